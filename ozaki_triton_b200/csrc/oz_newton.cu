// oz_newton.cu -- orthogonalisation of a batch of matrices by quintic
// Newton-Schulz steps on the tile engine (oz_tile.cuh).
//
//   X_0 = G / (|G|_F + eps)
//   S = X X^T,  P = b S + c S S,  X <- a X + P X          `steps` times
//
// for G with at most as many rows as columns; a tall G is worked on through
// its transpose (the polynomial is odd, so it commutes with transposing).
//
// Every matrix is held as fp16 slices at a power-of-two scale of its own:
// high = fp16(v 2^e), low = fp16(v 2^e - high).  The host bounds the norms
// step by step: the singular values start in [0, 1] and a step's polynomial
// is known, so their largest value after it is too; no data is looked at.  It
// is the bound of exact steps: rounded ones go a little beyond it, and a factor
// for that must not enter the next step's bound, since polynomials chosen for
// an interval may be steep just outside it (1/64 a step took the bound of one such
// schedule from 2 to 10^15 in 5 steps, and the matrices to zero).  Instead e puts the bound
// at 2^12, which leaves a factor of 16 below the largest fp16 and, two slices
// having 22 bits down to 2^-3, one of 2^15 above the entries that keep them all.  Schedules
// whose bound leaves [0, 8] before their last step are refused.
//
// With one slice the products use `high` alone (11 bits) and
// only the term a X keeps X's 22: that term carries the directions that the
// products hardly touch, and rounding it as well as P X makes both sides of
// the sum consistent only for full-rank G (measured on a low-rank gradient:
// 2.2e-2 with 11 bits there, 4.5e-4 with 22).  With two slices the products add
// high*high + high*low + low*high.  S and P are symmetric: only the tiles on
// and below the diagonal are multiplied, each written twice.
//
// 5 steps measured: 4096 x 4096 fp32 (two slices) 3.71 ms under lasting load, 1110 TFLOP/s
// of fp16 products (3.45 ms in short runs; 2.46 at the burst rate), bound by the tensor cores
// under the power limit and by 136 tiles of S and P for 74 pairs of CTAs; 4 x 2048 x 2816
// bf16 (one slice) 1.04 ms under lasting load (0.89 in short runs; 0.52 at the burst rate),
// bound by what the products and the epilogues' slices move between L2 and the SMs; up to
// 1000 or so rows the launches' length (17 of 7 us or more: 256 x 256 122 us, 300 x 1000
// 173, 1024 x 1024 261).  The pairs' tiles with passes hold 128 sums a thread under a cap of
// 168 registers and spill 108 to 172 bytes.

#include <algorithm>
#include <cmath>

#include "oz_tile.cuh"

namespace oz {
int status_newton(int *value, bool clear) { return read_status_word(value, clear); }

namespace {
using namespace tile;

constexpr int kMostPartials = 256;     // blocks that add the squares of a matrix

__device__ __forceinline__ float load_value(const void *p, int dtype, int64_t i) {
  if (dtype == OZ_F32) return static_cast<const float *>(p)[i];
  if (dtype == OZ_F16) return __half2float(static_cast<const __half *>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

// A matrix in slices: plane q of member z at base + (q * batch + z) * mat.
struct Planes {
  __half *base;
  int64_t ld, mat, plane;
  __device__ __half *at(int q, int z, int64_t row, int64_t column) const {
    return base + q * plane + z * mat + row * ld + column;
  }
};

struct InitParams {
  const void *g;
  int dtype, partials;
  bool flat, vectors;               // G's member is one run of elements; its lines start on 16-byte boundaries
  int rows, cols;                   // rows <= cols, after the transposition of a tall G
  int64_t g_sb, g_sr, g_sc;         // strides of G's member, and of X's rows and columns in G
  double *partial;                  // (batch, partials) sums of squares
  Planes x;
  double eps, scale;
};

// 8 elements of G as they are stored.
template <int DTYPE> struct Eight {
  static constexpr int kWords = DTYPE == OZ_F32 ? 8 : 4;
  uint32_t w[kWords];
  // from a 16-byte boundary, one after the other
  __device__ __forceinline__ void load(const void *p, int64_t i) {
    const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const char *>(p) + i * (kWords / 2));
#pragma unroll
    for (int x = 0; x < kWords / 4; ++x) {
      const uint4 a = *(q + x);
      w[4 * x] = a.x, w[4 * x + 1] = a.y, w[4 * x + 2] = a.z, w[4 * x + 3] = a.w;
    }
  }
  // the first `left`, `step` apart; the others are zero
  __device__ __forceinline__ void load(const void *p, int64_t i, int64_t step, int left) {
#pragma unroll
    for (int x = 0; x < kWords; ++x) w[x] = 0;
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (x < left) {
        if (DTYPE == OZ_F32) w[x % kWords] = *(static_cast<const uint32_t *>(p) + i + x * step);
        else w[x / 2 % kWords] |= (uint32_t)*(static_cast<const unsigned short *>(p) + i + x * step) << x % 2 * 16;
      }
  }
  __device__ __forceinline__ void floats(float (&v)[8]) const {
#pragma unroll
    for (int x = 0; x < kWords; ++x) {
      if (DTYPE == OZ_F32) {
        v[x] = __uint_as_float(w[x]);
        continue;
      }
      const float2 f = DTYPE == OZ_F16 ? __half22float2(*reinterpret_cast<const __half2 *>(&w[x]))
                                       : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w[x]));
      v[2 * x % 8] = f.x;
      v[(2 * x + 1) % 8] = f.y;
    }
  }
};

__device__ double block_sum(double sum, double *part) {
  for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = sum;
  __syncthreads();
  sum = 0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) sum += part[w];
  return sum;
}

// sum + the squares of 8 elements: in fp32 where neither an overflow nor the loss of
// small ones beside the largest can matter (a group's sum is then 2^-22 off at most),
// since conversions to fp64 are slow (46 MB of bf16 in 25 us with one an element), else
// in fp64.
template <int DTYPE> __device__ __forceinline__ double add_squares(double sum, const float (&v)[8]) {
  float most = 0.f;
#pragma unroll
  for (int x = 0; x < 8; ++x) most = fmaxf(most, fabsf(v[x]));
  if (DTYPE == OZ_F16 || (most >= 0x1p-40f && most <= 0x1p60f)) {
    const float a = fmaf(v[3], v[3], fmaf(v[2], v[2], fmaf(v[1], v[1], v[0] * v[0])));
    const float b = fmaf(v[7], v[7], fmaf(v[6], v[6], fmaf(v[5], v[5], v[4] * v[4])));
    return sum + (double)(a + b);
  }
#pragma unroll
  for (int x = 0; x < 8; ++x) sum += (double)v[x] * v[x];
  return sum;
}

// Sums of squares, held in fp64, each block a fixed part: the order of the sum does
// not depend on the launch.
template <int DTYPE> __global__ void __launch_bounds__(256) squares_kernel(const InitParams p) {
  __shared__ double part[8];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t base = blockIdx.y * p.g_sb, stride = (int64_t)gridDim.x * 256;
  double sum = 0;
  if (p.flat) {
    const int64_t pieces = (int64_t)p.rows * p.cols / 8;
    int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (; i < pieces; i += 4 * stride) {
      Eight<DTYPE> some[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + u * stride < pieces) some[u].load(p.g, base + (i + u * stride) * 8);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float v[8];
        some[u].floats(v);
        if (i + u * stride < pieces) sum = add_squares<DTYPE>(sum, v);
      }
    }
  } else {
    // a line at a time, consecutive threads along the smaller stride
    const bool across = p.g_sr < p.g_sc;
    const int inner = across ? p.rows : p.cols, outer = across ? p.cols : p.rows;
    const int64_t s_in = across ? p.g_sr : p.g_sc, s_out = across ? p.g_sc : p.g_sr;
    const int wide = inner >= 256 ? 256 : 32;                // threads of a line
    for (int o = blockIdx.x * (256 / wide) + threadIdx.x / wide; o < outer; o += gridDim.x * (256 / wide))
      for (int i = threadIdx.x % wide; i < inner; i += wide) {
        const double v = load_value(p.g, DTYPE, base + o * s_out + i * s_in);
        sum += v * v;
      }
  }
  sum = block_sum(sum, part);
  if (threadIdx.x == 0) p.partial[(int64_t)blockIdx.y * p.partials + blockIdx.x] = sum;
}

// X_0 in slices, 64 x 64 tiles: 8 elements at a time from G along its smaller
// stride, through shared memory where that is across X's rows, and 8 at a
// time to X along its rows (whose pitch is a multiple of 8).  A block takes many tiles,
// each one's elements on their way while the one before is written (a block for
// each tile added up the partial sums 5632 times for 4 x 2048 x 2816 bf16: 35 us, this 29).
template <int DTYPE> __global__ void __launch_bounds__(256, 6) normalise_kernel(const InitParams p) {
  __shared__ double part[8];
  __shared__ float tile[64][65];
  const bool across = p.g_sr < p.g_sc;
  const int64_t step = across ? p.g_sr : p.g_sc;
  const int wide = (p.cols + 63) / 64, tiles = wide * ((p.rows + 63) / 64);
  Eight<DTYPE> next[2];
  auto fetch = [&](int t) {
    const int r0 = t / wide * 64, c0 = t % wide * 64;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // line and piece of G's tile
      const int line = threadIdx.x / 8 + h * 32, u = threadIdx.x % 8 * 8;
      const int r = r0 + (across ? u : line), c = c0 + (across ? line : u);
      const int left = r >= p.rows || c >= p.cols ? 0 : across ? p.rows - r : p.cols - c;
      const int64_t at = blockIdx.z * p.g_sb + r * p.g_sr + c * p.g_sc;
      if (p.vectors && left >= 8) next[h].load(p.g, at);
      else next[h].load(p.g, at, step, left);
    }
  };
  if (blockIdx.x < tiles) fetch(blockIdx.x);
  asm volatile("griddepcontrol.wait;" ::: "memory");      // the partial sums

  double sum = 0;
  for (int i = threadIdx.x; i < p.partials; i += 256) sum += p.partial[(int64_t)blockIdx.z * p.partials + i];
  sum = block_sum(sum, part);
  // the scale as a float in [1, 2) and two powers of two, which together have its
  // range: the product with each element is rounded once (the scale itself 2^-24 off)
  __shared__ float factors[3];
  if (threadIdx.x == 0) {
    const double scale = sum == 0 && p.eps == 0 ? 0.0 : p.scale / (sqrt(sum) + p.eps);   // a zero matrix stays zero
    int e = 0;
    factors[0] = isfinite(scale) ? (float)(2 * frexp(scale, &e)) : (float)scale;
    e = max(-250, min(250, e - 1));
    factors[1] = (float)ldexp(1.0, e / 2);
    factors[2] = (float)ldexp(1.0, e - e / 2);
  }
  __syncthreads();
  const float f0 = factors[0], f1 = factors[1], f2 = factors[2];
  for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int line = threadIdx.x / 8 + h * 32, u = threadIdx.x % 8 * 8;
      float v[8];
      next[h].floats(v);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const float f = v[x] * f1 * f0 * f2;
        if (across) tile[u + x][line] = f;
        else tile[line][u + x] = f;
      }
    }
    __syncthreads();
    if (t + gridDim.x < tiles) fetch(t + gridDim.x);
    const int r0 = t / wide * 64, c0 = t % wide * 64;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = threadIdx.x / 8 + h * 32, u = threadIdx.x % 8 * 8;
      if (r0 + r >= p.rows || c0 + u >= p.cols) continue;
      uint32_t high[4], low[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float a = tile[r][u + 2 * x], b = tile[r][u + 2 * x + 1];
        const __half2 high2 = __floats2half2_rn(a, b);
        const float2 f = __half22float2(high2);
        high[x] = *reinterpret_cast<const uint32_t *>(&high2);
        low[x] = pack2<__half>(a - f.x, b - f.y);
      }
      *reinterpret_cast<uint4 *>(p.x.at(0, blockIdx.z, r0 + r, c0 + u)) = make_uint4(high[0], high[1], high[2], high[3]);
      *reinterpret_cast<uint4 *>(p.x.at(1, blockIdx.z, r0 + r, c0 + u)) = make_uint4(low[0], low[1], low[2], low[3]);
    }
    __syncthreads();
  }
}

struct StepParams {
  uint32_t idesc;
  int batch, rows, cols, k;         // of the result; terms of the contraction
  int row_tiles, column_tiles, tiles;   // tiles of one member
  float alpha, beta;                // result = alpha * in + beta * accumulator
  Planes in, out;
  // S of few rows and many columns: `parts` CTAs a tile, each `part_blocks` blocks of
  // the contraction, whose sums go to partial (parts, batch, rows, part_ld)
  int parts, part_blocks;
  int64_t part_ld;
  float *partial;
  // the last step's result instead of `out`: element (z, r, c) of the type
  void *last;
  int last_dtype;
  int64_t last_sb, last_sr, last_sc;
  bool last_vectors;                // its rows start on 16-byte boundaries
};

// 32 rows x 32 fp16 columns: each lane 4 pieces of 8 columns, 64 bytes of a
// row by 4 lanes; the warp's staging turns them into each lane's own row.
struct Chunk { uint4 piece[4]; };

__device__ __forceinline__ void fetch(const __half *src, int64_t ld, int rows, int cols, Chunk &v) {
  const int lane = threadIdx.x % 32;
  const __half *from = src + (lane / 4) * ld + (lane % 4) * 8;
  if (rows >= 32 && cols >= 32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v.piece[i] = *reinterpret_cast<const uint4 *>(from + i * 8 * ld);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v.piece[i] = i * 8 + lane / 4 < rows && lane % 4 * 8 < cols
                       ? *reinterpret_cast<const uint4 *>(from + i * 8 * ld)
                       : make_uint4(0, 0, 0, 0);
  }
}
__device__ __forceinline__ void to_rows(unsigned char *mine, Chunk &v) {
  const int lane = threadIdx.x % 32;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) *staged(mine, i * 8 + lane / 4, lane % 4) = v.piece[i];
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 4; ++u) v.piece[u] = *staged(mine, lane, u);
}

// The way back: the chunk in the staging to memory.
__device__ __forceinline__ void flush(unsigned char *mine, __half *dst, int64_t ld, int rows, int cols) {
  const int lane = threadIdx.x % 32;
  __half *to = dst + (lane / 4) * ld + (lane % 4) * 8;
  __syncwarp();
  if (rows >= 32 && cols >= 32) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<uint4 *>(to + i * 8 * ld) = *staged(mine, i * 8 + lane / 4, lane % 4);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i * 8 + lane / 4 < rows && lane % 4 * 8 < cols)
        *reinterpret_cast<uint4 *>(to + i * 8 * ld) = *staged(mine, i * 8 + lane / 4, lane % 4);
  }
  __syncwarp();
}
// From each lane's row; and its mirror image, from each lane's column.
__device__ __forceinline__ void store_rows(unsigned char *mine, __half *dst, int64_t ld, int rows, int cols,
                                           const uint4 (&v)[4]) {
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 4; ++u) *staged(mine, threadIdx.x % 32, u) = v[u];
  flush(mine, dst, ld, rows, cols);
}
__device__ __forceinline__ void store_columns(unsigned char *mine, __half *dst, int64_t ld, int rows, int cols,
                                              const uint4 (&v)[4]) {
  const int lane = threadIdx.x % 32;
  const __half *h = reinterpret_cast<const __half *>(&v[0]);
#pragma unroll
  for (int x = 0; x < 32; ++x) reinterpret_cast<__half *>(staged(mine, x, lane / 8))[lane % 8] = h[x];
  flush(mine, dst, ld, rows, cols);
}

// The part of `in` under chunk c of the warp's columns, IN slices.
template <int IN>
__device__ __forceinline__ void fetch_in(const StepParams &p, int z, int row, int column, Chunk (&v)[IN + !IN]) {
#pragma unroll
  for (int q = 0; q < IN; ++q)
    fetch(p.in.at(q, z, row, column), p.in.ld, p.rows - row, p.cols - column, v[q]);
}

// alpha * in + beta * accumulator for 32 columns of the lane's row.
template <int IN, class Source>
__device__ __forceinline__ void combine(const StepParams &p, const Source &source, int c, unsigned char *mine,
                                        Chunk (&in)[IN + !IN], float (&v)[32]) {
#pragma unroll
  for (int h = 0; h < 32; h += 16) {
    float acc[16];
    source.read(c + h, acc);
#pragma unroll
    for (int x = 0; x < 16; ++x) v[h + x] = p.beta * acc[x];
  }
#pragma unroll
  for (int q = 0; q < IN; ++q) {
    to_rows(mine, in[q]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const __half2 *h = reinterpret_cast<const __half2 *>(&in[q].piece[u]);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float2 f = __half22float2(h[x]);
        v[u * 8 + x * 2] += p.alpha * f.x;
        v[u * 8 + x * 2 + 1] += p.alpha * f.y;
      }
    }
  }
}

__device__ __forceinline__ void slices_of(const float (&v)[32], uint4 (&high)[4], uint4 (&low)[4]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float a = v[u * 8 + x * 2], b = v[u * 8 + x * 2 + 1];
      const __half2 hh = __floats2half2_rn(a, b);
      const float2 f = __half22float2(hh);
      h[x] = *reinterpret_cast<const uint32_t *>(&hh);
      l[x] = pack2<__half>(a - f.x, b - f.y);
    }
    high[u] = make_uint4(h[0], h[1], h[2], h[3]);
    low[u] = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

struct StepTile { int z, row, column; bool mirror; };

// S = X X^T (IN 0) and P = b S + c S S (IN slices of S): tiles (i, j) on and
// below the diagonal, the others their mirror images.
template <int PAIR_, int NT_, int PLANES_, int IN, int PASS_> struct SymmetricJob {
  static constexpr int PAIR = PAIR_, NT = NT_, PLANES = PLANES_, PASS = PASS_;
  static constexpr bool AMN = false, BMN = false, RAGGED = false, VARIABLE = false;
  static constexpr int R = kRows * PAIR / NT;           // column tiles as wide as a tile is high
  using Params = StepParams;
  using Extra = StepTile;
  static __device__ int plane_stride(const Params &p) { return p.batch; }
  // The first chunk of `in` is fetched before the accumulators are there and
  // each next one before the one in hand is used (passes need the registers).
  struct Ahead { Chunk in[IN + !IN]; };
  template <class Tile>
  static __device__ void look_ahead(const Params &p, const Tile &t, int row, int column, Ahead &early) {
    if (PASS == 0 && t.extra.row + row < p.rows && t.extra.column + column < p.cols)
      fetch_in<IN>(p, t.extra.z, t.extra.row + row, t.extra.column + column, early.in);
  }
  struct Walk {
    __device__ Walk(const Params &) {}
    __device__ bool find(const Params &p, int t, TileOf<Extra> &tile) {
      const int z = t / p.tiles, local = t - z * p.tiles;
      if (z >= p.batch) return false;
      // rows of tiles 0 .. i-1 hold R i (i + 1) / 2 tiles
      int i = (int)((sqrtf(8.f * (float)(local / R) + 1.f) - 1.f) * 0.5f);
      while (R * (i + 1) * (i + 2) / 2 <= local) ++i;
      while (R * i * (i + 1) / 2 > local) --i;
      const int j = local - R * i * (i + 1) / 2;
      tile.a_row = i * kRows * PAIR;
      tile.b_row = j * NT;
      tile.a_mat = tile.b_mat = z;
      tile.k_begin = 0;
      tile.k_len = p.k;
      tile.extra = StepTile{z, tile.a_row, tile.b_row, j < R * i};
      return true;
    }
  };
  template <class Source>
  static __device__ void epilogue(const Params &p, const TileOf<Extra> &t, const Source &source, int row,
                                  int column, unsigned char *mine, Ahead &early) {
    const int r0 = t.extra.row + row, rows = p.rows - r0;
    if (rows <= 0) return;
#pragma unroll
    for (int c = 0; c < NT / 2; c += 32) {
      const int c0 = t.extra.column + column + c, cols = p.cols - c0;
      if (cols <= 0) continue;
      float v[32];
      Chunk in[IN + !IN];
      if constexpr (PASS == 0) {
#pragma unroll
        for (int q = 0; q < IN; ++q) in[q] = early.in[q];
        if (c + 32 < NT / 2 && cols > 32) fetch_in<IN>(p, t.extra.z, r0, c0 + 32, early.in);
      } else {
        fetch_in<IN>(p, t.extra.z, r0, c0, in);
      }
      combine<IN>(p, source, c, mine, in, v);
      uint4 high[4], low[4];
      slices_of(v, high, low);
      store_rows(mine, p.out.at(0, t.extra.z, r0, c0), p.out.ld, rows, cols, high);
      if constexpr (PLANES == 2)
        store_rows(mine, p.out.at(1, t.extra.z, r0, c0), p.out.ld, rows, cols, low);
      if (t.extra.mirror) {
        store_columns(mine, p.out.at(0, t.extra.z, c0, r0), p.out.ld, cols, rows, high);
        if constexpr (PLANES == 2)
          store_columns(mine, p.out.at(1, t.extra.z, c0, r0), p.out.ld, cols, rows, low);
      }
    }
  }
  static __device__ void finish(const Params &, int, int) {}
};

// S of few rows and many columns: the same tiles, each with a part of the
// contraction; its sums are left to add_parts_kernel.
template <int PLANES, int PASS> struct PartsJob : SymmetricJob<1, 64, PLANES, 0, PASS> {
  using Whole = SymmetricJob<1, 64, PLANES, 0, PASS>;
  using typename Whole::Params;
  using typename Whole::Extra;
  using typename Whole::Ahead;
  struct Walk : Whole::Walk {
    __device__ Walk(const Params &p) : Whole::Walk(p) {}
    __device__ bool find(const Params &p, int t, TileOf<Extra> &tile) {
      const int part = t / (p.tiles * p.batch);
      if (part >= p.parts || !Whole::Walk::find(p, t - part * p.tiles * p.batch, tile)) return false;
      tile.k_begin = (int64_t)part * p.part_blocks * kBlock;
      tile.k_len = min((int64_t)p.part_blocks * kBlock, p.k - tile.k_begin);
      tile.extra.z += part * p.batch;
      return true;
    }
  };
  template <class Source>
  static __device__ void epilogue(const Params &p, const TileOf<Extra> &t, const Source &source, int row,
                                  int column, unsigned char *mine, Ahead &) {
    const int r0 = t.extra.row + row, c0 = t.extra.column + column;
    if (r0 < p.rows && c0 < p.cols)
      write_rows<float, 32>(source, mine, p.partial + ((int64_t)t.extra.z * p.rows + r0) * p.part_ld + c0,
                            p.part_ld, p.rows - r0, p.cols - c0, true);
  }
};

// The parts of S added up in their order, sliced, and mirrored: 32 x 32 tiles on
// and below the diagonal.
__global__ void __launch_bounds__(256) add_parts_kernel(const StepParams p, int planes) {
  __shared__ float tile[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32, z = blockIdx.z;
  if (c0 > r0) return;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  for (int i = warp; i < 32; i += 8) {
    float sum = 0.f;
    // above the diagonal of a diagonal tile: the element below it (both are there)
    const int r = max(r0 + i, c0 + lane), c = min(r0 + i, c0 + lane);
    if (r < p.rows)
      for (int part = 0; part < p.parts; ++part)
        sum += p.partial[((int64_t)(part * p.batch + z) * p.rows + r) * p.part_ld + c];
    tile[i][lane] = p.beta * sum;
  }
  __syncthreads();
  for (int i = warp; i < 32; i += 8) {
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int r = (side ? c0 : r0) + i, c = (side ? r0 : c0) + lane;
      if (r >= p.rows || c >= p.rows || (side && r0 == c0)) continue;
      const float v = side ? tile[lane][i] : tile[i][lane];
      const __half high = __float2half_rn(v);
      *p.out.at(0, z, r, c) = high;
      if (planes == 2) *p.out.at(1, z, r, c) = __float2half_rn(v - __half2float(high));
    }
  }
}

// X <- a X + P X: A is the rows of P, B the columns of X.
template <int PAIR_, int NT_, int PLANES_, int PASS_> struct UpdateJob {
  static constexpr int IN = 2;
  static constexpr int PAIR = PAIR_, NT = NT_, PLANES = PLANES_, PASS = PASS_;
  static constexpr bool AMN = false, BMN = true, RAGGED = false, VARIABLE = false;
  using Params = StepParams;
  using Extra = StepTile;
  static __device__ int plane_stride(const Params &p) { return p.batch; }
  // The first chunk of `in` is fetched before the accumulators are there and
  // each next one before the one in hand is used (passes need the registers).
  struct Ahead { Chunk in[IN + !IN]; };
  template <class Tile>
  static __device__ void look_ahead(const Params &p, const Tile &t, int row, int column, Ahead &early) {
    if (PASS == 0 && t.extra.row + row < p.rows && t.extra.column + column < p.cols)
      fetch_in<IN>(p, t.extra.z, t.extra.row + row, t.extra.column + column, early.in);
  }
  struct Walk {
    __device__ Walk(const Params &) {}
    __device__ bool find(const Params &p, int t, TileOf<Extra> &tile) {
      const int z = t / p.tiles, local = t - z * p.tiles;
      if (z >= p.batch) return false;
      const int sweep = local / (8 * p.column_tiles), in = local - sweep * 8 * p.column_tiles;
      const int size = min(p.row_tiles - sweep * 8, 8);
      tile.a_row = (sweep * 8 + in % size) * kRows * PAIR;
      tile.b_row = in / size * NT;
      tile.a_mat = tile.b_mat = z;
      tile.k_begin = 0;
      tile.k_len = p.k;
      tile.extra = StepTile{z, tile.a_row, tile.b_row, false};
      return true;
    }
  };
  template <class Source>
  static __device__ void epilogue(const Params &p, const TileOf<Extra> &t, const Source &source, int row,
                                  int column, unsigned char *mine, Ahead &early) {
    const int r0 = t.extra.row + row, rows = p.rows - r0, lane = threadIdx.x % 32;
    if (rows <= 0) return;
#pragma unroll
    for (int c = 0; c < NT / 2; c += 32) {
      const int c0 = t.extra.column + column + c, cols = p.cols - c0;
      if (cols <= 0) continue;
      float v[32];
      Chunk in[IN + !IN];
      if constexpr (PASS == 0) {
#pragma unroll
        for (int q = 0; q < IN; ++q) in[q] = early.in[q];
        if (c + 32 < NT / 2 && cols > 32) fetch_in<IN>(p, t.extra.z, r0, c0 + 32, early.in);
      } else {
        fetch_in<IN>(p, t.extra.z, r0, c0, in);
      }
      combine<IN>(p, source, c, mine, in, v);
      if (!p.last) {
        uint4 high[4], low[4];
        slices_of(v, high, low);
        store_rows(mine, p.out.at(0, t.extra.z, r0, c0), p.out.ld, rows, cols, high);
        store_rows(mine, p.out.at(1, t.extra.z, r0, c0), p.out.ld, rows, cols, low);
      } else {
        // the result: through the staging where it is stored along the rows,
        // from the lanes where it is stored across them
        const int64_t at = t.extra.z * p.last_sb + r0 * p.last_sr + c0 * p.last_sc;
        float *out32 = static_cast<float *>(p.last) + at;
        __half *out16 = static_cast<__half *>(p.last) + at;   // or bf16: 2 bytes either way
        const bool wide = p.last_dtype == OZ_F32;
        auto bits = [&](float f) {
          return p.last_dtype == OZ_F16 ? __float2half_rn(f)
                                        : __ushort_as_half(__bfloat16_as_ushort(__float2bfloat16_rn(f)));
        };
        if (p.last_sr == 1) {
          if (lane < rows) {
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (x < cols) {
                if (wide) out32[lane + x * p.last_sc] = v[x];
                else out16[lane + x * p.last_sc] = bits(v[x]);
              }
          }
        } else if (p.last_vectors) {
          // 64 bytes of a row at a time (4 x 2048 x 2816 bf16: the last product 105 us with single elements,
          // 83 so)
          uint4 w[4];
          if (wide) {
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
#pragma unroll
              for (int u = 0; u < 4; ++u) w[u] = *reinterpret_cast<const uint4 *>(&v[h + u * 4]);
              store_rows(mine, reinterpret_cast<__half *>(out32 + h), 2 * p.last_sr, rows, 2 * (cols - h), w);
            }
          } else {
            __half h[32];
#pragma unroll
            for (int x = 0; x < 32; ++x) h[x] = bits(v[x]);
#pragma unroll
            for (int u = 0; u < 4; ++u) w[u] = *reinterpret_cast<const uint4 *>(&h[u * 8]);
            store_rows(mine, out16, p.last_sr, rows, cols, w);
          }
        } else {
#pragma unroll
          for (int h = 0; h < 32; h += 16) {
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 4; ++u)
              *staged(mine, lane, u) = *reinterpret_cast<const uint4 *>(&v[h + u * 4]);
            __syncwarp();
#pragma unroll 4
            for (int r = lane / 16; r < 32; r += 2)
              if (r < rows && h + lane % 16 < cols) {
                const float f = reinterpret_cast<const float *>(staged(mine, r, lane % 16 / 4))[lane % 4];
                const int64_t to = r * p.last_sr + h + lane % 16;
                if (wide) out32[to] = f;
                else out16[to] = bits(f);
              }
          }
        }
      }
    }
  }
  static __device__ void finish(const Params &, int, int) {}
};

// ---------------------------------------------------------------------------
// small matrices: all steps in one launch
// ---------------------------------------------------------------------------
// 17 launches of products that take a microsecond each cost 85 us for 12
// matrices of 64 x 250; here a cluster of up to 8 CTAs keeps one matrix in
// shared memory in fp32, a panel of X's columns in each CTA and S and P in
// all of them: the panels' X X^T are added in the order of the ranks, P is
// computed a few rows a CTA and handed to the others, and a X + P X needs
// nothing of another panel.  fp32 FMAs are enough here (and rounded sums more
// exact than the tensor core's): a step of 64 x 250 is 0.23 M FMAs a CTA.  12 of
// them take 44 us, one of 16 x 16 13: barriers, exchanges and the latency of each part.
constexpr int kSmallRows = 128;
constexpr int kSmallThreads = 256;
constexpr int kMicro = 4;                // rows and columns of a thread's tile

struct SmallParams {
  const void *g;
  void *out;
  int dtype, rows, cols, panel;     // columns of a CTA, a multiple of 4
  int steps;
  int x_ld, s_ld;                   // pitches in shared memory: odd multiples of 4 floats
  int64_t g_sb, g_sr, g_sc, o_sb, o_sr, o_sc;
  double eps;
  float abc[3 * 16];
};
constexpr int kSmallSteps = 16;

__device__ __forceinline__ float4 peer_load(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}
__device__ __forceinline__ void peer_store(uint32_t addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z),
               "f"(v.w)
               : "memory");
}

// 4 x 4 tile of sum over k of a[k][i] b[k][j], k = first, first + step, ..
__device__ __forceinline__ void tile_along(const float *a, int lda, const float *b, int ldb, int first, int step,
                                           int n, float (&acc)[kMicro][kMicro]) {
#pragma unroll 4
  for (int k = first; k < n; k += step) {
    const float4 u = *reinterpret_cast<const float4 *>(a + k * lda), w = *reinterpret_cast<const float4 *>(b + k * ldb);
    const float x[4] = {u.x, u.y, u.z, u.w}, y[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < kMicro; ++i)
#pragma unroll
      for (int j = 0; j < kMicro; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
  }
}

// log2 of the threads (up to 8) that share the terms of a tile when there are fewer
// tiles than threads.
__device__ __forceinline__ int sharing(int tiles) {
  static_assert(kSmallThreads == 256, "the limits below");
  return tiles <= 32 ? 3 : tiles <= 64 ? 2 : tiles <= 128 ? 1 : 0;
}

__device__ __forceinline__ void add_shared(float (&acc)[kMicro][kMicro], int log) {
  for (int o = 1; o < 1 << log; o *= 2)
#pragma unroll
    for (int i = 0; i < kMicro; ++i)
#pragma unroll
      for (int j = 0; j < kMicro; ++j) acc[i][j] += __shfl_xor_sync(0xffffffffu, acc[i][j], o);
}

__global__ void __launch_bounds__(kSmallThreads, 1) small_kernel(const SmallParams p) {
  extern __shared__ __align__(16) float smem_f[];
  __shared__ double norms[8], part[kSmallThreads / 32];
  const int ranks = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
  const int tid = threadIdx.x;
  const int member = blockIdx.x / ranks;
  // another CTA's shared memory may be used once that CTA is known to have started:
  // waited for below, before the first remote store
  if (ranks > 1) cluster_arrive_relaxed();
  auto together = [&]() {
    if (ranks > 1) cluster_sync();
    else __syncthreads();
  };
  const int rm = (p.rows + kMicro - 1) / kMicro * kMicro;           // rows, padded with zeros
  float *x = smem_f, *s = x + rm * p.x_ld, *q = s + rm * p.s_ld;   // q: partial S, then P
  const int c0 = rank * p.panel, width = max(0, min(p.panel, p.cols - c0));

  // X = G's panel, its squares, and zeros around it
  double sum = 0;
  const bool across = p.g_sr < p.g_sc;                  // G is stored along X's columns
  const int inner = across ? p.rows : width, outer = across ? width : p.rows;
  const int64_t from = member * p.g_sb + c0 * p.g_sc;
  for (int i = tid; i < rm * p.x_ld; i += kSmallThreads) x[i] = 0.f;
  __syncthreads();
  if (inner > 0) {
    const int per = inner >= 256 ? 256 : inner >= 128 ? 128 : inner >= 64 ? 64 : inner >= 32 ? 32 : 16;
    for (int o = tid / per; o < outer; o += kSmallThreads / per)
      for (int i = tid % per; i < inner; i += per) {
        const int r = across ? i : o, c = across ? o : i;
        const float v = load_value(p.g, p.dtype, from + r * p.g_sr + c * p.g_sc);
        sum += (double)v * v;
        x[r * p.x_ld + c] = v;
      }
  }
  sum = block_sum(sum, part);
  if (ranks > 1) cluster_wait();
  if (tid < ranks) {
    const uint32_t to = map_to_cta(smem_u32(&norms[rank]), (uint32_t)tid);
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(sum) : "memory");
  }
  together();
  sum = 0;
  for (int r = 0; r < ranks; ++r) sum += norms[r];
  const double scale = sum == 0 && p.eps == 0 ? 0.0 : 1.0 / (sqrt(sum) + p.eps);
  for (int i = tid; i < rm * p.x_ld; i += kSmallThreads) x[i] = (float)(x[i] * scale);
  __syncthreads();

  // What does not change from step to step is computed here: a step of a small
  // matrix is bound by latencies, and divisions by variables have long ones
  // (12 matrices of 64 x 250: 8.0 us a step with them in it, 7.1 so).
  const int side = rm / kMicro;
  const uint32_t inverse = ((1u << 20) + side - 1) / side;
  auto by_side = [&](int v) { return (int)((uint32_t)v * inverse >> 20); };   // v / side for v < 2^20 / side
  auto below = [&](int t, int &i, int &j) {                 // tile t on and below the diagonal
    i = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    j = t - i * (i + 1) / 2;
  };
  const int slice = (side + ranks - 1) / ranks * kMicro;    // rows of S and P that this CTA makes
  const int first = min(rank * slice, rm), last = min(first + slice, rm);
  const int s_tiles = side * (side + 1) / 2, p_tiles = (last - first) / kMicro * side;
  const int p_log = sharing(p_tiles), x_log = sharing(side * (p.panel / kMicro));
  const int abreast = by_side(kSmallThreads >> x_log);      // column tiles of a round of the update
  const int x_column = by_side(tid >> x_log), x_row = (tid >> x_log) - x_column * side;
  int first_i, first_j;
  below(tid >> sharing(s_tiles), first_i, first_j);
  for (int step = 0; step < p.steps; ++step) {
    const float a = p.abc[3 * step], b = p.abc[3 * step + 1], c = p.abc[3 * step + 2];
    // This panel's X X^T, tiles on and below the diagonal and their mirror images; a
    // tile takes every side-th row, so that the threads of a warp read neighbouring
    // rows (whose pitch is odd: no bank conflicts).  One CTA's is S itself.
    float *sums = ranks > 1 ? q : s;
    for (int t0 = 0; t0 < s_tiles;) {
      const int log = sharing(s_tiles - t0), kq = tid & ((1 << log) - 1), t = t0 + (tid >> log);
      int ti = first_i, tj = first_j;
      if (t0) below(t, ti, tj);
      float acc[kMicro][kMicro] = {};
      if (t < s_tiles) {
        const float *xi = x + ti * p.x_ld, *xj = x + tj * p.x_ld;
        for (int k = kq * 4; k < p.panel; k += 4 << log) {
          float4 u[kMicro], w[kMicro];
#pragma unroll
          for (int i = 0; i < kMicro; ++i) {
            u[i] = *reinterpret_cast<const float4 *>(xi + i * side * p.x_ld + k);
            w[i] = *reinterpret_cast<const float4 *>(xj + i * side * p.x_ld + k);
          }
#pragma unroll
          for (int i = 0; i < kMicro; ++i)
#pragma unroll
            for (int j = 0; j < kMicro; ++j)
              acc[i][j] = fmaf(u[i].w, w[j].w, fmaf(u[i].z, w[j].z, fmaf(u[i].y, w[j].y, fmaf(u[i].x, w[j].x, acc[i][j]))));
        }
      }
      add_shared(acc, log);
      if (t < s_tiles && kq == 0)
#pragma unroll
        for (int i = 0; i < kMicro; ++i)
#pragma unroll
          for (int j = 0; j < kMicro; ++j) {
            sums[(ti + i * side) * p.s_ld + tj + j * side] = acc[i][j];
            sums[(tj + j * side) * p.s_ld + ti + i * side] = acc[i][j];
          }
      t0 += kSmallThreads >> log;
    }
    together();
    if (ranks > 1) {
      // S, rows [first, last) of it here, for everyone
      for (int v = tid; v < (last - first) * side; v += kSmallThreads) {
        const int row = by_side(v), at = (first + row) * p.s_ld + (v - row * side) * 4;
        const uint32_t from_q = smem_u32(q + at), to_s = smem_u32(s + at);
        float4 o[8], f = make_float4(0.f, 0.f, 0.f, 0.f);   // all on their way before the first is used
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < ranks) o[r] = peer_load(map_to_cta(from_q, (uint32_t)r));
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < ranks) f.x += o[r].x, f.y += o[r].y, f.z += o[r].z, f.w += o[r].w;
        for (int r = 0; r < ranks; ++r) peer_store(map_to_cta(to_s, (uint32_t)r), f);
      }
      cluster_sync();
    }
    // the same rows of P = b S + c S S
    for (int t0 = 0; t0 < p_tiles; t0 += kSmallThreads >> p_log) {
      const int kq = tid & ((1 << p_log) - 1), t = t0 + (tid >> p_log), row = by_side(t);
      const int i0 = first + row * kMicro, j0 = (t - row * side) * kMicro;
      float acc[kMicro][kMicro] = {};
      if (t < p_tiles) tile_along(s + i0, p.s_ld, s + j0, p.s_ld, kq, 1 << p_log, rm, acc);
      add_shared(acc, p_log);
      if (t < p_tiles && kq == 0)
#pragma unroll
        for (int i = 0; i < kMicro; ++i) {
          const int at = (i0 + i) * p.s_ld + j0;
          const float4 o = *reinterpret_cast<const float4 *>(s + at);
          const float4 f = make_float4(b * o.x + c * acc[i][0], b * o.y + c * acc[i][1], b * o.z + c * acc[i][2],
                                       b * o.w + c * acc[i][3]);
          if (ranks == 1) {
            *reinterpret_cast<float4 *>(q + at) = f;
          } else {
            const uint32_t to = smem_u32(q + at);
            for (int r = 0; r < ranks; ++r) peer_store(map_to_cta(to, (uint32_t)r), f);
          }
        }
    }
    together();
    // X <- a X + P X, the columns of a round from registers once all have read them
    const int kq = tid & ((1 << x_log) - 1);
    for (int base = 0; base < p.panel; base += abreast * kMicro) {
      const int i0 = x_row * kMicro, j0 = base + x_column * kMicro;
      const bool mine = x_column < abreast && j0 < p.panel;
      float acc[kMicro][kMicro] = {};
      if (mine) tile_along(q + i0, p.s_ld, x + j0, p.x_ld, kq, 1 << x_log, rm, acc);
      add_shared(acc, x_log);
      __syncthreads();
      if (mine && kq == 0)
#pragma unroll
        for (int i = 0; i < kMicro; ++i) {
          float4 *at = reinterpret_cast<float4 *>(x + (i0 + i) * p.x_ld + j0);
          const float4 o = *at;
          *at = make_float4(fmaf(a, o.x, acc[i][0]), fmaf(a, o.y, acc[i][1]), fmaf(a, o.z, acc[i][2]),
                            fmaf(a, o.w, acc[i][3]));
        }
    }
    __syncthreads();
  }

  const int64_t to = member * p.o_sb + c0 * p.o_sc;
  const bool rows_in = p.o_sr < p.o_sc;                 // the result is stored along X's columns
  const int o_inner = rows_in ? p.rows : width, all = p.rows * width;
  for (int i = tid; i < all; i += kSmallThreads) {
    const int r = rows_in ? i % o_inner : i / o_inner, cc = rows_in ? i / o_inner : i % o_inner;
    const float v = x[r * p.x_ld + cc];
    const int64_t at = to + r * p.o_sr + cc * p.o_sc;
    if (p.dtype == OZ_F32) static_cast<float *>(p.out)[at] = v;
    else if (p.dtype == OZ_F16) static_cast<__half *>(p.out)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(v);
  }
}

// CTAs of a small matrix's cluster, 0 where the tiles of the general path are
// expected to be faster.  Cycles of a step: the FMAs of a CTA at 46 a cycle
// (shared memory feeds no more of these 4 x 4 tiles); 3500 for barriers and
// sums; with a cluster 2500 more and the exchange of S and P, which both slow down
// once many clusters are there.  The general path takes about 40,000 whatever its size
// here.  Measured, cycles a step with 1, 2, 4, 8 CTAs: 16 x 16 3769, 5683, 6367, 6584;
// 64 x 250 41637, 25490, 16577, 13215, and 37 of them 41659, 25608, 25799, 38276;
// 128 x 128 92266, 54462, 34929, 28684.
struct SmallShape { int ranks, panel, x_ld, s_ld, bytes; };
SmallShape small_shape(int64_t batch, int64_t rows, int64_t cols, int steps) {
  SmallShape best{};
  if (rows > kSmallRows || steps > kSmallSteps || batch > 4096) return best;
  double least = 40000;
  for (int ranks = 1; ranks <= 8; ranks *= 2) {
    const int64_t rm = (rows + 3) / 4 * 4, panel = ((cols + ranks - 1) / ranks + 3) / 4 * 4;
    auto odd = [](int64_t n) { return n / 4 % 2 ? n : n + 4; };
    const int64_t x_ld = odd(panel), s_ld = odd(rm), bytes = 4 * rm * (x_ld + 2 * s_ld);
    if (bytes > 220 * 1024) continue;
    const double fmas = (double)rm * rm * (1.5 * panel) + (double)rm * rm * rm / ranks;
    const int64_t waves = (batch * ranks + sm_count() - 1) / sm_count();
    const double crowd = std::max(1.0, (double)(batch * ranks) * (batch * ranks) / (80.0 * 80.0));
    const double exchange = ranks > 1 ? (2500 + 0.6 * rm * rm) * std::min(crowd, 3.0) : 0;
    const double t = (double)waves * (fmas / 46 + 3500 + exchange);
    if (t < least) {
      least = t;
      best = SmallShape{ranks, (int)panel, (int)x_ld, (int)s_ld, (int)bytes};
    }
  }
  return best;
}

int run_small(const SmallShape &shape, SmallParams p, int64_t batch, cudaStream_t st) {
  p.panel = shape.panel;
  p.x_ld = shape.x_ld;
  p.s_ld = shape.s_ld;
  auto kernel = small_kernel;
  if (int rc = set_smem_once((const void *)kernel, shape.bytes, "small_kernel shared memory")) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * shape.ranks));
  cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = shape.bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = shape.ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, p), "small_kernel launch");
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
int64_t pitch(int64_t n) { return (n + 7) / 8 * 8; }

// Workspace of a call: sums of squares, two X's, S and P in slices.
struct Layout {
  int64_t rows, cols, x_mat, s_mat, x0, x1, s, p, partial, total;
  int parts, part_blocks;           // of S's contraction
};
int64_t member_tiles(bool symmetric, int64_t rows, int64_t cols, int high, int wide);
bool use_pairs(bool symmetric, int64_t batch, int64_t rows, int64_t cols);
Layout layout(int64_t batch, int64_t m, int64_t n, int splits) {
  Layout l{};
  l.rows = m < n ? m : n;
  l.cols = m < n ? n : m;
  l.x_mat = l.rows * pitch(l.cols);
  l.s_mat = l.rows * pitch(l.rows);
  int64_t at = align256(batch * kMostPartials * 8);
  const int64_t x = align256(2 * batch * l.x_mat * 2), s = align256(splits * batch * l.s_mat * 2);
  l.x0 = at;
  l.x1 = l.x0 + x;
  l.s = l.x1 + x;
  l.p = l.s + s;
  l.partial = l.p + s;
  // S of few rows: parts of at least 8 blocks on the SMs that its tiles leave idle
  // (68 x 3686, 5 matrices: 309 us a call in one part, 178 in 10)
  const int64_t blocks = (l.cols + kBlock - 1) / kBlock;
  int64_t parts = 1;
  if (batch && l.rows && blocks >= 32 && !use_pairs(true, batch, l.rows, l.rows))
    parts = std::max<int64_t>(
        1, std::min<int64_t>({16, sm_count() / (batch * member_tiles(true, l.rows, l.rows, 128, 64)), blocks / 8}));
  l.part_blocks = (int)((blocks + parts - 1) / parts);
  l.parts = (int)((blocks + l.part_blocks - 1) / std::max(l.part_blocks, 1));  // none is empty
  l.total = l.partial + (l.parts > 1 ? align256(l.parts * batch * l.rows * pitch(l.rows) * 4) : 0);
  return l;
}

// The exponent that puts a bound on a matrix's entries at 2^12.  Past 100 (a bound below
// 2^-88) the entries sink below fp16's; the other end is not reached (bounded_steps).
int exponent(double bound) {
  if (!(bound > 0)) return 12;
  int e;
  frexp(bound, &e);                                    // bound <= 2^e
  return std::min(std::max(12 - e, -100), 100);
}

// Largest |a s + b s^3 + c s^5| for s in [0, most], and |b u + c u^2| for u = s^2.
double largest_value(double a, double b, double c, double most) {
  auto f = [&](double s) { return std::fabs(s * (a + s * s * (b + s * s * c))); };
  double v = f(most);
  const double disc = 9 * b * b - 20 * a * c;          // a + 3 b u + 5 c u^2 = 0
  if (c != 0 && disc >= 0)
    for (int sign = -1; sign <= 1; sign += 2) {
      const double u = (-3 * b + sign * std::sqrt(disc)) / (10 * c);
      if (u > 0 && u < most * most) v = std::max(v, f(std::sqrt(u)));
    }
  if (c == 0 && b != 0 && -a / (3 * b) > 0 && -a / (3 * b) < most * most)
    v = std::max(v, f(std::sqrt(-a / (3 * b))));
  return v;
}
double largest_poly(double b, double c, double most) {
  auto f = [&](double u) { return std::fabs(u * (b + u * c)); };
  const double end = most * most;
  double v = f(end);
  if (c != 0 && -b / (2 * c) > 0 && -b / (2 * c) < end) v = std::max(v, f(-b / (2 * c)));
  return v;
}

// Whether the slices can hold every matrix of the steps: S grows with the square of the
// bound and P with its fourth power, while their entries may stay near 1, so X's bound
// before a step may be 8 at most (P's entries then still lie 2^12 above the 2^-12 that
// costs them bits), and P's 2^60.
constexpr double kMostNorm = 8, kMostPoly = 0x1p60;
constexpr double kFirstNorm = 1 + 1e-6;                // of X = G / (|G| + eps)
int bounded_steps(int steps, const double *coefficients) {
  double most = kFirstNorm;
  for (int i = 0; i < steps; ++i) {
    const double a = coefficients[3 * i], b = coefficients[3 * i + 1], c = coefficients[3 * i + 2];
    if (!(most <= kMostNorm) || !(largest_poly(b, c, most) <= kMostPoly))
      return set_error(OZ_ERR_UNSUPPORTED,
                       "the coefficients let singular values grow to %g before step %d of %d; fp16 slices hold %g",
                       most, i + 1, steps, kMostNorm);
    most = largest_value(a, b, c, most);
  }
  return OZ_OK;
}

// Tile counts of a member, and the estimated time of all tiles: waves over the
// GPU times the bytes a CTA loads for each block, which is what bounds both
// shapes (pairs of CTAs load 32 KB for 256 x 256, one CTA 24 KB for 128 x 64).
int64_t member_tiles(bool symmetric, int64_t rows, int64_t cols, int high, int wide) {
  const int64_t tm = (rows + high - 1) / high, tn = (cols + wide - 1) / wide, r = high / wide;
  return symmetric ? r * tm * (tm + 1) / 2 - (r * tm - tn) : tm * tn;
}
bool use_pairs(bool symmetric, int64_t batch, int64_t rows, int64_t cols) {
  const int64_t pairs = sm_count() / 2, singles = sm_count();
  const int64_t two = batch * member_tiles(symmetric, rows, cols, 256, 256);
  const int64_t one = batch * member_tiles(symmetric, rows, cols, 128, 64);
  return 4 * ((two + pairs - 1) / pairs) <= 3 * ((one + singles - 1) / singles);
}

template <class J>
int step_product(const CUtensorMap &a, const CUtensorMap &b, StepParams p, bool symmetric, cudaStream_t st) {
  const int64_t tiles = member_tiles(symmetric, p.rows, p.cols, kRows * J::PAIR, J::NT);
  if (tiles * p.batch > INT32_MAX / 2) return set_error(OZ_ERR_INVALID, "too many tiles");
  p.row_tiles = (p.rows + kRows * J::PAIR - 1) / (kRows * J::PAIR);
  p.column_tiles = (p.cols + J::NT - 1) / J::NT;
  p.tiles = (int)tiles;
  return launch<J>(a, b, p, tiles * p.batch * max(p.parts, 1), st, "newton step launch");
}

// A launch of 256 threads that may start before the one before it has ended.
template <class... A>
int launch_after(void (*kernel)(A...), dim3 grid, const char *what, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}

int add_parts(const StepParams &p, int planes, cudaStream_t st) {
  const unsigned side = (unsigned)((p.rows + 31) / 32);
  return launch_after(add_parts_kernel, dim3(side, side, (unsigned)p.batch), "add_parts_kernel launch", st, p, planes);
}

template <int DTYPE> int start(const InitParams &init, int batch, cudaStream_t st) {
  count_launch();
  squares_kernel<DTYPE><<<dim3((unsigned)init.partials, (unsigned)batch), 256, 0, st>>>(init);
  if (int rc = check_cuda(cudaGetLastError(), "squares_kernel launch")) return rc;
  const int64_t tiles = (int64_t)((init.cols + 63) / 64) * ((init.rows + 63) / 64);
  const int64_t most = std::max<int64_t>(1, 6 * sm_count() / batch);          // tiles at a time of a member
  return launch_after(normalise_kernel<DTYPE>, dim3((unsigned)std::min(tiles, most), 1, (unsigned)batch),
                      "normalise_kernel launch", st, init);
}

// PASS: blocks an accumulator takes before it is added in registers (0: all of them).
template <int SPLITS, int PASS>
int run(const InitParams &init, const Layout &l, int batch, int steps, const double *coefficients,
        unsigned char *ws, StepParams last, cudaStream_t st) {
  const int rows = (int)l.rows, cols = (int)l.cols;
  const int64_t ldx = pitch(cols), lds = pitch(rows);
  auto planes = [&](int64_t offset, int64_t ld, int64_t mat) {
    return Planes{reinterpret_cast<__half *>(ws + offset), ld, mat, mat * batch};
  };
  Planes x[2] = {planes(l.x0, ldx, l.x_mat), planes(l.x1, ldx, l.x_mat)};
  const Planes s = planes(l.s, lds, l.s_mat), q = planes(l.p, lds, l.s_mat);

  if (int rc = init.dtype == OZ_F32   ? start<OZ_F32>(init, batch, st)
               : init.dtype == OZ_F16 ? start<OZ_F16>(init, batch, st)
                                      : start<OZ_BF16>(init, batch, st))
    return rc;

  const bool pair_s = use_pairs(true, batch, rows, rows), pair_x = use_pairs(false, batch, rows, cols);
  // each matrix in the boxes its products read: 128 rows (A), the columns of a
  // tile as rows (B of a symmetric product) or 64 rows across (B of the update)
  auto map = [&](CUtensorMap *m, const Planes &v, int64_t inner, int count, int box) {
    return make_map(m, v.base, inner, rows, (int64_t)batch * count, v.ld * 2, v.mat * 2, box);
  };
  CUtensorMap xa[2], xb[2], xu[2], sa, sb, pa;
  for (int i = 0; i < 2; ++i) {
    if (int rc = map(&xa[i], x[i], cols, 2, kRows)) return rc;
    if (int rc = map(&xb[i], x[i], cols, 2, pair_s ? 128 : 64)) return rc;
    if (int rc = map(&xu[i], x[i], cols, 2, kBlock)) return rc;
  }
  if (int rc = map(&sa, s, rows, SPLITS, kRows)) return rc;
  if (int rc = map(&sb, s, rows, SPLITS, pair_s ? 128 : 64)) return rc;
  if (int rc = map(&pa, q, rows, SPLITS, kRows)) return rc;

  StepParams sym{};
  sym.idesc = instruction(OZ_F16);
  sym.batch = batch;
  sym.rows = sym.cols = rows;
  double most = kFirstNorm;                            // largest singular value of X
  int ex = exponent(most), cur = 0;
  for (int i = 0; i < steps; ++i) {
    const double a = coefficients[3 * i], b = coefficients[3 * i + 1], c = coefficients[3 * i + 2];
    const int es = exponent(most * most), ep = exponent(largest_poly(b, c, most));
    sym.k = cols;
    sym.alpha = 0;
    sym.beta = (float)std::ldexp(1.0, es - 2 * ex);
    sym.out = s;
    sym.parts = l.parts;
    sym.part_blocks = l.part_blocks;
    sym.part_ld = pitch(rows);
    sym.partial = reinterpret_cast<float *>(ws + l.partial);
    int rc = pair_s ? step_product<SymmetricJob<2, 256, SPLITS, 0, PASS>>(xa[cur], xb[cur], sym, true, st)
             : l.parts > 1
                 ? step_product<PartsJob<SPLITS, PASS>>(xa[cur], xb[cur], sym, true, st)
                 : step_product<SymmetricJob<1, 64, SPLITS, 0, PASS>>(xa[cur], xb[cur], sym, true, st);
    if (rc == OZ_OK && l.parts > 1) rc = add_parts(sym, SPLITS, st);
    if (rc) return rc;
    sym.parts = 1;
    sym.k = rows;
    sym.in = s;
    sym.alpha = (float)std::ldexp(b, ep - es);
    sym.beta = (float)std::ldexp(c, ep - 2 * es);
    sym.out = q;
    rc = pair_s ? step_product<SymmetricJob<2, 256, SPLITS, SPLITS, PASS>>(sa, sb, sym, true, st)
                : step_product<SymmetricJob<1, 64, SPLITS, SPLITS, PASS>>(sa, sb, sym, true, st);
    if (rc) return rc;
    most = largest_value(a, b, c, most);
    const bool end = i + 1 == steps;
    const int en = end ? 0 : exponent(most);
    StepParams up = last;
    if (!end) up.last = nullptr;
    up.idesc = sym.idesc;
    up.batch = batch;
    up.rows = rows;
    up.cols = cols;
    up.k = rows;
    up.in = x[cur];
    up.out = x[cur ^ 1];
    up.alpha = (float)std::ldexp(a, en - ex);
    up.beta = (float)std::ldexp(1.0, en - ep - ex);
    rc = pair_x ? step_product<UpdateJob<2, 256, SPLITS, PASS>>(pa, xu[cur], up, false, st)
                : step_product<UpdateJob<1, 64, SPLITS, PASS>>(pa, xu[cur], up, false, st);
    if (rc) return rc;
    cur ^= 1;
    ex = en;
  }
  return OZ_OK;
}

bool valid(int dtype, int64_t batch, int64_t m, int64_t n, int splits) {
  return (dtype == OZ_F32 || dtype == OZ_F16 || dtype == OZ_BF16) && batch >= 0 && m >= 0 && n >= 0 &&
         splits >= 1 && splits <= 2;
}

}  // namespace
}  // namespace oz

extern "C" int64_t oz_orthogonalize_workspace_bytes(int dtype, int64_t batch, int64_t m, int64_t n,
                                                    int32_t steps, int32_t num_splits) {
  using namespace oz;
  if (!valid(dtype, batch, m, n, num_splits) || steps < 1) return OZ_ERR_INVALID;
  if (batch == 0 || m == 0 || n == 0 || small_shape(batch, std::min(m, n), std::max(m, n), steps).ranks) return 0;
  return layout(batch, m, n, num_splits).total;
}

extern "C" int oz_orthogonalize(const void *g, int dtype, int64_t batch, int64_t m, int64_t n,
                                int64_t g_sb, int64_t g_sr, int64_t g_sc, int32_t steps,
                                const double *coefficients, double eps, int32_t num_splits,
                                void *out, void *workspace, int64_t workspace_bytes,
                                void *stream) {
  using namespace oz;
  if (dtype != OZ_F32 && dtype != OZ_F16 && dtype != OZ_BF16)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported dtype %d (fp32, fp16 or bf16)", dtype);
  if (batch < 0 || m < 0 || n < 0) return set_error(OZ_ERR_INVALID, "negative size");
  if (m > (1 << 20) || n > (1 << 20) || batch > 65535)
    return set_error(OZ_ERR_INVALID, "size out of range");
  if (steps < 1 || !coefficients) return set_error(OZ_ERR_INVALID, "at least one step is needed");
  if (!(eps >= 0)) return set_error(OZ_ERR_INVALID, "eps must not be negative");
  if (num_splits < 1 || num_splits > 2)
    return set_error(OZ_ERR_INVALID, "num_splits must be 1 or 2, got %d", num_splits);
  for (int i = 0; i < 3 * steps; ++i)
    if (!std::isfinite(coefficients[i])) return set_error(OZ_ERR_INVALID, "coefficients must be finite");
  if (batch == 0 || m == 0 || n == 0) return OZ_OK;
  if (!g || !out) return set_error(OZ_ERR_INVALID, "null pointer");
  const bool tall = m > n;
  const SmallShape small = small_shape(batch, m < n ? m : n, m < n ? n : m, steps);
  if (small.ranks) {
    SmallParams p{};
    p.g = g;
    p.out = out;
    p.dtype = dtype;
    p.rows = (int)(tall ? n : m);
    p.cols = (int)(tall ? m : n);
    p.steps = steps;
    p.g_sb = g_sb;
    p.g_sr = tall ? g_sc : g_sr;
    p.g_sc = tall ? g_sr : g_sc;
    p.o_sb = m * n;
    p.o_sr = tall ? 1 : n;
    p.o_sc = tall ? n : 1;
    p.eps = eps;
    for (int i = 0; i < 3 * steps; ++i) p.abc[i] = (float)coefficients[i];
    return run_small(small, p, batch, reinterpret_cast<cudaStream_t>(stream));
  }
  if (int rc = bounded_steps(steps, coefficients)) return rc;
  const Layout l = layout(batch, m, n, num_splits);
  if (!workspace || workspace_bytes < l.total || (uintptr_t)workspace % 256 != 0)
    return set_error(OZ_ERR_INVALID,
                     "workspace of %lld bytes (256-byte aligned) needed, got %lld at %p",
                     (long long)l.total, (long long)workspace_bytes, workspace);
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  const int64_t blocks = (l.rows * l.cols + 4095) / 4096;
  const int64_t line = std::max(g_sr, g_sc), step = std::min(g_sr, g_sc);
  const int64_t in_line = g_sr < g_sc ? m : n, per16 = 16 / dtype_size(dtype);
  const bool vectors = (uintptr_t)g % 16 == 0 && step == 1 && line % per16 == 0 && (batch == 1 || g_sb % per16 == 0);
  const bool flat = vectors && line == in_line && m * n % 8 == 0;
  InitParams init{g, dtype, (int)std::min<int64_t>(blocks, kMostPartials), flat, vectors, (int)l.rows, (int)l.cols, g_sb,
                  tall ? g_sc : g_sr, tall ? g_sr : g_sc, reinterpret_cast<double *>(ws),
                  Planes{reinterpret_cast<__half *>(ws + l.x0), pitch(l.cols), l.x_mat, l.x_mat * batch}, eps,
                  std::ldexp(1.0, exponent(kFirstNorm))};
  StepParams last{};
  last.last = out;
  last.last_dtype = dtype;
  last.last_sb = m * n;
  last.last_sr = tall ? 1 : n;
  last.last_sc = tall ? n : 1;
  last.last_vectors = !tall && (uintptr_t)out % 16 == 0 && n * (dtype == OZ_F32 ? 4 : 2) % 16 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (num_splits == 1) return run<1, 0>(init, l, (int)batch, steps, coefficients, ws, last, st);
  // Two slices: sums cut off every block where the launches and not the products take
  // the time, every 4 blocks where it would cost (4096 x 4096: 4682 us and 6.4e-7 off
  // against 3531 us and 1.3e-6; fp32 sums 3.7e-6.  200 x 800: 3.7e-6 with 4, 1.0e-6
  // with 1, fp32 sums 1.5e-6), and every 2 for fewer rows, whose singular values start
  // nearer to 1, so that more steps feel S and P (6 x 1024 x 1536: 782 us and 5.1e-6
  // with 4, 800 us and 2.8e-6 with 2, fp32 sums 3.2e-6)
  const double work = (double)batch * l.rows * l.rows * (3.0 * l.cols + l.rows);
  return work < 2e10     ? run<2, 1>(init, l, (int)batch, steps, coefficients, ws, last, st)
         : l.rows < 1536 ? run<2, 2>(init, l, (int)batch, steps, coefficients, ws, last, st)
                         : run<2, 4>(init, l, (int)batch, steps, coefficients, ws, last, st);
}
