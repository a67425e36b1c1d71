// oz_linear.cu -- a product with what follows it, and its gradients:
//
//   u  = x w + bias,  y = act(u) + residual
//   du = dy act'(u),  dx = du w^T,  dw = x^T du,  dbias = sum of du's rows
//
// The products run on the tile engine (oz_tile.cuh), their epilogues read the
// accumulators from tensor memory and write y (and u, rounded, for the backward
// pass).  Operands are fp16 or bf16, sums fp32; bias, activation and residual are
// applied in fp32 and rounded once.  du is rounded to the operands' type before
// it is multiplied, its sum is not.

#include <algorithm>
#include <type_traits>

#include "oz_linear.cuh"

namespace oz {
int status_linear(int *value, bool clear) { return read_status_word(value, clear); }

namespace {
using namespace tile;
using namespace linear;

struct OutTile { int row, column; };

// 8 aligned values of E as they lie in memory.
template <typename E> struct Run8 {
  struct Raw { uint4 u[sizeof(E) / 2]; };
  static __device__ __forceinline__ Raw load(const E *p) {
    Raw r;
#pragma unroll
    for (int h = 0; h < (int)sizeof(E) / 2; ++h) r.u[h] = *(reinterpret_cast<const uint4 *>(p) + h);
    return r;
  }
  static __device__ __forceinline__ void values(const Raw &r, float (&v)[8]) {
    const E *e = reinterpret_cast<const E *>(&r);
#pragma unroll
    for (int x = 0; x < 8; ++x) v[x] = to_f32(e[x]);
  }
  static __device__ __forceinline__ void store(E *p, const float (&v)[8]) {
    constexpr int V = 16 / sizeof(E);
#pragma unroll
    for (int h = 0; h < 8 / V; ++h) {
      float w[V];
#pragma unroll
      for (int x = 0; x < V; ++x) w[x] = v[h * V + x];
      reinterpret_cast<uint4 *>(p)[h] = stream::pack<E>(w);
    }
  }
};

// The columns of a source 16 at a time, the next ones on their way (accumulators in tensor
// memory) while the ones before are worked on.
template <class Source> struct Ahead16;
template <> struct Ahead16<Columns> {
  const Columns &source;
  uint32_t r[16];
  __device__ __forceinline__ void start(int c) { tmem_ld16_at(source.addr + (uint32_t)c, r); }
  __device__ __forceinline__ void finish(float (&v)[16]) {
    tmem_ld_wait16(r);
#pragma unroll
    for (int x = 0; x < 16; ++x) v[x] = __uint_as_float(r[x]);
  }
};
template <int N> struct Ahead16<Registers<N>> {
  const Registers<N> &source;
  int at;
  __device__ __forceinline__ void start(int c) { at = c; }
  __device__ __forceinline__ void finish(float (&v)[16]) { source.read(at, v); }
};

// Finishes the warp's 32 x COLS accumulators: 16 columns at a time go through its staging
// in fp32, so that a lane has 8 columns of two rows, whose bias, residual and results are
// 16 bytes each, next to the neighbouring lane's.  Accumulators, bias and residual of the next
// columns are on their way meanwhile.  (A lane's own row instead, with the bias and the
// residual read element by element, took 8192 x 8192 results of 4096 terms from 338 us to
// 365 and 549.)  For rows of a multiple of 8 columns on 16-byte boundaries.
template <typename O, typename B, int COLS, int UNROLL, class Source>
__device__ __forceinline__ void finish_vectors(const Params &p, const Source &source, unsigned char *mine, int64_t r0,
                                               int64_t c0) {
  using Out = Run8<O>;
  using In = Run8<B>;
  const int lane = threadIdx.x % 32, half = lane % 2;
  const int rows = (int)min(p.rows - r0, (int64_t)32), columns = (int)min(p.n - c0, (int64_t)COLS);
  if (rows <= 0 || columns <= 0) return;
  const int64_t at = (r0 + lane / 2) * p.ld + c0 + half * 8, next_row = 16 * p.ld;
  O *out = static_cast<O *>(p.out) + at;
  B *pre = p.pre ? static_cast<B *>(p.pre) + at : nullptr;
  const O *residual = p.residual ? static_cast<const O *>(p.residual) + (r0 + lane / 2) * p.residual_ld + c0 + half * 8
                                 : nullptr;
  const int64_t residual_row = 16 * p.residual_ld;
  const B *bias = p.bias && !p.bias_f32 ? static_cast<const B *>(p.bias) + c0 + half * 8 : nullptr;
  const float *bias_f32 = p.bias && p.bias_f32 ? static_cast<const float *>(p.bias) + c0 + half * 8 : nullptr;
  const int act = p.act, mine_end = columns - half * 8;            // this lane's columns: c < mine_end
  const bool one = lane / 2 < rows, two = 16 + lane / 2 < rows;
  typename In::Raw b{};
  typename Run8<float>::Raw b32{};
  typename Out::Raw r[2]{};
  auto fetch = [&](int c) {
    if (c >= mine_end) return;
    if (bias) b = In::load(bias + c);
    if (bias_f32) b32 = Run8<float>::load(bias_f32 + c);
    if (residual) {
      if (one) r[0] = Out::load(residual + c);
      if (two) r[1] = Out::load(residual + c + residual_row);
    }
  };
  Ahead16<Source> ahead{source};
  ahead.start(0);
  fetch(0);
#pragma unroll(UNROLL)
  for (int c = 0; c < COLS; c += 16) {
    if (c >= columns) continue;
    float v[16], u[2][8], add[8];
    ahead.finish(v);
#pragma unroll
    for (int x = 0; x < 4; ++x) *staged(mine, lane, x) = *reinterpret_cast<uint4 *>(&v[x * 4]);
    if (c + 16 < columns) ahead.start(c + 16);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 raw = *staged(mine, i * 16 + lane / 2, half * 2 + h);
        const float *f = reinterpret_cast<const float *>(&raw);
#pragma unroll
        for (int x = 0; x < 4; ++x) u[i][h * 4 + x] = f[x];
      }
    __syncwarp();
    if (bias || bias_f32) {
      if (bias) In::values(b, add);
      else Run8<float>::values(b32, add);
#pragma unroll
      for (int x = 0; x < 8; ++x) u[0][x] += add[x], u[1][x] += add[x];
    }
    const bool there = c < mine_end;
    if (pre) {
      if (there && one) In::store(pre + c, u[0]);
      if (there && two) In::store(pre + c + next_row, u[1]);
    }
    if (act) {
      activate(u[0], act);
      activate(u[1], act);
    }
    if (residual)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        Out::values(r[i], add);
#pragma unroll
        for (int x = 0; x < 8; ++x) u[i][x] += add[x];
      }
    fetch(c + 16);
    if (there && one) Out::store(out + c, u[0]);
    if (there && two) Out::store(out + c + next_row, u[1]);
  }
}

// The same for any rows, element by element: a lane has one column of every other row, so an
// instruction touches 2 rows of 16 columns.
template <typename O, typename B, int COLS, int UNROLL, class Source>
__device__ __forceinline__ void finish_elements(const Params &p, const Source &source, unsigned char *mine, int64_t r0,
                                                int64_t c0) {
  const int lane = threadIdx.x % 32, side = lane / 16, in = lane % 16;
  const int rows = (int)min(p.rows - r0, (int64_t)32), columns = (int)min(p.n - c0, (int64_t)COLS);
  if (rows <= 0 || columns <= 0) return;
  const int64_t at = (r0 + side) * p.ld + c0 + in, residual_at = (r0 + side) * p.residual_ld + c0 + in;
  Ahead16<Source> ahead{source};
  ahead.start(0);
#pragma unroll(UNROLL)
  for (int c = 0; c < COLS; c += 16) {
    if (c >= columns) continue;
    const bool there = c + in < columns;
    O r[16];
    if (p.residual)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (there && 2 * i + side < rows)
          r[i] = static_cast<const O *>(p.residual)[residual_at + c + 2 * i * p.residual_ld];
    const float bias = p.bias && there ? bias_at<B>(p, c0 + c + in) : 0.f;
    float v[16], u[16];
    ahead.finish(v);
#pragma unroll
    for (int x = 0; x < 4; ++x) *staged(mine, lane, x) = *reinterpret_cast<uint4 *>(&v[x * 4]);
    if (c + 16 < columns) ahead.start(c + 16);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i)
      u[i] = reinterpret_cast<const float *>(staged(mine, 2 * i + side, in / 4))[in % 4] + bias;
    __syncwarp();
    if (p.pre)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (there && 2 * i + side < rows) static_cast<B *>(p.pre)[at + c + 2 * i * p.ld] = from_f32<B>(u[i]);
    activate(u, p.act);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (there && 2 * i + side < rows)
        static_cast<O *>(p.out)[at + c + 2 * i * p.ld] = from_f32<O>(p.residual ? u[i] + to_f32(r[i]) : u[i]);
  }
}

// What follows a product: nothing, or bias, activation and residual by vectors or by elements.
enum Form { kPlain, kByVectors, kByElements };
// What follows a product keeps 16 epilogue warps busy (a plain one's 8 wait for its stores;
// the sums of passes of an fp32 result leave no registers for 16, and where something follows
// them they lie in local memory: 4096^3 108 us plain, 175 to 190 with bias, gelu and residual).
// A 16-bit result's whole contraction is added in one accumulator, whose additions cut off below
// fp32's last bit: all-positive terms come out 2e-5 too small with 4096 of them, 1e-4 with 16384 and
// 4e-4 with 65536, as in cuBLAS, beside the half unit of 5e-4 (fp16) or 4e-3 (bf16) of the
// rounding.  Passes of 8 blocks added in registers, as for fp32 results, keep 2.5e-6 at any
// length, and cost registers and time that a 16-bit result seldom shows.
template <typename O, typename B, int PAIR_, int NT_, bool AMN_, bool BMN_, int FORM> struct LinearJob : NoLookAhead {
  static constexpr int EPILOGUE_WARPS = FORM == kPlain || NT_ < 256 || sizeof(O) == 4 ? 8 : 16;
  static constexpr int PAIR = PAIR_, NT = NT_, PLANES = 1, PASS = sizeof(O) == 4 ? 8 : 0;
  static constexpr bool AMN = AMN_, BMN = BMN_, RAGGED = false;
  using Params = linear::Params;
  using Extra = OutTile;
  static __device__ int plane_stride(const Params &) { return 0; }
  struct Walk {
    __device__ Walk(const Params &) {}
    // 8 row tiles at a time sweep the columns: their operands stay in L2
    __device__ bool find(const Params &p, int i, TileOf<Extra> &t) {
      if (i >= p.row_tiles * p.column_tiles) return false;
      const int sweep = i / (8 * p.column_tiles), in = i - sweep * 8 * p.column_tiles;
      const int size = min(p.row_tiles - sweep * 8, 8);
      t.a_row = (sweep * 8 + in % size) * kRows * PAIR;
      t.b_row = in / size * NT;
      t.a_mat = t.b_mat = 0;
      t.k_begin = 0;
      t.k_len = p.k;
      t.extra = OutTile{t.a_row, t.b_row};
      return true;
    }
  };
  template <class Source>
  static __device__ void epilogue(const Params &p, const TileOf<Extra> &t, const Source &source, int row, int column,
                                  unsigned char *mine, Ahead &) {
    const int64_t r0 = t.extra.row + row, c0 = t.extra.column + column;
    const int rows = (int)(p.rows - r0);
    O *out = static_cast<O *>(p.out) + r0 * p.ld + c0;
    if constexpr (FORM == kPlain) {
      write_rows<O, NT / 2>(source, mine, out, p.ld, rows, p.n - c0, p.vectors & kVectors);
    } else {
      constexpr int COLS = NT * 4 / EPILOGUE_WARPS, UNROLL = PASS ? COLS : 1;
      if constexpr (FORM == kByVectors) finish_vectors<O, B, COLS, UNROLL>(p, source, mine, r0, c0);
      else finish_elements<O, B, COLS, UNROLL>(p, source, mine, r0, c0);
    }
  }
  static __device__ void finish(const Params &, int, int) {}
};

template <class J>
int run_job(const Side &a, const Side &b, Params p, cudaStream_t st, const char *what) {
  CUtensorMap ta, tb;
  const int64_t ai = J::AMN ? p.rows : p.k, ar = J::AMN ? p.k : p.rows;
  const int64_t bi = J::BMN ? p.n : p.k, br = J::BMN ? p.k : p.n;
  const int64_t ap = pitch_bytes(a.pitch, ar, ai), bp = pitch_bytes(b.pitch, br, bi);
  if (int rc = make_map(&ta, a.p, ai, ar, 1, ap, ap, J::AMN ? kBlock : kRows)) return rc;
  if (int rc = make_map(&tb, b.p, bi, br, 1, bp, bp, J::BMN ? kBlock : J::NT / J::PAIR)) return rc;
  const int64_t rows = (p.rows + kRows * J::PAIR - 1) / (kRows * J::PAIR), columns = (p.n + J::NT - 1) / J::NT;
  if (rows * columns > INT32_MAX / 2) return set_error(OZ_ERR_INVALID, "too many tiles");
  p.row_tiles = (int)rows;
  p.column_tiles = (int)columns;
  return launch<J>(ta, tb, p, rows * columns, st, what);
}

template <typename O, typename B, int FORM>
int product(bool pair, const Side &a, const Side &b, const Params &p, cudaStream_t st, const char *what) {
  if (a.mn) {
    if constexpr (FORM == kPlain)
      return pair ? run_job<LinearJob<O, B, 2, 256, true, true, kPlain>>(a, b, p, st, what)
                  : run_job<LinearJob<O, B, 1, 128, true, true, kPlain>>(a, b, p, st, what);
    return set_error(OZ_ERR_UNSUPPORTED, "operand layout");
  }
  if (b.mn)
    return pair ? run_job<LinearJob<O, B, 2, 256, false, true, FORM>>(a, b, p, st, what)
                : run_job<LinearJob<O, B, 1, 128, false, true, FORM>>(a, b, p, st, what);
  return pair ? run_job<LinearJob<O, B, 2, 256, false, false, FORM>>(a, b, p, st, what)
              : run_job<LinearJob<O, B, 1, 128, false, false, FORM>>(a, b, p, st, what);
}

// How a product is divided, by the least estimated time (us, one B200, fitted to 2000 measured
// times of 180 sizes, 1 to 16000 rows, 8 to 8192 terms and columns, plain and with what may
// follow: half of them within 10%; the choice is 2% slower than the best one on average, 39% at
// most).  Engine: its start, and for each wave of tiles a tile's blocks of 64 terms and its
// end.  Split: for each wave of clusters (two CTAs an SM; clusters of 8 do not fit everywhere) a
// CTA's start and end and its blocks, which take longer where the SM has two.  Some sizes (bf16, us):
//   rows x terms x columns          128 x 128   256 x 256   split (rows of a tile, CTAs)
//   4 x 3904 x 2600                    22.3        25.1      7.2 (16, 8)    9.0 (16, 4)
//   131 x 7504 x 2688                  45          49       16.7 (64, 4)   20.4 (128, 4)
//   432 x 72 x 2136                     4.2         5.9      5.5 (64, 1)    7.4 (128, 1)
//   720 x 7904 x 3616                  76.8        45.2     67.0 (128, 4)
//   580 x 6504 x 1056, silu, added     36.9        48       24.9 (128, 4)  39.0 (128, 2)
//   8687 x 160 x 2369, the same        78.5        67.5
// and by pairs that share a contraction, silu: 299 x 4632 x 3880 27.9 (2 pairs) where the others take
// 34.0, 536 x 7504 x 2688 31.7 (2; 42.3), 580 x 6504 x 1024 18.3 (4).  4 pairs take 14 tiles at most:
// 580 x 6504 x 1056 has 15 and takes 24.3 (128 rows, 4 CTAs).
struct Plan {
  bool pair;                   // the engine's tiles: 256 x 256 by pairs of CTAs, or 128 x 128
  SplitPlan split;             // of 0 rows: the engine
  bool loose;                  // operands off the 16-byte boundaries are read as they are
};
struct Times {
  double start, block, end, start_pair, block_pair, end_pair;      // engine
  double split_end[3], split_block[3], split_shared[3], joined[3]; // for tiles of 16, 64, 128 rows
};
constexpr Times kTimes[3] = {
    {3.3, 0.320, 0.9, 3.6, 0.347, 1.9, {2.9, 4.4, 6.1}, {0.271, 0.290, 0.347}, {0.10, 0.21, 0.32}, {0.85, 0.37, 0}},
    {2.4, 0.300, 3.9, 0.4, 0.321, 6.7, {4.0, 6.0, 7.6}, {0.292, 0.322, 0.410}, {0.10, 0.15, 0.28}, {0.75, 0, 0}},
    {3.8, 0.306, 6.1, 2.6, 0.319, 11.2, {4.4, 6.4, 9.1}, {0.292, 0.311, 0.409}, {0.09, 0.21, 0.31}, {0.55, 0, 0}}};
constexpr int kTileRows[3] = {16, 64, 128};
int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
// Clusters that the GPU holds at once, two CTAs an SM.
int64_t clusters_at_once(int splits) {
  const int64_t sms = tile::sm_count();
  return splits == 1 ? 2 * sms : splits == 2 ? sms : splits == 4 ? sms * 70 / 148 : splits == 8 ? sms * 32 / 148
                                                                                               : sms * 14 / 148;
}

Plan plan_product(int64_t rows, int64_t k, int64_t n, bool rows_mn, Form form, bool fp32) {
  const int64_t sms = tile::sm_count(), blocks = up(k, kBlock);
  const Times &t = kTimes[form];
  Plan plan{false, {0, 1}, false};
  double best = t.start + up(up(rows, 128) * up(n, 128), sms) * (t.block * blocks + t.end);
  const double pairs = t.start_pair + up(up(rows, 256) * up(n, 256) * 2, sms) * (t.block_pair * blocks + t.end_pair);
  if (pairs < best) plan.pair = true, best = pairs;
  for (int shape = rows_mn ? 1 : 0; shape < 3; ++shape) {
    const int64_t tiles = up(rows, kTileRows[shape]) * up(n, 128);
    for (int splits = 1; splits <= kMostSplits && splits <= blocks; splits *= 2) {
      const int64_t held = clusters_at_once(splits), waves = up(tiles, held), halves = up(2 * tiles, held);
      const int64_t each = up(blocks, splits);
      if (waves > 2) break;                    // the engine's CTAs stay; the fit knows no more waves
      const double time = waves * (t.split_end[shape] + each * t.split_block[shape]) +
                          (halves - waves) * each * t.split_shared[shape] + (splits > 1 ? t.joined[shape] : 0.0) + (splits > 8 ? 1.0 : 0.0);
      if (time < best) plan.split = SplitPlan{kTileRows[shape], splits}, best = time;
    }
  }
  // tiles of 256 x 256 whose contraction 2 or 4 pairs of CTAs share, in one wave (as many as 34
  // and 14 clusters are held at once)
  for (int splits = 2; !fp32 && splits <= 4 && splits <= blocks; splits *= 2) {
    const double time = (splits == 2 ? 12.0 : 8.8) + up(blocks, splits) * 0.35;
    if (up(rows, 256) * up(n, 256) <= (splits == 2 ? sms * 34 / 148 : sms * 14 / 148) && time < best)
      plan.split = SplitPlan{kPairTile, splits}, best = time;
  }
  return plan;
}

// What follows the product and how its rows may be moved.
Form form_of(const Params &p) {
  if (!p.bias && !p.act && !p.residual && !p.pre) return kPlain;
  constexpr int kAll = kVectors | kResidualVectors | kBiasVectors;
  return (p.vectors & kAll) == kAll && p.n % 8 == 0 ? kByVectors : kByElements;
}

template <int FORM>
int product_in(bool pair, int dtype, int out_dtype, const Side &a, const Side &b, const Params &p, cudaStream_t st,
               const char *what) {
  if (dtype == OZ_F16)
    return out_dtype == OZ_F32 ? product<float, __half, FORM>(pair, a, b, p, st, what)
                               : product<__half, __half, FORM>(pair, a, b, p, st, what);
  return out_dtype == OZ_F32 ? product<float, __nv_bfloat16, FORM>(pair, a, b, p, st, what)
                             : product<__nv_bfloat16, __nv_bfloat16, FORM>(pair, a, b, p, st, what);
}

int product_of(const Plan &plan, int dtype, int out_dtype, const Side &a, const Side &b, const Params &p, cudaStream_t st,
               const char *what) {
  if (plan.split.tile_rows) return split_product(plan.split, dtype, out_dtype, a, b, p, st, what);
  switch (form_of(p)) {
    case kPlain: return product_in<kPlain>(plan.pair, dtype, out_dtype, a, b, p, st, what);
    case kByVectors: return product_in<kByVectors>(plan.pair, dtype, out_dtype, a, b, p, st, what);
    default: return product_in<kByElements>(plan.pair, dtype, out_dtype, a, b, p, st, what);
  }
}

// ---------------------------------------------------------------------------
// du = dy act'(u) and the sums of its columns
// ---------------------------------------------------------------------------
struct SlopeParams {
  const void *dy, *pre;        // pre: none without an activation
  void *du;                    // written where there is an activation
  float *sums;                 // a row for each block row; none: no sums
  int64_t dy_sr, pre_sr, du_sr;
  int64_t rows;
  int n, act, per;             // rows of a block
  int lanes;                   // of a row: a power of 2
};

constexpr int kSlopeRows = 8;  // warps of a block

// p.lanes lanes take a row's columns (or 32 V of them), so a warp has 32 / p.lanes rows; its
// next two sets of rows are on their way while it works on the two before.  8192 x 8192 (403
// MB, 62 us at the memory's rate): silu 74 us with the sums, gelu 92 (instructions); 5 blocks an
// SM spilled and took 88 and 108.
template <typename T, int V> __global__ void __launch_bounds__(256, 4) slope_kernel(const SlopeParams p) {
  constexpr int AT_ONCE = 2;
  using R = stream::Raw<T, V, true>;
  __shared__ float part[kSlopeRows][32 * V];
  stream::start_after_earlier_kernels();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int c = (blockIdx.x * 32 + lane % p.lanes) * V;
  const int first = warp * (32 / p.lanes) + lane / p.lanes, apart = kSlopeRows * (32 / p.lanes);
  const int64_t r0 = (int64_t)blockIdx.y * p.per;
  const int rows = (int)min((int64_t)p.per, p.rows - r0);
  float sum[V] = {};
  if (c < p.n) {
    const T *dy = static_cast<const T *>(p.dy) + r0 * p.dy_sr + c, *pre = static_cast<const T *>(p.pre) + r0 * p.pre_sr + c;
    T *du = static_cast<T *>(p.du) + r0 * p.du_sr + c;
    typename R::Type a[AT_ONCE], b[AT_ONCE], next_a[AT_ONCE], next_b[AT_ONCE];
    auto load = [&](int r, auto &to_a, auto &to_b) {
#pragma unroll
      for (int q = 0; q < AT_ONCE; ++q) {
        const int at = r + q * apart;
        if (at >= rows) continue;
        to_a[q] = R::load(dy + at * p.dy_sr);
        if (p.pre) to_b[q] = R::load(pre + at * p.pre_sr);
      }
    };
    load(first, a, b);
#pragma unroll 1
    for (int r = first; r < rows; r += AT_ONCE * apart) {
      load(r + AT_ONCE * apart, next_a, next_b);
#pragma unroll
      for (int q = 0; q < AT_ONCE; ++q) {
        const int at = r + q * apart;
        if (at >= rows) continue;
        float v[V], u[V];
        R::values(a[q], v);
        if (p.pre) {
          R::values(b[q], u);
          if constexpr (V == 1) {
            float v2[2] = {v[0], v[0]};
            const float u2[2] = {u[0], u[0]};
            times_slope(v2, u2, p.act);
            v[0] = v2[0];
          } else {
            times_slope(v, u, p.act);
          }
          stream::Run<T, V>::store(du + at * p.du_sr, v);
        }
#pragma unroll
        for (int x = 0; x < V; ++x) sum[x] += v[x];
      }
#pragma unroll
      for (int q = 0; q < AT_ONCE; ++q) {
        a[q] = next_a[q];
        b[q] = next_b[q];
      }
    }
  }
  if (!p.sums) return;
  for (int o = p.lanes; o < 32; o *= 2)
#pragma unroll
    for (int x = 0; x < V; ++x) sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], o);
  if (lane < p.lanes)
#pragma unroll
    for (int x = 0; x < V; ++x) part[warp][lane * V + x] = sum[x];
  __syncthreads();
  for (int i = threadIdx.x; i < p.lanes * V; i += 256) {
    const int column = blockIdx.x * 32 * V + i;
    if (column >= p.n) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kSlopeRows; ++w) s += part[w][i];
    p.sums[(int64_t)blockIdx.y * p.n + column] = s;
  }
}

// A block adds up 32 columns of the block rows' sums, a warp every eighth row.
__global__ void __launch_bounds__(256) sums_kernel(const float *sums, float *out, int rows, int n) {
  __shared__ double part[8][33];
  stream::start_after_earlier_kernels();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, c = blockIdx.x * 32 + lane;
  double s = 0;
  if (c < n)
#pragma unroll 8
    for (int r = warp; r < rows; r += 8) s += *(sums + (int64_t)r * n + c);
  part[warp][lane] = s;
  __syncthreads();
  if (warp || c >= n) return;
  for (int w = 1; w < 8; ++w) s += part[w][lane];
  out[c] = (float)s;
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

// Rows of a block of slope_kernel: as many blocks as the GPU holds at once.
int slope_rows(int64_t rows, int n) {
  const int64_t columns = (n + 255) / 256;
  const int64_t want = std::max<int64_t>(1, stream::sm_count() * 4 / columns);
  const int64_t per = std::max<int64_t>(64, (rows + want - 1) / want);
  return (int)((per + 15) / 16 * 16);
}

int check_linear(int dtype, int out_dtype, int act, int64_t rows, int64_t k, int64_t n) {
  if (dtype != OZ_F16 && dtype != OZ_BF16)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported operand dtype %d (fp16 or bf16)", dtype);
  if (out_dtype != dtype && out_dtype != OZ_F32)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported output dtype %d", out_dtype);
  if (act < OZ_ACT_NONE || act > OZ_ACT_SILU) return set_error(OZ_ERR_UNSUPPORTED, "unsupported activation %d", act);
  if (rows < 0 || k < 0 || n < 0) return set_error(OZ_ERR_INVALID, "negative size");
  if (rows > (1 << 30) || k > (1 << 30) || n > (1 << 30)) return set_error(OZ_ERR_INVALID, "size out of range");
  return OZ_OK;
}

// A weight (k, n) as an operand: stored across its rows' dimension or along it.
bool stored_across(int64_t n, int64_t w_sk, int64_t w_sn) { return w_sn == 1 || (n == 1 && w_sk != 1); }

// The operands x and w of a product and how it is divided.  Small products read operands off
// the 16-byte boundaries as they are where a CTA has few pieces of 64 lines of them: 0.75 us
// each, 1.1 where two CTAs share an SM (67 x 1000 x 1407, 4 pieces: 9.7 us; 300 x 2047 x 515, 12:
// 20 us).  A copy first takes 11 and 12 us on the device, and 4.4 us more of the host, which
// is what counts up to 13 us.  Not where fp32 results take their sums in passes: the warps that
// would load are busy with those.
// (Whether they are read so does not depend on the form.)
Plan linear_operands(const oz_linear_args &a, bool across, Form form, Operand (&ops)[2]) {
  ops[0] = Operand{a.x, a.rows, a.x_sr, 1, 0, (int)a.k};
  ops[1] = Operand{a.w, across ? a.k : a.n, across ? a.w_sk : a.w_sn, 1, 0, (int)(across ? a.n : a.k)};
  const Plan whole = plan_product(a.rows, a.k, a.n, false, form, a.out_dtype == OZ_F32);
  const bool loose_x = copy_bytes(ops[0]) != 0, loose_w = copy_bytes(ops[1]) != 0;
  if (!loose_x && !loose_w) return whole;
  const int64_t sms = tile::sm_count(), blocks = up(a.k, kBlock);
  Plan plan{false, {0, 1}, true};
  double best = 10.5;
  for (int shape = 0; shape < 3; ++shape) {
    const int64_t tiles = up(a.rows, kTileRows[shape]) * up(a.n, 128);
    for (int splits = 1; splits <= 8 && splits <= blocks; splits *= 2) {      // (16: 15 us where 8 take 12)
      const int64_t pieces = up(blocks, splits) * ((loose_w ? 2 : 0) + (loose_x ? up(kTileRows[shape], 64) : 0));
      if (a.out_dtype == OZ_F32 && up(blocks, splits) > 8) continue;
      const double time = up(tiles, clusters_at_once(splits)) *
                              (kTimes[kPlain].split_end[shape] + pieces * (tiles * splits > sms ? 1.1 : 0.75)) +
                          kTimes[kPlain].joined[shape];
      if (time < best) plan.split = SplitPlan{kTileRows[shape], splits}, best = time;
    }
  }
  return plan.split.tile_rows ? plan : whole;
}

// y of an empty contraction: the epilogue on zeros.
template <typename O, typename B> __global__ void __launch_bounds__(256) empty_kernel(const Params p) {
  stream::start_after_earlier_kernels();
  const int64_t end = (int64_t)p.rows * p.n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < end; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / p.n, c = i - r * p.n;
    const float u = p.bias ? bias_at<B>(p, c) : 0.f;
    if (p.pre) static_cast<B *>(p.pre)[r * p.ld + c] = from_f32<B>(u);
    float v[2] = {u, u};
    activate(v, p.act);
    float y = v[0];
    if (p.residual) y += to_f32(static_cast<const O *>(p.residual)[r * p.residual_ld + c]);
    static_cast<O *>(p.out)[r * p.ld + c] = from_f32<O>(y);
  }
}

}  // namespace
}  // namespace oz

extern "C" int64_t oz_linear_workspace_bytes(const oz_linear_args *args) {
  using namespace oz;
  if (!args) return OZ_ERR_INVALID;
  const oz_linear_args &a = *args;
  if (check_linear(a.dtype, a.out_dtype, a.act, a.rows, a.k, a.n)) return OZ_ERR_INVALID;
  if (a.rows == 0 || a.n == 0 || a.k == 0) return 0;
  Operand ops[2];
  if (linear_operands(a, stored_across(a.n, a.w_sk, a.w_sn), kPlain, ops).loose) return 0;
  return copy_bytes(ops[0]) + copy_bytes(ops[1]);
}

extern "C" int oz_linear(const oz_linear_args *args, void *stream) {
  if (!args) return oz::set_error(OZ_ERR_INVALID, "null arguments");
  using namespace oz;
  const oz_linear_args &a = *args;
  if (int rc = check_linear(a.dtype, a.out_dtype, a.act, a.rows, a.k, a.n)) return rc;
  if (a.bias && a.bias_dtype != a.dtype && a.bias_dtype != OZ_F32)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported bias dtype %d", a.bias_dtype);
  if (a.rows == 0 || a.n == 0) return OZ_OK;
  if (!a.y) return set_error(OZ_ERR_INVALID, "null pointer");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int es = dtype_size(a.out_dtype);
  if (!stream::aligned(es, {a.y, a.residual}) || !stream::aligned(2, {a.pre}) ||
      !stream::aligned(dtype_size(a.bias_dtype), {a.bias}))
    return stream::not_aligned();
  Params p{a.y, a.pre, a.bias, a.residual, a.n, a.residual_sr, (int)a.rows, (int)a.k, (int)a.n, 0, 0,
                 0, a.bias_dtype == OZ_F32, a.act, tile::instruction(a.dtype)};
  if ((uintptr_t)a.y % 16 == 0 && a.n * es % 16 == 0 && (!a.pre || ((uintptr_t)a.pre % 16 == 0 && a.n % 8 == 0)))
    p.vectors |= kVectors;
  if (!a.residual || ((uintptr_t)a.residual % 16 == 0 && (a.rows == 1 || a.residual_sr * es % 16 == 0)))
    p.vectors |= kResidualVectors;
  if ((uintptr_t)a.bias % 16 == 0) p.vectors |= kBiasVectors;
  if (a.k == 0) {
    const dim3 grid((unsigned)std::min<int64_t>((a.rows * a.n + 255) / 256, stream::sm_count() * 8));
    const char *what = "empty product launch";
    if (a.dtype == OZ_F16)
      return a.out_dtype == OZ_F32 ? stream::launch(empty_kernel<float, __half>, grid, 256, 0, st, what, p)
                                   : stream::launch(empty_kernel<__half, __half>, grid, 256, 0, st, what, p);
    return a.out_dtype == OZ_F32 ? stream::launch(empty_kernel<float, __nv_bfloat16>, grid, 256, 0, st, what, p)
                                 : stream::launch(empty_kernel<__nv_bfloat16, __nv_bfloat16>, grid, 256, 0, st, what, p);
  }
  if (!a.x || !a.w) return set_error(OZ_ERR_INVALID, "null pointer");
  const bool across = stored_across(a.n, a.w_sk, a.w_sn);
  if (!across && a.w_sk != 1 && a.k != 1) return set_error(OZ_ERR_INVALID, "w must have a unit stride along k or n");
  Operand ops[2];
  const Plan plan = linear_operands(a, across, form_of(p), ops);
  if ((uintptr_t)a.x % 2 != 0 || (uintptr_t)a.w % 2 != 0)
    return set_error(OZ_ERR_INVALID, "an operand is not aligned to its elements");
  if (!plan.loose)
    if (int rc = lay_out(ops, 2, a.workspace, a.workspace_bytes, st)) return rc;
  return product_of(plan, a.dtype, a.out_dtype, Side{ops[0].p, ops[0].row, false}, Side{ops[1].p, ops[1].row, across}, p,
                           st, "product launch");
}

// Workspace of the backward pass beside the operands' copies: du and partial sums.
extern "C" int64_t oz_linear_backward_workspace_bytes(int64_t rows, int64_t n, int32_t act, int32_t sums) {
  using namespace oz;
  if (rows < 0 || n < 0) return set_error(OZ_ERR_INVALID, "negative size");
  if (rows > (1 << 30) || n > (1 << 30)) return set_error(OZ_ERR_INVALID, "size out of range");
  if (rows == 0 || n == 0) return 0;
  const int64_t blocks = (rows + slope_rows(rows, (int)n) - 1) / slope_rows(rows, (int)n);
  return (act ? align256(rows * ((n + 7) / 8 * 8) * 2) : 0) + (sums && blocks > 1 ? align256(blocks * n * 4) : 0);
}

extern "C" int oz_linear_backward(const oz_linear_backward_args *args, void *stream) {
  if (!args) return oz::set_error(OZ_ERR_INVALID, "null arguments");
  using namespace oz;
  const oz_linear_backward_args &a = *args;
  if (int rc = check_linear(a.dtype, a.dw_dtype, a.act, a.rows, a.k, a.n)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int dw_size = dtype_size(a.dw_dtype);
  if (!stream::aligned(2, {a.dy, a.x, a.w, a.pre, a.dx}) || !stream::aligned(dw_size, {a.dw}) || !stream::aligned(4, {a.db}))
    return stream::not_aligned();
  if (a.rows == 0 || a.n == 0) {
    if (a.dx && a.rows * a.k)
      if (int rc = check_cuda(cudaMemsetAsync(a.dx, 0, (size_t)(a.rows * a.k * 2), st), "cudaMemsetAsync")) return rc;
    if (a.dw && a.k * a.n)
      if (int rc = check_cuda(cudaMemsetAsync(a.dw, 0, (size_t)(a.k * a.n * dw_size), st), "cudaMemsetAsync")) return rc;
    if (a.db && a.n) return check_cuda(cudaMemsetAsync(a.db, 0, (size_t)(a.n * 4), st), "cudaMemsetAsync");
    return OZ_OK;
  }
  if (!a.dy || (a.act && !a.pre)) return set_error(OZ_ERR_INVALID, "null pointer");
  const bool want_x = a.dx && a.k > 0, want_w = a.dw && a.k > 0;
  if ((want_x && !a.w) || (want_w && !a.x)) return set_error(OZ_ERR_INVALID, "null pointer");
  const int64_t own = oz_linear_backward_workspace_bytes(a.rows, a.n, a.act, a.db != nullptr);
  if (own && (!a.workspace || (uintptr_t)a.workspace % 256 != 0 || a.workspace_bytes < own))
    return set_error(OZ_ERR_INVALID, "workspace of %lld bytes (256-byte aligned) needed, got %lld at %p", (long long)own,
                     (long long)a.workspace_bytes, a.workspace);
  unsigned char *space = static_cast<unsigned char *>(a.workspace);
  const int per = slope_rows(a.rows, (int)a.n);
  const int64_t blocks = (a.rows + per - 1) / per;
  Operand du{a.dy, a.rows, a.dy_sr, 1, 0, (int)a.n};
  if (a.act || a.db) {
    const int64_t pitch = (a.n + 7) / 8 * 8;
    void *out = a.act ? space : nullptr;
    float *sums = !a.db ? nullptr : blocks == 1 ? a.db
                  : reinterpret_cast<float *>(space + (a.act ? align256(a.rows * pitch * 2) : 0));
    SlopeParams s{a.dy, a.act ? a.pre : nullptr, out, sums, a.dy_sr, a.pre_sr, pitch, a.rows, (int)a.n, a.act, per, 32};
    auto fits = [&](const void *base, int64_t sr) { return !base || ((uintptr_t)base % 16 == 0 && (a.rows == 1 || sr % 8 == 0)); };
    const bool wide = fits(s.dy, s.dy_sr) && fits(s.pre, s.pre_sr) && a.n % 8 == 0;
    const int v = wide ? 8 : 1;
    while (s.lanes > 1 && s.lanes / 2 * v >= a.n) s.lanes /= 2;
    if (blocks > 65535) return set_error(OZ_ERR_INVALID, "size out of range");
    const dim3 grid((unsigned)((a.n + 32 * v - 1) / (32 * v)), (unsigned)blocks);
    const char *what = "slope_kernel launch";
    int rc;
    if (a.dtype == OZ_F16)
      rc = wide ? stream::launch(slope_kernel<__half, 8>, grid, 256, 0, st, what, s)
                : stream::launch(slope_kernel<__half, 1>, grid, 256, 0, st, what, s);
    else
      rc = wide ? stream::launch(slope_kernel<__nv_bfloat16, 8>, grid, 256, 0, st, what, s)
                : stream::launch(slope_kernel<__nv_bfloat16, 1>, grid, 256, 0, st, what, s);
    if (rc) return rc;
    if (a.db && blocks > 1) {
      rc = stream::launch(sums_kernel, dim3((unsigned)((a.n + 31) / 32)), 256, 0, st, "sums_kernel launch",
                          (const float *)sums, a.db, (int)blocks, (int)a.n);
      if (rc) return rc;
    }
    if (a.act) {
      du.p = out;
      du.row = pitch;
    }
  }
  if (!want_x && !want_w) return OZ_OK;
  const bool across = stored_across(a.n, a.w_sk, a.w_sn);
  if (want_x && !across && a.w_sk != 1 && a.k != 1)
    return set_error(OZ_ERR_INVALID, "w must have a unit stride along k or n");
  Operand ops[3] = {du};
  int count = 1, at_w = 0, at_x = 0;
  if (want_x) {
    ops[at_w = count++] = Operand{a.w, across ? a.k : a.n, across ? a.w_sk : a.w_sn, 1, 0, (int)(across ? a.n : a.k)};
  }
  if (want_w) ops[at_x = count++] = Operand{a.x, a.rows, a.x_sr, 1, 0, (int)a.k};
  if (int rc = lay_out(ops, count, space + own, a.workspace_bytes - own, st)) return rc;
  if (want_x) {
    // dx (rows, k) = du (rows, n) w^T: w's rows along n where it is stored across
    Params p{a.dx, nullptr, nullptr, nullptr, a.k, 0, (int)a.rows, (int)a.n, (int)a.k, 0, 0,
                   (uintptr_t)a.dx % 16 == 0 && a.k % 8 == 0, 0, OZ_ACT_NONE, tile::instruction(a.dtype)};
    if (int rc = product_of(plan_product(a.rows, a.n, a.k, false, kPlain, false), a.dtype, a.dtype, Side{ops[0].p, ops[0].row, false},
                                  Side{ops[at_w].p, ops[at_w].row, !across}, p, st, "dx launch"))
      return rc;
  }
  if (want_w) {
    Params p{a.dw, nullptr, nullptr, nullptr, a.n, 0, (int)a.k, (int)a.rows, (int)a.n, 0, 0,
                   (uintptr_t)a.dw % 16 == 0 && a.n * dw_size % 16 == 0, 0, OZ_ACT_NONE, tile::instruction(a.dtype)};
    return product_of(plan_product(a.k, a.rows, a.n, true, kPlain, a.dw_dtype == OZ_F32),
                      a.dtype, a.dw_dtype, Side{ops[at_x].p, ops[at_x].row, true},
                            Side{ops[0].p, ops[0].row, true}, p, st, "dw launch");
  }
  return OZ_OK;
}
