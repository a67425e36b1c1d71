// oz_route.cu -- the router of an expert layer and the way of the tokens' rows.
//
//   p[t]       = softmax(logits[t])            0 for a row that is -inf throughout
//   picks      = the k largest logits of a row, the lowest index first among equals;
//                an expert at -inf is not picked
//   w[t, j]    = p[t, e(t, j)], or that over the sum of the row's picks
//   slots      : rows of the picks in the order of their experts, of their tokens
//                within one: offsets[e] + (earlier tokens that picked e)
//   loss       = E sum_e (count_e / sum count) (sum_t p[t, e] / tokens)
//   dlogits[t] = p (g - sum_e g p),  g_e = dloss E (count_e / sum count) / tokens + dw of e's pick
//
//   dispatch   : rows[slots[t, j]] = x[t]
//   combine    : y[t] = sum_j w[t, j] rows[slots[t, j]]
//
// Softmax and all sums are in fp32 (the sums over tokens of all blocks in
// fp64); results do not depend on the order in which blocks run.

#include <algorithm>
#include <cmath>

#include "oz_stream.cuh"

namespace oz {
namespace {
using namespace stream;

constexpr int kMaxPicks = 32, kMaxExperts = 1024;
constexpr int kMaxChunk = 256;                // tokens of a block's round
constexpr uint32_t kNothing = 0x007FFFFFu;    // ordered form of -inf

// Order-preserving whole numbers of fp32 values: NaN above all, the two zeros equal.
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  if (f != f) return 0xFFFFFFFFu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

struct RouteParams {
  const void *logits;
  float *weights, *loss;
  int *experts, *slots, *offsets, *counts, *tokens;
  int *hist;                   // picks of each block and expert, and ...
  float *psum;                 // ... its sums of p, and its tokens
  int *held;
  int64_t rows, row, col;
  int e, k, normalize, chunk, per, blocks;    // tokens of a round, rounds of a block
};

// A token's logits lie in LPT lanes, value i of lane l being expert i * LPT + l.
template <typename T, int LPT, int VPL> struct Row {
  static __device__ __forceinline__ void load(const RouteParams &p, int64_t t, bool there, int l, float (&v)[VPL]) {
    const T *from = static_cast<const T *>(p.logits) + t * p.row;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = i * LPT + l;
      v[i] = there && e < p.e ? to_f32(from[e * p.col]) : -INFINITY;
    }
  }
};
template <int LPT, typename F> __device__ __forceinline__ float over_lanes(float v, F f) {
#pragma unroll
  for (int o = LPT / 2; o > 0; o /= 2) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int LPT> __device__ __forceinline__ float lanes_sum(float v) {
  return over_lanes<LPT>(v, [](float a, float b) { return a + b; });
}

// Exclusive prefix sums of n counts in shared memory, by the first warp; total in from[n].
__device__ __forceinline__ void scan(int *from, int n) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int before = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int own = i0 + lane < n ? from[i0 + lane] : 0;
      int upto = own;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (i0 + lane < n) from[i0 + lane] = before + upto - own;
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) from[n] = before;
  }
  __syncthreads();
}

int route_smem(int e, int k, int chunk, int warps) {
  return 4 * (e * (chunk / 32) + 2 * (e + 1) + warps * e + chunk * k + chunk + 1) + 2 * chunk * k;
}

// Picks of `per` rounds of `chunk` tokens a block.  A token's picks are found by k
// maxima over its lanes; ranks among the tokens of a round come from one bit a
// token and expert in shared memory (set in any order, counted by popc), so there
// is no sort.  With one block of one round the rows are final, else they count
// from the block's first pick of the expert and route_place adds the rest.
template <typename T, int LPT, int VPL>
__global__ void __launch_bounds__(VPL <= 8 ? 1024 : VPL == 16 ? 512 : 256) route_pick(const RouteParams p) {
  extern __shared__ unsigned char smem[];
  const int words = p.chunk / 32, warps = blockDim.x / 32;
  uint32_t *bits = reinterpret_cast<uint32_t *>(smem);              // [e][words]
  int *count = reinterpret_cast<int *>(bits + p.e * words);         // [e + 1]
  int *first = count + p.e + 1;                                     // [e + 1]
  float *sums = reinterpret_cast<float *>(first + p.e + 1);         // [warps][e]
  float *pick_w = sums + warps * p.e;                               // [chunk][k]
  float *total = pick_w + p.chunk * p.k;                            // [chunk]
  int *held = reinterpret_cast<int *>(total + p.chunk);
  int16_t *pick_e = reinterpret_cast<int16_t *>(held + 1);          // [chunk][k]

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, l = lane % LPT;
  constexpr int GROUPS = 32 / LPT;
  start_after_earlier_kernels();
  if (threadIdx.x == 0) *held = 0;
  for (int e = threadIdx.x; e <= p.e; e += blockDim.x) count[e] = first[e] = 0;
  float acc[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) acc[i] = 0.f;

  for (int round = 0; round < p.per; ++round) {
    const int64_t t0 = ((int64_t)blockIdx.x * p.per + round) * p.chunk;
    if (t0 >= p.rows) break;
    const int here = (int)min((int64_t)p.chunk, p.rows - t0);
    for (int i = threadIdx.x; i < p.e * words; i += blockDim.x) bits[i] = 0;
    __syncthreads();
    for (int w0 = warp * GROUPS; w0 < here; w0 += warps * GROUPS) {
      const int tl = w0 + lane / LPT;
      float v[VPL];
      Row<T, LPT, VPL>::load(p, t0 + tl, tl < here, l, v);
      uint32_t key[VPL], best = 0;
      int at = 0;
      auto rescan = [&]() {
        best = 0;
        at = 0;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
          if (key[i] > best) {
            best = key[i];
            at = i;
          }
      };
#pragma unroll
      for (int i = 0; i < VPL; ++i) key[i] = ordered(v[i]);
      rescan();
      // the largest of all lanes and its expert
      auto largest = [&](uint32_t &m, int &e) {
        m = best;
        e = at * LPT + l;
        if constexpr (LPT == 32) {
          m = __reduce_max_sync(0xffffffffu, best);
          e = (int)__reduce_min_sync(0xffffffffu, best == m ? (uint32_t)e : 0xFFFFu);
        } else {
#pragma unroll
          for (int o = LPT / 2; o > 0; o /= 2) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, m, o);
            const int index = __shfl_xor_sync(0xffffffffu, e, o);
            if (other > m || (other == m && index < e)) {
              m = other;
              e = index;
            }
          }
        }
      };
      uint32_t m;
      int e;
      largest(m, e);
      const bool real_row = m > kNothing;
      const float top = real_row ? unordered(m) : 0.f;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        v[i] = expf(v[i] - top);
        sum += v[i];
      }
      sum = lanes_sum<LPT>(sum);
      const float inverse = real_row ? 1.f / sum : 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) acc[i] += real_row ? v[i] * inverse : 0.f;
      float picked = 0.f;
      for (int j = 0; j < p.k; ++j) {
        if (j) largest(m, e);
        const bool real = m > kNothing;
        const float x = real ? expf(unordered(m) - top) : 0.f;
        picked += x;
        if (l == 0 && tl < here) {
          pick_e[tl * p.k + j] = real ? (int16_t)e : (int16_t)-1;
          pick_w[tl * p.k + j] = x;
          if (real) atomicOr(&bits[e * words + tl / 32], 1u << (tl % 32));
        }
        if (e % LPT == l) {
#pragma unroll
          for (int i = 0; i < VPL; ++i)
            if (i == e / LPT) key[i] = 0;
          rescan();
        }
        __syncwarp();
      }
      if (l == 0 && tl < here) {
        total[tl] = real_row ? (p.normalize ? picked : sum) : 1.f;
        if (real_row) atomicAdd(held, 1);
      }
    }
    __syncthreads();
    const bool alone = p.blocks == 1;
    if (alone) {
      for (int e = threadIdx.x; e < p.e; e += blockDim.x) {
        int n = 0;
        for (int w = 0; w < words; ++w) n += __popc(bits[e * words + w]);
        count[e] = first[e] = n;
      }
      __syncthreads();
      scan(first, p.e);
    }
    for (int i = threadIdx.x; i < here * p.k; i += blockDim.x) {
      const int e = pick_e[i], tl = i / p.k;
      const int64_t to = t0 * p.k + i;
      p.experts[to] = e;
      p.weights[to] = pick_w[i] / total[tl];
      int rank = -1;
      if (e >= 0) {
        rank = alone ? first[e] : count[e];
        for (int w = 0; w < tl / 32; ++w) rank += __popc(bits[e * words + w]);
        rank += __popc(bits[e * words + tl / 32] & ((1u << (tl % 32)) - 1));
      }
      p.slots[to] = rank;
    }
    __syncthreads();
    if (!alone) {
      for (int e = threadIdx.x; e < p.e; e += blockDim.x) {
        int n = count[e];
        for (int w = 0; w < words; ++w) n += __popc(bits[e * words + w]);
        count[e] = n;
      }
      __syncthreads();
    }
  }
  // sums of p over the groups of a warp, then over the warps
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
#pragma unroll
    for (int o = LPT; o < 32; o *= 2) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    if (lane < LPT && i * LPT + l < p.e) sums[warp * p.e + i * LPT + l] = acc[i];
  }
  __syncthreads();
  if (p.blocks > 1) {
    for (int e = threadIdx.x; e < p.e; e += blockDim.x) {
      float s = 0.f;
      for (int w = 0; w < warps; ++w) s += sums[w * p.e + e];
      p.psum[(int64_t)blockIdx.x * p.e + e] = s;
      p.hist[(int64_t)blockIdx.x * p.e + e] = count[e];
    }
    if (threadIdx.x == 0) p.held[blockIdx.x] = *held;
    return;
  }
  for (int e = threadIdx.x; e <= p.e; e += blockDim.x) {
    p.offsets[e] = first[e];
    if (e < p.e) p.counts[e] = count[e];
  }
  if (threadIdx.x < 32) {
    double s = 0;
    for (int e = lane; e < p.e; e += 32)
      for (int w = 0; w < warps; ++w) s += (double)count[e] * sums[w * p.e + e];
#pragma unroll
    for (int o = 16; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      *p.tokens = *held;
      *p.loss = *held ? (float)(p.e * s / ((double)first[p.e] * *held)) : 0.f;
    }
  }
}

// The rows of each block's picks: its first of an expert follows those of the
// blocks before it.  Every block adds up the counts of all blocks for itself; the
// last one (of blocks + 1) writes offsets, counts and loss.
__global__ void __launch_bounds__(512) route_place(const RouteParams p) {
  extern __shared__ unsigned char smem[];
  const int groups = max(1, (int)blockDim.x / p.e);
  int *total = reinterpret_cast<int *>(smem);                       // [e + 1]
  int *base = total + p.e + 1;                                      // [e]
  int *part = base + p.e + 1;                                       // [2][groups][e]
  start_after_earlier_kernels();
  const bool last = blockIdx.x == p.blocks;
  const int lanes = groups * p.e;                                   // threads at work where e < blockDim
  for (int i = threadIdx.x; i < lanes; i += blockDim.x) {
    const int e = i % p.e, g = i / p.e;
    int all = 0, before = 0;
#pragma unroll 8
    for (int b = g; b < p.blocks; b += groups) {
      const int n = __ldg(p.hist + (int64_t)b * p.e + e);
      all += n;
      before += b < (int)blockIdx.x ? n : 0;
    }
    part[g * p.e + e] = all;
    part[(groups + g) * p.e + e] = before;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.e; e += blockDim.x) {
    int all = 0, before = 0;
    for (int g = 0; g < groups; ++g) {
      all += part[g * p.e + e];
      before += part[(groups + g) * p.e + e];
    }
    total[e] = all;
    base[e] = before;
  }
  __syncthreads();
  scan(total, p.e);
  if (!last) {
    const int64_t span = (int64_t)p.chunk * p.per * p.k, i0 = blockIdx.x * span;
    const int64_t end = min(i0 + span, p.rows * p.k);
    for (int64_t i = i0 + threadIdx.x; i < end; i += blockDim.x) {
      const int e = p.experts[i];
      if (e >= 0) p.slots[i] += total[e] + base[e];
    }
    return;
  }
  for (int e = threadIdx.x; e <= p.e; e += blockDim.x) {
    p.offsets[e] = total[e];
    if (e < p.e) p.counts[e] = total[e + 1] - total[e];
  }
  double s = 0;
  int tokens = 0;
  for (int i = threadIdx.x; i < lanes; i += blockDim.x) {
    const int e = i % p.e, g = i / p.e;
    double q = 0;
#pragma unroll 8
    for (int b = g; b < p.blocks; b += groups) q += __ldg(p.psum + (int64_t)b * p.e + e);
    s += q * (total[e + 1] - total[e]);
  }
  for (int b = threadIdx.x; b < p.blocks; b += blockDim.x) tokens += p.held[b];
#pragma unroll
  for (int o = 16; o > 0; o /= 2) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
  }
  __shared__ double warp_s[16];
  __shared__ int warp_n[16];
  if (threadIdx.x % 32 == 0) {
    warp_s[threadIdx.x / 32] = s;
    warp_n[threadIdx.x / 32] = tokens;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0;
    tokens = 0;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) {
      s += warp_s[w];
      tokens += warp_n[w];
    }
    *p.tokens = tokens;
    *p.loss = tokens ? (float)(p.e * s / ((double)total[p.e] * tokens)) : 0.f;
  }
}

// Lanes of a token and values of a lane for e experts, then f.run<T, LPT, VPL>().
template <typename T, typename F> int with_layout(int e, F f) {
  if (e <= 8) return f.template run<T, 1, 8>();
  if (e <= 16) return f.template run<T, 2, 8>();
  if (e <= 32) return f.template run<T, 4, 8>();
  if (e <= 64) return f.template run<T, 8, 8>();
  if (e <= 128) return f.template run<T, 16, 8>();
  if (e <= 256) return f.template run<T, 32, 8>();
  if (e <= 512) return f.template run<T, 32, 16>();
  return f.template run<T, 32, 32>();
}

struct RoutePlan { int chunk, per, blocks; };
// Rounds of 256 tokens, or fewer (down to 32) while that leaves SMs without a block.
RoutePlan route_plan(int64_t rows, int e) {
  const int lpt = e <= 8 ? 1 : e <= 256 ? (e <= 16 ? 2 : e <= 32 ? 4 : e <= 64 ? 8 : e <= 128 ? 16 : 32) : 32;
  const int most = e <= 256 ? 1024 : e <= 512 ? 512 : 256;
  RoutePlan r{kMaxChunk, 1, 1};
  if (rows <= kMaxChunk && rows <= 4 * most / lpt) {
    r.chunk = (int)((rows + 31) / 32 * 32);
    return r;
  }
  while (r.chunk > 32 && (rows + r.chunk - 1) / r.chunk < 128) r.chunk /= 2;
  const int64_t rounds = (rows + r.chunk - 1) / r.chunk;
  r.per = (int)((rounds + 511) / 512);
  r.blocks = (int)((rounds + r.per - 1) / r.per);
  return r;
}

struct PickLaunch {
  const RouteParams &p;
  cudaStream_t st;
  template <typename T, int LPT, int VPL> int run() const {
    const int most = VPL <= 8 ? 1024 : VPL == 16 ? 512 : 256;
    const int64_t busy = min((int64_t)p.chunk, p.rows) * LPT;
    const int threads = (int)max((int64_t)32, min((int64_t)most, (busy + 31) / 32 * 32));
    return launch(route_pick<T, LPT, VPL>, dim3(p.blocks), threads, route_smem(p.e, p.k, p.chunk, threads / 32), st,
                  "route_pick launch", p);
  }
};

struct RouteBackward {
  const void *logits;
  const float *dweights, *dloss, *weights;
  const int *experts, *counts, *tokens;
  void *dlogits;
  int64_t rows, row, col;
  int e, k, normalize;
};

// dlogits, LPT lanes a token: the softmax again from the logits, the picks' part
// added by the lanes that hold them.
template <typename T, int LPT, int VPL>
__global__ void __launch_bounds__(256) route_backward(const RouteBackward p) {
  extern __shared__ unsigned char smem[];
  float *slope = reinterpret_cast<float *>(smem);                   // [e]: the loss's part of g
  constexpr int GROUPS = 32 / LPT;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, l = lane % LPT;
  start_after_earlier_kernels();
  // sum of the counts, by every warp for itself
  int sum_n = 0;
  for (int e = lane; e < p.e; e += 32) sum_n += p.counts[e];
#pragma unroll
  for (int o = 16; o > 0; o /= 2) sum_n += __shfl_xor_sync(0xffffffffu, sum_n, o);
  const int tokens = *p.tokens;
  const double scale = p.dloss && tokens > 0 && sum_n > 0 ? (double)*p.dloss * p.e / ((double)tokens * sum_n) : 0.0;
  for (int e = threadIdx.x; e < p.e; e += blockDim.x) slope[e] = (float)(scale * p.counts[e]);
  __syncthreads();
  const int64_t step = (int64_t)gridDim.x * (blockDim.x / 32) * GROUPS;
  for (int64_t w0 = ((int64_t)blockIdx.x * (blockDim.x / 32) + warp) * GROUPS; w0 < p.rows; w0 += step) {
    const int64_t t = w0 + lane / LPT;
    const bool there = t < p.rows;
    float v[VPL];
    const T *from = static_cast<const T *>(p.logits) + t * p.row;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = i * LPT + l;
      v[i] = there && e < p.e ? to_f32(from[e * p.col]) : -INFINITY;
    }
    float top = v[0];
    bool odd = false;                                               // a NaN makes the sum one
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      top = fmaxf(top, v[i]);
      odd |= v[i] != v[i];
    }
    top = over_lanes<LPT>(top, [](float a, float b) { return fmaxf(a, b); });
    const bool real = top > -INFINITY;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      v[i] = real || odd ? expf(v[i] - top) : 0.f;
      sum += v[i];
    }
    sum = lanes_sum<LPT>(sum);
    const float inverse = sum != 0.f ? 1.f / sum : 0.f;
    float inner = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      v[i] *= inverse;
      const int e = i * LPT + l;
      inner += v[i] * (e < p.e ? slope[e] : 0.f);
    }
    inner = lanes_sum<LPT>(inner);
    // what the picks add: w dw over the row
    float dot = 0.f;
    if (p.dweights && there)
      for (int j = l; j < p.k; j += LPT)
        if (p.experts[t * p.k + j] >= 0) dot += p.weights[t * p.k + j] * p.dweights[t * p.k + j];
    dot = lanes_sum<LPT>(dot);
    if (!p.normalize) inner += dot;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = i * LPT + l;
      v[i] *= (e < p.e ? slope[e] : 0.f) - inner;
    }
    if (p.dweights && there)
      for (int j = 0; j < p.k; ++j) {
        const int e = p.experts[t * p.k + j];
        if (e < 0 || e % LPT != l) continue;
        const float w = p.weights[t * p.k + j], d = p.dweights[t * p.k + j];
        const float add = p.normalize ? w * (d - dot) : w * d;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
          if (i == e / LPT) v[i] += add;
      }
    T *to = static_cast<T *>(p.dlogits) + t * p.e;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = i * LPT + l;
      if (there && e < p.e) to[e] = from_f32<T>(v[i]);
    }
  }
}

struct BackwardLaunch {
  const RouteBackward &p;
  cudaStream_t st;
  template <typename T, int LPT, int VPL> int run() const {
    const int64_t blocks = (p.rows * LPT + 255) / 256;
    return launch(route_backward<T, LPT, VPL>, dim3((unsigned)min(blocks, (int64_t)sm_count() * 8)), 256, p.e * 4, st,
                  "route_backward launch", p);
  }
};

// ---------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------
struct RowsParams {
  const void *x, *rows;        // of tokens; of picks
  void *x_out, *rows_out;
  const int *slots, *offsets;
  const float *weights;
  float *dweights;
  int64_t tokens, row_count, x_row, rows_row;   // row pitches of the inputs
  int d, k, experts;
};

// A slot that is a row, else -1.
__device__ __forceinline__ int64_t slot_of(const RowsParams &p, int64_t pick) {
  const int s = __ldg(p.slots + pick);
  return s >= 0 && s < p.row_count ? s : -1;
}

// Zeros in the rows after the last pick's, by the blocks from `first` on.
template <typename T, int V> __device__ __forceinline__ void clear_rest(const RowsParams &p, int first) {
  const int64_t n = p.d / V, end = p.row_count * n;
  const int64_t from = min(max((int64_t)__ldg(p.offsets + p.experts), (int64_t)0), p.row_count) * n;
  float zero[V] = {};
  for (int64_t i = from + (int64_t)(blockIdx.x - first) * blockDim.x + threadIdx.x; i < end;
       i += (int64_t)(gridDim.x - first) * blockDim.x)
    Run<T, V>::store(static_cast<T *>(p.rows_out) + i * V, zero);
}

// How the threads of a block lie over tokens and columns: `tokens` tokens side by side,
// `threads` threads each, which take the columns in steps of threads * V.
struct Spread { int tokens, threads; };

// The slots of a token's picks, -1 where there is no row, loaded ahead of the rows they name.
template <int K> struct Picks {
  int slot[K];
  __device__ __forceinline__ void load(const RowsParams &p, int64_t t, int j0) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      slot[j] = -1;
      if (t < p.tokens && j0 + j < p.k) {
        const int s = __ldg(p.slots + t * p.k + j0 + j);
        slot[j] = s >= 0 && s < p.row_count ? s : -1;
      }
    }
  }
};

template <typename T, int V> __global__ void __launch_bounds__(256, 6) dispatch_kernel(const RowsParams p, const Spread at,
                                                                                       int blocks) {
  start_after_earlier_kernels();
  if ((int)blockIdx.x >= blocks) return clear_rest<T, V>(p, blocks);
  const int group = (int)threadIdx.x / at.threads, in = (int)threadIdx.x - group * at.threads;
  if (group >= at.tokens) return;
  for (int64_t t = (int64_t)blockIdx.x * at.tokens + group; t < p.tokens; t += (int64_t)blocks * at.tokens) {
    for (int c = in * V; c < p.d; c += at.threads * V) {
      const auto v = Raw<T, V>::load(static_cast<const T *>(p.x) + t * p.x_row + c);
      T *to = static_cast<T *>(p.rows_out) + c;
#pragma unroll 4
      for (int j = 0; j < p.k; ++j) {
        const int64_t s = slot_of(p, t * p.k + j);
        if (s >= 0) Raw<T, V>::store(to + s * p.d, v);
      }
    }
  }
}

// y[t] = sum_j w rows[slot], in the order of j, K loads on their way at a time; the next
// token's slots are loaded before this one's rows arrive.
template <typename T, int V, int K> __global__ void __launch_bounds__(256, K >= 8 ? 3 : K >= 4 ? 4 : 5) combine_kernel(
    const RowsParams p, const Spread at) {
  start_after_earlier_kernels();
  const int group = (int)threadIdx.x / at.threads, in = (int)threadIdx.x - group * at.threads;
  if (group >= at.tokens) return;
  const int64_t step = (int64_t)gridDim.x * at.tokens;
  int64_t t = (int64_t)blockIdx.x * at.tokens + group;
  Picks<K> picks, next;
  picks.load(p, t, 0);
  for (; t < p.tokens; t += step) {
    next.load(p, t + step, 0);
#pragma unroll 1
    for (int c = in * V; c < p.d; c += at.threads * V) {
      const T *from = static_cast<const T *>(p.rows) + c;
      float y[V] = {};
#pragma unroll 1
      for (int j0 = 0; j0 < p.k; j0 += K) {
        if (p.k > K) picks.load(p, t, j0);
        typename Raw<T, V>::Type v[K];
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (picks.slot[j] >= 0) v[j] = Raw<T, V>::load(from + (int64_t)picks.slot[j] * p.rows_row);
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (picks.slot[j] >= 0) {
            const float w = p.weights ? __ldg(p.weights + t * p.k + j0 + j) : 1.f;
            float u[V];
            Raw<T, V>::values(v[j], u);
#pragma unroll
            for (int i = 0; i < V; ++i) y[i] = fmaf(w, u[i], y[i]);
          }
      }
      Run<T, V>::store(static_cast<T *>(p.x_out) + t * p.d + c, y);
    }
    picks = next;
  }
}

// drows[slot] = w dy[t], dw[t, j] = dy[t] . rows[slot]: `at.threads` threads (whole warps) a
// token, K picks at a time.
template <typename T, int V, int K>
__global__ void __launch_bounds__(256, 3) combine_backward_kernel(const RowsParams p, const Spread at, int blocks) {
  __shared__ float sums[8][K];
  start_after_earlier_kernels();
  if ((int)blockIdx.x >= blocks) return clear_rest<T, V>(p, blocks);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, parts = at.threads / 32;
  const int group = warp / parts, in = (int)threadIdx.x - group * at.threads;
  const int64_t step = (int64_t)blocks * at.tokens;
  int64_t t = (int64_t)blockIdx.x * at.tokens + group;
  Picks<K> picks, next;
  picks.load(p, t, 0);
  // every warp takes part in every round: the sums are shared
  for (int64_t t0 = (int64_t)blockIdx.x * at.tokens; t0 < p.tokens; t0 += step, t += step) {
    next.load(p, t + step, 0);
    for (int j0 = 0; j0 < p.k; j0 += K) {
      if (j0) picks.load(p, t, j0);
      float dot[K], weight[K];
#pragma unroll
      for (int j = 0; j < K; ++j) {
        dot[j] = 0.f;
        weight[j] = picks.slot[j] >= 0 ? __ldg(p.weights + t * p.k + j0 + j) : 0.f;
      }
      if (t < p.tokens) {
        for (int c = in * V; c < p.d; c += at.threads * V) {
          typename Raw<T, V>::Type v[K];
          const auto raw = Raw<T, V>::load(static_cast<const T *>(p.x) + t * p.x_row + c);
#pragma unroll
          for (int j = 0; j < K; ++j)
            if (picks.slot[j] >= 0)
              v[j] = Raw<T, V>::load(static_cast<const T *>(p.rows) + (int64_t)picks.slot[j] * p.rows_row + c);
          float dy[V];
          Raw<T, V>::values(raw, dy);
#pragma unroll
          for (int j = 0; j < K; ++j) {
            if (picks.slot[j] < 0) continue;
            float u[V];
            Raw<T, V>::values(v[j], u);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              dot[j] = fmaf(dy[i], u[i], dot[j]);
              u[i] = weight[j] * dy[i];
            }
            Run<T, V>::store(static_cast<T *>(p.rows_out) + (int64_t)picks.slot[j] * p.d + c, u);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < K; ++j) {
#pragma unroll
        for (int o = 16; o > 0; o /= 2) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
        if (parts > 1 && lane == 0) sums[warp][j] = dot[j];
      }
      if (parts == 1) {
        if (t < p.tokens && lane == 0)
#pragma unroll
          for (int j = 0; j < K; ++j)
            if (j0 + j < p.k) p.dweights[t * p.k + j0 + j] = dot[j];
      } else {
        __syncthreads();
        if (in < K && j0 + in < p.k && t < p.tokens) {
          float all = 0.f;
          for (int w = 0; w < parts; ++w) all += sums[warp + w][in];
          p.dweights[t * p.k + j0 + in] = all;
        }
        __syncthreads();
      }
    }
    picks = next;
  }
}

// Threads for a token's `runs` runs of V columns, whole warps where `warps`, and blocks
// for all tokens: as many as the GPU holds, so that each takes several tokens in turn.
Spread spread_over(int64_t runs, int64_t tokens, bool warps, int resident, int64_t &blocks) {
  Spread s;
  if (warps) {
    // 3 steps over a row and more: a warp's sums cost 5 exchanges a pick however long they are
    s.threads = runs <= 96 ? 32 : runs <= 192 ? 64 : runs <= 640 ? 128 : 256;
  } else {
    // the fewest steps over a row that fit, with as few idle threads as may be
    const int64_t steps = (runs + 255) / 256;
    s.threads = (int)((runs + steps - 1) / steps);
  }
  s.tokens = 256 / s.threads;
  blocks = std::min<int64_t>((tokens + s.tokens - 1) / s.tokens, (int64_t)sm_count() * resident);
  return s;
}

bool vectors_ok(const void *base, int64_t pitch, int64_t rows, int es) {
  return (uintptr_t)base % 16 == 0 && (rows <= 1 || pitch * es % 16 == 0);
}

int check_rows(const oz_rows_args &a) {
  if (a.tokens < 0 || a.d < 0 || a.experts < 1 || a.picks < 1)
    return set_error(OZ_ERR_INVALID, "bad size (tokens=%lld d=%lld experts=%d picks=%d)", (long long)a.tokens,
                     (long long)a.d, a.experts, a.picks);
  if (a.dtype != OZ_F32 && a.dtype != OZ_F16 && a.dtype != OZ_BF16)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported dtype %d (fp32, fp16 or bf16)", a.dtype);
  if (a.tokens * a.picks > INT32_MAX / 2 || a.d > (1 << 24) || a.picks > kMaxPicks)
    return set_error(OZ_ERR_INVALID, "size out of range");
  return OZ_OK;
}

constexpr int kClearBlocks = 64;     // zero the rows that no pick has

}  // namespace
}  // namespace oz

extern "C" int64_t oz_route_workspace_bytes(int64_t rows, int32_t experts) {
  using namespace oz;
  if (rows < 0 || experts < 1 || experts > kMaxExperts) return OZ_ERR_INVALID;
  const RoutePlan r = route_plan(rows, experts);
  return r.blocks <= 1 ? 0 : (int64_t)r.blocks * (experts * 8 + 4);
}

extern "C" int oz_route(const oz_route_args *args, void *stream) {
  if (!args) return oz::set_error(OZ_ERR_INVALID, "null arguments");
  using namespace oz;
  const oz_route_args &a = *args;
  if (a.rows < 0) return set_error(OZ_ERR_INVALID, "negative size");
  if (a.experts < 1 || a.experts > kMaxExperts)
    return set_error(OZ_ERR_INVALID, "experts must be in [1, %d], got %d", kMaxExperts, a.experts);
  if (a.picks < 1 || a.picks > kMaxPicks || a.picks > a.experts)
    return set_error(OZ_ERR_INVALID, "picks must be in [1, %d] and at most the experts, got %d", kMaxPicks, a.picks);
  if (a.rows * a.picks > INT32_MAX / 2) return set_error(OZ_ERR_INVALID, "size out of range");
  if (!a.offsets || !a.counts || !a.tokens || !a.loss || (a.rows > 0 && (!a.logits || !a.weights || !a.chosen || !a.slots)))
    return set_error(OZ_ERR_INVALID, "null pointer");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const RoutePlan r = route_plan(a.rows, a.experts);
  const int64_t bytes = oz_route_workspace_bytes(a.rows, a.experts);
  if (bytes && (!a.workspace || (uintptr_t)a.workspace % 16 != 0 || a.workspace_bytes < bytes))
    return set_error(OZ_ERR_INVALID, "workspace of %lld bytes (16-byte aligned) needed, got %lld at %p",
                     (long long)bytes, (long long)a.workspace_bytes, a.workspace);
  RouteParams p{a.logits, a.weights, a.loss, a.chosen, a.slots, a.offsets, a.counts, a.tokens, nullptr, nullptr,
                nullptr, a.rows, a.row, a.col, a.experts, a.picks, a.normalize, r.chunk, r.per, r.blocks};
  if (p.chunk == 0) p.chunk = 32;
  if (bytes) {
    p.hist = static_cast<int *>(a.workspace);
    p.psum = reinterpret_cast<float *>(p.hist + (int64_t)r.blocks * a.experts);
    p.held = reinterpret_cast<int *>(p.psum + (int64_t)r.blocks * a.experts);
  }
  const int rc = with_type(a.dtype, [&](auto v) { return with_layout<decltype(v)>(a.experts, PickLaunch{p, st}); });
  if (rc || r.blocks <= 1) return rc;
  const int groups = max(1, 512 / a.experts);
  return launch(route_place, dim3(r.blocks + 1), 512, 4 * (2 * (a.experts + 1) + 2 * groups * a.experts), st,
                "route_place launch", p);
}

extern "C" int oz_route_backward(const oz_route_backward_args *args, void *stream) {
  if (!args) return oz::set_error(OZ_ERR_INVALID, "null arguments");
  using namespace oz;
  const oz_route_backward_args &a = *args;
  if (a.rows < 0) return set_error(OZ_ERR_INVALID, "negative size");
  if (a.experts < 1 || a.experts > kMaxExperts || a.picks < 1 || a.picks > kMaxPicks || a.picks > a.experts)
    return set_error(OZ_ERR_INVALID, "bad size (experts=%d picks=%d)", a.experts, a.picks);
  if (a.rows * a.picks > INT32_MAX / 2) return set_error(OZ_ERR_INVALID, "size out of range");
  if (a.rows == 0) return OZ_OK;
  if (!a.logits || !a.weights || !a.chosen || !a.counts || !a.tokens || !a.dlogits)
    return set_error(OZ_ERR_INVALID, "null pointer");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const RouteBackward p{a.logits, a.dweights, a.dloss, a.weights, a.chosen, a.counts, a.tokens, a.dlogits,
                        a.rows, a.row, a.col, a.experts, a.picks, a.normalize};
  return with_type(a.dtype, [&](auto v) { return with_layout<decltype(v)>(a.experts, BackwardLaunch{p, st}); });
}

extern "C" int oz_dispatch(const oz_rows_args *args, void *stream) {
  if (!args) return oz::set_error(OZ_ERR_INVALID, "null arguments");
  using namespace oz;
  const oz_rows_args &a = *args;
  if (int rc = check_rows(a)) return rc;
  if (a.tokens == 0 || a.d == 0) return OZ_OK;
  if (!a.x || !a.rows_out || !a.slots || !a.offsets) return set_error(OZ_ERR_INVALID, "null pointer");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  RowsParams p{a.x, nullptr, nullptr, a.rows_out, a.slots, a.offsets, nullptr, nullptr, a.tokens, a.tokens * a.picks,
               a.x_row, 0, (int)a.d, a.picks, a.experts};
  return with_type(a.dtype, [&](auto z) {
    using T = decltype(z);
    constexpr int ES = sizeof(T);
    const bool wide = vectors_ok(a.x, a.x_row, a.tokens, ES) && vectors_ok(a.rows_out, a.d, a.tokens * a.picks, ES) &&
                      a.d * ES % 16 == 0;
    int64_t blocks;
    const Spread at = spread_over(a.d / (wide ? 16 / ES : 1), a.tokens, false, 6, blocks);
    const dim3 grid((unsigned)(blocks + kClearBlocks));
    return wide ? launch(dispatch_kernel<T, 16 / ES>, grid, 256, 0, st, "dispatch_kernel launch", p, at, (int)blocks)
                : launch(dispatch_kernel<T, 1>, grid, 256, 0, st, "dispatch_kernel launch", p, at, (int)blocks);
  });
}

extern "C" int oz_combine(const oz_rows_args *args, void *stream) {
  if (!args) return oz::set_error(OZ_ERR_INVALID, "null arguments");
  using namespace oz;
  const oz_rows_args &a = *args;
  if (int rc = check_rows(a)) return rc;
  if (a.tokens == 0 || a.d == 0) return OZ_OK;
  if (!a.rows || !a.x_out || !a.slots) return set_error(OZ_ERR_INVALID, "null pointer");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  RowsParams p{nullptr, a.rows, a.x_out, nullptr, a.slots, nullptr, a.weights, nullptr, a.tokens, a.tokens * a.picks,
               0, a.rows_row, (int)a.d, a.picks, a.experts};
  return with_type(a.dtype, [&](auto z) {
    using T = decltype(z);
    constexpr int ES = sizeof(T);
    const bool wide = vectors_ok(a.rows, a.rows_row, a.tokens * a.picks, ES) && vectors_ok(a.x_out, a.d, a.tokens, ES) &&
                      a.d * ES % 16 == 0;
    int64_t blocks;
    const Spread at = spread_over(a.d / (wide ? 16 / ES : 1), a.tokens, false, a.picks > 4 ? 3 : a.picks > 2 ? 4 : 5, blocks);
    auto with = [&](auto k) {
      constexpr int K = decltype(k)::value;
      const dim3 grid((unsigned)blocks);
      return wide ? launch(combine_kernel<T, 16 / ES, K>, grid, 256, 0, st, "combine_kernel launch", p, at)
                  : launch(combine_kernel<T, 1, K>, grid, 256, 0, st, "combine_kernel launch", p, at);
    };
    if (a.picks <= 2) return with(std::integral_constant<int, 2>{});
    if (a.picks <= 4) return with(std::integral_constant<int, 4>{});
    return with(std::integral_constant<int, 8>{});
  });
}

extern "C" int oz_combine_backward(const oz_rows_args *args, void *stream) {
  if (!args) return oz::set_error(OZ_ERR_INVALID, "null arguments");
  using namespace oz;
  const oz_rows_args &a = *args;
  if (int rc = check_rows(a)) return rc;
  if (a.tokens == 0) return OZ_OK;
  if (!a.slots || !a.offsets || !a.weights || !a.dweights || (a.d > 0 && (!a.x || !a.rows || !a.rows_out)))
    return set_error(OZ_ERR_INVALID, "null pointer");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  RowsParams p{a.x, a.rows, nullptr, a.rows_out, a.slots, a.offsets, a.weights, a.dweights, a.tokens,
               a.tokens * a.picks, a.x_row, a.rows_row, (int)a.d, a.picks, a.experts};
  return with_type(a.dtype, [&](auto z) {
    using T = decltype(z);
    constexpr int ES = sizeof(T);
    const int64_t n = a.tokens * a.picks;
    const bool wide = vectors_ok(a.x, a.x_row, a.tokens, ES) && vectors_ok(a.rows, a.rows_row, n, ES) &&
                      vectors_ok(a.rows_out, a.d, n, ES) && a.d * ES % 16 == 0;
    int64_t blocks;
    const Spread at = spread_over(a.d / (wide ? 16 / ES : 1), a.tokens, true, 3, blocks);
    const dim3 grid((unsigned)(blocks + kClearBlocks));
    const char *what = "combine_backward_kernel launch";
    return wide ? launch(combine_backward_kernel<T, 16 / ES, 4>, grid, 256, 0, st, what, p, at, (int)blocks)
                : launch(combine_backward_kernel<T, 1, 4>, grid, 256, 0, st, what, p, at, (int)blocks);
  });
}
