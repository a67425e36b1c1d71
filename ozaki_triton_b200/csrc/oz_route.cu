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

// Whole numbers in the order of fp32 values: NaN above all (an addition gives the positive
// one), the two zeros equal.
__device__ __forceinline__ int key_of(float f) {
  const int u = __float_as_int(f + 0.f);
  return u ^ (u >> 31 & 0x7FFFFFFF);
}
// exp(x) for x <= 0: off by |x| + 3 units of 2^-24 of its value.
__device__ __forceinline__ float exp_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}

// Where logits lie: LPT lanes take a token, 4 consecutive experts each in turn, so lane l's
// element 4 q + x is expert 4 (q LPT + l) + x.
struct Logits {
  const void *p;
  int64_t rows, row, col;
  int e, dtype, vectors;       // rows may be read 4 elements at a time
};
template <int LPT> __device__ __forceinline__ int expert_of(int i, int l) { return (i / 4 * LPT + l) * 4 + i % 4; }

template <int LPT, int VPL, typename T>
__device__ __forceinline__ void load_row(const Logits &g, int64_t t, bool there, int l, float (&v)[VPL]) {
  const T *from = static_cast<const T *>(g.p) + t * g.row;
#pragma unroll
  for (int i = 0; i < VPL; i += 4) {
    const int e = expert_of<LPT>(i, l);
    if (g.vectors) {                          // whole groups of 4
      if (there && e < g.e) {
        if constexpr (sizeof(T) == 4) {
          const float4 u = *(reinterpret_cast<const float4 *>(from + e));
          v[i] = u.x, v[i + 1] = u.y, v[i + 2] = u.z, v[i + 3] = u.w;
        } else {
          const uint2 u = *(reinterpret_cast<const uint2 *>(from + e));
          const T *w = reinterpret_cast<const T *>(&u);
#pragma unroll
          for (int x = 0; x < 4; ++x) v[i + x] = to_f32(w[x]);
        }
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) v[i + x] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) v[i + x] = there && e + x < g.e ? to_f32(from[(e + x) * g.col]) : -INFINITY;
    }
  }
}
template <int LPT, int VPL>
__device__ __forceinline__ void load_row(const Logits &g, int64_t t, bool there, int l, float (&v)[VPL]) {
  if (g.dtype == OZ_F32) load_row<LPT, VPL, float>(g, t, there, l, v);
  else if (g.dtype == OZ_F16) load_row<LPT, VPL, __half>(g, t, there, l, v);
  else load_row<LPT, VPL, __nv_bfloat16>(g, t, there, l, v);
}

__device__ __forceinline__ float logit(const Logits &g, int64_t t, int e) {
  const int64_t at = t * g.row + e * g.col;
  if (g.dtype == OZ_F32) return *(static_cast<const float *>(g.p) + at);
  if (g.dtype == OZ_F16) return to_f32(*(static_cast<const __half *>(g.p) + at));
  return to_f32(*(static_cast<const __nv_bfloat16 *>(g.p) + at));
}

struct RouteParams {
  Logits logits;
  float *weights, *loss;
  int *experts, *slots, *offsets, *counts, *tokens;
  int *hist;                   // [e][blocks]: picks of each block and expert, then those before,
  float *psum;                 // [e][blocks]: sums of p
  int *held, *all;             // tokens of each block; picks of each expert ...
  double *mass;                // ... and its sum of p
  int64_t rows;
  int e, k, normalize, chunk, per, blocks;    // tokens of a round, rounds of a block
};

template <int LPT, typename F> __device__ __forceinline__ float over_lanes(float v, F f) {
#pragma unroll
  for (int o = LPT / 2; o > 0; o /= 2) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int LPT> __device__ __forceinline__ float lanes_sum(float v) {
  return over_lanes<LPT>(v, [](float a, float b) { return a + b; });
}

// The K largest of what has been put in, the largest first, the lowest expert first among
// equals.  A key and its expert, or with PACKED (logits of 16 bits) one number for both:
// the key above, the lower the expert the larger below.
constexpr int kNone = (int)0x80000000;
template <int K, bool PACKED> struct Largest {
  int key[K], expert[PACKED ? 1 : K];
  __device__ __forceinline__ Largest() {
#pragma unroll
    for (int j = 0; j < K; ++j) key[j] = kNone;
    if constexpr (!PACKED)
#pragma unroll
      for (int j = 0; j < K; ++j) expert[j] = 0;
  }
  // The i-th element; they come in the order of their experts: an equal one goes behind, and
  // from its place on all others move by one.
  __device__ __forceinline__ void put(int i, int x, int e) {
    bool before = false;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (j > i) continue;
      const int k0 = key[j];
      if constexpr (PACKED) {
        key[j] = max(k0, x);
        x = min(k0, x);
      } else {
        const int e0 = expert[j];
        before = before || x > k0;
        key[j] = before ? x : k0;
        expert[j] = before ? e : e0;
        x = before ? k0 : x;
        e = before ? e0 : e;
      }
    }
  }
  __device__ __forceinline__ bool precedes(int k0, int e0, int k1, int e1) const {
    if constexpr (PACKED) return k0 > k1;
    else return k0 > k1 || (k0 == k1 && e0 < e1);
  }
  // Joins the lists of LPT lanes: of two sorted lists the better of the j-th and the
  // other's j-th from the end are the K best, falling then rising, and are sorted in
  // log K steps.  Both lanes of a pair end with the same list.
  template <int LPT> __device__ __forceinline__ void join() {
#pragma unroll 1
    for (int o = 1; o < LPT; o *= 2) {
      int k1[K], e1[PACKED ? 1 : K];
#pragma unroll
      for (int j = 0; j < K; ++j) {
        k1[j] = __shfl_xor_sync(0xffffffffu, key[K - 1 - j], o);
        if constexpr (!PACKED) e1[j] = __shfl_xor_sync(0xffffffffu, expert[K - 1 - j], o);
      }
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if constexpr (PACKED) key[j] = max(key[j], k1[j]);
        else if (precedes(k1[j], e1[j], key[j], expert[j])) key[j] = k1[j], expert[j] = e1[j];
      }
#pragma unroll
      for (int s = K / 2; s > 0; s /= 2)
#pragma unroll
        for (int j = 0; j < K; ++j) {
          if (j & s) continue;
          const int k0 = key[j];
          if constexpr (PACKED) {
            key[j] = max(k0, key[j + s]);
            key[j + s] = min(k0, key[j + s]);
          } else if (precedes(key[j + s], expert[j + s], k0, expert[j])) {
            const int e0 = expert[j];
            key[j] = key[j + s], expert[j] = expert[j + s];
            key[j + s] = k0, expert[j + s] = e0;
          }
        }
    }
  }
  // exp(value - high) of the j-th, 0 where there is none
  __device__ __forceinline__ float share(int j, float high, int dtype) const {
    if (key[j] == kNone) return 0.f;
    float v;
    if constexpr (PACKED) {
      const int k16 = key[j] & (int)0xFFFF0000, bits = k16 ^ (k16 >> 31 & 0x7FFF0000);
      v = dtype == OZ_F16 ? __half2float(__ushort_as_half((unsigned short)((uint32_t)bits >> 16))) : __int_as_float(bits);
    } else {
      v = __int_as_float(key[j] ^ (key[j] >> 31 & 0x7FFFFFFF));
    }
    return exp_of(v - high);
  }
  __device__ __forceinline__ int chosen(int j) const {
    if (key[j] == kNone) return -1;
    if constexpr (PACKED) return 0xFFFF - (key[j] & 0xFFFF);
    else return expert[j];
  }
};
// An element's key; none for -inf and past the last expert.
template <bool PACKED> __device__ __forceinline__ int element_key(float v, int e, int experts, int dtype) {
  if (e >= experts || v == -INFINITY) return kNone;
  if constexpr (!PACKED) return key_of(v);
  int bits;                                   // 16 of them above
  if (dtype == OZ_F16) bits = (int)((uint32_t)__half_as_ushort(__float2half_rn(v + 0.f)) << 16);
  else bits = __float_as_int(v + 0.f) & (int)0xFFFF0000;
  return (bits ^ (bits >> 31 & 0x7FFF0000)) | (0xFFFF - e);
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

constexpr int kPickThreads = 256;
int route_smem(int e, int k, int chunk) {
  return 4 * (e * (chunk / 32) + 2 * (e + 1) + kPickThreads / 32 * e + 2 * chunk + 1) + 2 * chunk * k;
}

// Picks of `per` rounds of `chunk` tokens a block.  A lane puts its part of a token's logits
// into a sorted list of K, and the LPT lanes of the token join their lists: for each expert and
// place of the list 6 instructions, or 2 for logits of 16 bits (k maxima over all lanes took 2440
// for 4 tokens of 64 experts and 8 picks).  Ranks among the tokens of a round come from
// one bit a token and expert in shared memory (set in any order, counted by popc), so there
// is no sort.  With one block of one round the rows are final, else they count from the
// block's first pick of the expert, and route_scan and route_place add the rest.  32768 tokens,
// 64 experts, 8 picks, bf16: 15 us (58 % of the issue slots), with the other two 25.
template <int LPT, int VPL, int K, bool PACKED>
__global__ void __launch_bounds__(kPickThreads, VPL == 16 && K <= 8 ? 4 : 1) route_pick(const RouteParams p) {
  extern __shared__ unsigned char smem[];
  const int words = p.chunk / 32, warps = blockDim.x / 32;
  uint32_t *bits = reinterpret_cast<uint32_t *>(smem);              // [e][words]
  int *count = reinterpret_cast<int *>(bits + p.e * words);         // [e + 1]
  int *first = count + p.e + 1;                                     // [e + 1]
  float *sums = reinterpret_cast<float *>(first + p.e + 1);         // [warps][e]
  float *top = sums + kPickThreads / 32 * p.e;                      // [chunk]
  float *total = top + p.chunk;                                     // [chunk]
  int *held = reinterpret_cast<int *>(total + p.chunk);
  int16_t *pick = reinterpret_cast<int16_t *>(held + 1);            // [chunk][k]

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, l = lane % LPT;
  constexpr int GROUPS = 32 / LPT;
  const uint32_t per_pick = ((1u << 18) + p.k - 1) / p.k;           // i / k for i < 8192: i per_pick / 2^18
  start_after_earlier_kernels();
  if (threadIdx.x == 0) *held = 0;
  for (int e = threadIdx.x; e <= p.e; e += blockDim.x) count[e] = first[e] = 0;
  for (int i = threadIdx.x; i < warps * p.e; i += blockDim.x) sums[i] = 0.f;

  for (int round = 0; round < p.per; ++round) {
    const int64_t t0 = ((int64_t)blockIdx.x * p.per + round) * p.chunk;
    if (t0 >= p.rows) break;
    const int here = (int)min((int64_t)p.chunk, p.rows - t0);
    for (int i = threadIdx.x; i < p.e * words; i += blockDim.x) bits[i] = 0;
    __syncthreads();
#pragma unroll 1
    for (int w0 = warp * GROUPS; w0 < here; w0 += warps * GROUPS) {
      const int tl = w0 + lane / LPT;
      float v[VPL];
      load_row<LPT, VPL>(p.logits, t0 + tl, tl < here, l, v);
      Largest<K, PACKED> best;
      float high = -INFINITY;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (i / 4 * 4 * LPT < p.e) {                    // the same for all lanes
          const int e = expert_of<LPT>(i, l);
          best.put(i, element_key<PACKED>(v[i], e, p.e, p.logits.dtype), e);
          high = fmaxf(high, v[i]);
        }
      best.template join<LPT>();
      high = over_lanes<LPT>(high, [](float a, float b) { return fmaxf(a, b); });
      const bool real = best.key[0] != kNone;
      if (!real) high = 0.f;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (i / 4 * 4 * LPT < p.e) {
          v[i] = exp_of(v[i] - high);
          sum += v[i];
        }
      sum = lanes_sum<LPT>(sum);
      const float inverse = real ? 1.f / sum : 0.f;
      // this warp's sums of p: over its tokens, then to those of its tokens before
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (i / 4 * 4 * LPT < p.e) {
          float q = real ? v[i] * inverse : 0.f;
#pragma unroll
          for (int o = LPT; o < 32; o *= 2) q += __shfl_xor_sync(0xffffffffu, q, o);
          const int e = expert_of<LPT>(i, l);
          if (lane < LPT && e < p.e) sums[warp * p.e + e] += q;
        }
      if (p.normalize) {
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (j < p.k) sum += best.share(j, high, p.logits.dtype);
      }
      // picks l, l + LPT, ... are this lane's to write
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (j % LPT == l && j < p.k && tl < here) pick[tl * p.k + j] = (int16_t)best.chosen(j);
      if (l == 0 && tl < here) {
        top[tl] = high;
        total[tl] = real ? sum : 1.f;
      }
      const uint32_t with = __ballot_sync(0xffffffffu, l == 0 && tl < here && real);
      if (lane == 0) atomicAdd(held, __popc(with));
    }
    __syncthreads();
    // a thread a pick: its probability and its bit
    for (int i = threadIdx.x; i < here * p.k; i += blockDim.x) {
      const int e = pick[i], tl = (int)((uint32_t)i * per_pick >> 18);
      float x = 0.f;
      if (e >= 0) {
        x = exp_of(logit(p.logits, t0 + tl, e) - top[tl]) / total[tl];
        atomicOr(&bits[e * words + tl / 32], 1u << (tl % 32));
      }
      p.experts[t0 * p.k + i] = e;
      p.weights[t0 * p.k + i] = x;
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
      const int e = pick[i], tl = (int)((uint32_t)i * per_pick >> 18);
      int rank = -1;
      if (e >= 0) {
        rank = alone ? first[e] : count[e];
        for (int w = 0; w < tl / 32; ++w) rank += __popc(bits[e * words + w]);
        rank += __popc(bits[e * words + tl / 32] & ((1u << (tl % 32)) - 1));
      }
      p.slots[t0 * p.k + i] = rank;
    }
    if (!alone) {
      __syncthreads();
      for (int e = threadIdx.x; e < p.e; e += blockDim.x) {
        int n = count[e];
        for (int w = 0; w < words; ++w) n += __popc(bits[e * words + w]);
        count[e] = n;
      }
      __syncthreads();
    }
  }
  __syncthreads();
  if (p.blocks > 1) {
    for (int e = threadIdx.x; e < p.e; e += blockDim.x) {
      float s = 0.f;
      for (int w = 0; w < warps; ++w) s += sums[w * p.e + e];
      p.psum[(int64_t)e * p.blocks + blockIdx.x] = s;
      p.hist[(int64_t)e * p.blocks + blockIdx.x] = count[e];
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

// A warp an expert: the picks of the blocks before each, of all, and the sum of p.
__global__ void __launch_bounds__(256) route_scan(const RouteParams p) {
  start_after_earlier_kernels();
  const int e = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (e >= p.e) return;
  constexpr int MOST = 16;                    // of a lane: kMostBlocks / 32
  const int each = (p.blocks + 31) / 32;
  int *hist = p.hist + (int64_t)e * p.blocks;
  int n[MOST], own = 0;
  double mass = 0;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    const int b = lane * each + i;
    n[i] = i < each && b < p.blocks ? hist[b] : 0;
    if (i < each && b < p.blocks) mass += p.psum[(int64_t)e * p.blocks + b];
    own += n[i];
  }
  int upto = own;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
#pragma unroll
  for (int o = 16; o > 0; o /= 2) mass += __shfl_xor_sync(0xffffffffu, mass, o);
  int before = upto - own;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    const int b = lane * each + i;
    if (i < each && b < p.blocks) hist[b] = before;
    before += n[i];
  }
  if (lane == 31) p.all[e] = upto;
  if (lane == 0) p.mass[e] = mass;
}

// The rows of each block's picks: the expert's first row and the picks of the blocks before.
// The last block (of blocks + 1) writes offsets, counts and loss.
__global__ void __launch_bounds__(256) route_place(const RouteParams p) {
  extern __shared__ unsigned char smem[];
  int *from = reinterpret_cast<int *>(smem);                        // [e + 1]
  start_after_earlier_kernels();
  const bool last = blockIdx.x == p.blocks;
  // this block's picks, up to 4 a thread, are on their way meanwhile
  const int64_t span = (int64_t)p.chunk * p.per * p.k, i0 = blockIdx.x * span, end = min(i0 + span, p.rows * p.k);
  int expert[4], slot[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t i = i0 + threadIdx.x + j * 256;
    const bool there = !last && i < end;
    expert[j] = there ? p.experts[i] : -1;
    slot[j] = there ? p.slots[i] : 0;
  }
  int *before = from + p.e + 1;                                     // [e]
  for (int e = threadIdx.x; e < p.e; e += 256) {
    from[e] = p.all[e];
    before[e] = last ? 0 : p.hist[(int64_t)e * p.blocks + blockIdx.x];
  }
  __syncthreads();
  scan(from, p.e);
  if (!last) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (expert[j] >= 0) p.slots[i0 + threadIdx.x + j * 256] = slot[j] + from[expert[j]] + before[expert[j]];
    for (int64_t i = i0 + threadIdx.x + 4 * 256; i < end; i += 256) {
      const int e = p.experts[i];
      if (e >= 0) p.slots[i] += from[e] + before[e];
    }
    return;
  }
  double s = 0;
  int tokens = 0;
  for (int e = threadIdx.x; e <= p.e; e += 256) {
    p.offsets[e] = from[e];
    if (e == p.e) break;
    const int n = from[e + 1] - from[e];
    p.counts[e] = n;
    s += p.mass[e] * n;
  }
  for (int b = threadIdx.x; b < p.blocks; b += 256) tokens += p.held[b];
  __shared__ double warp_s[8];
  __shared__ int warp_n[8];
#pragma unroll
  for (int o = 16; o > 0; o /= 2) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
  }
  if (threadIdx.x % 32 == 0) {
    warp_s[threadIdx.x / 32] = s;
    warp_n[threadIdx.x / 32] = tokens;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) {
      s += warp_s[w];
      tokens += warp_n[w];
    }
    *p.tokens = tokens;
    *p.loss = tokens ? (float)(p.e * s / ((double)from[p.e] * tokens)) : 0.f;
  }
}

// Lanes of a token and values of a lane for e experts, then f.run<LPT, VPL>().  More lanes
// than e needs leave some of each lane's values unused.
template <typename F> int with_layout(int e, const F &f) {
  if (e <= 16) return f.template run<1, 16>();
  if (e <= 32) return f.template run<2, 16>();
  if (e <= 64) return f.template run<4, 16>();
  if (e <= 128) return f.template run<8, 16>();
  if (e <= 256) return f.template run<16, 16>();
  if (e <= 512) return f.template run<32, 16>();
  return f.template run<32, 32>();
}
int lanes_of(int e) {
  int lanes = 1;
  while (lanes < 32 && lanes * 16 < e) lanes *= 2;
  return lanes;
}
// Twice the lanes (8 values each) where there are few tokens: a lane's list is what takes the
// time then (8 tokens of 64 experts).
int spread_experts(int64_t rows, int e) {
  const int lanes = lanes_of(e);
  return lanes < 16 && e > 4 && rows * lanes <= 4096 ? lanes * 32 : e;
}
Logits logits_of(const void *p, int64_t rows, int64_t row, int64_t col, int e, int dtype) {
  const int es = dtype_size(dtype);
  return {p, rows, row, col, e, dtype, e % 4 == 0 && col == 1 && (uintptr_t)p % (4 * es) == 0 && (rows <= 1 || row % 4 == 0)};
}

constexpr int kMostBlocks = 512;
struct RoutePlan { int chunk, per, blocks; };
// One block where that takes 2 turns of its threads or fewer.  Else rounds of 256 tokens, or
// fewer (down to 32) while that leaves room on the GPU.
RoutePlan route_plan(int64_t rows, int e) {
  RoutePlan r{kMaxChunk, 1, 1};
  if (rows <= kMaxChunk && rows * lanes_of(spread_experts(rows, e)) <= 2 * kPickThreads) {
    r.chunk = (int)(std::max<int64_t>(rows, 1) + 31) / 32 * 32;
    return r;
  }
  while (r.chunk > 32 && (rows + r.chunk - 1) / r.chunk <= kMostBlocks / 2) r.chunk /= 2;
  const int64_t rounds = (rows + r.chunk - 1) / r.chunk;
  r.per = (int)((rounds + kMostBlocks - 1) / kMostBlocks);
  r.blocks = (int)((rounds + r.per - 1) / r.per);
  return r;
}

struct PickLaunch {
  const RouteParams &p;
  cudaStream_t st;
  template <int LPT, int VPL, int K> int launch_it() const {
    const int64_t busy = std::min((int64_t)p.chunk, p.rows) * LPT;
    const int threads = (int)std::max<int64_t>(128, std::min<int64_t>(kPickThreads, (busy + 31) / 32 * 32));
    const int smem = route_smem(p.e, p.k, p.chunk);
    const char *what = "route_pick launch";
    return p.logits.dtype == OZ_F32 ? launch(route_pick<LPT, VPL, K, false>, dim3(p.blocks), threads, smem, st, what, p)
                                    : launch(route_pick<LPT, VPL, K, true>, dim3(p.blocks), threads, smem, st, what, p);
  }
  template <int LPT, int VPL> int run() const {
    if (p.k <= 2) return launch_it<LPT, VPL, 2>();
    if (p.k <= 4) return launch_it<LPT, VPL, 4>();
    if (p.k <= 8) return launch_it<LPT, VPL, 8>();
    if (p.k <= 16) return launch_it<LPT, VPL, 16>();
    return launch_it<LPT, VPL, 32>();
  }
};

struct RouteBackward {
  Logits logits;
  const float *dweights, *dloss, *weights;
  const int *experts, *counts, *tokens;
  void *dlogits;
  int64_t rows;
  int e, k, normalize;
};

// dlogits, LPT lanes a token: the softmax again from the logits; a token's row then goes
// through shared memory, where one lane for each pick adds its part.  16384 tokens, 256 experts, 8
// picks, fp32 (35 MB, 5.4 us at the memory's rate): 15 us, bound by the latency of its sums over lanes
// (picks added by the lanes that hold them: 23 us).
template <int LPT, int VPL> __global__ void __launch_bounds__(256) route_backward(const RouteBackward p) {
  extern __shared__ unsigned char smem[];
  constexpr int GROUPS = 32 / LPT, WIDE = LPT * VPL;
  float *slope = reinterpret_cast<float *>(smem);                   // [WIDE]: the loss's part of g
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, l = lane % LPT;
  float *line = slope + WIDE + (warp * GROUPS + lane / LPT) * WIDE; // this token's row
  start_after_earlier_kernels();
  // sum of the counts, by every warp for itself
  int sum_n = 0;
  for (int e = lane; e < p.e; e += 32) sum_n += p.counts[e];
#pragma unroll
  for (int o = 16; o > 0; o /= 2) sum_n += __shfl_xor_sync(0xffffffffu, sum_n, o);
  const int tokens = *p.tokens;
  const double scale = p.dloss && tokens > 0 && sum_n > 0 ? (double)*p.dloss * p.e / ((double)tokens * sum_n) : 0.0;
  for (int e = threadIdx.x; e < WIDE; e += blockDim.x) slope[e] = e < p.e ? (float)(scale * p.counts[e]) : 0.f;
  __syncthreads();
  const int64_t step = (int64_t)gridDim.x * (blockDim.x / 32) * GROUPS;
  for (int64_t w0 = ((int64_t)blockIdx.x * (blockDim.x / 32) + warp) * GROUPS; w0 < p.rows; w0 += step) {
    const int64_t t = w0 + lane / LPT;
    const bool there = t < p.rows;
    float v[VPL];
    load_row<LPT, VPL>(p.logits, t, there, l, v);
    // the picks' part by lanes l, l + LPT, ...: w dw over the row first
    float dot = 0.f;
    if (p.dweights && there)
      for (int j = l; j < p.k; j += LPT)
        if (p.experts[t * p.k + j] >= 0) dot = fmaf(p.weights[t * p.k + j], p.dweights[t * p.k + j], dot);
    dot = lanes_sum<LPT>(dot);
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
      v[i] = real || odd ? exp_of(v[i] - top) : 0.f;
      sum += v[i];
    }
    sum = lanes_sum<LPT>(sum);
    const float inverse = sum != 0.f ? 1.f / sum : 0.f;
    float inner = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; i += 4) {
      const float4 g = *reinterpret_cast<const float4 *>(slope + expert_of<LPT>(i, l));
      v[i] *= inverse, v[i + 1] *= inverse, v[i + 2] *= inverse, v[i + 3] *= inverse;
      inner = fmaf(v[i], g.x, fmaf(v[i + 1], g.y, fmaf(v[i + 2], g.z, fmaf(v[i + 3], g.w, inner))));
    }
    inner = lanes_sum<LPT>(inner);
    if (!p.normalize) inner += dot;
#pragma unroll
    for (int i = 0; i < VPL; i += 4) {
      const float4 g = *reinterpret_cast<const float4 *>(slope + expert_of<LPT>(i, l));
      *reinterpret_cast<float4 *>(line + expert_of<LPT>(i, l)) =
          make_float4(v[i] * (g.x - inner), v[i + 1] * (g.y - inner), v[i + 2] * (g.z - inner), v[i + 3] * (g.w - inner));
    }
    __syncwarp();
    if (p.dweights && there)
      for (int j = l; j < p.k; j += LPT) {
        const int e = p.experts[t * p.k + j];
        if (e < 0 || e >= p.e) continue;
        const float w = p.weights[t * p.k + j], d = p.dweights[t * p.k + j];
        line[e] += p.normalize ? w * (d - dot) : w * d;
      }
    __syncwarp();
    if (there) {
      auto store = [&](auto z) {
        using T = decltype(z);
        T *to = static_cast<T *>(p.dlogits) + t * p.e;
#pragma unroll
        for (int i = 0; i < VPL; i += 4) {
          const int e = expert_of<LPT>(i, l);
          if (e >= p.e) continue;
          const float4 u = *reinterpret_cast<const float4 *>(line + e);
          if (p.e % 4 == 0) {                                       // rows of whole groups, aligned
            T w[4] = {from_f32<T>(u.x), from_f32<T>(u.y), from_f32<T>(u.z), from_f32<T>(u.w)};
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(to + e) = u;
            else *reinterpret_cast<uint2 *>(to + e) = *reinterpret_cast<const uint2 *>(w);
          } else {
            const float f[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (e + x < p.e) to[e + x] = from_f32<T>(f[x]);
          }
        }
      };
      if (p.logits.dtype == OZ_F32) store(float{});
      else if (p.logits.dtype == OZ_F16) store(__half{});
      else store(__nv_bfloat16{});
    }
    __syncwarp();
  }
}

struct BackwardLaunch {
  const RouteBackward &p;
  cudaStream_t st;
  template <int LPT, int VPL> int run() const {
    const int64_t blocks = (p.rows * LPT + 255) / 256;
    constexpr int smem = (1 + 8 * (32 / LPT)) * LPT * VPL * 4;
    return launch(route_backward<LPT, VPL>, dim3((unsigned)std::min(blocks, (int64_t)sm_count() * 4)), 256, smem, st,
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
  const int s = *(p.slots + pick);
  return s >= 0 && s < p.row_count ? s : -1;
}

// Zeros in the rows after the last pick's, by the blocks from `first` on.
template <typename T, int V> __device__ __forceinline__ void clear_rest(const RowsParams &p, int first) {
  const int64_t n = p.d / V, end = p.row_count * n;
  const int64_t from = min(max((int64_t)*(p.offsets + p.experts), (int64_t)0), p.row_count) * n;
  float zero[V] = {};
  for (int64_t i = from + (int64_t)(blockIdx.x - first) * blockDim.x + threadIdx.x; i < end;
       i += (int64_t)(gridDim.x - first) * blockDim.x)
    Run<T, V>::store(static_cast<T *>(p.rows_out) + i * V, zero);
}

// How the threads of a block lie over tokens and columns: `tokens` tokens side by side,
// `threads` threads each, which take the columns in steps of threads * V.
struct Spread { int tokens, threads; };
// Runs of a thread at a time: 4 where they are single elements.
__host__ __device__ constexpr int at_once(int v) { return v == 1 ? 4 : 1; }

// The slots of a token's picks, -1 where there is no row, loaded ahead of the rows they name.
template <int K> struct Picks {
  int slot[K];
  __device__ __forceinline__ void load(const RowsParams &p, int64_t t, int j0) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      slot[j] = -1;
      if (t < p.tokens && j0 + j < p.k) {
        const int s = *(p.slots + t * p.k + j0 + j);
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
  constexpr int U = at_once(V);
  const int step = at.threads * V;
  if (group >= at.tokens) return;
  for (int64_t t = (int64_t)blockIdx.x * at.tokens + group; t < p.tokens; t += (int64_t)blocks * at.tokens) {
    for (int c = in * V; c < p.d; c += U * step) {
      typename Raw<T, V>::Type v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * step < p.d) v[u] = Raw<T, V>::load(static_cast<const T *>(p.x) + t * p.x_row + c + u * step);
      T *to = static_cast<T *>(p.rows_out) + c;
#pragma unroll 4
      for (int j = 0; j < p.k; ++j) {
        const int64_t s = slot_of(p, t * p.k + j);
        if (s < 0) continue;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (c + u * step < p.d) Raw<T, V>::store(to + s * p.d + u * step, v[u]);
      }
    }
  }
}

constexpr int combine_blocks(int k) { return k >= 8 ? 3 : k >= 4 ? 4 : 5; }       // of an SM
// y[t] = sum_j w rows[slot], in the order of j, K loads on their way at a time; the next
// token's slots are loaded before this one's rows arrive.  32768 x 2048, 6 picks, bf16: 154 us
// (941 MB, 146 at the memory's rate); with loads converted as they came in 284, with registers for
// 8 loads 176.
template <typename T, int V, int K> __global__ void __launch_bounds__(256, combine_blocks(K)) combine_kernel(
    const RowsParams p, const Spread at) {
  start_after_earlier_kernels();
  const int group = (int)threadIdx.x / at.threads, in = (int)threadIdx.x - group * at.threads;
  if (group >= at.tokens) return;
  constexpr int U = at_once(V);
  const int width = at.threads * V;
  const int64_t step = (int64_t)gridDim.x * at.tokens;
  int64_t t = (int64_t)blockIdx.x * at.tokens + group;
  Picks<K> picks, next;
  picks.load(p, t, 0);
  for (; t < p.tokens; t += step) {
    next.load(p, t + step, 0);
#pragma unroll 1
    for (int c = in * V; c < p.d; c += U * width) {
      const T *from = static_cast<const T *>(p.rows) + c;
      float y[U][V] = {};
#pragma unroll 1
      for (int j0 = 0; j0 < p.k; j0 += K) {
        if (p.k > K) picks.load(p, t, j0);
        typename Raw<T, V>::Type v[K][U];
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (picks.slot[j] >= 0)
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (U == 1 || c + u * width < p.d)
                v[j][u] = Raw<T, V>::load(from + (int64_t)picks.slot[j] * p.rows_row + u * width);
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (picks.slot[j] >= 0) {
            const float w = p.weights ? *(p.weights + t * p.k + j0 + j) : 1.f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
              float e[V];
              Raw<T, V>::values(v[j][u], e);
#pragma unroll
              for (int i = 0; i < V; ++i) y[u][i] = fmaf(w, e[i], y[u][i]);
            }
          }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (U == 1 || c + u * width < p.d)
          Run<T, V>::store(static_cast<T *>(p.x_out) + t * p.d + c + u * width, y[u]);
    }
    picks = next;
  }
}

// Rows of 16-bit elements off the 16-byte boundaries: a warp moves 512 elements of a row at a
// time by aligned words, whatever the rows' parities.  Words holds 8 words a lane of a
// source from its element c0 on (they start in the middle of one where the source's
// address does: the halves that belong to neither stay unused, but share their word with
// an element, so they can be read).  pair(i) with parity h is elements h + 2 m, h + 2 m + 1, m
// = 32 i + lane, counted from c0.  dispatch, 5003 x 1001, 2 picks: 8.6 us, by elements 18.5.
constexpr int kWordSpan = 512;
struct Words {
  uint32_t direct[8], shifted[8];
  int off;
  __device__ __forceinline__ void load(const unsigned short *from, int count) {
    const int lane = threadIdx.x % 32;
    off = (int)((uintptr_t)from >> 1 & 1);
    const uint32_t *words = reinterpret_cast<const uint32_t *>(from - off);
    uint32_t w[9];
#pragma unroll
    for (int i = 0; i < 9; ++i) {
      const int j = i * 32 + lane;
      w[i] = 2 * j - off < count && (i < 8 || lane == 0) ? *(words + j) : 0;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t down = __shfl_down_sync(0xffffffffu, w[i], 1), over = __shfl_sync(0xffffffffu, w[i + 1], 0);
      const uint32_t next = lane == 31 ? over : down;
      direct[i] = off ? next : w[i];
      shifted[i] = __funnelshift_r(w[i], next, 16);
    }
  }
  __device__ __forceinline__ uint32_t pair(int i, int h) const { return off == h ? direct[i] : shifted[i]; }
};

__global__ void __launch_bounds__(256, 4) dispatch_words_kernel(const RowsParams p, int blocks) {
  using E = unsigned short;
  start_after_earlier_kernels();
  if ((int)blockIdx.x >= blocks) return clear_rest<__half, 1>(p, blocks);
  const int lane = threadIdx.x % 32, parts = (p.d + kWordSpan - 1) / kWordSpan;
  const int64_t all = p.tokens * parts;
  for (int64_t v = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; v < all; v += (int64_t)blocks * 8) {
    const int64_t t = v / parts;
    const int c0 = (int)(v - t * parts) * kWordSpan, count = min(p.d - c0, kWordSpan);
    const E *from = static_cast<const E *>(p.x) + t * p.x_row + c0;
    Words words;
    words.load(from, count);
    for (int j = 0; j < p.k; ++j) {
      const int64_t s = slot_of(p, t * p.k + j);
      if (s < 0) continue;
      E *to = static_cast<E *>(p.rows_out) + s * p.d + c0;
      const int h = (int)((uintptr_t)to >> 1 & 1);
      uint32_t *pairs = reinterpret_cast<uint32_t *>(to + h);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (h + 2 * (i * 32 + lane) + 1 < count) pairs[i * 32 + lane] = words.pair(i, h);
      if (lane == 0 && h) to[0] = from[0];
      if (lane == 1 && (count - h) % 2) to[count - 1] = from[count - 1];
    }
  }
}

template <typename T> __global__ void __launch_bounds__(256, 3) combine_words_kernel(const RowsParams p) {
  using E = unsigned short;
  start_after_earlier_kernels();
  const int lane = threadIdx.x % 32, parts = (p.d + kWordSpan - 1) / kWordSpan;
  const int64_t all = p.tokens * parts;
  auto low = [](uint32_t u) { const E e = (E)u; return to_f32(*reinterpret_cast<const T *>(&e)); };
  for (int64_t v = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; v < all; v += (int64_t)gridDim.x * 8) {
    const int64_t t = v / parts;
    const int c0 = (int)(v - t * parts) * kWordSpan, count = min(p.d - c0, kWordSpan);
    T *to = static_cast<T *>(p.x_out) + t * p.d + c0;
    const int h = (int)((uintptr_t)to >> 1 & 1);
    float y[8][2] = {}, edge = 0.f;               // edge: lane 0's first element, lane 1's last
    const int at = lane == 0 ? 0 : count - 1;
    const bool single = lane == 0 ? h != 0 : lane == 1 && (count - h) % 2;
#pragma unroll 2
    for (int j = 0; j < p.k; ++j) {
      const int64_t s = slot_of(p, t * p.k + j);
      if (s < 0) continue;
      const float w = p.weights ? *(p.weights + t * p.k + j) : 1.f;
      const E *from = static_cast<const E *>(p.rows) + s * p.rows_row + c0;
      Words words;
      words.load(from, count);
      if (single) edge = fmaf(w, low(*(from + at)), edge);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t u = words.pair(i, h);
        y[i][0] = fmaf(w, low(u), y[i][0]);
        y[i][1] = fmaf(w, low(u >> 16), y[i][1]);
      }
    }
    uint32_t *pairs = reinterpret_cast<uint32_t *>(to + h);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      T e[2] = {from_f32<T>(y[i][0]), from_f32<T>(y[i][1])};
      if (h + 2 * (i * 32 + lane) + 1 < count) pairs[i * 32 + lane] = *reinterpret_cast<const uint32_t *>(e);
    }
    if (single) to[at] = from_f32<T>(edge);
  }
}

// drows[slot] = w dy[t], dw[t, j] = dy[t] . rows[slot]: `at.threads` threads (whole warps) a
// token, K picks at a time.  8192 x 2816, 4 picks, bf16: 74 us (416 MB, 64 at the memory's rate).
// Single elements (rows off the 16-byte boundaries) go 4 at a time: 20000 x 1001, 4 picks, bf16 137
// us, one at a time 206.
template <typename T, int V, int K>
__global__ void __launch_bounds__(256, 3) combine_backward_kernel(const RowsParams p, const Spread at, int blocks) {
  __shared__ float sums[8][K];
  start_after_earlier_kernels();
  if ((int)blockIdx.x >= blocks) return clear_rest<T, V>(p, blocks);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, parts = at.threads / 32;
  const int group = warp / parts, in = (int)threadIdx.x - group * at.threads;
  constexpr int U = at_once(V);
  const int width = at.threads * V;
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
        weight[j] = picks.slot[j] >= 0 ? *(p.weights + t * p.k + j0 + j) : 0.f;
      }
      if (t < p.tokens) {
        for (int c = in * V; c < p.d; c += U * width) {
          typename Raw<T, V>::Type v[K][U], raw[U];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (U == 1 || c + u * width < p.d)
              raw[u] = Raw<T, V>::load(static_cast<const T *>(p.x) + t * p.x_row + c + u * width);
#pragma unroll
          for (int j = 0; j < K; ++j)
            if (picks.slot[j] >= 0)
#pragma unroll
              for (int u = 0; u < U; ++u)
                if (U == 1 || c + u * width < p.d)
                  v[j][u] = Raw<T, V>::load(static_cast<const T *>(p.rows) + (int64_t)picks.slot[j] * p.rows_row + c +
                                            u * width);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (U > 1 && c + u * width >= p.d) continue;
            float dy[V];
            Raw<T, V>::values(raw[u], dy);
#pragma unroll
            for (int j = 0; j < K; ++j) {
              if (picks.slot[j] < 0) continue;
              float e[V];
              Raw<T, V>::values(v[j][u], e);
#pragma unroll
              for (int i = 0; i < V; ++i) {
                dot[j] = fmaf(dy[i], e[i], dot[j]);
                e[i] = weight[j] * dy[i];
              }
              Run<T, V>::store(static_cast<T *>(p.rows_out) + (int64_t)picks.slot[j] * p.d + c + u * width, e);
            }
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

// Blocks of 8 warps, a warp 512 elements of a row at a time.
int64_t word_blocks(int64_t tokens, int64_t d, int resident) {
  const int64_t warps = tokens * ((d + kWordSpan - 1) / kWordSpan);
  return std::min<int64_t>((warps + 7) / 8, (int64_t)sm_count() * resident);
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
  if (a.tokens > INT32_MAX / 2 / a.picks || a.d > (1 << 24) || a.picks > kMaxPicks)
    return set_error(OZ_ERR_INVALID, "size out of range");
  if (!aligned(dtype_size(a.dtype), {a.x, a.rows, a.x_out, a.rows_out}) ||
      !aligned(4, {a.slots, a.offsets, a.weights, a.dweights}))
    return not_aligned();
  return OZ_OK;
}

constexpr int kClearBlocks = 64;     // zero the rows that no pick has

}  // namespace
}  // namespace oz

extern "C" int64_t oz_route_workspace_bytes(int64_t rows, int32_t experts) {
  using namespace oz;
  if (rows < 0 || experts < 1 || experts > kMaxExperts)
    return set_error(OZ_ERR_INVALID, "bad size (rows=%lld experts=%d)", (long long)rows, experts);
  if (rows > INT32_MAX / 2) return set_error(OZ_ERR_INVALID, "size out of range");
  const RoutePlan r = route_plan(rows, experts);
  // sums of p, then what the blocks counted
  return r.blocks <= 1 ? 0 : (int64_t)experts * 8 + (int64_t)r.blocks * (experts * 8 + 4) + experts * 4;
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
  if (a.rows > INT32_MAX / 2 / a.picks) return set_error(OZ_ERR_INVALID, "size out of range");
  if (!a.offsets || !a.counts || !a.tokens || !a.loss || (a.rows > 0 && (!a.logits || !a.weights || !a.chosen || !a.slots)))
    return set_error(OZ_ERR_INVALID, "null pointer");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const RoutePlan r = route_plan(a.rows, a.experts);
  const int64_t bytes = oz_route_workspace_bytes(a.rows, a.experts);
  if (bytes && (!a.workspace || (uintptr_t)a.workspace % 16 != 0 || a.workspace_bytes < bytes))
    return set_error(OZ_ERR_INVALID, "workspace of %lld bytes (16-byte aligned) needed, got %lld at %p",
                     (long long)bytes, (long long)a.workspace_bytes, a.workspace);
  if (a.dtype != OZ_F32 && a.dtype != OZ_F16 && a.dtype != OZ_BF16)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported dtype %d (fp32, fp16 or bf16)", a.dtype);
  if (!aligned(dtype_size(a.dtype), {a.logits}) ||
      !aligned(4, {a.weights, a.loss, a.chosen, a.slots, a.offsets, a.counts, a.tokens}))
    return not_aligned();
  RouteParams p{logits_of(a.logits, a.rows, a.row, a.col, a.experts, a.dtype), a.weights, a.loss, a.chosen, a.slots,
                a.offsets, a.counts, a.tokens, nullptr, nullptr, nullptr, nullptr, nullptr, a.rows, a.experts, a.picks,
                a.normalize, r.chunk, r.per, r.blocks};
  if (bytes) {
    p.mass = static_cast<double *>(a.workspace);
    p.hist = reinterpret_cast<int *>(p.mass + a.experts);
    p.psum = reinterpret_cast<float *>(p.hist + (int64_t)r.blocks * a.experts);
    p.held = reinterpret_cast<int *>(p.psum + (int64_t)r.blocks * a.experts);
    p.all = p.held + r.blocks;
  }
  int rc = with_layout(spread_experts(a.rows, a.experts), PickLaunch{p, st});
  if (rc || r.blocks <= 1) return rc;
  rc = launch(route_scan, dim3((a.experts + 7) / 8), 256, 0, st, "route_scan launch", p);
  if (rc) return rc;
  return launch(route_place, dim3(r.blocks + 1), 256, 4 * (2 * a.experts + 1), st, "route_place launch", p);
}

extern "C" int oz_route_backward(const oz_route_backward_args *args, void *stream) {
  if (!args) return oz::set_error(OZ_ERR_INVALID, "null arguments");
  using namespace oz;
  const oz_route_backward_args &a = *args;
  if (a.rows < 0) return set_error(OZ_ERR_INVALID, "negative size");
  if (a.experts < 1 || a.experts > kMaxExperts || a.picks < 1 || a.picks > kMaxPicks || a.picks > a.experts)
    return set_error(OZ_ERR_INVALID, "bad size (experts=%d picks=%d)", a.experts, a.picks);
  if (a.rows > INT32_MAX / 2 / a.picks) return set_error(OZ_ERR_INVALID, "size out of range");
  if (a.rows == 0) return OZ_OK;
  if (!a.logits || !a.weights || !a.chosen || !a.counts || !a.tokens || !a.dlogits)
    return set_error(OZ_ERR_INVALID, "null pointer");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a.dtype != OZ_F32 && a.dtype != OZ_F16 && a.dtype != OZ_BF16)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported dtype %d (fp32, fp16 or bf16)", a.dtype);
  if (!aligned(dtype_size(a.dtype), {a.logits}) ||
      !aligned(4, {a.dweights, a.dloss, a.weights, a.chosen, a.counts, a.tokens}))
    return not_aligned();
  if ((uintptr_t)a.dlogits % 16 != 0) return set_error(OZ_ERR_INVALID, "dlogits must start on a 16-byte boundary");
  const RouteBackward p{logits_of(a.logits, a.rows, a.row, a.col, a.experts, a.dtype), a.dweights, a.dloss, a.weights,
                        a.chosen, a.counts, a.tokens, a.dlogits, a.rows, a.experts, a.picks, a.normalize};
  return with_layout(a.experts, BackwardLaunch{p, st});
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
    if (!wide && ES == 2 && a.d >= 64) {
      blocks = word_blocks(a.tokens, a.d, 4);
      return launch(dispatch_words_kernel, dim3((unsigned)(blocks + kClearBlocks)), 256, 0, st,
                    "dispatch_words_kernel launch", p, (int)blocks);
    }
    const Spread at = spread_over(wide ? a.d / (16 / ES) : (a.d + 3) / 4, a.tokens, false, 6, blocks);
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
    if constexpr (ES == 2)
      if (!wide && a.d >= 64) {
        blocks = word_blocks(a.tokens, a.d, 3);
        return launch(combine_words_kernel<T>, dim3((unsigned)blocks), 256, 0, st, "combine_words_kernel launch", p);
      }
    const Spread at = spread_over(wide ? a.d / (16 / ES) : (a.d + 3) / 4, a.tokens, false, combine_blocks(a.picks <= 6 ? a.picks : 8), blocks);
    auto with = [&](auto k) {
      constexpr int K = decltype(k)::value;
      const dim3 grid((unsigned)blocks);
      return wide ? launch(combine_kernel<T, 16 / ES, K>, grid, 256, 0, st, "combine_kernel launch", p, at)
                  : launch(combine_kernel<T, 1, K>, grid, 256, 0, st, "combine_kernel launch", p, at);
    };
    if (a.picks <= 2) return with(std::integral_constant<int, 2>{});
    if (a.picks <= 4) return with(std::integral_constant<int, 4>{});
    if (a.picks <= 6) return with(std::integral_constant<int, 6>{});
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
    const Spread at = spread_over(wide ? a.d / (16 / ES) : (a.d + 3) / 4, a.tokens, true, 3, blocks);
    const dim3 grid((unsigned)(blocks + kClearBlocks));
    const char *what = "combine_backward_kernel launch";
    return wide ? launch(combine_backward_kernel<T, 16 / ES, 4>, grid, 256, 0, st, what, p, at, (int)blocks)
                : launch(combine_backward_kernel<T, 1, 4>, grid, 256, 0, st, what, p, at, (int)blocks);
  });
}
