// oz_linear.cuh -- what the two forms of a fused product share: its parameters and
// the arithmetic after the sums.
#pragma once

#include "oz_operands.cuh"
#include "oz_stream.cuh"

namespace oz {
namespace linear {
using stream::from_f32;
using stream::to_f32;

// ---------------------------------------------------------------------------
// activations
// ---------------------------------------------------------------------------
// Two values at a time: sm_100 multiplies and adds fp32 pairs in one instruction.
//
// The normal distribution's function below 0 is its density's exponential times a smooth
// ratio: Phi(-z) = exp(-z^2 / 2) t Q(t), t = 1 / (1 + 0.3 z), z >= 0.  Q (degree 7) is a
// weighted least-squares fit of erfcx(z / sqrt 2) / 2, off by at most 1.5e-7 of its value up
// to z = 14 (4.8e-7 as evaluated in fp32), so the tails keep their relative accuracy; above 14
// the exponential is below fp32's smallest.  8192 x 8192 results of 4096 terms, under lasting
// load: 416 us without what follows, 430 with a bias, 432 with silu, 442 with gelu (normcdff: 516).
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Smaller and larger of two, NaN if one is.
__device__ __forceinline__ float smaller(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float larger(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 exp2_of(float2 x) { return make_float2(exp2_of(x.x), exp2_of(x.y)); }
__device__ __forceinline__ float2 reciprocal(float2 x) { return make_float2(reciprocal(x.x), reciprocal(x.y)); }
constexpr float kLog2E = 1.4426950408889634f;
// Phi(nz) for nz in [-40, 0]; e: exp(-nz^2 / 2).
__device__ __forceinline__ float2 normal_tail(float2 nz, float2 &e) {
  const float2 t = reciprocal(__ffma2_rn(both(-0.3f), nz, both(1.f)));
  float2 q = both(0.03567512333393097f);
  q = __ffma2_rn(q, t, both(-0.1572044938802719f));
  q = __ffma2_rn(q, t, both(0.20635586977005005f));
  q = __ffma2_rn(q, t, both(-0.053685761988162994f));
  q = __ffma2_rn(q, t, both(0.12856271862983704f));
  q = __ffma2_rn(q, t, both(0.09991317242383957f));
  q = __ffma2_rn(q, t, both(0.12075400352478027f));
  q = __ffma2_rn(q, t, both(0.11962929368019104f));
  e = exp2_of(__fmul2_rn(__fmul2_rn(nz, nz), both(-0.5f * kLog2E)));
  return __fmul2_rn(__fmul2_rn(t, q), e);
}
// 1 / (1 + exp(-u)); 0 below -87.33, where that is no normal number any more (silu is then 0 where it
// should be -1.1e-36 at most).
__device__ __forceinline__ float2 sigmoid(float2 u) {
  return reciprocal(__fadd2_rn(both(1.f), exp2_of(__fmul2_rn(u, both(-kLog2E)))));
}

__device__ __forceinline__ float2 relu(float2 u) { return make_float2(larger(u.x, 0.f), larger(u.y, 0.f)); }
__device__ __forceinline__ float2 gelu(float2 u) {        // u Phi(u) = max(u, 0) - |u| Phi(-|u|)
  float2 e;
  const float2 nz = make_float2(larger(-fabsf(u.x), -40.f), larger(-fabsf(u.y), -40.f));
  return __ffma2_rn(nz, normal_tail(nz, e), relu(u));
}
__device__ __forceinline__ float2 silu(float2 u) { return __fmul2_rn(u, sigmoid(u)); }
__device__ __forceinline__ float relu_slope(float u) { return u > 0.f ? 1.f : u != u ? u : 0.f; }
__device__ __forceinline__ float2 relu_slope(float2 u) { return make_float2(relu_slope(u.x), relu_slope(u.y)); }
__device__ __forceinline__ float2 gelu_slope(float2 u) {  // Phi(u) + u times the density
  float2 e;
  u = make_float2(smaller(larger(u.x, -40.f), 40.f), smaller(larger(u.y, -40.f), 40.f));
  const float2 h = normal_tail(make_float2(-fabsf(u.x), -fabsf(u.y)), e), rest = __ffma2_rn(h, both(-1.f), both(1.f));
  const float2 phi = make_float2(u.x >= 0.f ? rest.x : h.x, u.y >= 0.f ? rest.y : h.y);
  return __ffma2_rn(__fmul2_rn(u, both(0.3989422804014327f)), e, phi);
}
__device__ __forceinline__ float2 silu_slope(float2 u) {
  const float2 s = sigmoid(u);
  return __fmul2_rn(s, __ffma2_rn(u, __ffma2_rn(s, both(-1.f), both(1.f)), both(1.f)));
}
template <int N, typename F> __device__ __forceinline__ void in_pairs(float (&v)[N], F f) {
  static_assert(N % 2 == 0, "pairs");
#pragma unroll
  for (int x = 0; x < N; x += 2) {
    const float2 y = f(x, make_float2(v[x], v[x + 1]));
    v[x] = y.x;
    v[x + 1] = y.y;
  }
}
// act of each value; v times act' of each u.  One branch for all of them.
template <int N> __device__ __forceinline__ void activate(float (&v)[N], int act) {
  switch (act) {
    case OZ_ACT_RELU: return in_pairs(v, [](int, float2 u) { return relu(u); });
    case OZ_ACT_GELU: return in_pairs(v, [](int, float2 u) { return gelu(u); });
    case OZ_ACT_SILU: return in_pairs(v, [](int, float2 u) { return silu(u); });
    default: return;
  }
}
template <int N> __device__ __forceinline__ void times_slope(float (&v)[N], const float (&u)[N], int act) {
  auto at = [&](int x) { return make_float2(u[x], u[x + 1]); };
  switch (act) {
    case OZ_ACT_RELU: return in_pairs(v, [&](int x, float2 d) { return __fmul2_rn(d, relu_slope(at(x))); });
    case OZ_ACT_GELU: return in_pairs(v, [&](int x, float2 d) { return __fmul2_rn(d, gelu_slope(at(x))); });
    case OZ_ACT_SILU: return in_pairs(v, [&](int x, float2 d) { return __fmul2_rn(d, silu_slope(at(x))); });
    default: return;
  }
}

struct Params {
  void *out, *pre;
  const void *bias, *residual;
  int64_t ld, residual_ld;
  int rows, k, n;              // of the result, and the contraction
  int row_tiles, column_tiles;
  int vectors;                 // what may be moved 16 bytes at a time (below)
  int bias_f32, act;
  uint32_t idesc;
};

constexpr int kVectors = 1, kResidualVectors = 2, kBiasVectors = 4;    // rows of out and pre; of the residual; the bias

// The bias has the operands' type B or fp32.
template <typename B> __device__ __forceinline__ float bias_at(const Params &p, int64_t c) {
  if (p.bias_f32) return *(static_cast<const float *>(p.bias) + c);
  return to_f32(*(static_cast<const B *>(p.bias) + c));
}

// Two operands of a result (rows, n): one along its rows, one along its columns, each
// stored across the contraction (`mn`) or along it, with its row pitch.
struct Side {
  const void *p;
  int64_t pitch;               // elements
  bool mn;
};

// oz_linear_split.cu: results of few tiles of 128 columns by `tile_rows` (16, 64 or 128; 16
// only where the rows are not stored across the contraction), the contraction over `splits`
// CTAs of a cluster.
constexpr int kMostSplits = 16;
// Or, for 16-bit results, of tiles of 256 x 256 by pairs of CTAs, 2 or 4 pairs a cluster.
constexpr int kPairTile = 256;
struct SplitPlan { int tile_rows, splits; };
int split_product(const SplitPlan &plan, int dtype, int out_dtype, const Side &a, const Side &b, const Params &p,
                  cudaStream_t st, const char *what);

}  // namespace linear
}  // namespace oz
