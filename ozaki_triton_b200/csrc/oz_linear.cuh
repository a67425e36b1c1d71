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
// The normal distribution's function below 0 is its density's exponential times a smooth
// ratio: Phi(-z) = exp(-z^2 / 2) t Q(t), t = 1 / (1 + 0.3 z), z >= 0.  Q (degree 7) is a
// weighted least-squares fit of erfcx(z / sqrt 2) / 2, off by at most 1.5e-7 of its value up
// to z = 14 (4.8e-7 as evaluated in fp32), so the tails keep their relative accuracy; above 14
// the exponential is below fp32's smallest.  16 instructions; with normcdff 8192 x 8192 results of 4096
// terms took 516 us where they take 365 without an activation.
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
constexpr float kLog2E = 1.4426950408889634f;
// Phi(-z) for z in [0, 40]; e: exp(-z^2 / 2).
__device__ __forceinline__ float normal_tail(float z, float &e) {
  const float t = reciprocal(fmaf(0.3f, z, 1.f));
  float q = 0.03567512333393097f;
  q = fmaf(q, t, -0.1572044938802719f);
  q = fmaf(q, t, 0.20635586977005005f);
  q = fmaf(q, t, -0.053685761988162994f);
  q = fmaf(q, t, 0.12856271862983704f);
  q = fmaf(q, t, 0.09991317242383957f);
  q = fmaf(q, t, 0.12075400352478027f);
  q = fmaf(q, t, 0.11962929368019104f);
  e = exp2_of(z * z * (-0.5f * kLog2E));
  return t * q * e;
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
// 1 / (1 + exp(-u)); below -88 the exponential is infinite and the result 0.
__device__ __forceinline__ float sigmoid(float u) { return reciprocal(1.f + exp2_of(u * -kLog2E)); }

__device__ __forceinline__ float relu(float u) { return larger(u, 0.f); }
__device__ __forceinline__ float gelu(float u) {          // u Phi(u) = max(u, 0) - |u| Phi(-|u|)
  float e;
  const float z = smaller(fabsf(u), 40.f);
  return larger(u, 0.f) - z * normal_tail(z, e);
}
__device__ __forceinline__ float silu(float u) { return u * sigmoid(u); }
__device__ __forceinline__ float relu_slope(float u) { return u > 0.f ? 1.f : u != u ? u : 0.f; }
__device__ __forceinline__ float gelu_slope(float u) {
  float e;
  const float z = smaller(fabsf(u), 40.f), h = normal_tail(z, e);
  return fmaf(copysignf(z, u) * 0.3989422804014327f, e, u >= 0.f ? 1.f - h : h);
}
__device__ __forceinline__ float silu_slope(float u) {
  const float s = sigmoid(u);
  return s * fmaf(u, 1.f - s, 1.f);
}
// act of each value; v times act' of each u.  One branch for all of them.
template <int N> __device__ __forceinline__ void activate(float (&v)[N], int act) {
  switch (act) {
    case OZ_ACT_RELU:
#pragma unroll
      for (int x = 0; x < N; ++x) v[x] = relu(v[x]);
      break;
    case OZ_ACT_GELU:
#pragma unroll
      for (int x = 0; x < N; ++x) v[x] = gelu(v[x]);
      break;
    case OZ_ACT_SILU:
#pragma unroll
      for (int x = 0; x < N; ++x) v[x] = silu(v[x]);
      break;
    default: break;
  }
}
template <int N> __device__ __forceinline__ void times_slope(float (&v)[N], const float (&u)[N], int act) {
  switch (act) {
    case OZ_ACT_RELU:
#pragma unroll
      for (int x = 0; x < N; ++x) v[x] *= relu_slope(u[x]);
      break;
    case OZ_ACT_GELU:
#pragma unroll
      for (int x = 0; x < N; ++x) v[x] *= gelu_slope(u[x]);
      break;
    case OZ_ACT_SILU:
#pragma unroll
      for (int x = 0; x < N; ++x) v[x] *= silu_slope(u[x]);
      break;
    default: break;
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
  if (p.bias_f32) return __ldg(static_cast<const float *>(p.bias) + c);
  return to_f32(__ldg(static_cast<const B *>(p.bias) + c));
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
constexpr int kMostSplits = 8;
struct SplitPlan { int tile_rows, splits; };
int split_product(const SplitPlan &plan, int dtype, int out_dtype, const Side &a, const Side &b, const Params &p,
                  cudaStream_t st, const char *what);

}  // namespace linear
}  // namespace oz
