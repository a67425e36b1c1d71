// oz_linear.cuh -- what the two forms of a fused product share: its parameters and
// the arithmetic after the sums.
#pragma once

#include <cmath>

#include "oz_operands.cuh"
#include "oz_stream.cuh"

namespace oz {
namespace linear {
using stream::from_f32;
using stream::to_f32;

__device__ __forceinline__ float activated(float u, int act) {
  switch (act) {
    case OZ_ACT_RELU: return u > 0.f ? u : u != u ? u : 0.f;
    case OZ_ACT_GELU: return u * normcdff(u);
    case OZ_ACT_SILU: return u / (1.f + expf(-u));
    default: return u;
  }
}
__device__ __forceinline__ float slope(float u, int act) {
  switch (act) {
    case OZ_ACT_RELU: return u > 0.f ? 1.f : u != u ? u : 0.f;
    case OZ_ACT_GELU: return normcdff(u) + u * (0.3989422804014327f * expf(-0.5f * u * u));
    case OZ_ACT_SILU: {
      const float s = 1.f / (1.f + expf(-u));
      return s * (1.f + u * (1.f - s));
    }
    default: return 1.f;
  }
}

struct Params {
  void *out, *pre;
  const void *bias, *residual;
  int64_t ld, residual_ld;
  int rows, k, n;              // of the result, and the contraction
  int row_tiles, column_tiles;
  int vectors;                 // rows of out and pre may be written 16 bytes at a time
  int bias_f32, act;
  uint32_t idesc;
};

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

// oz_linear_split.cu: results of few tiles, the contraction over the CTAs of a cluster.
// `plan` says how (rows of a tile, CTAs of a cluster), or 0 rows where the tile engine is
// the faster way.
struct SplitPlan { int tile_rows, splits; };
SplitPlan split_plan(int64_t rows, int64_t k, int64_t n, bool rows_mn);
int split_product(const SplitPlan &plan, int dtype, int out_dtype, const Side &a, const Side &b, const Params &p,
                  cudaStream_t st, const char *what);

}  // namespace linear
}  // namespace oz
