// oz_w4.cu -- products of a few rows with 4-bit weights and group scales.
//
//   y[r, n] = sum_k x[r, k] (q[n, k] - z[n, k / g]) s[n, k / g]
//
// q: two values a byte along k, the even k in the low half; z is 8 where no
// zero points are given.  With offsets the rows come in groups, each with the
// weights of its own expert.  q - z is an exact small integer; the products
// and sums are held in fp32, the scale is applied to a group's sum.

#include "oz_common.cuh"

namespace oz {
namespace {

struct W4Params {
  const void *x, *scales, *offsets;
  const uint8_t *packed, *zeros;
  void *y;
  int wide, experts, group, scale_dtype;
  int64_t rows, k, n;
  int64_t x_sr, ldy;
  int64_t p_se, p_sn;          // packed: expert and row strides, bytes
  int64_t s_se, s_sn;          // scales (and zeros): expert and row strides, elements
};

__device__ __forceinline__ float load_scale(const void *s, int dtype, int64_t i) {
  if (dtype == OZ_F32) return __ldg(static_cast<const float *>(s) + i);
  if (dtype == OZ_F16) return __half2float(__ldg(static_cast<const __half *>(s) + i));
  return __bfloat162float(__ldg(static_cast<const __nv_bfloat16 *>(s) + i));
}

__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }

// A warp per weight row and input row.
template <typename T, typename O> __global__ void __launch_bounds__(256) w4_kernel(const W4Params p) {
  const int lane = threadIdx.x % 32;
  const int64_t n = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (n >= p.n) return;
  for (int64_t r = blockIdx.y; r < p.rows; r += gridDim.y) {
    int64_t e = 0;
    if (p.offsets) {
      // the expert whose group holds the row; none: the row is zero
      for (; e < p.experts; ++e) {
        const int64_t end = p.wide ? static_cast<const long long *>(p.offsets)[e + 1]
                                   : static_cast<const int *>(p.offsets)[e + 1];
        const int64_t begin = p.wide ? static_cast<const long long *>(p.offsets)[e]
                                     : static_cast<const int *>(p.offsets)[e];
        if (r >= begin && r < end) break;
      }
    }
    float sum = 0.f;
    if (e < p.experts) {
      const T *x = static_cast<const T *>(p.x) + r * p.x_sr;
      const uint8_t *q = p.packed + e * p.p_se + n * p.p_sn;
      const int64_t s = e * p.s_se + n * p.s_sn;
      for (int64_t k = lane * 2; k < p.k; k += 64) {
        const int64_t g = k / p.group;
        const float zero = p.zeros ? (float)p.zeros[s + g] : 8.f;
        const uint8_t v = q[k / 2];
        const float part = InTraits<T>::to_float(x[k]) * ((float)(v & 15) - zero) +
                           InTraits<T>::to_float(x[k + 1]) * ((float)(v >> 4) - zero);
        sum += part * load_scale(p.scales, p.scale_dtype, s + g);
      }
    }
    for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) put(static_cast<O *>(p.y) + r * p.ldy + n, sum);
  }
}

}  // namespace
}  // namespace oz

extern "C" int oz_matmul_w4(const void *x, const void *packed, const void *scales,
                            const void *zeros, const void *offsets, int offsets_64, int dtype,
                            int scale_dtype, int out_dtype, int32_t experts, int64_t rows,
                            int64_t k, int64_t n, int32_t group, int64_t x_sr, int64_t p_se,
                            int64_t p_sn, int64_t s_se, int64_t s_sn, void *y, int64_t ldy,
                            void *stream) {
  using namespace oz;
  if (dtype != OZ_F16 && dtype != OZ_BF16)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported operand dtype %d (fp16 or bf16)", dtype);
  if (scale_dtype != OZ_F16 && scale_dtype != OZ_BF16 && scale_dtype != OZ_F32)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported scale dtype %d", scale_dtype);
  if (out_dtype != dtype && out_dtype != OZ_F32)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported output dtype %d", out_dtype);
  if (experts < 1) return set_error(OZ_ERR_INVALID, "at least one expert is needed, got %d", experts);
  if (rows < 0 || k < 0 || n < 0) return set_error(OZ_ERR_INVALID, "negative size");
  if (rows > (1 << 30) || k > (1 << 30) || n > (1 << 30))
    return set_error(OZ_ERR_INVALID, "size out of range");
  if (group < 32 || group % 32 != 0 || k % group != 0)
    return set_error(OZ_ERR_INVALID, "the group size must be a multiple of 32 that divides k (group=%d k=%lld)",
                     group, (long long)k);
  if (rows == 0 || n == 0) return OZ_OK;
  if (!y || ldy < n)
    return set_error(OZ_ERR_INVALID, "bad output (ldy=%lld n=%lld)", (long long)ldy, (long long)n);
  if (k > 0 && (!x || !packed || !scales)) return set_error(OZ_ERR_INVALID, "null pointer");
  if (!offsets && experts != 1) return set_error(OZ_ERR_INVALID, "several experts need offsets");
  W4Params p{x, scales, offsets, static_cast<const uint8_t *>(packed),
             static_cast<const uint8_t *>(zeros), y, offsets_64, experts, group, scale_dtype,
             rows, k, n, x_sr, ldy, p_se, p_sn, s_se, s_sn};
  const dim3 grid((unsigned)((n + 7) / 8), (unsigned)(rows < 65535 ? rows : 65535));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  count_launch();
  if (dtype == OZ_F16 && out_dtype == OZ_F32) w4_kernel<__half, float><<<grid, 256, 0, st>>>(p);
  else if (dtype == OZ_F16) w4_kernel<__half, __half><<<grid, 256, 0, st>>>(p);
  else if (out_dtype == OZ_F32) w4_kernel<__nv_bfloat16, float><<<grid, 256, 0, st>>>(p);
  else w4_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "w4_kernel launch");
}
