// oz_newton.cu -- orthogonalisation of a batch of matrices by quintic
// Newton-Schulz steps.
//
//   X_0 = G / (|G|_F + eps)
//   A = X X^T,  X <- a X + (b A + c A^2) X        `steps` times
//
// for G with at most as many rows as columns; a tall G is worked on through
// its transpose (the polynomial is odd, so it commutes with transposing).
// Everything is held in fp32; the sum of squares in fp64.

#include "oz_common.cuh"

namespace oz {
namespace {

constexpr int kTile = 64;
constexpr int kStep = 16;
constexpr int kNormBlocks = 64;

template <typename T> __device__ __forceinline__ float get(const void *p, int64_t i) {
  return InTraits<T>::to_float(static_cast<const T *>(p)[i]);
}

struct InitParams {
  const void *g;
  int64_t rows, cols;               // rows <= cols, after the transposition of a tall G
  int64_t g_sb, g_sr, g_sc;
  double *partial;                  // (batch, kNormBlocks) sums of squares
  float *x;                         // (batch, rows, cols)
  double eps;
};

template <typename T> __global__ void __launch_bounds__(256) squares_kernel(const InitParams p) {
  __shared__ double part[8];
  const int64_t total = p.rows * p.cols;
  double sum = 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += kNormBlocks * 256) {
    const double v = get<T>(p.g, blockIdx.y * p.g_sb + i / p.cols * p.g_sr + i % p.cols * p.g_sc);
    sum += v * v;
  }
  for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) part[0] += part[w];
    p.partial[(int64_t)blockIdx.y * kNormBlocks + blockIdx.x] = part[0];
  }
}

template <typename T> __global__ void __launch_bounds__(256) normalise_kernel(const InitParams p) {
  double sum = 0;
  for (int i = 0; i < kNormBlocks; ++i) sum += p.partial[(int64_t)blockIdx.y * kNormBlocks + i];
  const double scale = 1.0 / (sqrt(sum) + p.eps);
  const int64_t total = p.rows * p.cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256)
    p.x[blockIdx.y * total + i] = (float)(
        get<T>(p.g, blockIdx.y * p.g_sb + i / p.cols * p.g_sr + i % p.cols * p.g_sc) * scale);
}

// out = alpha * D + beta * (a b), a (ni, nq) and b (nq, nj) by their strides.
struct ProductParams {
  const float *a, *b, *d;
  void *out;
  float alpha, beta;
  int64_t ni, nj, nq;
  int64_t a_sb, a_i, a_q, b_sb, b_q, b_j, d_sb, o_sb, o_i, o_j;
};

template <typename O> __device__ __forceinline__ void put(void *p, int64_t i, float v) {
  if constexpr (sizeof(O) == 4) static_cast<float *>(p)[i] = v;
  else if constexpr (__is_same(O, __half)) static_cast<__half *>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

template <typename O> __global__ void __launch_bounds__(256) product_kernel(const ProductParams p) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t i0 = (int64_t)blockIdx.y * kTile, j0 = (int64_t)blockIdx.x * kTile;
  const float *a = p.a + blockIdx.z * p.a_sb, *b = p.b + blockIdx.z * p.b_sb;
  float acc[4][4] = {};
  for (int64_t q0 = 0; q0 < p.nq; q0 += kStep) {
    for (int v = threadIdx.x; v < kStep * kTile; v += 256) {
      const int q = v / kTile, i = v % kTile;
      const bool in = q0 + q < p.nq;
      sa[q][i] = in && i0 + i < p.ni ? a[(i0 + i) * p.a_i + (q0 + q) * p.a_q] : 0.f;
      sb[q][i] = in && j0 + i < p.nj ? b[(q0 + q) * p.b_q + (j0 + i) * p.b_j] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kStep; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += sa[q][ty * 4 + i] * sb[q][tx * 4 + j];
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t r = i0 + ty * 4 + i, c = j0 + tx * 4 + j;
      if (r >= p.ni || c >= p.nj) continue;
      float v = p.beta * acc[i][j];
      if (p.d) v += p.alpha * p.d[blockIdx.z * p.d_sb + r * p.nj + c];
      put<O>(p.out, blockIdx.z * p.o_sb + r * p.o_i + c * p.o_j, v);
    }
}

template <typename O> int product(const ProductParams &p, int64_t batch, cudaStream_t st) {
  const dim3 grid((unsigned)((p.nj + kTile - 1) / kTile), (unsigned)((p.ni + kTile - 1) / kTile),
                  (unsigned)batch);
  count_launch();
  product_kernel<O><<<grid, 256, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "product_kernel launch");
}

template <typename T>
int run(const void *g, int64_t batch, int64_t m, int64_t n, int64_t g_sb, int64_t g_sr,
        int64_t g_sc, int steps, const double *coefficients, double eps, void *out, void *workspace,
        cudaStream_t st) {
  const bool tall = m > n;
  const int64_t rows = tall ? n : m, cols = tall ? m : n;
  double *partial = static_cast<double *>(workspace);
  float *x0 = reinterpret_cast<float *>(partial + batch * kNormBlocks);
  float *x1 = x0 + batch * rows * cols, *s = x1 + batch * rows * cols, *q = s + batch * rows * rows;
  const InitParams ip{g, rows, cols, g_sb, tall ? g_sc : g_sr, tall ? g_sr : g_sc, partial, x0, eps};
  count_launch();
  squares_kernel<T><<<dim3(kNormBlocks, (unsigned)batch), 256, 0, st>>>(ip);
  if (int rc = check_cuda(cudaGetLastError(), "squares_kernel launch")) return rc;
  const int64_t blocks = (rows * cols + 255) / 256;
  count_launch();
  normalise_kernel<T><<<dim3((unsigned)(blocks < 4096 ? blocks : 4096), (unsigned)batch), 256, 0, st>>>(ip);
  if (int rc = check_cuda(cudaGetLastError(), "normalise_kernel launch")) return rc;
  const int64_t xs = rows * cols, ss = rows * rows;
  for (int i = 0; i < steps; ++i) {
    const float a = (float)coefficients[3 * i], b = (float)coefficients[3 * i + 1],
                c = (float)coefficients[3 * i + 2];
    if (int rc = product<float>({x0, x0, nullptr, s, 0.f, 1.f, rows, rows, cols, xs, cols, 1, xs, 1,
                                 cols, 0, ss, rows, 1}, batch, st)) return rc;
    if (int rc = product<float>({s, s, s, q, b, c, rows, rows, rows, ss, rows, 1, ss, rows, 1, ss,
                                 ss, rows, 1}, batch, st)) return rc;
    const ProductParams last{q, x0, x0, i + 1 < steps ? (void *)x1 : out, a, 1.f, rows, cols, rows,
                             ss, rows, 1, xs, cols, 1, xs, xs,
                             i + 1 < steps || !tall ? cols : 1, i + 1 < steps || !tall ? 1 : rows};
    if (int rc = i + 1 < steps ? product<float>(last, batch, st) : product<T>(last, batch, st))
      return rc;
    float *t = x0;
    x0 = x1;
    x1 = t;
  }
  return OZ_OK;
}

}  // namespace
}  // namespace oz

extern "C" int64_t oz_orthogonalize_workspace_bytes(int dtype, int64_t batch, int64_t m, int64_t n,
                                                    int32_t num_splits) {
  using namespace oz;
  if ((dtype != OZ_F32 && dtype != OZ_F16 && dtype != OZ_BF16) || batch < 0 || m < 0 || n < 0 ||
      num_splits < 1 || num_splits > 2)
    return OZ_ERR_INVALID;
  const int64_t rows = m < n ? m : n, cols = m < n ? n : m;
  return batch * (kNormBlocks * 8 + (2 * rows * cols + 2 * rows * rows) * 4);
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
  if (m > (1 << 30) || n > (1 << 30) || batch > 65535)
    return set_error(OZ_ERR_INVALID, "size out of range");
  if (steps < 1 || !coefficients) return set_error(OZ_ERR_INVALID, "at least one step is needed");
  if (!(eps >= 0)) return set_error(OZ_ERR_INVALID, "eps must not be negative");
  if (num_splits < 1 || num_splits > 2)
    return set_error(OZ_ERR_INVALID, "num_splits must be 1 or 2, got %d", num_splits);
  if (batch == 0 || m == 0 || n == 0) return OZ_OK;
  if (!g || !out) return set_error(OZ_ERR_INVALID, "null pointer");
  const int64_t need = oz_orthogonalize_workspace_bytes(dtype, batch, m, n, num_splits);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256 != 0)
    return set_error(OZ_ERR_INVALID,
                     "workspace of %lld bytes (256-byte aligned) needed, got %lld at %p",
                     (long long)need, (long long)workspace_bytes, workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == OZ_F32) return run<float>(g, batch, m, n, g_sb, g_sr, g_sc, steps, coefficients, eps, out, workspace, st);
  if (dtype == OZ_F16) return run<__half>(g, batch, m, n, g_sb, g_sr, g_sc, steps, coefficients, eps, out, workspace, st);
  return run<__nv_bfloat16>(g, batch, m, n, g_sb, g_sr, g_sc, steps, coefficients, eps, out, workspace, st);
}
