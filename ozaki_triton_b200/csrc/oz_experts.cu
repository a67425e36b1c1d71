// oz_experts.cu -- ragged products of an expert layer and their gradients.
//
//   y[r]  = x[r] @ w[e]                     offsets[e] <= r < offsets[e + 1]
//   dx[r] = dy[r] @ w[e]^T                  (the same product with w transposed)
//   dw[e] = sum_r x[r]^T dy[r]              r over the group's rows
//
// The groups are runs of rows given by device offsets, so no size of a group
// is known on the host: every block finds its group itself.  Offsets are
// clamped to [0, rows] before they are used as row numbers.  Products of
// fp16 / bf16 values are exact in fp32; sums are held in fp32 and rounded once.

#include "oz_common.cuh"

namespace oz {
namespace {

constexpr int kTile = 64;       // rows and columns of a block's tile
constexpr int kStep = 16;       // contraction steps staged at a time

__device__ __forceinline__ int64_t load_offset(const void *offsets, int wide, int64_t i) {
  return wide ? __ldg(static_cast<const long long *>(offsets) + i)
              : (int64_t)__ldg(static_cast<const int *>(offsets) + i);
}

// Row range of group e, clamped so that a bad offset never leaves the tensor.
__device__ __forceinline__ void group_rows(const void *offsets, int wide, int e, int64_t rows,
                                           int64_t &begin, int64_t &end) {
  begin = min(max(load_offset(offsets, wide, e), (int64_t)0), rows);
  end = min(max(load_offset(offsets, wide, e + 1), begin), rows);
}

template <typename T> __device__ __forceinline__ void store_out(void *p, int64_t i, float v);
template <> __device__ __forceinline__ void store_out<float>(void *p, int64_t i, float v) {
  static_cast<float *>(p)[i] = v;
}
template <> __device__ __forceinline__ void store_out<__half>(void *p, int64_t i, float v) {
  static_cast<__half *>(p)[i] = __float2half_rn(v);
}
template <> __device__ __forceinline__ void store_out<__nv_bfloat16>(void *p, int64_t i, float v) {
  static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// One 64 x 64 tile of sum_q a(i, q) b(q, j): 256 threads, 4 x 4 values each.
template <typename T>
__device__ __forceinline__ void tile_product(const T *a, int64_t a_i, int64_t a_q, int64_t ni,
                                             const T *b, int64_t b_q, int64_t b_j, int64_t nj,
                                             int64_t nq, float (&acc)[4][4]) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  for (int64_t q0 = 0; q0 < nq; q0 += kStep) {
    for (int v = threadIdx.x; v < kStep * kTile; v += 256) {
      const int q = v / kTile, i = v % kTile;
      const bool in_q = q0 + q < nq;
      sa[q][i] = in_q && i < ni ? InTraits<T>::to_float(a[i * a_i + (q0 + q) * a_q]) : 0.f;
      sb[q][i] = in_q && i < nj ? InTraits<T>::to_float(b[(q0 + q) * b_q + i * b_j]) : 0.f;
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
}

struct GroupedParams {
  const void *a, *b, *offsets;
  void *c;
  int wide, groups;
  int64_t rows, k, n;
  int64_t a_sr, a_sk;          // x: row and inner strides
  int64_t b_se, b_sk, b_sn;    // w: expert, k and n strides (wgrad: dy's row and column ones)
  int64_t ldc;
};

// Block (row block, column tile): row blocks count the groups' 64-row tiles in
// order; the blocks after the last one zero the rows that no group holds.
template <typename T, typename O>
__global__ void __launch_bounds__(256) grouped_kernel(const GroupedParams p) {
  int64_t block = blockIdx.x, begin = 0, end = 0;
  int e = 0;
  for (; e < p.groups; ++e) {
    group_rows(p.offsets, p.wide, e, p.rows, begin, end);
    const int64_t tiles = (end - begin + kTile - 1) / kTile;
    if (block < tiles) break;
    block -= tiles;
  }
  const int64_t n0 = (int64_t)blockIdx.y * kTile, nj = min((int64_t)kTile, p.n - n0);
  if (e == p.groups) {
    int64_t first, last;
    group_rows(p.offsets, p.wide, 0, p.rows, first, last);
    group_rows(p.offsets, p.wide, p.groups - 1, p.rows, begin, last);
    const int64_t outside = first + p.rows - last;
    for (int64_t v = block * kTile * nj + threadIdx.x; v < min((block + 1) * kTile, outside) * nj;
         v += 256) {
      const int64_t r = v / nj, row = r < first ? r : last + r - first;
      store_out<O>(p.c, row * p.ldc + n0 + v % nj, 0.f);
    }
    return;
  }
  const int64_t row = begin + block * kTile, ni = min((int64_t)kTile, end - row);
  float acc[4][4] = {};
  tile_product<T>(static_cast<const T *>(p.a) + row * p.a_sr, p.a_sr, p.a_sk, ni,
                  static_cast<const T *>(p.b) + e * p.b_se + n0 * p.b_sn, p.b_sk, p.b_sn, nj, p.k,
                  acc);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (ty * 4 + i < ni && tx * 4 + j < nj)
        store_out<O>(p.c, (row + ty * 4 + i) * p.ldc + n0 + tx * 4 + j, acc[i][j]);
}

// Block (n tile, k tile, group): dw[e] tile over the rows of the group.
template <typename T, typename O>
__global__ void __launch_bounds__(256) grouped_wgrad_kernel(const GroupedParams p) {
  int64_t begin, end;
  const int e = blockIdx.z;
  group_rows(p.offsets, p.wide, e, p.rows, begin, end);
  const int64_t n0 = (int64_t)blockIdx.x * kTile, nj = min((int64_t)kTile, p.n - n0);
  const int64_t k0 = (int64_t)blockIdx.y * kTile, ni = min((int64_t)kTile, p.k - k0);
  float acc[4][4] = {};
  tile_product<T>(static_cast<const T *>(p.a) + begin * p.a_sr + k0 * p.a_sk, p.a_sk, p.a_sr, ni,
                  static_cast<const T *>(p.b) + begin * p.b_sk + n0 * p.b_sn, p.b_sk, p.b_sn, nj,
                  end - begin, acc);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (ty * 4 + i < ni && tx * 4 + j < nj)
        store_out<O>(p.c, ((int64_t)e * p.k + k0 + ty * 4 + i) * p.n + n0 + tx * 4 + j, acc[i][j]);
}

int check_grouped(int dtype, int out_dtype, int32_t groups, int64_t rows, int64_t k, int64_t n) {
  if (dtype != OZ_F16 && dtype != OZ_BF16)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported operand dtype %d (fp16 or bf16)", dtype);
  if (out_dtype != dtype && out_dtype != OZ_F32)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported output dtype %d", out_dtype);
  if (groups < 1) return set_error(OZ_ERR_INVALID, "at least one group is needed, got %d", groups);
  if (rows < 0 || k < 0 || n < 0) return set_error(OZ_ERR_INVALID, "negative size");
  if (rows > (1 << 30) || k > (1 << 30) || n > (1 << 30))
    return set_error(OZ_ERR_INVALID, "size out of range");
  return OZ_OK;
}

}  // namespace
}  // namespace oz

extern "C" int oz_grouped_matmul(const void *x, const void *w, const void *offsets,
                                 int offsets_64, int dtype, int out_dtype, int32_t groups,
                                 int64_t rows, int64_t k, int64_t n, int64_t x_sr, int64_t x_sk,
                                 int64_t w_se, int64_t w_sk, int64_t w_sn, void *y, int64_t ldy,
                                 void *stream) {
  using namespace oz;
  if (int rc = check_grouped(dtype, out_dtype, groups, rows, k, n)) return rc;
  if (rows == 0 || n == 0) return OZ_OK;
  if (!y || ldy < n) return set_error(OZ_ERR_INVALID, "bad output (ldy=%lld n=%lld)",
                                      (long long)ldy, (long long)n);
  if (!offsets || (k > 0 && (!x || !w))) return set_error(OZ_ERR_INVALID, "null pointer");
  GroupedParams p{x, w, offsets, y, offsets_64, groups, rows, k, n, x_sr, x_sk, w_se, w_sk, w_sn,
                  ldy};
  const int64_t blocks = (rows + kTile - 1) / kTile + groups + 1;
  const dim3 grid((unsigned)blocks, (unsigned)((n + kTile - 1) / kTile));
  if (grid.y > 65535) return set_error(OZ_ERR_INVALID, "size out of range");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  count_launch();
  if (dtype == OZ_F16 && out_dtype == OZ_F32) grouped_kernel<__half, float><<<grid, 256, 0, st>>>(p);
  else if (dtype == OZ_F16) grouped_kernel<__half, __half><<<grid, 256, 0, st>>>(p);
  else if (out_dtype == OZ_F32) grouped_kernel<__nv_bfloat16, float><<<grid, 256, 0, st>>>(p);
  else grouped_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "grouped_kernel launch");
}

extern "C" int oz_grouped_wgrad(const void *x, const void *dy, const void *offsets,
                                int offsets_64, int dtype, int out_dtype, int32_t groups,
                                int64_t rows, int64_t k, int64_t n, int64_t x_sr, int64_t x_sk,
                                int64_t dy_sr, int64_t dy_sn, void *dw, void *stream) {
  using namespace oz;
  if (int rc = check_grouped(dtype, out_dtype, groups, rows, k, n)) return rc;
  if (k == 0 || n == 0) return OZ_OK;
  if (!dw || !offsets || (rows > 0 && (!x || !dy)))
    return set_error(OZ_ERR_INVALID, "null pointer");
  if (groups > 65535) return set_error(OZ_ERR_INVALID, "too many groups");
  GroupedParams p{x, dy, offsets, dw, offsets_64, groups, rows, k, n, x_sr, x_sk, 0, dy_sr, dy_sn,
                  n};
  const dim3 grid((unsigned)((n + kTile - 1) / kTile), (unsigned)((k + kTile - 1) / kTile),
                  (unsigned)groups);
  if (grid.y > 65535) return set_error(OZ_ERR_INVALID, "size out of range");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  count_launch();
  if (dtype == OZ_F16 && out_dtype == OZ_F32)
    grouped_wgrad_kernel<__half, float><<<grid, 256, 0, st>>>(p);
  else if (dtype == OZ_F16) grouped_wgrad_kernel<__half, __half><<<grid, 256, 0, st>>>(p);
  else if (out_dtype == OZ_F32)
    grouped_wgrad_kernel<__nv_bfloat16, float><<<grid, 256, 0, st>>>(p);
  else grouped_wgrad_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "grouped_wgrad_kernel launch");
}
