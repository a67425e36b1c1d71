// oz_clip.cu -- gradients of many tensors, scaled so that their common norm is at
// most max_norm:
//
//   norm = sqrt(sum of all squares),  out = g min(1, max_norm / (norm + eps))
//
// Two launches read the gradients: the first sums squares (fp32 within 16
// bytes whose squares fit it, fp64 beyond, in an order that does not depend on timing),
// the second has every block add up the first's sums and scales.  Bound by memory:
// the gradients are read twice and the results written once.  48 tensors of 4e8 bf16 gradients
// to fp32 (3.2 GB): 540 us, 5.9 TB/s; to bf16 392 us, 6.1 TB/s.

#include <algorithm>
#include <cmath>
#include <vector>

#include "oz_stream.cuh"

namespace oz {
namespace {
using namespace stream;

constexpr int kThreads = 256;
constexpr int kBlocksPerSm = 4, kScaleBlocksPerSm = 3;      // resident together
constexpr int kSmallPiece = 8192, kLargePiece = 16384;     // elements of a block's turn
constexpr int kAtOnce = 4;            // 16-byte loads of a thread: these are worked on while as many are on their way

struct Tensor {
  const void *g;
  void *out;
  int64_t n;
  int first;                          // pieces of the tensors before it
  int types;                          // type of g, of out (4 bits each), 16-byte runs (bit 8)
};
template <int N> struct Table {
  Tensor t[N];
  int tensors, pieces, piece;          // piece: its elements
};
struct Sums {
  double *partial;                    // one of each block of each summing launch
  float *norm;
  int blocks;
  float max_norm, eps;
};

template <int N> __device__ __forceinline__ int tensor_of(const Table<N> &table, int piece) {
  int low = 0, high = table.tensors - 1;      // the last tensor whose first piece is not after it
  while (low < high) {
    const int mid = (low + high + 1) / 2;
    if (table.t[mid].first <= piece) low = mid;
    else high = mid - 1;
  }
  return low;
}

// sum + the squares of 16 bytes of T: in fp32 where their sum shows that none overflowed and that
// what fp32 loses below its smallest numbers cannot matter (8 times 2^-150 of 2^-120 and more; with
// the additions 2^-21 off at most), else in fp64.  48 tensors, 4e8 bf16 gradients: 543 us
// with the test as without it; by the largest of the 8 instead of their sum 556.
template <typename T> __device__ __forceinline__ double add_squares(double sum, const uint4 &u) {
  constexpr int V = 16 / sizeof(T);
  float v[V], s = 0.f;
  unpack<T>(u, v);
#pragma unroll
  for (int x = 0; x < V; ++x) s = fmaf(v[x], v[x], s);
  if (std::is_same<T, __half>::value || (s >= 0x1p-120f && s <= 0x1p120f)) return sum + s;
  if (((u.x | u.y | u.z | u.w) & (sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu)) == 0) return sum;
#pragma unroll
  for (int x = 0; x < V; ++x) sum += (double)v[x] * v[x];
  return sum;
}
// An element of a type known at run time.
__device__ __forceinline__ float element(const void *g, int64_t i, int type) {
  if (type == OZ_F32) return static_cast<const float *>(g)[i];
  if (type == OZ_F16) return to_f32(static_cast<const __half *>(g)[i]);
  return to_f32(static_cast<const __nv_bfloat16 *>(g)[i]);
}
__device__ __forceinline__ void set_element(void *out, int64_t i, int type, float v) {
  if (type == OZ_F32) static_cast<float *>(out)[i] = v;
  else if (type == OZ_F16) static_cast<__half *>(out)[i] = from_f32<__half>(v);
  else static_cast<__nv_bfloat16 *>(out)[i] = from_f32<__nv_bfloat16>(v);
}

// Calls f(run, bits) for this thread's runs (16 bytes, or 8) of a piece.
template <typename U, typename F> __device__ __forceinline__ void each_run(const U *g, int runs, F f) {
  constexpr int kAtOnce = oz::kAtOnce * 16 / sizeof(U);
  U u[kAtOnce], next[kAtOnce];
  auto load = [&](int i, U (&to)[kAtOnce]) {
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (i + j * kThreads < runs) to[j] = g[i + j * kThreads];
  };
  load(threadIdx.x, u);
#pragma unroll 1
  for (int i = threadIdx.x; i < runs; i += kThreads * kAtOnce) {
    load(i + kThreads * kAtOnce, next);
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (i + j * kThreads < runs) f(i + j * kThreads, u[j]);
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) u[j] = next[j];
  }
}

template <int N>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) norm_kernel(const __grid_constant__ Table<N> table, double *partial) {
  start_after_earlier_kernels();
  double all = 0;
  // neighbouring blocks take neighbouring pieces: what is read at a time lies together
  int at = tensor_of(table, min((int)blockIdx.x, table.pieces - 1));
  for (int piece = blockIdx.x; piece < table.pieces; piece += gridDim.x) {
    while (at + 1 < table.tensors && table.t[at + 1].first <= piece) ++at;
    const Tensor &t = table.t[at];
    const int64_t from = (int64_t)(piece - t.first) * table.piece;
    const int n = (int)min(t.n - from, (int64_t)table.piece), type = t.types & 15, es = type == OZ_F32 ? 4 : 2;
    const char *g = static_cast<const char *>(t.g) + from * es;
    const int runs = t.types >> 8 & 1 ? n * es / 16 : 0;
    each_run(reinterpret_cast<const uint4 *>(g), runs, [&](int, const uint4 &u) {
      if (type == OZ_F32) all = add_squares<float>(all, u);
      else if (type == OZ_F16) all = add_squares<__half>(all, u);
      else all = add_squares<__nv_bfloat16>(all, u);
    });
#pragma unroll 1
    for (int i = runs * (16 / es) + threadIdx.x; i < n; i += kThreads) {
      const double v = element(g, i, type);
      all += v * v;
    }
  }
  __shared__ double warp_sum[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o /= 2) all += __shfl_xor_sync(0xffffffffu, all, o);
  if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = all;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) all += warp_sum[w];
    partial[blockIdx.x] = all;
  }
}

// A run of T, scaled, to run r of out.
template <typename T, typename O> __device__ __forceinline__ void scaled(const uint4 &u, O *out, int r, float scale) {
  constexpr int V = 16 / sizeof(T);
  float v[V];
  unpack<T>(u, v);
#pragma unroll
  for (int x = 0; x < V; ++x) v[x] *= scale;
  out += (int64_t)r * V;
  if constexpr (sizeof(O) == sizeof(T)) {
    *reinterpret_cast<uint4 *>(out) = pack<O>(v);
  } else {                                    // fp32 to 16 bits
    O w[V];
#pragma unroll
    for (int x = 0; x < V; ++x) w[x] = from_f32<O>(v[x]);
    *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<const uint2 *>(w);
  }
}
// 16 bits to fp32: 8 bytes, so that a warp's results are next to each other (from 16 bytes a lane
// wrote two halves of 32: 631 us for 400 million gradients, this 543).
template <typename T> __device__ __forceinline__ void widened(const uint2 &u, float *out, int r, float scale) {
  const T *e = reinterpret_cast<const T *>(&u);
  reinterpret_cast<float4 *>(out)[r] =
      make_float4(to_f32(e[0]) * scale, to_f32(e[1]) * scale, to_f32(e[2]) * scale, to_f32(e[3]) * scale);
}

// PAIR: the types of all gradients and results (type | to << 4), or 0 where they differ.
template <int N, int PAIR>
__global__ void __launch_bounds__(kThreads, kScaleBlocksPerSm) scale_kernel(const __grid_constant__ Table<N> table, const Sums sums) {
  __shared__ float shared_scale;
  __shared__ double warp_sum[kThreads / 32];
  start_after_earlier_kernels();
  double all = 0;
  for (int i = threadIdx.x; i < sums.blocks; i += kThreads) all += *(sums.partial + i);
#pragma unroll
  for (int o = 16; o > 0; o /= 2) all += __shfl_xor_sync(0xffffffffu, all, o);
  if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = all;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) all += warp_sum[w];
    const float norm = (float)sqrt(all);
    const float ratio = sums.max_norm / (norm + sums.eps);
    shared_scale = ratio >= 1.f ? 1.f : ratio;                 // NaN stays
    if (blockIdx.x == 0) *sums.norm = norm;
  }
  __syncthreads();
  const float scale = shared_scale;
  if ((int)blockIdx.x >= table.pieces) return;
  // the pieces read last are the first here: some of them are still in L2
  int at = tensor_of(table, table.pieces - 1 - (int)blockIdx.x);
  for (int piece = table.pieces - 1 - (int)blockIdx.x; piece >= 0; piece -= gridDim.x) {
    while (table.t[at].first > piece) --at;
    const Tensor &t = table.t[at];
    const int64_t from = (int64_t)(piece - t.first) * table.piece;
    const int types = PAIR ? PAIR : t.types, type = types & 15, to = types >> 4 & 15;
    const int n = (int)min(t.n - from, (int64_t)table.piece);
    const int es = type == OZ_F32 ? 4 : 2, os = to == OZ_F32 ? 4 : 2;
    const char *g = static_cast<const char *>(t.g) + from * es;
    char *out = static_cast<char *>(t.out) + from * os;
    const int runs = t.types >> 8 & 1 ? n * es / 16 : 0;
    if (es == 2 && os == 4) {
      each_run(reinterpret_cast<const uint2 *>(g), 2 * runs, [&](int r, const uint2 &u) {
        if (type == OZ_F16) widened<__half>(u, reinterpret_cast<float *>(out), r, scale);
        else widened<__nv_bfloat16>(u, reinterpret_cast<float *>(out), r, scale);
      });
    } else {
      each_run(reinterpret_cast<const uint4 *>(g), runs, [&](int r, const uint4 &u) {
        if (type == OZ_F32) {
          if (to == OZ_F32) scaled<float>(u, reinterpret_cast<float *>(out), r, scale);
          else if (to == OZ_F16) scaled<float>(u, reinterpret_cast<__half *>(out), r, scale);
          else scaled<float>(u, reinterpret_cast<__nv_bfloat16 *>(out), r, scale);
        } else if (type == OZ_F16) {
          if (to == OZ_F16) scaled<__half>(u, reinterpret_cast<__half *>(out), r, scale);
          else scaled<__half>(u, reinterpret_cast<__nv_bfloat16 *>(out), r, scale);
        } else {
          if (to == OZ_F16) scaled<__nv_bfloat16>(u, reinterpret_cast<__half *>(out), r, scale);
          else scaled<__nv_bfloat16>(u, reinterpret_cast<__nv_bfloat16 *>(out), r, scale);
        }
      });
    }
#pragma unroll 1
    for (int i = runs * (16 / es) + threadIdx.x; i < n; i += kThreads)
      set_element(out, i, to, element(g, i, type) * scale);
  }
}

// A launch takes the addresses of at most this many tensors as arguments.
constexpr int kFew = 64, kMany = 640;

int blocks_of(int64_t pieces, int per_sm) { return (int)std::min<int64_t>(pieces, (int64_t)sm_count() * per_sm); }

template <int N> Table<N> table_of(const oz_clip_args &a, int first, int count, int piece) {
  Table<N> table;
  table.piece = piece;
  int64_t pieces = 0;
  table.tensors = 0;
  for (int i = first; i < first + count; ++i) {
    const int64_t n = a.sizes[i];
    if (n == 0) continue;
    const int es = dtype_size(a.dtypes[i]), os = dtype_size(a.out_dtypes[i]);
    const bool runs = (uintptr_t)a.grads[i] % 16 == 0 && (uintptr_t)a.outs[i] % (es == 4 && os == 2 ? 8 : 16) == 0;
    table.t[table.tensors++] = Tensor{a.grads[i], a.outs[i], n, (int)pieces,
                                      a.dtypes[i] | a.out_dtypes[i] << 4 | (runs ? 1 << 8 : 0)};
    pieces += (n + piece - 1) / piece;
  }
  table.pieces = (int)pieces;
  return table;
}
int64_t pieces_of(const oz_clip_args &a, int piece) {
  int64_t pieces = 0;
  for (int i = 0; i < a.tensors; ++i) pieces += (a.sizes[i] + piece - 1) / piece;
  return pieces;
}

template <int N> int run(const oz_clip_args &a, Sums sums, cudaStream_t st) {
  sums.blocks = 0;
  // large pieces where every block has several of them
  const int piece = pieces_of(a, kLargePiece) >= (int64_t)sm_count() * kBlocksPerSm * 4 ? kLargePiece : kSmallPiece;
  for (int i = 0; i < a.tensors; i += N) {
    const auto table = table_of<N>(a, i, std::min(N, a.tensors - i), piece);
    if (!table.pieces) continue;
    const int blocks = blocks_of(table.pieces, kBlocksPerSm);
    if (int rc = launch(norm_kernel<N>, dim3(blocks), kThreads, 0, st, "norm_kernel launch", table,
                        sums.partial + sums.blocks))
      return rc;
    sums.blocks += blocks;
  }
  // the last tensors first, like the pieces in a launch
  const int last = a.tensors ? (a.tensors - 1) / N * N : 0;
  for (int i = last; i >= 0; i -= N) {
    const auto table = table_of<N>(a, i, std::min(N, a.tensors - i), piece);
    if (!table.pieces && i != last) continue;                   // one launch at least writes the norm
    int types = table.tensors ? table.t[0].types & 255 : 0;
    for (int j = 1; j < table.tensors; ++j)
      if ((table.t[j].types & 255) != types) types = 0;
    auto scale = [&](auto pair) {
      return launch(scale_kernel<N, decltype(pair)::value>, dim3(std::max(1, blocks_of(table.pieces, kScaleBlocksPerSm))),
                    kThreads, 0, st, "scale_kernel launch", table, sums);
    };
    constexpr int F = OZ_F32, H = OZ_F16, B = OZ_BF16;
    int rc;
    if (types == (F | F << 4)) rc = scale(std::integral_constant<int, F | F << 4>{});
    else if (types == (H | H << 4)) rc = scale(std::integral_constant<int, H | H << 4>{});
    else if (types == (B | B << 4)) rc = scale(std::integral_constant<int, B | B << 4>{});
    else if (types == (H | F << 4)) rc = scale(std::integral_constant<int, H | F << 4>{});
    else if (types == (B | F << 4)) rc = scale(std::integral_constant<int, B | F << 4>{});
    else rc = scale(std::integral_constant<int, 0>{});
    if (rc) return rc;
  }
  return OZ_OK;
}

}  // namespace
}  // namespace oz

extern "C" int64_t oz_clip_workspace_bytes(int32_t tensors) {
  if (tensors < 0) return OZ_ERR_INVALID;
  const int64_t launches = tensors <= oz::kFew ? 1 : (tensors + oz::kMany - 1) / oz::kMany;
  return launches * oz::stream::sm_count() * oz::kBlocksPerSm * 8;
}

extern "C" int oz_clip(const oz_clip_args *args, void *stream) {
  if (!args) return oz::set_error(OZ_ERR_INVALID, "null arguments");
  using namespace oz;
  const oz_clip_args &a = *args;
  if (a.tensors < 0) return set_error(OZ_ERR_INVALID, "negative size");
  if (!a.norm || (a.tensors > 0 && (!a.grads || !a.outs || !a.sizes || !a.dtypes || !a.out_dtypes)))
    return set_error(OZ_ERR_INVALID, "null pointer");
  if (!aligned(4, {a.norm})) return not_aligned();
  if (!(a.max_norm >= 0) || !(a.eps >= 0)) return set_error(OZ_ERR_INVALID, "max_norm and eps must not be negative");
  const int64_t bytes = oz_clip_workspace_bytes(a.tensors);
  if (!a.workspace || (uintptr_t)a.workspace % 16 != 0 || a.workspace_bytes < bytes)
    return set_error(OZ_ERR_INVALID, "workspace of %lld bytes (16-byte aligned) needed, got %lld at %p",
                     (long long)bytes, (long long)a.workspace_bytes, a.workspace);
  struct Range { uintptr_t from, to; };
  thread_local std::vector<Range> ranges;
  try {
    ranges.clear();
    ranges.reserve(a.tensors);
    for (int i = 0; i < a.tensors; ++i) {
      for (int dt : {a.dtypes[i], a.out_dtypes[i]})
        if (dt != OZ_F32 && dt != OZ_F16 && dt != OZ_BF16)
          return set_error(OZ_ERR_UNSUPPORTED, "unsupported dtype %d of tensor %d (fp32, fp16 or bf16)", dt, i);
      if (a.sizes[i] < 0) return set_error(OZ_ERR_INVALID, "negative size of tensor %d", i);
      if (a.sizes[i] > (int64_t)1 << 42) return set_error(OZ_ERR_INVALID, "size out of range");
      if (a.sizes[i] == 0) continue;
      if (!a.grads[i] || !a.outs[i]) return set_error(OZ_ERR_INVALID, "null pointer of tensor %d", i);
      const int es = dtype_size(a.dtypes[i]), os = dtype_size(a.out_dtypes[i]);
      if ((uintptr_t)a.grads[i] % es || (uintptr_t)a.outs[i] % os)
        return set_error(OZ_ERR_INVALID, "tensor %d is not aligned to its elements", i);
      ranges.push_back({(uintptr_t)a.outs[i], (uintptr_t)a.outs[i] + (uintptr_t)a.sizes[i] * os});
    }
  } catch (...) {
    return set_error(OZ_ERR_INVALID, "out of host memory");
  }
  if (pieces_of(a, kSmallPiece) > INT32_MAX / 2) return set_error(OZ_ERR_INVALID, "size out of range");
  // results that share memory would be scaled twice, or in parts
  std::sort(ranges.begin(), ranges.end(), [](const Range &x, const Range &y) { return x.from < y.from; });
  for (size_t i = 1; i < ranges.size(); ++i)
    if (ranges[i].from < ranges[i - 1].to) return set_error(OZ_ERR_INVALID, "two results share memory");
  // and so would a result over another tensor's gradient, which is read again
  for (int i = 0; i < a.tensors; ++i) {
    if (a.sizes[i] == 0) continue;
    const uintptr_t g0 = (uintptr_t)a.grads[i], g1 = g0 + (uintptr_t)a.sizes[i] * dtype_size(a.dtypes[i]);
    const uintptr_t o0 = (uintptr_t)a.outs[i];
    auto it = std::upper_bound(ranges.begin(), ranges.end(), g0, [](uintptr_t v, const Range &r) { return v < r.to; });
    for (; it != ranges.end() && it->from < g1; ++it)
      if (!(it->from == o0 && g0 == o0 && a.dtypes[i] == a.out_dtypes[i]))
        return set_error(OZ_ERR_INVALID, "a result shares memory with a gradient, and is not that gradient");
  }
  const Sums sums{static_cast<double *>(a.workspace), a.norm, 0, (float)a.max_norm, (float)a.eps};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return a.tensors <= kFew ? run<kFew>(a, sums, st) : run<kMany>(a, sums, st);
}
