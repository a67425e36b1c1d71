// oz_stream.cuh -- pieces of the kernels that stream through memory: elements
// in 32 bits, 16 bytes of them at a time, and launches that overlap their start
// with the end of the kernel before.
#pragma once

#include <initializer_list>
#include <type_traits>

#include "oz_common.cuh"

namespace oz {
namespace stream {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of T as fp32 values and back.
template <typename T> __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[16 / sizeof(T)]) {
  const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i) v[i] = to_f32(e[i]);
}
template <typename T> __device__ __forceinline__ uint4 pack(const float (&v)[16 / sizeof(T)]) {
  uint4 u;
  T *e = reinterpret_cast<T *>(&u);
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i) e[i] = from_f32<T>(v[i]);
  return u;
}

// 16 bytes that are read once: they take no place in L1.  Not held in order against stores: for
// memory that the kernel does not write.  (du of 8192 x 8192 and its products 538 us a call, by plain
// loads 553; rows to tokens and back are 1 to 2 us faster by plain ones, of 75 and 168.)
__device__ __forceinline__ uint4 read_once(const void *p) {
  uint4 u;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
               : "l"(p));
  return u;
}

// V consecutive elements of T: 16 bytes, or one element where rows do not start
// on 16-byte boundaries.
template <typename T, int V> struct Run {
  static_assert(V == 1 || V * sizeof(T) == 16, "one element or 16 bytes");
  static __device__ __forceinline__ void load(const T *p, float (&v)[V]) {
    if constexpr (V == 1) v[0] = to_f32(*p);
    else unpack<T>(*reinterpret_cast<const uint4 *>(p), v);
  }
  static __device__ __forceinline__ void store(T *p, const float (&v)[V]) {
    if constexpr (V == 1) *p = from_f32<T>(v[0]);
    else *reinterpret_cast<uint4 *>(p) = pack<T>(v);
  }
};

// The same as it lies in memory: few registers for loads on their way.
template <typename T, int V, bool ONCE = false> struct Raw {
  using Type = typename std::conditional<V == 1, T, uint4>::type;
  static __device__ __forceinline__ Type load(const T *p) {
    if constexpr (V == 1) return *p;
    else if constexpr (ONCE) return read_once(p);
    else return *reinterpret_cast<const uint4 *>(p);
  }
  static __device__ __forceinline__ void store(T *p, const Type &v) { *reinterpret_cast<Type *>(p) = v; }
  static __device__ __forceinline__ void values(const Type &r, float (&v)[V]) {
    if constexpr (V == 1) v[0] = to_f32(r);
    else unpack<T>(r, v);
  }
};

// What follows reads by plain loads alone: a read-only one (ld.global.nc, __ldg) may be moved before
// the wait, and may find in L1 what stood there before an earlier kernel wrote it, as that kernel
// runs during this one's life.
__device__ __forceinline__ void start_after_earlier_kernels() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// A launch whose blocks may start while the kernel before ends; every kernel
// launched so calls start_after_earlier_kernels() before it touches memory.
template <typename... P, typename... A>
int launch(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t st, const char *what, A... args) {
  if (smem > 48 * 1024)
    if (int rc = set_smem_once((const void *)kernel, smem, what)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...), what);
}

inline int sm_count() {
  static const int n = [] {
    int dev = 0, v = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    return v > 0 ? v : 148;
  }();
  return n;
}

// Whether all addresses are multiples of an element's size (NULL is).
inline bool aligned(int size, std::initializer_list<const void *> addresses) {
  for (const void *p : addresses)
    if ((uintptr_t)p % size != 0) return false;
  return true;
}
inline int not_aligned() { return set_error(OZ_ERR_INVALID, "a tensor is not aligned to its elements"); }

// Calls f with a value of the element type that `dtype` names.
template <typename F> int with_type(int dtype, F f) {
  if (dtype == OZ_F32) return f(float{});
  if (dtype == OZ_F16) return f(__half{});
  if (dtype == OZ_BF16) return f(__nv_bfloat16{});
  return set_error(OZ_ERR_UNSUPPORTED, "unsupported dtype %d (fp32, fp16 or bf16)", dtype);
}

}  // namespace stream
}  // namespace oz
