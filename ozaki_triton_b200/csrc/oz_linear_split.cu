// oz_linear_split.cu -- fused products whose result has few tiles: one token against
// a weight matrix, a short chunk, the gradient of a small weight.
//
//   y = act(x w + bias) + residual     (or a plain product)
//
// What bounds them is the way of the operands' bytes to the SMs, so the contraction is
// divided over the CTAs of a cluster (up to 16), each with 128 columns of the result
// by up to 128 of its rows: tcgen05 products with the columns as A (their weights are
// read once, however few rows there are), fp32 sums in tensor memory.  The CTAs
// then put their sums into shared memory and each adds up, over the cluster, the
// rows that are its own, in the order of the CTAs, and finishes them.  No second
// launch, no atomics.  Two CTAs share an SM, so that one's start and end run under
// the other's loads.  1 x 2048 x 2816 (11.5 MB of weights, 1.8 us at the memory's rate): 6.7 us
// in a CUDA graph, bound by the launch, the first load's latency and the joining; 1 x 8192 x
// 8192: 25 us where the bytes need 21; the tile engine took 18 and 66.

#include <algorithm>
#include <cstring>

#include "oz_linear.cuh"

namespace oz {
int status_linear_split(int *value, bool clear) { return read_status_word(value, clear); }

namespace {
using namespace tile;
using namespace linear;

constexpr int kFinishWarps = 8;               // they read the sums, join and finish them
constexpr int kSplitThreads = 64 + 32 * kFinishWarps;
constexpr int kSplitRoom = 106 * 1024;        // shared memory of a CTA: two an SM
constexpr int kPassBlocks = 8;                // of an accumulator where the result is fp32

template <int NT> __host__ __device__ constexpr int split_stage() { return kRows * kLine + NT * kLine; }
template <int NT> __host__ __device__ constexpr int split_stages() {
  return (kSplitRoom - 2048) / split_stage<NT>() < 8 ? (kSplitRoom - 2048) / split_stage<NT>() : 8;
}
template <int NT> __host__ __device__ constexpr int split_smem() { return 1024 + split_stages<NT>() * split_stage<NT>() + 256; }

__device__ __forceinline__ float4 load_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
// 4 consecutive columns, at once or, up to `count`, one by one.
template <typename E> __device__ __forceinline__ void load4(const E *from, bool vectors, int count, float (&v)[4]) {
  if (vectors && count >= 4) {
    if constexpr (sizeof(E) == 4) {
      const float4 a = *(reinterpret_cast<const float4 *>(from));
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
      const uint2 a = *(reinterpret_cast<const uint2 *>(from));
      const E *e = reinterpret_cast<const E *>(&a);
#pragma unroll
      for (int x = 0; x < 4; ++x) v[x] = to_f32(e[x]);
    }
  } else {
#pragma unroll
    for (int x = 0; x < 4; ++x) v[x] = x < count ? to_f32(*(from + x)) : 0.f;
  }
}
template <typename E> __device__ __forceinline__ void store4(E *to, bool vectors, int count, const float (&v)[4]) {
  if (vectors && count >= 4) {
    if constexpr (sizeof(E) == 4) {
      *reinterpret_cast<float4 *>(to) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      uint2 a;
      E *e = reinterpret_cast<E *>(&a);
#pragma unroll
      for (int x = 0; x < 4; ++x) e[x] = from_f32<E>(v[x]);
      *reinterpret_cast<uint2 *>(to) = a;
    }
  } else {
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (x < count) to[x] = from_f32<E>(v[x]);
  }
}

// An operand off the 16-byte boundaries: the copy unit cannot read it, so the warps that
// finish the tile load it meanwhile.  A tile is lines of 64 elements, along the contraction or across it; a thread
// makes 16 bytes of a line from the one or two aligned 16 bytes that hold them (which share
// their 16 bytes with an element, so they can be read).
struct Loose {
  const void *p;               // none: the copy unit's
  int64_t pitch;
  int inner, outer;            // extents along a row and across
};
struct LooseTwo { Loose a, b; };

struct Piece {
  uint4 low, high;
  int shift, count;            // bytes into `low`; elements
  // elements [at, at + 8) of row `row`, as far as there are
  __device__ __forceinline__ void load(const Loose &o, int64_t row, int at) {
    count = row < o.outer ? min(max(o.inner - at, 0), 8) : 0;
    low = high = make_uint4(0, 0, 0, 0);
    shift = 0;
    if (count == 0) return;
    const uintptr_t from = (uintptr_t)o.p + 2 * (uintptr_t)(row * o.pitch + at);
    shift = (int)(from & 15);
    const uint4 *v = reinterpret_cast<const uint4 *>(from - shift);
    low = *(v);
    if (shift + 2 * count > 16) high = *(v + 1);
  }
  __device__ __forceinline__ uint4 value() const {
    uint32_t w[8] = {low.x, low.y, low.z, low.w, high.x, high.y, high.z, high.w};
    if (shift & 8)
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    if (shift & 4)
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[i] = shift & 2 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
      const int left = count - 2 * i;
      if (left < 2) out[i] = left == 1 ? out[i] & 0xFFFFu : 0u;
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
  }
};

// Adds up rows part, part + splits, ... of the cluster's sums (128 columns from column0 on; CTA
// first + apart s holds the s-th part of the contraction) and finishes them: the 8 last warps, a
// warp a row, 4 columns a lane.
template <typename O, typename T>
__device__ __forceinline__ void join_rows(const Params &p, const float *partial, int part, int splits, int first, int apart,
                                          int row0, int rows, int column0) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int column = column0 + lane * 4, count = min(p.n - column, 4);
  const uint32_t mine = smem_u32(partial) + (uint32_t)lane * 16;
  float bias[4] = {};
  if (p.bias && count > 0) {
    if (p.bias_f32) load4(static_cast<const float *>(p.bias) + column, p.vectors & kBiasVectors, count, bias);
    else load4(static_cast<const T *>(p.bias) + column, p.vectors & kBiasVectors, count, bias);
  }
  if (count > 0) {
    // two rows side by side: one's way through the instructions hides the other's
    constexpr int AT_ONCE = 2;
    const int step = kFinishWarps * splits;
    for (int r0 = part + (warp - 2) * splits; r0 < rows; r0 += AT_ONCE * step) {
      float u[AT_ONCE][4], residual[AT_ONCE][4];
      if (p.residual)
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
          if (r0 + i * step < rows)
            load4(static_cast<const O *>(p.residual) + (int64_t)(row0 + r0 + i * step) * p.residual_ld + column,
                  p.vectors & kResidualVectors, count, residual[i]);
      // 8 CTAs' sums on their way at a time, added in the order of the CTAs
      float4 v[AT_ONCE][8];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const int r = min(r0 + i * step, rows - 1);
        if (splits > 1) {
#pragma unroll
          for (int s = 0; s < 8; ++s)
            if (s < splits) v[i][s] = load_cluster(map_to_cta(mine + (uint32_t)(r * kRows * 4), first + apart * s));
        } else {
          v[i][0] = *reinterpret_cast<const float4 *>(partial + r * kRows + lane * 4);
        }
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        u[i][0] = v[i][0].x, u[i][1] = v[i][0].y, u[i][2] = v[i][0].z, u[i][3] = v[i][0].w;
#pragma unroll
        for (int s = 1; s < 8; ++s)
          if (s < splits) u[i][0] += v[i][s].x, u[i][1] += v[i][s].y, u[i][2] += v[i][s].z, u[i][3] += v[i][s].w;
      }
      if (splits > 8)
#pragma unroll 1
        for (int i = 0; i < AT_ONCE; ++i) {
          const int r = min(r0 + i * step, rows - 1);
#pragma unroll
          for (int s = 0; s < 8; ++s) v[0][s] = load_cluster(map_to_cta(mine + (uint32_t)(r * kRows * 4), first + apart * (8 + s)));
#pragma unroll
          for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j)
              if (i == j) u[j][0] += v[0][s].x, u[j][1] += v[0][s].y, u[j][2] += v[0][s].z, u[j][3] += v[0][s].w;
        }
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) u[i][x] += bias[x];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        if (r0 + i * step >= rows) continue;
        const int64_t at = (int64_t)(row0 + r0 + i * step) * p.ld + column;
        if (p.pre) store4(static_cast<T *>(p.pre) + at, p.vectors & kVectors, count, u[i]);
        activate(u[i], p.act);
        if (p.residual)
#pragma unroll
          for (int x = 0; x < 4; ++x) u[i][x] += residual[i][x];
        store4(static_cast<O *>(p.out) + at, p.vectors & kVectors, count, u[i]);
      }
    }
  }
}

// A: 128 columns of the result, B: NT rows.  O: the result's type, T: the operands'.
template <typename O, typename T, int NT, bool AMN, bool BMN>
__global__ void __launch_bounds__(kSplitThreads, 2)
    split_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const Params p,
                 const __grid_constant__ LooseTwo loose, const int splits) {
  constexpr int S = split_stages<NT>(), SB = split_stage<NT>(), A_BYTES = kRows * kLine;
  constexpr int PASS = sizeof(O) == 4 ? kPassBlocks : 1 << 28;
  constexpr int kTmemColumns = 2 * NT < 32 ? 32 : 2 * NT;
  static_assert(S >= 3 && NT * kRows * 4 <= S * SB, "shared memory");
  static_assert(NT % 16 == 0 && (!BMN || NT % 64 == 0), "rows of a tile");

  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  float *partial = reinterpret_cast<float *>(smem);            // [NT][128], after the products
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + S * SB);
  uint64_t *empty = full + S;
  uint64_t *acc_full = empty + S;                              // [2]
  uint64_t *acc_empty = acc_full + 2;                          // [2]
  uint64_t *drain = acc_empty + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = splits > 1 ? (int)cluster_ctarank() : 0;
  const int tile = blockIdx.x / splits;
  const int column0 = tile / p.row_tiles * kRows, row0 = tile % p.row_tiles * NT;
  const int blocks = (p.k + kBlock - 1) / kBlock;
  const int first = (int)((int64_t)blocks * rank / splits), last = (int)((int64_t)blocks * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], loose.a.p || loose.b.p ? 1 + kFinishWarps : 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kFinishWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    if (!loose.a.p) prefetch_tmap(&tm_a);
    if (!loose.b.p) prefetch_tmap(&tm_b);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  stream::start_after_earlier_kernels();

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (int kb = first; kb < last; ++kb, ++it) {
        const int slot = it % S;
        if (!mbar_wait_bounded(&empty[slot], ((it / S) & 1) ^ 1, abort_flag, DEV_TIMEOUT_PRODUCER)) break;
        unsigned char *sa = smem + slot * SB, *sb = sa + A_BYTES;
        mbar_arrive_expect_tx(&full[slot], (loose.a.p ? 0 : A_BYTES) + (loose.b.p ? 0 : NT * kLine));
        if (loose.a.p) {
        } else if constexpr (AMN) {
          tma_load_3d(sa, &tm_a, &full[slot], column0, kb * kBlock, 0);
          tma_load_3d(sa + kBlock * kLine, &tm_a, &full[slot], column0 + 64, kb * kBlock, 0);
        } else {
          tma_load_3d(sa, &tm_a, &full[slot], kb * kBlock, column0, 0);
        }
        if (loose.b.p) {
        } else if constexpr (BMN) {
#pragma unroll
          for (int c = 0; c < NT / 64; ++c)
            tma_load_3d(sb + c * kBlock * kLine, &tm_b, &full[slot], row0 + c * 64, kb * kBlock, 0);
        } else {
          tma_load_3d(sb, &tm_b, &full[slot], kb * kBlock, row0, 0);
        }
      }
      // every load has landed before shared memory is used for something else or goes away
      for (int k = max(it - S, 0); k < it; ++k)
        if (!mbar_settle(&full[k % S], (k / S) & 1, abort_flag, DEV_TIMEOUT_PRODUCER)) break;
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t base = smem_u32(smem);
      const uint64_t a_desc = operand_desc<AMN>(base), b_desc = operand_desc<BMN>(base + A_BYTES);
      constexpr uint64_t a_step = AMN ? (16 * kLine) >> 4 : 2, b_step = BMN ? (16 * kLine) >> 4 : 2;
      const uint32_t idesc = p.idesc | (uint32_t)(NT >> 3) << 17 | (uint32_t)(kRows >> 4) << 24 |
                             (AMN ? 1u << 15 : 0u) | (BMN ? 1u << 16 : 0u);
      int slot = 0;
      uint32_t phase = 0, done = 0;
      bool ok = true;
      for (int kb = first; ok && kb < last;) {
        const int stop = min(last - kb, PASS) + kb, buf = done & 1;
        if (!(ok = mbar_wait_bounded(&acc_empty[buf], ((done >> 1) & 1) ^ 1, abort_flag, DEV_TIMEOUT_MMA))) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(buf * NT);
        for (const int from = kb; kb < stop; ++kb) {
          if (!(ok = mbar_wait_bounded(&full[slot], phase, abort_flag, DEV_TIMEOUT_MMA))) break;
          tc_fence_after();
          const uint64_t ad = a_desc + slot * (SB >> 4), bd = b_desc + slot * (SB >> 4);
#pragma unroll
          for (int kk = 0; kk < kBlock / 16; ++kk)
            tc_mma<1>(d, ad + kk * a_step, bd + kk * b_step, idesc, kk || kb > from ? 1u : 0u);
          tc_commit(&empty[slot]);
          if (++slot == S) {
            slot = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        tc_commit(&acc_full[buf]);
        ++done;
      }
      tc_commit(drain);
      mbar_settle(drain, 0, abort_flag, DEV_TIMEOUT_MMA);
    }
  } else {
    if (loose.a.p || loose.b.p) {
      // 64 lines at a time, two 16 bytes a thread; the next ones are on their way while these
      // are stored
      constexpr int A_PARTS = kRows / 64, B_PARTS = (NT + 63) / 64;
      const int thread = threadIdx.x - 64, line = thread / 8, j = thread % 8;
      const int a_parts = loose.a.p ? A_PARTS : 0, parts = a_parts + (loose.b.p ? B_PARTS : 0);
      const int units = (last - first) * parts;
      auto load = [&](int unit, Piece (&to)[2]) {
        const int block = (first + unit / parts) * kBlock, part = unit % parts;
        const bool a = part < a_parts;
        const int at = (a ? part : part - a_parts) * 64;           // first line, or first element of lines
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int l = line + h * 32;
          if (a) {
            if (AMN) to[h].load(loose.a, block + l, column0 + at + j * 8);
            else to[h].load(loose.a, column0 + at + l, block + j * 8);
          } else {
            if (BMN) to[h].load(loose.b, block + l, row0 + at + j * 8);
            else to[h].load(loose.b, row0 + at + l, block + j * 8);
          }
        }
      };
      Piece now[2], next[2];
      load(0, now);
      bool ok = true;
#pragma unroll 1
      for (int unit = 0; unit < units; ++unit) {
        if (unit + 1 < units) load(unit + 1, next);
        const int it = unit / parts, part = unit - it * parts, slot = it % S;
        if (part == 0) {
          ok = mbar_wait_bounded(&empty[slot], ((it / S) & 1) ^ 1, abort_flag, DEV_TIMEOUT_PRODUCER);
          if (!__all_sync(0xffffffffu, ok)) break;
        }
        const bool a = part < a_parts;
        unsigned char *to = smem + slot * SB + (a ? part * (64 * kLine) : A_BYTES + (part - a_parts) * (64 * kLine));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int l = line + h * 32;
          // (a K-major B of fewer than 64 rows has no more lines than those)
          if (a || BMN || (part - a_parts) * 64 + l < NT)
            *reinterpret_cast<uint4 *>(to + l * kLine + ((j ^ (l & 7)) << 4)) = now[h].value();
          now[h] = next[h];
        }
        if (part == parts - 1) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[slot]);
        }
      }
    }
    // sums to shared memory (once the last accumulator is there, the products are done with
    // it): two warps a quarter of the lanes, half of the rows each
    constexpr int HALF = NT / 2 < 16 ? 16 : NT / 2;
    const int sub = warp & 3, from = (warp - 2) / 4 * HALF, rows = min(min(p.rows - row0, NT) - from, min(HALF, NT - from));
    const uint32_t columns = tmem + ((uint32_t)(sub * 32) << 16) + (uint32_t)from;
    float *to = partial + from * kRows + sub * 32 + lane;
    uint32_t done = 0;
    auto acquire = [&]() {
      const bool ok = mbar_wait_bounded(&acc_full[done & 1], (done >> 1) & 1, abort_flag, DEV_TIMEOUT_EPILOGUE);
      if (!__all_sync(0xffffffffu, ok)) return false;
      tc_fence_after();
      return true;
    };
    if constexpr (sizeof(O) == 4) {
      float sum[HALF];
#pragma unroll
      for (int r = 0; r < HALF; ++r) sum[r] = 0.f;
      for (int kb = first; kb < last; kb += PASS) {
        if (!acquire()) break;
        if (rows > 0) {
#pragma unroll
          for (int r0 = 0; r0 < HALF; r0 += 16) {
            uint32_t v[16];
            tmem_ld16_at(columns + (uint32_t)((done & 1) * NT + r0), v);
            tmem_ld_wait16(v);
#pragma unroll
            for (int x = 0; x < 16; ++x) sum[r0 + x] += __uint_as_float(v[x]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[done & 1]);
        ++done;
      }
#pragma unroll
      for (int r = 0; r < HALF; ++r)
        if (r < rows) to[r * kRows] = sum[r];
    } else {
      acquire();
#pragma unroll 1
      for (int r0 = 0; r0 < rows; r0 += 16) {
        uint32_t v[16];
        tmem_ld16_at(columns + (uint32_t)r0, v);
        tmem_ld_wait16(v);
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (r0 + x < rows) to[(r0 + x) * kRows] = __uint_as_float(v[x]);
      }
    }
  }
  __syncwarp();                                // lane 0 of the first two warps comes from its loop
  if (splits > 1) cluster_sync();
  else __syncthreads();
  if (warp >= 2) {
    join_rows<O, T>(p, partial, rank, splits, 0, 1, row0, min(p.rows - row0, NT), column0);
  }
  tc_fence_before();
  if (splits > 1) cluster_sync();              // nobody's sums go away while they are read
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemColumns);
  }
}

// The same for results of a few tiles of 256 x 256, whose operands' way from L2 to the SMs
// bounds them: pairs of CTAs hold half of a tile's columns and rows each (as in the tile engine)
// and multiply them by one instruction, and the 2 or 4 pairs of a cluster share the contraction.
// 16-bit results only: their sums are of one pass.
constexpr int kPairRows = 256, kPairStage = 2 * kRows * kLine, kPairStages = 6;
constexpr int kPairSmem = 1024 + kPairStages * kPairStage + 256;

// Arrive on the barrier at this offset of both CTAs of pair q once the products so far are done.
__device__ __forceinline__ void commit_to_pair(uint32_t bar, int q) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((uint16_t)(3 << (2 * q)))
      : "memory");
}

template <typename T, bool AMN, bool BMN>
__global__ void __launch_bounds__(kSplitThreads, 1)
    pair_split_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const Params p,
                      const int splits) {
  constexpr int S = kPairStages, SB = kPairStage, A_BYTES = kRows * kLine, NT = kPairRows;
  static_assert(NT * kRows * 4 <= S * SB && kPairSmem <= kSmemLimit, "shared memory");
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  float *partial = reinterpret_cast<float *>(smem);            // [NT][128], after the products
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + S * SB);
  uint64_t *empty = full + S;
  uint64_t *acc_full = empty + S;
  uint64_t *drain = acc_full + 1;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = (int)cluster_ctarank(), q = rank / 2, half = rank % 2;
  const bool leader = half == 0;
  const int tile = blockIdx.x / (2 * splits);
  const int column0 = tile / p.row_tiles * (2 * kRows) + half * kRows, row0 = tile % p.row_tiles * NT;
  const int blocks = (p.k + kBlock - 1) / kBlock;
  const int first = (int)((int64_t)blocks * q / splits), last = (int)((int64_t)blocks * (q + 1) / splits);

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, NT);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  stream::start_after_earlier_kernels();

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      const int br = row0 + half * kRows;
      for (int kb = first; kb < last; ++kb, ++it) {
        const int slot = it % S;
        if (!mbar_wait_bounded(&empty[slot], ((it / S) & 1) ^ 1, abort_flag, DEV_TIMEOUT_PRODUCER)) break;
        unsigned char *sa = smem + slot * SB, *sb = sa + A_BYTES;
        if (leader) mbar_arrive_expect_tx(&full[slot], 2 * SB);
        const uint32_t bar = map_to_cta(smem_u32(&full[slot]), 2 * q);
        if constexpr (AMN) {
          tma_load_3d_pair(sa, &tm_a, bar, column0, kb * kBlock, 0);
          tma_load_3d_pair(sa + kBlock * kLine, &tm_a, bar, column0 + 64, kb * kBlock, 0);
        } else {
          tma_load_3d_pair(sa, &tm_a, bar, kb * kBlock, column0, 0);
        }
        if constexpr (BMN) {
          tma_load_3d_pair(sb, &tm_b, bar, br, kb * kBlock, 0);
          tma_load_3d_pair(sb + kBlock * kLine, &tm_b, bar, br + 64, kb * kBlock, 0);
        } else {
          tma_load_3d_pair(sb, &tm_b, bar, kb * kBlock, br, 0);
        }
      }
      // every load has landed, and every stage is reported as read, before shared memory is used for
      // something else or goes away
      if (leader)
        for (int k = max(it - S, 0); k < it; ++k)
          if (!mbar_settle(&full[k % S], (k / S) & 1, abort_flag, DEV_TIMEOUT_PRODUCER)) break;
      for (int k = max(it - S, 0); k < it; ++k)
        if (!mbar_settle(&empty[k % S], (k / S) & 1, abort_flag, DEV_TIMEOUT_PRODUCER)) break;
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      const uint32_t base = smem_u32(smem);
      const uint64_t a_desc = operand_desc<AMN>(base), b_desc = operand_desc<BMN>(base + A_BYTES);
      constexpr uint64_t a_step = AMN ? (16 * kLine) >> 4 : 2, b_step = BMN ? (16 * kLine) >> 4 : 2;
      const uint32_t idesc = p.idesc | (uint32_t)(NT >> 3) << 17 | (uint32_t)((2 * kRows) >> 4) << 24 |
                             (AMN ? 1u << 15 : 0u) | (BMN ? 1u << 16 : 0u);
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = first; kb < last; ++kb) {
        if (!(ok = wait_cluster(&full[slot], phase, abort_flag, DEV_TIMEOUT_MMA))) break;
        tc_fence_after();
        const uint64_t ad = a_desc + slot * (SB >> 4), bd = b_desc + slot * (SB >> 4);
#pragma unroll
        for (int kk = 0; kk < kBlock / 16; ++kk)
          tc_mma_pair<1>(tmem, ad + kk * a_step, bd + kk * b_step, idesc, kk || kb > first ? 1u : 0u);
        commit_to_pair(smem_u32(&empty[slot]), q);
        if (++slot == S) {
          slot = 0;
          phase ^= 1;
        }
      }
      if (ok) commit_to_pair(smem_u32(acc_full), q);
      tc_commit_pair(smem_u32(drain));
      mbar_settle(drain, 0, abort_flag, DEV_TIMEOUT_MMA);
    }
  } else {
    // sums to shared memory (once they are there, the products are done with it): two warps a
    // quarter of the lanes, half of the rows each
    const int sub = warp & 3, from = (warp - 2) / 4 * (NT / 2), rows = min(p.rows - row0 - from, NT / 2);
    const uint32_t columns = tmem + ((uint32_t)(sub * 32) << 16) + (uint32_t)from;
    float *to = partial + from * kRows + sub * 32 + lane;
    const bool ok = mbar_wait_bounded(acc_full, 0, abort_flag, DEV_TIMEOUT_EPILOGUE);
    if (__all_sync(0xffffffffu, ok)) {
      tc_fence_after();
#pragma unroll 1
      for (int r0 = 0; r0 < rows; r0 += 16) {
        uint32_t v[16];
        tmem_ld16_at(columns + (uint32_t)r0, v);
        tmem_ld_wait16(v);
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (r0 + x < rows) to[(r0 + x) * kRows] = __uint_as_float(v[x]);
      }
    }
  }
  __syncwarp();
  cluster_sync();
  if (warp >= 2) join_rows<T, T>(p, partial, q, splits, half, 2, row0, min(p.rows - row0, NT), column0);
  tc_fence_before();
  cluster_sync();                              // nobody's sums go away while they are read
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, NT);
  }
}

// Clusters of 16 are past what every GPU of the kind must hold: a kernel has to ask, once a device.
int allow_large_clusters(const void *kernel, const char *what) {
  constexpr int kDevs = 64;
  static std::mutex mu;
  static std::unordered_map<const void *, bool> asked[kDevs];
  int dev = -1;
  const bool known = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kDevs;
  if (known) {
    std::lock_guard<std::mutex> lk(mu);
    if (asked[dev].count(kernel)) return OZ_OK;
  }
  const int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), what);
  if (rc == OZ_OK && known) {
    std::lock_guard<std::mutex> lk(mu);
    asked[dev][kernel] = true;
  }
  return rc;
}

template <typename O, typename T, int NT, bool AMN, bool BMN>
int run_split(const Side &a, const Side &b, Params p, int splits, cudaStream_t st, const char *what) {
  // a lies along the result's rows: the kernel's B
  CUtensorMap tc, tr;
  const int64_t ci = AMN ? p.n : p.k, cr = AMN ? p.k : p.n, ri = BMN ? p.rows : p.k, rr = BMN ? p.k : p.rows;
  const int64_t cp = pitch_bytes(b.pitch, cr, ci), rp = pitch_bytes(a.pitch, rr, ri);
  LooseTwo loose{};
  if (!readable(b.p, cr, b.pitch, 1, 0)) {
    loose.a = Loose{b.p, b.pitch, (int)ci, (int)cr};
    memset(&tc, 0, sizeof(tc));                // not used
  } else if (int rc = make_map(&tc, b.p, ci, cr, 1, cp, cp, AMN ? kBlock : kRows)) {
    return rc;
  }
  if (!readable(a.p, rr, a.pitch, 1, 0)) {
    loose.b = Loose{a.p, a.pitch, (int)ri, (int)rr};
    memset(&tr, 0, sizeof(tr));
  } else if (int rc = make_map(&tr, a.p, ri, rr, 1, rp, rp, BMN ? kBlock : NT)) {
    return rc;
  }
  const int64_t rows = (p.rows + NT - 1) / NT, columns = (p.n + kRows - 1) / kRows;
  if (rows * columns * splits > INT32_MAX / 2) return set_error(OZ_ERR_INVALID, "too many tiles");
  p.row_tiles = (int)rows;
  p.column_tiles = (int)columns;
  auto kernel = split_kernel<O, T, NT, AMN, BMN>;
  constexpr int smem = split_smem<NT>();
  if (int rc = set_smem_once((const void *)kernel, smem, what)) return rc;
  if (splits > 8)
    if (int rc = allow_large_clusters((const void *)kernel, what)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * columns * splits));
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  count_launch();
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, tc, tr, p, loose, splits), what);
}

template <typename T, bool AMN, bool BMN>
int run_pairs(const Side &a, const Side &b, Params p, int splits, cudaStream_t st, const char *what) {
  CUtensorMap tc, tr;
  const int64_t ci = AMN ? p.n : p.k, cr = AMN ? p.k : p.n, ri = BMN ? p.rows : p.k, rr = BMN ? p.k : p.rows;
  const int64_t cp = pitch_bytes(b.pitch, cr, ci), rp = pitch_bytes(a.pitch, rr, ri);
  if (int rc = make_map(&tc, b.p, ci, cr, 1, cp, cp, AMN ? kBlock : kRows)) return rc;
  if (int rc = make_map(&tr, a.p, ri, rr, 1, rp, rp, BMN ? kBlock : kRows)) return rc;
  const int64_t rows = (p.rows + kPairRows - 1) / kPairRows, columns = (p.n + 2 * kRows - 1) / (2 * kRows);
  if (rows * columns * splits > INT32_MAX / 4) return set_error(OZ_ERR_INVALID, "too many tiles");
  p.row_tiles = (int)rows;
  p.column_tiles = (int)columns;
  auto kernel = pair_split_kernel<T, AMN, BMN>;
  if (int rc = set_smem_once((const void *)kernel, kPairSmem, what)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * columns * splits * 2));
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2 * splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  count_launch();
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, tc, tr, p, splits), what);
}

template <typename T>
int pairs_of(int splits, const Side &a, const Side &b, const Params &p, cudaStream_t st, const char *what) {
  if (a.mn) return b.mn ? run_pairs<T, true, true>(a, b, p, splits, st, what)
                        : set_error(OZ_ERR_UNSUPPORTED, "operand layout");
  return b.mn ? run_pairs<T, true, false>(a, b, p, splits, st, what)
              : run_pairs<T, false, false>(a, b, p, splits, st, what);
}

template <typename O, typename T>
int split_of(const SplitPlan &plan, const Side &a, const Side &b, const Params &p, cudaStream_t st, const char *what) {
  const int s = plan.splits;
  if (a.mn) {
    if (!b.mn) return set_error(OZ_ERR_UNSUPPORTED, "operand layout");
    return plan.tile_rows <= 64 ? run_split<O, T, 64, true, true>(a, b, p, s, st, what)
                                : run_split<O, T, 128, true, true>(a, b, p, s, st, what);
  }
  if (b.mn)
    return plan.tile_rows <= 16   ? run_split<O, T, 16, true, false>(a, b, p, s, st, what)
           : plan.tile_rows <= 64 ? run_split<O, T, 64, true, false>(a, b, p, s, st, what)
                                  : run_split<O, T, 128, true, false>(a, b, p, s, st, what);
  return plan.tile_rows <= 16   ? run_split<O, T, 16, false, false>(a, b, p, s, st, what)
         : plan.tile_rows <= 64 ? run_split<O, T, 64, false, false>(a, b, p, s, st, what)
                                : run_split<O, T, 128, false, false>(a, b, p, s, st, what);
}

}  // namespace

namespace linear {

int split_product(const SplitPlan &plan, int dtype, int out_dtype, const Side &a, const Side &b, const Params &p,
                  cudaStream_t st, const char *what) {
  if (plan.tile_rows == kPairTile) {
    if (out_dtype != dtype) return set_error(OZ_ERR_UNSUPPORTED, "output dtype %d", out_dtype);
    return dtype == OZ_F16 ? pairs_of<__half>(plan.splits, a, b, p, st, what)
                           : pairs_of<__nv_bfloat16>(plan.splits, a, b, p, st, what);
  }
  if (dtype == OZ_F16)
    return out_dtype == OZ_F32 ? split_of<float, __half>(plan, a, b, p, st, what)
                               : split_of<__half, __half>(plan, a, b, p, st, what);
  return out_dtype == OZ_F32 ? split_of<float, __nv_bfloat16>(plan, a, b, p, st, what)
                             : split_of<__nv_bfloat16, __nv_bfloat16>(plan, a, b, p, st, what);
}

}  // namespace linear
}  // namespace oz
