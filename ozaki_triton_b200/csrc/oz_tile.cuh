// oz_tile.cuh -- a persistent tcgen05 tile engine for products of fp16 / bf16
// operands whose tiles, extents and epilogues differ from job to job.
//
// A job (a class with the members used below) says which tiles there are,
// where their operands lie and what becomes of an accumulator; the engine
// moves the data and issues the matrix instructions:
//   warp 0     TMA producer: 64-deep blocks of A and B into a ring of stages;
//   warp 1     TMEM allocator and the one thread that issues tcgen05.mma;
//   warps 2-9  epilogue: the job's, from TMEM (fp32 accumulators, two buffers,
//              so the epilogue of one tile runs under the products of the next;
//              16 warps and a stage less were 2% slower forward, 10% for dw).
// A tile is 128 * PAIR rows by NT columns; with PAIR = 2 two CTAs of a
// cluster hold half of A's rows and half of B's columns each and one
// cta_group::2 instruction multiplies both halves: each CTA then feeds 256
// rows or columns of products with 128 of its own loads.
//
// An operand is stored either along the contraction ("K-major") or across it
// ("MN-major": AMN / BMN).  Both are staged with the 128-byte swizzle; an
// MN-major tile is a row of chunks of 64 elements, each chunk 64 contraction
// rows of 128 bytes.  Elements outside a tensor's extents arrive as zeros.
// With RAGGED the contraction runs over a tile's own range of rows
// [k_begin, k_begin + k_len) of longer operands: the rows of the last block
// past the range are overwritten with zeros in shared memory before they are
// multiplied (in both operands: a zero times a stray NaN is a NaN), as far as
// the last instruction of 16 reads.  A warp of its own does that as soon as the
// block is there, ahead of the products (done by the MMA warp in its turn it
// cost 8 of 48 us on 256 tiles of 4 blocks).
//
// With VARIABLE a tile has t.n <= NT columns, a multiple of 32, and both the loads
// (B's rows in one or two boxes of 64) and the instructions go by that.
//
// With PASS > 0 an accumulator takes at most PASS blocks and the epilogue adds
// the passes in registers: the tensor core cuts each sum off instead of
// rounding it, an error that grows with the number of blocks (relative 1.1e-6
// at 2048 terms of one sign), and that an fp32 result would show.
//
// With PLANES = 2 each operand is a sum of two fp16 slices and a block adds
// high*high, high*low and low*high to the accumulator (low*low is below the
// last bit of the others).
//
// Every wait is bounded (oz_common.cuh).
#pragma once

#include "oz_common.cuh"

namespace oz {
namespace tile {

constexpr int kRows = 128;              // rows of one CTA's part of a tile
constexpr int kBlock = 64;              // contraction elements of a stage
constexpr int kLine = 128;              // bytes of a swizzled row
constexpr int kMaxStages = 10;
constexpr int kStagingBytes = 2048;     // of each epilogue warp: 32 rows of 64 bytes
constexpr int kBarrierBytes = 512;
constexpr int kSmemLimit = 227 * 1024;

// For jobs whose epilogue reads nothing but the accumulators.
struct NoLookAhead {
  static constexpr bool VARIABLE = false;
  struct Ahead {};
  template <class P, class T> static __device__ void look_ahead(const P &, const T &, int, int, Ahead &) {}
};

// epilogue warps: 8, or what the job says
template <class J, class = void> struct EpilogueWarps { static constexpr int value = 8; };
template <class J> struct EpilogueWarps<J, decltype((void)J::EPILOGUE_WARPS)> { static constexpr int value = J::EPILOGUE_WARPS; };
template <class J> __host__ __device__ constexpr int epilogue_warps() { return EpilogueWarps<J>::value; }
template <class J> __host__ __device__ constexpr int threads() { return 64 + 32 * epilogue_warps<J>() + (J::RAGGED ? 32 : 0); }
// columns of an epilogue warp (4 warps share the rows of a tile, a quarter each)
template <class J> __host__ __device__ constexpr int warp_columns() { return J::NT * 4 / epilogue_warps<J>(); }
template <class J> __host__ __device__ constexpr int a_bytes() { return kRows * kLine; }
template <class J> __host__ __device__ constexpr int b_bytes() { return J::NT / J::PAIR * kLine; }
template <class J> __host__ __device__ constexpr int stage_bytes() { return J::PLANES * (a_bytes<J>() + b_bytes<J>()); }
template <class J> __host__ __device__ constexpr int stages() {
  constexpr int room = kSmemLimit - 1024 - kBarrierBytes - epilogue_warps<J>() * kStagingBytes;
  constexpr int n = room / stage_bytes<J>();
  return n < kMaxStages ? n : kMaxStages;
}
template <class J> __host__ __device__ constexpr int smem_bytes() {
  return 1024 + stages<J>() * stage_bytes<J>() + epilogue_warps<J>() * kStagingBytes + kBarrierBytes;
}

// Where a tile's operands lie: first row (or column) and matrix of A and B in
// their tensor maps, the contraction range, and what the job's epilogue wants.
template <class Extra> struct TileOf {
  int a_row, a_mat, b_row, b_mat, n;
  int64_t k_begin, k_len;
  Extra extra;
};

// 3-D tensor map: `inner` contiguous elements, `rows` of them `row_bytes`
// apart, `mats` of those `mat_bytes` apart, and the box of a copy.
inline int encode(CUtensorMap *map, CUtensorMapDataType type, const void *base, int64_t inner, int64_t rows,
                  int64_t mats, int64_t row_bytes, int64_t mat_bytes, int box_inner, int box_rows, int box_mats,
                  CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)mats};
  const cuuint64_t strides[2] = {(cuuint64_t)row_bytes, (cuuint64_t)mat_bytes};
  const cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows, (cuuint32_t)box_mats};
  return encode_tiled(map, type, base, dims, strides, box, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

// A 16-bit operand of the engine: boxes of 64 elements x box_rows, swizzled.
inline int make_map(CUtensorMap *map, const void *base, int64_t inner, int64_t rows, int64_t mats,
                    int64_t row_bytes, int64_t mat_bytes, int box_rows) {
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, base, inner, rows, mats, row_bytes, mat_bytes, kBlock,
                box_rows, 1, CU_TENSOR_MAP_SWIZZLE_128B);
}

inline int sm_count() {
  static int n = 0;
  if (!n) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (n <= 0) n = 148;
  }
  return n;
}

// Shared-memory descriptors (128-byte swizzle).  K-major: rows of 128 bytes,
// 1024 bytes from one group of 8 rows to the next.  MN-major: chunks of 64
// elements 64 * 128 bytes apart, 1024 bytes from 8 contraction rows to the next.
template <bool MN> __device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  if constexpr (!MN) return smem_desc_sw128(addr);
  uint64_t d = (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)((kBlock * kLine) >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// Wait for arrivals of the other CTA of a pair too (acquire over the cluster).
__device__ __forceinline__ bool wait_cluster(uint64_t *bar, uint32_t parity, volatile int *abort,
                                             int code) {
  const uint32_t a = smem_u32(bar);
  auto there = [&]() {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(a), "r"(parity)
        : "memory");
    return ok != 0;
  };
  if (there()) return true;
  const long long t0 = clock64();
  for (uint32_t it = 0;; ++it) {
    if (there()) return true;
    if ((it & 63u) == 63u) {
      if (*abort) return false;
      if (clock64() - t0 > kWaitBoundCycles) {
        *abort = code;
        atomicCAS(&g_device_status, 0, code);
        return false;
      }
    }
  }
}

// Where an epilogue finds its warp's accumulators, 32 rows (one a lane) by
// its columns, 16 at a time: in TMEM (zeros for an empty
// contraction), or summed over the passes in registers.
struct Columns {
  bool some;
  uint32_t addr;
  __device__ __forceinline__ void read(int c, float (&v)[16]) const {
    if (some) {
      uint32_t r[16];
      tmem_ld16_at(addr + (uint32_t)c, r);
      tmem_ld_wait16(r);
#pragma unroll
      for (int x = 0; x < 16; ++x) v[x] = __uint_as_float(r[x]);
    } else {
#pragma unroll
      for (int x = 0; x < 16; ++x) v[x] = 0.f;
    }
  }
};
template <int N> struct Registers {
  const float (&sum)[N];
  __device__ __forceinline__ void read(int c, float (&v)[16]) const {
#pragma unroll
    for (int x = 0; x < 16; ++x) v[x] = sum[c + x];
  }
};

// Tell the pair's leader that this warp has read its accumulators.  No memory is
// handed over (TMEM is ordered by the tcgen05 fence before), so the arrival is not
// a release over the cluster, which would wait for the warp's stores to land.
__device__ __forceinline__ void arrive_at_leader(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <class J>
__global__ void __launch_bounds__(threads<J>(), 1)
    tile_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                const typename J::Params p) {
  using Tile = TileOf<typename J::Extra>;
  constexpr int PAIR = J::PAIR, NT = J::NT, S = stages<J>(), SB = stage_bytes<J>();
  constexpr int kEpilogueWarps = epilogue_warps<J>();
  constexpr int BR = NT / PAIR;                       // B rows (columns of the tile) of one CTA
  constexpr int kTmemColumns = 2 * NT < 32 ? 32 : 2 * NT;
  static_assert((NT & (NT - 1)) == 0 && NT >= 32 && NT <= 256 && 2 * NT <= 512, "tile columns");
  static_assert(!J::BMN || BR % 64 == 0, "an MN-major B comes in chunks of 64");
  static_assert(S >= 3, "too few stages");
  static_assert(!J::VARIABLE || !J::BMN, "a variable B is stored along the contraction");

  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char *staging = smem + S * SB;
  uint64_t *full = reinterpret_cast<uint64_t *>(staging + kEpilogueWarps * kStagingBytes);
  uint64_t *empty = full + kMaxStages;
  uint64_t *acc_full = empty + kMaxStages;            // [2]
  uint64_t *acc_empty = acc_full + 2;                 // [2]
  uint64_t *drain = acc_empty + 2;
  uint64_t *tail = drain + 1;                         // RAGGED: this CTA's last block has landed
  uint64_t *peer_tail = tail + kMaxStages;            // RAGGED: the other CTA's has been cleared
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(peer_tail + kMaxStages);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = PAIR == 2 ? cluster_ctarank() : 0;
  const bool leader = rank == 0;
  const int unit = blockIdx.x / PAIR, units = gridDim.x / PAIR;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&tail[i], 1);
      mbar_init(&peer_tail[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], PAIR * kEpilogueWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
  }
  if (warp == 1) {
    if constexpr (PAIR == 2) {
      tmem_alloc_pair(tmem_slot, kTmemColumns);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, kTmemColumns);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (PAIR == 2) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // up to here nothing depends on earlier kernels: the next launch may do as
  // much while this one runs, and this one waits here for what came before
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  auto leader_addr = [&](uint64_t *bar) -> uint32_t {
    if constexpr (PAIR == 2) return map_to_cta(smem_u32(bar), 0);
    else return smem_u32(bar);
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    typename J::Walk walk(p);
    Tile t;
    uint32_t it = 0, ended = 0, turn = 0;             // slots whose tail was used; parity of the last use
    bool ok = true;
    for (int i = unit; ok && walk.find(p, i, t); i += units) {
      const int blocks = (int)((t.k_len + kBlock - 1) / kBlock);
      const bool ragged = J::RAGGED && t.k_len % kBlock;
      if (lane == 0) {
        const int ar = t.a_row + (int)rank * kRows;
        const int br = t.b_row + (int)rank * (J::VARIABLE ? t.n / PAIR : BR);
        const bool two = t.n / PAIR > 64;
        const uint32_t bytes = J::VARIABLE ? J::PLANES * (a_bytes<J>() + (two ? 128 : 64) * kLine) : SB;
        // the boxes of block kb: into this CTA, counted on the leader's barrier, or for a
        // block that ends the range on each CTA's own, for its clearing warp
        auto block = [&](int kb, unsigned char *st, uint32_t bar, uint64_t *own) {
          auto load = [&](void *dst, const CUtensorMap *map, int c0, int c1, int c2) {
            if constexpr (PAIR == 2) {
              if (!own) tma_load_3d_pair(dst, map, bar, c0, c1, c2);
              else tma_load_3d(dst, map, own, c0, c1, c2);
            } else {
              tma_load_3d(dst, map, own, c0, c1, c2);
            }
          };
          const int k = (int)(t.k_begin + (int64_t)kb * kBlock);
#pragma unroll
          for (int pl = 0; pl < J::PLANES; ++pl) {
            unsigned char *sa = st + pl * a_bytes<J>();
            unsigned char *sb = st + J::PLANES * a_bytes<J>() + pl * b_bytes<J>();
            const int am = t.a_mat + pl * J::plane_stride(p), bm = t.b_mat + pl * J::plane_stride(p);
            if constexpr (J::AMN) {
#pragma unroll
              for (int c = 0; c < kRows / 64; ++c)
                load(sa + c * kBlock * kLine, &tm_a, ar + c * 64, k, am);
            } else {
              load(sa, &tm_a, k, ar, am);
            }
            if constexpr (J::BMN) {
#pragma unroll
              for (int c = 0; c < BR / 64; ++c)
                load(sb + c * kBlock * kLine, &tm_b, br + c * 64, k, bm);
            } else if constexpr (J::VARIABLE) {
              load(sb, &tm_b, k, br, bm);
              if (two) load(sb + 64 * kLine, &tm_b, k, br + 64, bm);
            } else {
              load(sb, &tm_b, k, br, bm);
            }
          }
        };
        const int whole = blocks - (ragged ? 1 : 0);
        for (int kb = 0; kb < whole; ++kb, ++it) {
          const int slot = it % S;
          if (!(ok = mbar_wait_bounded(&empty[slot], ((it / S) & 1) ^ 1, abort_flag, DEV_TIMEOUT_PRODUCER))) break;
          if (leader) mbar_arrive_expect_tx(&full[slot], PAIR * bytes);
          block(kb, smem + slot * SB, leader_addr(&full[slot]), PAIR == 2 ? nullptr : &full[slot]);
        }
        if (ragged && ok) {
          const int slot = it % S;
          ok = mbar_wait_bounded(&empty[slot], ((it / S) & 1) ^ 1, abort_flag, DEV_TIMEOUT_PRODUCER);
          if (ok) {
            mbar_arrive_expect_tx(&tail[slot], SB);
            turn ^= ((ended >> slot) & 1) << slot;
            ended |= 1u << slot;
            block(whole, smem + slot * SB, 0, &tail[slot]);
            ++it;
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
    }
    // every load must have landed before shared memory goes away (a block that ends a
    // range counts on `full` only through the clearing warp); past the first that does not
    // within its limit, nothing can still be under way
    if (lane == 0)
      for (int slot = 0; J::RAGGED && slot < S; ++slot)
        if (((ended >> slot) & 1) && !mbar_settle(&tail[slot], (turn >> slot) & 1, abort_flag, DEV_TIMEOUT_PRODUCER))
          break;
    if (lane == 0 && leader)
      for (uint32_t k = (it > (uint32_t)S ? it - S : 0); k < it; ++k)
        if (!mbar_settle(&full[k % S], (k / S) & 1, abort_flag, DEV_TIMEOUT_PRODUCER)) break;
    // nor may this CTA leave while the pair's leader still reports a stage as read to its
    // barriers (the reports come from the other SM)
    if (lane == 0)
      for (uint32_t k = (it > (uint32_t)S ? it - S : 0); k < it; ++k)
        if (!mbar_settle(&empty[k % S], (k / S) & 1, abort_flag, DEV_TIMEOUT_PRODUCER)) break;
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    typename J::Walk walk(p);
    Tile t;
    uint32_t done = 0;
    bool ok = true;
    const uint32_t base = smem_u32(smem);
    const uint32_t fixed = p.idesc | (J::VARIABLE ? 0u : (uint32_t)(NT >> 3) << 17) |
                           ((uint32_t)((kRows * PAIR) >> 4) << 24) | (J::AMN ? 1u << 15 : 0u) |
                           (J::BMN ? 1u << 16 : 0u);
    constexpr uint64_t a_step = J::AMN ? (16 * kLine) >> 4 : 2, b_step = J::BMN ? (16 * kLine) >> 4 : 2;
    auto release = [&](uint64_t *bar) {
      if constexpr (PAIR == 2) tc_commit_both(smem_u32(bar));
      else tc_commit(bar);
    };
    auto wait = [&](uint64_t *bar, uint32_t parity) {
      if constexpr (PAIR == 2) return wait_cluster(bar, parity, abort_flag, DEV_TIMEOUT_MMA);
      else return mbar_wait_bounded(bar, parity, abort_flag, DEV_TIMEOUT_MMA);
    };
    // the issuing thread must not fall behind the tensor core, which holds only
    // a few instructions: descriptors are one base plus the slot's offset
    const uint64_t a_desc = operand_desc<J::AMN>(base);
    const uint64_t b_desc = operand_desc<J::BMN>(base + J::PLANES * a_bytes<J>());
    uint32_t slot = 0, phase = 0;
    uint32_t idesc = fixed;
    auto instruction = [&](uint32_t d, uint64_t ad, uint64_t bd, uint32_t add) {
      if constexpr (PAIR == 2) tc_mma_pair<1>(d, ad, bd, idesc, add);
      else tc_mma<1>(d, ad, bd, idesc, add);
    };
    auto multiply = [&](uint32_t d, bool first) {
      const uint64_t ad = a_desc + slot * (SB >> 4), bd = b_desc + slot * (SB >> 4);
#pragma unroll
      for (int q = 0; q < (J::PLANES == 2 ? 3 : 1); ++q) {
        // the small products first: what the sum cuts off is relative to its size
        const uint64_t aq = ad + (J::PLANES == 2 && q == 0 ? a_bytes<J>() >> 4 : 0);
        const uint64_t bq = bd + (q == 1 ? b_bytes<J>() >> 4 : 0);
#pragma unroll
        for (int kk = 0; kk < kBlock / 16; ++kk)
          instruction(d, aq + kk * a_step, bq + kk * b_step, (kk | q) ? 1u : (first ? 0u : 1u));
      }
      release(&empty[slot]);
    };
    auto advance = [&]() {
      if (++slot == S) {
        slot = 0;
        phase ^= 1;
      }
    };
    for (int i = unit; ok && walk.find(p, i, t); i += units) {
      if (lane == 0 && leader) {
        const int blocks = (int)((t.k_len + kBlock - 1) / kBlock);   // none: the epilogue writes zeros
        const int rest = J::RAGGED ? (int)(t.k_len % kBlock) : 0;
        const int whole = blocks - (rest ? 1 : 0);
        if constexpr (J::VARIABLE) idesc = fixed | (uint32_t)(t.n >> 3) << 17;
        // accumulator by accumulator: all blocks, or PASS at a time
        int kb = 0;
        while (kb < blocks) {
          const int stop = J::PASS ? min(blocks, kb + J::PASS) : blocks;
          const int buf = done & 1;
          if (!(ok = wait(&acc_empty[buf], ((done >> 1) & 1) ^ 1))) break;
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(buf * NT);
          bool first = true;
          for (const int to = min(stop, whole); kb < to; ++kb) {
            if (!(ok = wait(&full[slot], phase))) break;
            multiply(d, first);
            first = false;
            advance();
          }
          // a block that ends the range: the instructions that hold some of it.  Apart
          // from the loop above, whose instructions have to come without a pause (with
          // a test in it 8192^3 took 1084 us, without 715)
          if (J::RAGGED && ok && kb < stop) {
            ok = wait(&full[slot], phase);
            if (ok) {
              for (int kk = 0; kk * 16 < rest; ++kk)
                instruction(d, a_desc + slot * (SB >> 4) + kk * a_step, b_desc + slot * (SB >> 4) + kk * b_step,
                            kk ? 1u : (first ? 0u : 1u));
              release(&empty[slot]);
              advance();
              ++kb;
            }
          }
          if (!ok) break;
          release(&acc_full[buf]);
          ++done;
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
    }
    if (lane == 0 && leader) {
      if constexpr (PAIR == 2) tc_commit_pair(smem_u32(drain));
      else tc_commit(drain);
      mbar_settle(drain, 0, abort_flag, DEV_TIMEOUT_MMA);
    }
  } else if (J::RAGGED && warp == 2 + kEpilogueWarps) {
    // ------------------------------------------------------------ clearing
    typename J::Walk walk(p);
    Tile t;
    uint32_t it = 0, turn = 0;                        // parity of each slot's tail barriers
    bool ok = true;
    for (int i = unit; ok && walk.find(p, i, t); i += units) {
      const int blocks = (int)((t.k_len + kBlock - 1) / kBlock), rest = (int)(t.k_len % kBlock);
      it += blocks;
      if (rest == 0) continue;
      const uint32_t slot = (it - 1) % S, parity = (turn >> slot) & 1;
      turn ^= 1u << slot;
      unsigned char *st = smem + slot * SB;
      ok = mbar_wait_bounded(&tail[slot], parity, abort_flag, DEV_TIMEOUT_PRODUCER);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      // rows [rest, up to a multiple of 16) of every chunk: whole 128-byte lines, so
      // the swizzle does not matter
      constexpr int chunks = SB / (kBlock * kLine);
      const int pieces = ((rest + 15) / 16 * 16 - rest) * 8;  // 16-byte pieces of a chunk's lines
      for (int c = 0; c < chunks; ++c)
        for (int v = lane; v < pieces; v += 32)
          *reinterpret_cast<uint4 *>(st + c * (kBlock * kLine) + rest * kLine + v * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (leader) {
          if constexpr (PAIR == 2) ok = wait_cluster(&peer_tail[slot], parity, abort_flag, DEV_TIMEOUT_PRODUCER);
          if (ok) mbar_arrive(&full[slot]);
        } else {
          mbar_arrive_remote(leader_addr(&peer_tail[slot]));
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    constexpr int CW = warp_columns<J>();
    const int sub = warp & 3, part = (warp - 2) >> 2;
    unsigned char *mine = staging + (warp - 2) * kStagingBytes;
    const uint32_t columns = tmem + ((uint32_t)(sub * 32) << 16) + (uint32_t)(part * CW);
    typename J::Walk walk(p);
    Tile t;
    uint32_t done = 0;
    auto acquire = [&]() {
      const bool ok = mbar_wait_bounded(&acc_full[done & 1], (done >> 1) & 1, abort_flag,
                                        DEV_TIMEOUT_EPILOGUE);
      if (!__all_sync(0xffffffffu, ok)) return false;
      tc_fence_after();
      return true;
    };
    auto hand_back = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader) mbar_arrive(&acc_empty[done & 1]);
        else arrive_at_leader(leader_addr(&acc_empty[done & 1]));
      }
      ++done;
    };
    for (int i = unit; walk.find(p, i, t); i += units) {
      const int row = (int)rank * kRows + sub * 32, column = part * CW;
      typename J::Ahead early;                        // what the epilogue reads besides the accumulators
      J::look_ahead(p, t, row, column, early);
      if constexpr (J::PASS > 0) {
        float sum[CW];
#pragma unroll
        for (int c = 0; c < CW; ++c) sum[c] = 0.f;
        const int blocks = (int)((t.k_len + kBlock - 1) / kBlock);
        bool ok = true;
        for (int kb = 0; ok && kb < blocks; kb += J::PASS) {
          if (!(ok = acquire())) break;
#pragma unroll
          for (int c = 0; c < CW; c += 16) {
            uint32_t r[16];
            tmem_ld16_at(columns + (uint32_t)((done & 1) * NT + c), r);
            tmem_ld_wait16(r);
#pragma unroll
            for (int x = 0; x < 16; ++x) sum[c + x] += __uint_as_float(r[x]);
          }
          hand_back();
        }
        if (!ok) break;
        J::epilogue(p, t, Registers<CW>{sum}, row, column, mine, early);
      } else {
        const bool some = t.k_len > 0;
        if (some && !acquire()) break;
        J::epilogue(p, t, Columns{some, columns + (uint32_t)((done & 1) * NT)}, row, column, mine, early);
        if (some) hand_back();
      }
    }
    J::finish(p, (blockIdx.x * kEpilogueWarps + warp - 2), gridDim.x * kEpilogueWarps);
  }

  tc_fence_before();
  if constexpr (PAIR == 2) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR == 2) tmem_dealloc_pair(tmem, kTmemColumns);
    else tmem_dealloc(tmem, kTmemColumns);
  }
}

template <class J>
int launch(const CUtensorMap &a, const CUtensorMap &b, const typename J::Params &p, int64_t tiles,
           cudaStream_t st, const char *what) {
  auto kernel = tile_kernel<J>;
  constexpr int smem = smem_bytes<J>();
  static_assert(smem <= kSmemLimit, "shared memory");
  if (int rc = set_smem_once((const void *)kernel, smem, what)) return rc;
  const int64_t most = sm_count() / J::PAIR;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((tiles < most ? tiles : most) * J::PAIR));
  cfg.blockDim = dim3(threads<J>());
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = J::PAIR;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  count_launch();
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, a, b, p), what);
}

// ---------------------------------------------------------------------------
// epilogue pieces
// ---------------------------------------------------------------------------
template <typename O> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// The 16-byte piece u of row r in a warp's staging (32 rows of 64 bytes,
// pieces swizzled so that neither row-wise nor piece-wise access conflicts).
__device__ __forceinline__ uint4 *staged(unsigned char *mine, int r, int u) {
  return reinterpret_cast<uint4 *>(mine + r * 64 + ((u ^ ((r >> 1) & 3)) << 4));
}

// Rounds the warp's 32 x COLS accumulators to O and writes the first `rows`
// rows and `cols` columns of them to out (row pitch ld): every lane rounds
// its row into the staging, then 4 lanes write 64 consecutive bytes of a row.
template <typename O, int COLS, class Source>
__device__ __forceinline__ void write_rows(const Source &source, unsigned char *mine, O *out, int64_t ld,
                                           int rows, int64_t cols, bool vectors) {
  constexpr int ES = (int)sizeof(O), CH = 64 / ES;        // columns staged at a time
  const int lane = threadIdx.x % 32;
  O *to = out + (lane / 4) * ld + (lane % 4) * (16 / ES);
  const bool whole = vectors && rows >= 32;
#pragma unroll
  for (int c0 = 0; c0 < COLS; c0 += CH) {
    if (c0 >= cols || rows <= 0) continue;
#pragma unroll
    for (int c = 0; c < CH; c += 16) {
      float v[16];
      source.read(c0 + c, v);
      if constexpr (ES == 4) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          *staged(mine, lane, u) = *reinterpret_cast<uint4 *>(&v[u * 4]);
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u)
          *staged(mine, lane, c / 8 + u) =
              make_uint4(pack2<O>(v[u * 8], v[u * 8 + 1]), pack2<O>(v[u * 8 + 2], v[u * 8 + 3]),
                         pack2<O>(v[u * 8 + 4], v[u * 8 + 5]), pack2<O>(v[u * 8 + 6], v[u * 8 + 7]));
      }
    }
    __syncwarp();
    if (whole && c0 + CH <= cols) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4 *>(to + c0 + i * 8 * ld) = *staged(mine, i * 8 + lane / 4, lane % 4);
    } else if (vectors && c0 + CH <= cols) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i * 8 + lane / 4 < rows)
          *reinterpret_cast<uint4 *>(to + c0 + i * 8 * ld) = *staged(mine, i * 8 + lane / 4, lane % 4);
    } else {
      // rows off the 16-byte boundaries: element by element (pairs from 4-byte
      // boundary to 4-byte boundary took 30 us where this takes 23)
#pragma unroll 8
      for (int r = lane / CH; r < 32; r += 32 / CH)
        if (r < rows && c0 + lane % CH < cols)
          out[r * ld + c0 + lane % CH] =
              reinterpret_cast<const O *>(staged(mine, r, lane % CH * ES / 16))[lane % CH % (16 / ES)];
    }
    __syncwarp();
  }
}

// The same where the lanes hold columns of the output and the accumulator
// columns are its rows: `rows` of them from out on, 32 columns wide.
template <typename O, int COLS, class Source>
__device__ __forceinline__ void write_columns(const Source &source, unsigned char *mine, O *out, int64_t ld,
                                              int rows, int64_t cols, bool vectors) {
  constexpr int ES = (int)sizeof(O), RH = 64 / ES;        // rows staged at a time, 32 ES bytes each
  constexpr int PIECES = 32 * ES / 16, PER = 32 / PIECES;
  const int lane = threadIdx.x % 32;
  O *to = out + (int64_t)(lane / PIECES) * ld + lane % PIECES * (16 / ES);
  // 16-byte piece u of row r: shifted by the row, so that a row's write and the
  // pieces' reads touch every bank once
  auto piece = [&](int r, int u) {
    return reinterpret_cast<uint4 *>(mine + r * (32 * ES) + ((ES == 2 ? u ^ (r >> 1 & 3) : u ^ (r & 7)) << 4));
  };
#pragma unroll
  for (int r0 = 0; r0 < COLS; r0 += RH) {
    if (r0 >= rows || cols <= 0) continue;
#pragma unroll
    for (int c = 0; c < RH; c += 16) {
      float v[16];
      source.read(r0 + c, v);
#pragma unroll
      for (int x = 0; x < 16; ++x)
        reinterpret_cast<O *>(piece(c + x, lane * ES / 16))[lane % (16 / ES)] = O(v[x]);
    }
    __syncwarp();
    if (vectors && cols >= 32) {
#pragma unroll
      for (int i = 0; i < RH; i += PER)
        if (r0 + i + lane / PIECES < rows)
          *reinterpret_cast<uint4 *>(to + (r0 + i) * ld) = *piece(i + lane / PIECES, lane % PIECES);
    } else {
#pragma unroll 8
      for (int r = 0; r < RH; ++r)
        if (r0 + r < rows && lane < cols)
          out[(r0 + r) * ld + lane] = reinterpret_cast<const O *>(piece(r, lane * ES / 16))[lane % (16 / ES)];
    }
    __syncwarp();
  }
}

// fp16 operands (0) or bf16 (1), fp32 accumulator.
inline uint32_t instruction(int dtype) {
  const uint32_t f = dtype == OZ_BF16 ? 1 : 0;
  return 1u << 4 | f << 7 | f << 10;
}

}  // namespace tile
}  // namespace oz
