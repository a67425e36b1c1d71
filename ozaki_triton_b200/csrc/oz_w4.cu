// oz_w4.cu -- products of a few rows with 4-bit weights and group scales.
//
//   y[r, n] = sum_k x[r, k] (q[n, k] - z[n, k / g]) s[n, k / g]
//
// q: two values a byte along k, the even k in the low half; z is 8 where no
// zero points are given.  With offsets the rows come in groups, each with the
// weights of its own expert.
//
// The weights' bytes bound it, so they stream through shared memory (one
// bulk copy of 16 RT rows x 128 k at a time into a ring that each warp keeps
// for itself: no barrier between warps while they stream) and everything else
// is kept out of their way: q - z is an exact fp16 / bf16 integer, made with a
// mask and one subtraction a pair from the 4-bit fields, and mma.sync
// multiplies 16 weight rows by 8 rows of x with fp32 sums: the matrix unit
// only has to keep up with memory here (2 flops for each half byte and row),
// and its registers take the weights without another trip through shared
// memory.  The order of k inside a block of 8 follows the fields of a word
// (0 4, 1 5, 2 6, 3 7) on both sides.  A group's sum is scaled in fp32.
// The warps of a tile share k and are summed in shared memory in a fixed order.

#include "oz_tile.cuh"

namespace oz {
int status_w4(int *value, bool clear) { return read_status_word(value, clear); }

namespace {

constexpr int kWarps = 8;
constexpr int kDepth = 2;              // chunks of a warp's ring
constexpr int kChunk = 128;            // k of a chunk

struct W4Params {
  const void *scales, *offsets;
  const uint8_t *zeros;
  void *y;
  int wide, experts, group, groups, scale_dtype, out_dtype;
  int rows, k, n;
  int64_t ldy;
  int64_t s_se, s_sn;                  // scales (and zeros): expert and row strides, elements
  int along;                           // warps that share the k of a tile (1, 2, 4 or 8)
  int column_tiles;
};

__device__ __forceinline__ float load_scale(const void *s, int dtype, int64_t i) {
  if (dtype == OZ_F32) return __ldg(static_cast<const float *>(s) + i);
  if (dtype == OZ_F16) return __half2float(__ldg(static_cast<const __half *>(s) + i));
  return __bfloat162float(__ldg(static_cast<const __nv_bfloat16 *>(s) + i));
}

// Rows of expert e, clamped to the tensor; without offsets every row.
__device__ __forceinline__ void expert_rows(const W4Params &p, int e, int &begin, int &end) {
  if (!p.offsets) {
    begin = 0;
    end = p.rows;
    return;
  }
  auto at = [&](int i) {
    return p.wide ? (int64_t)__ldg(static_cast<const long long *>(p.offsets) + i)
                  : (int64_t)__ldg(static_cast<const int *>(p.offsets) + i);
  };
  begin = (int)min(max(at(e), (int64_t)0), (int64_t)p.rows);
  end = (int)min(max(at(e + 1), (int64_t)begin), (int64_t)p.rows);
}

// Tiles: expert by expert, `per` rows of x a block, every column tile of it.
// A warp holds the ranges of 32 experts, one a lane.
struct W4Walk {
  int first = -32, before = 0, begin = 0, end = 0, tiles = 0, upto = 0;
  __device__ bool find(const W4Params &p, int per, int i, int &e, int &row, int &rows, int &column) {
    const int lane = threadIdx.x % 32;
    int total = __shfl_sync(0xffffffffu, upto, 31);
    while (first < 0 || i >= before + total) {
      before += total;
      first += 32;
      if (first >= p.experts) return false;
      begin = end = 0;
      if (first + lane < p.experts) expert_rows(p, first + lane, begin, end);
      tiles = (end - begin + per - 1) / per * p.column_tiles;
      upto = tiles;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      total = __shfl_sync(0xffffffffu, upto, 31);
    }
    const int src = __ffs(__ballot_sync(0xffffffffu, i < before + upto)) - 1;
    e = first + src;
    const int lo = __shfl_sync(0xffffffffu, begin, src), hi = __shfl_sync(0xffffffffu, end, src);
    const int local = i - before - __shfl_sync(0xffffffffu, upto - tiles, src);
    // blocks of the same columns one after the other: their weights are in L2
    const int blocks = (hi - lo + per - 1) / per;
    column = local / blocks;
    row = lo + local % blocks * per;
    rows = min(per, hi - row);
    return true;
  }
};

// Two 16-bit values q - z from bits [SHIFT, SHIFT + 4) of both halves of a
// word: as 1024 + q (fp16) or 128 + q (bf16), less the same with z.
template <typename T> struct Unpack;
template <> struct Unpack<__half> {
  static __device__ __forceinline__ uint32_t zero(int z) { return 0x64006400u | (uint32_t)(z * 0x10001); }
  static __device__ __forceinline__ uint32_t value(uint32_t w, uint32_t z) {
    const uint32_t v = (w & 0x000f000fu) | 0x64006400u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&v), *reinterpret_cast<const __half2 *>(&z));
    return *reinterpret_cast<const uint32_t *>(&d);
  }
};
template <> struct Unpack<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t zero(int z) { return 0x43004300u | (uint32_t)(z * 0x10001); }
  static __device__ __forceinline__ uint32_t value(uint32_t w, uint32_t z) {
    const uint32_t v = (w & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 d =
        __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), *reinterpret_cast<const __nv_bfloat162 *>(&z));
    return *reinterpret_cast<const uint32_t *>(&d);
  }
};

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __half))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                 "{%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                 "{%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void put(const W4Params &p, int64_t i, float v) {
  if (p.out_dtype == OZ_F32) static_cast<float *>(p.y)[i] = v;
  else if (p.out_dtype == OZ_F16) static_cast<__half *>(p.y)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(p.y)[i] = __float2bfloat16_rn(v);
}

template <int RT, int NB> struct W4Shape {
  static constexpr int kRows = 16 * RT;                    // weight rows of a tile
  static constexpr int kWeights = kRows * kChunk / 2;      // bytes of a chunk
  static constexpr int kX = 8 * NB * kChunk * 2;
  static constexpr int kStage = kWeights + kX;
  static constexpr int kSums = kRows * 8 * NB * 4;         // of a warp
  static constexpr int kBytes = 512 + kWarps * (kDepth * kStage + kSums) + kWarps * kDepth * 8 + 16;
};

// RT: 16-row blocks of weights of a tile; NB: 8-row blocks of x.
// WHOLE: a group covers whole chunks (g a multiple of 128), one scale a chunk.
template <typename T, int RT, int NB, bool WHOLE>
__global__ void __launch_bounds__(kWarps * 32, RT * NB >= 8 ? 1 : 2)
    w4_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
              const W4Params p) {
  using Shape = W4Shape<RT, NB>;
  extern __shared__ unsigned char raw[];
  unsigned char *smem = raw + ((512 - (smem_u32(raw) & 511)) & 511);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  unsigned char *ring = smem + warp * kDepth * Shape::kStage;
  float *sums = reinterpret_cast<float *>(smem + kWarps * kDepth * Shape::kStage);
  uint64_t *full = reinterpret_cast<uint64_t *>(sums + kWarps * Shape::kSums / 4) + warp * kDepth;
  volatile int *abort_flag =
      reinterpret_cast<volatile int *>(reinterpret_cast<uint64_t *>(sums + kWarps * Shape::kSums / 4) +
                                       kWarps * kDepth);
  if (threadIdx.x == 0) *abort_flag = 0;
  if (lane == 0)
    for (int i = 0; i < kDepth; ++i) mbar_init(&full[i], 1);
  fence_mbar_init();
  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
  }
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int team = warp / p.along, member = warp % p.along, teams = kWarps / p.along;
  const int unit = blockIdx.x * teams + team, units = gridDim.x * teams;
  const int chunks = (p.k + kChunk - 1) / kChunk;

  // this warp's chunks of this team's tiles, in order: what is copied (ahead)
  // and what is multiplied walk the same sequence
  W4Walk ahead;
  int a_tile = unit, a_chunk = member, a_e = 0, a_row = 0, a_rows = 0, a_column = 0;
  bool a_more = ahead.find(p, 8 * NB, a_tile, a_e, a_row, a_rows, a_column);
  uint32_t issued = 0;
  auto issue = [&]() {
    while (a_more && a_chunk >= chunks) {
      a_tile += units;
      a_chunk = member;
      a_more = ahead.find(p, 8 * NB, a_tile, a_e, a_row, a_rows, a_column);
    }
    if (!a_more) return;
    if (lane == 0) {
      unsigned char *st = ring + issued % kDepth * Shape::kStage;
      uint64_t *bar = &full[issued % kDepth];
      mbar_arrive_expect_tx(bar, Shape::kStage);
      tma_load_3d(st, &tm_w, bar, a_chunk * (kChunk / 2), a_column * Shape::kRows, a_e);
      tma_load_3d(st + Shape::kWeights, &tm_x, bar, 0, a_row, a_chunk * (kChunk / 32));
    }
    a_chunk += p.along;
    ++issued;
  };
  if (member < chunks)
    for (int i = 0; i < kDepth; ++i) issue();

  W4Walk walk;
  uint32_t used = 0;
  bool ok = true;
  for (int tile = unit; ok; tile += units) {
    int e, row, rows, column;
    if (!walk.find(p, 8 * NB, tile, e, row, rows, column)) break;
    const int n0 = column * Shape::kRows;
    float acc[RT][NB][4];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][b][c] = 0.f;
    const int64_t s0 = e * p.s_se;
    for (int chunk = member; chunk < chunks; chunk += p.along) {
      float scale[RT][2];
      uint32_t zero[RT][2];
      auto load_group = [&](int k) {
        const int group = k / p.group;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int n = n0 + r * 16 + h * 8 + g;
            const bool in = n < p.n && group < p.groups;
            const int64_t at = s0 + n * p.s_sn + group;
            scale[r][h] = in ? load_scale(p.scales, p.scale_dtype, at) : 0.f;
            zero[r][h] = Unpack<T>::zero(in && p.zeros ? __ldg(p.zeros + at) : 8);
          }
      };
      if constexpr (WHOLE) load_group(chunk * kChunk);
      const unsigned char *st = ring + used % kDepth * Shape::kStage;
      ok = mbar_wait_bounded(&full[used % kDepth], used / kDepth & 1, abort_flag, DEV_TIMEOUT_PRODUCER);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      float part[RT][NB][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {                       // 32 k at a time
        if constexpr (!WHOLE) load_group(chunk * kChunk + i * 32);
        if (!WHOLE || i == 0) {
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int c = 0; c < 4; ++c) part[r][b][c] = 0.f;
        }
        // x: row g of each block of 8, the lane's 8 k, as the pairs (0 4) (1 5) (2 6) (3 7)
        uint32_t x[NB][4];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint4 v = *reinterpret_cast<const uint4 *>(st + Shape::kWeights + i * (NB * 512) + b * 512 +
                                                           g * 64 + t * 16);
          x[b][0] = __byte_perm(v.x, v.z, 0x5410);
          x[b][1] = __byte_perm(v.x, v.z, 0x7632);
          x[b][2] = __byte_perm(v.y, v.w, 0x5410);
          x[b][3] = __byte_perm(v.y, v.w, 0x7632);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          uint32_t w[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int rr = r * 16 + h * 8 + g;
            w[h] = *reinterpret_cast<const uint32_t *>(st + rr * 64 + ((i ^ ((rr >> 1) & 3)) << 4) + t * 4);
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t a[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              a[h] = Unpack<T>::value(w[h] >> (8 * half), zero[r][h]);
              a[2 + h] = Unpack<T>::value(w[h] >> (8 * half + 4), zero[r][h]);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) mma<T>(part[r][b], a, x[b][2 * half], x[b][2 * half + 1]);
          }
        }
        if (!WHOLE || i == 3) {
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int c = 0; c < 4; ++c) acc[r][b][c] += scale[r][c / 2] * part[r][b][c];
        }
      }
      __syncwarp();
      ++used;
      issue();                                            // into the slot just read
    }
    // the team's sums: rows of x by weight rows, summed in the order of the warps
    float *own = sums + warp * (Shape::kSums / 4);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          own[(b * 8 + t * 2 + (c & 1)) * Shape::kRows + r * 16 + (c >> 1) * 8 + g] = acc[r][b][c];
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(p.along * 32) : "memory");
    const float *all = sums + team * p.along * (Shape::kSums / 4);
    for (int v = member * 32 + lane; v < rows * Shape::kRows; v += p.along * 32) {
      float sum = 0.f;
      for (int w = 0; w < p.along; ++w) sum += all[w * (Shape::kSums / 4) + v];
      const int n = n0 + v % Shape::kRows;
      if (n < p.n) put(p, (row + v / Shape::kRows) * p.ldy + n, sum);
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(p.along * 32) : "memory");
    ok = !*abort_flag;
  }
  // copies still in flight after a wait gave up
  if (lane == 0)
    for (; used < issued; ++used)
      mbar_wait_bounded(&full[used % kDepth], used / kDepth & 1, abort_flag, DEV_TIMEOUT_PRODUCER);

  if (p.offsets) {                                        // rows that no group holds are zero
    int first, last, a, b;
    expert_rows(p, 0, first, a);
    expert_rows(p, p.experts - 1, b, last);
    for (int v = blockIdx.x * kWarps + warp; v < first + p.rows - last; v += gridDim.x * kWarps)
      for (int n = lane; n < p.n; n += 32) put(p, (v < first ? v : last + v - first) * p.ldy + n, 0.f);
  }
}

int make_maps(CUtensorMap *w, CUtensorMap *x, const void *packed, const void *xp, const W4Params &p, int dtype,
              int64_t x_sr, int64_t p_se, int64_t p_sn, int rows, int x_rows) {
  if (int rc = tile::encode(w, CU_TENSOR_MAP_DATA_TYPE_UINT8, packed, p.k / 2, p.n, p.experts, p_sn,
                            p.experts > 1 ? p_se : p_sn, kChunk / 2, rows, 1, CU_TENSOR_MAP_SWIZZLE_64B))
    return rc;
  // 32 k, rows, blocks of 32 k: a chunk lands as 4 blocks of x_rows rows of 64 bytes
  return tile::encode(x, CU_TENSOR_MAP_DATA_TYPE_UINT16, xp, 32, p.rows, p.k / 32, x_sr * 2, 64, 32, x_rows,
                      kChunk / 32, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <typename T, int RT, int NB>
int run(const void *packed, const void *x, W4Params p, int dtype, int64_t x_sr, int64_t p_se, int64_t p_sn,
        cudaStream_t st) {
  using Shape = W4Shape<RT, NB>;
  CUtensorMap tw, tx;
  if (int rc = make_maps(&tw, &tx, packed, x, p, dtype, x_sr, p_se, p_sn, Shape::kRows, 8 * NB)) return rc;
  p.column_tiles = (p.n + Shape::kRows - 1) / Shape::kRows;
  const int64_t blocks = p.rows / (8 * NB) + min(p.experts, p.rows);
  const int64_t tiles = blocks * p.column_tiles;
  if (tiles > INT32_MAX / 2) return set_error(OZ_ERR_INVALID, "too many tiles");
  const int teams = kWarps / p.along;
  const int64_t most = (RT * NB >= 8 ? 1 : 2) * (int64_t)tile::sm_count();
  const int64_t need = (tiles + teams - 1) / teams;
  auto kernel = p.group % kChunk == 0 ? w4_kernel<T, RT, NB, true> : w4_kernel<T, RT, NB, false>;
  if (int rc = set_smem_once((const void *)kernel, Shape::kBytes, "w4_kernel shared memory")) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(need < most ? need : most));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = Shape::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, tw, tx, p), "w4_kernel launch");
}

template <typename T>
int choose(const void *packed, const void *x, const W4Params &p, int dtype, int64_t x_sr, int64_t p_se,
           int64_t p_sn, cudaStream_t st) {
  // rows of x a tile: as many as the mean group has (more would be read for nothing)
  const int64_t mean = (p.rows + p.experts - 1) / p.experts;
  if (mean > 16) return run<T, 2, 4>(packed, x, p, dtype, x_sr, p_se, p_sn, st);
  if (mean > 8) return run<T, 4, 2>(packed, x, p, dtype, x_sr, p_se, p_sn, st);
  // 64 weight rows a tile share the reading of x; 16 where that would leave SMs idle
  const int64_t used = min(p.experts, p.rows);
  if (used * ((p.n + 63) / 64) * p.along >= 2 * kWarps * (int64_t)tile::sm_count())
    return run<T, 4, 1>(packed, x, p, dtype, x_sr, p_se, p_sn, st);
  return run<T, 1, 1>(packed, x, p, dtype, x_sr, p_se, p_sn, st);
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
  if (rows > (1 << 30) || k > (1 << 30) || n > (1 << 30) || experts > (1 << 24))
    return set_error(OZ_ERR_INVALID, "size out of range");
  if (k == 0 || group < 32 || group % 32 != 0 || k % group != 0)
    return set_error(OZ_ERR_INVALID, "the group size must be a multiple of 32 that divides k (group=%d k=%lld)",
                     group, (long long)k);
  if (rows == 0 || n == 0) return OZ_OK;
  if (!y || ldy < n)
    return set_error(OZ_ERR_INVALID, "bad output (ldy=%lld n=%lld)", (long long)ldy, (long long)n);
  if (!x || !packed || !scales) return set_error(OZ_ERR_INVALID, "null pointer");
  if (!offsets && experts != 1) return set_error(OZ_ERR_INVALID, "several experts need offsets");
  if (rows == 1) x_sr = (k + 7) / 8 * 8;
  if (n == 1) p_sn = k / 2;
  if (((uintptr_t)x | (uintptr_t)packed) % 16 != 0 || x_sr <= 0 || x_sr % 8 != 0 || p_sn <= 0 ||
      p_sn % 16 != 0 || (experts > 1 && (p_se <= 0 || p_se % 16 != 0)))
    return set_error(OZ_ERR_INVALID,
                     "x and packed must start on 16-byte boundaries with row pitches of multiples of 16 bytes");
  const int64_t chunks = (k + kChunk - 1) / kChunk;
  W4Params p{scales, offsets, static_cast<const uint8_t *>(zeros), y, offsets_64, experts, group,
             (int)(k / group), scale_dtype, out_dtype, (int)rows, (int)k, (int)n, ldy, s_se, s_sn,
             chunks >= 8 ? 8 : chunks >= 4 ? 4 : chunks >= 2 ? 2 : 1, 0};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == OZ_F16 ? choose<__half>(packed, x, p, dtype, x_sr, p_se, p_sn, st)
                         : choose<__nv_bfloat16>(packed, x, p, dtype, x_sr, p_se, p_sn, st);
}
