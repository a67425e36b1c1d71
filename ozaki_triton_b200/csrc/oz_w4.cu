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
//
// 8 rows, 28672 x 8192, groups of 128: 46.7 us (123 MB: 2.6 TB/s); 24 rows over 64
// experts of 2816 x 2048: 31 us; one row, 2048 x 2048: 5.4 us on the device, 11 a call.
// The warps' own instructions bound it, 690 a chunk of 64 x 128 weights (four warps a
// scheduler do not cover their latencies) and the last round of tiles.  Two blocks an SM
// leave 128 registers: with 64 weight rows, groups of 64 spill 32 (fp16) and 44 bytes
// (bf16), groups of 128 spill 4 (fp16).  Many rows are not what it is for: 4096 x 11008, 64
// rows 47 us, 512 291, 2048 934 (each 32 of them unpack the weights again).

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
  uint32_t per_group;                  // 2^32 / (group / 32), rounded up
  int column_tiles;
};

// Rows of expert e, clamped to the tensor; without offsets every row.
__device__ __forceinline__ void expert_rows(const W4Params &p, int e, int &begin, int &end) {
  if (!p.offsets) {
    begin = 0;
    end = p.rows;
    return;
  }
  auto at = [&](int i) {
    return p.wide ? (int64_t)*(static_cast<const long long *>(p.offsets) + i)
                  : (int64_t)*(static_cast<const int *>(p.offsets) + i);
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

// Four pairs of 16-bit values q - z from a word's eight fields (bits 0-3 and
// 16-19 first), exactly: a field becomes the low mantissa bits of a constant
// that is a power of two, and the same constant plus z is subtracted.  fp16
// has room for a field in bits 4-7 too (64 + q beside 1024 + q), bf16 has not.
// z is any byte.  fp16 holds 1024 + z and 64 + z exactly.  bf16 holds whole numbers up to
// 256, and 128 + z is more from 129 on: there the fields are flipped in the mantissa of
// -255, which makes q - 255, and z - 255 is subtracted (24 rows / 64 experts, 2816 x 2048:
// 30.9 us; 128 + q below z = 128 and q - 255 above 31.6).
// A constant that stays in a register (as an immediate it is moved there again at
// each use, and a mask and an or with two immediates become two instructions).
__device__ __forceinline__ uint32_t kept(uint32_t c) {
  uint32_t v;
  asm volatile("mov.b32 %0, %1;" : "=r"(v) : "r"(c));
  return v;
}
// (w & m) ^ c
__device__ __forceinline__ uint32_t field(uint32_t w, uint32_t m, uint32_t c) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(v) : "r"(w), "r"(m), "r"(c));
  return v;
}
template <typename T> struct Unpack;
template <> struct Unpack<__half> {
  uint32_t m0 = kept(0x000f000fu), c0 = kept(0x64006400u), m1 = kept(0x00f000f0u), c1 = kept(0x54005400u);
  static __device__ __forceinline__ uint32_t zero(uint32_t z) { return 0x64006400u | z * 0x10001u; }
  // 1024 + z and 64 + z
  __device__ __forceinline__ uint2 both(uint32_t z) const { return make_uint2(z, less(z, 0x63806380u)); }
  static __device__ __forceinline__ uint32_t less(uint32_t v, uint32_t z) {
    const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&v), *reinterpret_cast<const __half2 *>(&z));
    return *reinterpret_cast<const uint32_t *>(&d);
  }
  __device__ __forceinline__ void values(uint32_t w, uint2 z, uint32_t (&v)[4]) const {
    v[0] = less(field(w, m0, c0), z.x);
    v[1] = less(field(w, m1, c1), z.y);
    w >>= 8;
    v[2] = less(field(w, m0, c0), z.x);
    v[3] = less(field(w, m1, c1), z.y);
  }
};
template <> struct Unpack<__nv_bfloat16> {
  uint32_t m0 = kept(0x000f000fu), c0 = kept(0xc37fc37fu);
  // z - 255
  static __device__ __forceinline__ uint32_t zero(uint32_t z) {
    return (__float_as_uint((float)((int)z - 255)) >> 16) * 0x10001u;
  }
  __device__ __forceinline__ uint2 both(uint32_t z) const { return make_uint2(z, 0); }
  __device__ __forceinline__ void values(uint32_t w, uint2 z, uint32_t (&v)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = field(w >> (4 * i), m0, c0);
      const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&u),
                                       *reinterpret_cast<const __nv_bfloat162 *>(&z.x));
      v[i] = *reinterpret_cast<const uint32_t *>(&d);
    }
  }
};

// d = c + a b, 16 weight rows x 16 k by 8 rows of x
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1, float c0, float c1, float c2, float c3) {
  if constexpr (__is_same(T, __half))
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                 "{%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                 "{%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

__device__ __forceinline__ void put(const W4Params &p, int64_t i, float v) {
  if (p.out_dtype == OZ_F32) static_cast<float *>(p.y)[i] = v;
  else if (p.out_dtype == OZ_F16) static_cast<__half *>(p.y)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(p.y)[i] = __float2bfloat16_rn(v);
}

template <int RT, int NB, int PER> struct W4Shape {
  static constexpr int kRows = 16 * RT;                    // weight rows of a tile
  static constexpr int kWeights = kRows * kChunk / 2;      // bytes of a chunk
  static constexpr int kX = 8 * NB * kChunk * 2;
  static constexpr int kStage = kWeights + kX;
  static constexpr int kEntries = kRows * PER;             // scales of a chunk
  static constexpr int kSumRows = kRows < 32 ? kRows : 32; // summed over the warps at a time
  static constexpr int kSums = kSumRows * 8 * NB * 4;      // of a warp
  static constexpr int kWarpBytes = kDepth * kStage + kEntries * 8 + kSums;
  static constexpr int kBytes = 512 + kWarps * kWarpBytes + kWarps * kDepth * 8 + 16;
  static constexpr int kCtas = 2 * (kBytes + 1024) <= 228 * 1024 ? 2 : 1;
};

// RT: 16-row blocks of weights of a tile; NB: 8-row blocks of x.
// PER: scales of a chunk and row: 1 where a group covers whole chunks (g a
// multiple of 128), 2 where g is a multiple of 64, otherwise one for every 32 k.
template <typename T, int RT, int NB, int PER>
__global__ void __launch_bounds__(kWarps * 32, (W4Shape<RT, NB, PER>::kCtas))
    w4_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
              const W4Params p) {
  using Shape = W4Shape<RT, NB, PER>;
  static_assert(kDepth == 2, "the scales of a chunk are loaded two chunks ahead");
  extern __shared__ unsigned char raw[];
  unsigned char *smem = raw + ((512 - (smem_u32(raw) & 511)) & 511);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  unsigned char *ring = smem + warp * kDepth * Shape::kStage;
  // of the chunk in hand: scale and zero of each row and group
  uint2 *entries = reinterpret_cast<uint2 *>(smem + kWarps * kDepth * Shape::kStage) + warp * Shape::kEntries;
  float *sums = reinterpret_cast<float *>(smem + kWarps * (kDepth * Shape::kStage + Shape::kEntries * 8));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kWarps * Shape::kWarpBytes);
  uint64_t *full = bars + warp * kDepth;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + kWarps * kDepth);
  if (threadIdx.x == 0) *abort_flag = 0;
  if (lane == 0)
    for (int i = 0; i < kDepth; ++i) mbar_init(&full[i], 1);
  fence_mbar_init();
  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
  }
  __syncthreads();
  // what follows reads by plain loads alone: read-only ones may find what stood there before
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int team = warp / p.along, member = warp % p.along, teams = kWarps / p.along;
  const int unit = blockIdx.x * teams + team, units = gridDim.x * teams;
  const int chunks = (p.k + kChunk - 1) / kChunk;

  // This warp's chunks of this team's tiles, in order; what is copied runs two
  // chunks ahead of what is multiplied.  A chunk's scales and zeros are loaded
  // into registers with its copy and put into shared memory, ready for use, a
  // chunk later (when the chunk before it has been multiplied).
  constexpr int kMine = (Shape::kEntries + 31) / 32;
  W4Walk ahead;
  int a_tile = unit, a_chunk = member, a_e = 0, a_row = 0, a_rows = 0, a_column = 0;
  bool a_more = ahead.find(p, 8 * NB, a_tile, a_e, a_row, a_rows, a_column);
  uint32_t issued = 0;
  uint32_t scale_bits[kMine], zero_bits[kMine];
  // where the scales and zeros of this lane's entries start (kNowhere: no such row)
  constexpr int64_t kNowhere = INT64_MIN;
  int64_t entry_at[kMine];
  const int scale_bytes = p.scale_dtype == OZ_F32 ? 4 : 2;
  auto enter = [&]() {                                    // the tile that is copied next
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int r = (i * 32 + lane) % Shape::kRows, n = a_column * Shape::kRows + r;
      const bool in = n < p.n && (Shape::kEntries >= 32 || lane < Shape::kEntries);
      entry_at[i] = in ? a_e * p.s_se + n * p.s_sn : kNowhere;
    }
  };
  if (a_more) enter();
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    scale_bits[i] = 0;
    zero_bits[i] = 8;
  }
  auto issue = [&]() {
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const uint32_t bits = scale_bits[i];
      const float f = p.scale_dtype == OZ_F32 ? __uint_as_float(bits)
                      : p.scale_dtype == OZ_BF16 ? __uint_as_float(bits << 16)
                                                 : __half2float(__ushort_as_half((unsigned short)bits));
      if (Shape::kEntries >= 32 || lane < Shape::kEntries) {
        entries[i * 32 + lane] = make_uint2(__float_as_uint(f), Unpack<T>::zero(zero_bits[i]));
      }
    }
    while (a_more && a_chunk >= chunks) {
      a_tile += units;
      a_chunk = member;
      a_more = ahead.find(p, 8 * NB, a_tile, a_e, a_row, a_rows, a_column);
      if (a_more) enter();
    }
    if (a_more) {
      if (lane == 0) {
        unsigned char *st = ring + (issued & 1) * Shape::kStage;
        uint64_t *bar = &full[issued & 1];
        mbar_arrive_expect_tx(bar, Shape::kStage);
        tma_load_3d(st, &tm_w, bar, a_chunk * (kChunk / 2), a_column * Shape::kRows, a_e);
        tma_load_3d(st + Shape::kWeights, &tm_x, bar, 0, a_row, a_chunk * (kChunk / 32));
      }
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const uint32_t k32 = (uint32_t)(a_chunk * (kChunk / 32) + (i * 32 + lane) / Shape::kRows * (4 / PER));
        const uint32_t group = p.group == kChunk ? k32 / 4 : p.group == 32 ? k32 : __umulhi(k32, p.per_group);
        if (entry_at[i] != kNowhere && (int)group < p.groups) {
          const int64_t at = entry_at[i] + group;
          scale_bits[i] = scale_bytes == 4 ? *(static_cast<const uint32_t *>(p.scales) + at)
                                           : *(static_cast<const unsigned short *>(p.scales) + at);
          if (p.zeros) zero_bits[i] = *(p.zeros + at);
        } else {
          scale_bits[i] = 0;                              // nothing there: adds nothing
        }
      }
      a_chunk += p.along;
      ++issued;
    }
    __syncwarp();
  };
  issue();
  issue();

  // the lane's word of the 32-k piece i of a row, and its 8 k of x
  uint32_t piece[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) piece[i] = g * 64 + ((i ^ ((g >> 1) & 3)) << 4) + t * 4;
  const uint32_t x_at = Shape::kWeights + g * 64 + t * 16;

  const Unpack<T> unpack;
  W4Walk walk;
  uint32_t used = 0;
  // Once a wait has given up a warp multiplies nothing more but goes through all its
  // tiles: the other warps of its team wait for it at each tile's barriers.
  bool ok = true;
  for (int tile = unit;; tile += units) {
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
    for (int chunk = member; ok && chunk < chunks; chunk += p.along) {
      const unsigned char *st = ring + (used & 1) * Shape::kStage;
      ok = mbar_wait_bounded(&full[used & 1], used >> 1 & 1, abort_flag, DEV_TIMEOUT_PRODUCER);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      float part[RT][NB][4];
      uint2 zero[RT][2];
      float scale[RT][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {                       // 32 k at a time
        if (i % (4 / PER) == 0) {
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int entry = i / (4 / PER) * Shape::kRows + r * 16 + h * 8 + g;
              const uint2 v = entries[entry];
              scale[r][h] = __uint_as_float(v.x);
              zero[r][h] = unpack.both(v.y);
            }
        }
        // x: row g of each block of 8, the lane's 8 k, as the pairs (0 4) (1 5) (2 6) (3 7)
        uint32_t x[NB][4];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint4 v = *reinterpret_cast<const uint4 *>(st + x_at + i * (NB * 512) + b * 512);
          x[b][0] = __byte_perm(v.x, v.z, 0x5410);
          x[b][1] = __byte_perm(v.x, v.z, 0x7632);
          x[b][2] = __byte_perm(v.y, v.w, 0x5410);
          x[b][3] = __byte_perm(v.y, v.w, 0x7632);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          uint32_t w[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            unpack.values(*reinterpret_cast<const uint32_t *>(st + piece[i] + (r * 16 + h * 8) * 64), zero[r][h],
                              w[h]);
          }
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            float(&d)[4] = part[r][b];
            if (i % (4 / PER) == 0)
              mma<T>(d, w[0][0], w[1][0], w[0][1], w[1][1], x[b][0], x[b][1], 0.f, 0.f, 0.f, 0.f);
            else
              mma<T>(d, w[0][0], w[1][0], w[0][1], w[1][1], x[b][0], x[b][1], d[0], d[1], d[2], d[3]);
            mma<T>(d, w[0][2], w[1][2], w[0][3], w[1][3], x[b][2], x[b][3], d[0], d[1], d[2], d[3]);
          }
        }
        if ((i + 1) % (4 / PER) == 0) {
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
    // the team's sums, 32 weight rows (by rows of x) at a time, in the order of the warps
    float *own = sums + warp * (Shape::kSums / 4);
    const float *all = sums + team * p.along * (Shape::kSums / 4);
    constexpr int kSumRows = Shape::kSumRows;
#pragma unroll
    for (int r0 = 0; r0 < RT; r0 += kSumRows / 16) {
#pragma unroll
      for (int r = r0; r < r0 + kSumRows / 16; ++r)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            own[(b * 8 + t * 2 + (c & 1)) * kSumRows + (r - r0) * 16 + (c >> 1) * 8 + g] = acc[r][b][c];
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(p.along * 32) : "memory");
      for (int v = member * 32 + lane; v < rows * kSumRows; v += p.along * 32) {
        float sum = 0.f;
        for (int w = 0; w < p.along; ++w) sum += all[w * (Shape::kSums / 4) + v];
        const int n = n0 + r0 * 16 + v % kSumRows;
        if (n < p.n) put(p, (row + v / kSumRows) * p.ldy + n, sum);
      }
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(p.along * 32) : "memory");
    }
  }
  // copies still in flight after a wait gave up
  if (lane == 0)
    for (; used < issued; ++used)
      mbar_settle(&full[used & 1], used >> 1 & 1, abort_flag, DEV_TIMEOUT_PRODUCER);

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

template <typename T, int RT, int NB, int PER>
int run_shape(const void *packed, const void *x, W4Params p, int dtype, int64_t x_sr, int64_t p_se, int64_t p_sn,
              cudaStream_t st) {
  using Shape = W4Shape<RT, NB, PER>;
  CUtensorMap tw, tx;
  if (int rc = make_maps(&tw, &tx, packed, x, p, dtype, x_sr, p_se, p_sn, Shape::kRows, 8 * NB)) return rc;
  p.column_tiles = (p.n + Shape::kRows - 1) / Shape::kRows;
  const int64_t blocks = p.rows / (8 * NB) + min(p.experts, p.rows);
  const int64_t tiles = blocks * p.column_tiles;
  if (tiles > INT32_MAX / 2) return set_error(OZ_ERR_INVALID, "too many tiles");
  const int teams = kWarps / p.along;
  const int64_t most = Shape::kCtas * (int64_t)tile::sm_count();
  const int64_t need = (tiles + teams - 1) / teams;
  auto kernel = w4_kernel<T, RT, NB, PER>;
  static_assert(Shape::kBytes <= 227 * 1024, "shared memory");
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

template <typename T, int RT, int NB>
int run(const void *packed, const void *x, const W4Params &p, int dtype, int64_t x_sr, int64_t p_se, int64_t p_sn,
        cudaStream_t st) {
  return p.group % 128 == 0  ? run_shape<T, RT, NB, 1>(packed, x, p, dtype, x_sr, p_se, p_sn, st)
         : p.group % 64 == 0 ? run_shape<T, RT, NB, 2>(packed, x, p, dtype, x_sr, p_se, p_sn, st)
                             : run_shape<T, RT, NB, 4>(packed, x, p, dtype, x_sr, p_se, p_sn, st);
}

template <typename T>
int choose(const void *packed, const void *x, W4Params p, int dtype, int64_t x_sr, int64_t p_se,
           int64_t p_sn, cudaStream_t st) {
  // Rows of x a tile: as many as the mean group has (more would be read for
  // nothing).  Weight rows and warps a tile: the least estimated time, rounds of
  // tiles over the GPU times a warp's chunks of a tile and half a one for the
  // tile itself; a chunk of 16 weight rows takes 0.58 of one of 64 (instructions
  // counted: 411 and 714).  9 rows / 64 experts, 1088 x 15288, 9 chunks: 8 warps a
  // tile 61 us, 1 warp 37 us; 30 rows, 3520 x 11715: 8 warps 27 us, 2 warps 38 us.
  const int64_t mean = (p.rows + p.experts - 1) / p.experts, used = min(p.experts, p.rows);
  const int wide = mean > 16 ? 4 : mean > 8 ? 2 : 1;
  const int64_t chunks = (p.k + kChunk - 1) / kChunk;
  const int per = p.group % 128 == 0 ? 1 : p.group % 64 == 0 ? 2 : 4;
  auto time = [&](int rt, int nb, int ctas, int along) {
    const int64_t tiles = used * ((mean + 8 * nb - 1) / (8 * nb)) * ((p.n + 16 * rt - 1) / (16 * rt));
    const int64_t teams = (int64_t)tile::sm_count() * ctas * (kWarps / along);
    return (double)((tiles + teams - 1) / teams) * ((double)((chunks + along - 1) / along) + 0.5);
  };
  double best = 0;
  bool narrow = false;
  p.along = 0;
  for (int along = kWarps; along; along /= 2) {
    if (along > 1 && along > chunks) continue;
    const double t = wide == 1 ? time(4, 1, per == 4 ? 1 : 2, along) : time(wide == 2 ? 4 : 2, wide, 1, along);
    const double u = wide == 1 ? 0.58 * time(1, 1, 2, along) : t;
    if (!p.along || min(t, u) < 0.93 * best) {           // more warps a tile unless it pays
      best = min(t, u);
      narrow = u < t;
      p.along = along;
    }
  }
  if (wide == 4) return run<T, 2, 4>(packed, x, p, dtype, x_sr, p_se, p_sn, st);
  if (wide == 2) return run<T, 4, 2>(packed, x, p, dtype, x_sr, p_se, p_sn, st);
  return narrow ? run<T, 1, 1>(packed, x, p, dtype, x_sr, p_se, p_sn, st)
                : run<T, 4, 1>(packed, x, p, dtype, x_sr, p_se, p_sn, st);
}

}  // namespace
}  // namespace oz

extern "C" int oz_matmul_w4(const oz_w4_args *args, void *stream) {
  if (!args) return oz::set_error(OZ_ERR_INVALID, "null arguments");
  auto [x, packed, scales, zeros, offsets, y, rows, k, n, x_sr, p_se, p_sn, s_se, s_sn, ldy, experts, group,
        offsets_64, dtype, scale_dtype, out_dtype] = *args;
  using namespace oz;
  if (dtype != OZ_F16 && dtype != OZ_BF16)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported operand dtype %d (fp16 or bf16)", dtype);
  if (scale_dtype != OZ_F16 && scale_dtype != OZ_BF16 && scale_dtype != OZ_F32)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported scale dtype %d", scale_dtype);
  if (out_dtype != dtype && out_dtype != OZ_F32)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported output dtype %d", out_dtype);
  if (experts < 1) return set_error(OZ_ERR_INVALID, "at least one expert is needed, got %d", experts);
  if (rows < 0 || k < 0 || n < 0) return set_error(OZ_ERR_INVALID, "negative size");
  // (k / 32) (group / 32) < 2^32 keeps the kernel's division by a product exact
  if (rows > (1 << 30) || k > (1 << 20) || n > (1 << 30) || experts > (1 << 24))
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
  W4Params p{scales, offsets, static_cast<const uint8_t *>(zeros), y, offsets_64, experts, group,
             (int)(k / group), scale_dtype, out_dtype, (int)rows, (int)k, (int)n, ldy, s_se, s_sn,
             0,
             group == 32 ? 0 : (uint32_t)(((1ull << 32) + group / 32 - 1) / (group / 32)), 0};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == OZ_F16 ? choose<__half>(packed, x, p, dtype, x_sr, p_se, p_sn, st)
                         : choose<__nv_bfloat16>(packed, x, p, dtype, x_sr, p_se, p_sn, st);
}
