// oz_experts.cu -- ragged products of an expert layer and their gradients on
// the tile engine (oz_tile.cuh).
//
//   y[r]  = x[r] @ w[e]                     offsets[e] <= r < offsets[e + 1]
//   dx[r] = dy[r] @ w[e]^T                  (the same product with w transposed)
//   dw[e] = sum_r x[r]^T dy[r]              r over the group's rows
//
// The groups are runs of rows given by device offsets, so the number of tiles
// is not known on the host: the grid is sized for the most there can be and
// every role of every CTA walks the groups itself.  Offsets are clamped to
// [0, rows] before they are used as row numbers.  Products of fp16 / bf16
// values are exact in fp32; sums are held in fp32 and rounded once.

#include <cmath>

#include "oz_tile.cuh"

namespace oz {
int status_experts(int *value, bool clear) { return read_status_word(value, clear); }

namespace {
using namespace tile;

__device__ __forceinline__ int64_t load_offset(const void *offsets, int wide, int64_t i) {
  return wide ? __ldg(static_cast<const long long *>(offsets) + i)
              : (int64_t)__ldg(static_cast<const int *>(offsets) + i);
}

// Row range of group e, clamped so that a bad offset never leaves the tensor.
__device__ __forceinline__ void group_rows(const void *offsets, int wide, int e, int rows,
                                           int &begin, int &end) {
  begin = (int)min(max(load_offset(offsets, wide, e), (int64_t)0), (int64_t)rows);
  end = (int)min(max(load_offset(offsets, wide, e + 1), (int64_t)begin), (int64_t)rows);
}

struct GroupedParams {
  const void *offsets;
  void *out;
  int64_t ld;                  // output row pitch
  int wide, groups, rows, k, n;
  int column_tiles;
  int vectors;                 // output rows may be written 16 bytes at a time
  uint32_t idesc;
};

// Tiles of row blocks: group by group, `per_rows` rows a block, every column
// tile of a block.  A warp holds the ranges of 32 groups, one a lane.
struct GroupWalk {
  int first, before, begin, end, tiles, upto;   // first group of the 32; tiles before it
  __device__ GroupWalk(const GroupedParams &) : first(-32), before(0), tiles(0), upto(0) {}

  // The group, block and column tile of tile i; false past the last one.  Calls
  // have increasing i.  Blocks of `span` consecutive rows of tiles sweep all columns
  // together (their operands stay in L2).
  __device__ bool find(const GroupedParams &p, int per_rows, int span, int i, int &e, int &lo, int &hi,
                       int &block, int &column) {
    const int lane = threadIdx.x % 32;
    int total = __shfl_sync(0xffffffffu, upto, 31);
    while (first < 0 || i >= before + total) {
      before += total;
      first += 32;
      if (first >= p.groups) return false;
      begin = end = 0;
      if (first + lane < p.groups) group_rows(p.offsets, p.wide, first + lane, p.rows, begin, end);
      tiles = (end - begin + per_rows - 1) / per_rows * p.column_tiles;
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
    lo = __shfl_sync(0xffffffffu, begin, src);
    hi = __shfl_sync(0xffffffffu, end, src);
    const int local = i - before - __shfl_sync(0xffffffffu, upto - tiles, src);
    const int blocks = (hi - lo + per_rows - 1) / per_rows;
    const int sweep = local / (span * p.column_tiles);
    const int in = local - sweep * span * p.column_tiles;
    const int size = min(blocks - sweep * span, span);
    block = sweep * span + in % size;
    column = in / size;
    return true;
  }
};

// Zeros in the rows that no group holds, warp `me` of `warps`.
template <typename O>
__device__ __forceinline__ void clear_outside(const GroupedParams &p, int me, int warps) {
  int first, last, a, b;
  group_rows(p.offsets, p.wide, 0, p.rows, first, a);
  group_rows(p.offsets, p.wide, p.groups - 1, p.rows, b, last);
  for (int v = me; v < first + p.rows - last; v += warps) {
    O *row = static_cast<O *>(p.out) + (int64_t)(v < first ? v : last + v - first) * p.ld;
    for (int c = threadIdx.x % 32; c < p.n; c += 32) row[c] = O(0.f);
  }
}

struct RowTile { int row, rows, column; };   // first row, rows from there to the group's end

// y = x w: A is the rows of x, B the columns of w[e].  For groups of many rows:
// one of 8192 rows, 8192 x 8192, runs at the rate of the tensor cores under the
// power limit (715 us in short runs, 1540 TFLOP/s).
template <typename O, int PAIR_, int NT_, bool BMN_> struct RowsJob : NoLookAhead {
  static constexpr int PAIR = PAIR_, NT = NT_, PLANES = 1, PASS = sizeof(O) == 4 ? 8 : 0;
  static constexpr bool AMN = false, BMN = BMN_, RAGGED = false;
  using Params = GroupedParams;
  using Extra = RowTile;
  static __device__ int plane_stride(const Params &) { return 0; }
  struct Walk : GroupWalk {
    using GroupWalk::GroupWalk;
    __device__ bool find(const Params &p, int i, TileOf<Extra> &t) {
      int e, lo, hi, block, column;
      if (!GroupWalk::find(p, kRows * PAIR, 8, i, e, lo, hi, block, column)) return false;
      t.a_row = lo + block * kRows * PAIR;
      t.a_mat = 0;
      t.b_row = column * NT;
      t.b_mat = e;
      t.k_begin = 0;
      t.k_len = p.k;
      t.extra = RowTile{t.a_row, hi - t.a_row, t.b_row};
      return true;
    }
  };
  template <class Source>
  static __device__ void epilogue(const Params &p, const TileOf<Extra> &t, const Source &source, int row,
                                  int column, unsigned char *mine, Ahead &) {
    const int64_t c0 = t.extra.column + column;
    write_rows<O, NT / 2>(source, mine,
                          static_cast<O *>(p.out) + (int64_t)(t.extra.row + row) * p.ld + c0, p.ld,
                          t.extra.rows - row, p.n - c0, p.vectors);
  }
  static __device__ void finish(const Params &p, int me, int warps) { clear_outside<O>(p, me, warps); }
};

// The same product with the roles exchanged, for groups of a few rows: A is
// 128 columns of w[e], B up to NT rows of x, so a tile's weights are read
// once and hardly any of the staged bytes belong to rows that are not there.
// 16 rows over 8 experts, 1024 x 2048: 8 us on the device, 9.1 a call (30 MB of
// weights at 6.5 TB/s: 4.6), bound by the way from the launch to the first block.
template <typename O, int NT_, bool AMN_> struct ColumnsJob : NoLookAhead {
  static constexpr int PAIR = 1, NT = NT_, PLANES = 1, PASS = sizeof(O) == 4 ? 8 : 0;
  static constexpr bool AMN = AMN_, BMN = false, RAGGED = false;
  using Params = GroupedParams;
  using Extra = RowTile;
  static __device__ int plane_stride(const Params &) { return 0; }
  struct Walk : GroupWalk {
    using GroupWalk::GroupWalk;
    __device__ bool find(const Params &p, int i, TileOf<Extra> &t) {
      int e, lo, hi, block, column;
      if (!GroupWalk::find(p, NT, 1 << 16, i, e, lo, hi, block, column)) return false;
      t.a_row = column * kRows;
      t.a_mat = e;
      t.b_row = lo + block * NT;
      t.b_mat = 0;
      t.k_begin = 0;
      t.k_len = p.k;
      t.extra = RowTile{t.b_row, hi - t.b_row, t.a_row};
      return true;
    }
  };
  template <class Source>
  static __device__ void epilogue(const Params &p, const TileOf<Extra> &t, const Source &source, int row,
                                  int column, unsigned char *, Ahead &) {
    const int64_t c = t.extra.column + row + threadIdx.x % 32;
    O *out = static_cast<O *>(p.out) + (int64_t)(t.extra.row + column) * p.ld + c;
    const int rows = t.extra.rows - column;
#pragma unroll
    for (int r0 = 0; r0 < NT / 2; r0 += 16) {
      if (r0 >= rows) continue;
      float v[16];
      source.read(r0, v);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (r0 + r < rows && c < p.n) out[(r0 + r) * p.ld] = O(v[r]);
    }
  }
  static __device__ void finish(const Params &p, int me, int warps) { clear_outside<O>(p, me, warps); }
};

// The exchanged roles for pairs of CTAs: 256 columns of w[e] by up to 256 rows of
// x.  A group's rows are dealt out evenly to as few tiles as hold them, in multiples
// of 32: with rows as A every group ends in a tile of 256 rows whatever is left
// (32768 rows over 64 experts, 2048 x 2816, in short runs: 356 us, this 344; 8192 rows
// over 64, 2048 x 1408: 93 and 78).  Under lasting load the power limit makes the first
// 405 us.  Its epilogue turns the tile, which a short contraction does not hide.  With
// fp32 results the sums of the passes spill 28 bytes under 168 registers (15% slower: 369
// us where bf16 results take 320).
template <typename O, bool AMN_> struct PairsJob : NoLookAhead {
  static constexpr int PAIR = 2, NT = 256, PLANES = 1, PASS = sizeof(O) == 4 ? 8 : 0;
  static constexpr bool AMN = AMN_, BMN = false, RAGGED = false, VARIABLE = true;
  using Params = GroupedParams;
  using Extra = RowTile;
  static __device__ int plane_stride(const Params &) { return 0; }
  struct Walk : GroupWalk {
    using GroupWalk::GroupWalk;
    __device__ bool find(const Params &p, int i, TileOf<Extra> &t) {
      int e, lo, hi, block, column;
      if (!GroupWalk::find(p, NT, 8, i, e, lo, hi, block, column)) return false;
      const int blocks = (hi - lo + NT - 1) / NT, each = (hi - lo + blocks - 1) / blocks;
      t.n = (each + 31) / 32 * 32;
      t.a_row = column * 2 * kRows;
      t.a_mat = e;
      t.b_row = lo + block * t.n;
      t.b_mat = 0;
      t.k_begin = 0;
      t.k_len = p.k;
      t.extra = RowTile{t.b_row, min(t.n, hi - t.b_row), t.a_row};
      return true;
    }
  };
  template <class Source>
  static __device__ void epilogue(const Params &p, const TileOf<Extra> &t, const Source &source, int row,
                                  int column, unsigned char *mine, Ahead &) {
    const int64_t c = t.extra.column + row;
    write_columns<O, NT / 2>(source, mine, static_cast<O *>(p.out) + (int64_t)(t.extra.row + column) * p.ld + c, p.ld,
                             t.extra.rows - column, p.n - c, p.vectors);
  }
  static __device__ void finish(const Params &p, int me, int warps) { clear_outside<O>(p, me, warps); }
};

struct WeightTile { int row, column, group; };

// dw[e] = x^T dy over the group's rows: both operands are stored across the
// contraction, whose range is the group.  32768 rows over 16 groups, 4096 x 2048, with
// dx: 855 us (both are 1100 GFLOP: 1290 TFLOP/s; under lasting load the power limit makes
// it 1010; with bf16 results 826 where fp32 ones take 869), bound by the tensor cores; 3989
// rows over 16, 1024 x 1536, with dx: 63 us, bound by the 100 MB of fp32 results and by tiles
// of only 4 blocks.  The contraction is not divided: few tiles of many rows leave SMs idle
// (one group of 32768 rows, 256 x 256: 245 us with dx, which takes 18).
template <typename O, int PAIR_, int NT_> struct WeightsJob : NoLookAhead {
  static constexpr int PAIR = PAIR_, NT = NT_, PLANES = 1, PASS = sizeof(O) == 4 ? 8 : 0;
  static constexpr bool AMN = true, BMN = true, RAGGED = true;
  using Params = GroupedParams;
  using Extra = WeightTile;
  static __device__ int plane_stride(const Params &) { return 0; }
  struct Walk {
    int group, begin, end;
    __device__ Walk(const Params &) : group(-1) {}
    __device__ bool find(const Params &p, int i, TileOf<Extra> &t) {
      const int row_tiles = (p.k + kRows * PAIR - 1) / (kRows * PAIR);
      const int per = row_tiles * p.column_tiles;
      const int e = i / per;
      if (e >= p.groups) return false;
      if (e != group) group_rows(p.offsets, p.wide, group = e, p.rows, begin, end);
      // 8 row tiles at a time sweep the columns, so that the tiles of a wave
      // share their operands in L2
      const int local = i - e * per, sweep = local / (8 * p.column_tiles);
      const int in = local - sweep * 8 * p.column_tiles, size = min(row_tiles - sweep * 8, 8);
      t.a_row = (sweep * 8 + in % size) * kRows * PAIR;
      t.b_row = in / size * NT;
      t.a_mat = t.b_mat = 0;
      t.k_begin = begin;
      t.k_len = end - begin;
      t.extra = WeightTile{t.a_row, t.b_row, e};
      return true;
    }
  };
  template <class Source>
  static __device__ void epilogue(const Params &p, const TileOf<Extra> &t, const Source &source, int row,
                                  int column, unsigned char *mine, Ahead &) {
    const int64_t r0 = t.extra.row + row, c0 = t.extra.column + column;
    write_rows<O, NT / 2>(source, mine,
                          static_cast<O *>(p.out) + ((int64_t)t.extra.group * p.k + r0) * p.ld + c0,
                          p.ld, (int)(p.k - r0), p.n - c0, p.vectors);
  }
  static __device__ void finish(const Params &, int, int) {}
};

int check_grouped(int dtype, int out_dtype, int32_t groups, int64_t rows, int64_t k, int64_t n) {
  if (dtype != OZ_F16 && dtype != OZ_BF16)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported operand dtype %d (fp16 or bf16)", dtype);
  if (out_dtype != dtype && out_dtype != OZ_F32)
    return set_error(OZ_ERR_UNSUPPORTED, "unsupported output dtype %d", out_dtype);
  if (groups < 1) return set_error(OZ_ERR_INVALID, "at least one group is needed, got %d", groups);
  if (rows < 0 || k < 0 || n < 0) return set_error(OZ_ERR_INVALID, "negative size");
  if (rows > (1 << 30) || k > (1 << 30) || n > (1 << 30) || groups > (1 << 24))
    return set_error(OZ_ERR_INVALID, "size out of range");
  return OZ_OK;
}

// Whether the copy unit can read rows (and matrices) that far apart.
bool pitch_ok(int64_t stride, int64_t count) {
  return count <= 1 || (stride > 0 && stride % 8 == 0 && stride < ((int64_t)1 << 38));
}
int64_t pitch_bytes(int64_t stride, int64_t count, int64_t inner) {
  return 2 * (count <= 1 ? (inner + 7) / 8 * 8 : stride);
}

bool readable(const void *p, int64_t rows, int64_t row_stride, int64_t mats, int64_t mat_stride) {
  return (uintptr_t)p % 16 == 0 && pitch_ok(row_stride, rows) && pitch_ok(mat_stride, mats);
}

// Copies of operands whose rows the copy unit cannot address (16-byte boundaries
// and pitches): rows of 2-byte elements with unit stride to rows 16 bytes apart,
// both operands of a call in one launch.  A warp takes up to 2048 elements of a
// row, 9 words a lane on their way at a time.  1003 rows / 12 experts, 1000 x 1407,
// most of whose time is this copy of 34 MB: 33.1 us with 6 blocks an SM, 39.4
// with 4, 35.3 with 8 (and so fewer registers), 34.5 with 13 words.
struct Repitch {
  const unsigned short *from;
  unsigned short *to;
  int64_t from_row, from_mat, to_row;
  uint32_t rows, lines, parts;         // rows of a matrix, of all, and parts of 2048 elements of a row
  int inner;
};
struct RepitchTwo { Repitch job[2]; };
constexpr int kPart = 2048;

__global__ void __launch_bounds__(256, 6) repitch_kernel(const __grid_constant__ RepitchTwo two) {
  const Repitch &p = two.job[blockIdx.y];
  const int lane = threadIdx.x % 32;
  const uint64_t all = (uint64_t)p.lines * p.parts;
  for (uint64_t v = (uint64_t)blockIdx.x * 8 + threadIdx.x / 32; v < all; v += (uint64_t)gridDim.x * 8) {
    const uint32_t line = p.parts == 1 ? (uint32_t)v : (uint32_t)(v / p.parts);
    const int first = p.parts == 1 ? 0 : (int)(v - (uint64_t)line * p.parts) * kPart;
    const uint32_t mat = line / p.rows;
    const unsigned short *from = p.from + mat * p.from_mat + (int64_t)(line - mat * p.rows) * p.from_row;
    uint32_t *to = reinterpret_cast<uint32_t *>(p.to + line * p.to_row);
    const int count = min(p.inner - first, kPart);
    // aligned words: a row that starts in the middle of one gets its pairs from two
    // neighbouring words (the halves that belong to neither row nor part stay unused;
    // they share their word with an element, so they can be read)
    const unsigned short *start = from + first;
    const int off = (int)((uintptr_t)start >> 1 & 1);
    const uint32_t *words = reinterpret_cast<const uint32_t *>(start - off);
    to += first / 2;
    for (int j0 = 0; j0 * 2 < count; j0 += 256) {
      uint32_t w[9];
#pragma unroll
      for (int i = 0; i < 9; ++i) {
        const int j = j0 + i * 32 + lane;
        w[i] = 2 * j - off < count && (i < 8 || lane == 0) ? __ldg(words + j) : 0;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t down = __shfl_down_sync(0xffffffffu, w[i], 1), over = __shfl_sync(0xffffffffu, w[i + 1], 0);
        const int j = j0 + i * 32 + lane;
        if (2 * j < count) to[j] = off ? __funnelshift_r(w[i], lane == 31 ? over : down, 16) : w[i];
      }
    }
  }
}

// An operand as it is, or its copy in the workspace.
struct Operand {
  const void *p;
  int64_t rows, row, mats, mat;
  int inner;
};
int64_t copy_bytes(const Operand &o) {
  if (o.p && readable(o.p, o.rows, o.row, o.mats, o.mat)) return 0;
  return (o.rows * o.mats * ((o.inner + 7) / 8 * 8) * 2 + 255) / 256 * 256;
}
int lay_out(Operand *ops, void *workspace, int64_t workspace_bytes, cudaStream_t st) {
  RepitchTwo two{};
  int n = 0;
  int64_t at = 0, most = 0;
  for (int i = 0; i < 2; ++i) {
    Operand &o = ops[i];
    const int64_t bytes = copy_bytes(o);
    if (!bytes) continue;
    if (!workspace || (uintptr_t)workspace % 256 != 0 || workspace_bytes < at + bytes)
      return set_error(OZ_ERR_INVALID,
                       "an operand off the 16-byte boundaries needs a workspace of %lld bytes (256-byte "
                       "aligned), got %lld at %p",
                       (long long)(at + bytes), (long long)workspace_bytes, workspace);
    if ((uintptr_t)o.p % 2 != 0) return set_error(OZ_ERR_INVALID, "an operand is not aligned to its elements");
    unsigned char *to = static_cast<unsigned char *>(workspace) + at;
    const int64_t pitch = (o.inner + 7) / 8 * 8;
    const int64_t parts = (o.inner + kPart - 1) / kPart;
    if (o.rows * o.mats > INT32_MAX) return set_error(OZ_ERR_INVALID, "size out of range");
    two.job[n++] = Repitch{static_cast<const unsigned short *>(o.p), reinterpret_cast<unsigned short *>(to), o.row,
                           o.mat, pitch, (uint32_t)o.rows, (uint32_t)(o.rows * o.mats), (uint32_t)parts, o.inner};
    o.p = to;
    o.row = pitch;
    o.mat = pitch * o.rows;
    at += bytes;
    most = max(most, (o.rows * o.mats * parts + 7) / 8);
  }
  if (!n) return OZ_OK;
  count_launch();
  repitch_kernel<<<dim3((unsigned)min(most, (int64_t)sm_count() * 16), n), 256, 0, st>>>(two);
  return check_cuda(cudaGetLastError(), "repitch_kernel launch");
}

template <class J>
int run(const CUtensorMap &a, const CUtensorMap &b, GroupedParams p, int64_t row_tiles, int64_t n_side,
        int n_per_tile, cudaStream_t st, const char *what) {
  const int64_t columns = (n_side + n_per_tile - 1) / n_per_tile;
  if (row_tiles * columns > INT32_MAX / 2) return set_error(OZ_ERR_INVALID, "too many tiles");
  p.column_tiles = (int)columns;
  return launch<J>(a, b, p, row_tiles * columns, st, what);
}

template <typename O>
int grouped(const void *x, const void *w, int64_t x_sr, int64_t w_se, bool across, int64_t w_row,
            const GroupedParams &p, cudaStream_t st) {
  // The least estimated time of three tile shapes: waves of tiles over the GPU,
  // from the mean group (half a tile of each group is empty on average), times a
  // tile's blocks and four more for its start and end, times the bytes a CTA loads a
  // block: 128 columns by at most 32 rows (20 KB), 128 rows by 128 columns (32),
  // pairs of CTAs 256 by 256 (32 each).  Measured, 128 x 128 against pairs: 256
  // rows / 8 experts, 2048 x 2048, 23 and 16 us; 1003 rows / 12 experts, 1000 x 1408,
  // 14 and 12 us.
  const int64_t groups = min(p.groups, p.rows);
  const double mean = (double)p.rows / groups;
  const double blocks64 = (p.k + kBlock - 1) / kBlock + 4;
  auto time = [&](int high, int wide, int bytes, int ctas) {
    const double tiles = groups * max(1.0, mean / high + 0.5) * ((p.n + wide - 1) / wide);
    return ceil(tiles * ctas / sm_count()) * blocks64 * bytes;
  };
  const double few_time = time(32, kRows, 20, 1), one_time = time(kRows, 128, 32, 1);
  const double two_time = time(256, 2 * kRows, 32, 2);
  const bool few = few_time <= one_time && few_time <= two_time;
  const int pair = two_time <= one_time ? 2 : 1;
  // columns as A: 32 experts of 256 rows on average, 4096 columns: k 256 32 us (rows as
  // A 30), k 512 45 (47), k 2048 143 (152); one of 20000 rows, k 2048: 234 (226)
  const bool turned = pair == 2 && p.k >= 512 && mean < 2048;
  CUtensorMap tx, tw;
  const int64_t wr = across ? p.k : p.n, wi = across ? p.n : p.k;
  const int64_t xb = pitch_bytes(x_sr, p.rows, p.k), wb = pitch_bytes(w_row, wr, wi);
  if (int rc = make_map(&tx, x, p.k, p.rows, 1, xb, xb, few ? 32 : turned ? 64 : kRows)) return rc;
  if (int rc = make_map(&tw, w, wi, wr, p.groups, wb, p.groups > 1 ? 2 * w_se : wb, across ? kBlock : kRows))
    return rc;
  const char *what = "grouped product launch";
  const int64_t per = few ? 32 : kRows * pair;
  const int64_t blocks = p.rows / per + groups;
  if (few)
    return across ? run<ColumnsJob<O, 32, true>>(tw, tx, p, blocks, p.n, kRows, st, what)
                  : run<ColumnsJob<O, 32, false>>(tw, tx, p, blocks, p.n, kRows, st, what);
  if (pair == 1)
    return across ? run<RowsJob<O, 1, 128, true>>(tx, tw, p, blocks, p.n, 128, st, what)
                  : run<RowsJob<O, 1, 128, false>>(tx, tw, p, blocks, p.n, 128, st, what);
  if (!turned)
    return across ? run<RowsJob<O, 2, 256, true>>(tx, tw, p, blocks, p.n, 256, st, what)
                  : run<RowsJob<O, 2, 256, false>>(tx, tw, p, blocks, p.n, 256, st, what);
  return across ? run<PairsJob<O, true>>(tw, tx, p, blocks, p.n, 256, st, what)
                : run<PairsJob<O, false>>(tw, tx, p, blocks, p.n, 256, st, what);
}

template <typename O>
int wgrad(const void *x, const void *dy, int64_t x_sr, int64_t dy_sr, const GroupedParams &p,
          cudaStream_t st) {
  CUtensorMap tx, ty;
  const int64_t xb = pitch_bytes(x_sr, p.rows, p.k), yb = pitch_bytes(dy_sr, p.rows, p.n);
  if (int rc = make_map(&tx, x, p.k, p.rows, 1, xb, xb, kBlock)) return rc;
  if (int rc = make_map(&ty, dy, p.n, p.rows, 1, yb, yb, kBlock)) return rc;
  const char *what = "grouped weight gradient launch";
  if (p.k > kRows && p.n > 128)
    return run<WeightsJob<O, 2, 256>>(tx, ty, p, (int64_t)p.groups * ((p.k + 255) / 256), p.n, 256, st, what);
  return run<WeightsJob<O, 1, 128>>(tx, ty, p, (int64_t)p.groups * ((p.k + 127) / 128), p.n, 128, st, what);
}

}  // namespace
}  // namespace oz

extern "C" int oz_grouped_matmul(const oz_grouped_args *args, void *stream) {
  if (!args) return oz::set_error(OZ_ERR_INVALID, "null arguments");
  const auto [x, w, offsets, y, rows, k, n, x_sr, w_se, w_sk, w_sn, ldy, workspace, workspace_bytes, groups,
              offsets_64, dtype, out_dtype] = *args;
  using namespace oz;
  if (int rc = check_grouped(dtype, out_dtype, groups, rows, k, n)) return rc;
  if (rows == 0 || n == 0) return OZ_OK;
  if (!y || ldy < n) return set_error(OZ_ERR_INVALID, "bad output (ldy=%lld n=%lld)",
                                      (long long)ldy, (long long)n);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int es = dtype_size(out_dtype);
  if (k == 0)
    return check_cuda(cudaMemset2DAsync(y, (size_t)(ldy * es), 0, (size_t)(n * es), (size_t)rows, st),
                      "cudaMemset2DAsync");
  if (!offsets || !x || !w) return set_error(OZ_ERR_INVALID, "null pointer");
  // stored across the contraction (unit stride along n) or along it
  const bool across = w_sn == 1 || (n == 1 && w_sk != 1);
  if (!across && w_sk != 1 && k != 1)
    return set_error(OZ_ERR_INVALID, "w must have a unit stride along k or n");
  Operand ops[2] = {{x, rows, x_sr, 1, 0, (int)k},
                    {w, across ? k : n, across ? w_sk : w_sn, groups, w_se, (int)(across ? n : k)}};
  if (int rc = lay_out(ops, workspace, workspace_bytes, st)) return rc;
  GroupedParams p{offsets, y, ldy, offsets_64, groups, (int)rows, (int)k, (int)n, 0,
                  (uintptr_t)y % 16 == 0 && ldy * es % 16 == 0, tile::instruction(dtype)};
  if (out_dtype == OZ_F32) return grouped<float>(ops[0].p, ops[1].p, ops[0].row, ops[1].mat, across, ops[1].row, p, st);
  if (dtype == OZ_F16) return grouped<__half>(ops[0].p, ops[1].p, ops[0].row, ops[1].mat, across, ops[1].row, p, st);
  return grouped<__nv_bfloat16>(ops[0].p, ops[1].p, ops[0].row, ops[1].mat, across, ops[1].row, p, st);
}

extern "C" int oz_grouped_wgrad(const oz_grouped_wgrad_args *args, void *stream) {
  if (!args) return oz::set_error(OZ_ERR_INVALID, "null arguments");
  const auto [x, dy, offsets, dw, rows, k, n, x_sr, dy_sr, workspace, workspace_bytes, groups, offsets_64, dtype,
              out_dtype] = *args;
  using namespace oz;
  if (int rc = check_grouped(dtype, out_dtype, groups, rows, k, n)) return rc;
  if (k == 0 || n == 0) return OZ_OK;
  if (!dw) return set_error(OZ_ERR_INVALID, "null pointer");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int es = dtype_size(out_dtype);
  if (rows == 0)
    return check_cuda(cudaMemsetAsync(dw, 0, (size_t)(groups * k * n * es), st), "cudaMemsetAsync");
  if (!offsets || !x || !dy) return set_error(OZ_ERR_INVALID, "null pointer");
  Operand ops[2] = {{x, rows, x_sr, 1, 0, (int)k}, {dy, rows, dy_sr, 1, 0, (int)n}};
  if (int rc = lay_out(ops, workspace, workspace_bytes, st)) return rc;
  GroupedParams p{offsets, dw, n, offsets_64, groups, (int)rows, (int)k, (int)n, 0,
                  (uintptr_t)dw % 16 == 0 && n * es % 16 == 0, tile::instruction(dtype)};
  if (out_dtype == OZ_F32) return wgrad<float>(ops[0].p, ops[1].p, ops[0].row, ops[1].row, p, st);
  if (dtype == OZ_F16) return wgrad<__half>(ops[0].p, ops[1].p, ops[0].row, ops[1].row, p, st);
  return wgrad<__nv_bfloat16>(ops[0].p, ops[1].p, ops[0].row, ops[1].row, p, st);
}
