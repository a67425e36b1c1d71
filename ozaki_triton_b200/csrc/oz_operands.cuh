// oz_operands.cuh -- operands of the tile engine (oz_tile.cuh) as the copy unit can
// read them: where their rows do not start on 16-byte boundaries they are copied first.
#pragma once

#include "oz_stream.cuh"
#include "oz_tile.cuh"

namespace oz {
namespace {
using namespace tile;

// Whether the copy unit can read rows (and matrices) that far apart.
inline bool pitch_ok(int64_t stride, int64_t count) {
  return count <= 1 || (stride > 0 && stride % 8 == 0 && stride < ((int64_t)1 << 38));
}
inline int64_t pitch_bytes(int64_t stride, int64_t count, int64_t inner) {
  return 2 * (count <= 1 ? (inner + 7) / 8 * 8 : stride);
}

inline bool readable(const void *p, int64_t rows, int64_t row_stride, int64_t mats, int64_t mat_stride) {
  return (uintptr_t)p % 16 == 0 && pitch_ok(row_stride, rows) && pitch_ok(mat_stride, mats);
}

// Copies of operands whose rows the copy unit cannot address (16-byte boundaries
// and pitches): rows of 2-byte elements with unit stride to rows 16 bytes apart,
// all operands of a call in one launch.  A warp takes up to 2048 elements of a
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
struct RepitchAll { Repitch job[3]; };
constexpr int kPart = 2048;

__global__ void __launch_bounds__(256, 6) repitch_kernel(const __grid_constant__ RepitchAll all_jobs) {
  const Repitch &p = all_jobs.job[blockIdx.y];
  stream::start_after_earlier_kernels();
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
        w[i] = 2 * j - off < count && (i < 8 || lane == 0) ? *(words + j) : 0;
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

// An operand as it is, or its copy in the workspace; at most 3 to a call.
struct Operand {
  const void *p;
  int64_t rows, row, mats, mat;
  int inner;
};
inline int64_t copy_bytes(const Operand &o) {
  if (o.p && readable(o.p, o.rows, o.row, o.mats, o.mat)) return 0;
  return (o.rows * o.mats * ((o.inner + 7) / 8 * 8) * 2 + 255) / 256 * 256;
}
inline int lay_out(Operand *ops, int count, void *workspace, int64_t workspace_bytes, cudaStream_t st) {
  RepitchAll all{};
  int n = 0;
  int64_t at = 0, most = 0;
  for (int i = 0; i < count; ++i) {
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
    all.job[n++] = Repitch{static_cast<const unsigned short *>(o.p), reinterpret_cast<unsigned short *>(to), o.row,
                           o.mat, pitch, (uint32_t)o.rows, (uint32_t)(o.rows * o.mats), (uint32_t)parts, o.inner};
    o.p = to;
    o.row = pitch;
    o.mat = pitch * o.rows;
    at += bytes;
    most = max(most, (o.rows * o.mats * parts + 7) / 8);
  }
  if (!n) return OZ_OK;
  return stream::launch(repitch_kernel, dim3((unsigned)min(most, (int64_t)tile::sm_count() * 16), n), 256, 0, st,
                        "repitch_kernel launch", all);
}

}  // namespace
}  // namespace oz
