// grouped.hpp — products over ragged groups of rows ("experts"): which rows
// and which weight a workgroup of the tiled GEMM kernels works on.
//
//   GroupedRows   C[r] = epi(op(B[e]) A[r] (+ bias[e])) for the rows r of
//                 group e: the M axis is cut into groups, each with its own B
//   GroupedSums   C[e] = sum over the rows r of group e of A[r]^T B[r]: the
//                 K axis is cut into groups, each with its own C
//
// Groups come as offsets[groups + 1] in device memory, written by the launch
// before (a router): the host never knows the sizes, so nothing waits for
// them.  Group e holds rows [end(e - 1), end(e)), end(e) being the largest of
// offsets[1 .. e + 1] cut to [0, rows] (end(-1) = 0): for ascending offsets
// that start at 0 these are the offsets themselves, and any other content
// still gives disjoint ranges within the operands.  Rows behind the last
// group form one more range, which GroupedRows fills with zeros.
//
// GroupedRows' grid covers the largest number of BM-row tiles that any group
// sizes can give; each wave finds its tile by itself, with one load of the
// offsets and two 64-lane scans (largest end so far, tiles so far), and
// surplus workgroups leave.  That costs about 1 us at the start of a
// workgroup; a launch of its own that wrote a tile table would cost 4-5.
#pragma once

#include <type_traits>

#include "gemm16.hpp"

namespace sf {

// M, N, K, tiles_* as GemmParams says, but M (GroupedRows) and K (GroupedSums)
// are the sizes over all groups.
struct GroupedRows : GemmParams {
  const int* offsets;
  int groups, rows;
  int cus;  // > 0: one of a pair of launches (GroupPart), on this many CUs
};
struct GroupedSums : GemmParams {
  const int* offsets;
  int groups, rows;
};

// A size that is fixed in an ordinary launch and set per group in a grouped one.
template <bool VARIES>
struct GroupVar {
  typedef int type;
};
template <>
struct GroupVar<false> {
  typedef const int type;
};

constexpr int kMaxGroups = 1024;

struct GroupTile {
  int e;     // group, or `groups` for the rows behind the last one
  int row;   // first row of the tile
  int rows;  // rows of the tile, 1 .. BM
  int tn;    // column tile
};

__device__ __forceinline__ int group_clamp(int v, int rows) { return v < 0 ? 0 : (v < rows ? v : rows); }

// Inclusive scans over the 64 lanes.
__device__ __forceinline__ int wave_scan_max(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(v, off, 64);
    if (lane >= off && o > v) v = o;
  }
  return v;
}
__device__ __forceinline__ int wave_scan_sum(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(v, off, 64);
    if (lane >= off) v += o;
  }
  return v;
}

// Which part of the tile list a launch works on.
//   ALL   every tile
//   HEAD  the whole rounds of one tile a CU (p.cus), and the rest where it is
//         more than half a round
//   REST  what HEAD leaves, in quarters: tile t's quarter q is the BM x BM / 2
//         rows and columns at row (q & 1) BM and column tile 2 tn + (q >> 1) of
//         a launch with tiles of half the edge
// A last round of a few 256 x 256 tiles costs as much as a full one; in
// quarters it runs on all CUs.
enum GroupPart { GROUP_ALL, GROUP_HEAD, GROUP_REST };

// The tile of workgroup `pid` (see above), every wave for itself; false for a
// surplus workgroup.  Tiles run group by group, within a group in the column
// bands of group_tile, and each XCD takes a contiguous range.  BM and tiles_n
// are those of the tile list (REST: of HEAD's).
template <int BM, GroupPart PART>
__device__ __forceinline__ bool group_find_at(const int* __restrict__ offsets, int groups, int rows, int tiles_n,
                                              int cus, int pid, GroupTile& out) {
  const int lane = threadIdx.x & 63;
  const int per = (groups + 1 + 63) / 64;  // groups per lane, the range behind the last among them
  const int i0 = lane * per;
  auto end_of = [&](int i) { return i < groups ? group_clamp(offsets[i + 1], rows) : rows; };
  int top = 0;
  for (int i = i0; i < i0 + per && i <= groups; ++i) {
    const int v = end_of(i);
    top = v > top ? v : top;
  }
  const int incl = wave_scan_max(top);
  int start = __shfl_up(incl, 1, 64);
  if (lane == 0) start = 0;
  int tiles = 0;
  {
    int s = start;
    for (int i = i0; i < i0 + per && i <= groups; ++i) {
      const int v = end_of(i);
      if (v > s) {
        tiles += (v - s + BM - 1) / BM;
        s = v;
      }
    }
  }
  const int upto = wave_scan_sum(tiles);
  const int active = __builtin_amdgcn_readlane(upto, 63) * tiles_n;
  int lo = 0, hi = active;  // this launch's tiles
  if constexpr (PART != GROUP_ALL) {
    const int left = active % cus;
    const int cut = 2 * left <= cus ? active - left : active;
    if constexpr (PART == GROUP_HEAD) hi = cut;
    else lo = cut;
  }
  constexpr int Q = PART == GROUP_REST ? 4 : 1;
  if (pid >= (hi - lo) * Q) return false;
  const int sub = xcd_remap(pid, (hi - lo) * Q);
  const int tile = lo + sub / Q;
  const bool mine = tile >= (upto - tiles) * tiles_n && tile < upto * tiles_n;
  int e = 0, row = 0, cnt = 0, first = 0;  // group, its first row, its rows, its first tile
  if (mine) {
    int s = start, t = (upto - tiles) * tiles_n;
    for (int i = i0; i < i0 + per && i <= groups; ++i) {
      const int v = end_of(i);
      if (v > s) {
        const int n = (v - s + BM - 1) / BM * tiles_n;
        if (tile < t + n) {
          e = i;
          row = s;
          cnt = v - s;
          first = t;
          break;
        }
        t += n;
        s = v;
      }
    }
  }
  const int src = __builtin_ctzll(__ballot(mine));
  e = __builtin_amdgcn_readlane(e, src);
  row = __builtin_amdgcn_readlane(row, src);
  cnt = __builtin_amdgcn_readlane(cnt, src);
  first = __builtin_amdgcn_readlane(first, src);
  int tm, tn;
  group_tile(tile - first, (cnt + BM - 1) / BM, tiles_n, 8, tm, tn);
  constexpr int H = PART == GROUP_REST ? BM / 2 : BM;  // rows of this launch's tiles
  const int r0 = tm * BM + (PART == GROUP_REST ? (sub & 1) * H : 0);
  if (PART == GROUP_REST && r0 >= cnt) return false;
  out.e = e;
  out.row = row + r0;
  out.rows = cnt - r0 < H ? cnt - r0 : H;
  out.tn = PART == GROUP_REST ? 2 * tn + ((sub >> 1) & 1) : tn;
  return true;
}

template <int BM, typename P>
__device__ __forceinline__ bool group_find(const P& p, GroupTile& out) {
  return group_find_at<BM, GROUP_ALL>(p.offsets, p.groups, p.rows, p.tiles_n, 0, (int)blockIdx.x, out);
}
// 256-row tiles: all of them, or HEAD where the launch is one of a pair.
template <typename P>
__device__ __forceinline__ bool group_find_head(const P& p, GroupTile& out) {
  if (p.cus == 0) return group_find<256>(p, out);
  return group_find_at<256, GROUP_HEAD>(p.offsets, p.groups, p.rows, p.tiles_n, p.cus, (int)blockIdx.x, out);
}
// 128-row tiles: all of them, or the quarters of what the 256-row launch left.
template <typename P>
__device__ __forceinline__ bool group_find_rest(const P& p, GroupTile& out) {
  if (p.cus == 0) return group_find<128>(p, out);
  return group_find_at<256, GROUP_REST>(p.offsets, p.groups, p.rows, p.tiles_n, p.cus, (int)blockIdx.x, out);
}

// Zeros to `rows` rows of C (leading dimension ld) in columns n0 .. n0 + width
// - 1 below N, by the whole workgroup.
__device__ __forceinline__ void group_zero_tile(uint16_t* C, int64_t ld, int rows, int n0, int N, int width) {
  const int w = N - n0 < width ? N - n0 : width;
  for (int i = threadIdx.x; i < rows * w; i += blockDim.x) C[(int64_t)(i / w) * ld + n0 + i % w] = 0;
}

// First row and rows of group e, every wave for itself.
__device__ __forceinline__ void group_bounds(const int* __restrict__ offsets, int e, int rows, int& first, int& cnt) {
  const int lane = threadIdx.x & 63;
  int top = 0;  // largest end of the groups before e
  for (int i = lane; i < e; i += 64) {
    const int v = group_clamp(offsets[i + 1], rows);
    top = v > top ? v : top;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const int o = __shfl_xor(top, off, 64);
    top = o > top ? o : top;
  }
  top = __builtin_amdgcn_readfirstlane(top);
  const int end = group_clamp(offsets[e + 1], rows);
  first = top;
  cnt = end > top ? end - top : 0;
}

// Most tiles of `bm` rows that `rows` rows in at most `groups` groups (and
// the range behind the last) can take.
inline int64_t grouped_max_tiles(int64_t rows, int64_t groups, int64_t bm) {
  const int64_t g = groups + 1 < rows ? groups + 1 : rows;  // ranges with a row at all
  return (rows + g * (bm - 1)) / bm;
}

}  // namespace sf
