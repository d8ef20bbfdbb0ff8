// What the kernels of ivakv_rows.hip and the wide shared walk of ivakv_prefill.hip have in common: their
// arguments, and how groups of rows and their pages are cut into pieces.  Internal to libivakv.
#pragma once

#include "ivakv_tile.h"

namespace ivakv {

struct RowArgs {
  const void* q;  // [n_rows, Hq, D]
  const void* k_pool;
  const void* v_pool;
  const float* k_scale;  // FP8 pools
  const float* v_scale;
  void* out;             // like q
  const int32_t* bt;     // [tables, max_blocks]
  const int32_t* ctx;    // cross: keys of each group; prefix: length of each row's sequence
  const int32_t* start;  // [n_groups + 1] first query row of each group
  const int32_t* shared; // prefix: [n_groups] shared tokens
  float* part_acc;       // shared partials [slot][16 NR][D]
  float* part_ml;        // [slot][16 NR][2]  (running max, sum)
  float* own_acc;        // own partials [slot][G][D]
  float* own_ml;         // [slot][G][2]
  int32_t* own_pref;     // [n_rows + 1] own page sets before each row
  int n_groups, n_rows, Hkv, G, max_blocks, num_pages;
  int prefix;            // 1: prefix groups, 0: cross
  int max_rows;          // query rows of the largest group
  int rows_shift;        // log2 of the rows of a chunk (16 NR)
  int items, split;      // (piece, row chunk) pairs the grid holds for a kv head; whether pages are cut
  int unit;              // pages a shared workgroup's waves take at once
  int shared_wgs, own_waves;  // workgroups of the shared walk, waves of the own walk
  float scale_log2;
  int window, n_sink;
};

// The shared walk for many rows (ivakv_prefill.hip): 16-bit pools of the queries' type, head_dim 128 or
// 256, chunks of wide_rows(head_dim) rows, pieces of a multiple of four pages.
int wide_rows(int head_dim);
void launch_rows_wide(int dtype, int head_dim, const RowArgs& a, hipStream_t stream);

namespace {

// Rows [r0, r1) of group g, inside [0, n_rows].
__device__ inline void group_rows(const RowArgs& a, int g, int& r0, int& r1) {
  r0 = min(max(a.start[g], 0), a.n_rows);
  r1 = min(max(a.start[g + 1], r0), a.n_rows);
}

// One group as a lane holds it: its rows, their chunks and its pages.  prefix: the full pages of the
// shared tokens, inside the table.  A group without rows has no chunks.
struct Group {
  int r0, r1, chunks, pages;
};
__device__ inline Group load_group(const RowArgs& a, int g) {
  Group x{0, 0, 0, 0};
  if (g >= a.n_groups) return x;
  const int n = a.prefix ? a.shared[g] / kBS : cdiv(max(a.ctx[g], 0), kBS);
  group_rows(a, g, x.r0, x.r1);
  x.chunks = (min(x.r1 - x.r0, a.max_rows) * a.G + (1 << a.rows_shift) - 1) >> a.rows_shift;
  x.pages = x.chunks > 0 ? min(max(n, 0), a.max_blocks) : 0;
  return x;
}

// Whether a sequence of length len takes part in its group's shared walk of `blocks` pages: it has
// the whole prefix and its window cuts nothing off.  (Any other row walks all of its visible pages
// itself, so the shared walk needs no mask of its own.)
__device__ inline bool takes_part(const RowArgs& a, int len, int blocks) {
  return len >= blocks * kBS && (a.window <= 0 || len <= a.window);
}

// The first row of [r0, r1) that takes part, whose table the shared walk reads (-1: none, and then no
// row asks for the walk's partials).
__device__ inline int prefix_row(const RowArgs& a, int blocks, int r0, int r1, int lane) {
  for (int r = r0; r < r1; r += 64) {
    const uint64_t has =
        __builtin_amdgcn_ballot_w64(r + lane < r1 && takes_part(a, a.ctx[min(r + lane, r1 - 1)], blocks));
    if (has != 0) return r + __builtin_ctzll(has);
  }
  return -1;
}

// Inclusive scan over the wave's lanes (row shifts, then the rows' last lanes broadcast).
__device__ inline int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
  return x;
}
__device__ inline int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// How the groups' pages are cut: every list into pieces of `len` pages (a multiple of the pages that a
// workgroup's waves take at once), the shortest of four lengths with which all groups' items, pieces
// times row chunks, number at most a.items.  The last of the four, sum (pages x chunks) / (items -
// sum chunks), always does: a group has at most one piece that is not whole.  Without a.split
// every group is one piece.  Partials are numbered group by group, in it piece by piece, kv head by kv
// head, chunk by chunk; the shared workgroups kv head by kv head, so that an XCD, which takes a
// contiguous run of them, gets its share of every group, long or short (bf16, 16 sequences of 97 .. 448
// rows on 700 .. 1500 keys, 16 heads of 64: 44 us against 51 group by group; 32 / 8 heads of 128 on FP8
// pages 186 against 204; 64 FP8 rows behind one prefix 54.8 against 53.8).  A cross group without keys
// has one empty piece, which writes its rows' zeros.  Each wave works this out for itself, 64 groups
// at a time, the first 64 (`own`, group `lane`) from registers.
struct Pieces {
  int len, least, items;  // items: of all groups
  __device__ inline int of(const Group& x) const {
    return x.chunks == 0 ? 0 : max((int)(((uint32_t)x.pages + (uint32_t)len - 1) / (uint32_t)len), least);
  }

  __device__ inline Pieces(const RowArgs& a, const Group& own, int lane) {
    least = a.prefix ? 0 : 1;
    len = 1 << 30;
    int work = 0, chunks = 0;
    if (a.split) {  // (then items x max_blocks, and so the work, is below 2^31)
      work = wave_sum(own.pages * own.chunks);
      chunks = wave_sum(own.chunks);
      for (int g0 = 64; g0 < a.n_groups; g0 += 64) {
        const Group x = load_group(a, g0 + lane);
        work += wave_sum(x.pages * x.chunks);
        chunks += wave_sum(x.chunks);
      }
    }
#pragma unroll 1
    for (int k = a.split ? 0 : 3; k < 4; ++k) {
      if (a.split) {
        const uint32_t parts = (uint32_t)max(a.items - k * chunks / 3, 1), unit = (uint32_t)a.unit;
        len = (int)max(((uint32_t)work + parts * unit - 1) / (parts * unit) * unit, unit);
      }
      items = wave_sum(of(own) * own.chunks);
      for (int g0 = 64; g0 < a.n_groups; g0 += 64) {
        const Group x = load_group(a, g0 + lane);
        items += wave_sum(of(x) * x.chunks);
      }
      if (items <= a.items) return;
    }
  }

  // What shared workgroup `wg` does: the group, which of its pieces, kv head and chunk, and its
  // partial; false when there is nothing for it.
  __device__ inline bool find(const RowArgs& a, const Group& own, int wg, int lane, Group& group, int& g, int& piece,
                              int& h, int& chunk, int& slot) const {
    h = (int)((uint32_t)wg / (uint32_t)items);
    const int item = wg - h * items;
    int before = 0;
    for (int g0 = 0; g0 < a.n_groups; g0 += 64) {
      const Group x = g0 == 0 ? own : load_group(a, g0 + lane);
      const int n = of(x) * x.chunks, incl = wave_scan(n);
      const uint64_t has = __builtin_amdgcn_ballot_w64(item < before + incl);
      if (has != 0) {
        const int w = __builtin_ctzll(has);
        g = g0 + w;
        group = Group{__builtin_amdgcn_readlane(x.r0, w), __builtin_amdgcn_readlane(x.r1, w),
                      __builtin_amdgcn_readlane(x.chunks, w), __builtin_amdgcn_readlane(x.pages, w)};
        const int first = before + __builtin_amdgcn_readlane(incl, w) - __builtin_amdgcn_readlane(n, w);
        const uint32_t at = (uint32_t)(item - first);
        chunk = (int)(at % (uint32_t)group.chunks);
        piece = (int)(at / (uint32_t)group.chunks);
        slot = first * a.Hkv + (piece * a.Hkv + h) * group.chunks + chunk;
        return true;
      }
      before += __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
  }

  // First partial of group g, and its pieces.
  __device__ inline void of_group(const RowArgs& a, const Group& own, int g, int lane, int64_t& first,
                                  int& pieces) const {
    int before = 0, n = 0, mine = 0;
    for (int g0 = 0; g0 <= g; g0 += 64) {
      const Group x = g0 == 0 ? own : load_group(a, g0 + lane);
      mine = of(x);
      n = g0 + lane <= g ? mine * x.chunks : 0;
      before += wave_sum(n);
    }
    pieces = __builtin_amdgcn_readlane(mine, g & 63);
    first = (int64_t)(before - __builtin_amdgcn_readlane(n, g & 63)) * a.Hkv;
  }
};

}  // namespace
}  // namespace ivakv
