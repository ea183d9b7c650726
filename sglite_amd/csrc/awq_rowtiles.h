// Tiles of consecutive sorted rows of one expert, counted over the experts'
// buckets in order.
#pragma once

#include "awq_device.h"

namespace sgl_awq {

// One lane per EPL (2 or 8) experts; every wave of a workgroup finds its tiles
// by itself.  Offsets are clamped to the sorted table, whatever they hold.
template <int EPL>
struct RowTiles {
  int r0[EPL], nr[EPL];  // first sorted row and rows of the lane's experts
  int excl, incl;        // tiles before the lane's first expert and past its last one

  __device__ __forceinline__ void load(const int32_t* offsets, int E, int sorted_cap, int lane) {
    int o[EPL + 1];
#pragma unroll
    for (int i = 0; i <= EPL; ++i) o[i] = offsets[min(lane * EPL + i, E)];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      r0[i] = min(max(o[i], 0), sorted_cap);
      const int r1 = min(max(o[i + 1], r0[i]), sorted_cap);
      nr[i] = lane * EPL + i < E ? r1 - r0[i] : 0;
    }
  }

  __device__ __forceinline__ void scan(int tile_rows, int lane) {
    int sum = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) sum += (nr[i] + tile_rows - 1) / tile_rows;
    incl = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(incl, d);
      if (lane >= d) incl += u;
    }
    excl = incl - sum;
  }

  __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(incl, 63); }

  // Tile t's expert, first sorted row and rows (at most tile_rows); e = -1 past the last tile.
  __device__ __forceinline__ void find(int t, int tile_rows, int lane, int& e, int& rb, int& rows) const {
    const uint64_t hit = __ballot(t >= excl && t < incl);
    if (hit == 0) {
      e = -1;
      return;
    }
    int fe = 0, fb = 0, fn = 0, pos = excl;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int n = (nr[i] + tile_rows - 1) / tile_rows;
      if (t >= pos && t < pos + n) {
        fe = lane * EPL + i;
        fb = r0[i] + (t - pos) * tile_rows;
        fn = min(tile_rows, r0[i] + nr[i] - fb);
      }
      pos += n;
    }
    const int src = __builtin_ctzll(hit);
    e = __builtin_amdgcn_readlane(fe, src);
    rb = __builtin_amdgcn_readlane(fb, src);
    rows = __builtin_amdgcn_readlane(fn, src);
  }

  // Unit u of the (tile, column group) pairs, the experts in order and inside
  // an expert its tiles for one column group after the other's: neighbours read
  // the same weights.  The tiles of an expert are of nearly equal size, rounded
  // up to `grain` rows.  e = -1 past the last unit.
  __device__ __forceinline__ void find_unit(int u, int groups, int tile_rows, int grain, int lane, int& e, int& rb,
                                            int& rows, int& group) const {
    const uint64_t hit = __ballot(u >= excl * groups && u < incl * groups);
    if (hit == 0) {
      e = -1;
      return;
    }
    int fe = 0, fb = 0, fn = 0, fg = 0, pos = excl;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int n = (nr[i] + tile_rows - 1) / tile_rows;
      if (u >= pos * groups && u < (pos + n) * groups) {
        const int at = u - pos * groups;
        fg = at / n;
        const int per = ((nr[i] + n - 1) / n + grain - 1) / grain * grain;
        fe = lane * EPL + i;
        fb = r0[i] + (at - fg * n) * per;
        fn = min(per, r0[i] + nr[i] - fb);
      }
      pos += n;
    }
    const int src = __builtin_ctzll(hit);
    e = __builtin_amdgcn_readlane(fe, src);
    rb = __builtin_amdgcn_readlane(fb, src);
    rows = __builtin_amdgcn_readlane(fn, src);
    group = __builtin_amdgcn_readlane(fg, src);
  }

  // Tiles of at most tile_rows rows, and the rows that they compute when each
  // takes `more` beyond its own.
  __device__ __forceinline__ void weigh(int tile_rows, int grain, int more, int& tiles, int& work) const {
    tiles = work = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int n = (nr[i] + tile_rows - 1) / tile_rows;
      const int per = n > 0 ? ((nr[i] + n - 1) / n + grain - 1) / grain * grain : 0;
      tiles += n;
      work += n * (per + more);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      tiles += __shfl_xor(tiles, d);
      work += __shfl_xor(work, d);
    }
  }
};

}  // namespace sgl_awq
