// Low-rank adapters of many requests beside a shared projection.
//
// A row m of the batch names an adapter e (or none).  With the adapter's A
// [P * R, K] (R ranks for each of the projection's P column parts), B [N, R],
// its rank r_e <= R and its scaling s_e, the projection's output y becomes
//
//   v[m, p, r] = sum_k x[m, k] A[p R + r, k]                       (shrink)
//   y'[m, n]   = y[m, n] + s_e sum_{r < r_e} v[m, part(n), r] B[n, r]   (expand)
//
// and with a gate/up activation out[m, j] = act(y'[m, j]) * y'[m, N/2 + j].
//
// Rows are taken in the order of their adapters (the alignment kernel's sorted
// table, 16-row blocks of one adapter, the rows without one in a bucket behind
// the last adapter), so both steps are MFMA products of a block's rows with one
// adapter's matrices as they lie in memory: A's and B's rows are contiguous in
// the summed index, which is the MFMA operand order of 8 consecutive values
// per lane.  v stays in fp32 between the launches, at the rows' sorted
// positions, one partial sum per k-slice, added in slice order: no atomics.
//
// Three sizes of batch:
//   few rows   every row is a block of its own, its adapter read from the ids:
//              nothing is sorted, and the shrink waits for two loads in a row
//              (id, then weights) and no more; the expand, as compiled, for v
//              first.  (Both steps in one launch, every workgroup computing v
//              for itself, took as long: a CU by itself draws the 80 to 160 KB
//              of A in 4 us and more.)
//   batches    16-row blocks of the sorted table
//   prefill    64-row tiles, what their waves share staged in LDS
#include <math.h>

#include <algorithm>

#include "awq_buffer.h"
#include "awq_epilogue.h"
#include "awq_launch.h"

namespace sgl_awq {

namespace {

constexpr int kLoraWaves = 4;
// k-slices of the shrink at most, for few rows and batches, and for prefill.
constexpr int kLoraSlices = 8;
constexpr int kTileSlices = 4;
constexpr int kStepK = 64;  // k per step of the shrink: 128 bytes of a row

// Loads above stay above: the wait counts of the rings below rely on how many
// a step issues.
__device__ __forceinline__ void stay_here() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// A value that no kernel writes while this one runs, at an address all lanes
// share: a scalar load.
template <typename T>
__device__ __forceinline__ T load_uniform(const T* p) {
  return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// Rows of block b (16 of the sorted table, or the one row b), their adapter and
// their positions in v.
struct BlockArgs {
  const int32_t* ids;     // adapter of each row (ROWS)
  const int32_t* sorted;  // rows by adapter, M in padding
  const int32_t* bucket;  // adapter of each 16-row block, L: none, -1: past the last block
  int M, L, blocks;       // blocks that the grid covers
};

template <bool ROWS>
__device__ __forceinline__ int block_adapter(const BlockArgs& a, int b) {
  if (!ROWS) return load_uniform(a.bucket + b);
  const int e = load_uniform(a.ids + b);
  return e >= 0 && e < a.L ? e : a.L;
}
// Prefill: workgroup `id` runs on XCD id % 8.  Each XCD takes neighbouring row
// tiles, so that it reads few adapters' matrices through its L2 (tiles dealt
// round, every L2 fetched all of them).  False past the last tile.
__device__ __forceinline__ bool row_tile(int id, int tiles, int& tile, int& rest) {
  const int per = (tiles + 7) >> 3, j = id >> 3;
  rest = j / per;
  tile = (id & 7) * per + j - rest * per;
  return tile < tiles;
}
int row_tile_workgroups(int64_t tiles, int64_t rest) { return (int)((tiles + 7) / 8 * 8 * rest); }

// The adapters of the four blocks from b, lane m's that of block b + m: 64 rows
// of the prefill kernels in one load.
__device__ __forceinline__ int four_adapters(const BlockArgs& a, int b, int lane) {
  return lane < 4 && b + lane < a.blocks ? a.bucket[b + lane] : -1;
}
// Past the blocks of adapter e among them, from block m on.
__device__ __forceinline__ int blocks_end(int adapters, int e, int m) {
  int n = m + 1;
  while (n < 4 && __builtin_amdgcn_readlane(adapters, n) == e) ++n;
  return n;
}
template <bool ROWS>
__device__ __forceinline__ int block_row(const BlockArgs& a, int b, int c) {
  if (ROWS) return c == 0 ? b : -1;
  const int sid = a.sorted[b * 16 + c];
  return sid < a.M ? sid : -1;
}

// ---------------------------------------------------------------------------
// Shrink.
// ---------------------------------------------------------------------------
struct ShrinkArgs {
  BlockArgs b;
  const void* x;
  const void* a;
  const int32_t* ranks;
  float* v;                   // [k-slices][positions][VR]
  uint32_t x_bytes, a_bytes;  // of x, and of one adapter's A (both below 2^31)
  int K, R;
  int rt;                     // rank tiles of 16 per part
  int tiles;                  // P * rt
  int VR;                     // 16 * tiles
  int steps, slices;          // k-steps, and into how many slices they are cut
  int row_tiles;              // groups of four blocks (prefill)
  int positions;              // rows of v
  int64_t v_slice;            // positions * VR
};

// Byte offset of the lane's row of A in rank tile q, at k = `k`; past the end for tiles that A lacks.
__device__ __forceinline__ uint32_t a_offset(const ShrinkArgs& a, int q, int i, int rank, int k) {
  const int p = q / a.rt, r = (q - p * a.rt) * 16 + i;
  return q < a.tiles && r < rank ? ((uint32_t)(p * a.R + r) * (uint32_t)a.K + (uint32_t)k) * 2u : kPastEnd;
}

// One rank tile of one block; a wave's share of the k-steps, one step ahead,
// straight from global memory: no other wave reads these k.  The waves of other
// workgroups fill the time.  Depths measured on this loop (layers of Qwen3-4B at
// 1 row / 32 rows unsorted / Llama-3-8B at 128 rows over 32 adapters of rank 64):
// one step ahead 263 / 424 / 484 us, two 266 / 435 / 491, three 270 / 444 / 500,
// five 275 / 460 / 513.  (The break between the two steps of its body gives the
// loop two ways back to its head, where the compiler waits for three of the four
// loads in flight: every second step starts nearly empty.  What a loop without
// it would gain from depth is not known.)
// Bound by the chain id -> weights -> sum for single rows (Qwen3-4B qkv, rank 16,
// 0.25 MB of A: 2.2 to 4.6 us under the profiler), by the loads of A for batches
// (Llama-3-8B qkv, 128 rows over 32 adapters of rank 64: 50 MB in 16 us, 3.1 TB/s).
// grid: (blocks, k-slices, rank tiles).
constexpr int kShrinkWaves = 4;

template <bool ROWS, typename DT>
__global__ __launch_bounds__(64 * kShrinkWaves) void lora_shrink_kernel(ShrinkArgs a) {
  using V8 = typename DT::vec8;
  constexpr int D = 2;
  __shared__ f32x4 red[kShrinkWaves * 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int i = lane & 15, g = lane >> 4;
  const int b = blockIdx.x, q = blockIdx.z;
  const int e = block_adapter<ROWS>(a.b, b);
  if (e < 0 || e >= a.b.L) return;
  const int sid = block_row<ROWS>(a.b, b, i);
  // A row block waits for the rank, to leave out what lies past it; a single
  // row reads it beside the weights (the expand takes no value past the rank).
  const int rank = ROWS ? a.R : min(load_uniform(a.ranks + e), a.R);
  const __amdgpu_buffer_rsrc_t ar = make_rsrc((const char*)a.a + (int64_t)e * a.a_bytes, a.a_bytes);
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, a.x_bytes);
  const uint32_t ao = a_offset(a, q, i, rank, 16 * g);
  const uint32_t xo = sid >= 0 ? ((uint32_t)sid * (uint32_t)a.K + 16u * g) * 2u : kPastEnd;
  // Slice (blockIdx.y, wave) of the k-steps.
  const int parts = gridDim.y * kShrinkWaves, part = blockIdx.y * kShrinkWaves + wave;
  const int s0 = (int)((int64_t)part * a.steps / parts), s1 = (int)((int64_t)(part + 1) * a.steps / parts);

  struct Stage {
    u32x4 a[2], x[2];
  };
  auto load = [&](Stage& st, int s) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // K is a multiple of 8, so a lane's vector lies in its row or past its end.
      const uint32_t dead = s < s1 && s * kStepK + 16 * g + 8 * h < a.K ? 0u : kPastEnd;
      st.a[h] = __builtin_amdgcn_raw_buffer_load_b128(ar, (ao + 16u * h) | dead, s * kStepK * 2, 0);
      st.x[h] = __builtin_amdgcn_raw_buffer_load_b128(xr, (xo + 16u * h) | dead, s * kStepK * 2, 0);
    }
  };
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  Stage st[D];
#pragma unroll
  for (int p = 0; p + 1 < D; ++p) load(st[p], s0 + p);
  for (int s = s0; s < s1;) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      load(st[(d + D - 1) % D], s + D - 1);
      __builtin_amdgcn_sched_barrier(0);  // the prefetch stays ahead of this step's math
#pragma unroll
      for (int h = 0; h < 2; ++h)
        acc = mfma16x16x32(__builtin_bit_cast(V8, st[d].a[h]), __builtin_bit_cast(V8, st[d].x[h]), acc);
      if (++s >= s1) break;
    }
  }
  // Sum over the waves; lane (row i, ranks 4 g .. 4 g + 3).
  red[wave * 64 + lane] = acc;
  __syncthreads();
  if (wave != 0 || sid < 0) return;  // (the expand reads no padding)
  f32x4 s = red[lane];
#pragma unroll
  for (int w = 1; w < kShrinkWaves; ++w) s += red[w * 64 + lane];
  *(f32x4*)(a.v + blockIdx.y * a.v_slice + (int64_t)(ROWS ? b : b * 16 + i) * a.VR + q * 16 + 4 * g) = s;
}

// Prefill: 64 rows (four blocks) and 64 RT ranks, the wave's RT rank tiles read
// straight into MFMA operands and the rows shared through a ring of LDS slots
// filled by LDS-DMA, whole 128-byte lines of a row at a time.  Blocks of
// different adapters in the four are taken in turn, the others' rows as zeros.
// 8192 rows over 8 adapters of rank 64, Llama-3-8B qkv / o / gate_up / down: 55 /
// 29 / 44 / 87 us, x at 1.2 to 2.7 TB/s.  Bound by the reads of A through L2,
// three times x's bytes for qkv's 192 ranks, and the wait for them at each step.
// grid: (groups of four blocks and k-slices, groups of 4 RT rank tiles).
constexpr int kShrinkRows = 64;
constexpr int shrink_slots(int rt) { return rt <= 2 ? 6 : 4; }

template <int RT, typename DT>
__global__ __launch_bounds__(64 * kLoraWaves) void lora_shrink_tile_kernel(ShrinkArgs a) {
  using V8 = typename DT::vec8;
  constexpr int SLOTS = shrink_slots(RT);
  constexpr int D = SLOTS - 1;              // steps in flight ahead of the multiply
  constexpr int VECS = kShrinkRows * 8;     // 16-byte vectors of a slot
  constexpr int LOADS = 2 + 2 * RT;         // a wave's loads of a step
  extern __shared__ u32x4 xs[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const int slice = blockIdx.x / a.row_tiles, tile = blockIdx.x - slice * a.row_tiles;
  const int q0 = (blockIdx.y * kLoraWaves + wave) * RT;
  const int s0 = (int)((int64_t)slice * a.steps / a.slices);
  const int s1 = (int)((int64_t)(slice + 1) * a.steps / a.slices);
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, a.x_bytes);
  // The DMA's lanes: row lane / 8 of eight, the vector that its place holds.
  const int kq = ((lane & 7) ^ (lane >> 3)) * 8;
  const int b0 = tile * 4, adapters = four_adapters(a.b, b0, lane);
  int sids[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int pos = b0 * 16 + (n * kLoraWaves + wave) * 8 + (lane >> 3);
    sids[n] = pos < a.positions ? a.b.sorted[pos] : -1;
  }
  for (int m0 = 0; m0 < 4;) {
    const int e = __builtin_amdgcn_readlane(adapters, m0);
    if (e < 0 || e >= a.b.L) break;  // none and past the end are the last ones
    const int m1 = blocks_end(adapters, e, m0);
    const int rank = min(load_uniform(a.ranks + e), a.R);
    const __amdgpu_buffer_rsrc_t ar = make_rsrc((const char*)a.a + (int64_t)e * a.a_bytes, a.a_bytes);
    uint32_t ao[RT], xo[2];
#pragma unroll
    for (int t = 0; t < RT; ++t) ao[t] = a_offset(a, q0 + t, c, rank, 8 * g);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int m = (n * kLoraWaves + wave) >> 1, sid = m >= m0 && m < m1 ? sids[n] : -1;
      xo[n] = sid >= 0 && sid < a.b.M ? ((uint32_t)sid * (uint32_t)a.K + (uint32_t)kq) * 2u : kPastEnd;
    }
    u32x4 aw[D + 1][RT][2];
    auto issue = [&](u32x4 (&w)[RT][2], int s, int slot) {
      const uint32_t dead = s < s1 && s * kStepK + kq < a.K ? 0u : kPastEnd;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        load_lds16(xr, xs + slot * VECS + (i * kLoraWaves + wave) * 64, xo[i] | dead, s * kStepK * 2);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t gone = s < s1 && s * kStepK + 32 * h + 8 * g < a.K ? 0u : kPastEnd;
#pragma unroll
        for (int t = 0; t < RT; ++t)
          w[t][h] = __builtin_amdgcn_raw_buffer_load_b128(ar, (ao[t] + 64u * h) | gone, s * kStepK * 2, 0);
      }
      stay_here();
    };
    f32x4 acc[RT][4];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int m = 0; m < 4; ++m) acc[t][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Step s: wait until its loads have landed (the D - 1 steps after it may be
    // in flight), meet the other waves -- all of it is in LDS then, and every
    // wave is done with the slot that step s + D takes -- and issue that one.
#pragma unroll
    for (int p = 0; p < D; ++p) issue(aw[p], s0 + p, p);
    for (int s = s0; s < s1; s += SLOTS) {  // (steps past the slice multiply zeros)
#pragma unroll
      for (int d = 0; d <= D; ++d) {
        __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm((D - 1) * LOADS));
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        issue(aw[(d + D) % (D + 1)], s + d + D, (d + D) % (D + 1));
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const V8 x = __builtin_bit_cast(V8, xs[d * VECS + (16 * m + c) * 8 + ((4 * h + g) ^ (c & 7))]);
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[t][m] = mfma16x16x32(__builtin_bit_cast(V8, aw[d][t][h]), x, acc[t][m]);
          }
      }
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    __syncthreads();  // before the ring is filled again
    float* v = a.v + slice * a.v_slice;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (m < m0 || m >= m1) continue;
#pragma unroll
      for (int t = 0; t < RT; ++t)
        if (q0 + t < a.tiles)
          *(f32x4*)(v + (int64_t)((b0 + m) * 16 + c) * a.VR + (q0 + t) * 16 + 4 * g) = acc[t][m];
    }
    m0 = m1;
  }
}

// ---------------------------------------------------------------------------
// v as MFMA operands.
//
// v enters the expand's MFMAs as a sum of values of the operand type, each the
// remainder of those before: three in bf16, which hold all 24 bits of the fp32
// sum, two in fp16, which hold 23 of them (down to 2^-39 of the row's largest).
// (Two in bf16 hold 16 bits: where B takes the difference of two sums, outputs
// were off by whole percents; of a qkv of 32 rows 5.9e-4 of the outputs rounded
// the other way than the exact value, with three terms 2.5e-5, in torch's fp32
// products 5.1e-5.)  A part's row is
// brought to a largest value in [2^14, 2^15) by a power of two first: fp16
// holds no more than 65504, and the remainders stay normal numbers.  A row with
// an infinity or NaN keeps those, and its finite values no longer count.
// ---------------------------------------------------------------------------
template <typename DT>
constexpr int kTerms = 3;
template <>
constexpr int kTerms<F16> = 2;

struct VArgs {
  const float* v;    // partial sums [slices][positions][VR]
  int64_t v_slice;
  int positions, slices, VR, rp;  // rp: ranks of a part in v, a multiple of 16
};

// The lane's row of a part: 8 consecutive ranks of each 32, the k-slices added in order.
template <int KC, int S>
__device__ __forceinline__ void load_v(const VArgs& a, int64_t pos, int part, int limit, int g, f32x4 (&v)[KC][2]) {
  const float* p = a.v + pos * a.VR + part * a.rp + 8 * g;
#pragma unroll
  for (int k = 0; k < KC; ++k) {
    v[k][0] = v[k][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (32 * k + 8 * g >= limit) continue;
    // Asked for ahead of the first sum.  The compiler keeps a branch for each
    // slice and waits at joins: up to 32 ranks of a block have all slices in
    // flight, further ranks and the prefill kernel's slices mostly come one after
    // the other, a single row's first slice by itself.
    f32x4 t[S][2];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < a.slices) {
        t[s][0] = *(const f32x4*)(p + s * a.v_slice + 32 * k);
        t[s][1] = *(const f32x4*)(p + s * a.v_slice + 32 * k + 4);
      }
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < a.slices) {
        v[k][0] += t[s][0];
        v[k][1] += t[s][1];
      }
    }
  }
}

// Its operands, and the exponent that brings the products back.
template <int KC, typename DT>
__device__ __forceinline__ int split_v(const f32x4 (&v)[KC][2], int rank, int g,
                                       typename DT::vec8 (&t)[kTerms<DT>][KC]) {
  using E = typename DT::elem;
  float f[KC][8], top = 0.f;
#pragma unroll
  for (int k = 0; k < KC; ++k)
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      f[k][w] = 32 * k + 8 * g + w < rank ? v[k][w >> 2][w & 3] : 0.f;
      top = f[k][w] != f[k][w] ? INFINITY : fmaxf(top, fabsf(f[k][w]));
    }
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  const bool finite = top < INFINITY;
  const int ex = finite ? __builtin_amdgcn_frexp_expf(top) - 15 : 128;
#pragma unroll
  for (int k = 0; k < KC; ++k)
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      float rest = __builtin_ldexpf(f[k][w], -ex);
#pragma unroll
      for (int i = 0; i < kTerms<DT>; ++i) {
        t[i][k][w] = (E)rest;
        rest = finite ? rest - (float)t[i][k][w] : 0.f;
      }
    }
  return ex;
}

// ---------------------------------------------------------------------------
// Expand.
// ---------------------------------------------------------------------------
struct ExpandArgs {
  BlockArgs b;
  VArgs v;
  const void* y;
  void* out;
  const void* w;    // B
  const float* scaling;
  const int32_t* ranks;
  uint32_t w_bytes;  // one adapter's B (below 2^31)
  int N, R;
  int inplace;       // out is y: rows without an adapter stay as they are
  int per;           // column steps of a group
  int groups;        // column groups
  int row_tiles;     // groups of four row blocks (prefill)
  int col[kLoraParts + 1];    // first column of each part
  int group[kLoraParts + 1];  // first column group of each part
};

// One wave's columns: 16 CT of each of H ranges (gate and up with an
// activation).  Column j of MFMA tile t of the group is column
// 32 (t / 2) + 8 (j / 4) + 4 (t % 2) + j % 4, so that lane (row, g) holds the 8
// columns from 8 g of every 32, and the four lanes of a row 64 bytes in a row.
template <int KC, int CT, int ACT, typename DT>
struct ExpandCols {
  using E = typename DT::elem;
  using V8 = typename DT::vec8;
  static constexpr int H = ACT == kActNone ? 1 : 2;
  static constexpr int VEC = CT / 2;  // 8-column vectors a lane holds in each range

  const ExpandArgs& a;
  int c, g, part, base, end, half, ncols;

  // Group `grp` of `per` times 16 CT columns.
  __device__ __forceinline__ ExpandCols(const ExpandArgs& args, int grp, int lane, int per)
      : a(args), c(lane & 15), g(lane >> 4), part(0) {
    if (H == 1)
      while (part + 1 < kLoraParts && grp >= a.group[part + 1]) ++part;
    base = a.col[part] + (grp - a.group[part]) * per * 16 * CT;
    end = a.col[part + 1];
    half = a.N >> 1;
    ncols = H == 1 ? a.N : half;
  }
  __device__ __forceinline__ int first(int q) const { return base + 32 * q + 8 * g; }
  // Column j of tile t, from the group's first.
  static __device__ __forceinline__ int column(int t, int j) { return 32 * (t >> 1) + 8 * (j >> 2) + 4 * (t & 1) + (j & 3); }

  __device__ __forceinline__ void load_y(int sid, u32x4 (&y)[H][VEC]) const {
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int q = 0; q < VEC; ++q) {
        y[h][q] = u32x4{0u, 0u, 0u, 0u};
        if (sid >= 0 && first(q) < end)
          y[h][q] = *(const u32x4*)((const E*)a.y + (int64_t)sid * a.N + h * half + first(q));
      }
  }

  // The columns' rows of adapter e's B, up to `limit` ranks.
  __device__ __forceinline__ void load_b(int e, int limit, u32x4 (&w)[H][CT][KC]) const {
    const __amdgpu_buffer_rsrc_t br = make_rsrc((const char*)a.w + (int64_t)e * a.w_bytes, a.w_bytes);
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        const int n = base + column(t, c);
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          const int r0 = 32 * k + 8 * g;
          const uint32_t off =
              n < end && r0 < limit ? ((uint32_t)(h * half + n) * (uint32_t)a.R + (uint32_t)r0) * 2u : kPastEnd;
          w[h][t][k] = __builtin_amdgcn_raw_buffer_load_b128(br, off, 0, 0);
        }
      }
  }

  // Zeros in place of what lies at and past the rank.
  __device__ __forceinline__ void cut(int rank, u32x4 (&w)[CT][KC]) const {
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      const int live = rank - (32 * k + 8 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t m = live >= 2 * i + 2 ? ~0u : live == 2 * i + 1 ? 0xFFFFu : 0u;
#pragma unroll
        for (int t = 0; t < CT; ++t) w[t][k][i] &= m;
      }
    }
  }

  // The smallest terms of v first.
  static __device__ __forceinline__ void mul(const u32x4 (&w)[CT][KC], const V8 (&v)[kTerms<DT>][KC],
                                             f32x4 (&acc)[CT]) {
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = kTerms<DT> - 1; i >= 0; --i)
#pragma unroll
      for (int k = 0; k < KC; ++k)
#pragma unroll
        for (int t = 0; t < CT; ++t) acc[t] = mfma16x16x32(__builtin_bit_cast(V8, w[t][k]), v[i][k], acc[t]);
  }

  // y plus f times the products, f the scaling and the power of two that
  // brings them back.
  __device__ __forceinline__ void combine(int q, const u32x4 (&y)[H][VEC], const f32x4 (&acc)[H][CT],
                                          const float (&f)[H], V8& r) const {

    const V8 y0 = __builtin_bit_cast(V8, y[0][q]), y1 = __builtin_bit_cast(V8, y[H - 1][q]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = 2 * q + (i >> 2);
      const float v = __builtin_fmaf(acc[0][t][i & 3], f[0], (float)y0[i]);
      if constexpr (ACT == kActNone)
        r[i] = (E)v;
      else
        r[i] = (E)(gated_act_fast(ACT, v) * __builtin_fmaf(acc[H - 1][t][i & 3], f[H - 1], (float)y1[i]));
    }
  }

  __device__ __forceinline__ void store(int sid, const u32x4 (&y)[H][VEC], const f32x4 (&acc)[H][CT],
                                        const float (&f)[H]) const {
#pragma unroll
    for (int q = 0; q < VEC; ++q) {
      V8 r;
      combine(q, y, acc, f, r);
      if (sid >= 0 && first(q) < end) *(V8*)((E*)a.out + (int64_t)sid * ncols + first(q)) = r;
    }
  }
};

// Few rows and batches: a wave is a row block and one or two column steps, v
// split by every wave for itself.  A single row's y and v are asked for first;
// the compiled code adds v's slices before it loads the id, and the weights
// follow that.  A block's y and weights go out ahead of its v, whose waits
// (load_v) take them in too; the second step's go out ahead of the first one's
// stores.
// Bound by that chain for single rows (Qwen3-4B gate_up, rank 16, silu: 4.7 us
// under the profiler); for batches by it and by the waves that the operands'
// registers leave room for (Llama-3-8B gate_up, 128 rows over 32 adapters of
// rank 64: 128 MB in 34.8 us, 3.7 TB/s).
template <bool ROWS, int KC, int CT, int ACT, typename DT>
__global__ __launch_bounds__(64 * kLoraWaves, KC > 2 ? 1 : ROWS || KC == 1 ? 4 : 3) void lora_expand_kernel(ExpandArgs a) {
  using Cols = ExpandCols<KC, CT, ACT, DT>;
  constexpr int H = Cols::H;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // Column groups fastest: neighbours read and write one row's neighbouring columns.
  const int wgs = (a.groups + kLoraWaves - 1) / kLoraWaves;
  const int b = blockIdx.x / wgs, grp = (blockIdx.x - b * wgs) * kLoraWaves + wave;
  if (grp >= a.groups) return;
  Cols cols(a, grp, lane, ROWS ? 1 : a.per);
  u32x4 y[H][Cols::VEC];
  f32x4 v[H][KC][2];
  if (ROWS) {
    cols.load_y(block_row<true>(a.b, b, cols.c), y);
#pragma unroll
    for (int h = 0; h < H; ++h) load_v<KC, kLoraSlices>(a.v, b, H == 1 ? cols.part : h, a.R, cols.g, v[h]);
  }
  const int e = block_adapter<ROWS>(a.b, b);
  if (e < 0) return;  // past the last block
  const bool adapter = e < a.b.L;
  if (!adapter && H == 1 && a.inplace) return;
  const int sid = block_row<ROWS>(a.b, b, cols.c);
  u32x4 w[H][CT][KC];
  if (ROWS && adapter) cols.load_b(e, a.R, w);
  if (!ROWS) cols.load_y(sid, y);
  const int rank = adapter ? min(load_uniform(a.ranks + e), a.R) : 0;
  const float scale = adapter ? load_uniform(a.scaling + e) : 0.f;
  if (!ROWS && adapter) cols.load_b(e, rank, w);
  typename DT::vec8 vt[H][kTerms<DT>][KC];
  float f[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    // Padding rows take none: with all 16 rows v was more bytes than B.
    if (!ROWS)
      load_v<KC, kLoraSlices>(a.v, b * 16 + cols.c, H == 1 ? cols.part : h, sid >= 0 ? rank : 0, cols.g, v[h]);
    f[h] = __builtin_ldexpf(scale, split_v<KC, DT>(v[h], rank, cols.g, vt[h]));
  }
  for (int s = 0;;) {
    f32x4 acc[H][CT];
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[h][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (adapter) {
        if ((ROWS && rank < a.R) || (rank & 7)) cols.cut(rank, w[h]);
        Cols::mul(w[h], vt[h], acc[h]);
      }
    }
    const bool more = !ROWS && ++s < a.per && cols.base + 16 * CT < cols.end;
    if (!more) {
      cols.store(sid, y, acc, f);
      return;
    }
    cols.base += 16 * CT;
    if (adapter) cols.load_b(e, rank, w);
    __builtin_amdgcn_sched_barrier(0);
    cols.base -= 16 * CT;
    cols.store(sid, y, acc, f);
    cols.base += 16 * CT;
    cols.load_y(sid, y);
  }
}

// Prefill: a workgroup is four row blocks, one a wave, and `per` steps of 64
// columns (32 gate and their 32 up ones).  A wave's v becomes MFMA operands
// once; the columns' rows of B come through a ring of LDS slots filled by
// LDS-DMA, shared by the waves, and y into registers, both issued D steps ahead.
// (The wait leaves room for D - 1 steps' loads; the stores in between count among
// them, so that it takes in the next step's loads too, half of them with an
// activation.)  Blocks of different adapters in the four are taken in turn.  Bound
// by reading y and writing the output, and by each workgroup's start, most of it
// v's slices one after the other (load_v): 8192 rows of rank 64, bf16, Llama-3-8B
// gate_up with silu 246 us for 705 MB, 2.9 TB/s; qkv 84 us, o 52 us.
constexpr int kExpandSlots = 4;

// Waves a SIMD: with three terms of 64 ranks two, since three spill 8 to 9
// registers (8192 rows of a Llama-3-8B layer, bf16, rank 64: 635 us against 661).
constexpr int expand_tile_waves(int kc, int terms) { return kc * terms <= 4 ? 3 : kc <= 2 ? 2 : 1; }

template <int KC, int ACT, typename DT>
__global__ __launch_bounds__(64 * kLoraWaves, expand_tile_waves(KC, kTerms<DT>)) void lora_expand_tile_kernel(ExpandArgs a) {
  constexpr int CT = kLoraColTiles / (ACT == kActNone ? 1 : 2);
  using Cols = ExpandCols<KC, CT, ACT, DT>;
  using V8 = typename DT::vec8;
  constexpr int H = Cols::H, VEC = Cols::VEC;
  constexpr int D = kExpandSlots - 1;
  constexpr int PL = 4 * KC;              // 16-byte places of a column in a slot
  constexpr int VECS = 64 * PL;           // ... and of a slot
  constexpr int LOADS = KC + H * VEC;     // a wave's loads of a step
  extern __shared__ u32x4 bs[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int tile, chunk;
  if (!row_tile(blockIdx.x, a.row_tiles, tile, chunk)) return;
  const int b0 = tile * 4;
  Cols cols(a, chunk, lane, a.per);
  const int c = cols.c, g = cols.g, base = cols.base;
  const int steps = min(a.per, (cols.end - base + 16 * CT - 1) / (16 * CT));
  // Place p of slot row r holds the vector p ^ swap(r) of its column: reads of
  // one vector of 8 rows meet all banks.
  auto swap = [](int r) { return KC == 1 ? (r >> 1) & 3 : r & 7; };
  // What does not hang on the adapter is loaded beside it.
  const int adapters = four_adapters(a.b, b0, lane);
  const int pos = (b0 + wave) * 16 + c;
  const bool have = pos < a.v.positions;
  const int mine = have ? a.b.sorted[pos] : -1;
  V8 vt[H][kTerms<DT>][KC];
  float f[H];
  {
    f32x4 v[H][KC][2];
#pragma unroll
    for (int h = 0; h < H; ++h) load_v<KC, kTileSlices>(a.v, have ? pos : 0, H == 1 ? cols.part : h, a.R, g, v[h]);
    const int e = __builtin_amdgcn_readlane(adapters, wave);  // of the wave's own block
    const bool adapter = e >= 0 && e < a.b.L;
    const int rank = adapter ? min(load_uniform(a.ranks + e), a.R) : 0;
    const float scale = adapter ? load_uniform(a.scaling + e) : 0.f;
#pragma unroll
    for (int h = 0; h < H; ++h) f[h] = __builtin_ldexpf(scale, split_v<KC, DT>(v[h], rank, g, vt[h]));
  }

  for (int m0 = 0; m0 < 4;) {
    const int e = __builtin_amdgcn_readlane(adapters, m0);
    if (e < 0) break;  // past the last block
    const bool adapter = e < a.b.L;
    if (!adapter && H == 1 && a.inplace) break;  // the rows without an adapter are the last ones
    const int m1 = blocks_end(adapters, e, m0);
    const int sid = wave >= m0 && wave < m1 && mine < a.b.M ? mine : -1;
    const int rank = adapter ? min(load_uniform(a.ranks + e), a.R) : 0;
    const __amdgpu_buffer_rsrc_t br = make_rsrc((const char*)a.w + (int64_t)(adapter ? e : 0) * a.w_bytes, a.w_bytes);

    // The wave's places in a slot, and what it fills them with at step 0.
    uint32_t bo[KC];
    int bn0[KC];
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      const int u = (k * kLoraWaves + wave) * 64 + lane, r = u / PL, i = r & 15, t = r >> 4;
      const int r0 = ((u % PL) ^ swap(r)) * 8;
      bn0[k] = base + Cols::column(t % CT, i);
      bo[k] = r0 < rank ? ((uint32_t)(t / CT * cols.half + bn0[k]) * (uint32_t)a.R + (uint32_t)r0) * 2u : kPastEnd;
    }
    const typename DT::elem* yrow = (const typename DT::elem*)a.y + (int64_t)max(sid, 0) * a.N;
    u32x4 y[D + 1][H][VEC];
    auto issue = [&](u32x4 (&v)[H][VEC], int s, int slot) {
#pragma unroll
      for (int k = 0; k < KC; ++k) {
        const uint32_t dead = bn0[k] + s * 16 * CT < cols.end ? 0u : kPastEnd;
        load_lds16(br, bs + slot * VECS + (k * kLoraWaves + wave) * 64, bo[k] | dead, s * 16 * CT * a.R * 2);
      }
      __builtin_amdgcn_sched_barrier(0);
      // Past the last column the lane's loads repeat it, so that every wave counts the same loads.
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int q = 0; q < VEC; ++q)
          v[h][q] = *(const u32x4*)(yrow + h * cols.half + min(base + s * 16 * CT + 32 * q + 8 * g, cols.end - 8));
      stay_here();
    };
#pragma unroll
    for (int p = 0; p < D; ++p) issue(y[p], p, p);
    // Step s: wait until its loads have landed (with no stores between, those of
    // the D - 1 steps after it may be in flight), meet the other waves and issue
    // step s + D into the slot that every wave is done with.  Steps past the last
    // store nothing.
    for (int s0 = 0; s0 < steps; s0 += kExpandSlots) {
#pragma unroll
      for (int d = 0; d <= D; ++d) {
        const int s = s0 + d;
        __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm((D - 1) * LOADS));
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        issue(y[(d + D) % (D + 1)], s + D, (d + D) % (D + 1));
        f32x4 acc[H][CT];
#pragma unroll
        for (int h = 0; h < H; ++h) {
          u32x4 w[CT][KC];
#pragma unroll
          for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int k = 0; k < KC; ++k)
              w[t][k] = bs[d * VECS + ((h * CT + t) * 16 + c) * PL + ((4 * k + g) ^ swap(c))];
          if (rank & 7) cols.cut(rank, w);
          Cols::mul(w, vt[h], acc[h]);
        }
        cols.base = base + s * 16 * CT;
        cols.store(sid, y[d], acc, f);
      }
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    __syncthreads();  // before the ring is filled again
    m0 = m1;
  }
}

template <int KC, int ACT, typename DT>
hipError_t launch_expand(const ExpandArgs& a, int mode, hipStream_t s) {
  constexpr int CT = kLoraColTiles / (ACT == kActNone ? 1 : 2);
  const dim3 block(64 * kLoraWaves);
  if constexpr (KC <= 4) {
    if (mode == kLoraTiles) {
      constexpr int lds = kExpandSlots * 64 * 4 * KC * 16;
      hipLaunchKernelGGL((lora_expand_tile_kernel<KC, ACT, DT>),
                         dim3((unsigned)row_tile_workgroups(a.row_tiles, a.groups)), block, lds, s, a);
      return hipGetLastError();
    }
  }
  const dim3 grid((unsigned)((a.groups + kLoraWaves - 1) / kLoraWaves * a.b.blocks));
  if (mode == kLoraRows)
    hipLaunchKernelGGL((lora_expand_kernel<true, KC, CT, ACT, DT>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((lora_expand_kernel<false, KC, CT, ACT, DT>), grid, block, 0, s, a);
  return hipGetLastError();
}

template <int KC, typename DT>
hipError_t launch_expand_act(const ExpandArgs& a, int mode, int act, hipStream_t s) {
  if (act == kActSilu) return launch_expand<KC, kActSilu, DT>(a, mode, s);
  if (act == kActGelu) return launch_expand<KC, kActGelu, DT>(a, mode, s);
  return launch_expand<KC, kActNone, DT>(a, mode, s);
}

template <typename DT>
hipError_t launch_shrink(const ShrinkArgs& a, const LoraPlan& p, hipStream_t s) {
  const dim3 block(64 * kLoraWaves);
  const unsigned ks = (unsigned)p.slices;
  if (p.mode != kLoraTiles) {
    const dim3 grid((unsigned)p.blocks, ks, (unsigned)a.tiles);
    if (p.mode == kLoraRows)
      hipLaunchKernelGGL((lora_shrink_kernel<true, DT>), grid, dim3(64 * kShrinkWaves), 0, s, a);
    else
      hipLaunchKernelGGL((lora_shrink_kernel<false, DT>), grid, dim3(64 * kShrinkWaves), 0, s, a);
    return hipGetLastError();
  }
  const int rt = p.rank_tiles;
  const dim3 grid((unsigned)(a.row_tiles * p.slices),
                  (unsigned)((a.tiles + kLoraWaves * rt - 1) / (kLoraWaves * rt)));
#define SGL_TILE(RT_) \
  if (rt == RT_)      \
  hipLaunchKernelGGL((lora_shrink_tile_kernel<RT_, DT>), grid, block, shrink_slots(RT_) * kShrinkRows * 128, s, a)
  SGL_TILE(1);
  SGL_TILE(2);
  SGL_TILE(3);
  SGL_TILE(4);
#undef SGL_TILE
  return hipGetLastError();
}

}  // namespace

LoraPlan plan_lora(int64_t M, int64_t N, int64_t K, int64_t L, int64_t R, int parts, bool routed) {
  LoraPlan p{};
  const int cus = device_cu_count();
  const int tiles = parts * (int)((R + 15) / 16);
  // (Ranks beyond 128 leave the prefill kernels too few registers.)
  p.mode = !routed ? kLoraRows : M < lora_tile_rows(R) || R > 128 ? kLoraBlocks : kLoraTiles;
  const int64_t cap = moe_sorted_capacity(M, L + 1, kLoraBlock);
  // A block holds a row at least.
  p.blocks = routed ? std::min(moe_block_capacity(M, L + 1, kLoraBlock), M) : M;
  p.positions = routed ? cap : M;
  p.rank_tiles = p.mode == kLoraTiles ? std::min(4, (tiles + kLoraWaves - 1) / kLoraWaves) : 1;
  const int per = p.mode == kLoraTiles ? kLoraWaves * p.rank_tiles : 1;
  const int64_t wgs = (int64_t)((tiles + per - 1) / per) * (p.mode == kLoraTiles ? (p.blocks + 3) / 4 : p.blocks);
  const int64_t steps = (K + kStepK - 1) / kStepK;
  // Two workgroups a CU, and eight (tiles) or two steps a wave at least.
  const bool tile = p.mode == kLoraTiles;
  p.slices = (int)std::max<int64_t>(
      1, std::min<int64_t>({tile ? kTileSlices : kLoraSlices, steps / (tile ? 8 : 2 * kShrinkWaves),
                            (2 * cus + wgs - 1) / wgs}));
  p.per = 1;
  // Two column steps for each split of v once there are four waves a SIMD with
  // one step each (a projection alone, both steps of it; one / two / three steps,
  // us: rank 64, N = 28672 gated, 64 rows over 8 adapters 32.4 / 22.9 / 24.4, 128
  // over 32 58.3 / 48.5 / 48.1; N = 6144 128 over 32 21.8 / 21.8 / 23.5, 64 over 8
  // 13.2 / 14.3 / 15.7; rank 16, N = 4096, 40 rows over 4 9.2 / 10.0 / 10.6).
  if (p.mode == kLoraBlocks && p.blocks * N / (16 * kLoraColTiles) >= 16 * cus) p.per = 2;
  if (p.mode == kLoraTiles) {
    // A workgroup waits for its rows, v and the first columns once (as long as
    // 5 to 8 steps take) however many steps it has, so they are many, as far as
    // two workgroups a CU remain (8192 rows, rank 64, N = 6144 / 4096 / 28672
    // gated: 24 steps 72 / 52 / 228 us, 16 71 / 51 / 243, 8 75 / 52 / 304).
    const int64_t row_tiles = (p.blocks + 3) / 4;
    for (p.per = 24; p.per > 4 && row_tiles * ((N + 64 * p.per - 1) / (64 * p.per)) < 2 * cus;) p.per -= 4;
  }
  p.ws_bytes = (int64_t)p.slices * p.positions * tiles * 16 * 4;
  return p;
}

hipError_t launch_lora(const LoraParams& p, hipStream_t s) {
  const LoraPlan plan = plan_lora(p.M, p.N, p.K, p.L, p.R, p.parts, p.sorted != nullptr);
  const int rt = (int)((p.R + 15) / 16), tiles = p.parts * rt;
  ShrinkArgs a{};
  a.b.ids = p.ids;
  a.b.sorted = p.sorted;
  a.b.bucket = p.bucket;
  a.b.M = (int)p.M;
  a.b.L = (int)p.L;
  a.b.blocks = (int)plan.blocks;
  a.x = p.x;
  a.a = p.a;
  a.ranks = p.ranks;
  a.v = (float*)p.ws;
  a.x_bytes = (uint32_t)(p.M * p.K * 2);
  a.a_bytes = (uint32_t)(p.parts * p.R * p.K * 2);
  a.K = (int)p.K;
  a.R = (int)p.R;
  a.rt = rt;
  a.tiles = tiles;
  a.VR = 16 * tiles;
  a.steps = (int)((p.K + kStepK - 1) / kStepK);
  a.slices = plan.slices;
  a.row_tiles = (int)((plan.blocks + 3) / 4);
  a.positions = (int)plan.positions;
  a.v_slice = plan.positions * a.VR;
  const hipError_t st = p.dtype == 0 ? launch_shrink<F16>(a, plan, s) : launch_shrink<BF16>(a, plan, s);
  if (st != hipSuccess) return st;

  ExpandArgs x{};
  x.b = a.b;
  x.v.v = a.v;
  x.v.v_slice = a.v_slice;
  x.v.positions = (int)plan.positions;
  x.v.slices = plan.slices;
  x.v.VR = a.VR;
  x.v.rp = 16 * rt;
  x.y = p.y;
  x.out = p.out;
  x.w = p.b;
  x.scaling = p.scaling;
  x.ranks = p.ranks;
  x.w_bytes = (uint32_t)(p.N * p.R * 2);
  x.N = (int)p.N;
  x.R = a.R;
  x.per = plan.per;
  x.inplace = p.out == p.y;
  x.row_tiles = a.row_tiles;
  const int cols = plan.per * 16 * kLoraColTiles / (p.act ? 2 : 1);
  for (int i = 0, c = 0, n = 0; i <= kLoraParts; ++i) {
    // With an activation the groups cover the gate half and its up columns.
    const int width = i < p.parts ? (int)p.part_cols[i] : 0;
    x.col[i] = c;
    x.group[i] = n;
    if (p.act && i > 0) continue;
    c += width;
    n += (width + cols - 1) / cols;
    x.groups = n;
  }
#define SGL_KC(KC_) \
  (p.dtype == 0 ? launch_expand_act<KC_, F16>(x, plan.mode, p.act, s) : launch_expand_act<KC_, BF16>(x, plan.mode, p.act, s))
  if (p.R <= 32) return SGL_KC(1);
  if (p.R <= 64) return SGL_KC(2);
  if (p.R <= 128) return SGL_KC(4);
  return SGL_KC(8);
#undef SGL_KC
}

}  // namespace sgl_awq
