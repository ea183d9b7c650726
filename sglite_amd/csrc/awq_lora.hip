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
//              nothing is sorted, and a kernel waits for two loads in a row
//              (id, then weights) and no more
//   batches    16-row blocks of the sorted table
//   prefill    64-row tiles through LDS in the shrink, and v split once into
//              MFMA operands by a launch of its own, not by every column group
#include <math.h>

#include <algorithm>

#include "awq_buffer.h"
#include "awq_epilogue.h"
#include "awq_launch.h"

namespace sgl_awq {

namespace {

constexpr int kLoraWaves = 4;
constexpr int kStepK = 64;  // k per step of the shrink: 128 bytes of a row

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
  if (!ROWS) return a.bucket[b];
  const int e = a.ids[b];
  return e >= 0 && e < a.L ? e : a.L;
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
  int steps;                  // k-steps
  int64_t v_slice;            // positions * VR
};

// Byte offset of the lane's row of A in rank tile q, at k = `k`; past the end for tiles that A lacks.
__device__ __forceinline__ uint32_t a_offset(const ShrinkArgs& a, int q, int i, int rank, int k) {
  const int p = q / a.rt, r = (q - p * a.rt) * 16 + i;
  return q < a.tiles && r < rank ? ((uint32_t)(p * a.R + r) * (uint32_t)a.K + (uint32_t)k) * 2u : kPastEnd;
}

// One rank tile of one block; a wave's share of the k-steps with D - 1 of them
// in flight, straight from global memory: no other wave reads these k.
// grid: (blocks, k-slices, rank tiles).
template <bool ROWS, typename DT>
__global__ __launch_bounds__(64 * kLoraWaves) void lora_shrink_kernel(ShrinkArgs a) {
  using V8 = typename DT::vec8;
  constexpr int D = 4;
  __shared__ f32x4 red[kLoraWaves * 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int i = lane & 15, g = lane >> 4;
  const int b = blockIdx.x, q = blockIdx.z;
  const int e = block_adapter<ROWS>(a.b, b);
  if (e < 0 || e >= a.b.L) return;
  const int sid = block_row<ROWS>(a.b, b, i);
  // A row block waits for the rank, to leave out what lies past it; a single
  // row reads it beside the weights (the expand takes no value past the rank).
  const int rank = ROWS ? a.R : min(a.ranks[e], a.R);
  const __amdgpu_buffer_rsrc_t ar = make_rsrc((const char*)a.a + (int64_t)e * a.a_bytes, a.a_bytes);
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, a.x_bytes);
  const uint32_t ao = a_offset(a, q, i, rank, 16 * g);
  const uint32_t xo = sid >= 0 ? ((uint32_t)sid * (uint32_t)a.K + 16u * g) * 2u : kPastEnd;
  // Slice (blockIdx.y, wave) of the k-steps.
  const int parts = gridDim.y * kLoraWaves, part = blockIdx.y * kLoraWaves + wave;
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
  if (wave != 0 || (ROWS && i != 0)) return;
  f32x4 s = red[lane];
#pragma unroll
  for (int w = 1; w < kLoraWaves; ++w) s += red[w * 64 + lane];
  *(f32x4*)(a.v + blockIdx.y * a.v_slice + (int64_t)(ROWS ? b : b * 16 + i) * a.VR + q * 16 + 4 * g) = s;
}

// Prefill: 64 rows (four blocks) and 64 RT ranks, the wave's RT rank tiles read
// straight into MFMA operands and the rows shared through a ring of LDS slots
// filled by LDS-DMA, whole 128-byte lines of a row at a time.  Blocks of
// different adapters in the four are taken in turn, the others' rows as zeros.
// grid: (groups of four blocks, k-slices, groups of 4 RT rank tiles).
constexpr int kShrinkRows = 64;
constexpr int kShrinkSlots = 4;

template <int RT, typename DT>
__global__ __launch_bounds__(64 * kLoraWaves) void lora_shrink_tile_kernel(ShrinkArgs a) {
  using V8 = typename DT::vec8;
  constexpr int D = kShrinkSlots - 1;       // steps in flight ahead of the multiply
  constexpr int VECS = kShrinkRows * 8;     // 16-byte vectors of a slot
  constexpr int LOADS = 2 + 2 * RT;         // a wave's loads of a step
  extern __shared__ u32x4 xs[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const int q0 = (blockIdx.z * kLoraWaves + wave) * RT;
  const int s0 = (int)((int64_t)blockIdx.y * a.steps / gridDim.y);
  const int s1 = (int)((int64_t)(blockIdx.y + 1) * a.steps / gridDim.y);
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, a.x_bytes);
  // The DMA's lanes: row lane / 8 of eight, the vector that its place holds.
  const int kq = ((lane & 7) ^ (lane >> 3)) * 8;
  const int b1 = min((int)(blockIdx.x + 1) * 4, a.b.blocks);
  for (int b = blockIdx.x * 4; b < b1;) {
    const int e = a.b.bucket[b];
    if (e < 0 || e >= a.b.L) break;  // none and past the end are the last ones
    int bn = b + 1;
    while (bn < b1 && a.b.bucket[bn] == e) ++bn;
    const int rank = min(a.ranks[e], a.R);
    const __amdgpu_buffer_rsrc_t ar = make_rsrc((const char*)a.a + (int64_t)e * a.a_bytes, a.a_bytes);
    uint32_t ao[RT], xo[2];
#pragma unroll
    for (int t = 0; t < RT; ++t) ao[t] = a_offset(a, q0 + t, c, rank, 8 * g);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int pos = blockIdx.x * kShrinkRows + (n * kLoraWaves + wave) * 8 + (lane >> 3);
      const int sid = pos >= 16 * b && pos < 16 * bn ? a.b.sorted[pos] : -1;
      xo[n] = sid >= 0 && sid < a.b.M ? ((uint32_t)sid * (uint32_t)a.K + (uint32_t)kq) * 2u : kPastEnd;
    }
    u32x4 aw[D + 1][RT][2];
    auto issue = [&](u32x4 (&w)[RT][2], int s, int slot) {
      const uint32_t dead = s < s1 && s * kStepK + kq < a.K ? 0u : kPastEnd;
#pragma unroll
      for (int n = 0; n < 2; ++n)
        load_lds16(xr, xs + slot * VECS + (n * kLoraWaves + wave) * 64, xo[n] | dead, s * kStepK * 2);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t gone = s < s1 && s * kStepK + 32 * h + 8 * g < a.K ? 0u : kPastEnd;
#pragma unroll
        for (int t = 0; t < RT; ++t)
          w[t][h] = __builtin_amdgcn_raw_buffer_load_b128(ar, (ao[t] + 64u * h) | gone, s * kStepK * 2, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
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
    [&] {
      for (int s = s0;;) {
#pragma unroll
        for (int d = 0; d <= D; ++d) {
          __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm((D - 1) * LOADS));
          __builtin_amdgcn_s_barrier();
          __builtin_amdgcn_sched_barrier(0);
          issue(aw[(d + D) % (D + 1)], s + D, (d + D) % (D + 1));
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const V8 x = __builtin_bit_cast(V8, xs[d * VECS + (16 * m + c) * 8 + ((4 * h + g) ^ (c & 7))]);
#pragma unroll
              for (int t = 0; t < RT; ++t) acc[t][m] = mfma16x16x32(__builtin_bit_cast(V8, aw[d][t][h]), x, acc[t][m]);
            }
          if (++s >= s1) return;
        }
      }
    }();
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    __syncthreads();  // before the ring is filled again
    float* v = a.v + blockIdx.y * a.v_slice;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int blk = blockIdx.x * 4 + m;
      if (blk < b || blk >= bn) continue;
#pragma unroll
      for (int t = 0; t < RT; ++t)
        if (q0 + t < a.tiles) *(f32x4*)(v + (int64_t)(blk * 16 + c) * a.VR + (q0 + t) * 16 + 4 * g) = acc[t][m];
    }
    b = bn;
  }
}

// ---------------------------------------------------------------------------
// v as MFMA operands.
//
// v enters the expand's MFMAs as two values of the operand type, the second
// the first one's remainder: together 22 (fp16) or 16 (bf16) bits of the row's
// largest, so that the rounding stays far below the output's.  A part's row is
// brought to a largest value in [2^14, 2^15) by a power of two first: fp16
// holds no more than 65504, and the remainders stay normal numbers.  A row with
// an infinity or NaN keeps those, and its finite values no longer count.
// ---------------------------------------------------------------------------
struct VArgs {
  const float* v;    // partial sums [slices][positions][VR]
  int64_t v_slice;
  int slices, VR, rp;  // rp: ranks of a part in v, a multiple of 16
};

// The lane's row of a part: 8 consecutive ranks of each 32, the k-slices added in order.
template <int KC>
__device__ __forceinline__ void load_v(const VArgs& a, int64_t pos, int part, int limit, int g, f32x4 (&v)[KC][2]) {
  const float* p = a.v + pos * a.VR + part * a.rp + 8 * g;
#pragma unroll
  for (int k = 0; k < KC; ++k) {
    v[k][0] = v[k][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (32 * k + 8 * g >= limit) continue;
    for (int s = 0; s < a.slices; ++s) {
      v[k][0] += *(const f32x4*)(p + s * a.v_slice + 32 * k);
      v[k][1] += *(const f32x4*)(p + s * a.v_slice + 32 * k + 4);
    }
  }
}

// Its operands, and the exponent that brings the products back.
template <int KC, typename DT>
__device__ __forceinline__ int split_v(const f32x4 (&v)[KC][2], int rank, int g, typename DT::vec8 (&hi)[KC],
                                       typename DT::vec8 (&lo)[KC]) {
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
      const float t = __builtin_ldexpf(f[k][w], -ex);
      hi[k][w] = (E)t;
      lo[k][w] = finite ? (E)(t - (float)hi[k][w]) : (E)0.f;
    }
  return ex;
}

// Prefill: the operands of every block and part, once.  One wave each:
// vs[(block P + part) KC + k][hi, lo][lane], ve[(block P + part) 16 + row].
struct SplitArgs {
  BlockArgs b;
  VArgs v;
  const int32_t* ranks;
  u32x4* vs;
  int32_t* ve;
  int P, R;
};

template <int KC, typename DT>
__global__ __launch_bounds__(64 * kLoraWaves) void lora_split_kernel(SplitArgs a) {
  const int unit = blockIdx.x * kLoraWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int b = unit / a.P, p = unit - b * a.P, c = lane & 15, g = lane >> 4;
  if (b >= a.b.blocks) return;
  const int e = a.b.bucket[b];
  if (e < 0 || e >= a.b.L) return;
  const int rank = min(a.ranks[e], a.R);
  f32x4 v[KC][2];
  typename DT::vec8 hi[KC], lo[KC];
  load_v<KC>(a.v, b * 16 + c, p, rank, g, v);
  const int ex = split_v<KC, DT>(v, rank, g, hi, lo);
#pragma unroll
  for (int k = 0; k < KC; ++k) {
    a.vs[((int64_t)unit * KC + k) * 128 + lane] = __builtin_bit_cast(u32x4, hi[k]);
    a.vs[((int64_t)unit * KC + k) * 128 + 64 + lane] = __builtin_bit_cast(u32x4, lo[k]);
  }
  if (g == 0) a.ve[unit * 16 + c] = ex;
}

// ---------------------------------------------------------------------------
// Expand.
// ---------------------------------------------------------------------------
struct ExpandArgs {
  BlockArgs b;
  VArgs v;
  const u32x4* vs;  // operands from lora_split_kernel (prefill)
  const int32_t* ve;
  const void* y;
  void* out;
  const void* w;    // B
  const float* scaling;
  const int32_t* ranks;
  uint32_t w_bytes;  // one adapter's B (below 2^31)
  int N, R, P;
  int per;           // row blocks that a workgroup takes in turn
  int inplace;       // out is y: rows without an adapter stay as they are
  int groups;        // column groups
  int col[kLoraParts + 1];    // first column of each part
  int group[kLoraParts + 1];  // first column group of each part
};

// One wave's columns: 16 CT of each of H ranges (gate and up with an
// activation).  Column j of MFMA tile t of the group is column
// 4 CT (j / 4) + 4 t + j % 4, so that lane (row, g) holds 4 CT consecutive
// columns of its row.
template <int KC, int CT, int ACT, typename DT>
struct ExpandCols {
  using E = typename DT::elem;
  using V8 = typename DT::vec8;
  static constexpr int H = ACT == kActNone ? 1 : 2;
  static constexpr int VEC = CT / 2;  // 8-column vectors a lane holds in each range

  const ExpandArgs& a;
  int c, g, part, base, end, half, ncols;

  __device__ __forceinline__ ExpandCols(const ExpandArgs& args, int grp, int lane)
      : a(args), c(lane & 15), g(lane >> 4), part(0) {
    if (H == 1)
      while (part + 1 < kLoraParts && grp >= a.group[part + 1]) ++part;
    base = a.col[part] + (grp - a.group[part]) * 16 * CT;
    end = a.col[part + 1];
    half = a.N >> 1;
    ncols = H == 1 ? a.N : half;
  }
  __device__ __forceinline__ int first(int q) const { return base + 4 * CT * g + 8 * q; }

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
        const int n = base + 4 * CT * (c >> 2) + 4 * t + (c & 3);
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
  __device__ __forceinline__ void cut_b(int rank, u32x4 (&w)[H][CT][KC]) const {
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      const int live = rank - (32 * k + 8 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t m = live >= 2 * i + 2 ? ~0u : live == 2 * i + 1 ? 0xFFFFu : 0u;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int t = 0; t < CT; ++t) w[h][t][k][i] &= m;
      }
    }
  }

  static __device__ __forceinline__ void mul(const u32x4 (&w)[CT][KC], const V8 (&hi)[KC], const V8 (&lo)[KC],
                                             f32x4 (&acc)[CT]) {
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KC; ++k)
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[t] = mfma16x16x32(__builtin_bit_cast(V8, w[t][k]), lo[k], acc[t]);
#pragma unroll
    for (int k = 0; k < KC; ++k)
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[t] = mfma16x16x32(__builtin_bit_cast(V8, w[t][k]), hi[k], acc[t]);
  }

  // Bring the products back and scale them.
  static __device__ __forceinline__ void scale(f32x4 (&acc)[CT], int ex, float s) {
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][i] = __builtin_ldexpf(acc[t][i], ex) * s;
  }

  __device__ __forceinline__ void store(int sid, const u32x4 (&y)[H][VEC], const f32x4 (&acc)[H][CT]) const {
#pragma unroll
    for (int q = 0; q < VEC; ++q) {
      V8 r;
      const V8 y0 = __builtin_bit_cast(V8, y[0][q]), y1 = __builtin_bit_cast(V8, y[H - 1][q]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = 2 * q + (i >> 2);
        const float f = (float)y0[i] + acc[0][t][i & 3];
        if constexpr (ACT == kActNone)
          r[i] = (E)f;
        else
          r[i] = (E)(gated_act_fast(ACT, f) * ((float)y1[i] + acc[H - 1][t][i & 3]));
      }
      if (sid >= 0 && first(q) < end) *(V8*)((E*)a.out + (int64_t)sid * ncols + first(q)) = r;
    }
  }
};

// Few rows and batches: row block after row block, v split by every wave for
// itself.  A single row's loads go out beside its id as far as they do not
// hang on it: v's partial sums and y; the weights follow the id alone.
template <bool ROWS, int KC, int CT, int ACT, typename DT>
__global__ __launch_bounds__(64 * kLoraWaves) void lora_expand_kernel(ExpandArgs a) {
  using Cols = ExpandCols<KC, CT, ACT, DT>;
  constexpr int H = Cols::H;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // Column groups fastest: neighbours read and write one row's neighbouring columns.
  const int wgs = (a.groups + kLoraWaves - 1) / kLoraWaves;
  const int b = blockIdx.x / wgs, grp = (blockIdx.x - b * wgs) * kLoraWaves + wave;
  if (grp >= a.groups) return;
  const Cols cols(a, grp, lane);
  u32x4 y[H][Cols::VEC];
  f32x4 v[H][KC][2];
  if (ROWS) {
    cols.load_y(block_row<true>(a.b, b, cols.c), y);
#pragma unroll
    for (int h = 0; h < H; ++h) load_v<KC>(a.v, b, H == 1 ? cols.part : h, a.R, cols.g, v[h]);
  }
  const int e = block_adapter<ROWS>(a.b, b);
  if (e < 0) return;  // past the last block
  const bool adapter = e < a.b.L;
  if (!adapter && H == 1 && a.inplace) return;
  const int sid = block_row<ROWS>(a.b, b, cols.c);
  if (!ROWS) cols.load_y(sid, y);
  f32x4 acc[H][CT];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[h][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (adapter) {
    u32x4 w[H][CT][KC];
    if (ROWS) cols.load_b(e, a.R, w);
    const int rank = min(a.ranks[e], a.R);
    if (!ROWS) {
      cols.load_b(e, rank, w);
#pragma unroll
      for (int h = 0; h < H; ++h) load_v<KC>(a.v, b * 16 + cols.c, H == 1 ? cols.part : h, rank, cols.g, v[h]);
    }
    if ((ROWS && rank < a.R) || (rank & 7)) cols.cut_b(rank, w);
#pragma unroll
    for (int h = 0; h < H; ++h) {
      typename DT::vec8 hi[KC], lo[KC];
      const int ex = split_v<KC, DT>(v[h], rank, cols.g, hi, lo);
      Cols::mul(w[h], hi, lo, acc[h]);
      Cols::scale(acc[h], ex, a.scaling[e]);
    }
  }
  cols.store(sid, y, acc);
}

// Prefill: v comes as operands, and what block b + 1 reads is in flight while
// block b is computed.
template <int KC, int CT, int ACT, typename DT>
__global__ __launch_bounds__(64 * kLoraWaves) void lora_expand_tile_kernel(ExpandArgs a) {
  using Cols = ExpandCols<KC, CT, ACT, DT>;
  using V8 = typename DT::vec8;
  constexpr int H = Cols::H;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wgs = (a.groups + kLoraWaves - 1) / kLoraWaves;
  const int rows = blockIdx.x / wgs, grp = (blockIdx.x - rows * wgs) * kLoraWaves + wave;
  if (grp >= a.groups) return;
  const Cols cols(a, grp, lane);
  const int b0 = rows * a.per, b1 = min(b0 + a.per, a.b.blocks);

  struct Stage {
    int e, sid;
    u32x4 y[H][Cols::VEC];
    u32x4 v[H][KC][2];
    int ex[H];
  };
  auto find = [&](Stage& s, int b) {
    s.e = b < b1 ? a.b.bucket[b] : -1;
    if (H == 1 && a.inplace && s.e >= a.b.L) s.e = -1;  // the rows without an adapter are the last ones
    s.sid = s.e >= 0 ? block_row<false>(a.b, b, cols.c) : -1;
  };
  auto load = [&](Stage& s, int b) {
    cols.load_y(s.sid, s.y);
    if (s.e < 0 || s.e >= a.b.L) return;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int unit = b * a.P + (H == 1 ? cols.part : h);
#pragma unroll
      for (int k = 0; k < KC; ++k) {
        s.v[h][k][0] = a.vs[((int64_t)unit * KC + k) * 128 + lane];
        s.v[h][k][1] = a.vs[((int64_t)unit * KC + k) * 128 + 64 + lane];
      }
      s.ex[h] = a.ve[unit * 16 + cols.c];
    }
  };
  u32x4 w[H][CT][KC];
  int prev = -1;
  float scale = 0.f;
  auto work = [&](const Stage& s) {
    f32x4 acc[H][CT];
    if (s.e < a.b.L) {
      if (s.e != prev) {
        prev = s.e;
        const int rank = min(a.ranks[prev], a.R);
        scale = a.scaling[prev];
        cols.load_b(prev, rank, w);
        if (rank & 7) cols.cut_b(rank, w);
      }
#pragma unroll
      for (int h = 0; h < H; ++h) {
        V8 hi[KC], lo[KC];
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          hi[k] = __builtin_bit_cast(V8, s.v[h][k][0]);
          lo[k] = __builtin_bit_cast(V8, s.v[h][k][1]);
        }
        Cols::mul(w[h], hi, lo, acc[h]);
        Cols::scale(acc[h], s.ex[h], scale);
      }
    } else {
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int t = 0; t < CT; ++t) acc[h][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    cols.store(s.sid, s.y, acc);
  };

  Stage st[2];
  find(st[0], b0);
  if (st[0].e < 0) return;
  load(st[0], b0);
  find(st[1], b0 + 1);
  for (int b = b0;;) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      Stage next;
      load(st[1 - d], b + 1);
      find(next, b + 2);
      work(st[d]);
      if (st[1 - d].e < 0) return;
      st[d].e = next.e;
      st[d].sid = next.sid;
      ++b;
    }
  }
}

template <int KC, int ACT, typename DT>
hipError_t launch_expand(const ExpandArgs& a, int mode, dim3 grid, hipStream_t s) {
  constexpr int CT = kLoraColTiles / (ACT == kActNone ? 1 : 2);
  const dim3 block(64 * kLoraWaves);
  if (mode == kLoraRows)
    hipLaunchKernelGGL((lora_expand_kernel<true, KC, CT, ACT, DT>), grid, block, 0, s, a);
  else if (mode == kLoraBlocks)
    hipLaunchKernelGGL((lora_expand_kernel<false, KC, CT, ACT, DT>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((lora_expand_tile_kernel<KC, CT, ACT, DT>), grid, block, 0, s, a);
  return hipGetLastError();
}

template <int KC, typename DT>
hipError_t launch_split_expand(const SplitArgs& sp, const ExpandArgs& a, int mode, int act, dim3 grid, hipStream_t s) {
  if (mode == kLoraTiles) {
    const int64_t units = (int64_t)sp.b.blocks * sp.P;
    hipLaunchKernelGGL((lora_split_kernel<KC, DT>), dim3((unsigned)((units + kLoraWaves - 1) / kLoraWaves)),
                       dim3(64 * kLoraWaves), 0, s, sp);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (act == kActSilu) return launch_expand<KC, kActSilu, DT>(a, mode, grid, s);
  if (act == kActGelu) return launch_expand<KC, kActGelu, DT>(a, mode, grid, s);
  return launch_expand<KC, kActNone, DT>(a, mode, grid, s);
}

template <typename DT>
hipError_t launch_shrink(const ShrinkArgs& a, const LoraPlan& p, hipStream_t s) {
  const dim3 block(64 * kLoraWaves);
  const unsigned ks = (unsigned)p.slices;
  if (p.mode != kLoraTiles) {
    const dim3 grid((unsigned)p.blocks, ks, (unsigned)a.tiles);
    if (p.mode == kLoraRows)
      hipLaunchKernelGGL((lora_shrink_kernel<true, DT>), grid, block, 0, s, a);
    else
      hipLaunchKernelGGL((lora_shrink_kernel<false, DT>), grid, block, 0, s, a);
    return hipGetLastError();
  }
  const int rt = p.rank_tiles;
  const dim3 grid((unsigned)((p.blocks + 3) / 4), ks, (unsigned)((a.tiles + kLoraWaves * rt - 1) / (kLoraWaves * rt)));
  constexpr int lds = kShrinkSlots * kShrinkRows * 128;
#define SGL_TILE(RT_) \
  if (rt == RT_) hipLaunchKernelGGL((lora_shrink_tile_kernel<RT_, DT>), grid, block, lds, s, a)
  SGL_TILE(1);
  SGL_TILE(2);
  SGL_TILE(3);
  SGL_TILE(4);
#undef SGL_TILE
  return hipGetLastError();
}

int rank_chunks(int64_t R) { return R <= 32 ? 1 : R <= 64 ? 2 : R <= 128 ? 4 : 8; }

}  // namespace

LoraPlan plan_lora(int64_t M, int64_t K, int64_t L, int64_t R, int parts, bool routed) {
  LoraPlan p{};
  const int cus = device_cu_count();
  const int tiles = parts * (int)((R + 15) / 16);
  p.mode = !routed ? kLoraRows : M < kLoraTileRows ? kLoraBlocks : kLoraTiles;
  const int64_t cap = moe_sorted_capacity(M, L + 1, kLoraBlock);
  // A block holds a row at least.
  p.blocks = routed ? std::min(moe_block_capacity(M, L + 1, kLoraBlock), M) : M;
  p.positions = routed ? cap : M;
  p.rank_tiles = p.mode == kLoraTiles ? std::min(4, (tiles + kLoraWaves - 1) / kLoraWaves) : 1;
  const int per = p.mode == kLoraTiles ? kLoraWaves * p.rank_tiles : 1;
  const int64_t wgs = (int64_t)((tiles + per - 1) / per) * (p.mode == kLoraTiles ? (p.blocks + 3) / 4 : p.blocks);
  const int64_t steps = (K + kStepK - 1) / kStepK;
  // Two workgroups a CU, two steps a wave at least, and no more than eight partial sums.
  p.slices = (int)std::max<int64_t>(
      1, std::min<int64_t>({8, steps / (p.mode == kLoraTiles ? 8 : 2 * kLoraWaves), (2 * cus + wgs - 1) / wgs}));
  p.per = p.mode == kLoraTiles ? 8 : 1;
  p.v_bytes = (int64_t)p.slices * p.positions * tiles * 16 * 4;
  p.vs_bytes = p.mode == kLoraTiles ? p.blocks * parts * rank_chunks(R) * 2048 : 0;
  p.ve_bytes = p.mode == kLoraTiles ? p.blocks * parts * 16 * 4 : 0;
  p.ws_bytes = p.v_bytes + p.vs_bytes + p.ve_bytes;
  return p;
}

hipError_t launch_lora(const LoraParams& p, hipStream_t s) {
  const LoraPlan plan = plan_lora(p.M, p.K, p.L, p.R, p.parts, p.sorted != nullptr);
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
  a.v_slice = plan.positions * a.VR;
  const hipError_t st = p.dtype == 0 ? launch_shrink<F16>(a, plan, s) : launch_shrink<BF16>(a, plan, s);
  if (st != hipSuccess) return st;

  ExpandArgs x{};
  x.b = a.b;
  x.v.v = a.v;
  x.v.v_slice = a.v_slice;
  x.v.slices = plan.slices;
  x.v.VR = a.VR;
  x.v.rp = 16 * rt;
  u32x4* vs = (u32x4*)((char*)p.ws + plan.v_bytes);
  int32_t* ve = (int32_t*)((char*)p.ws + plan.v_bytes + plan.vs_bytes);
  x.vs = vs;
  x.ve = ve;
  x.y = p.y;
  x.out = p.out;
  x.w = p.b;
  x.scaling = p.scaling;
  x.ranks = p.ranks;
  x.w_bytes = (uint32_t)(p.N * p.R * 2);
  x.N = (int)p.N;
  x.R = a.R;
  x.P = p.parts;
  x.per = plan.per;
  x.inplace = p.out == p.y;
  const int cols = 16 * kLoraColTiles / (p.act ? 2 : 1);
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
  const SplitArgs sp{a.b, x.v, p.ranks, vs, ve, p.parts, a.R};
  const dim3 grid((unsigned)((x.groups + kLoraWaves - 1) / kLoraWaves * ((plan.blocks + x.per - 1) / x.per)));
#define SGL_KC(KC_)                                                                    \
  (p.dtype == 0 ? launch_split_expand<KC_, F16>(sp, x, plan.mode, p.act, grid, s)      \
                : launch_split_expand<KC_, BF16>(sp, x, plan.mode, p.act, grid, s))
  switch (rank_chunks(p.R)) {
    case 1: return SGL_KC(1);
    case 2: return SGL_KC(2);
    case 4: return SGL_KC(4);
    default: return SGL_KC(8);
  }
#undef SGL_KC
}

}  // namespace sgl_awq
