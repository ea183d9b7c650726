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
// per lane.  v stays in fp32 between the two launches, at the rows' sorted
// positions, one partial sum per k-slice, added in slice order: no atomics.
#include <math.h>

#include <algorithm>

#include "awq_buffer.h"
#include "awq_epilogue.h"
#include "awq_launch.h"

namespace sgl_awq {

namespace {

constexpr int kLoraWaves = 4;
constexpr int kStepK = 64;  // k per step of the shrink: two 16-byte loads a lane, 128 bytes of a row

// ---------------------------------------------------------------------------
// Shrink.
// ---------------------------------------------------------------------------
struct ShrinkArgs {
  const void* x;
  const void* a;
  const int32_t* sorted;
  const int32_t* bucket;  // adapter of each 16-row block, L: none, -1: past the last block
  const int32_t* ranks;
  float* v;               // [k-slices][sorted_cap][VR]
  uint32_t x_bytes, a_bytes;  // of x, and of one adapter's A (both below 2^31)
  int M, K, L, R;
  int rt;                 // rank tiles of 16 per part
  int tiles;              // P * rt
  int VR;                 // 16 * tiles
  int blocks;             // entries of `bucket` that the grid covers
  int steps;              // k-steps
  int64_t v_slice;        // sorted_cap * VR
};

// RT rank tiles (from tile q0) of MT 16-row blocks (from sorted position pos0)
// of one adapter, over the wave's k-steps.  D - 1 steps are in flight ahead.
template <int RT, int MT, int D, typename DT>
__device__ __forceinline__ void shrink_tile(const ShrinkArgs& a, f32x4* red, int e, int q0, int pos0, int wave,
                                            int lane) {
  using V8 = typename DT::vec8;
  const int i = lane & 15, g = lane >> 4;
  const int rank = min(a.ranks[e], a.R);
  const __amdgpu_buffer_rsrc_t ar = make_rsrc((const char*)a.a + (int64_t)e * a.a_bytes, a.a_bytes);
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, a.x_bytes);
  uint32_t ao[RT], xo[MT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int q = q0 + t, p = q / a.rt, r = (q - p * a.rt) * 16 + i;
    ao[t] = q < a.tiles && r < rank ? ((uint32_t)(p * a.R + r) * (uint32_t)a.K + 16u * g) * 2u : kPastEnd;
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int sid = a.sorted[pos0 + 16 * m + i];
    xo[m] = sid >= 0 && sid < a.M ? ((uint32_t)sid * (uint32_t)a.K + 16u * g) * 2u : kPastEnd;
  }
  // Slice (blockIdx.y, wave) of the k-steps.
  const int parts = gridDim.y * kLoraWaves, part = blockIdx.y * kLoraWaves + wave;
  const int s0 = (int)((int64_t)part * a.steps / parts), s1 = (int)((int64_t)(part + 1) * a.steps / parts);

  struct Stage {
    u32x4 a[RT][2], x[MT][2];
  };
  auto load = [&](Stage& st, int s) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // K is a multiple of 8, so a lane's vector lies in its row or past its end.
      const uint32_t dead = s < s1 && s * kStepK + 16 * g + 8 * h < a.K ? 0u : kPastEnd;
#pragma unroll
      for (int t = 0; t < RT; ++t)
        st.a[t][h] = __builtin_amdgcn_raw_buffer_load_b128(ar, (ao[t] + 16u * h) | dead, s * kStepK * 2, 0);
#pragma unroll
      for (int m = 0; m < MT; ++m)
        st.x[m][h] = __builtin_amdgcn_raw_buffer_load_b128(xr, (xo[m] + 16u * h) | dead, s * kStepK * 2, 0);
    }
  };
  f32x4 acc[RT][MT];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[t][m] = f32x4{0.f, 0.f, 0.f, 0.f};
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
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int m = 0; m < MT; ++m)
            acc[t][m] = mfma16x16x32(__builtin_bit_cast(V8, st[d].a[t][h]), __builtin_bit_cast(V8, st[d].x[m][h]),
                                     acc[t][m]);
      if (++s >= s1) break;
    }
  }

  // Sum over the waves; lane (row i, ranks 4 g .. 4 g + 3) of each tile.
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) red[((wave * RT + t) * MT + m) * 64 + lane] = acc[t][m];
  __syncthreads();
  float* v = a.v + (int64_t)blockIdx.y * a.v_slice;
  for (int u = wave; u < RT * MT; u += kLoraWaves) {
    const int t = u / MT, m = u - t * MT;
    if (q0 + t >= a.tiles) continue;
    f32x4 s = red[u * 64 + lane];
#pragma unroll
    for (int w = 1; w < kLoraWaves; ++w) s += red[(w * RT * MT + u) * 64 + lane];
    *(f32x4*)(v + (int64_t)(pos0 + 16 * m + i) * a.VR + (q0 + t) * 16 + 4 * g) = s;
  }
}

// grid: (groups of MT row blocks, k-slices, groups of RT rank tiles).
template <int RT, int MT, int D, typename DT>
__global__ __launch_bounds__(64 * kLoraWaves) void lora_shrink_kernel(ShrinkArgs a) {
  __shared__ f32x4 red[kLoraWaves * RT * MT * 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int q0 = blockIdx.z * RT, b0 = blockIdx.x * MT;
  // Buckets are in order: equal ends are one adapter's blocks throughout.
  const int e0 = a.bucket[b0];
  if (e0 < 0 || e0 >= a.L) return;
  if (MT > 1 && (b0 + MT > a.blocks || a.bucket[b0 + MT - 1] != e0)) {
    for (int b = b0; b < min(b0 + MT, a.blocks); ++b) {
      const int e = a.bucket[b];
      if (e < 0 || e >= a.L) break;
      shrink_tile<RT, 1, D, DT>(a, red, e, q0, b * 16, wave, lane);
      __syncthreads();  // before the next block's partial sums
    }
    return;
  }
  shrink_tile<RT, MT, D, DT>(a, red, e0, q0, b0 * 16, wave, lane);
}

// ---------------------------------------------------------------------------
// Expand.
// ---------------------------------------------------------------------------
struct ExpandArgs {
  const void* y;
  void* out;
  const void* b;
  const float* v;
  const float* scaling;
  const int32_t* sorted;
  const int32_t* bucket;
  const int32_t* ranks;
  uint32_t b_bytes;  // one adapter's B (below 2^31)
  int M, N, L, R, rp, VR, slices;
  int64_t v_slice;
  int blocks, per;   // row blocks, and how many a workgroup takes in turn
  int inplace;       // out is y: rows without an adapter stay as they are
  int groups;        // column groups
  int col[kLoraParts + 1];    // first column of each part
  int group[kLoraParts + 1];  // first column group of each part
};

// One wave: a group of 16 CT columns of each of HALVES column ranges (gate and
// up with an activation), row block after row block.
//
// Column j of MFMA tile t of a group is column 4 CT (j / 4) + 4 t + j % 4: lane
// (row, g) then holds 4 CT consecutive columns of its row.
template <int KC, int CT, int ACT, typename DT>
__global__ __launch_bounds__(64 * kLoraWaves) void lora_expand_kernel(ExpandArgs a) {
  using E = typename DT::elem;
  using V8 = typename DT::vec8;
  constexpr int H = ACT == kActNone ? 1 : 2;
  constexpr int VEC = CT / 2;  // 8-column vectors a lane holds in each half
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  // Column groups fastest: neighbours read and write one row's neighbouring columns.
  const int wgs = (a.groups + kLoraWaves - 1) / kLoraWaves;
  const int rows = blockIdx.x / wgs, grp = (blockIdx.x - rows * wgs) * kLoraWaves + wave;
  if (grp >= a.groups) return;
  int part = 0;
  if (H == 1)
    while (part + 1 < kLoraParts && grp >= a.group[part + 1]) ++part;
  const int base = a.col[part] + (grp - a.group[part]) * 16 * CT, end = a.col[part + 1];
  const int half = a.N >> 1, ncols = H == 1 ? a.N : half;

  u32x4 bw[H][CT][KC];
  int prev = -1, rank = 0;
  float scale = 0.f;
  const int b1 = min((rows + 1) * a.per, a.blocks);
  for (int b = rows * a.per; b < b1; ++b) {
    const int e = a.bucket[b];
    if (e < 0) break;  // past the last block
    const bool adapter = e < a.L;
    if (!adapter && H == 1 && a.inplace) break;  // the rows without an adapter are the last ones
    const int sid = a.sorted[b * 16 + c];
    const bool valid = sid >= 0 && sid < a.M;

    u32x4 yv[H][VEC];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int q = 0; q < VEC; ++q) {
        const int n = base + 4 * CT * g + 8 * q;
        yv[h][q] = u32x4{0u, 0u, 0u, 0u};
        if (valid && n < end) yv[h][q] = *(const u32x4*)((const E*)a.y + (int64_t)sid * a.N + h * half + n);
      }

    f32x4 acc[H][CT];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[h][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (adapter) {
      if (e != prev) {
        prev = e;
        rank = min(a.ranks[e], a.R);
        scale = a.scaling[e];
        const __amdgpu_buffer_rsrc_t br = make_rsrc((const char*)a.b + (int64_t)e * a.b_bytes, a.b_bytes);
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int t = 0; t < CT; ++t) {
            const int n = base + 4 * CT * (c >> 2) + 4 * t + (c & 3);
#pragma unroll
            for (int k = 0; k < KC; ++k) {
              const int r0 = 32 * k + 8 * g;
              const uint32_t off = n < end && r0 < rank
                                       ? ((uint32_t)(h * half + n) * (uint32_t)a.R + (uint32_t)r0) * 2u
                                       : kPastEnd;
              bw[h][t][k] = __builtin_amdgcn_raw_buffer_load_b128(br, off, 0, 0);
            }
          }
        if (rank & 7) {  // values past the rank inside a vector
#pragma unroll
          for (int k = 0; k < KC; ++k) {
            const int live = rank - (32 * k + 8 * g);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t m = live >= 2 * w + 2 ? ~0u : live == 2 * w + 1 ? 0xFFFFu : 0u;
#pragma unroll
              for (int h = 0; h < H; ++h)
#pragma unroll
                for (int t = 0; t < CT; ++t) bw[h][t][k][w] &= m;
            }
          }
        }
      }
#pragma unroll
      for (int h = 0; h < H; ++h) {
        // The lane's row of v: 8 consecutive ranks per 32, the k-slices added in order.
        float v[KC][8];
        float top = 0.f;
        const float* vp = a.v + (int64_t)(b * 16 + c) * a.VR + (H == 1 ? part : h) * a.rp + 8 * g;
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
          if (32 * k + 8 * g < rank) {
            for (int s = 0; s < a.slices; ++s) {
              lo += *(const f32x4*)(vp + s * a.v_slice + 32 * k);
              hi += *(const f32x4*)(vp + s * a.v_slice + 32 * k + 4);
            }
          }
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            const float f = w < 4 ? lo[w] : hi[w - 4];
            v[k][w] = 32 * k + 8 * g + w < rank ? f : 0.f;
            top = fmaxf(top, fabsf(v[k][w]));
            if (v[k][w] != v[k][w]) top = INFINITY;
          }
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        // v enters the MFMAs as two values of the operand type, the second the
        // first one's remainder: 22 (fp16) or 16 (bf16) bits of the row's
        // largest, so its rounding stays far below the output's.  The row is
        // brought into [-1, 1] by a power of two first (fp16 holds no more than
        // 65504); a row with an infinity or NaN keeps those, and its finite
        // values no longer count.
        const int ex = top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 128;
        constexpr float kUp = sizeof(E) == 2 && __is_same(E, _Float16) ? 2048.f : 256.f;
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          V8 r;
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            v[k][w] = __builtin_ldexpf(v[k][w], -ex);
            const float rem = v[k][w] - (float)(E)v[k][w];
            r[w] = top < INFINITY ? (E)(rem * kUp) : (E)0.f;
          }
#pragma unroll
          for (int t = 0; t < CT; ++t) acc[h][t] = mfma16x16x32(__builtin_bit_cast(V8, bw[h][t][k]), r, acc[h][t]);
        }
#pragma unroll
        for (int t = 0; t < CT; ++t) acc[h][t] *= 1.f / kUp;
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          V8 r;
#pragma unroll
          for (int w = 0; w < 8; ++w) r[w] = (E)v[k][w];
#pragma unroll
          for (int t = 0; t < CT; ++t) acc[h][t] = mfma16x16x32(__builtin_bit_cast(V8, bw[h][t][k]), r, acc[h][t]);
        }
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int w = 0; w < 4; ++w) acc[h][t][w] = __builtin_ldexpf(acc[h][t][w], ex) * scale;
      }
    }
#pragma unroll
    for (int q = 0; q < VEC; ++q) {
      const int n = base + 4 * CT * g + 8 * q;
      V8 r;
      const V8 y0 = __builtin_bit_cast(V8, yv[0][q]), y1 = __builtin_bit_cast(V8, yv[H - 1][q]);
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const int t = 2 * q + (w >> 2);
        const float f = (float)y0[w] + acc[0][t][w & 3];
        if constexpr (ACT == kActNone) {
          r[w] = (E)f;
        } else {
          r[w] = (E)(gated_act(ACT, f) * ((float)y1[w] + acc[H - 1][t][w & 3]));
        }
      }
      if (valid && n < end) *(V8*)((E*)a.out + (int64_t)sid * ncols + n) = r;
    }
  }
}

template <int RT, int MT, int D>
hipError_t launch_shrink(const ShrinkArgs& a, dim3 grid, int dtype, hipStream_t s) {
  if (dtype == 0)
    hipLaunchKernelGGL((lora_shrink_kernel<RT, MT, D, F16>), grid, dim3(64 * kLoraWaves), 0, s, a);
  else
    hipLaunchKernelGGL((lora_shrink_kernel<RT, MT, D, BF16>), grid, dim3(64 * kLoraWaves), 0, s, a);
  return hipGetLastError();
}

template <int KC, int ACT>
hipError_t launch_expand(const ExpandArgs& a, dim3 grid, int dtype, hipStream_t s) {
  constexpr int CT = kLoraColTiles / (ACT == kActNone ? 1 : 2);
  if (dtype == 0)
    hipLaunchKernelGGL((lora_expand_kernel<KC, CT, ACT, F16>), grid, dim3(64 * kLoraWaves), 0, s, a);
  else
    hipLaunchKernelGGL((lora_expand_kernel<KC, CT, ACT, BF16>), grid, dim3(64 * kLoraWaves), 0, s, a);
  return hipGetLastError();
}

template <int KC>
hipError_t launch_expand_act(const ExpandArgs& a, dim3 grid, int act, int dtype, hipStream_t s) {
  if (act == kActSilu) return launch_expand<KC, kActSilu>(a, grid, dtype, s);
  if (act == kActGelu) return launch_expand<KC, kActGelu>(a, grid, dtype, s);
  return launch_expand<KC, kActNone>(a, grid, dtype, s);
}

}  // namespace

LoraPlan plan_lora(int64_t M, int64_t K, int64_t L, int64_t R, int parts) {
  LoraPlan p{};
  const int cus = device_cu_count();
  const int tiles = parts * (int)((R + 15) / 16);
  p.blocks = moe_block_capacity(M, L + 1, 16);
  p.blocks = std::min(p.blocks, M);  // a block holds a row at least
  p.row_tiles = p.blocks * 16 > 4 * M || M < 64 ? 1 : 4;
  p.rank_tiles = p.row_tiles == 4 ? std::min(tiles, 4) : 1;
  if (p.rank_tiles == 3) p.rank_tiles = 4;
  const int64_t groups = (tiles + p.rank_tiles - 1) / p.rank_tiles;
  const int64_t wgs = groups * ((p.blocks + p.row_tiles - 1) / p.row_tiles);
  const int64_t steps = (K + kStepK - 1) / kStepK;
  // Two steps a wave at least, and no more than eight partial sums.
  p.slices = (int)std::max<int64_t>(
      1, std::min<int64_t>({8, steps / (2 * kLoraWaves), (2 * cus + wgs - 1) / std::max<int64_t>(wgs, 1)}));
  p.per = M >= 1024 ? 8 : 1;
  p.ws_bytes = (int64_t)p.slices * moe_sorted_capacity(M, L + 1, 16) * tiles * 16 * 4;
  return p;
}

hipError_t launch_lora(const LoraParams& p, hipStream_t s) {
  const LoraPlan plan = plan_lora(p.M, p.K, p.L, p.R, p.parts);
  const int rt = (int)((p.R + 15) / 16), tiles = p.parts * rt;
  ShrinkArgs a{};
  a.x = p.x;
  a.a = p.a;
  a.sorted = p.sorted;
  a.bucket = p.bucket;
  a.ranks = p.ranks;
  a.v = p.ws;
  a.x_bytes = (uint32_t)(p.M * p.K * 2);
  a.a_bytes = (uint32_t)(p.parts * p.R * p.K * 2);
  a.M = (int)p.M;
  a.K = (int)p.K;
  a.L = (int)p.L;
  a.R = (int)p.R;
  a.rt = rt;
  a.tiles = tiles;
  a.VR = 16 * tiles;
  a.blocks = (int)plan.blocks;
  a.steps = (int)((p.K + kStepK - 1) / kStepK);
  a.v_slice = moe_sorted_capacity(p.M, p.L + 1, 16) * a.VR;
  const dim3 sg((unsigned)((plan.blocks + plan.row_tiles - 1) / plan.row_tiles), (unsigned)plan.slices,
                (unsigned)((tiles + plan.rank_tiles - 1) / plan.rank_tiles));
  hipError_t st;
  if (plan.row_tiles == 1)
    st = launch_shrink<1, 1, 4>(a, sg, p.dtype, s);
  else if (plan.rank_tiles == 1)
    st = launch_shrink<1, 4, 3>(a, sg, p.dtype, s);
  else if (plan.rank_tiles == 2)
    st = launch_shrink<2, 4, 2>(a, sg, p.dtype, s);
  else
    st = launch_shrink<4, 4, 2>(a, sg, p.dtype, s);
  if (st != hipSuccess) return st;

  ExpandArgs x{};
  x.y = p.y;
  x.out = p.out;
  x.b = p.b;
  x.v = p.ws;
  x.scaling = p.scaling;
  x.sorted = p.sorted;
  x.bucket = p.bucket;
  x.ranks = p.ranks;
  x.b_bytes = (uint32_t)(p.N * p.R * 2);
  x.M = a.M;
  x.N = (int)p.N;
  x.L = a.L;
  x.R = a.R;
  x.rp = 16 * rt;
  x.VR = a.VR;
  x.slices = plan.slices;
  x.v_slice = a.v_slice;
  x.blocks = a.blocks;
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
  const dim3 eg((unsigned)((x.groups + kLoraWaves - 1) / kLoraWaves * ((x.blocks + x.per - 1) / x.per)));
  if (p.R <= 32) return launch_expand_act<1>(x, eg, p.act, p.dtype, s);
  if (p.R <= 64) return launch_expand_act<2>(x, eg, p.act, p.dtype, s);
  if (p.R <= 128) return launch_expand_act<4>(x, eg, p.act, p.dtype, s);
  return launch_expand_act<8>(x, eg, p.act, p.dtype, s);
}

}  // namespace sgl_awq
