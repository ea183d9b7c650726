// Grouped products of dense (fp16 or bf16) experts over ragged row buckets.
//
//   out[r, n] = w_r sum_k a[r / top_k, k] W[e(r)][n, k]
//
// with W [E, N, K] as a checkpoint holds it, or, with a gate/up activation,
// out[r, j] = act(g) * u of the sums g of row j and u of row N / 2 + j of W, each
// times w_r first where routed weights are asked for; fp32 throughout, rounded
// once.  Rows are taken in the order of their experts (the alignment kernel's
// sorted table), in tiles of one expert's rows.
//
// W's and a's rows are contiguous in k, which is the MFMA operand order of 8
// consecutive values per lane: neither is rearranged beforehand.
#include <math.h>

#include <algorithm>

#include "awq_buffer.h"
#include "awq_epilogue.h"
#include "awq_launch.h"
#include "awq_rowtiles.h"

namespace sgl_awq {

namespace {

constexpr int kDenseStepK = 64;  // k per step: two 16-byte loads a lane, 128 bytes of a row

struct DenseArgs {
  const void* x;
  const void* w;
  const int32_t* sorted;
  const int32_t* offsets;  // padded bucket offsets [E + 1]
  const float* topk_w;
  void* out;
  uint32_t x_bytes, w_bytes;  // of the activation rows, and of one expert's W (both below 2^31)
  int a_div, num_routed, sorted_cap, E;
  int N, K;
  int cols;   // output columns: N, or N / 2 with an activation
  int groups; // column groups of a row tile
  int slots;  // row tiles the grid covers at a time
};

// The outputs of lane (row c of an m-tile, columns n .. n + 3).
template <int ACT, typename DT>
__device__ __forceinline__ void dense_store4(const DenseArgs& a, int sid, float rw, int n, f32x4 g, f32x4 u) {
  using E = typename DT::elem;
  typename DT::vec4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = (E)(ACT == kActNone ? g[i] * rw : gated_act(ACT, g[i] * rw) * (u[i] * rw));
  *(typename DT::vec4*)((E*)a.out + (int64_t)sid * a.cols + n) = r;
}

// Few rows per expert: a workgroup is one tile of up to 16 MT rows and 16 NT
// columns (of each half, with an activation), its four waves split K and load
// weights and rows straight into MFMA operands: each wave reads other k, so
// LDS would share nothing.  Bound by reading each busy expert's weights once.
constexpr int kDenseWaves = 4;

template <int EPL, int MT, int NT, int D, int ACT, typename DT>
__global__ __launch_bounds__(64 * kDenseWaves) void dense_rows_kernel(DenseArgs a) {
  using V8 = typename DT::vec8;
  constexpr int H = ACT == kActNone ? 1 : 2;
  __shared__ f32x4 red[kDenseWaves * H * NT * MT * 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const int slot = blockIdx.x / a.groups, base = (blockIdx.x - slot * a.groups) * 16 * NT;
  const int steps = (a.K + kDenseStepK - 1) / kDenseStepK;
  const int s0 = wave * steps / kDenseWaves, s1 = (wave + 1) * steps / kDenseWaves;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, a.x_bytes);

  RowTiles<EPL> tiles;
  tiles.scan(a.offsets, a.E, a.sorted_cap, 16 * MT, lane);
  for (int t = slot;; t += a.slots) {
    int e, rb, rows;
    tiles.find(t, 16 * MT, lane, e, rb, rows);
    if (e < 0) break;  // the same in every wave
    int sid[MT];
    uint32_t xo[MT];
    bool some = false;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      sid[m] = 16 * m + c < rows ? a.sorted[rb + 16 * m + c] : -1;
      if (sid[m] >= a.num_routed) sid[m] = -1;
      xo[m] = sid[m] >= 0 ? ((uint32_t)(sid[m] / a.a_div) * (uint32_t)a.K + 16u * g) * 2u : kPastEnd;
      some |= sid[m] >= 0;
    }
    if (__ballot(some) == 0) continue;  // padding alone: the same in every wave

    const __amdgpu_buffer_rsrc_t wr = make_rsrc((const char*)a.w + (int64_t)e * a.w_bytes, a.w_bytes);
    uint32_t wo[H][NT];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int n = base + 16 * j + c;
        wo[h][j] = n < a.cols ? ((uint32_t)(h * a.cols + n) * (uint32_t)a.K + 16u * g) * 2u : kPastEnd;
      }
    struct Stage {
      u32x4 w[H][NT][2], x[MT][2];
    };
    auto load = [&](Stage& st, int s) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        // K is a multiple of 8, so a lane's vector lies in its row or past its end.
        const uint32_t dead = s < s1 && s * kDenseStepK + 16 * g + 8 * q < a.K ? 0u : kPastEnd;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int j = 0; j < NT; ++j)
            st.w[h][j][q] = __builtin_amdgcn_raw_buffer_load_b128(wr, (wo[h][j] + 16u * q) | dead, s * kDenseStepK * 2,
                                                                  kCacheStream);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          st.x[m][q] = __builtin_amdgcn_raw_buffer_load_b128(xr, (xo[m] + 16u * q) | dead, s * kDenseStepK * 2, 0);
      }
    };
    f32x4 acc[H][NT][MT];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[h][j][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    Stage st[D];
#pragma unroll
    for (int p = 0; p + 1 < D; ++p) load(st[p], s0 + p);
    for (int s = s0; s < s1;) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        load(st[(d + D - 1) % D], s + D - 1);
        __builtin_amdgcn_sched_barrier(0);  // the prefetch stays ahead of this step's math
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int m = 0; m < MT; ++m)
                acc[h][j][m] = mfma16x16x32(__builtin_bit_cast(V8, st[d].w[h][j][q]),
                                            __builtin_bit_cast(V8, st[d].x[m][q]), acc[h][j][m]);
        if (++s >= s1) break;
      }
    }
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m) red[((wave * H + h) * NT * MT + j * MT + m) * 64 + lane] = acc[h][j][m];
    __syncthreads();
    auto sum = [&](int h, int u) {
      f32x4 v = red[(h * NT * MT + u) * 64 + lane];
#pragma unroll
      for (int w = 1; w < kDenseWaves; ++w) v += red[((w * H + h) * NT * MT + u) * 64 + lane];
      return v;
    };
    // Wave w stores the (column tile, m-tile) pairs w, w + 4, ...: lane (row c, columns 4 g .. 4 g + 3).
    for (int u = wave; u < NT * MT; u += kDenseWaves) {
      const int j = u / MT, m = u - j * MT;
      const int n = base + 16 * j + 4 * g;
      int id = -1;
#pragma unroll
      for (int i = 0; i < MT; ++i) id = i == m ? sid[i] : id;
      const f32x4 v0 = sum(0, u), v1 = sum(H - 1, u);
      if (id >= 0 && n < a.cols)
        dense_store4<ACT, DT>(a, id, a.topk_w != nullptr ? a.topk_w[id] : 1.f, n, v0, v1);
    }
    __syncthreads();  // before the next tile's partial sums
  }
}

// Many rows per expert: a workgroup of eight waves is one tile of up to 256
// rows of an expert and 256 rows of its W (with an activation 128 gate and their
// 128 up rows), both staged through two LDS buffers of 64 k by LDS-DMA.  Wave
// (wm, wn) of 2 x 4 holds half the tile's rows and 64 columns.
constexpr int kTileWaves = 8;
constexpr int kTileM = 256;
constexpr int kTileN = 256;
constexpr int kTileVecs = 2048;  // 16-byte vectors of one operand's stage: 256 rows of 128 bytes
constexpr int kTileLds = 4 * kTileVecs * 16 + kTileM * 4;

// One tile: MT m-tiles of 16 rows a wave.
//
// Row r of a stage lies at 128 r, its 16-byte vector q (k = 8 q .. 8 q + 7) in
// place q ^ (r & 7): the DMA's lanes then read whole lines of a row, and the
// MFMA operand reads of 8 rows at one q meet all banks.
template <int MT, int ACT, typename DT>
__device__ __forceinline__ void dense_tile(const DenseArgs& a, u32x4* lds, const int32_t* sids,
                                           const __amdgpu_buffer_rsrc_t& wr, const uint32_t (&wo)[4],
                                           const __amdgpu_buffer_rsrc_t& xr, const uint32_t (&xo)[4], int base,
                                           int wave, int lane) {
  using E = typename DT::elem;
  using V8 = typename DT::vec8;
  constexpr int H = ACT == kActNone ? 1 : 2;
  constexpr int NTH = 4 / H;  // column tiles of each half
  const int c = lane & 15, g = lane >> 4;
  const int wm = wave >> 2, wn = wave & 3;
  const int steps = (a.K + kDenseStepK - 1) / kDenseStepK;
  const int kq = ((lane & 7) ^ (lane >> 3)) * 8;  // the lane's k in a step's DMA

  auto issue = [&](int s) {
    u32x4* buf = lds + (s & 1) * 2 * kTileVecs;
    const uint32_t dead = s * kDenseStepK + kq < a.K ? 0u : kPastEnd;  // K is a multiple of 8
#pragma unroll
    for (int q = 0; q < 4; ++q)
      load_lds16(wr, buf + kTileVecs + (q * kTileWaves + wave) * 64, wo[q] | dead, s * kDenseStepK * 2);
#pragma unroll
    for (int q = 0; q < (MT + 1) / 2; ++q)
      if (q * kTileWaves + wave < 4 * MT)
        load_lds16(xr, buf + (q * kTileWaves + wave) * 64, xo[q] | dead, s * kDenseStepK * 2);
  };
  f32x4 acc[MT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Step s: wait until its loads have landed, meet the other waves -- all of it
  // is in LDS then, and every wave is done with step s - 1, whose buffer step
  // s + 1 takes -- and issue step s + 1.
  issue(0);
  for (int s = 0; s < steps; ++s) {
    __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(0));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (s + 1 < steps) issue(s + 1);
    __builtin_amdgcn_sched_barrier(0);
    const u32x4* xs = lds + (s & 1) * 2 * kTileVecs + wm * MT * 128 + c * 8;
    const u32x4* ws = lds + (s & 1) * 2 * kTileVecs + kTileVecs + wn * 512 + c * 8;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int at = (k * 4 + g) ^ (c & 7);
      V8 b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = __builtin_bit_cast(V8, ws[j * 128 + at]);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const V8 x = __builtin_bit_cast(V8, xs[m * 128 + at]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[m][j] = mfma16x16x32(b[j], x, acc[m][j]);
      }
    }
  }

  // Lane (row c of each m-tile) holds 4 NTH consecutive columns of each half.
  const int n0 = base + wn * 16 * NTH + 4 * NTH * g;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int sid = sids[(wm * MT + m) * 16 + c];
    if (sid < 0) continue;
    const float rw = a.topk_w != nullptr ? a.topk_w[sid] : 1.f;
#pragma unroll
    for (int v = 0; v < NTH / 2; ++v) {
      V8 r;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const int j = 2 * v + (w >> 2);
        if constexpr (ACT == kActNone)
          r[w] = (E)(acc[m][j][w & 3] * rw);
        else
          r[w] = (E)(gated_act(ACT, acc[m][j][w & 3] * rw) * (acc[m][j + NTH][w & 3] * rw));
      }
      if (n0 + 8 * v < a.cols) *(V8*)((E*)a.out + (int64_t)sid * a.cols + n0 + 8 * v) = r;
    }
  }
}

template <int EPL, int ACT, typename DT>
__global__ __launch_bounds__(64 * kTileWaves) void dense_tile_kernel(DenseArgs a) {
  constexpr int H = ACT == kActNone ? 1 : 2;
  constexpr int NTH = 4 / H;
  extern __shared__ u32x4 lds[];
  int32_t* sids = (int32_t*)(lds + 4 * kTileVecs);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;

  // Workgroup b runs on XCD b % 8: each XCD takes a run of consecutive units,
  // so that the tiles that read one expert's weights share an L2.
  RowTiles<EPL> tiles;
  tiles.scan(a.offsets, a.E, a.sorted_cap, kTileM, lane);
  const int per_xcd = (tiles.total() * a.groups + 7) >> 3, u = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd) return;
  int e, rb, rows, group;
  tiles.find_unit(u, a.groups, kTileM, 32, lane, e, rb, rows, group);
  if (e < 0) return;  // the same in every wave
  const int base = group * 64 * NTH;

  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, a.x_bytes);
  const __amdgpu_buffer_rsrc_t wr = make_rsrc((const char*)a.w + (int64_t)e * a.w_bytes, a.w_bytes);
  const uint32_t kq = ((lane & 7) ^ (lane >> 3)) * 8;
  uint32_t xo[4], wo[4];
  bool some = false;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = (q * kTileWaves + wave) * 8 + (lane >> 3);
    int sid = r < rows ? a.sorted[rb + r] : -1;
    if (sid >= a.num_routed) sid = -1;
    some |= sid >= 0;
    if ((lane & 7) == 0) sids[r] = sid;
    xo[q] = sid >= 0 ? ((uint32_t)(sid / a.a_div) * (uint32_t)a.K + kq) * 2u : kPastEnd;
    // Row 64 wn + 16 j + i of the stage: column 4 NTH (i / 4) + 4 (j % NTH) + i % 4 of half j / NTH of
    // wave wn's columns, so that a lane's MFMA outputs are consecutive columns.
    const int i = r & 15, j = (r >> 4) & 3;
    const int n = base + (r >> 6) * 16 * NTH + 4 * NTH * (i >> 2) + 4 * (j % NTH) + (i & 3);
    wo[q] = n < a.cols ? ((uint32_t)(j / NTH * a.cols + n) * (uint32_t)a.K + kq) * 2u : kPastEnd;
  }
  if (!__syncthreads_or(some)) return;  // padding alone
  if (rows <= 64)
    dense_tile<2, ACT, DT>(a, lds, sids, wr, wo, xr, xo, base, wave, lane);
  else if (rows <= 128)
    dense_tile<4, ACT, DT>(a, lds, sids, wr, wo, xr, xo, base, wave, lane);
  else if (rows <= 192)
    dense_tile<6, ACT, DT>(a, lds, sids, wr, wo, xr, xo, base, wave, lane);
  else
    dense_tile<8, ACT, DT>(a, lds, sids, wr, wo, xr, xo, base, wave, lane);
}

template <int EPL, int ACT, typename DT>
hipError_t launch_tile(const DenseArgs& a, dim3 grid, hipStream_t s) {
  hipLaunchKernelGGL((dense_tile_kernel<EPL, ACT, DT>), grid, dim3(64 * kTileWaves), kTileLds, s, a);
  return hipGetLastError();
}

int tile_groups(const MoeDenseParams& p) {
  const int64_t cols = p.act ? p.N / 2 : p.N, bn = p.act ? kTileN / 2 : kTileN;
  return (int)((cols + bn - 1) / bn);
}

// Workgroups that every (tile, column group) pair fits in: of the buckets' rows,
// padding included, each expert has one tile more than its full ones at most.
int64_t tile_units(const MoeDenseParams& p) {
  return (p.sorted_cap / kTileM + std::min(p.num_routed, p.E)) * tile_groups(p);
}

hipError_t launch_tile_act(const DenseArgs& args, const MoeDenseParams& p, hipStream_t s) {
  DenseArgs a = args;
  a.groups = tile_groups(p);
  const dim3 grid((unsigned)((tile_units(p) + 7) / 8 * 8));
#define SGL_TILE(ACT_, DT_) (p.E <= 128 ? launch_tile<2, ACT_, DT_>(a, grid, s) : launch_tile<8, ACT_, DT_>(a, grid, s))
#define SGL_TILE_A(ACT_) (p.dtype == 0 ? SGL_TILE(ACT_, F16) : SGL_TILE(ACT_, BF16))
  if (p.act == kActSilu) return SGL_TILE_A(kActSilu);
  if (p.act == kActGelu) return SGL_TILE_A(kActGelu);
  return SGL_TILE_A(kActNone);
#undef SGL_TILE_A
#undef SGL_TILE
}

template <int EPL, int MT, int NT, int D, int ACT>
hipError_t launch_rows(const DenseArgs& a, int64_t slots, int dtype, hipStream_t s) {
  const dim3 grid((unsigned)(slots * a.groups));
  if (dtype == 0)
    hipLaunchKernelGGL((dense_rows_kernel<EPL, MT, NT, D, ACT, F16>), grid, dim3(64 * kDenseWaves), 0, s, a);
  else
    hipLaunchKernelGGL((dense_rows_kernel<EPL, MT, NT, D, ACT, BF16>), grid, dim3(64 * kDenseWaves), 0, s, a);
  return hipGetLastError();
}

template <int MT, int NT, int D>
hipError_t launch_rows_act(const DenseArgs& args, const MoeDenseParams& p, hipStream_t s) {
  // With an activation a workgroup's tiles are half gate and half up.
  constexpr int NA = NT / 2;
  DenseArgs a = args;
  const int nt = p.act ? NA : NT;
  a.groups = (a.cols + 16 * nt - 1) / (16 * nt);
  // Every tile with rows at once, as far as a launch of 2^24 workgroups goes.
  const int64_t slots = std::min<int64_t>({p.num_routed, p.num_routed / (16 * MT) + p.E, ((1 << 24) - 1) / a.groups});
  a.slots = (int)slots;
#define SGL_ROWS(ACT_, NT_)                                                              \
  (p.E <= 128 ? launch_rows<2, MT, NT_, D, ACT_>(a, slots, p.dtype, s)                   \
              : launch_rows<8, MT, NT_, D, ACT_>(a, slots, p.dtype, s))
  if (p.act == kActSilu) return SGL_ROWS(kActSilu, NA);
  if (p.act == kActGelu) return SGL_ROWS(kActGelu, NA);
  return SGL_ROWS(kActNone, NT);
#undef SGL_ROWS
}

}  // namespace

hipError_t launch_moe_dense(const MoeDenseParams& p, hipStream_t s) {
  DenseArgs a{};
  a.x = p.x;
  a.w = p.w;
  a.sorted = p.sorted;
  a.offsets = p.offsets;
  a.topk_w = p.mul_rw ? p.topk_w : nullptr;
  a.out = p.out;
  a.x_bytes = (uint32_t)((p.num_routed + p.a_div - 1) / p.a_div * p.K * 2);
  a.w_bytes = (uint32_t)(p.N * p.K * 2);
  a.a_div = (int)p.a_div;
  a.num_routed = (int)p.num_routed;
  a.sorted_cap = (int)p.sorted_cap;
  a.E = (int)p.E;
  a.N = (int)p.N;
  a.K = (int)p.K;
  a.cols = (int)(p.act ? p.N / 2 : p.N);
  if (p.num_routed <= 4 * p.E) return launch_rows_act<1, 2, 4>(a, p, s);
  if (p.num_routed >= 64 * p.E && tile_units(p) < (1 << 24)) return launch_tile_act(a, p, s);
  return launch_rows_act<4, 4, 2>(a, p, s);
}

}  // namespace sgl_awq
