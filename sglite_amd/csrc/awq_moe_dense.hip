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
  int K;
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

// Few rows per expert: a workgroup is one 16-row tile and 16 NT columns (of each
// half, with an activation), its four waves split K and load weights and rows
// straight into MFMA operands: each wave reads other k, so LDS would share
// nothing.  Bound by reading each busy expert's weights once; the loads in flight
// are those of many short waves.  One step ahead against two and three took 223 /
// 229 / 238 us for both products of E = 128, H = 2048, I = 768 top-8 at 32 tokens
// (4.7 TB/s of weights), 31.5 / 32.3 / 32.5 at one; two waves 227 and 32.0, eight
// 268 and 33.0.  (Measured on this loop, whose break between the two steps of its
// body gives it two ways back to its head: the compiler waits there for all loads,
// and every second step starts with none in flight.)
constexpr int kDenseWaves = 4;

template <int EPL, int NT, int ACT, typename DT>
__global__ __launch_bounds__(64 * kDenseWaves) void dense_rows_kernel(DenseArgs a) {
  using V8 = typename DT::vec8;
  constexpr int H = ACT == kActNone ? 1 : 2;
  constexpr int D = 2;
  __shared__ f32x4 red[kDenseWaves * H * NT * 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const int slot = blockIdx.x / a.groups, base = (blockIdx.x - slot * a.groups) * 16 * NT;
  const int steps = (a.K + kDenseStepK - 1) / kDenseStepK;
  const int s0 = wave * steps / kDenseWaves, s1 = (wave + 1) * steps / kDenseWaves;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, a.x_bytes);

  RowTiles<EPL> tiles;
  tiles.load(a.offsets, a.E, a.sorted_cap, lane);
  tiles.scan(16, lane);
  for (int t = slot;; t += a.slots) {
    int e, rb, rows;
    tiles.find(t, 16, lane, e, rb, rows);
    if (e < 0) break;  // the same in every wave
    int sid = c < rows ? a.sorted[rb + c] : -1;
    if (sid >= a.num_routed) sid = -1;
    if (__ballot(sid >= 0) == 0) continue;  // padding alone: the same in every wave
    const uint32_t xo = sid >= 0 ? ((uint32_t)(sid / a.a_div) * (uint32_t)a.K + 16u * g) * 2u : kPastEnd;
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
      u32x4 w[H][NT][2], x[2];
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
        st.x[q] = __builtin_amdgcn_raw_buffer_load_b128(xr, (xo + 16u * q) | dead, s * kDenseStepK * 2, 0);
      }
    };
    f32x4 acc[H][NT];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[h][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    Stage st[D];
    load(st[0], s0);
    for (int s = s0; s < s1;) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        load(st[1 - d], s + 1);
        __builtin_amdgcn_sched_barrier(0);  // the prefetch stays ahead of this step's math
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int j = 0; j < NT; ++j)
              acc[h][j] = mfma16x16x32(__builtin_bit_cast(V8, st[d].w[h][j][q]), __builtin_bit_cast(V8, st[d].x[q]),
                                       acc[h][j]);
        if (++s >= s1) break;
      }
    }
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int j = 0; j < NT; ++j) red[((wave * H + h) * NT + j) * 64 + lane] = acc[h][j];
    __syncthreads();
    auto sum = [&](int h, int j) {
      f32x4 v = red[(h * NT + j) * 64 + lane];
#pragma unroll
      for (int w = 1; w < kDenseWaves; ++w) v += red[((w * H + h) * NT + j) * 64 + lane];
      return v;
    };
    // Wave j sums and stores column tile j: lane (row c, columns 4 g .. 4 g + 3).
    const int n = base + 16 * wave + 4 * g;
    if (wave < NT) {
      const f32x4 v0 = sum(0, wave), v1 = sum(H - 1, wave);
      if (sid >= 0 && n < a.cols)
        dense_store4<ACT, DT>(a, sid, a.topk_w != nullptr ? a.topk_w[sid] : 1.f, n, v0, v1);
    }
    __syncthreads();  // before the next tile's partial sums
  }
}

template <int EPL, int NT, int ACT>
hipError_t launch_rows(const DenseArgs& a, int64_t slots, int dtype, hipStream_t s) {
  const dim3 grid((unsigned)(slots * a.groups));
  if (dtype == 0)
    hipLaunchKernelGGL((dense_rows_kernel<EPL, NT, ACT, F16>), grid, dim3(64 * kDenseWaves), 0, s, a);
  else
    hipLaunchKernelGGL((dense_rows_kernel<EPL, NT, ACT, BF16>), grid, dim3(64 * kDenseWaves), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_rows_act(const DenseArgs& args, const MoeDenseParams& p, hipStream_t s) {
  DenseArgs a = args;
  const int cols = p.act ? 16 : 32;  // a gate and an up tile, or two tiles
  a.groups = (a.cols + cols - 1) / cols;
  // Every tile with rows at once, as far as a launch of 2^24 workgroups goes.
  const int64_t slots = std::min<int64_t>({p.num_routed, p.num_routed / 16 + p.E, ((1 << 24) - 1) / a.groups});
  a.slots = (int)slots;
#define SGL_ROWS(ACT_, NT_) \
  (p.E <= 128 ? launch_rows<2, NT_, ACT_>(a, slots, p.dtype, s) : launch_rows<8, NT_, ACT_>(a, slots, p.dtype, s))
  if (p.act == kActSilu) return SGL_ROWS(kActSilu, 1);
  if (p.act == kActGelu) return SGL_ROWS(kActGelu, 1);
  return SGL_ROWS(kActNone, 2);
#undef SGL_ROWS
}

// Many rows per expert: a workgroup of eight waves is one tile of up to 320
// rows of an expert and 256 rows of its W (with an activation 128 gate and their
// 128 up rows), both staged through two LDS buffers of 64 k by LDS-DMA.  Wave
// (wm, wn) of 2 x 4 holds half the tile's rows and 64 columns.  One workgroup a
// CU takes unit after unit.  Bound by the weights' bytes where experts are short
// (E = 128, H = 2048, I = 768 top-8 at 512 tokens: gate/up and down 196 + 95 us,
// 4.2 TB/s) and by the MFMA loop and the last round of units where they are long
// (E = 16, H = 4096, I = 1408 top-4 at 4001 tokens: 555 GFLOP in 419 + 233 us under
// the profiler; an eager pass of both and the alignment takes 592 us, 0.94 PFLOP/s).
// The form for more than 128 experts (EPL = 8) keeps 16 registers of buckets a lane
// and spills 26 (44 with gelu), outside the loop over k: E = 256, H = 2048, I = 768
// top-8 at 512 / 4096 tokens 553 / 693 us, E = 512 of I = 384 566 / 682 us, for
// 2.4 GB of weights (4.4 and 4.3 TB/s at 512 tokens).
constexpr int kTileWaves = 8;
constexpr int kTileM = 320;
constexpr int kTileN = 256;
constexpr int kTileGrain = 32;               // a tile's rows come in multiples of two m-tiles
constexpr int kTileX = kTileM * 8;           // 16-byte vectors of the rows' stage: 128 bytes a row
constexpr int kTileStage = (kTileM + kTileN) * 8;
constexpr int kTileLds = 2 * kTileStage * 16 + kTileM * 4;  // and the row ids
constexpr int kTileXLoads = kTileM / (8 * kTileWaves);      // a wave's DMAs of a stage's rows, at most
constexpr int kTileMore = 64;  // what a tile takes beside its rows, in rows

// One unit: MT m-tiles of 16 rows a wave.
//
// Row r of a stage lies at 128 r, its 16-byte vector q (k = 8 q .. 8 q + 7) in
// place q ^ (r & 7): the DMA's lanes then read whole lines of a row, and the
// MFMA operand reads of 8 rows at one q meet all banks.
//
// (Starting the following unit's first stage ahead of the epilogue takes the
// registers that the products need: with what it keeps spilled, 478 against
// 422 us for both products of E = 128, H = 2048, I = 768 top-8 at 4096 tokens.)
template <int MT, int ACT, typename DT>
__device__ __forceinline__ void dense_tile(const DenseArgs& a, u32x4* lds, const int32_t* sids,
                                           const __amdgpu_buffer_rsrc_t& wr, const uint32_t (&wo)[4],
                                           const __amdgpu_buffer_rsrc_t& xr, const uint32_t (&xo)[kTileXLoads],
                                           int base, int wave, int lane) {
  using E = typename DT::elem;
  using V8 = typename DT::vec8;
  constexpr int H = ACT == kActNone ? 1 : 2;
  constexpr int NTH = 4 / H;  // column tiles of each half
  const int c = lane & 15, g = lane >> 4;
  const int wm = wave >> 2, wn = wave & 3;
  const int steps = (a.K + kDenseStepK - 1) / kDenseStepK;
  const int kq = ((lane & 7) ^ (lane >> 3)) * 8;  // the lane's k in a step's DMA

  auto issue = [&](int s) {
    u32x4* buf = lds + (s & 1) * kTileStage;
    const uint32_t dead = s * kDenseStepK + kq < a.K ? 0u : kPastEnd;  // K is a multiple of 8
#pragma unroll
    for (int q = 0; q < 4; ++q)
      load_lds16(wr, buf + kTileX + (q * kTileWaves + wave) * 64, wo[q] | dead, s * kDenseStepK * 2);
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
    const u32x4* xs = lds + (s & 1) * kTileStage + wm * MT * 128 + c * 8;
    const u32x4* ws = lds + (s & 1) * kTileStage + kTileX + wn * 512 + c * 8;
    const int at0 = g ^ (c & 7), at1 = (4 + g) ^ (c & 7);
    V8 w[2][4], x[MT];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[0][j] = __builtin_bit_cast(V8, ws[j * 128 + at0]);
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = __builtin_bit_cast(V8, xs[m * 128 + at0]);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[1][j] = __builtin_bit_cast(V8, ws[j * 128 + at1]);
    // The second half of a row operand follows its first into the same
    // registers, MT m-tiles of products ahead of its use.
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[m][j] = mfma16x16x32(w[0][j], x[m], acc[m][j]);
      x[m] = __builtin_bit_cast(V8, xs[m * 128 + at1]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[m][j] = mfma16x16x32(w[1][j], x[m], acc[m][j]);
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
      for (int i = 0; i < 8; ++i) {
        const int j = 2 * v + (i >> 2);
        if constexpr (ACT == kActNone)
          r[i] = (E)(acc[m][j][i & 3] * rw);
        else
          r[i] = (E)(gated_act_fast(ACT, acc[m][j][i & 3] * rw) * (acc[m][j + NTH][i & 3] * rw));
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
  int32_t* sids = (int32_t*)(lds + 2 * kTileStage);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;

  // The tile height: with units of nearly equal length the last round of them
  // leaves CUs idle, so the height is the one with the shortest rounds for
  // these buckets (every workgroup finds the same).
  RowTiles<EPL> tiles;
  tiles.load(a.offsets, a.E, a.sorted_cap, lane);
  int height = kTileM;
  float best = INFINITY;
  for (int h = kTileM; h >= 128; h -= kTileGrain) {
    int n, work;
    tiles.weigh(h, kTileGrain, kTileMore, n, work);
    const int units = n * a.groups, cus = gridDim.x;
    const float cost = (float)((units + cus - 1) / cus) * (float)work / (float)max(n, 1);
    if (cost < best) {
      best = cost;
      height = h;
    }
  }
  tiles.scan(height, lane);

  // Workgroup b runs on XCD b % 8: each XCD takes a run of consecutive units,
  // so that the tiles that read one expert's weights share an L2.
  const int per_xcd = (tiles.total() * a.groups + 7) >> 3;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, a.x_bytes);
  const uint32_t kq = ((lane & 7) ^ (lane >> 3)) * 8;
  for (int at = blockIdx.x >> 3; at < per_xcd; at += gridDim.x >> 3) {
    int e, rb, rows, group;
    tiles.find_unit((blockIdx.x & 7) * per_xcd + at, a.groups, height, kTileGrain, lane, e, rb, rows, group);
    if (e < 0) break;  // the same in every wave
    const int base = group * 64 * NTH;
    const __amdgpu_buffer_rsrc_t wr = make_rsrc((const char*)a.w + (int64_t)e * a.w_bytes, a.w_bytes);
    uint32_t xo[kTileXLoads], wo[4];
    int sid[kTileXLoads];
    bool some = false;
#pragma unroll
    for (int q = 0; q < kTileXLoads; ++q) {
      const int r = (q * kTileWaves + wave) * 8 + (lane >> 3);
      sid[q] = r < rows ? a.sorted[rb + r] : -1;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      // Row 64 wn + 16 j + i of the stage: column 4 NTH (i / 4) + 4 (j % NTH) + i % 4 of half j / NTH of
      // wave wn's columns, so that a lane's MFMA outputs are consecutive columns.
      const int r = (q * kTileWaves + wave) * 8 + (lane >> 3), i = r & 15, j = (r >> 4) & 3;
      const int n = base + (r >> 6) * 16 * NTH + 4 * NTH * (i >> 2) + 4 * (j % NTH) + (i & 3);
      wo[q] = n < a.cols ? ((uint32_t)(j / NTH * a.cols + n) * (uint32_t)a.K + kq) * 2u : kPastEnd;
    }
    __syncthreads();  // the unit before is done with LDS
#pragma unroll
    for (int q = 0; q < kTileXLoads; ++q) {
      if (sid[q] >= a.num_routed) sid[q] = -1;
      some |= sid[q] >= 0;
      if ((lane & 7) == 0) sids[(q * kTileWaves + wave) * 8 + (lane >> 3)] = sid[q];
      xo[q] = sid[q] >= 0 ? ((uint32_t)(sid[q] / a.a_div) * (uint32_t)a.K + kq) * 2u : kPastEnd;
    }
    if (!__syncthreads_or(some)) continue;  // padding alone
#define SGL_MT(MT_) \
  case MT_: dense_tile<MT_, ACT, DT>(a, lds, sids, wr, wo, xr, xo, base, wave, lane); break
    switch ((rows + kTileGrain - 1) / kTileGrain) {
      SGL_MT(1);
      SGL_MT(2);
      SGL_MT(3);
      SGL_MT(4);
      SGL_MT(5);
      SGL_MT(6);
      SGL_MT(7);
      SGL_MT(8);
      SGL_MT(9);
      default: dense_tile<10, ACT, DT>(a, lds, sids, wr, wo, xr, xo, base, wave, lane);
    }
#undef SGL_MT
  }
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

// (Tile, column group) pairs, counted in 32 bits: of the buckets' rows, padding
// included, each expert has one tile more than its full ones at most.
int64_t tile_units(const MoeDenseParams& p) {
  return (p.sorted_cap / 128 + std::min(p.num_routed, p.E)) * tile_groups(p);
}

hipError_t launch_tile_act(const DenseArgs& args, const MoeDenseParams& p, hipStream_t s) {
  DenseArgs a = args;
  a.groups = tile_groups(p);
  const dim3 grid((unsigned)std::max(8, device_cu_count() / 8 * 8));
#define SGL_TILE(ACT_, DT_) (p.E <= 128 ? launch_tile<2, ACT_, DT_>(a, grid, s) : launch_tile<8, ACT_, DT_>(a, grid, s))
#define SGL_TILE_A(ACT_) (p.dtype == 0 ? SGL_TILE(ACT_, F16) : SGL_TILE(ACT_, BF16))
  if (p.act == kActSilu) return SGL_TILE_A(kActSilu);
  if (p.act == kActGelu) return SGL_TILE_A(kActGelu);
  return SGL_TILE_A(kActNone);
#undef SGL_TILE_A
#undef SGL_TILE
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
  a.K = (int)p.K;
  a.cols = (int)(p.act ? p.N / 2 : p.N);
  // From a few rows per expert the tiles read weights no slower and follow
  // uneven buckets better: E = 128, H = 2048, I = 768 top-8 at 4 rows an expert
  // 269 us both ways, at 8 260 against 306 (with 64-row tiles); E = 64, I = 1408
  // top-6 at 3 rows 220 row by row against 225, at 6 247 against 259.
  if (p.num_routed <= 4 * p.E || tile_units(p) >= (1 << 30)) return launch_rows_act(a, p, s);
  return launch_tile_act(a, p, s);
}

}  // namespace sgl_awq
