// Products with MXFP4 weights: activations quantised to MXFP4 on the way, scaled
// 16x16x128 MFMAs, fp32 sums, one rounding.
//
//   out[m, n] = sum_k Q(x)[m, k] W[n, k] (+ bias[n])
//   out[m, j] = act(g) u of those sums, g column j and u column N / 2 + j
//
// and the same over the routed rows of a stack of experts, times the routed
// weight.  The products of two codes and their scales are exact; a lane's 32 k
// are one block of each operand (awq_mx4.h).
#include <algorithm>
#include <type_traits>

#include "awq_buffer.h"
#include "awq_epilogue.h"
#include "awq_launch.h"
#include "awq_mx4.h"
#include "awq_rowtiles.h"

namespace sgl_awq {

namespace {

struct MxArgs {
  const void* x;       // activations, or their codes
  const uint8_t* xs;   // the codes' scales
  const char* w;
  const char* s;
  const void* bias;
  const float* topk_w;
  const int32_t* sorted;
  const int32_t* offsets;
  void* out;
  int M, K, cols;      // rows (of x, for experts), inner size, output columns
  int NT, KT, KS, half;  // column tiles, k-tiles, scale steps; NT / 2 with an activation
  int groups, slots, E, a_div, num_routed, sorted_cap;
};

// Few rows: a workgroup owns 16 MT rows and NTW column tiles (with an activation
// a gate tile and its up tile); its waves take steps of 512 k in turn, load
// weights straight into MFMA operands, a step ahead, and meet in LDS at the end.
// RM = 0: the rows come quantised, in the weights' layout.  Else a wave quantises
// the step's part of up to 16 rows itself, RM of them loaded ahead: four lanes a
// block, and through LDS into the operands' order.
//
// Bound by the weights' stream and the launch's own length: one row through
// Qwen3-4B's qkv, o, gate/up with silu and down (8.4, 5.6, 26.5 and 13.2 MB) takes
// 4.5, 4.0, 8.7 and 6.1 us in a graph.  From 64 rows on what counts is the rows'
// way from the L2 (10 TB/s at 128 rows of 14336 x 4096, 18 us).  Quantising a block
// a lane, with 16 loads a k-tile, took 35 us in place of 23 for those four layers.
// Tried without gain: 16 rows loaded ahead (9 to 16 rows: 8.8 against 7.7 us for
// qkv), rows a whole step ahead (128 rows of qkv 14.9 against 13.0: registers),
// four column tiles a workgroup (128 rows of 14336 x 4096 26 against 21; experts
// at one token 10.9 -> 12.3, at 32 43 -> 41.5).
constexpr int kMxRowsWaves = 8;        // at most
constexpr int kMxRowWords = 68;        // a quantised row's step in LDS: 256 bytes of codes, and 16 against bank conflicts
constexpr int kMxExpertRows = 4;       // of an expert's rows, loaded ahead
constexpr int kMxRowsLds = 16 * (kMxRowWords + 4) * 4;  // a wave's, with the scales

template <typename DT, int RM, int MT, int NTW, int ACT>
struct RowsBody {
  using E = typename DT::elem;
  using V4 = typename DT::vec4;
  // Weights that one row block reads pass the caches as a stream.
  static constexpr int kPolicy = MT == 4 ? 0 : kCacheStream;
  static constexpr int XM = RM == 0 ? MT : 1;

  const MxArgs& a;
  const int wave, waves, lane;
  __amdgpu_buffer_rsrc_t wr[NTW], sr[NTW], xr, xsr;
  int tile[XM];     // RM = 0: row tiles, one past the last is the last
  int rows;         // else: rows, and the lane's (row lane % 16) offset in xr
  uint32_t row_at;

  __device__ __forceinline__ RowsBody(const MxArgs& args)
      : a(args),
        wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
        waves(blockDim.x >> 6),
        lane(threadIdx.x & 63) {}

  __device__ __forceinline__ void set_tiles(int64_t e, int group) {
#pragma unroll
    for (int j = 0; j < NTW; ++j) {
      const int t = ACT != kActNone ? group + j * a.half : group * NTW + j;
      wr[j] = make_rsrc(a.w + (e * a.NT + t) * (int64_t)a.KT * 1024, (uint32_t)a.KT * 1024u);
      sr[j] = make_rsrc(a.s + (e * a.NT + t) * (int64_t)a.KS * 256, (uint32_t)a.KS * 256u);
    }
  }
  __device__ __forceinline__ void load_w(u32x4 (&w)[NTW], int kt) const {
    const uint32_t past = kt < a.KT ? 0u : kPastEnd;
#pragma unroll
    for (int j = 0; j < NTW; ++j)
      w[j] = __builtin_amdgcn_raw_buffer_load_b128(wr[j], (uint32_t)lane * 16u | past, kt * 1024, kPolicy);
  }
  __device__ __forceinline__ void load_s(uint32_t (&s)[NTW], int step) const {
    const uint32_t at = (uint32_t)lane * 4u | (step < a.KS ? 0u : kPastEnd);
#pragma unroll
    for (int j = 0; j < NTW; ++j) s[j] = __builtin_amdgcn_raw_buffer_load_b32(sr[j], at, step * 256, 0);
  }
  template <int B>
  __device__ __forceinline__ void mul(const u32x4 (&w)[NTW], const uint32_t (&sw)[NTW], const u32x4 (&x)[XM],
                                      const uint32_t (&sx)[XM], f32x4 (&acc)[MT][NTW]) const {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < NTW; ++j) acc[mt][j] = mfma_mx4<B, B>(w[j], x[mt], sw[j], sx[mt], acc[mt][j]);
  }

  // Quantised rows.
  __device__ __forceinline__ void load_x(u32x4 (&x)[XM], int kt) const {
    const uint32_t at = (uint32_t)lane * 16u | (kt < a.KT ? 0u : kPastEnd);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      x[mt] = __builtin_amdgcn_raw_buffer_load_b128(xr, at, (tile[mt] * a.KT + kt) * 1024, 0);
  }
  __device__ __forceinline__ void load_sx(uint32_t (&s)[XM], int step) const {
    const uint32_t at = (uint32_t)lane * 4u | (step < a.KS ? 0u : kPastEnd);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      s[mt] = __builtin_amdgcn_raw_buffer_load_b32(xsr, at, (tile[mt] * a.KS + step) * 256, 0);
  }
  __device__ __forceinline__ void steps_quantized(f32x4 (&acc)[MT][NTW]) const {
    u32x4 w[4][NTW], x[2][XM];
    uint32_t sw[NTW], sx[XM], sw1[NTW], sx1[XM];
    load_s(sw, wave);
    load_sx(sx, wave);
#pragma unroll
    for (int b = 0; b < 4; ++b) load_w(w[b], 4 * wave + b);
    load_x(x[0], 4 * wave);
    load_x(x[1], 4 * wave + 1);
    for (int s = wave; s < a.KS; s += waves) {
      const int s1 = s + waves;  // a step past the last one loads zeros, and reads nothing
      load_s(sw1, s1);
      load_sx(sx1, s1);
      mul<0>(w[0], sw, x[0], sx, acc);
      load_w(w[0], 4 * s1);
      load_x(x[0], 4 * s + 2);
      mul<1>(w[1], sw, x[1], sx, acc);
      load_w(w[1], 4 * s1 + 1);
      load_x(x[1], 4 * s + 3);
      mul<2>(w[2], sw, x[0], sx, acc);
      load_w(w[2], 4 * s1 + 2);
      load_x(x[0], 4 * s1);
      mul<3>(w[3], sw, x[1], sx, acc);
      load_w(w[3], 4 * s1 + 3);
      load_x(x[1], 4 * s1 + 1);
#pragma unroll
      for (int j = 0; j < NTW; ++j) sw[j] = sw1[j];
#pragma unroll
      for (int mt = 0; mt < XM; ++mt) sx[mt] = sx1[mt];
    }
  }

  // Rows r0 .. r0 + RM - 1 of a step, 8 values a lane.
  __device__ __forceinline__ void load_rows(u32x4 (&v)[RM ? RM : 1], int r0, int step) const {
    // K is a multiple of 32: four lanes' block lies in its row or past its end.
    const uint32_t dead = step * 512 + 8 * lane < a.K ? 0u : kPastEnd;
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const uint32_t none = r0 + i < rows ? dead : kPastEnd;
      const uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)row_at, min(r0 + i, 15));
      v[i] = __builtin_amdgcn_raw_buffer_load_b128(xr, (at + 16u * lane) | none, step * 1024, 0);
    }
  }
  __device__ __forceinline__ void put_rows(const u32x4 (&v)[RM ? RM : 1], int r0, uint32_t* codes) const {
    uint8_t* scales = (uint8_t*)(codes + 16 * kMxRowWords);
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      if (r0 + i >= rows) break;
      uint32_t byte;
      codes[(r0 + i) * kMxRowWords + lane] = mx4_quarter<DT>(v[i], byte);
      if ((lane & 3) == 0) scales[16 * (r0 + i) + mx4_row_byte(lane >> 2)] = (uint8_t)byte;
    }
  }
  __device__ __forceinline__ void steps_rows(f32x4 (&acc)[MT][NTW], uint32_t* codes) const {
    u32x4 w[4][NTW], v[RM ? RM : 1];
    uint32_t sw[NTW], sw1[NTW];
    load_rows(v, 0, wave);  // ahead of the weights: loads come back in order
    load_s(sw, wave);
#pragma unroll
    for (int b = 0; b < 4; ++b) load_w(w[b], 4 * wave + b);
    // Lanes of rows that are not there read the last one.
    const int r = min(lane & 15, rows - 1), g = lane >> 4;
    for (int s = wave; s < a.KS; s += waves) {
      const int s1 = s + waves;
      put_rows(v, 0, codes);
      for (int r0 = RM; r0 < rows; r0 += RM) {
        load_rows(v, r0, s);
        put_rows(v, r0, codes);
      }
      load_rows(v, 0, s1);
      load_s(sw1, s1);
      const uint32_t sx[XM] = {codes[16 * kMxRowWords + 4 * r + g]};
      const u32x4* at = (const u32x4*)(codes + r * kMxRowWords) + g;
      const u32x4 x[4][XM] = {{at[0]}, {at[4]}, {at[8]}, {at[12]}};
      mul<0>(w[0], sw, x[0], sx, acc);
      load_w(w[0], 4 * s1);
      mul<1>(w[1], sw, x[1], sx, acc);
      load_w(w[1], 4 * s1 + 1);
      mul<2>(w[2], sw, x[2], sx, acc);
      load_w(w[2], 4 * s1 + 2);
      mul<3>(w[3], sw, x[3], sx, acc);
      load_w(w[3], 4 * s1 + 3);
#pragma unroll
      for (int j = 0; j < NTW; ++j) sw[j] = sw1[j];
    }
  }

  // The wave's steps, and every wave's sums in red; what the waves quantise lies behind it.
  __device__ __forceinline__ void run(f32x4* red) const {
    f32x4 acc[MT][NTW];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < NTW; ++j) acc[mt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (RM == 0)
      steps_quantized(acc);
    else
      steps_rows(acc, (uint32_t*)(red + waves * MT * NTW * 64) + wave * (kMxRowsLds / 4));
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < NTW; ++j) red[((wave * MT + mt) * NTW + j) * 64 + lane] = acc[mt][j];
  }
  __device__ __forceinline__ f32x4 sum(const f32x4* red, int mt, int j) const {
    f32x4 v = red[(mt * NTW + j) * 64 + lane];
    for (int w = 1; w < waves; ++w) v += red[((w * MT + mt) * NTW + j) * 64 + lane];
    return v;
  }
  __device__ __forceinline__ f32x4 biased(f32x4 v, int n, float rw) const {
    v *= rw;
    if (a.bias != nullptr) {
      const V4 b = *(const V4*)((const E*)a.bias + n);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += (float)b[i];
    }
    return v;
  }
  // The lane's 4 columns of m-tile mt and output tile j, row `row` of out.
  static constexpr int kOutTiles = ACT != kActNone ? NTW / 2 : NTW;
  __device__ __forceinline__ void store(const f32x4* red, int mt, int j, int64_t row, int group, float rw) const {
    const int t = group * kOutTiles + j, n = 32 * (t >> 1) + 8 * (lane >> 4) + 4 * (t & 1);
    if (n >= a.cols) return;  // N is a multiple of 8
    const f32x4 v = biased(sum(red, mt, j), n, rw);
    V4 r;
    if constexpr (ACT != kActNone) {
      const f32x4 up = biased(sum(red, mt, j + kOutTiles), a.cols + n, rw);
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = (E)(gated_act(ACT, v[i]) * up[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = (E)v[i];
    }
    *(V4*)((E*)a.out + row * a.cols + n) = r;
  }
};

template <typename DT, int RM, int MT, int NTW, int ACT>
__global__ __launch_bounds__(64 * kMxRowsWaves) void mx4_rows_kernel(MxArgs a) {
  extern __shared__ f32x4 red[];
  RowsBody<DT, RM, MT, NTW, ACT> b(a);
  // Workgroup b runs on XCD b % 8: all row blocks of a column group share an L2.
  const int local = blockIdx.x >> 3, group = (blockIdx.x & 7) + 8 * (local / a.slots);
  if (group >= a.groups) return;
  const int block = local % a.slots, m0 = block * 16 * MT;
  b.rows = min(16 * MT, a.M - m0);
  b.set_tiles(0, group);
  if constexpr (RM == 0) {
    const uint32_t tiles = (b.rows + 15) / 16;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) b.tile[mt] = min(mt, (int)tiles - 1);
    b.xr = make_rsrc((const char*)a.x + (int64_t)block * MT * a.KT * 1024, tiles * a.KT * 1024u);
    b.xsr = make_rsrc(a.xs + (int64_t)block * MT * a.KS * 256, tiles * a.KS * 256u);
  } else {
    b.xr = make_rsrc((const char*)a.x + (int64_t)m0 * a.K * 2, (uint32_t)b.rows * (uint32_t)a.K * 2u);
    b.row_at = (uint32_t)(b.lane & 15) * (uint32_t)a.K * 2u;
  }
  b.run(red);
  __syncthreads();
  for (int i = b.wave; i < MT * b.kOutTiles; i += b.waves) {
    const int mt = i / b.kOutTiles, r = 16 * mt + (b.lane & 15);
    if (r < b.rows) b.store(red, mt, i - mt * b.kOutTiles, m0 + r, group, 1.f);
  }
}

// The same for 16 sorted rows of one expert at a time.
template <typename DT, int NTW, int ACT, int EPL>
__global__ __launch_bounds__(64 * kMxRowsWaves) void mx4_expert_rows_kernel(MxArgs a) {
  extern __shared__ f32x4 red[];
  RowsBody<DT, kMxExpertRows, 1, NTW, ACT> b(a);
  const int slot = blockIdx.x / a.groups, group = blockIdx.x - slot * a.groups, c = b.lane & 15;
  RowTiles<EPL> tiles;
  tiles.load(a.offsets, a.E, a.sorted_cap, b.lane);
  tiles.scan(16, b.lane);
  b.xr = make_rsrc(a.x, (uint32_t)a.M * (uint32_t)a.K * 2u);
  for (int t = slot;; t += a.slots) {
    int e, rb, rows;
    tiles.find(t, 16, b.lane, e, rb, rows);
    if (e < 0) break;  // the same in every wave
    int sid = c < rows ? a.sorted[rb + c] : -1;
    if (sid >= a.num_routed) sid = -1;
    // Rows up to the last one that is no padding (the table has it behind them).
    const uint32_t live = (uint32_t)__ballot(sid >= 0) & 0xFFFFu;
    if (live == 0) continue;  // padding alone: the same in every wave
    b.rows = 32 - __builtin_clz(live);
    b.row_at = sid >= 0 ? (uint32_t)(sid / a.a_div) * (uint32_t)a.K * 2u : kPastEnd;
    b.set_tiles(e, group);
    b.run(red);
    __syncthreads();
    if (sid >= 0)
      for (int j = b.wave; j < b.kOutTiles; j += b.waves)
        b.store(red, 0, j, sid, group, a.topk_w != nullptr ? a.topk_w[sid] : 1.f);
    __syncthreads();  // before the next tile's partial sums
  }
}

// Many rows: a workgroup of four waves is up to 128 quantised rows and 64 NTW rows
// of W (with an activation half of them gate rows, the others their up rows).  The
// rows go through LDS stages of 512 k by LDS-DMA, in the order of the MFMA
// operands; a wave's weights are its own (NTW column tiles) and go straight to
// registers.
constexpr int kMxTileM = kMx4TileRows;
constexpr int kMxTileGrain = 32;  // a tile's rows come in multiples of two m-tiles
constexpr int kMxCodes = 4 * (kMxTileM / 16) * 64;      // 16-byte vectors of a stage's codes
constexpr int kMxStage = kMxCodes + kMxTileM;           // and its scales, 16 bytes a row
// NTW = 4: two stages, weights two k-tiles ahead, two workgroups a CU.  NTW = 2,
// for grids that leave CUs idle: three stages and weights six k-tiles ahead.
//
// 8192 rows of Llama-3-8B's gate/up with silu take 470 to 500 us between the
// layer's other launches, 3.9 to 4.1 PFLOP/s (qkv and o 3.5 to 3.7, down 4.5 to
// 4.7); the MFMA alone, its operands in registers, reaches 6.2 on random data (9.0
// on zeros: power).  MFMAs are busy 53 % of the time there, the L2 gives 12 TB/s.
// Tiles of 256 x 256 by eight waves, both operands through a ring of LDS stages,
// take a third less from the L2 and were no faster (526 us, when these took 509);
// neither were row operands further ahead, or
// workgroups of one CU on one column group.  E = 128, H = 2048, I = 768 top-8 at
// 4096 tokens: 93 and 86 us, MFMAs busy 20 %: four and two stages a tile, between
// its start and its scattered rows' stores.
constexpr int mx4_stages(int ntw) { return ntw == 4 ? 2 : 3; }
constexpr int mx4_tile_lds(int ntw) { return (mx4_stages(ntw) * kMxStage + kMxTileM / 2) * 16; }  // row ids, routed weights

struct MxUnit {
  __amdgpu_buffer_rsrc_t xr, xsr;
  int64_t e;    // expert
  int64_t row0; // first row of the ranges (linear)
  int group;    // column group
  int tiles;    // m-tiles (linear)
};

// ROWS: the codes row by row; a DMA brings 256 bytes of each of four rows (xrow:
// offsets of the lane's rows, with its 16 bytes), block j of row r lands in place
// j ^ (r % 16) of the row's 256 bytes of LDS, and the operand reads of 16 rows meet
// all banks.  Else in the weights' layout.  xsrow: the lane's 16 bytes of the
// wave's scales.
template <int MT, int NTW, int ACT, bool ROWS, typename DT>
__device__ __forceinline__ void mx4_tile(const MxArgs& a, u32x4* lds, const int32_t* sids, const MxUnit& u,
                                         const uint32_t (&xrow)[kMxTileM / 16], uint32_t xsrow, int wave, int lane) {
  using E = typename DT::elem;
  constexpr int NS = mx4_stages(NTW);
  constexpr int R = NTW == 4 ? 4 : 8, D = NTW == 4 ? 2 : 6;  // k-tiles of weights in registers, and ahead
  const int c = lane & 15, g = lane >> 4;
  // The wave's tiles are two runs of H: of its columns, or gate and up.  A run
  // past the last one is the last one again and not stored.
  constexpr int H = NTW / 2;
  const int runs = (ACT == kActNone ? a.NT : a.half) / H;
  __amdgpu_buffer_rsrc_t wr[2], sr[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = ACT == kActNone ? min((u.group * 4 + wave) * 2 + h, runs - 1) : min(u.group * 4 + wave, runs - 1) + h * runs;
    const int64_t t = u.e * a.NT + (int64_t)r * H;
    wr[h] = make_rsrc(a.w + t * a.KT * 1024, (uint32_t)(a.KT * H) * 1024u);
    sr[h] = make_rsrc(a.s + t * a.KS * 256, (uint32_t)(a.KS * H) * 256u);
  }
  struct Weights {
    u32x4 q[NTW];
  };
  auto load_w = [&](Weights& w, int kt) {
    kt = min(kt, a.KT - 1);
#pragma unroll
    for (int j = 0; j < NTW; ++j)
      w.q[j] = __builtin_amdgcn_raw_buffer_load_b128(wr[j / H], lane * 16, (j % H * a.KT + kt) * 1024, 0);
  };
  auto load_s = [&](uint32_t (&sw)[NTW], int s) {
    s = min(s, a.KS - 1);
#pragma unroll
    for (int j = 0; j < NTW; ++j)
      sw[j] = __builtin_amdgcn_raw_buffer_load_b32(sr[j / H], lane * 4, (j % H * a.KS + s) * 256, 0);
  };
  // Stage s's codes of m-tiles m0 .. m1 - 1: of each, wave w brings rows 4 w .. 4 w + 3,
  // or k-tile w.
  auto dma = [&](int s, int m0, int m1) {
    u32x4* buf = lds + s % NS * kMxStage;
    const int kt = 4 * s + wave;
    if constexpr (ROWS) {
      const uint32_t dead = s * 512 + 32 * (c ^ (4 * wave + g)) < a.K ? 0u : kPastEnd;
#pragma unroll
      for (int m = m0; m < m1; ++m) load_lds16(u.xr, buf + (4 * m + wave) * 64, xrow[m] | dead, s * 256);
    } else {
      const uint32_t at = lane * 16u | (kt < a.KT ? 0u : kPastEnd);
#pragma unroll
      for (int m = m0; m < m1; ++m)
        load_lds16(u.xr, buf + (wave * MT + m) * 64, at, (min(m, u.tiles - 1) * a.KT + kt) * 1024);
    }
  };
  // Their scales: rows 64 w .. 64 w + 63 by waves w and w + 2, both the same.
  auto dma_scales = [&](int s) {
    load_lds16(u.xsr, lds + s % NS * kMxStage + kMxCodes + (wave & 1) * 64, xsrow | (s < a.KS ? 0u : kPastEnd),
               s * (ROWS ? 16 : 256));
  };

  f32x4 acc[MT][NTW];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NTW; ++j) acc[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  Weights w[R];
  uint32_t sw[2][NTW];
  load_s(sw[0], 0);
  dma(0, 0, MT);
  dma_scales(0);
  __builtin_amdgcn_sched_barrier(0);  // the waits count the loads behind a stage's own
  if constexpr (NS == 3) {
    dma(1, 0, MT);
    dma_scales(1);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int k = 0; k < D; ++k) load_w(w[k], k);
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(D * NTW + (NS == 3 ? MT : 0)));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);

  constexpr int XMAX = NTW == 4 ? 3 : 7, XD = MT < XMAX ? MT : XMAX;  // row operands in registers: all but one ahead
  u32x4 x[XD];
  // Where the lane's operand of k-tile b and m-tile m lies in a stage.
  int xat[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) xat[b] = ROWS ? c * 16 + ((4 * b + g) ^ c) : b * MT * 64 + lane;
  constexpr int kRowTile = ROWS ? 256 : 64;
  auto step = [&](auto pp, auto bb, int s, uint32_t (&now)[NTW], uint32_t (&later)[NTW], const uint32_t (&sx)[MT]) {
    constexpr int P = decltype(pp)::value, b = decltype(bb)::value;
    if constexpr (b == 0) {
      load_s(later, s + 1);
      dma(s + NS - 1, 0, MT / 2);
    }
    if constexpr (b == 1) {
      dma(s + NS - 1, MT / 2, MT);
      dma_scales(s + NS - 1);
    }
    load_w(w[(4 * P + b + D) % R], 4 * s + b + D);
    __builtin_amdgcn_sched_barrier(0);
    if (b > 0 && ROWS && 4 * s + b >= a.KT) return;  // past K
    const u32x4* xs = lds + s % NS * kMxStage;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      // Operand b MT + m of the stage's 4 MT; the first ones are read ahead of the stage's first step.
      const int next = b * MT + m + XD - 1;
      if (next < 4 * MT) x[next % XD] = xs[xat[next / MT] + next % MT * kRowTile];
#pragma unroll
      for (int j = 0; j < NTW; ++j)
        acc[m][j] = mfma_mx4<b, b>(w[(4 * P + b) % R].q[j], x[(b * MT + m) % XD], now[j], sx[m], acc[m][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto super = [&](auto pp, int s, uint32_t (&now)[NTW], uint32_t (&later)[NTW]) {
    uint32_t sx[MT];
    const u32x4* stage = lds + s % NS * kMxStage;
    const uint32_t* at = (const uint32_t*)(stage + kMxCodes) + (ROWS ? c * 4 + g : lane);
#pragma unroll
    for (int m = 0; m < XD - 1; ++m) x[m] = stage[xat[0] + m * kRowTile];
#pragma unroll
    for (int m = 0; m < MT; ++m) sx[m] = at[m * 64];
    step(pp, std::integral_constant<int, 0>{}, s, now, later, sx);
    step(pp, std::integral_constant<int, 1>{}, s, now, later, sx);
    step(pp, std::integral_constant<int, 2>{}, s, now, later, sx);
    step(pp, std::integral_constant<int, 3>{}, s, now, later, sx);
    // Stage s + 1 has landed when at most the loads behind its own are
    // outstanding: two k-tiles' weights, and with three stages all of this step's
    // (but for the row scales').  Every wave is done with stage s.
    __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(2 * NTW + (NS == 3 ? MT + 5 * NTW : 0)));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int s = 0; s < a.KS; s += 2) {
    super(std::integral_constant<int, 0>{}, s, sw[0], sw[1]);
    if (s + 1 < a.KS) super(std::integral_constant<int, 1>{}, s + 1, sw[1], sw[0]);
  }

  // What was issued past the last stage has landed before LDS is another unit's.
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));

  // A lane holds 4 H consecutive columns of each run.
  constexpr int C = 4 * H;
  typedef E VC __attribute__((ext_vector_type(C)));
  const float* rws = (const float*)(sids + kMxTileM);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int sid = sids[m * 16 + c];
    if (sid < 0) continue;
    const float rw = a.topk_w != nullptr ? rws[m * 16 + c] : 1.f;
    E* out = (E*)a.out + (u.row0 + sid) * a.cols;
#pragma unroll
    for (int h = 0; h < (ACT == kActNone ? 2 : 1); ++h) {
      const int t = (ACT == kActNone ? (u.group * 4 + wave) * 2 + h : u.group * 4 + wave) * H;
      const int n = 32 * (t >> 1) + 8 * g + 4 * (t & 1);
      if (n >= a.cols) continue;  // columns come in multiples of 8
      float v[2][C];
#pragma unroll
      for (int i = 0; i < C; ++i) {
        v[0][i] = acc[m][H * h + (i >> 2)][i & 3] * rw;
        if constexpr (ACT != kActNone) v[1][i] = acc[m][H + (i >> 2)][i & 3] * rw;
      }
      if (a.bias != nullptr) {
#pragma unroll
        for (int k = 0; k < (ACT == kActNone ? 1 : 2); ++k) {
          const VC bias = *(const VC*)((const E*)a.bias + k * a.cols + n);
#pragma unroll
          for (int i = 0; i < C; ++i) v[k][i] += (float)bias[i];
        }
      }
      VC r;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        if constexpr (ACT == kActNone)
          r[i] = (E)v[0][i];
        else
          r[i] = (E)(gated_act_fast(ACT, v[0][i]) * v[1][i]);
      }
      *(VC*)(out + n) = r;
    }
  }
}

template <int NTW, int ACT, bool ROWS, typename DT>
__device__ __forceinline__ void mx4_tile_of(int rows, const MxArgs& a, u32x4* lds, const int32_t* sids, const MxUnit& u,
                                            const uint32_t (&xrow)[kMxTileM / 16], uint32_t xsrow, int wave, int lane) {
  switch ((rows + kMxTileGrain - 1) / kMxTileGrain) {
    case 1: mx4_tile<2, NTW, ACT, ROWS, DT>(a, lds, sids, u, xrow, xsrow, wave, lane); break;
    case 2: mx4_tile<4, NTW, ACT, ROWS, DT>(a, lds, sids, u, xrow, xsrow, wave, lane); break;
    case 3: mx4_tile<6, NTW, ACT, ROWS, DT>(a, lds, sids, u, xrow, xsrow, wave, lane); break;
    default: mx4_tile<8, NTW, ACT, ROWS, DT>(a, lds, sids, u, xrow, xsrow, wave, lane);
  }
}

// Linear layers: unit after unit of (row tile, column group), 8 row tiles by 8
// groups in turn, so that the workgroups of an XCD (b % 8) share rows and weights
// in its L2.
template <int NTW, int ACT, typename DT>
__global__ __launch_bounds__(256, 2) void mx4_tile_kernel(MxArgs a) {
  extern __shared__ u32x4 lds[];
  int32_t* sids = (int32_t*)(lds + mx4_stages(NTW) * kMxStage);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int units = a.slots * a.groups, per_xcd = (units + 7) >> 3;
  // Row tiles of nearly equal height.
  const int height = ((a.M + a.slots - 1) / a.slots + kMxTileGrain - 1) / kMxTileGrain * kMxTileGrain;
  for (int at = blockIdx.x >> 3; at < per_xcd; at += gridDim.x >> 3) {
    const int unit = (blockIdx.x & 7) * per_xcd + at;
    if (unit >= units) break;
    const int band = unit / (8 * a.groups), in = unit - band * 8 * a.groups, high = min(8, a.slots - 8 * band);
    MxUnit u;
    u.e = 0;
    u.group = in / high;
    u.row0 = (int64_t)(8 * band + in - u.group * high) * height;
    const int rows = (int)min((int64_t)height, a.M - u.row0);
    if (rows <= 0) continue;
    u.tiles = (rows + 15) / 16;  // row0 is a multiple of 16
    u.xr = make_rsrc((const char*)a.x + u.row0 / 16 * a.KT * 1024, (uint32_t)u.tiles * (uint32_t)a.KT * 1024u);
    u.xsr = make_rsrc(a.xs + u.row0 / 16 * a.KS * 256, (uint32_t)u.tiles * (uint32_t)a.KS * 256u);
    __syncthreads();  // the unit before is done with LDS
    if (threadIdx.x < kMxTileM) sids[threadIdx.x] = threadIdx.x < rows ? threadIdx.x : -1;
    __syncthreads();
    // 16 bytes of the scales of one of four m-tiles.
    const int m = 4 * (wave & 1) + (lane >> 4);
    const uint32_t xsrow = m < u.tiles ? (uint32_t)m * a.KS * 256u + 16u * (lane & 15) : kPastEnd;
    const uint32_t none[kMxTileM / 16] = {};
    mx4_tile_of<NTW, ACT, false, DT>(rows, a, lds, sids, u, none, xsrow, wave, lane);
  }
}

// Experts: a workgroup is one (tile of one expert's sorted rows, column group) of
// those that there are; the grid covers as many as there can be.  Each XCD (b % 8)
// takes a run of consecutive ones, so that the tiles that read one expert's
// weights share an L2.
template <int EPL, int NTW, int ACT, typename DT>
__global__ __launch_bounds__(256, 2) void mx4_expert_tile_kernel(MxArgs a) {
  extern __shared__ u32x4 lds[];
  int32_t* sids = (int32_t*)(lds + mx4_stages(NTW) * kMxStage);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  MxUnit u;
  int e, rb, rows;
  {
    RowTiles<EPL> tiles;
    tiles.load(a.offsets, a.E, a.sorted_cap, lane);
    tiles.scan(kMxTileM, lane);
    const int per_xcd = (tiles.total() * a.groups + 7) >> 3, at = blockIdx.x >> 3;
    if (at >= per_xcd) return;
    tiles.find_unit((blockIdx.x & 7) * per_xcd + at, a.groups, kMxTileM, kMxTileGrain, lane, e, rb, rows, u.group);
    if (e < 0) return;  // the same in every wave
  }
  int sid = -1;
  if (threadIdx.x < kMxTileM && (int)threadIdx.x < rows) sid = a.sorted[rb + threadIdx.x];
  if (sid >= a.num_routed) sid = -1;
  if (threadIdx.x < kMxTileM) {
    sids[threadIdx.x] = sid;
    if (a.topk_w != nullptr && sid >= 0) ((float*)sids)[kMxTileM + threadIdx.x] = a.topk_w[sid];
  }
  if (!__syncthreads_or(sid >= 0)) return;  // padding alone
  u.e = e;
  u.row0 = 0;
  u.xr = make_rsrc(a.x, (uint32_t)a.M * (uint32_t)(a.K / 2));
  u.xsr = make_rsrc(a.xs, (uint32_t)a.M * (uint32_t)a.KS * 16u);
  uint32_t xrow[kMxTileM / 16];
#pragma unroll
  for (int m = 0; m < kMxTileM / 16; ++m) {
    const int r = 4 * wave + (lane >> 4), id = sids[16 * m + r];
    xrow[m] = id < 0 ? kPastEnd : (uint32_t)(id / a.a_div) * (uint32_t)(a.K / 2) + 16u * ((lane & 15) ^ r);
  }
  const int id = sids[64 * (wave & 1) + lane];
  const uint32_t xsrow = id < 0 ? kPastEnd : (uint32_t)(id / a.a_div) * (uint32_t)(a.KS * 16);
  mx4_tile_of<NTW, ACT, true, DT>(rows, a, lds, sids, u, xrow, xsrow, wave, lane);
}

template <typename DT, int ACT>
hipError_t launch_tile(const MxArgs& a, const Mx4Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)p.grid), block(256);
  if (a.sorted == nullptr && p.ntw == 2)
    hipLaunchKernelGGL((mx4_tile_kernel<2, ACT, DT>), grid, block, mx4_tile_lds(2), s, a);
  else if (a.sorted == nullptr)
    hipLaunchKernelGGL((mx4_tile_kernel<4, ACT, DT>), grid, block, mx4_tile_lds(4), s, a);
  else if (a.E <= 128)
    hipLaunchKernelGGL((mx4_expert_tile_kernel<2, 4, ACT, DT>), grid, block, mx4_tile_lds(4), s, a);
  else
    hipLaunchKernelGGL((mx4_expert_tile_kernel<8, 4, ACT, DT>), grid, block, mx4_tile_lds(4), s, a);
  return hipGetLastError();
}

template <typename DT>
hipError_t launch_tiles(const MxArgs& a, const Mx4Plan& p, int act, hipStream_t s) {
  if (act == kActSilu) return launch_tile<DT, kActSilu>(a, p, s);
  if (act == kActGelu) return launch_tile<DT, kActGelu>(a, p, s);
  return launch_tile<DT, kActNone>(a, p, s);
}

template <typename DT, int RM, int MT, int NTW, int ACT>
hipError_t launch_rows_form(const MxArgs& a, const Mx4Plan& p, hipStream_t s) {
  hipLaunchKernelGGL((mx4_rows_kernel<DT, RM, MT, NTW, ACT>), dim3((unsigned)p.grid), dim3(64 * p.waves),
                     p.waves * (MT * NTW * 1024 + (RM ? kMxRowsLds : 0)), s, a);
  return hipGetLastError();
}

template <typename DT, int NTW, int ACT>
hipError_t launch_rows(const MxArgs& a, const Mx4Plan& p, hipStream_t s) {
  if (!p.pre) {
    if (a.M == 1) return launch_rows_form<DT, 1, 1, NTW, ACT>(a, p, s);
    if (a.M <= 4) return launch_rows_form<DT, 4, 1, NTW, ACT>(a, p, s);
    return launch_rows_form<DT, 8, 1, NTW, ACT>(a, p, s);
  }
  if (p.mt == 1) return launch_rows_form<DT, 0, 1, NTW, ACT>(a, p, s);
  if (p.mt == 2) return launch_rows_form<DT, 0, 2, NTW, ACT>(a, p, s);
  if (p.mt == 3) return launch_rows_form<DT, 0, 3, NTW, ACT>(a, p, s);
  return launch_rows_form<DT, 0, 4, NTW, ACT>(a, p, s);
}

template <typename DT>
hipError_t launch_linear(const MxArgs& a, const Mx4Plan& p, int act, hipStream_t s) {
  if (act == kActSilu) return launch_rows<DT, 2, kActSilu>(a, p, s);
  if (act == kActGelu) return launch_rows<DT, 2, kActGelu>(a, p, s);
  return p.ntw == 1 ? launch_rows<DT, 1, kActNone>(a, p, s) : launch_rows<DT, 2, kActNone>(a, p, s);
}

template <typename DT, int ACT, int EPL>
hipError_t launch_expert_form(const MxArgs& a, const Mx4Plan& p, hipStream_t s) {
  hipLaunchKernelGGL((mx4_expert_rows_kernel<DT, 2, ACT, EPL>), dim3((unsigned)p.grid), dim3(64 * p.waves),
                     p.waves * (2 * 1024 + kMxRowsLds), s, a);
  return hipGetLastError();
}

template <typename DT, int ACT>
hipError_t launch_expert_rows(const MxArgs& a, const Mx4Plan& p, hipStream_t s) {
  return a.E <= 128 ? launch_expert_form<DT, ACT, 2>(a, p, s) : launch_expert_form<DT, ACT, 8>(a, p, s);
}

template <typename DT>
hipError_t launch_experts(const MxArgs& a, const Mx4Plan& p, int act, hipStream_t s) {
  if (act == kActSilu) return launch_expert_rows<DT, kActSilu>(a, p, s);
  if (act == kActGelu) return launch_expert_rows<DT, kActGelu>(a, p, s);
  return launch_expert_rows<DT, kActNone>(a, p, s);
}

// Rows up to which a product quantises them itself (us, itself / by a launch ahead:
// Qwen3-4B's qkv, gate/up with silu and down at 8 rows 6.2 / 8.4, 12.7 / 12.3, 8.6 /
// 10.2; at 16 rows 7.7 / 9.0, 15.0 / 12.9, 12.6 / 10.7).
constexpr int kMxInlineRows = 8;

// Waves of a workgroup of few rows: as many as leave none without a step, in
// rounds of equal length.
int rows_waves(int64_t K) {
  const int64_t steps = mx4_ksteps(K), rounds = (steps + kMxRowsWaves - 1) / kMxRowsWaves;
  return (int)((steps + rounds - 1) / rounds);
}

// Quantised rows ahead of the product, codes and scales: of a linear layer in the
// weights' layout (16 rows a tile), of experts row by row.
int64_t linear_codes(int64_t rows, int64_t K) { return (rows + 15) / 16 * mx4_ktiles(K) * 1024; }
int64_t linear_scales(int64_t rows, int64_t K) { return (rows + 15) / 16 * mx4_ksteps(K) * 256; }
int64_t expert_codes(int64_t rows, int64_t K) { return rows * K / 2; }  // a multiple of 16
int64_t expert_scales(int64_t rows, int64_t K) { return rows * mx4_ksteps(K) * 16; }

// Column groups of tiles whose waves hold ntw column tiles.
int64_t tile_groups(int64_t N, int act, int ntw) {
  const int64_t cols = act ? N / 2 : N, per = act ? 32 * ntw : 64 * ntw;
  return (cols + per - 1) / per;
}

}  // namespace

Mx4Plan plan_mx4(int64_t M, int64_t N, int64_t K, int act) {
  Mx4Plan p{};
  const int64_t tiles = mx4_tiles(N);
  p.pre = M > kMxInlineRows;
  // By tiles where they give half the CUs a workgroup: of 128 columns while all of
  // them run at once, else of 256 (us, 128-column tiles / 256 / few rows at a time,
  // with the quantising launch: 128 rows of 2560 x 6144 17.4 / 22.7 / 13.0, of 4096 x
  // 28672 gated 25 / 31 / 40; 333 rows of 2560 x 19456 gated 27.9 / 23.7 / 49, of
  // 2560 x 6144 17.6 / 22.6 / 21.3, of 9728 x 2560 31 / 49 / 21.8; 1024 rows of
  // 4096 x 2560 22 / 30 / 25).
  const int64_t row_tiles = (M + kMxTileM - 1) / kMxTileM;
  int64_t col_groups = tile_groups(N, act, 2);
  if (M > 64 && row_tiles * col_groups >= device_cu_count() / 2) {
    p.tile = true;
    p.ntw = row_tiles * col_groups > device_cu_count() ? 4 : 2;
    col_groups = tile_groups(N, act, p.ntw);
    p.groups = col_groups;
    p.slots = row_tiles;
    p.grid = std::min<int64_t>((row_tiles * col_groups + 7) / 8 * 8, 2 * device_cu_count() / 8 * 8);
    p.ws_bytes = linear_codes(M, K) + linear_scales(M, K);
    return p;
  }
  p.mt = (int)std::min<int64_t>(4, (M + 15) / 16);
  p.slots = (M + 16 * p.mt - 1) / (16 * p.mt);
  // Two column tiles where the grid still fills the CUs: a row operand then serves both.
  p.ntw = act || tiles / 2 * p.slots >= device_cu_count() ? 2 : 1;
  p.groups = act ? tiles / 2 : tiles / p.ntw;
  p.grid = (p.groups + 7) / 8 * 8 * p.slots;
  p.waves = rows_waves(K);
  p.ws_bytes = p.pre ? linear_codes(M, K) + linear_scales(M, K) : 0;
  return p;
}

Mx4Plan plan_mx4_moe(int64_t num_routed, int64_t top_k, int64_t E, int64_t N, int64_t K, int act, int64_t sorted_cap) {
  Mx4Plan p{};
  const int64_t tiles = mx4_tiles(N);
  const int64_t rows = (num_routed + top_k - 1) / top_k;
  // From three rows an expert the tiles are ahead, although they quantise in a
  // launch of their own (us of both products, row by row / by tiles: E = 128, H =
  // 2048, I = 768 top-8 at 24 tokens 64 / 66, 32 70 / 75, 48 78 / 77, 96 87 / 82; E =
  // 16, H = 4096, I = 1408 top-2 at 8 tokens 31 / 37, at 24 45 / 42).  Fewer and
  // wider experts, of whose tiles there are less than CUs, were not measured.
  p.pre = num_routed > 2 * E;
  p.ws_bytes = p.pre ? expert_codes(rows, K) + expert_scales(rows, K) : 0;
  if (p.pre) {
    p.tile = true;
    p.ntw = 4;
    p.groups = tile_groups(N, act, 4);
    // Of the sorted rows, padding included, each expert has one tile more than its full ones at most.
    p.grid = (sorted_cap / kMxTileM + std::min(num_routed, E)) * p.groups / 8 * 8 + 8;
    return p;
  }
  p.mt = 1;
  p.ntw = 2;
  p.groups = tiles / 2;
  p.waves = rows_waves(K);
  // Every tile with rows at once, as far as a launch of kMx4MaxGrid workgroups goes.
  p.slots = std::max<int64_t>(1, std::min<int64_t>({num_routed, num_routed / 16 + E, kMx4MaxGrid / p.groups}));
  p.grid = p.slots * p.groups;
  return p;
}

hipError_t launch_mx4_gemm(const Mx4Params& p, const Mx4Plan& plan, hipStream_t s) {
  MxArgs a{};
  a.x = p.x;
  if (plan.pre) {
    const bool experts = p.sorted != nullptr;
    uint8_t* scales = (uint8_t*)p.ws + (experts ? expert_codes(p.rows, p.K) : linear_codes(p.rows, p.K));
    const hipError_t e = experts ? launch_mx4_rows_quantize(p.x, p.dtype, p.rows, p.K, p.ws, scales, s)
                                 : launch_mx4_tile_quantize(p.x, p.dtype, p.rows, p.K, p.ws, scales, s);
    if (e != hipSuccess) return e;
    a.x = p.ws;
    a.xs = scales;
  }
  a.w = (const char*)p.w;
  a.s = (const char*)p.s;
  a.bias = p.bias;
  a.topk_w = p.topk_w;
  a.sorted = p.sorted;
  a.offsets = p.offsets;
  a.out = p.out;
  a.M = (int)p.rows;
  a.K = (int)p.K;
  a.cols = (int)(p.act ? p.N / 2 : p.N);
  a.NT = (int)mx4_tiles(p.N);
  a.KT = (int)mx4_ktiles(p.K);
  a.KS = (int)mx4_ksteps(p.K);
  a.half = a.NT / 2;
  a.groups = (int)plan.groups;
  a.slots = (int)plan.slots;
  a.E = (int)p.E;
  a.a_div = (int)p.a_div;
  a.num_routed = (int)p.num_routed;
  a.sorted_cap = (int)p.sorted_cap;
  if (plan.tile) return p.dtype == 0 ? launch_tiles<F16>(a, plan, p.act, s) : launch_tiles<BF16>(a, plan, p.act, s);
  if (p.sorted == nullptr) return p.dtype == 0 ? launch_linear<F16>(a, plan, p.act, s) : launch_linear<BF16>(a, plan, p.act, s);
  return p.dtype == 0 ? launch_experts<F16>(a, plan, p.act, s) : launch_experts<BF16>(a, plan, p.act, s);
}

}  // namespace sgl_awq
