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

#include "awq_buffer.h"
#include "awq_epilogue.h"
#include "awq_launch.h"
#include "awq_mx4.h"
#include "awq_rowtiles.h"

namespace sgl_awq {

namespace {

struct MxArgs {
  const void* x;       // activations, or their codes
  const uint8_t* xs;   // the codes' scales, in the rows' order
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
// a gate tile and its up tile); its waves take k-tiles in turn, load weights
// straight into MFMA operands and meet in LDS at the end.  PRE: the rows come
// quantised; else a lane's 32 values are one block, which it quantises itself.
template <typename DT, bool PRE, int MT, int NTW, int ACT, int EPL>
struct RowsBody {
  using E = typename DT::elem;
  using V4 = typename DT::vec4;
  using V8 = typename DT::vec8;
  static constexpr int D = !PRE && MT > 1 ? 2 : 4;  // k-tiles in flight
  static constexpr int kPolicy = MT == 4 ? 0 : kCacheStream;

  struct Stage {
    u32x4 w[NTW], x[MT][PRE ? 1 : 4];
    uint32_t sw[NTW], sx[MT];
  };

  const MxArgs& a;
  const int wave, waves, lane;
  __amdgpu_buffer_rsrc_t wr[NTW], sr[NTW], xr, xsr;
  uint32_t xo[MT], xso[MT];

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
  // Row of the lane in m-tile mt, relative to the ranges' first; -1 for none.
  __device__ __forceinline__ void set_row(int mt, int row) {
    const int g = lane >> 4;
    xo[mt] = row < 0 ? kPastEnd : PRE ? (uint32_t)row * (uint32_t)(a.K / 2) + 16u * g : (uint32_t)row * (uint32_t)a.K * 2u + 64u * g;
    xso[mt] = row < 0 ? kPastEnd : (uint32_t)row * (uint32_t)(a.KS * 16) + 4u * g;
  }
  __device__ __forceinline__ void load(Stage& st, int kt) const {
    const uint32_t past = kt < a.KT ? 0u : kPastEnd;
    const uint32_t dead = kt * 128 + 32 * (lane >> 4) < a.K ? 0u : kPastEnd;  // K is a multiple of 32
#pragma unroll
    for (int j = 0; j < NTW; ++j) {
      st.w[j] = __builtin_amdgcn_raw_buffer_load_b128(wr[j], (uint32_t)lane * 16u | past, kt * 1024, kPolicy);
      st.sw[j] = __builtin_amdgcn_raw_buffer_load_b8(sr[j], ((uint32_t)lane * 4u + (kt & 3)) | past, (kt >> 2) * 256, 0);
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if constexpr (PRE) {
        st.x[mt][0] = __builtin_amdgcn_raw_buffer_load_b128(xr, xo[mt] | dead, kt * 64, 0);
        st.sx[mt] = __builtin_amdgcn_raw_buffer_load_b8(xsr, (xso[mt] + (kt & 3)) | dead, (kt >> 2) * 16, 0);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          st.x[mt][q] = __builtin_amdgcn_raw_buffer_load_b128(xr, (xo[mt] + 16u * q) | dead, kt * 256, 0);
      }
    }
  }
  __device__ __forceinline__ void mul(Stage& st, f32x4 (&acc)[MT][NTW]) const {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      u32x4 x;
      uint32_t sx;
      if constexpr (PRE) {
        x = st.x[mt][0];
        sx = st.sx[mt];
      } else {
        x = mx4_block<DT>(st.x[mt], sx);
      }
#pragma unroll
      for (int j = 0; j < NTW; ++j) acc[mt][j] = mfma_mx4<0, 0>(st.w[j], x, st.sw[j], sx, acc[mt][j]);
    }
  }
  // The wave's k-tiles, and every wave's sums in red.
  __device__ __forceinline__ void run(f32x4* red) const {
    f32x4 acc[MT][NTW];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < NTW; ++j) acc[mt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    Stage st[D];
#pragma unroll
    for (int d = 0; d < D; ++d) load(st[d], wave + d * waves);
    // Whole rounds of D: a k-tile past the last one loads zeros.
    for (int kt = wave; kt < a.KT; kt += D * waves) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        mul(st[d], acc);
        load(st[d], kt + (D + d) * waves);
      }
    }
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
  // m-tile mt's outputs of row `row` of out: the lane's 4 columns of each tile.
  __device__ __forceinline__ void store(const f32x4* red, int mt, int64_t row, int group, float rw) const {
    const int g = lane >> 4;
    E* out = (E*)a.out + row * a.cols;
    if constexpr (ACT != kActNone) {
      const int n = 32 * (group >> 1) + 8 * g + 4 * (group & 1);
      const f32x4 gate = biased(sum(red, mt, 0), n, rw), up = biased(sum(red, mt, 1), a.cols + n, rw);
      V4 r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = (E)(gated_act(ACT, gate[i]) * up[i]);
      *(V4*)(out + n) = r;
    } else {
      const int t = group * NTW, n = 32 * (t >> 1) + 8 * g + 4 * (t & 1);
      if (n >= a.cols) return;  // N is a multiple of 8
#pragma unroll
      for (int j = 0; j < NTW; ++j) {
        const f32x4 v = biased(sum(red, mt, j), n + 4 * j, rw);
        V4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = (E)v[i];
        *(V4*)(out + n + 4 * j) = r;
      }
    }
  }
};

template <typename DT, bool PRE, int MT, int NTW, int ACT>
__global__ __launch_bounds__(1024) void mx4_rows_kernel(MxArgs a) {
  extern __shared__ f32x4 red[];
  RowsBody<DT, PRE, MT, NTW, ACT, 0> b(a);
  // Workgroup b runs on XCD b % 8: all row blocks of a column group share an L2.
  const int local = blockIdx.x >> 3, group = (blockIdx.x & 7) + 8 * (local / a.slots);
  if (group >= a.groups) return;
  const int m0 = local % a.slots * 16 * MT, rows = min(16 * MT, a.M - m0);
  b.set_tiles(0, group);
  const uint32_t pitch = PRE ? a.K / 2 : a.K * 2;
  b.xr = make_rsrc((const char*)a.x + (int64_t)m0 * pitch, (uint32_t)rows * pitch);
  if constexpr (PRE) b.xsr = make_rsrc(a.xs + (int64_t)m0 * a.KS * 16, (uint32_t)rows * a.KS * 16u);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = 16 * mt + (b.lane & 15);
    b.set_row(mt, r < rows ? r : -1);
  }
  b.run(red);
  __syncthreads();
  for (int mt = b.wave; mt < MT; mt += b.waves) {
    const int r = 16 * mt + (b.lane & 15);
    if (r < rows) b.store(red, mt, m0 + r, group, 1.f);
  }
}

// The same for 16 sorted rows of one expert at a time.
template <typename DT, bool PRE, int NTW, int ACT, int EPL>
__global__ __launch_bounds__(1024) void mx4_expert_rows_kernel(MxArgs a) {
  extern __shared__ f32x4 red[];
  RowsBody<DT, PRE, 1, NTW, ACT, EPL> b(a);
  const int slot = blockIdx.x / a.groups, group = blockIdx.x - slot * a.groups, c = b.lane & 15;
  RowTiles<EPL> tiles;
  tiles.load(a.offsets, a.E, a.sorted_cap, b.lane);
  tiles.scan(16, b.lane);
  const uint32_t pitch = PRE ? a.K / 2 : a.K * 2;
  b.xr = make_rsrc(a.x, (uint32_t)a.M * pitch);
  if constexpr (PRE) b.xsr = make_rsrc(a.xs, (uint32_t)a.M * a.KS * 16u);
  for (int t = slot;; t += a.slots) {
    int e, rb, rows;
    tiles.find(t, 16, b.lane, e, rb, rows);
    if (e < 0) break;  // the same in every wave
    int sid = c < rows ? a.sorted[rb + c] : -1;
    if (sid >= a.num_routed) sid = -1;
    if (__ballot(sid >= 0) == 0) continue;  // padding alone: the same in every wave
    b.set_tiles(e, group);
    b.set_row(0, sid < 0 ? -1 : sid / a.a_div);
    b.run(red);
    __syncthreads();
    if (b.wave == 0 && sid >= 0) b.store(red, 0, sid, group, a.topk_w != nullptr ? a.topk_w[sid] : 1.f);
    __syncthreads();  // before the next tile's partial sums
  }
}

template <typename DT, bool PRE, int MT, int NTW, int ACT>
hipError_t launch_rows_form(const MxArgs& a, const Mx4Plan& p, hipStream_t s) {
  hipLaunchKernelGGL((mx4_rows_kernel<DT, PRE, MT, NTW, ACT>), dim3((unsigned)p.grid), dim3(64 * p.waves),
                     p.waves * MT * NTW * 1024, s, a);
  return hipGetLastError();
}

template <typename DT, int NTW, int ACT>
hipError_t launch_rows(const MxArgs& a, const Mx4Plan& p, hipStream_t s) {
  if (!p.pre) return launch_rows_form<DT, false, 1, NTW, ACT>(a, p, s);
  if (p.mt == 1) return launch_rows_form<DT, true, 1, NTW, ACT>(a, p, s);
  if (p.mt == 2) return launch_rows_form<DT, true, 2, NTW, ACT>(a, p, s);
  if (p.mt == 3) return launch_rows_form<DT, true, 3, NTW, ACT>(a, p, s);
  return launch_rows_form<DT, true, 4, NTW, ACT>(a, p, s);
}

template <typename DT>
hipError_t launch_linear(const MxArgs& a, const Mx4Plan& p, int act, hipStream_t s) {
  if (act == kActSilu) return launch_rows<DT, 2, kActSilu>(a, p, s);
  if (act == kActGelu) return launch_rows<DT, 2, kActGelu>(a, p, s);
  return p.ntw == 1 ? launch_rows<DT, 1, kActNone>(a, p, s) : launch_rows<DT, 2, kActNone>(a, p, s);
}

template <typename DT, bool PRE, int ACT, int EPL>
hipError_t launch_expert_form(const MxArgs& a, const Mx4Plan& p, hipStream_t s) {
  hipLaunchKernelGGL((mx4_expert_rows_kernel<DT, PRE, 2, ACT, EPL>), dim3((unsigned)p.grid), dim3(64 * p.waves),
                     p.waves * 2 * 1024, s, a);
  return hipGetLastError();
}

template <typename DT, int ACT>
hipError_t launch_expert_rows(const MxArgs& a, const Mx4Plan& p, hipStream_t s) {
  if (p.pre) return a.E <= 128 ? launch_expert_form<DT, true, ACT, 2>(a, p, s) : launch_expert_form<DT, true, ACT, 8>(a, p, s);
  return a.E <= 128 ? launch_expert_form<DT, false, ACT, 2>(a, p, s) : launch_expert_form<DT, false, ACT, 8>(a, p, s);
}

template <typename DT>
hipError_t launch_experts(const MxArgs& a, const Mx4Plan& p, int act, hipStream_t s) {
  if (act == kActSilu) return launch_expert_rows<DT, kActSilu>(a, p, s);
  if (act == kActGelu) return launch_expert_rows<DT, kActGelu>(a, p, s);
  return launch_expert_rows<DT, kActNone>(a, p, s);
}

int rows_waves(int64_t KT) { return KT >= 64 ? 16 : KT > 20 ? 8 : 4; }

// Quantised rows ahead of the product: codes, then scales.
int64_t quantized_bytes(int64_t rows, int64_t K) { return (rows * K / 2 + 15) / 16 * 16 + rows * mx4_ksteps(K) * 16; }

}  // namespace

Mx4Plan plan_mx4(int64_t M, int64_t N, int64_t K, int act) {
  Mx4Plan p{};
  const int64_t tiles = mx4_tiles(N);
  p.pre = M > 16;
  p.mt = (int)std::min<int64_t>(4, (M + 15) / 16);
  p.slots = (M + 16 * p.mt - 1) / (16 * p.mt);
  p.ntw = act || tiles / 2 * p.slots >= 256 ? 2 : 1;
  p.groups = act ? tiles / 2 : tiles / p.ntw;
  p.grid = (p.groups + 7) / 8 * 8 * p.slots;
  p.waves = rows_waves(mx4_ktiles(K));
  p.ws_bytes = p.pre ? quantized_bytes(M, K) : 0;
  return p;
}

Mx4Plan plan_mx4_moe(int64_t num_routed, int64_t top_k, int64_t E, int64_t N, int64_t K, int act) {
  Mx4Plan p{};
  const int64_t tiles = mx4_tiles(N);
  p.pre = num_routed > 4 * E;
  p.mt = 1;
  p.ntw = 2;
  p.groups = tiles / 2;
  p.waves = rows_waves(mx4_ktiles(K));
  // Every tile with rows at once, as far as a launch of kMx4MaxGrid workgroups goes.
  p.slots = std::max<int64_t>(1, std::min<int64_t>({num_routed, num_routed / 16 + E, kMx4MaxGrid / p.groups}));
  p.grid = p.slots * p.groups;
  p.ws_bytes = p.pre ? quantized_bytes((num_routed + top_k - 1) / top_k, K) : 0;
  return p;
}

hipError_t launch_mx4_gemm(const Mx4Params& p, const Mx4Plan& plan, hipStream_t s) {
  MxArgs a{};
  a.x = p.x;
  if (plan.pre) {
    uint8_t* scales = (uint8_t*)p.ws + (p.rows * p.K / 2 + 15) / 16 * 16;
    const hipError_t e = launch_mx4_rows_quantize(p.x, p.dtype, p.rows, p.K, p.ws, scales, s);
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
  if (p.sorted == nullptr) return p.dtype == 0 ? launch_linear<F16>(a, plan, p.act, s) : launch_linear<BF16>(a, plan, p.act, s);
  return p.dtype == 0 ? launch_experts<F16>(a, plan, p.act, s) : launch_experts<BF16>(a, plan, p.act, s);
}

}  // namespace sgl_awq
