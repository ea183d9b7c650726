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
  return launch_rows_act<4, 4, 2>(a, p, s);
}

}  // namespace sgl_awq
