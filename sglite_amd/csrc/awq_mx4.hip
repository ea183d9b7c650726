// MXFP4 blocks from activations and weights, their values, and the weights'
// tile layout (awq_mx4.h).
#include "awq_launch.h"
#include "awq_mx4.h"

namespace sgl_awq {

namespace {

constexpr int kMxThreads = 256;

// What four neighbouring lanes hold of a block, 8 values each.
struct MxF32 {};

template <typename DT>
struct Vec8 {
  u32x4 v;
  __device__ __forceinline__ void load(const void* x, int64_t i) { v = ((const u32x4*)x)[i]; }
  __device__ __forceinline__ uint32_t quantize(uint32_t& byte) const { return mx4_quarter<DT>(v, byte); }
};
template <>
struct Vec8<MxF32> {
  f32x4 v[2];
  __device__ __forceinline__ void load(const void* x, int64_t i) {
    v[0] = ((const f32x4*)x)[2 * i];
    v[1] = ((const f32x4*)x)[2 * i + 1];
  }
  __device__ __forceinline__ uint32_t quantize(uint32_t& byte) const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = v[i >> 2][i & 3];  // a bit cast of the element itself would take the vector's first
      m = max(m, __builtin_bit_cast(uint32_t, f) & 0x7FFFFFFFu);
    }
    byte = mx4_byte_of(max4(m));
    const float s = mx4_scale(byte);
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0][0], v[0][1], s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0][2], v[0][3], s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[1][0], v[1][1], s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[1][2], v[1][3], s, 3);
  }
};

// Codes and scales in the order that they are kept in: a tensor of rows of whole
// blocks is one run of blocks.  Bound by memory: 28672 x 4096 bf16 in 46 to 57 us,
// 5.2 to 6.4 TB/s.
template <typename DT>
__global__ __launch_bounds__(kMxThreads) void mx4_quantize_kernel(const void* x, uint32_t* codes, uint8_t* scales,
                                                                  int64_t vecs) {
  const int64_t i = (int64_t)blockIdx.x * kMxThreads + threadIdx.x;
  if (i >= vecs) return;  // vecs is a multiple of 4: four lanes of a block leave together
  Vec8<DT> t;
  t.load(x, i);
  uint32_t byte;
  codes[i] = t.quantize(byte);
  if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
}

// The same of a product's activations, scales in the rows' order, with those of
// the blocks past K.
template <typename DT>
__global__ __launch_bounds__(kMxThreads) void mx4_rows_quantize_kernel(const void* x, uint32_t* codes, uint8_t* scales,
                                                                       uint32_t total, uint32_t kv, uint32_t ks) {
  const uint32_t i = blockIdx.x * kMxThreads + threadIdx.x;  // 8-value vectors, 64 ks a row
  if (i >= total) return;
  const uint32_t row = i / (64 * ks), v = i - row * (64 * ks);
  uint32_t byte = 0;
  if (v < kv) {
    Vec8<DT> t;
    const int64_t at = (int64_t)row * kv + v;
    t.load(x, at);
    codes[at] = t.quantize(byte);
  }
  if ((v & 3) == 0) scales[(int64_t)row * (16 * ks) + mx4_row_byte((int)(v >> 2))] = (uint8_t)byte;
}

// The same in the weights' layout: a wave takes 16 rows and NB k-tiles, a lane its
// block of each.  Rows past the last are read as the last.  With few rows a wave
// is one k-tile, with many a whole step whose scales leave as words: 128 rows of
// 14336 take 5.6 us by steps and 4.7 by k-tiles under the profiler, 8192 rows 66 to
// 70 by steps (4.3 to 4.5 TB/s).
template <typename DT, int NB>
__global__ __launch_bounds__(kMxThreads) void mx4_tile_quantize_kernel(const void* x, u32x4* codes, uint8_t* scales,
                                                                       uint32_t waves, int M, int K, int KT, int KS) {
  const uint32_t w = blockIdx.x * (kMxThreads / 64) + (threadIdx.x >> 6);
  if (w >= waves) return;
  const int lane = threadIdx.x & 63;
  const int tile = w / (4 * KS / NB), kt = (w - tile * (4 * KS / NB)) * NB;
  const u32x4* row = (const u32x4*)x + (int64_t)min(16 * tile + (lane & 15), M - 1) * (K / 8);
  u32x4 v[NB][4];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int kb = 4 * (kt + b) + (lane >> 4);
#pragma unroll
    for (int q = 0; q < 4; ++q) v[b][q] = kb * kMxBlock < K ? row[4 * kb + q] : u32x4{0, 0, 0, 0};
  }
  uint32_t word = 0;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    uint32_t byte;
    const u32x4 c = mx4_block<DT>(v[b], byte);
    word |= byte << (8 * b);
    if (kt + b < KT) codes[((int64_t)tile * KT + kt + b) * 64 + lane] = c;
  }
  uint8_t* at = scales + (((int64_t)tile * KS + (kt >> 2)) * 64 + lane) * 4 + (kt & 3);
  if constexpr (NB == 4)
    *(uint32_t*)at = word;
  else
    *at = (uint8_t)word;
}

__device__ __forceinline__ float mx4_value(uint32_t code) {
  const uint32_t m = code & 7;
  const uint32_t bits = m >= 2 ? ((m >> 1) + 126) << 23 | (m & 1) << 22 : m ? 0x3F000000u : 0u;
  return __builtin_bit_cast(float, bits | (code & 8) << 28);
}

// Values, each rounded once to the type asked for and stored past the caches: 28672
// x 4096 bf16 in 44 us, 6.7 TB/s (69 us through them).
template <typename E>
__global__ __launch_bounds__(kMxThreads) void mx4_dequantize_kernel(const uint32_t* codes, const uint8_t* scales,
                                                                    E* out, int64_t vecs) {
  typedef E V4 __attribute__((ext_vector_type(4)));
  const int64_t i = (int64_t)blockIdx.x * kMxThreads + threadIdx.x;
  if (i >= vecs) return;
  const uint32_t c = codes[i];
  const float s = mx4_scale(scales[i >> 2]);
  V4 r[2];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j >> 2][j & 3] = (E)(mx4_value(c >> (4 * j)) * s);
  __builtin_nontemporal_store(r[0], (V4*)out + 2 * i);
  __builtin_nontemporal_store(r[1], (V4*)out + 2 * i + 1);
}

// Column of MFMA row i of tile t.
__device__ __forceinline__ int tile_column(int t, int i) { return 32 * (t >> 1) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3); }

// Weights between a checkpoint's order and the tiles, one 16-byte block a thread;
// BACK restores the former.  Bound by memory: 28672 x 4096 in 24 us, a stack of 256
// weights 4096 x 4096 in 860 us, 5.2 to 5.3 TB/s read and written (a copy of its
// codes alone takes as long); back 22 and 1150 us, 5.6 and 4.0 TB/s.
template <bool BACK>
__global__ __launch_bounds__(kMxThreads) void mx4_repack_kernel(u32x4* codes, uint8_t* scales, u32x4* w, uint8_t* s,
                                                                int64_t total, int N, int KB, int NT, int KT, int KS) {
  const int64_t at = (int64_t)blockIdx.x * kMxThreads + threadIdx.x;
  if (at >= total) return;
  // at = ((expert NT + tile) 4 KS + k-tile) 64 + lane, over whole scale steps.
  const int lane = (int)(at & 63);
  int64_t q = at >> 6;
  const int kt = (int)(q % (4 * KS));
  q /= 4 * KS;
  const int t = (int)(q % NT);
  const int64_t e = q / NT;
  const int n = tile_column(t, lane & 15), kb = 4 * kt + (lane >> 4);
  const bool in = n < N && kb < KB;
  const int64_t src = (e * N + n) * KB + kb;
  const int64_t so = (((e * NT + t) * KS + (kt >> 2)) * 64 + lane) * 4 + (kt & 3);
  const int64_t wo = ((e * NT + t) * KT + kt) * 64 + lane;
  if constexpr (BACK) {
    if (in) {
      codes[src] = w[wo];
      scales[src] = s[so];
    }
  } else {
    if (kt < KT) w[wo] = in ? codes[src] : u32x4{0, 0, 0, 0};
    s[so] = in ? scales[src] : (uint8_t)0;
  }
}

dim3 blocks_for(int64_t threads) { return dim3((unsigned)((threads + kMxThreads - 1) / kMxThreads)); }

}  // namespace

hipError_t launch_mx4_quantize(const void* x, int dtype, int64_t rows, int64_t K, void* codes, void* scales,
                               hipStream_t s) {
  const int64_t vecs = rows * K / 8;
  const dim3 grid = blocks_for(vecs), block(kMxThreads);
  uint32_t* c = (uint32_t*)codes;
  uint8_t* b = (uint8_t*)scales;
  if (dtype == 0) hipLaunchKernelGGL(mx4_quantize_kernel<F16>, grid, block, 0, s, x, c, b, vecs);
  else if (dtype == 1) hipLaunchKernelGGL(mx4_quantize_kernel<BF16>, grid, block, 0, s, x, c, b, vecs);
  else hipLaunchKernelGGL(mx4_quantize_kernel<MxF32>, grid, block, 0, s, x, c, b, vecs);
  return hipGetLastError();
}

hipError_t launch_mx4_rows_quantize(const void* x, int dtype, int64_t rows, int64_t K, void* codes, void* scales,
                                    hipStream_t s) {
  const int64_t ks = mx4_ksteps(K), total = rows * ks * 64;
  const dim3 grid = blocks_for(total), block(kMxThreads);
  uint32_t* c = (uint32_t*)codes;
  uint8_t* b = (uint8_t*)scales;
  if (dtype == 0)
    hipLaunchKernelGGL(mx4_rows_quantize_kernel<F16>, grid, block, 0, s, x, c, b, (uint32_t)total, (uint32_t)(K / 8),
                       (uint32_t)ks);
  else
    hipLaunchKernelGGL(mx4_rows_quantize_kernel<BF16>, grid, block, 0, s, x, c, b, (uint32_t)total, (uint32_t)(K / 8),
                       (uint32_t)ks);
  return hipGetLastError();
}

hipError_t launch_mx4_tile_quantize(const void* x, int dtype, int64_t rows, int64_t K, void* codes, void* scales,
                                    hipStream_t s) {
  const int64_t KT = mx4_ktiles(K), KS = mx4_ksteps(K), steps = (rows + 15) / 16 * KS;
  const bool many = steps >= 4 * device_cu_count();
  const int64_t waves = many ? steps : 4 * steps;
  const dim3 grid = blocks_for(waves * 64), block(kMxThreads);
  const auto kernel = dtype == 0 ? (many ? mx4_tile_quantize_kernel<F16, 4> : mx4_tile_quantize_kernel<F16, 1>)
                                 : (many ? mx4_tile_quantize_kernel<BF16, 4> : mx4_tile_quantize_kernel<BF16, 1>);
  hipLaunchKernelGGL(kernel, grid, block, 0, s, x, (u32x4*)codes, (uint8_t*)scales, (uint32_t)waves, (int)rows, (int)K,
                     (int)KT, (int)KS);
  return hipGetLastError();
}

hipError_t launch_mx4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t K, int dtype, void* out,
                                 hipStream_t s) {
  const int64_t vecs = rows * K / 8;
  const dim3 grid = blocks_for(vecs), block(kMxThreads);
  const uint32_t* c = (const uint32_t*)codes;
  const uint8_t* b = (const uint8_t*)scales;
  if (dtype == 0) hipLaunchKernelGGL(mx4_dequantize_kernel<_Float16>, grid, block, 0, s, c, b, (_Float16*)out, vecs);
  else if (dtype == 1) hipLaunchKernelGGL(mx4_dequantize_kernel<__bf16>, grid, block, 0, s, c, b, (__bf16*)out, vecs);
  else hipLaunchKernelGGL(mx4_dequantize_kernel<float>, grid, block, 0, s, c, b, (float*)out, vecs);
  return hipGetLastError();
}

hipError_t launch_mx4_repack(void* codes, void* scales, void* w, void* ws, int64_t E, int64_t N, int64_t K, bool back,
                             hipStream_t s) {
  const int64_t NT = mx4_tiles(N), KT = mx4_ktiles(K), KS = mx4_ksteps(K);
  const int64_t total = E * NT * KS * 256;
  const auto kernel = back ? mx4_repack_kernel<true> : mx4_repack_kernel<false>;
  hipLaunchKernelGGL(kernel, blocks_for(total), dim3(kMxThreads), 0, s, (u32x4*)codes, (uint8_t*)scales, (u32x4*)w,
                     (uint8_t*)ws, total, (int)N, (int)(K / kMxBlock), (int)NT, (int)KT, (int)KS);
  return hipGetLastError();
}

}  // namespace sgl_awq
