// Storage conversion to 8-bit floating point with one float scale per block of 128 columns (gfx950):
//
//   a = max(largest |x| of the block, 2^-100),  s = a / 448,  q = e4m3(448 x / a)
//
// for blocks of 1 row (activations) or 128 rows (weights).  HBM-bound: x is read once, q (one
// byte) and the scales (4 bytes per 128 or 16384 elements) are written once; a block's values stay in
// registers between its maximum and its conversion.  132612 x 2048 bfloat16: 142 to 157 us, 5.2 to 5.8
// TB/s, split-bfloat16 232 us, 5.9 TB/s; 2048 x 4096 floats in 128 x 128 blocks: 8.1 us, 5.2 TB/s; 1 x 512: 3.2
// us, a launch.
#include <algorithm>

#include "fss_common.h"

namespace fss {
namespace {

constexpr float kE4m3Max = 448.f;
constexpr unsigned kTinyBits = 0x0d800000u;      // 2^-100: blocks below it (zeros) share its scale
constexpr unsigned kInfBits = 0x7f800000u;
constexpr long long kMaxGrid256 = (1ll << 24) - 1;       // workgroups of 256

// 16 consecutive elements as floats
template <typename T>
__device__ __forceinline__ void load16(const T* p, float (&v)[16]) {
  constexpr int N = Chunk<T>::N;
#pragma unroll
  for (int i = 0; i < 16 / N; ++i) {
    Chunk<T> c;
    c.load(p + i * N);
#pragma unroll
    for (int e = 0; e < N; ++e) v[i * N + e] = c.v[e];
  }
}

// Largest magnitude as bits: orders like the floats, and a NaN is above every number, so that it
// is never lost the way fmaxf loses it.
__device__ __forceinline__ unsigned amax16(const float (&v)[16]) {
  unsigned a = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) a = max(a, __float_as_uint(v[e]) & 0x7fffffffu);
  return a;
}

__device__ __forceinline__ void scale_of(unsigned amax_bits, float& a, float& scale, float& inv) {
  a = __uint_as_float(max(amax_bits, kTinyBits));
  scale = amax_bits < kInfBits ? a / kE4m3Max : __uint_as_float(0x7fc00000u);
  inv = amax_bits < kInfBits ? kE4m3Max / a : __uint_as_float(0x7fc00000u);
}

// The byte of one element whose quotient 448 x / a lies within 2^-20 of a midpoint: `hi` and `lo` are
// the two e4m3 neighbours.  Compares 448 |x| with mid * a (both over 512: no overflow).  16-bit types hold at most
// 11 bits, so that in float 0.875 |x| is exact, and the side that the fused difference is on; floats, and the sums of
// two bfloat16 values with a gap between them, have up to 24 bits and take both products in double.
template <typename T> __device__ __forceinline__ unsigned settle(unsigned hi, unsigned lo, float x, float a) {
  const float mid = 0x1p-10f * (fabsf(__builtin_amdgcn_cvt_f32_fp8((int)hi, 0)) + fabsf(__builtin_amdgcn_cvt_f32_fp8((int)lo, 0)));
  float above;
  if constexpr (sizeof(T) == 4) above = (float)(0.875 * fabs((double)x) - (double)mid * (double)a);
  else above = fmaf(-mid, a, 0.875f * fabsf(x));
  return above > 0.f || (above == 0.f && (lo & 1)) ? hi : lo;
}

// In float, x * (448 / a) is within 2^-22 of the quotient.  Rounding it with 448 / a made larger and smaller by 2^-21
// gives the same byte unless a midpoint lies between, and then it is the quotient's byte; where the two
// differ (ties are common: bfloat16 values over a bfloat16 maximum), settle decides.
template <typename T> __device__ __forceinline__ uint4 to_fp8(const float (&v)[16], float inv, float a) {
  const float more = inv * (1.f + 0x1p-21f), less = inv * (1.f - 0x1p-21f);
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float* x = v + 4 * i;
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * more, x[1] * more, 0, false);
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * less, x[1] * less, 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * more, x[3] * more, hi, true);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * less, x[3] * less, lo, true);
    w[i] = (unsigned)lo;
    if (hi != lo) {
      unsigned r = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned h = (unsigned)hi >> (8 * e) & 0xffu, l = (unsigned)lo >> (8 * e) & 0xffu;
        r |= (h == l ? l : settle<T>(h, l, x[e], a)) << (8 * e);
      }
      w[i] = r;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Blocks of one row: 8 lanes x 16 columns hold one block, a workgroup 32 rows x 1 block column, so
// that its scales are 32 consecutive floats.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T* __restrict__ x, long long x_ld, uint8_t* __restrict__ q, long long q_ld,
                     float* __restrict__ scales, long long scale_ld, long long rows, int cols, int col_blocks) {
  const long long wg = blockIdx.x;
  const int kb = (int)(wg % col_blocks);
  const long long row = wg / col_blocks * 32 + (threadIdx.x >> 3);
  const int part = threadIdx.x & 7, col = kb * 128 + part * 16;
  const bool in = row < rows && col < cols;
  float v[16];
  if (in) load16(x + row * x_ld + col, v);
  else {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = 0.f;
  }
  unsigned a = amax16(v);
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) a = max(a, (unsigned)__shfl_xor((int)a, d));
  float top, scale, inv;
  scale_of(a, top, scale, inv);
  if (in) *reinterpret_cast<uint4*>(q + row * q_ld + col) = to_fp8<T>(v, inv, top);
  if (part == 0 && row < rows) scales[kb * scale_ld + row] = scale;
}

// Blocks of 128 x 128: one workgroup each.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_tiles_kernel(const T* __restrict__ x, long long x_ld, uint8_t* __restrict__ q, long long q_ld,
                      float* __restrict__ scales, long long scale_ld, long long rows, int cols, int col_blocks) {
  const long long wg = blockIdx.x;
  const int kb = (int)(wg % col_blocks);
  const long long rb = wg / col_blocks;
  const int col = kb * 128 + (threadIdx.x & 7) * 16;
  float v[4][16];
  unsigned a = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long row = rb * 128 + i * 32 + (threadIdx.x >> 3);
    if (row < rows && col < cols) load16(x + row * x_ld + col, v[i]);
    else {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[i][e] = 0.f;
    }
    a = max(a, amax16(v[i]));
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) a = max(a, (unsigned)__shfl_xor((int)a, d));
  __shared__ unsigned wave_max[4];
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = a;
  __syncthreads();
  a = max(max(wave_max[0], wave_max[1]), max(wave_max[2], wave_max[3]));
  float top, scale, inv;
  scale_of(a, top, scale, inv);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long row = rb * 128 + i * 32 + (threadIdx.x >> 3);
    if (row < rows && col < cols) *reinterpret_cast<uint4*>(q + row * q_ld + col) = to_fp8<T>(v[i], inv, top);
  }
  if (threadIdx.x == 0) scales[kb * scale_ld + rb] = scale;
}

}  // namespace
}  // namespace fss

using namespace fss;

extern "C" int fss_quantize_fp8(const void* x, long long x_ld, void* q, long long q_ld, float* scales,
                                long long scale_ld, long long rows, int cols, int block_rows, int dtype,
                                void* stream) {
  FSS_REQUIRE(dtype == FSS_F32 || dtype == FSS_BF16 || dtype == FSS_F16 || dtype == FSS_F32_BF16X3, "bad dtype");
  FSS_REQUIRE(block_rows == 1 || block_rows == 128, "block_rows must be 1 or 128");
  FSS_REQUIRE(rows >= 0 && rows < (1ll << 40), "rows must be in [0, 2^40)");
  FSS_REQUIRE(cols > 0 && cols % 16 == 0, "cols must be a positive multiple of 16");
  if (rows == 0) return 0;
  FSS_REQUIRE(x && q && scales, "null argument");
  const int chunk = dtype == FSS_F32 ? 4 : 8;
  FSS_REQUIRE(x_ld >= cols && x_ld % chunk == 0, "x_ld must be at least cols and a multiple of 16 bytes (split: 32)");
  FSS_REQUIRE(q_ld >= cols && q_ld % 16 == 0, "q_ld must be at least cols and a multiple of 16");
  FSS_REQUIRE(((uintptr_t)x & (dtype == FSS_F32_BF16X3 ? 31 : 15)) == 0 && ((uintptr_t)q & 15) == 0 &&
              ((uintptr_t)scales & 3) == 0, "unaligned pointer");
  const long long row_blocks = (rows + block_rows - 1) / block_rows;
  FSS_REQUIRE(scale_ld >= row_blocks, "scale_ld is less than the number of row blocks");
  const int col_blocks = ceil_div(cols, 128);
  // A launch holds fewer than 2^32 threads (more are cut off without an error): rows in parts
  const int unit = block_rows == 1 ? 32 : 128;
  FSS_REQUIRE(col_blocks <= kMaxGrid256, "too many columns");
  const long long part = kMaxGrid256 / col_blocks * unit;
  hipStream_t s = (hipStream_t)stream;
  for (long long r0 = 0; r0 < rows; r0 += part) {
    const long long n = std::min(part, rows - r0);
    const dim3 grid((unsigned)((n + unit - 1) / unit * col_blocks));
#define FSS_QUANT(T)                                                                                                 \
  do {                                                                                                               \
    const T* xp = (const T*)x + r0 * x_ld;                                                                           \
    uint8_t* qp = (uint8_t*)q + r0 * q_ld;                                                                           \
    float* sp = scales + r0 / block_rows;                                                                            \
    if (block_rows == 1)                                                                                             \
      hipLaunchKernelGGL(quantize_rows_kernel<T>, grid, dim3(256), 0, s, xp, x_ld, qp, q_ld, sp, scale_ld, n, cols,  \
                         col_blocks);                                                                                \
    else                                                                                                             \
      hipLaunchKernelGGL(quantize_tiles_kernel<T>, grid, dim3(256), 0, s, xp, x_ld, qp, q_ld, sp, scale_ld, n, cols, \
                         col_blocks);                                                                                \
  } while (0)
    if (dtype == FSS_F32) FSS_QUANT(float);
    else if (dtype == FSS_BF16) FSS_QUANT(bf16_t);
    else if (dtype == FSS_F16) FSS_QUANT(f16_t);
    else FSS_QUANT(f32s_t);
#undef FSS_QUANT
    FSS_LAUNCH_CHECK();
  }
  return 0;
}
