// Matrix product of two e4m3 tensors with a float scale per block of 128 along k (gfx950):
//
//   y[m][n] = act( sum_b sx[b][m] * sw[b][n / 128] * (x[m][b] . w[n][b]) + bias[n] + res[m][n] )
//
// One v_mfma_f32_16x16x128_f8f6f4 is exactly one block of k: it forms 16 x 16 dot products of 128
// e4m3 values from a zero accumulator, and its 4 results per lane are folded into the float sums
// with one multiply-add each.  Operands are exchanged (D[channel][row] = w x^T), so that a lane's 4
// results belong to ONE row of x and the block's factor sx * sw is one number per lane and MFMA.
// The rows of a pair of weight tiles are interleaved (tile t takes channels 8 (r / 4) + 4 t + r % 4),
// which leaves a lane with 8 consecutive channels of its row: 16-byte stores straight from the
// accumulators.  The order of the 128 products inside an MFMA is free (both operands are read in the
// same one), so a lane simply takes 16-byte pieces g and g + 4 of its row's 128 bytes.
#include <type_traits>

#include "fss_common.h"

namespace fss {
namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

struct MmArgs {
  const char* x;
  const char* w;
  const float* sx;
  const float* sw;
  const float* bias;
  const void* res;
  void* y;
  long long rows, x_ld, x_scale_ld, w_ld, w_scale_ld, res_ld, y_ld;
  int cout, k, kblocks, act, vec;   // vec: y, residual and their strides allow 16-byte accesses
};

// 16 e4m3 values of a lane as two operands of 8 half-precision values (exact)
__device__ __forceinline__ void widen(const uint4& q, uint4& lo, uint4& hi) {
  auto pair = [](unsigned w, auto high) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, decltype(high)::value));
  };
  const std::false_type l{};
  const std::true_type h{};
  lo = make_uint4(pair(q.x, l), pair(q.x, h), pair(q.y, l), pair(q.y, h));
  hi = make_uint4(pair(q.z, l), pair(q.z, h), pair(q.w, l), pair(q.w, h));
}

// One block of k for a 16-row operand, ready for the matrix cores: the 32 bytes of a lane, or the same
// values in half precision for the float outputs (T of 4 bytes), see mma.
template <typename T> struct Block {
  static constexpr bool kWide = sizeof(T) == 4;
  uint4 v[kWide ? 4 : 2];
  __device__ __forceinline__ void set(const uint4& p0, const uint4& p1) {
    if constexpr (kWide) {
      widen(p0, v[0], v[1]);
      widen(p1, v[2], v[3]);
    } else {
      v[0] = p0;
      v[1] = p1;
    }
  }
};

// The 128 products of a block.  The 8-bit matrix instructions (this one and the K = 32 form alike) align
// each group of 8 products to the largest and drop what lies below about 2^-13 of it: measured 2e-5 of
// the result's size, a tenth of a half-precision output's rounding, but visible in a float.  Float
// outputs are therefore formed from the same values in half precision (exact), at half the rate.
template <typename T>
__device__ __forceinline__ fss_f32x4 mma(const Block<T>& a, const Block<T>& b) {
  fss_f32x4 c = {0.f, 0.f, 0.f, 0.f};
  if constexpr (Block<T>::kWide) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = mfma_16x16x32<f16_t>(a.v[i], b.v[i], c);
    return c;
  } else {
    const i32x8_t x = {(int)a.v[0].x, (int)a.v[0].y, (int)a.v[0].z, (int)a.v[0].w,
                       (int)a.v[1].x, (int)a.v[1].y, (int)a.v[1].z, (int)a.v[1].w};
    const i32x8_t y = {(int)b.v[0].x, (int)b.v[0].y, (int)b.v[0].z, (int)b.v[0].w,
                       (int)b.v[1].x, (int)b.v[1].y, (int)b.v[1].z, (int)b.v[1].w};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 0, 0, 0, 0, 0, 0);
  }
}

// (comparisons instead of min / max: a NaN stays one)
__device__ __forceinline__ float activate(float v, int act) {
  if (act != FSS_ACT_NONE) v = v < 0.f ? 0.f : v;
  if (act == FSS_ACT_RELU6) v = v > 6.f ? 6.f : v;
  return v;
}
template <typename T> __device__ __forceinline__ float storable(float v) { return v; }
template <> __device__ __forceinline__ float storable<f16_t>(float v) {
  return v > 65504.f ? 65504.f : v < -65504.f ? -65504.f : v;
}

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  constexpr int N = Chunk<T>::N;
#pragma unroll
  for (int i = 0; i < 8 / N; ++i) {
    Chunk<T> c;
    c.load(p + i * N);
#pragma unroll
    for (int e = 0; e < N; ++e) v[i * N + e] = c.v[e];
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = Half16<T>::pack2(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    constexpr int N = Chunk<T>::N;
#pragma unroll
    for (int i = 0; i < 8 / N; ++i) {
      Chunk<T> c;
#pragma unroll
      for (int e = 0; e < N; ++e) c.v[e] = v[i * N + e];
      c.store(p + i * N);
    }
  }
}
// one element (slow path: odd widths and strides)
template <typename T> __device__ __forceinline__ void store1(T* p, float v) {
  if constexpr (sizeof(T) == 2) *reinterpret_cast<unsigned short*>(p) = (unsigned short)Half16<T>::bits(v);
  else ElemTraits<T>::store(p, v);
}

// Bias, residual, activation and store of 8 consecutive channels of one row.
template <typename T>
__device__ __forceinline__ void finish8(const MmArgs& a, long long row, int c0, float (&v)[8]) {
  if (row >= a.rows || c0 >= a.cout) return;
  T* y = reinterpret_cast<T*>(a.y) + row * a.y_ld + c0;
  const T* res = a.res != nullptr ? reinterpret_cast<const T*>(a.res) + row * a.res_ld + c0 : nullptr;
  if (a.vec && c0 + 8 <= a.cout) {
    if (a.bias != nullptr) {
      float b[8];
      load8(a.bias + c0, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += b[e];
    }
    if (res != nullptr) {
      float r[8];
      load8(res, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += r[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = storable<T>(activate(v[e], a.act));
    store8(y, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (c0 + e < a.cout) {
      float t = v[e];
      if (a.bias != nullptr) t += a.bias[c0 + e];
      if (res != nullptr) t += ElemTraits<T>::load(res + e);
      store1(y + e, storable<T>(activate(t, a.act)));
    }
}

// ------------------------------------------------------------------------------- few rows
// 32 channels x 16 rows per workgroup, the blocks of k dealt to its 4 waves, operands straight from
// memory to registers; the waves' sums are added in LDS in a fixed order.
constexpr int kFewWaves = 4;

template <typename T>
__global__ void __launch_bounds__(kFewWaves * 64)
matmul_fp8_few_kernel(const MmArgs a, int chan_tiles) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const long long wg = blockIdx.x;
  const int n0 = (int)(wg % chan_tiles) * 32;
  const long long m0 = wg / chan_tiles * 16;

  const long long row = m0 + r;
  const bool row_ok = row < a.rows;
  const int ch0 = n0 + 8 * (r >> 2) + (r & 3), ch1 = ch0 + 4;
  const bool ch0_ok = ch0 < a.cout, ch1_ok = ch1 < a.cout;
  const char* px = a.x + (row_ok ? row : 0) * a.x_ld + g * 16;
  const char* pw0 = a.w + (long long)(ch0_ok ? ch0 : 0) * a.w_ld + g * 16;
  const char* pw1 = a.w + (long long)(ch1_ok ? ch1 : 0) * a.w_ld + g * 16;
  const float* psx = a.sx + (row_ok ? row : 0);
  const float* psw = a.sw + (n0 >> 7);

  fss_f32x4 acc0 = {0.f, 0.f, 0.f, 0.f}, acc1 = {0.f, 0.f, 0.f, 0.f};
  const uint4 zero = make_uint4(0, 0, 0, 0);
  auto piece = [&](const char* p, int off, bool ok) {
    return ok && off + g * 16 < a.k ? *reinterpret_cast<const uint4*>(p + off) : zero;
  };
  for (int kb = wave; kb < a.kblocks; kb += kFewWaves) {
    const int o0 = kb * 128, o1 = o0 + 64;
    Block<T> fx, f0, f1;
    fx.set(piece(px, o0, row_ok), piece(px, o1, row_ok));
    f0.set(piece(pw0, o0, ch0_ok), piece(pw0, o1, ch0_ok));
    f1.set(piece(pw1, o0, ch1_ok), piece(pw1, o1, ch1_ok));
    const float s = (row_ok ? psx[kb * a.x_scale_ld] : 0.f) * psw[kb * a.w_scale_ld];
    const fss_f32x4 p0 = mma<T>(f0, fx), p1 = mma<T>(f1, fx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc0[i] = fmaf(p0[i], s, acc0[i]);
      acc1[i] = fmaf(p1[i], s, acc1[i]);
    }
  }
  __shared__ float part[kFewWaves][8][64];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    part[wave][i][lane] = acc0[i];
    part[wave][4 + i][lane] = acc1[i];
  }
  __syncthreads();
  if (wave != 0) return;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = part[0][e][lane];
#pragma unroll
    for (int i = 1; i < kFewWaves; ++i) v[e] += part[i][e][lane];
  }
  finish8<T>(a, row, n0 + 8 * g, v);
}

int check_desc(const fss_matmul_fp8_desc* d) {
  FSS_REQUIRE(d != nullptr, "null descriptor");
  FSS_REQUIRE(d->rows >= 0 && d->cout > 0, "cout must be positive, rows not negative");
  FSS_REQUIRE(d->k > 0 && d->k % 16 == 0, "k must be a positive multiple of 16");
  FSS_REQUIRE(d->out_dtype == FSS_F32 || d->out_dtype == FSS_BF16 || d->out_dtype == FSS_F16 ||
                  d->out_dtype == FSS_F32_BF16X3, "bad out_dtype");
  FSS_REQUIRE(d->act == FSS_ACT_NONE || d->act == FSS_ACT_RELU || d->act == FSS_ACT_RELU6, "bad act");
  return 0;
}

}  // namespace
}  // namespace fss

using namespace fss;

extern "C" {

int fss_matmul_fp8_workspace_bytes(const fss_matmul_fp8_desc* desc, size_t* bytes) {
  FSS_REQUIRE(bytes != nullptr, "null argument");
  if (int e = check_desc(desc)) return e;
  *bytes = 0;
  return 0;
}

int fss_matmul_fp8(const fss_matmul_fp8_desc* desc, const void* x, const float* x_scales, const void* w,
                   const float* w_scales, const float* bias, const void* residual, void* y, void* workspace,
                   size_t workspace_bytes, void* stream) {
  if (int e = check_desc(desc)) return e;
  const fss_matmul_fp8_desc& d = *desc;
  if (d.rows == 0) return 0;
  FSS_REQUIRE(x && x_scales && w && w_scales && y, "null argument");
  constexpr int64_t kMaxLd = 1 << 23;
  FSS_REQUIRE(d.x_ld >= d.k && d.x_ld % 16 == 0 && d.w_ld >= d.k && d.w_ld % 16 == 0,
              "x_ld and w_ld must be at least k and multiples of 16");
  FSS_REQUIRE(d.x_ld < kMaxLd && d.w_ld < kMaxLd, "x_ld and w_ld must be below 2^23");
  FSS_REQUIRE(d.x_scale_ld >= d.rows && d.w_scale_ld >= ceil_div(d.cout, 128), "scale stride too small");
  FSS_REQUIRE(d.y_ld >= d.cout && (residual == nullptr || d.res_ld >= d.cout), "y_ld or res_ld is less than cout");
  const int es = d.out_dtype == FSS_BF16 || d.out_dtype == FSS_F16 ? 2 : 4;
  const int align = d.out_dtype == FSS_F32_BF16X3 ? 32 : es;
  FSS_REQUIRE((((uintptr_t)x | (uintptr_t)w | (uintptr_t)bias) & 15) == 0, "x, w and bias must be 16-byte aligned");
  FSS_REQUIRE((((uintptr_t)x_scales | (uintptr_t)w_scales) & 3) == 0, "unaligned scales");
  FSS_REQUIRE((((uintptr_t)y | (uintptr_t)residual) & (align - 1)) == 0, "unaligned y or residual");
  if (d.out_dtype == FSS_F32_BF16X3)
    FSS_REQUIRE(d.cout % 8 == 0 && d.y_ld % 8 == 0 && (residual == nullptr || d.res_ld % 8 == 0),
                "split-bfloat16 output needs cout, y_ld and res_ld in multiples of 8");
  MmArgs a;
  a.x = (const char*)x; a.w = (const char*)w; a.sx = x_scales; a.sw = w_scales; a.bias = bias;
  a.res = residual; a.y = y;
  a.rows = d.rows; a.x_ld = d.x_ld; a.x_scale_ld = d.x_scale_ld; a.w_ld = d.w_ld; a.w_scale_ld = d.w_scale_ld;
  a.res_ld = d.res_ld; a.y_ld = d.y_ld;
  a.cout = d.cout; a.k = d.k; a.kblocks = ceil_div(d.k, 128); a.act = d.act;
  a.vec = (((uintptr_t)y | (uintptr_t)residual) & 15) == 0 && d.y_ld * es % 16 == 0 &&
          (residual == nullptr || d.res_ld * es % 16 == 0);
  hipStream_t s = (hipStream_t)stream;
  const int chan_tiles = ceil_div(d.cout, 32);
  const long long groups = (d.rows + 15) / 16 * chan_tiles;
  FSS_REQUIRE(groups < 0x7fffffffLL, "too many tiles");
#define FSS_MM(T) \
  hipLaunchKernelGGL(matmul_fp8_few_kernel<T>, dim3((unsigned)groups), dim3(kFewWaves * 64), 0, s, a, chan_tiles)
  if (d.out_dtype == FSS_F32) FSS_MM(float);
  else if (d.out_dtype == FSS_BF16) FSS_MM(bf16_t);
  else if (d.out_dtype == FSS_F16) FSS_MM(f16_t);
  else FSS_MM(f32s_t);
#undef FSS_MM
  FSS_LAUNCH_CHECK();
  return 0;
}

}  // extern "C"
