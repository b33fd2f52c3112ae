// Matrix product of two e4m3 tensors with a float scale per block of 128 along k (gfx950):
//
//   y[m][n] = act( sum_b sx[b][m] * sw[b][n / 128] * (x[m][b] . w[n][b]) + bias[n] + res[m][n] )
//
// One v_mfma_f32_16x16x128_f8f6f4 is exactly one block of k: it forms 16 x 16 dot products of 128
// e4m3 values from a zero accumulator, and its 4 results per lane are folded into the float sums
// with one multiply-add each.  Operands are exchanged (D[channel][row] = w x^T), so that a lane's 4
// results belong to ONE row of x and the block's factor sx * sw is one number per lane and MFMA.
// The rows of a pair of weight tiles are interleaved (tile t takes channels 8 (r / 4) + 4 t + r % 4, put
// side by side when they are copied to LDS), which leaves a lane with 8 consecutive channels of its row:
// 16-byte stores straight from the accumulators.  The order of the 128 products inside an MFMA is free (both operands are read in the
// same one), so a lane simply takes 16-byte pieces g and g + 4 of its row's 128 bytes.
//
// 16-bit outputs: 8192 x 8192, k 8192: 480 us, 2.3 PFLOP/s; 132612 x 2048, k 2048: 588 - 630 us, 1.8 PFLOP/s (all waves drain
// and meet at every block of k: matrix cores busy 45 % of the cycles, waves at waits and barriers 31 %); 33153 x 256, k
// 512: 15 us, 2.3 TB/s; 1 x 512, k 2048: 5.0 us.  Float outputs: 8192^3 897 us, 1.23 PFLOP/s.
#include <algorithm>
#include <type_traits>

#include "fss_conv_args.h"

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
  int cout, k, kblocks, act, vec;   // vec: cout, y, residual and their strides allow 16-byte accesses
  float* part;                      // k split over the grid: [splits][rows][part_ld] sums, else null
  int splits, per, part_ld;         // blocks of k per split
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

// Bounds of the activation, for half precision cut to its largest value; minimum and maximum that keep a
// NaN (v_minimum3_f32, v_maximum3_f32).
struct Limits {
  float lo, hi;
};
template <typename T> __device__ __forceinline__ Limits limits_of(int act) {
  const float top = __is_same(T, f16_t) ? 65504.f : INFINITY;
  return {act == FSS_ACT_NONE ? -top : 0.f, act == FSS_ACT_RELU6 ? 6.f : top};
}
__device__ __forceinline__ float clip(float v, const Limits& l) {
  return __builtin_elementwise_minimum(__builtin_elementwise_maximum(v, l.lo), l.hi);
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

// Bias and residual of 8 consecutive channels of a row, as far as they exist
template <typename T, bool VEC>
__device__ __forceinline__ void bias8(const MmArgs& a, int c0, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  if (a.bias == nullptr) return;
  if constexpr (VEC) {
    load8(a.bias + c0, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < a.cout) v[e] = a.bias[c0 + e];
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void residual8(const MmArgs& a, long long row, int c0, float (&v)[8]) {
  const T* res = reinterpret_cast<const T*>(a.res) + row * a.res_ld + c0;
  if constexpr (VEC) {
    load8(res, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c0 + e < a.cout ? ElemTraits<T>::load(res + e) : 0.f;
  }
}
// Stores 8 consecutive channels of a row that exists.  VEC: cout and the strides allow
// 16-byte accesses.  (Two kernels instead of a branch: a launch that does little is bound by
// fetching its instructions.)
template <typename T, bool VEC>
__device__ __forceinline__ void finish8(const MmArgs& a, long long row, int c0, const float (&v)[8]) {
  T* y = reinterpret_cast<T*>(a.y) + row * a.y_ld + c0;
  if constexpr (VEC) {
    store8(y, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < a.cout) store1(y + e, v[e]);
  }
}

// ------------------------------------------------------------------------------- few rows
// 32 channels x 16 rows per workgroup, the blocks of k dealt to its 16 waves, operands straight from
// memory to registers (lanes without a row, a channel or a piece of k read zeros past the buffer's
// end); the waves' sums are added in LDS in a fixed order, one output per thread.  Latency-bound: one
// round trip per 2048 of k, and few instructions, as fetching them is most of a launch this small.
constexpr int kFewWaves = 16;
constexpr unsigned kMmBytes = 0xe0000000u;       // window of a tile's rows: 256 rows of at most 2^23 bytes
constexpr unsigned kMmOutside = 0xf0000000u;     // an offset past it that stays past it for every k

typedef int i32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 load_piece(__amdgpu_buffer_rsrc_t rsrc, unsigned off) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)off, 0, 0));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t window(const void* base, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}

template <typename T>
__global__ void __launch_bounds__(kFewWaves * 64)
matmul_fp8_few_kernel(const MmArgs a, int chan_tiles) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int wg = blockIdx.x;
  const int n0 = wg % chan_tiles * 32;
  const long long m0 = (long long)(wg / chan_tiles) * 16;
  const int rows_left = (int)min(16ll, a.rows - m0), chans_left = a.cout - n0;

  const __amdgpu_buffer_rsrc_t bx = window(a.x + m0 * a.x_ld, kMmBytes);
  const __amdgpu_buffer_rsrc_t bw = window(a.w + (long long)n0 * a.w_ld, kMmBytes);
  const int ch = 8 * (r >> 2) + (r & 3);
  const unsigned x0 = r < rows_left ? (unsigned)(r * (int)a.x_ld) : kMmOutside;
  const unsigned w0 = ch < chans_left ? (unsigned)(ch * (int)a.w_ld) : kMmOutside;
  const unsigned w1 = ch + 4 < chans_left ? (unsigned)((ch + 4) * (int)a.w_ld) : kMmOutside;

  fss_f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  for (int kb = wave; kb < a.kblocks; kb += kFewWaves) {
    const int o0 = kb * 128 + g * 16, o1 = o0 + 64;
    const unsigned t0 = o0 < a.k ? (unsigned)o0 : kMmOutside, t1 = o1 < a.k ? (unsigned)o1 : kMmOutside;
    auto at = [](unsigned row, unsigned k) { return row >= kMmOutside || k >= kMmOutside ? kMmOutside : row + k; };
    const float sx = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
                                                   window(a.sx + kb * a.x_scale_ld + m0, rows_left * 4), r * 4, 0, 0));
    const float sw = a.sw[kb * a.w_scale_ld + (n0 >> 7)];
    Block<T> fx, f[2];
    fx.set(load_piece(bx, at(x0, t0)), load_piece(bx, at(x0, t1)));
    f[0].set(load_piece(bw, at(w0, t0)), load_piece(bw, at(w0, t1)));
    f[1].set(load_piece(bw, at(w1, t0)), load_piece(bw, at(w1, t1)));
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const fss_f32x4 p = mma<T>(f[t], fx);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(p[i], sx * sw, acc[t][i]);
    }
  }
  __shared__ float part[kFewWaves][8][64];
#pragma unroll
  for (int e = 0; e < 8; ++e) part[wave][e][lane] = acc[e >> 2][e & 3];
  __syncthreads();
  if (wave >= 8) return;
  float v = 0.f;
  for (int i = 0; i < min(kFewWaves, a.kblocks); ++i) v += part[i][wave][lane];
  const int c = 8 * g + wave;
  if (r >= rows_left || c >= chans_left) return;
  if (a.bias != nullptr) v += a.bias[n0 + c];
  if (a.res != nullptr) v += ElemTraits<T>::load(reinterpret_cast<const T*>(a.res) + (m0 + r) * a.res_ld + n0 + c);
  store1(reinterpret_cast<T*>(a.y) + (m0 + r) * a.y_ld + n0 + c, clip(v, limits_of<T>(a.act)));
}

// ------------------------------------------------------------------------------ many rows
// BM rows x BN channels per workgroup of WM x WN waves (and WK groups of them, which take turns along k).
// Blocks of k (128 bytes of every row) are copied to one of two LDS stages while the other is multiplied (more
// stages changed nothing); 16-byte chunks of a row are exchanged by an XOR with the row, so that a
// fragment's reads spread over all banks.  Rows and channels past the end and the tail of k are filled
// with zeros by out-of-range offsets.  The scales travel in the same stages (a scalar load in the loop
// would make every LDS read wait for memory, as both count on one counter): 64 rows per wave, and the
// tile's weight scales in the next one.
template <int BM, int BN, int WM, int WN, int WK> struct MmTile {
  static constexpr int kThreads = 64 * WM * WN * WK, kWaves = WM * WN;
  static constexpr int TJ = BM / WM / 16, TI = BN / WN / 16;
  static constexpr int kXPieces = BM / 8 / kWaves, kWPieces = BN / 8 / kWaves;   // 1 KiB each, per wave
  static constexpr int kSPieces = BM / 64 + 1;                                   // 256 bytes each, one per wave
  static constexpr int kXBytes = BM * 128, kWBytes = BN * 128;
  static constexpr int kStage = kXBytes + kWBytes + kSPieces * 256;
  static constexpr int kLds = 2 * WK * kStage;
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0 && TI % 2 == 0 && kSPieces <= kWaves &&
                    BM % 64 == 0 && BN % (TI * 16) == 0 && 128 % (TI * 16) == 0, "tile shape");
  static_assert(kLds <= 160 * 1024, "LDS");
};

// 64 lanes x 4 bytes to the 256 bytes of LDS at lds_dst
__device__ __forceinline__ void blds4(unsigned voff, fss_i32x4 rsrc, unsigned lds_dst) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %0, %1, 0 offen lds"
      :
      : "v"(voff), "s"(rsrc), "s"(lds_dst)
      : "memory", "m0");
}

template <typename T, bool VEC, bool PART, int BM, int BN, int WM, int WN, int WK>
__global__ void __launch_bounds__(64 * WM * WN * WK, 2)
matmul_fp8_tile_kernel(const MmArgs a, int tiles_n) {
  typedef MmTile<BM, BN, WM, WN, WK> L;
  constexpr int TJ = L::TJ, TI = L::TI;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = waves / L::kWaves, wave = waves % L::kWaves;      // group along k, wave of the group
  const int wm = wave / WN, wn = wave % WN;
  char* ring = smem + wk * 2 * L::kStage;                          // each group has stages of its own
  const unsigned ring_base = (unsigned)(size_t)(__attribute__((address_space(3))) char*)ring;

  // the tiles of one XCD are neighbours, taken in columns of 8: what runs at a time shares rows
  // and channels in its L2
  const int nwg = gridDim.x, bid = blockIdx.x;
  const int q8 = nwg >> 3, rr = nwg & 7, xcd = bid & 7;
  const int wg = (xcd < rr ? xcd * (q8 + 1) : rr * (q8 + 1) + (xcd - rr) * q8) + (bid >> 3);
  const int kb0 = PART ? blockIdx.y * a.per : 0, kcount = PART ? min(a.per, a.kblocks - kb0) : a.kblocks;
  const int kend = PART ? min(a.k, (kb0 + kcount) * 128) : a.k;
  const int tiles_m = nwg / tiles_n, band = wg / (8 * tiles_n), in_band = wg - band * 8 * tiles_n;
  const int band_m = min(8, tiles_m - band * 8);
  const long long m0 = (long long)(band * 8 + in_band % band_m) * BM;
  const int n0 = in_band / band_m * BN;
  const int rows_left = (int)min((long long)BM, a.rows - m0), chans_left = min(BN, a.cout - n0);

  const fss_i32x4 rx = dma_resource(a.x + m0 * a.x_ld, kMmBytes);
  const fss_i32x4 rw = dma_resource(a.w + (long long)n0 * a.w_ld, kMmBytes);
  unsigned xoff[L::kXPieces], woff[L::kWPieces];
  const int prow = lane >> 3, phys = lane & 7;
#pragma unroll
  for (int i = 0; i < L::kXPieces; ++i) {
    const int row = (wave * L::kXPieces + i) * 8 + prow, chunk = phys ^ ((row >> 1) & 7);
    xoff[i] = row < rows_left ? (unsigned)(row * (int)a.x_ld + chunk * 16) : kMmOutside + chunk * 16;
  }
#pragma unroll
  for (int i = 0; i < L::kWPieces; ++i) {
    const int row = (wave * L::kWPieces + i) * 8 + prow, chunk = phys ^ ((row >> 1) & 7);
    // rows of a fragment lie together: row 16 t + r of a pair holds channel 8 (r / 4) + 4 t + r % 4
    const int chan = (row & ~31) + 8 * ((row & 15) >> 2) + (row >> 4 & 1) * 4 + (row & 3);
    woff[i] = chan < chans_left ? (unsigned)(chan * (int)a.w_ld + chunk * 16) : kMmOutside + chunk * 16;
  }
  auto stage = [&](int kb, unsigned dst) {
    const unsigned k0 = (unsigned)kb * 128u;
    const bool whole = (int)k0 + 128 <= kend, past = (int)k0 >= kend;            // uniform
#pragma unroll
    for (int i = 0; i < L::kXPieces; ++i) {
      const int row = (wave * L::kXPieces + i) * 8 + prow, chunk = phys ^ ((row >> 1) & 7);
      blds16(whole || (int)k0 + chunk * 16 < kend ? xoff[i] + k0 : kMmOutside, rx,
             dst + (wave * L::kXPieces + i) * 1024);
    }
#pragma unroll
    for (int i = 0; i < L::kWPieces; ++i) {
      const int row = (wave * L::kWPieces + i) * 8 + prow, chunk = phys ^ ((row >> 1) & 7);
      blds16(whole || (int)k0 + chunk * 16 < kend ? woff[i] + k0 : kMmOutside, rw,
             dst + L::kXBytes + (wave * L::kWPieces + i) * 1024);
    }
    const unsigned sdst = dst + L::kXBytes + L::kWBytes + wave * 256;
    if (wave < BM / 64) {
      const fss_i32x4 rs = dma_resource(a.sx + kb * a.x_scale_ld + m0, past ? 0 : BM * 4);
      const int row = wave * 64 + lane;
      blds4(row < rows_left ? row * 4u : kMmOutside, rs, sdst);
    } else if (wave == BM / 64) {
      const fss_i32x4 rs = dma_resource(a.sw + kb * a.w_scale_ld + (n0 >> 7), past ? 0 : 1024);
      blds4(lane * 128 < chans_left ? lane * 4u : kMmOutside, rs, sdst);
    }
  };

  fss_f32x4 acc[TJ][TI];
#pragma unroll
  for (int j = 0; j < TJ; ++j)
#pragma unroll
    for (int i = 0; i < TI; ++i) acc[j][i] = fss_f32x4{0.f, 0.f, 0.f, 0.f};

  const int r = lane & 15, g = lane >> 4;
  const int swz = (r >> 1) & 7;
  const char* px = ring + (wm * TJ * 16 + r) * 128;
  const char* psx = ring + L::kXBytes + L::kWBytes + (wm * TJ * 16 + r) * 4;
  const char* pw = ring + L::kXBytes + (wn * TI * 16 + r) * 128;
  const char* psw = ring + L::kXBytes + L::kWBytes + BM * 4 + ((n0 & 127) + wn * TI * 16 >> 7) * 4;

  // blocks wk, wk + WK, ... of k; all groups make the same number of rounds (a round past the end of
  // k deposits zeros), as they share the barriers
  const int rounds = (kcount + WK - 1) / WK;
  stage(kb0 + wk, ring_base);
  unsigned cur = 0;
  for (int round = 0; round < rounds; ++round, cur = L::kStage - cur) {
    wait_vmcnt<0>();
    __syncthreads();       // the stage has landed for every wave, and nobody reads the other one any more
    if (round + 1 < rounds) stage(kb0 + (round + 1) * WK + wk, ring_base + L::kStage - cur);
    const float sw = *reinterpret_cast<const float*>(psw + cur);
    Block<T> fw[TI];
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const char* p = pw + cur + i * 16 * 128;
      fw[i].set(*reinterpret_cast<const uint4*>(p + ((g ^ swz) << 4)),
                *reinterpret_cast<const uint4*>(p + (((4 + g) ^ swz) << 4)));
    }
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      Block<T> fx;
      const char* p = px + cur + j * 16 * 128;
      fx.set(*reinterpret_cast<const uint4*>(p + ((g ^ swz) << 4)),
             *reinterpret_cast<const uint4*>(p + (((4 + g) ^ swz) << 4)));
      const float s = sw * *reinterpret_cast<const float*>(psx + cur + j * 64);
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        const fss_f32x4 t = mma<T>(fw[i], fx);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][i][e] = fmaf(t[e], s, acc[j][i][e]);
      }
    }
  }

  if constexpr (WK > 1) {
    // the groups' sums are added in a fixed order; the stages are free after the barrier
    static_assert(L::kLds >= (WK - 1) * L::kWaves * TJ * TI * 1024, "sums do not fit");
    fss_f32x4* part = reinterpret_cast<fss_f32x4*>(smem) + (wave * TJ * TI) * 64 + lane;
    constexpr int kGroup = L::kWaves * TJ * TI * 64;
    __syncthreads();
    if (wk > 0) {
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int i = 0; i < TI; ++i) part[(wk - 1) * kGroup + (j * TI + i) * 64] = acc[j][i];
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int z = 0; z < WK - 1; ++z) acc[j][i] += part[z * kGroup + (j * TI + i) * 64];
  }
  const Limits lim = limits_of<T>(a.act);
  // Two 16-byte pieces a and b of every row, at byte offsets oa and ob, as two stores that cover whole lines of
  // 8 rows instead of parts of 16: lanes r and r + 8 exchange their pieces b (132612 x 2048, k 2048:
  // 622 against 675 us).
  auto put2 = [&](char* base, long long ld, int row, int oa, int ob, const uint4& pa, const uint4& pb, bool in_a, bool in_b) {
    const bool upper = (r & 8) != 0;
    auto other = [](unsigned w) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)w, 0x128, 0xf, 0xf, true); };   // row_ror:8
    const uint4 q = make_uint4(other(pb.x), other(pb.y), other(pb.z), other(pb.w));
    const int row1 = row & ~8, row2 = row | 8;
    if (row1 < rows_left && (upper ? in_b : in_a))
      *reinterpret_cast<uint4*>(base + (m0 + row1) * ld + (upper ? ob : oa)) =
          make_uint4(upper ? q.x : pa.x, upper ? q.y : pa.y, upper ? q.z : pa.z, upper ? q.w : pa.w);
    if (row2 < rows_left && (upper ? in_a : in_b))
      *reinterpret_cast<uint4*>(base + (m0 + row2) * ld + (upper ? oa : ob)) =
          make_uint4(upper ? pa.x : q.x, upper ? pa.y : q.y, upper ? pa.z : q.z, upper ? pa.w : q.w);
  };
  // sums of 8 channels with bias and residual, activated
  auto final8 = [&](int i, int j, int row, int c0, bool ok, const float (&bias)[8], float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = acc[j][i + (e >> 2)][e & 3] + bias[e];
    if (a.res != nullptr && ok) {
      float t[8];
      residual8<T, VEC>(a, m0 + row, n0 + c0, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += t[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = clip(v[e], lim);
  };
  if constexpr (PART) {
#pragma unroll
    for (int i = 0; i < TI; i += 2) {
      const int c0 = (wn * TI + i) * 16 + 8 * g;
#pragma unroll
      for (int j = 0; j < TJ; ++j)
        put2(reinterpret_cast<char*>(a.part + (long long)blockIdx.y * a.rows * a.part_ld), a.part_ld * 4ll, (wm * TJ + j) * 16 + r,
             (n0 + c0) * 4, (n0 + c0) * 4 + 16, __builtin_bit_cast(uint4, acc[j][i]), __builtin_bit_cast(uint4, acc[j][i + 1]),
             c0 < chans_left, c0 < chans_left);
    }
    return;
  } else if constexpr (VEC && (sizeof(T) == 4 || TI == 4)) {
    constexpr int STEP = sizeof(T) == 4 ? 2 : 4;       // a piece pair is 8 floats, or 2 x 8 16-bit channels
#pragma unroll
    for (int i = 0; i < TI; i += STEP) {
      const int ca = (wn * TI + i) * 16 + 8 * g, cb = ca + 32;
      const bool in_a = ca < chans_left, in_b = STEP == 2 ? in_a : cb < chans_left;
      float ba[8], bb[8];
      bias8<T, VEC>(a, in_a ? n0 + ca : 0, ba);
      if constexpr (STEP == 4) bias8<T, VEC>(a, in_b ? n0 + cb : 0, bb);
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        const int row = (wm * TJ + j) * 16 + r;
        const bool ok = row < rows_left;
        float v[8];
        final8(i, j, row, ca, ok && in_a, ba, v);
        uint4 p[2];
        if constexpr (STEP == 4) {
          store8(reinterpret_cast<T*>(&p[0]), v);
          final8(i + 2, j, row, cb, ok && in_b, bb, v);
          store8(reinterpret_cast<T*>(&p[1]), v);
        } else {
          store8(reinterpret_cast<T*>(p), v);
        }
        constexpr int ES = sizeof(T);
        put2(reinterpret_cast<char*>(a.y), a.y_ld * ES, row, (n0 + ca) * ES, STEP == 4 ? (n0 + cb) * ES : (n0 + ca) * ES + 16,
             p[0], p[1], in_a, in_b);
      }
    }
    return;
  }
  // bias once per 8 channels, the residuals of a column before its first store (the compiler would keep each
  // load behind the stores in front of it)
#pragma unroll
  for (int i = 0; i < TI; i += 2) {
    const int c0 = (wn * TI + i) * 16 + 8 * g;
    if (c0 >= chans_left) break;
    float bias[8], v[TJ][8];
    bias8<T, VEC>(a, n0 + c0, bias);
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const int row = (wm * TJ + j) * 16 + r;
      final8(i, j, row, c0, row < rows_left, bias, v[j]);
    }
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const int row = (wm * TJ + j) * 16 + r;
      if (row < rows_left) finish8<T, VEC>(a, m0 + row, n0 + c0, v[j]);
    }
  }
}

// Adds the splits in index order and finishes 8 channels of a row per thread.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) matmul_fp8_join_kernel(const MmArgs a) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int units = a.part_ld / 8;
  const long long row = i / units;
  if (row >= a.rows) return;
  const int c0 = (int)(i - row * units) * 8;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int z = 0; z < a.splits; ++z) {
    float t[8];
    load8(a.part + (z * a.rows + row) * a.part_ld + c0, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += t[e];
  }
  float t[8];
  bias8<T, VEC>(a, c0, t);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += t[e];
  if (a.res != nullptr) {
    residual8<T, VEC>(a, row, c0, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += t[e];
  }
  const Limits lim = limits_of<T>(a.act);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = clip(v[e], lim);
  finish8<T, VEC>(a, row, c0, v);
}

// 64 x 64 tiles with k split over the grid
template <typename T>
int launch_split(const MmArgs& a, hipStream_t stream) {
  typedef MmTile<64, 64, 2, 2, 2> L;
  typedef std::conditional_t<sizeof(T) == 4, float, bf16_t> M;            // which products, nothing else
  const auto kern = matmul_fp8_tile_kernel<M, true, true, 64, 64, 2, 2, 2>;
  FSS_CHECK_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, L::kLds));
  const int tiles_n = ceil_div(a.cout, 64);
  const dim3 grid((unsigned)((a.rows + 63) / 64 * tiles_n), a.splits);
  hipLaunchKernelGGL(kern, grid, dim3(L::kThreads), L::kLds, stream, a, tiles_n);
  FSS_LAUNCH_CHECK();
  const dim3 join((unsigned)((a.rows * (a.part_ld / 8) + 255) / 256));
  if (a.vec) hipLaunchKernelGGL((matmul_fp8_join_kernel<T, true>), join, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((matmul_fp8_join_kernel<T, false>), join, dim3(256), 0, stream, a);
  FSS_LAUNCH_CHECK();
  return 0;
}

template <typename T, bool VEC, int BM, int BN, int WM, int WN, int WK>
int launch_tile(const MmArgs& a, hipStream_t stream) {
  typedef MmTile<BM, BN, WM, WN, WK> L;
  const int tiles_n = ceil_div(a.cout, BN);
  const long long tiles = (a.rows + BM - 1) / BM * tiles_n;
  FSS_REQUIRE(tiles < (1ll << 32) / L::kThreads, "too many tiles");        // more threads are cut off without an error
  if (L::kLds > 64 * 1024)
    FSS_CHECK_HIP(hipFuncSetAttribute((const void*)matmul_fp8_tile_kernel<T, VEC, false, BM, BN, WM, WN, WK>,
                                      hipFuncAttributeMaxDynamicSharedMemorySize, L::kLds));
  hipLaunchKernelGGL((matmul_fp8_tile_kernel<T, VEC, false, BM, BN, WM, WN, WK>), dim3((unsigned)tiles), dim3(L::kThreads), L::kLds,
                     stream, a, tiles_n);
  FSS_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int launch_few(const MmArgs& a, hipStream_t stream) {
  const int chan_tiles = ceil_div(a.cout, 32);
  const long long groups = (a.rows + 15) / 16 * chan_tiles;                // at most 2560, see few_rows
  hipLaunchKernelGGL(matmul_fp8_few_kernel<T>, dim3((unsigned)groups), dim3(kFewWaves * 64), 0, stream, a, chan_tiles);
  FSS_LAUNCH_CHECK();
  return 0;
}

// Rules measured over 1 to 132612 rows, 19 to 8192 channels and k from 128 to 16384 (us, 16-bit outputs).
// Few rows, while their work is at most 10 blocks of k per compute unit (1 x 512, k 2048: 5.0 against 7.2;
// 300 x 1024, k 1024: 8.0 against 6.1).
bool few_rows(long long rows, int cout, int kblocks) {
  return (double)((rows + 15) / 16) * ceil_div(cout, 32) * kblocks <= 2560;      // (past 2^63 for rows near 2^40)
}
// Pieces of k for the grid, where few 64 x 64 tiles meet a long k: to one workgroup per compute unit, of 8
// blocks each at least (128 x 128, k 16384: 16 pieces 9.4 against 33.0 us whole; 512 x 512, k 8192: 4 pieces 14.3
// against 24.4; 300 x 1024, k 2048, 80 tiles: 2 pieces 9.2 against 7.8).
int splits_of(long long rows, int cout, int kblocks) {
  const long long tiles = (rows + 63) / 64 * ceil_div(cout, 64);
  if (few_rows(rows, cout, kblocks) || tiles > 64 || kblocks < 32) return 1;
  const long long splits = std::min(256 / tiles, (long long)kblocks / 8);
  return (int)std::min(splits, 16ll);
}

template <typename T>
int launch_matmul(const MmArgs& a, hipStream_t stream) {
  auto tiles = [&](int bm, int bn) { return (a.rows + bm - 1) / bm * ceil_div(a.cout, bn); };
  if (few_rows(a.rows, a.cout, a.kblocks)) return launch_few<T>(a, stream);
  if (a.splits > 1) return launch_split<T>(a, stream);
#define FSS_TILE(...) \
  return a.vec ? launch_tile<T, true, __VA_ARGS__>(a, stream) : launch_tile<T, false, __VA_ARGS__>(a, stream)
  // 256 x 256 where they fill whole rounds of the 256 compute units and k is long enough to hide a tile's
  // ends (8192 x 8192, k 8192: 485 against 560; 33153 x 1024, k 2048, 2.03 rounds: 110 against 94);
  const long long big = tiles(256, 256), rounds = (big + 255) / 256;
  if (big >= 240 && big * 10 >= rounds * 256 * 9 && a.kblocks >= 8) FSS_TILE(256, 256, 2, 4, 1);
  // 128 x 128 from three per compute unit (33153 x 1024, k 2048: 94 against 129; 8385 x 1024, k 1024,
  // 528 tiles: 24.0 against 21.7);
  if (tiles(128, 128) >= 768) FSS_TILE(128, 128, 2, 2, 1);
  // 64 x 64 with two groups of waves along k where the chain of its blocks is what takes the time (2145 x
  // 512, k 2048: 10.0 against 11.6; 8385 x 256, k 1024: 11.4 against 9.3), else with one.
  if (tiles(64, 64) <= 512 && a.kblocks >= 8) FSS_TILE(64, 64, 2, 2, 2);
  FSS_TILE(64, 64, 2, 2, 1);
#undef FSS_TILE
}

size_t workspace_of(const fss_matmul_fp8_desc& d) {
  const int splits = splits_of(d.rows, d.cout, ceil_div(d.k, 128));
  return splits == 1 ? 0 : (size_t)splits * d.rows * ceil_div(d.cout, 8) * 8 * sizeof(float);
}

int check_desc(const fss_matmul_fp8_desc* d) {
  FSS_REQUIRE(d != nullptr, "null descriptor");
  FSS_REQUIRE(d->rows >= 0 && d->rows < (1ll << 40), "rows must be in [0, 2^40)");
  FSS_REQUIRE(d->cout > 0 && d->cout < (1 << 28), "cout must be in [1, 2^28)");
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
  *bytes = workspace_of(*desc);
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
  a.vec = d.cout % 8 == 0 && (((uintptr_t)y | (uintptr_t)residual) & 15) == 0 && d.y_ld * es % 16 == 0 &&
          (residual == nullptr || d.res_ld * es % 16 == 0);
  const size_t need = workspace_of(d);
  FSS_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
              "workspace missing, too small or unaligned");
  a.splits = splits_of(d.rows, d.cout, a.kblocks);
  a.per = ceil_div(a.kblocks, a.splits);
  a.splits = ceil_div(a.kblocks, a.per);
  a.part = (float*)workspace;
  a.part_ld = ceil_div(d.cout, 8) * 8;
  hipStream_t s = (hipStream_t)stream;
  if (d.out_dtype == FSS_F32) return launch_matmul<float>(a, s);
  if (d.out_dtype == FSS_BF16) return launch_matmul<bf16_t>(a, s);
  if (d.out_dtype == FSS_F16) return launch_matmul<f16_t>(a, s);
  return launch_matmul<f32s_t>(a, s);
}

}  // extern "C"
