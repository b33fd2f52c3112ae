// Attention of queries to the keys and values of another set of tokens (gfx950), one pass over the keys
// with a running maximum and sum per query:
//
//   y[i] = sum_j p[i][j] v[j] / sum_j p[i][j],   p[i][j] = exp(scale * q[i] . k[j] - max_j)
//
// The query heads that share a key / value head are rows of one problem (row r = token r / G, head r % G
// of the group), so keys and values are read once for all of them.  Both products keep a query in
// ONE matrix column: S^T = K Q^T and O^T = V^T P^T.  A lane of v_mfma_f32_32x32x16 then holds 16 scores
// of its query (column lane % 32, keys 8 (i / 4) + 4 (lane / 32) + i % 4), the softmax needs one
// exchange between lanes l and l + 32 and otherwise stays inside a lane, the rescaling of the sums is
// one factor per lane, and the rounded p are the second product's operand where they are: its 16 keys may
// be taken in any order as long as V is read in the same one, which the transposing LDS read
// (ds_read_b64_tr_b16: 4 keys x 16 channels -> 4 keys per lane) does at no cost.
//
// 2 x 16 heads of 128, 8385 queries, 8385 and 6288 keys: 1.05 ms, 0.96 PFLOP/s (matrix cores 50 %, exponentials
// and roundings 48 % of the cycles); of 64, 8385 keys: 0.72 ms, 0.80; 8 heads of 256, 4096 queries and keys: 0.17 ms,
// 0.80; 8 heads of 64, 2 x 33153 queries, 50 keys: 31 us, 4.3 TB/s; 8 x 32 heads of 128 in 8 groups, one query, 8385 keys:
// 51 us, 5.3 TB/s; 8 heads of 32, one query, 2145 keys: 8.6 us.
#include <algorithm>

#include "fss_conv_args.h"

namespace fss {
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

constexpr int kKeys = 64;              // keys per tile
constexpr float kFar = 256.f;          // see `far` in attention_kernel
constexpr int kMfma = 0x8, kDsRead = 0x100, kValu = 0x402;     // instruction classes of sched_group_barrier

struct AttnArgs {
  const char* q;
  const char* k;
  const char* v;
  char* y;
  const int32_t* lens;
  const uint8_t* mask;
  float* part_o;                       // [splits][all rows][head_dim] sums, not yet divided
  float* part_ml;                      // [splits][all rows][2]: maximum of q . k, sum
  long long qs[3], ks[3], vs[3], ys[3], ms[3];
  int batch, kv_len, kv_heads, group, rows, d, qtiles, splits, negate;
  float c;                             // |scale| * log2(e)
};

template <typename T> __device__ __forceinline__ f32x16_t mfma32(const uint4& a, const uint4& b, f32x16_t c) {
  if constexpr (__is_same(T, f16_t))
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(fss_f16x8, a), __builtin_bit_cast(fss_f16x8, b), c,
                                                  0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(fss_bf16x8, a),
                                                   __builtin_bit_cast(fss_bf16x8, b), c, 0, 0, 0);
}

// Byte layout of a K or V tile in LDS: rows of DP channels, 16-byte chunks exchanged by an XOR with
// the row so that the lanes of one read spread over all banks.  K is read as one chunk of 8 and
// more consecutive rows, V as 64 consecutive bytes of 4 consecutive rows.
template <int DP> struct Tile {
  static constexpr int kRow = DP * 2, kChunks = DP / 8, kPerLine = kRow < 256 ? 256 / kRow : 1;
  static constexpr int kBytes = kKeys * kRow;
  static constexpr int kPieces = kBytes / 1024;
  static __device__ __forceinline__ int kswz(int row) { return (row / kPerLine) & (kChunks < 16 ? kChunks - 1 : 15); }
  static __device__ __forceinline__ int vswz(int row) {
    return ((row / kPerLine) & ((kChunks < 16 ? kChunks : 16) / 4 - 1)) << 2;
  }
};

// sum + both values of a pair, in float (one v_dot2): the rounded p, as the product with v takes them, so
// that their errors partly cancel in the quotient
template <typename T> __device__ __forceinline__ float add_pair(unsigned pair, float sum) {
  if constexpr (__is_same(T, f16_t))
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(fss_f16x2, pair), __builtin_bit_cast(fss_f16x2, Half16<T>::kOnePair),
                                  sum, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(fss_bf16x2, pair),
                                           __builtin_bit_cast(fss_bf16x2, Half16<T>::kOnePair), sum, false);
}

// largest of lanes l and l + 32, in both
__device__ __forceinline__ float other_half_max(float v) {
  const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

// p is carried at 2^kUp of its size, which the quotient drops again: half precision then holds p down to 2^-39 of a
// query's largest (2^-24 as it is), so that many weak keys are not lost one by one
template <typename T> constexpr float kUp = __is_same(T, f16_t) ? 15.f : 0.f;

typedef __attribute__((address_space(3))) const char* lds_ptr;
typedef __attribute__((address_space(3))) i16x4_t* lds_tr_ptr;
__device__ __forceinline__ uint4 lds16(lds_ptr p) {
  return __builtin_bit_cast(uint4, *(const __attribute__((address_space(3))) fss_u32x4*)p);
}

template <typename T> __device__ __forceinline__ unsigned pack2_sat(float a, float b) {
  if constexpr (__is_same(T, f16_t)) {
    a = a > 65504.f ? 65504.f : a < -65504.f ? -65504.f : a;
    b = b > 65504.f ? 65504.f : b < -65504.f ? -65504.f : b;
  }
  return Half16<T>::pack2(a, b);
}

// Buffers of a tile: as many as leave LDS for three (head_dim above 64: two) workgroups of four waves per
// compute unit; two where mask loads share the counter that the copies are waited for with.
template <int DP, bool MASK> constexpr int kStages = MASK || DP > 64 ? 2 : DP > 32 ? 3 : 4;

// blds16 with a wave-uniform byte offset besides the per-lane one (which alone is checked against the
// buffer's end, less soff)
__device__ __forceinline__ void blds16_at(unsigned voff, fss_i32x4 rsrc, unsigned soff, unsigned lds_dst) {
  asm volatile(
      "s_mov_b32 m0, %3\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %0, %1, %2 offen lds"
      :
      : "v"(voff), "s"(rsrc), "s"(soff), "s"(lds_dst)
      : "memory", "m0");
}

// One masked query (row rq of its head's problem) again, without matrix instructions, so that the values of
// keys it does not see never enter: 64 keys at a time, a lane each for scores and p, then a lane for each channel.
// Same sums, in the same places.  A wave does its queries in turn: where one hidden value that is not finite
// concerns all of them, the call takes ten to twenty times as long (2 x 100 queries, 8 heads of 32, 33153 keys: 0.71 ms
// instead of 0.05).
template <typename T, int DP, bool SPLIT>
__device__ __forceinline__ void recompute_row(const AttnArgs& a, int b, int rq, int head, long long part, const char* kbase,
                                              const char* vbase, int first, int end) {
  const int lane = threadIdx.x & 63, token = rq / a.group;
  const uint4* qp = reinterpret_cast<const uint4*>(a.q + 2 * (b * a.qs[0] + token * a.qs[1] + head * a.qs[2]));
  const uint8_t* mq = a.mask + b * a.ms[0] + token * a.ms[1] + head * a.ms[2];
  constexpr int PER = (DP + 63) / 64;
  float m = -INFINITY, l = 0.f, acc[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) acc[i] = 0.f;
  for (int j0 = first; j0 < end; j0 += 64) {
    const bool seen = j0 + lane < end && mq[j0 + lane] != 0;
    const unsigned long long keys = __ballot(seen);
    if (keys == 0) continue;
    float dot = -INFINITY;
    if (seen) {
      const uint4* kp = reinterpret_cast<const uint4*>(kbase + 2 * ((j0 + lane) * a.ks[1]));
      float t = 0.f;
#pragma unroll 2
      for (int i = 0; i < a.d / 8; ++i) {
        Chunk<T> cq, ck;
        cq.load(reinterpret_cast<const T*>(qp + i));
        ck.load(reinterpret_cast<const T*>(kp + i));
#pragma unroll
        for (int e = 0; e < 8; ++e) t = fmaf(cq.v[e], ck.v[e], t);
      }
      dot = a.negate ? -t : t;
    }
    float top = dot;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    if (top > m) {
      const float alpha = __builtin_amdgcn_exp2f((m - top) * a.c);
      m = top;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] *= alpha;
    }
    const float p = seen ? Half16<T>::value(Half16<T>::bits(__builtin_amdgcn_exp2f(
                               fmaf(dot - (m == -INFINITY ? 0.f : m), a.c, kUp<T>)))) : 0.f;
    l += p;
    for (int n = 0; n < 64; n += 4) {
      const unsigned now = (unsigned)(keys >> n) & 0xfu;
      if (now == 0) continue;
      float v[4][PER];
#pragma unroll
      for (int e = 0; e < 4; ++e) {       // (a row that is seen in the place of one that is not)
        const T* vp = reinterpret_cast<const T*>(vbase) + (j0 + n + (now >> e & 1 ? e : __ffs((int)now) - 1)) * a.vs[1];
#pragma unroll
        for (int i = 0; i < PER; ++i) v[e][i] = ElemTraits<T>::load(vp + min(lane + 64 * i, a.d - 1));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float pe = __shfl(p, n + e);
        if (now >> e & 1) {
#pragma unroll
          for (int i = 0; i < PER; ++i) acc[i] = fmaf(pe, v[e][i], acc[i]);
        }
      }
    }
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x);
  if (SPLIT && lane == 0) {
    a.part_ml[part * 2] = m;
    a.part_ml[part * 2 + 1] = l;
  }
  const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int ch = lane + 64 * i;
    if (ch >= a.d) continue;
    if constexpr (SPLIT) a.part_o[part * a.d + ch] = acc[i];
    else
      reinterpret_cast<unsigned short*>(a.y)[b * a.ys[0] + token * a.ys[1] + head * a.ys[2] + ch] =
          (unsigned short)(l == 0.f ? 0u : pack2_sat<T>(acc[i] * f, 0.f));
  }
}

template <typename T, int DP, int NW, bool MASK, bool SPLIT>
__global__ void __launch_bounds__(NW * 64, DP <= 64 ? 3 : DP <= 128 || NW == 8 ? 2 : 1)
attention_kernel(const AttnArgs a) {
  typedef Tile<DP> L;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const unsigned smem_base = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;

  // Query tiles of one head follow each other and so run at about the same time, spread over all XCDs: each
  // XCD's L2 holds the keys and values once, and batch entries of different length load all XCDs alike
  // (one head per XCD instead: 1.23 against 1.12 ms for 2 x 16 heads, 8385 queries, 8385 and 6288 keys).
  const int qt = blockIdx.x % a.qtiles, rest = blockIdx.x / a.qtiles;
  const int z = rest % a.splits, bh = rest / a.splits;
  const int b = bh / a.kv_heads, hk = bh % a.kv_heads;

  int len = a.kv_len;
  if (a.lens != nullptr) len = min(max(a.lens[b], 0), a.kv_len);
  const int tiles = (len + kKeys - 1) / kKeys;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int tile0 = min(z * per, tiles), tile1 = min(tile0 + per, tiles);

  // this lane's query
  const int r = (qt * NW + wave) * 32 + col;
  const bool row_ok = r < a.rows;
  const int token = (row_ok ? r : 0) / a.group, head = hk * a.group + (row_ok ? r : 0) % a.group;
  uint4 qf[DP / 16];
  {
    const char* qp = a.q + 2 * (b * a.qs[0] + token * a.qs[1] + head * a.qs[2]);
    const unsigned flip = a.negate ? 0x80008000u : 0u;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int chunk = 2 * s + h;
      uint4 t = make_uint4(0, 0, 0, 0);
      if (row_ok && chunk * 8 < a.d) t = *reinterpret_cast<const uint4*>(qp + chunk * 16);
      qf[s] = make_uint4(t.x ^ flip, t.y ^ flip, t.z ^ flip, t.w ^ flip);
    }
  }
  const uint8_t* mp = nullptr;
  if constexpr (MASK) mp = a.mask + b * a.ms[0] + token * a.ms[1] + head * a.ms[2];
  const char* kbase = a.k + 2 * (b * a.ks[0] + hk * a.ks[2]);
  const char* vbase = a.v + 2 * (b * a.vs[0] + hk * a.vs[2]);

  f32x16_t o[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) o[i] = f32x16_t{};
  // Largest q . k so far and the sum of the p, which are exp2(c q.k - c m): one multiply-add each, the
  // rounded c m shared by all.  Its error, 2^-24 of itself, is the same factor in the sum and in the output, but far from
  // zero that factor itself leaves the range of p (f16 q and k of 5000 did).  Where some query of the wave has |c m|
  // above kFar, m is therefore taken off the scores first, exactly near the maximum.
  float m = -INFINITY, l = 0.f;
  bool far = false;

  // copies a tile to a buffer, 1 KiB pieces dealt to the waves: keys at or behind the length and channels
  // behind head_dim are zeros.  The XOR of a row is the XOR of its piece's first row and of the
  // lane's row in the piece (they share no bits), and the former takes few values per wave.
  constexpr int kMine = L::kPieces / NW, kRows = 64 / L::kChunks;
  constexpr int kKPat = DP / 32 / NW > 0 ? DP / 32 / NW : 1, kVPat = DP == 256 && NW == 1 ? 2 : 1;
  static_assert(L::kPieces % NW == 0 && kMine % kKPat == 0, "pieces per wave");
  const int lrow = lane / L::kChunks;
  unsigned koff[kKPat], voff[kVPat];
#pragma unroll
  for (int i = 0; i < kKPat; ++i) {
    const int c = lane % L::kChunks ^ L::kswz(lrow) ^ L::kswz((i * NW + wave) * kRows);
    koff[i] = c * 8 < a.d ? lrow * 2 * (unsigned)a.ks[1] + c * 16 : kDmaOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < kVPat; ++i) {
    const int c = lane % L::kChunks ^ L::vswz(lrow) ^ L::vswz((i * NW + wave) * kRows);
    voff[i] = c * 8 < a.d ? lrow * 2 * (unsigned)a.vs[1] + c * 16 : kDmaOutOfRange;
  }
  auto stage = [&](int tile, unsigned dst) {
    const int key0 = tile * kKeys, left = len - key0;
    const fss_i32x4 rk = dma_resource(kbase + 2 * (long long)key0 * a.ks[1], ~0ull);
    const fss_i32x4 rv = dma_resource(vbase + 2 * (long long)key0 * a.vs[1], ~0ull);
    if (left >= kKeys) {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int piece = i * NW + wave, row0 = piece * kRows;
        blds16_at(koff[i % kKPat], rk, row0 * 2 * (unsigned)a.ks[1], dst + piece * 1024);
        blds16_at(voff[i % kVPat], rv, row0 * 2 * (unsigned)a.vs[1], dst + L::kBytes + piece * 1024);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int piece = i * NW + wave, row0 = piece * kRows;
        const bool in = lrow + row0 < left;
        blds16_at(in ? koff[i % kKPat] : kDmaOutOfRange, rk, row0 * 2 * (unsigned)a.ks[1], dst + piece * 1024);
        blds16_at(in ? voff[i % kVPat] : kDmaOutOfRange, rv, row0 * 2 * (unsigned)a.vs[1],
                  dst + L::kBytes + piece * 1024);
      }
    }
  };
  // Mask of a tile: this lane reads 32 consecutive keys (those of score tile h) of its query, of the last tile the last 32
  // that there are, shifted when they are used (the loads of a tile are a tile ahead).
  uint4 mnext[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  auto mask_ahead = [&](int tile) {
    const int at = min(tile * kKeys + 32 * h, len - 32);
    __builtin_memcpy(&mnext[0], mp + at, 16);               // any alignment
    __builtin_memcpy(&mnext[1], mp + at + 16, 16);
  };

  // Transposing reads of V: each group of 16 lanes takes 4 keys x 16 channels.  The row XOR depends on the
  // lane alone and moves 64-byte pieces among 4 (2, 1 for short rows), hence one base per piece.
  constexpr int kVBases = L::kChunks < 16 ? L::kChunks / 4 : 4;
  lds_ptr vfrag[kVBases];
  {
    const int key = 4 * (lane >> 5) + ((lane & 15) >> 2), in64 = (lane >> 4 & 1) * 32 + (lane & 3) * 8;
#pragma unroll
    for (int i = 0; i < kVBases; ++i)
      vfrag[i] = (lds_ptr)smem + L::kBytes + key * L::kRow + ((i * 4 ^ L::vswz(key)) << 4) + in64;
  }
  lds_ptr kfrag[DP / 16];
#pragma unroll
  for (int st = 0; st < DP / 16; ++st) kfrag[st] = (lds_ptr)smem + col * L::kRow + (((2 * st + h) ^ L::kswz(col)) << 4);

  if constexpr (MASK) {
    if (tile0 < tile1 && len >= 32) {
      mask_ahead(tile0);
    } else if (tile0 < tile1 && h == 0) {
      unsigned w[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < len) w[i / 4] |= (unsigned)mp[i] << (8 * (i % 4));
      mnext[0] = make_uint4(w[0], w[1], w[2], w[3]);
      mnext[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  constexpr int NS = kStages<DP, MASK>, kTile = 2 * L::kBytes;
#pragma unroll
  for (int i = 0; i < NS - 1; ++i)
    if (tile0 + i < tile1) stage(tile0 + i, smem_base + i * kTile);
  unsigned cur = 0, ahead = (NS - 1) * kTile;
  for (int tile = tile0; tile < tile1; ++tile) {
    const int key0 = tile * kKeys, left = len - key0;
    // everything but the tiles behind this one (those that exist) has landed
    const int behind = tile1 - 1 - tile;
    if (NS > 3 && behind >= 2) wait_vmcnt<(NS > 3 ? 4 * kMine : 0)>();
    else if (NS > 2 && behind >= 1) wait_vmcnt<(NS > 2 ? 2 * kMine : 0)>();
    else wait_vmcnt<0>();
    __syncthreads();     // ... for every wave, and nobody reads the buffer refilled next any more
    // mask dwords, 4 keys each: own keys of score tile 0 and 1, exchanged with lane + 32
    unsigned md[2][4];
    if constexpr (MASK) {
      unsigned w[8] = {mnext[0].x, mnext[0].y, mnext[0].z, mnext[0].w, mnext[1].x, mnext[1].y, mnext[1].z, mnext[1].w};
      if (left < kKeys && len >= 32) {
        asm volatile("");      // keeps the shift out of the path of whole tiles
        const int shift = max(key0 + 32 * h - (len - 32), 0);      // in bytes; what comes in is behind the length: unseen
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __builtin_amdgcn_alignbit(i < 7 ? w[i + 1] : 0u, w[i], shift % 4 * 8);
#pragma unroll
        for (int n = 1; n < 8; n *= 2)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (shift & 4 * n) w[i] = i + n < 8 ? w[i + n] : 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (shift >= 32) w[i] = 0u;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const auto t = __builtin_amdgcn_permlane32_swap(w[2 * j], w[2 * j + 1], false, false);
        md[0][j] = t[0];
        md[1][j] = t[1];
      }
    }
    if constexpr (MASK) {
      if (tile + 1 < tile1) mask_ahead(tile + 1);
    }
    if (tile + NS - 1 < tile1) stage(tile + NS - 1, smem_base + ahead);

    // scores of 64 keys
    f32x16_t s[2];
    s[0] = f32x16_t{};
    s[1] = f32x16_t{};
#pragma unroll
    for (int st = 0; st < DP / 16; ++st)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
        s[kt] = mfma32<T>(lds16(kfrag[st] + cur + kt * 32 * L::kRow), qf[st], s[kt]);
    // issue order: reads four ahead of the products that take them
    __builtin_amdgcn_sched_group_barrier(kDsRead, 4, 0);
#pragma unroll
    for (int i = 0; i < DP / 8 - 4; ++i) {
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kMfma, 4, 0);
    if constexpr (MASK) {
      // (head_dim above 128: a block of its own for the selects, 153 -> 141 us for 8 heads, 2000 queries, 4096 keys,
      // head_dim 256; with 32 it costs 5 %)
      if (DP > 128 && left < kKeys) asm volatile("");
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[kt][i] = (md[kt][i / 4] >> (8 * (i % 4)) & 0xffu) != 0 ? s[kt][i] : -INFINITY;
    } else if (left < kKeys) {
      asm volatile("");      // keeps the comparisons below out of the path of whole tiles
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kt][i] = kt * 32 + 8 * (i / 4) + 4 * h + i % 4 < left ? s[kt][i] : -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kt][i]);
    top = other_half_max(top);
    // the sums are rescaled only where some query's maximum has grown (after a few tiles, hardly ever)
    if (__any(top > m) || far) {
      const float m_new = fmaxf(m, top), base = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f((m - base) * a.c);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) o[i] *= alpha;
      far = __any(fabsf(base * a.c) > kFar);
      if (far) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[kt][i] -= base;
      }
    }
    const float m_use = (far || m == -INFINITY ? 0.f : m * a.c) - kUp<T>;
    unsigned pf[2][8];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[kt][2 * i], a.c, -m_use));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[kt][2 * i + 1], a.c, -m_use));
        pf[kt][i] = Half16<T>::pack2(p0, p1);
        l = add_pair<T>(pf[kt][i], l);
      }
    // O^T += V^T P^T, 16 keys at a time
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const uint4 pb = make_uint4(pf[ks / 2][4 * (ks & 1)], pf[ks / 2][4 * (ks & 1) + 1], pf[ks / 2][4 * (ks & 1) + 2],
                                  pf[ks / 2][4 * (ks & 1) + 3]);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const lds_ptr at = vfrag[dt % kVBases] + cur + (dt / kVBases) * kVBases * 64 + ks * 16 * L::kRow;
        const uint2 v0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)at));
        const uint2 v1 =
            __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(at + 8 * L::kRow)));
        o[dt] = mfma32<T>(make_uint4(v0.x, v0.y, v1.x, v1.y), pb, o[dt]);
      }
    }
    // issue order: the exponentials of the second 32 keys between the products of the first
    constexpr int kHalf = DP / 16;                    // products per 32 keys
    __builtin_amdgcn_sched_group_barrier(kDsRead, 4, 1);
    __builtin_amdgcn_sched_group_barrier(kValu, 48, 1);
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 1);
      __builtin_amdgcn_sched_group_barrier(kDsRead, 2, 1);
      __builtin_amdgcn_sched_group_barrier(kValu, 48 / kHalf, 1);
    }
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 1);
      __builtin_amdgcn_sched_group_barrier(kDsRead, 2, 1);
    }
    cur = cur + kTile == NS * kTile ? 0 : cur + kTile;
    ahead = ahead + kTile == NS * kTile ? 0 : ahead + kTile;
  }

  l += __shfl_xor(l, 32);
  // An infinity or a NaN in the value of a key that a query does not see has met p = 0 and left a NaN: such
  // queries are left to recompute_row.  (If the sum is a NaN, so is every channel, and that is the result.)
  unsigned redo = 0;
  if constexpr (MASK) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) nan = nan || o[i][e] != o[i][e];
    const unsigned long long lanes = __ballot(nan && row_ok && l == l);
    redo = (unsigned)lanes | (unsigned)(lanes >> 32);
  }
  const bool store = row_ok && !(redo >> col & 1);
  const long long part0 = ((long long)z * a.batch * a.kv_heads + bh) * a.rows, part = part0 + r;
  if constexpr (SPLIT) {
    if (store) {
      if (h == 0) {
        a.part_ml[part * 2] = m;
        a.part_ml[part * 2 + 1] = l;
      }
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int ch = dt * 32 + 8 * j + 4 * h;
          if (ch < a.d)
            *reinterpret_cast<float4*>(a.part_o + part * a.d + ch) =
                make_float4(o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]);
        }
    }
  } else {
    const float f = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    char* yp = a.y + 2 * (b * a.ys[0] + token * a.ys[1] + head * a.ys[2]);
    // lanes l and l + 32 hold 4 channels each of 8; an exchange of two such groups leaves each lane with 8
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        unsigned w[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          w[0][e] = l == 0.f ? 0u : pack2_sat<T>(o[dt][4 * j + 2 * e] * f, o[dt][4 * j + 2 * e + 1] * f);
          w[1][e] = l == 0.f ? 0u : pack2_sat<T>(o[dt][4 * j + 4 + 2 * e] * f, o[dt][4 * j + 5 + 2 * e] * f);
        }
        const auto t0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
        const auto t1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
        const int ch = dt * 32 + 8 * (j + h);
        if (store && ch < a.d)
          *reinterpret_cast<uint4*>(yp + ch * 2) = make_uint4(t0[0], t1[0], t0[1], t1[1]);
      }
  }
  if constexpr (MASK) {
    for (; redo != 0; redo &= redo - 1) {
      const int rq = (qt * NW + wave) * 32 + __ffs((int)redo) - 1;
      recompute_row<T, DP, SPLIT>(a, b, rq, hk * a.group + rq % a.group, part0 + rq, kbase, vbase, tile0 * kKeys,
                                  min(tile1 * kKeys, len));
    }
  }
}

// y of a row's 4 channels from their joined sums
template <typename T>
__device__ __forceinline__ void store_joined(const AttnArgs& a, int row, int ch, const float4& v, float l) {
  const int bh = row / a.rows, r = row - bh * a.rows;
  const int b = bh / a.kv_heads, head = (bh - b * a.kv_heads) * a.group + r % a.group;
  const float f = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(a.y + 2 * (b * a.ys[0] + r / a.group * a.ys[1] + head * a.ys[2] + ch)) =
      make_uint2(pack2_sat<T>(v.x * f, v.y * f), pack2_sat<T>(v.z * f, v.w * f));
}
// Weight of a piece with maximum m and sum l: none without a key of the query; a NaN among its scores, which
// may have left no maximum, stays one
__device__ __forceinline__ float piece_weight(const float2& ml, float top, float c) {
  return ml.y == 0.f || ml.y != ml.y ? ml.y : __builtin_amdgcn_exp2f((ml.x - top) * c);
}
__device__ __forceinline__ void add_piece(float4& v, float w, const float4& o) {
  if (w != 0.f) v = make_float4(fmaf(w, o.x, v.x), fmaf(w, o.y, v.y), fmaf(w, o.z, v.z), fmaf(w, o.w, v.w));
}

// Joins few pieces of the key axis, weights 2^(c (m_z - max m)), in index order: one thread per 4 channels.
constexpr int kFewSplits = 8;

template <typename T>
__global__ void __launch_bounds__(256) attention_join_few_kernel(const AttnArgs a, long long all_rows) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int quads = a.d / 4;
  const long long row = i / quads;
  if (row >= all_rows) return;
  const int ch = (int)(i - row * quads) * 4;
  float2 ml[kFewSplits];
  float4 o[kFewSplits];
  float top = -INFINITY;
#pragma unroll
  for (int z = 0; z < kFewSplits; ++z) {
    const long long at = (long long)min(z, a.splits - 1) * all_rows + row;
    ml[z] = reinterpret_cast<const float2*>(a.part_ml)[at];
    o[z] = *reinterpret_cast<const float4*>(a.part_o + at * a.d + ch);
    top = fmaxf(top, ml[z].x);
  }
  float l = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int z = 0; z < kFewSplits; ++z) {
    const float w = z >= a.splits ? 0.f : piece_weight(ml[z], top, a.c);
    if (w != 0.f) l = fmaf(w, ml[z].y, l);
    add_piece(v, w, o[z]);
  }
  store_joined<T>(a, (int)row, ch, v, l);
}

// Joins many pieces: one row per workgroup; thread z forms the weight of piece z, then QP threads of 4
// channels x 256 / QP groups of pieces add them, all loads of a row in flight at once (a serial walk over 34
// pieces took 10 us), in a fixed order.
constexpr int kMaxSplits = 256;

template <typename T, int QP>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnArgs a, int all_rows) {
  constexpr int G = 256 / QP;
  __shared__ float weight[kMaxSplits], red[8];
  __shared__ float4 sums[256];
  const int row = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  float2 ml = make_float2(-INFINITY, 0.f);
  if (t < a.splits) ml = reinterpret_cast<const float2*>(a.part_ml)[(long long)t * all_rows + row];
  float top = ml.x;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
  if (lane == 0) red[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float w = piece_weight(ml, top, a.c);
  weight[t] = w;
  float l = w == 0.f ? 0.f : w * ml.y;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x);
  if (lane == 0) red[4 + wave] = l;
  __syncthreads();
  l = (red[4] + red[5]) + (red[6] + red[7]);

  const int ch = t % QP * 4;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (ch < a.d)
    for (int z = t / QP; z < a.splits; z += G) {
      const float4 o = *reinterpret_cast<const float4*>(a.part_o + ((long long)z * all_rows + row) * a.d + ch);
      add_piece(v, weight[z], o);
    }
  sums[t] = v;
  __syncthreads();
  if (t >= QP || ch >= a.d) return;
  for (int g = 1; g < G; ++g) {
    const float4 o = sums[g * QP + t];
    v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
  }
  store_joined<T>(a, row, ch, v, l);
}

struct Shape {
  int waves, qtiles, splits;
};

// Queries of a workgroup: 32 per wave, four waves from 33 queries on.  Where the query tiles do not give
// two workgroups per compute unit, the key axis is cut into pieces, joined by a second launch: of 64 keys at
// least for single waves (one query, 8 heads, 2145 keys: 34 pieces 8.4, 9 pieces 9.7, 5 pieces 11.8 us), of 512
// for four (300 queries and keys, 8 heads: whole 9.1, halves 10.5 us).  More workgroups than two per unit
// cost more in joining than they hide (100 queries, 33153 keys, 2 x 8 heads: 512 of them 31, 2048 36 us).
Shape shape_of(const fss_attention_desc& d) {
  Shape s;
  const long long rows = (long long)d.q_len * (d.q_heads / d.kv_heads);
  s.waves = rows > 32 ? 4 : 1;
  s.qtiles = ceil_div(rows, 32 * s.waves);
  const long long blocks = (long long)d.batch * d.kv_heads * s.qtiles;
  long long splits = 512 / blocks, most = d.kv_len / (s.waves == 4 ? 512 : 64);
  if (splits > most) splits = most;
  if (splits > kMaxSplits) splits = kMaxSplits;
  s.splits = splits > 1 ? (int)splits : 1;
  return s;
}

int check_desc(const fss_attention_desc* d) {
  FSS_REQUIRE(d != nullptr, "null descriptor");
  FSS_REQUIRE(d->dtype == FSS_BF16 || d->dtype == FSS_F16, "dtype must be FSS_BF16 or FSS_F16");
  FSS_REQUIRE(d->batch >= 0 && d->q_len >= 0 && d->kv_len >= 0, "negative size");
  FSS_REQUIRE(d->kv_heads > 0 && d->q_heads > 0 && d->q_heads % d->kv_heads == 0,
              "q_heads must be a positive multiple of kv_heads");
  FSS_REQUIRE(d->head_dim > 0 && d->head_dim <= 256 && d->head_dim % 8 == 0,
              "head_dim must be a multiple of 8 and at most 256");
  FSS_REQUIRE(fabsf(d->scale) < 0x1p127f, "scale must be below 2^127");       // finite in log2 units, too
  FSS_REQUIRE((long long)d->q_len * (d->q_heads / d->kv_heads) < 0x7fff0000LL && d->kv_len < 0x7fff0000, "too long");
  // (a launch holds fewer than 2^32 threads, more are cut off without an error; waves of 32 queries in ones, fours, eights)
  const long long rows = (long long)d->q_len * (d->q_heads / d->kv_heads);
  const int waves = rows <= 32 ? 1 : d->head_dim > 128 && rows > 128 ? 8 : 4;
  FSS_REQUIRE((long long)d->batch * d->kv_heads <= ((1ll << 26) - 1) / (std::max(1, ceil_div(rows, 32 * waves)) * waves),
              "too many query tiles");
  return 0;
}

size_t workspace_of(const fss_attention_desc& d, const Shape& s) {
  return s.splits == 1 ? 0 : (size_t)s.splits * d.batch * d.q_len * d.q_heads * (d.head_dim + 2) * 4;
}

template <typename T, int DP, int NW>
int launch(const AttnArgs& a, const Shape& s, hipStream_t stream) {
  const dim3 grid((unsigned)((long long)a.batch * a.kv_heads * a.qtiles * a.splits));
  // a piece of the key axis with fewer tiles than buffers touches no more buffers than it has tiles
  const int tiles = std::max(1, ceil_div(ceil_div(a.kv_len, kKeys), a.splits));
  const size_t lds = 2 * Tile<DP>::kBytes * std::min(tiles, a.mask != nullptr ? kStages<DP, true> : kStages<DP, false>);
#define FSS_ATTN(MASK, SPLIT)                                                                                       \
  do {                                                                                                              \
    if (lds > 64 * 1024)                                                                                            \
      FSS_CHECK_HIP(hipFuncSetAttribute((const void*)attention_kernel<T, DP, NW, MASK, SPLIT>,                      \
                                        hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));                     \
    hipLaunchKernelGGL((attention_kernel<T, DP, NW, MASK, SPLIT>), grid, dim3(NW * 64), lds, stream, a);            \
  } while (0)
  if (NW < 8 && a.mask != nullptr) {
    if constexpr (NW < 8) {
      if (s.splits > 1) FSS_ATTN(true, true); else FSS_ATTN(true, false);
    }
  } else {
    if (s.splits > 1) FSS_ATTN(false, true); else FSS_ATTN(false, false);
  }
#undef FSS_ATTN
  FSS_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int launch_type(const AttnArgs& a, const Shape& s, hipStream_t stream) {
#define FSS_DP(DP) return s.waves == 4 ? launch<T, DP, 4>(a, s, stream) : launch<T, DP, 1>(a, s, stream)
  if (a.d <= 32) FSS_DP(32);
  if (a.d <= 64) FSS_DP(64);
  if (a.d <= 128) FSS_DP(128);
  if (s.waves == 8) return launch<T, 256, 8>(a, s, stream);
  FSS_DP(256);
#undef FSS_DP
}

}  // namespace
}  // namespace fss

using namespace fss;

extern "C" {

int fss_cross_attention_workspace_bytes(const fss_attention_desc* desc, size_t* bytes) {
  FSS_REQUIRE(bytes != nullptr, "null argument");
  if (int e = check_desc(desc)) return e;
  *bytes = desc->batch == 0 || desc->q_len == 0 ? 0 : workspace_of(*desc, shape_of(*desc));
  return 0;
}

int fss_cross_attention(const fss_attention_desc* desc, const void* q, const void* k, const void* v,
                        const int32_t* kv_lens, const uint8_t* mask, void* y, void* workspace,
                        size_t workspace_bytes, void* stream) {
  if (int e = check_desc(desc)) return e;
  const fss_attention_desc& d = *desc;
  if (d.batch == 0 || d.q_len == 0) return 0;
  FSS_REQUIRE(q && y && ((k && v) || d.kv_len == 0), "null argument");
  for (int i = 0; i < 3; ++i) {
    const int64_t st[4] = {d.q_stride[i], d.k_stride[i], d.v_stride[i], d.y_stride[i]};
    for (int t = 0; t < 4; ++t)
      FSS_REQUIRE(st[t] >= 0 && st[t] % 8 == 0 && (i != 1 || st[t] < (1 << 24)),
                  "strides must be multiples of 8 and not negative, token strides below 2^24");
    FSS_REQUIRE(mask == nullptr || d.mask_stride[i] >= 0, "negative mask stride");
  }
  FSS_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)y | (uintptr_t)workspace) & 15) == 0 &&
                  ((uintptr_t)kv_lens & 3) == 0, "unaligned pointer");
  Shape s = shape_of(d);
  const size_t need = workspace_of(d, s);
  FSS_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), "workspace too small");
  // Eight waves with head_dim above 128, where the tiles leave LDS for one workgroup per compute unit (8 heads,
  // 4096 queries and keys, head_dim 256: 195 against 260 us); not with a mask, whose registers would
  // not fit (416 against 259 us).
  const long long rows = (long long)d.q_len * (d.q_heads / d.kv_heads);
  if (d.head_dim > 128 && rows > 128 && mask == nullptr) {
    s.waves = 8;
    s.qtiles = ceil_div(rows, 256);
  }
  AttnArgs a;
  a.q = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.y = (char*)y;
  a.lens = kv_lens; a.mask = mask;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = d.q_stride[i]; a.ks[i] = d.k_stride[i]; a.vs[i] = d.v_stride[i]; a.ys[i] = d.y_stride[i];
    a.ms[i] = d.mask_stride[i];
  }
  a.batch = d.batch; a.kv_len = d.kv_len; a.kv_heads = d.kv_heads; a.group = d.q_heads / d.kv_heads;
  a.rows = d.q_len * a.group; a.d = d.head_dim; a.qtiles = s.qtiles; a.splits = s.splits;
  a.negate = d.scale < 0.f;
  // (a scale of 0 gives equal scores; the smallest float in its place keeps 0 * infinity out)
  a.c = fmaxf(fabsf(d.scale) * 1.44269504088896340736f, 1.17549435e-38f);
  const long long all_rows = (long long)d.batch * d.q_len * d.q_heads;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + (need == 0 ? 0 : s.splits * all_rows * d.head_dim);
  hipStream_t st = (hipStream_t)stream;
  const int e = d.dtype == FSS_F16 ? launch_type<f16_t>(a, s, st) : launch_type<bf16_t>(a, s, st);
  if (e != 0 || s.splits == 1) return e;
  if (s.splits <= kFewSplits) {
    const long long threads = all_rows * (d.head_dim / 4);
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (d.dtype == FSS_F16) hipLaunchKernelGGL(attention_join_few_kernel<f16_t>, grid, dim3(256), 0, st, a, all_rows);
    else hipLaunchKernelGGL(attention_join_few_kernel<bf16_t>, grid, dim3(256), 0, st, a, all_rows);
    FSS_LAUNCH_CHECK();
    return 0;
  }
  const dim3 grid((unsigned)all_rows);
#define FSS_JOIN(QP)                                                                                                 \
  do {                                                                                                               \
    if (d.dtype == FSS_F16)                                                                                          \
      hipLaunchKernelGGL((attention_join_kernel<f16_t, QP>), grid, dim3(256), 0, st, a, (int)all_rows);              \
    else                                                                                                             \
      hipLaunchKernelGGL((attention_join_kernel<bf16_t, QP>), grid, dim3(256), 0, st, a, (int)all_rows);             \
  } while (0)
  if (d.head_dim <= 32) FSS_JOIN(8);
  else if (d.head_dim <= 64) FSS_JOIN(16);
  else if (d.head_dim <= 128) FSS_JOIN(32);
  else FSS_JOIN(64);
#undef FSS_JOIN
  FSS_LAUNCH_CHECK();
  return 0;
}

}  // extern "C"
