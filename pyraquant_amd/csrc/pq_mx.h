// Microscaled 4-bit blocks (gfx950): the format, its conversions and its packed layout.
//
// 32 consecutive values of a row share one power of two 2^E, E = floor(log2(max |x|)) - 2 (at least -127), stored as the
// byte E + 127. Each value is the nearest of {0, 0.5, 1, 1.5, 2, 3, 4, 6} 2^E with its sign (1 sign, 2 exponent, 1 mantissa
// bit), ties to the even mantissa, saturated at 6. With that E the largest |x| 2^-E lies in [4, 8), so the top of the grid
// is used and only values in (7, 8) 2^E lose more than half a step. A block holding an infinity or a NaN has byte 255 (the
// whole block is NaN) and codes 0; a block of zeros has byte 0 and codes 0.
//
// The 8-bit codes of a training layer's checkpoint are rint(x 2^(4 - E)) in [-127, 127] on the same E, worth 2^(E - 4)
// each: |x| < 2^(E + 3), so seven bits and the sign cover the block, and one scale array serves both.
#pragma once

#include "pq_common.h"

namespace pq {
namespace mx {

// t = x l1t^T [M, R] in fp32 and, unless codes is NULL, the codes of x (and q8), in one pass (pq_mx.hip). K % 16 == 0 (32 with
// codes), 16-byte aligned rows, R 32 or 64, l1f: l1t in fragment order (pq_mx_factors); arguments checked by the caller.
int lowrank(const void* x, int32_t dtype, int64_t M, int64_t K, int64_t ldx, const void* l1f, int64_t R, uint8_t* codes,
            uint8_t* scales, int8_t* q8, float* t, void* workspace, hipStream_t stream);
int64_t lowrank_workspace(int64_t M, int64_t K, int64_t R);   // bytes of its workspace (0: none)

constexpr int kBlock = 32;     // values that share a scale
constexpr int kNaN = 255;      // scale byte of a block that is NaN

typedef int v8i __attribute__((ext_vector_type(8)));

// ---- packed layout ---------------------------------------------------------------------------------------------------
// A matrix [R, K] (K % 32 == 0) is cut into KT = ceil(K / 128) stages of 128 values and ceil(R / 16) row blocks.
// Codes: block (rb, kt), 1 KB at (rb KT + kt) 1024, is the packed K64 layout of the bytes (two values each, the even k in the
// low nibble): the 32 values of scale block b (of 4) of row r are the 16 bytes at 64 r + 16 (b ^ k64_swz(r)).
// Scales: 64 bytes at (rb KT + kt) 64, four for each row, in the order of blocks 0, 2, 1, 3: a matrix instruction over 64
// values takes blocks 2 s (lanes 0-31) and 2 s + 1 (lanes 32-63) in its step s, so each half reads the two bytes it needs
// as one 16-bit word. Rows past R and blocks past K are zeros.
__host__ __device__ __forceinline__ int stages(int64_t K) { return (int)((K + 127) / 128); }
__host__ __device__ __forceinline__ int64_t code_offset(int64_t row, int kt, int b, int KT) {
  const int r = (int)(row & 15);
  return ((row >> 4) * KT + kt) * 1024 + r * 64 + ((b ^ k64_swz(r)) << 4);
}
__host__ __device__ __forceinline__ int scale_slot(int b) { return (b >> 1) | ((b & 1) << 1); }
__host__ __device__ __forceinline__ int64_t scale_offset(int64_t row, int kt, int b, int KT) {
  return ((row >> 4) * KT + kt) * 64 + (row & 15) * 4 + scale_slot(b);
}

// 2^(byte - 127) as the conversion instructions take it (they read the exponent field; 0x400000 is 2^-127 itself).
__device__ __forceinline__ float scale_value(int byte) {
  return __uint_as_float(max((uint32_t)byte << 23, 0x400000u));
}

// ---- a block of 32 values in registers, as 16 words of two 16-bit values or 32 floats ------------------------------
template <int DT>
struct Block {
  static constexpr int WORDS = DT == PQ_F32 ? 32 : 16;
  uint32_t w[WORDS];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
  }
  // 32 values at p: 16-byte loads where VEC, else one by one
  template <bool VEC>
  __device__ __forceinline__ void load(const void* p) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const v4u v = reinterpret_cast<const v4u*>(p)[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * i + e] = v[e];
      }
    } else if constexpr (DT == PQ_F32) {
#pragma unroll
      for (int i = 0; i < 32; ++i) w[i] = static_cast<const uint32_t*>(p)[i];
    } else {
      const uint16_t* h = static_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
    }
  }
  __device__ __forceinline__ float value(int i) const {   // i: a constant after unrolling
    if constexpr (DT == PQ_F32) return __uint_as_float(w[i]);
    else return i & 1 ? hi16_to_f32<DT>(w[i >> 1]) : lo16_to_f32<DT>(w[i >> 1]);
  }
  // The scale byte. The largest magnitude is found on the bits without the sign, which order as the values do (and put
  // infinities and NaNs on top).
  __device__ __forceinline__ int scale_byte() const {
    uint32_t e;
    if constexpr (DT == PQ_F32) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) m = max(m, w[i] & 0x7fffffffu);
      e = m >> 23;
    } else {
      us2 m = us2{0, 0};
#pragma unroll
      for (int i = 0; i < 16; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, w[i] & 0x7fff7fffu));
      const uint32_t a = max((uint32_t)m[0], (uint32_t)m[1]);
      if constexpr (DT == PQ_BF16) e = a >> 7;
      else e = a >= 0x7c00u ? 255u : __float_as_uint(lo16_to_f32<PQ_F16>(a)) >> 23;
    }
    return e == 255u ? kNaN : max((int)e - 2, 0);
  }
  // the 4-bit codes, two to a byte
  __device__ __forceinline__ v4i codes(int byte) const {
    const float s = scale_value(byte);
    v4i c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t o = 0;
      if constexpr (DT == PQ_F32) {
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, value(8 * i + 0), value(8 * i + 1), s, 0);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, value(8 * i + 2), value(8 * i + 3), s, 1);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, value(8 * i + 4), value(8 * i + 5), s, 2);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, value(8 * i + 6), value(8 * i + 7), s, 3);
      } else if constexpr (DT == PQ_BF16) {
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(v2bf, w[4 * i + 0]), s, 0);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(v2bf, w[4 * i + 1]), s, 1);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(v2bf, w[4 * i + 2]), s, 2);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(v2bf, w[4 * i + 3]), s, 3);
      } else {
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(v2h, w[4 * i + 0]), s, 0);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(v2h, w[4 * i + 1]), s, 1);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(v2h, w[4 * i + 2]), s, 2);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(v2h, w[4 * i + 3]), s, 3);
      }
      c[i] = byte == kNaN ? 0 : (int)o;
    }
    return c;
  }
  // the 8-bit codes: x 2^(131 - byte), rounded by adding 1.5 2^23 (to nearest even; the sum's low byte is the code). ldexp,
  // not a product: below byte 4 that power of two is no float.
  __device__ __forceinline__ void codes8(int byte, v4i (&q)[2]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f = __builtin_amdgcn_ldexpf(value(4 * i + e), 131 - byte);
        f = __builtin_amdgcn_fmed3f(f, -127.0f, 127.0f) + 12582912.0f;
        b[e] = __float_as_uint(f);
      }
      const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400);
      q[i >> 2][i & 3] = byte == kNaN ? 0 : (int)(lo | (hi << 16));
    }
  }
};

// Two 4-bit values (byte SEL of `c`) as two 16-bit values times `s` (scale_value); exact for bf16, and for fp16 where the
// result is a normal or a two-bit subnormal number.
template <int DT, int SEL>
__device__ __forceinline__ uint32_t widen2(uint32_t c, float s) {
  if constexpr (DT == PQ_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, SEL));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, SEL));
}
// Eight 4-bit values (one word) as four words of two 16-bit values.
template <int DT>
__device__ __forceinline__ v4u widen8(uint32_t c, float s) {
  return v4u{widen2<DT, 0>(c, s), widen2<DT, 1>(c, s), widen2<DT, 2>(c, s), widen2<DT, 3>(c, s)};
}
template <int DT>
constexpr uint32_t nan2() { return DT == PQ_BF16 ? 0x7fc07fc0u : 0x7e007e00u; }

// Four 8-bit codes (one word) times 2^(byte - 131), as two words of two 16-bit values.
template <int DT>
__device__ __forceinline__ v2u restore4(uint32_t q, float s) {
  float f[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = (float)((int)(q << (24 - 8 * e)) >> 24) * s;
  return v2u{pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3])};
}
// 2^(byte - 131), NaN for a block that is NaN.
__device__ __forceinline__ float restore_scale(int byte) {
  return byte == kNaN ? __uint_as_float(0x7fc00000u) : __builtin_amdgcn_ldexpf(1.0f, byte - 131);
}

// t and dt are kept in fp32 and taken as two 16-bit parts by the products that read them, hi + lo: twice the bits. With the first
// alone the rounding of t shows in every result, as large as the results' own where the low-rank term is the larger one.
// hi is cut towards zero from the next value nearer zero, so that lo has the sign of the value and is no zero where hi is none: an
// infinity on the other side of a product meets two parts of one sign and gives what it gives with the value itself, where a lo of
// 0 or of the other sign would make it NaN. (An infinite value is a finite hi and an infinite lo; in fp16, whose lo must not fall
// below the smallest subnormal, hi lies at least that much nearer zero, and values under 2^-23 may have a hi of 0.)
template <int DT>
__device__ __forceinline__ void two_parts(float a, float b, uint32_t& hi, uint32_t& lo) {
  auto nearer = [](float v) { return __uint_as_float(__builtin_elementwise_sub_sat(__float_as_uint(v), 1u)); };
  a += 0.0f;   // (-0 to 0: its bits are no magnitude to step down from)
  b += 0.0f;
  if constexpr (DT == PQ_BF16) {
    hi = __builtin_amdgcn_perm(__float_as_uint(nearer(b)), __float_as_uint(nearer(a)), 0x07060302);
  } else {
    const float tiny = 0x1p-24f;
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(nearer(a) - copysignf(tiny, a), nearer(b) - copysignf(tiny, b)));
  }
  lo = pack2<DT>(a - lo16_to_f32<DT>(hi), b - hi16_to_f32<DT>(hi));
}

// ---- shared by the products ------------------------------------------------------------------------------------------
// Products of 16-bit operands, fp32 sums. From registers alone, at the power limit, 32 x 32 x 16 runs at 1.75 PFLOP/s in bf16
// and 16 x 16 x 32 at 2.0; for 4-bit operands 32 x 32 x 64 at 6.5 and 16 x 16 x 128 at 6.95. The large kernels take the 32 x 32
// shapes all the same: the others read half as much again from LDS for a block, and the product was 12 % slower with them, the
// input gradient 6-8 % in one round of blocks. 16 x 16 x 32 serves the low-rank products, whose operand is a quantizer's lane.
template <int DT>
__device__ __forceinline__ v4f mfma16_16(v4i a, v4i b, v4f c) {
  if constexpr (DT == PQ_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ v16f mfma16(v4i a, v4i b, v16f c) {
  if constexpr (DT == PQ_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// fp16 ends at 65504, and t and dt may go past it where the results do not. Values of a row (of a column, where sums run over
// rows) whose largest magnitude is 2^16 or more are taken times 2^-e, so that it falls below 2^16, and the sums that they join times
// 2^-e before and 2^e after: no bit changes. 2^-e from that largest magnitude's bits (2^-113 for an infinity: its sums are no numbers).
__device__ __forceinline__ float scale_down(uint32_t bits) {
  const int e = max((int)(bits >> 23) - 127 - 15, 0);
  return __uint_as_float((uint32_t)(127 - min(e, 113)) << 23);
}
__device__ __forceinline__ float scale_back(float down) { return __uint_as_float(0x7f000000u - __float_as_uint(down)); }   // 1 / down

// Below 2^-10 a second part is cut to fp16's smallest subnormal, and below 2^-24 nothing is left of the first. Where the sums are t's or
// dt's alone, values are therefore taken times a power of two that brings the largest of them to 2^15 .. 2^16, up or down, and what is cut off is
// 2^-40 of that one. scale_exponent: minus that power's exponent (of zeros -126, so that both powers are normal numbers; of an infinity 113).
__device__ __forceinline__ int scale_exponent(float largest) { return max((int)(__float_as_uint(largest) >> 23) - 127 - 15, -126); }
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// The scales of a step's values v [64][P] in sums over rows, four consecutive ranks of four rows of each of P / 16 a lane: each rank's from the largest
// of its values, so that neither other ranks nor other steps lose bits to it. Only exponents count, so two ranks share a word and its instructions
// (upper halves of fp32; with a word each, 16384 x 3072 x 12288 of rank 32 took 139 us). The waves tell each other in top[4][P / 2]: tell_largest() before a barrier,
// scale_values() after it, and after the next one back[P] holds what brings a rank's sums back.
__device__ __forceinline__ us2 halves_of(uint32_t w) { return __builtin_bit_cast(us2, w); }   // (by value: the cast takes a vector's element for its first one)
__device__ __forceinline__ uint32_t most(uint32_t x, uint32_t y) { return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(halves_of(x), halves_of(y))); }
template <int P>
__device__ __forceinline__ void tell_largest(const v4f (&v)[P / 16], uint32_t* top, int tid) {
  auto upper = [](float lo, float hi) { return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302) & 0x7fff7fffu; };
  v2u m;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    m[h] = upper(v[0][2 * h], v[0][2 * h + 1]);
#pragma unroll
    for (int i = 1; i < P / 16; ++i) m[h] = most(m[h], upper(v[i][2 * h], v[i][2 * h + 1]));
    if constexpr (P == 16) m[h] = most(m[h], (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m[h], 0x124, 0xf, 0xf, false));   // row_ror 4
    if constexpr (P <= 32) m[h] = most(m[h], (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m[h], 0x128, 0xf, 0xf, false));   // row_ror 8
    const auto rows = __builtin_amdgcn_permlane16_swap(m[h], m[h], false, false);   // lanes 16 apart
    m[h] = most(rows[0], rows[1]);
    const auto halves = __builtin_amdgcn_permlane32_swap(m[h], m[h], false, false);
    m[h] = most(halves[0], halves[1]);
  }
  if ((tid & 63) < P / 4) *reinterpret_cast<v2u*>(top + (tid >> 6) * (P / 2) + 2 * (tid & 63)) = m;
}
template <int P>
__device__ __forceinline__ void scale_values(v4f (&v)[P / 16], const uint32_t* top, float* back, int tid) {
  v2u m = {0, 0};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const v2u o = *reinterpret_cast<const v2u*>(top + w * (P / 2) + tid % (P / 4) * 2);
#pragma unroll
    for (int h = 0; h < 2; ++h) m[h] = most(m[h], o[h]);
  }
  v4f by, inverse;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // exponents E of both ranks, biased and 16 at least (a NaN's is an infinity's): the scale 2^(142 - E), as bits (269 - E) << 23
    const us2 e = __builtin_elementwise_max(halves_of(m[h]) >> (uint16_t)7, us2{16, 16});
    const uint32_t w = __builtin_bit_cast(uint32_t, us2{269, 269} - e);
    by[2 * h] = __uint_as_float(w << 23);
    by[2 * h + 1] = __uint_as_float((w & 0xffff0000u) << 7);
  }
#pragma unroll
  for (int i = 0; i < P / 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[i][e] *= by[e];
  if (tid < P / 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) inverse[e] = __uint_as_float(0x7f000000u - __float_as_uint(by[e]));
    *reinterpret_cast<v4f*>(back + 4 * tid) = inverse;
  }
}

// Eight consecutive ranks of a row of t (or dt), lane % 32 of which is the operand of a low-rank product: lanes l and l + 32 hold
// the 16 ranks of a step.
struct RankPiece {
  v4f raw[2];
  __device__ __forceinline__ void load(const float* at) {
    raw[0] = reinterpret_cast<const v4f*>(at)[0];
    raw[1] = reinterpret_cast<const v4f*>(at)[1];
  }
  __device__ __forceinline__ float largest() const {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(raw[e >> 2][e & 3]));
    return m;
  }
};
struct RankParts {
  v4i hi, lo;
};
template <int DT>
__device__ __forceinline__ RankParts parts_of(const RankPiece& p) {
  RankParts t;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t h, l;
    two_parts<DT>(p.raw[e >> 1][2 * (e & 1)], p.raw[e >> 1][2 * (e & 1) + 1], h, l);
    t.hi[e] = (int)h;
    t.lo[e] = (int)l;
  }
  return t;
}
// acc[i] += l_i t^T for NI tiles of 32 x 32 whose rows (lane % 32) are the pieces' and for NP pieces; l(i, s): the other operand.
// Where some row's values are far (rare) its pieces and sums are scaled. (Small ones are not, the sums being the layer's own too: fp16 values
// below 2^-4 are held to 2^-25, and that times |l| is what a result loses, of which fp16 itself holds no more than 2^-25.)
template <int DT, int NI, int NP, typename L>
__device__ __forceinline__ void rank_products(v16f* const (&acc)[NI], RankPiece (&piece)[NP], L l) {
  bool far = false;
  float down = 1.0f;
  auto scale = [&](float by) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) (*acc[i])[e] *= by;
  };
  if constexpr (DT == PQ_F16) {
    float m = piece[0].largest();
#pragma unroll
    for (int s = 1; s < NP; ++s) m = fmaxf(m, piece[s].largest());
    far = __ballot(m >= 65536.0f) != 0;
    if (far) {
      down = scale_down(__float_as_uint(fmaxf(m, __shfl_xor(m, 32))));
#pragma unroll
      for (int s = 0; s < NP; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) piece[s].raw[e >> 2][e & 3] *= down;
      scale(down);
    }
  }
#pragma unroll
  for (int s = 0; s < NP; ++s) {
    const RankParts t = parts_of<DT>(piece[s]);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const v4i a = l(i, s);
      *acc[i] = mfma16<DT>(a, t.hi, mfma16<DT>(a, t.lo, *acc[i]));
    }
  }
  if (DT == PQ_F16 && far) scale(scale_back(down));
}

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s_t;

// Matrix operand from a tile held row-major along the other axis: lane l gets, of column c0 + l % 32, the 8 rows
// r0 + 8 (l / 32) .. + 7. Each 16 lanes read a 4 x 16 patch (8 bytes a lane) that the transposing read hands back by
// columns. `at(row, chunk)`: address of the 16 bytes holding columns 8 chunk .. of a row.
//
// Such a tile's rows are a multiple of 256 bytes, and 16 lanes read 32 bytes of each of 4 consecutive rows (32 lanes 64): chunk c
// of a row sits at c ^ spread(row), so that those fall on distinct banks in 128- and in 256-byte windows (bits 1-2 of the
// four values of spread are distinct, and so are bits 2-3).
__device__ __forceinline__ int spread(int row) { return (0xca60 >> ((row & 3) << 2)) & 15; }
template <typename At>
__device__ __forceinline__ v4i read_columns(At at, int r0, int c0, int lane) {
  const int i = lane & 15, row = r0 + 8 * (lane >> 5) + (i >> 2), col = c0 + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
  union { v4s h[2]; v4i v; } u;
  u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(at(row, col >> 3) + (col & 4) * 2));
  u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(at(row + 4, col >> 3) + (col & 4) * 2));
  return u.v;
}

// Workgroup id -> (tile_m, tile_n): ids are dealt round-robin over the 8 XCDs, so each XCD takes a contiguous run of the
// tiles, rastered in groups of `group` m-tiles so that the tiles it works on at a time share rows of both operands in its L2.
__device__ __forceinline__ void tile_of(int bid, int blocks, int tiles_m, int tiles_n, int group, int& tm, int& tn) {
  const int per = blocks >> 3, rem = blocks & 7, xcd = bid & 7;
  const int at = (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + (bid >> 3);
  const int g = at / (group * tiles_n), first = g * group, size = min(tiles_m - first, group), r = at - g * group * tiles_n;
  tm = first + r % size;
  tn = r / size;
}

// Lanes of a wave hand each other values through LDS (which keeps a wave's accesses in order): no instruction, but the compiler
// may take a lane's own view of memory past it neither way.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Workgroup barrier that leaves LDS-DMA in flight (__syncthreads() would wait for all of it): this wave's LDS reads are done,
// and nothing moves across it.
__device__ __forceinline__ void ring_barrier() {
  __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

}  // namespace mx
}  // namespace pq
