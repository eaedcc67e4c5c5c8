// Microscaled 4-bit quantization (pq_mx.h): rows to packed codes and scales, with the 8-bit codes of a training layer's
// checkpoint in the same pass, and back to values.
//
// One lane takes one block of 32 values: its largest magnitude, its scale byte and its 16 bytes of codes need no other lane.
// A wave takes 16 rows x 4 blocks, which is one 1 KB block of the packed layout, so its codes go out as one contiguous
// 1 KB store and a row's 4 blocks are whole 128-byte lines of the input. Bound by memory: 2 bytes read per value, 1/2 +
// 1/32 written (and 1 for the 8-bit codes).
#include "pq_mx.h"

namespace pq {
namespace mx {
namespace {

// DT: input type. VEC: 16-byte loads. CKPT: also the 8-bit codes, q8 [M, K] row-major.
template <int DT, bool VEC, bool CKPT>
__global__ __launch_bounds__(256) void mx_quant_kernel(const void* __restrict__ x, int64_t ldx, int64_t M, int K, int KT,
                                                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                       int8_t* __restrict__ q8, int64_t units) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);   // (row block, stage)
  if (unit >= units) return;
  const int64_t rb = unit / KT;
  const int kt = (int)(unit - rb * KT);
  const int64_t row = rb * 16 + (lane & 15);
  const int b = lane >> 4, k = kt * 128 + b * kBlock;
  constexpr int ES = DT == PQ_F32 ? 4 : 2;
  Block<DT> blk;
  const bool inside = row < M && k < K;
  if (inside) blk.template load<VEC>(static_cast<const uint8_t*>(x) + (row * ldx + k) * ES);
  else blk.zero();
  const int byte = blk.scale_byte();
  scales[scale_offset(row, kt, b, KT)] = (uint8_t)byte;
  *reinterpret_cast<v4i*>(codes + code_offset(row, kt, b, KT)) = blk.codes(byte);
  if constexpr (CKPT) {
    if (inside) {
      v4i q[2];
      blk.codes8(byte, q);
      v4i* const o = reinterpret_cast<v4i*>(q8 + row * K + k);
      o[0] = q[0];
      o[1] = q[1];
    }
  }
}

// Values of the 4-bit codes (EIGHT: of the 8-bit ones), one lane a block. ODT: output type.
template <int ODT, bool EIGHT>
__global__ __launch_bounds__(256) void mx_values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                        int64_t M, int K, int KT, void* __restrict__ out, int64_t ldo,
                                                        int64_t units) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int64_t rb = unit / KT;
  const int kt = (int)(unit - rb * KT);
  const int64_t row = rb * 16 + (lane & 15);
  const int b = lane >> 4, k = kt * 128 + b * kBlock;
  if (row >= M || k >= K) return;
  const int byte = scales[scale_offset(row, kt, b, KT)];
  if constexpr (EIGHT) {
    const v4u* const q = reinterpret_cast<const v4u*>(codes + row * K + k);
    const float s = restore_scale(byte);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = q[i >> 2][i & 3];
      if constexpr (ODT == PQ_F32) {
        v4f f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = (float)((int)(w << (24 - 8 * e)) >> 24) * s;
        *reinterpret_cast<v4f*>(static_cast<float*>(out) + row * ldo + k + 4 * i) = f;
      } else {
        *reinterpret_cast<v2u*>(static_cast<uint16_t*>(out) + row * ldo + k + 4 * i) = restore4<ODT>(w, s);
      }
    }
  } else {
    const v4u c = *reinterpret_cast<const v4u*>(codes + code_offset(row, kt, b, KT));
    const float s = scale_value(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (ODT == PQ_F32) {
        float* const o = static_cast<float*>(out) + row * ldo + k + 8 * i;
        const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], s, 0), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], s, 1);
        const v2f e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], s, 2), f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], s, 3);
        const float nan = __uint_as_float(0x7fc00000u);
        const bool bad = byte == kNaN;
        reinterpret_cast<v4f*>(o)[0] = bad ? v4f{nan, nan, nan, nan} : v4f{a[0], a[1], d[0], d[1]};
        reinterpret_cast<v4f*>(o)[1] = bad ? v4f{nan, nan, nan, nan} : v4f{e[0], e[1], f[0], f[1]};
      } else {
        constexpr uint32_t n = nan2<ODT>();
        *reinterpret_cast<v4u*>(static_cast<uint16_t*>(out) + row * ldo + k + 8 * i) =
            byte == kNaN ? v4u{n, n, n, n} : widen8<ODT>(c[i], s);
      }
    }
  }
}

// lr_A [K, R] -> At [P, K] and Ap [K, P]; lr_B [R, N] -> Bt [N, P] and Bp [P, N]: the four orders in which the layer's
// kernels read the factors, zero-padded from rank R to P. A workgroup takes 64 rows k (or columns n) of one factor.
__global__ __launch_bounds__(256) void mx_factors_kernel(const uint16_t* __restrict__ A, int64_t lda,
                                                         const uint16_t* __restrict__ B, int64_t ldb, int K, int N, int R,
                                                         int P, uint16_t* __restrict__ At, uint16_t* __restrict__ Ap,
                                                         uint16_t* __restrict__ Bt, uint16_t* __restrict__ Bp, int blocks_a) {
  __shared__ uint16_t tile[64][66];   // [k or n][r]; a pitch of 33 words: both directions spread over the banks
  const bool is_a = (int)blockIdx.x < blocks_a;
  const int c0 = ((int)blockIdx.x - (is_a ? 0 : blocks_a)) * 64, C = is_a ? K : N;
  for (int i = threadIdx.x; i < 64 * P; i += 256) {
    int c, r;
    if (is_a) { c = i / P; r = i - c * P; }   // read along r
    else { r = i >> 6; c = i & 63; }          // read along n
    const bool in = c0 + c < C && r < R;
    tile[c][r] = !in ? 0 : is_a ? A[(int64_t)(c0 + c) * lda + r] : B[(int64_t)r * ldb + c0 + c];
  }
  __syncthreads();
  uint16_t* const by_c = is_a ? Ap : Bt;   // [C, P]
  uint16_t* const by_r = is_a ? At : Bp;   // [P, C]
  for (int i = threadIdx.x; i < 64 * P; i += 256) {
    const int c = i / P, r = i - c * P;
    if (by_c && c0 + c < C) by_c[(int64_t)(c0 + c) * P + r] = tile[c][r];
    const int r2 = i >> 6, c2 = i & 63;
    if (by_r && c0 + c2 < C) by_r[(int64_t)r2 * C + c0 + c2] = tile[c2][r2];
  }
}

template <int DT, bool VEC>
int launch_quant(const void* x, int64_t M, int64_t K, int64_t ldx, uint8_t* codes, uint8_t* scales, int8_t* q8,
                 hipStream_t stream) {
  const int KT = stages(K);
  const int64_t units = (M + 15) / 16 * KT;
  if (const int st = check_grid((units + 3) / 4, 256, "mx_quant")) return st;
  const dim3 grid((unsigned)((units + 3) / 4)), block(256);
  if (q8)
    hipLaunchKernelGGL((mx_quant_kernel<DT, VEC, true>), grid, block, 0, stream, x, ldx, M, (int)K, KT, codes, scales, q8, units);
  else
    hipLaunchKernelGGL((mx_quant_kernel<DT, VEC, false>), grid, block, 0, stream, x, ldx, M, (int)K, KT, codes, scales, q8, units);
  return check_launch("mx_quant");
}

}  // namespace
}  // namespace mx
}  // namespace pq

using namespace pq;
using namespace pq::mx;

extern "C" int pq_mx_quant(const void* x, int32_t dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* codes, uint8_t* scales,
                           int8_t* q8, hipStream_t stream) {
  if (M < 0 || K < 32 || K % 32 || ldx < K || K > (1 << 30))
    return set_error(PQ_ESHAPE, "pq_mx_quant: M=%lld K=%lld ldx=%lld (K %% 32 == 0, ldx >= K)", (long long)M, (long long)K,
                     (long long)ldx);
  if (dtype != PQ_BF16 && dtype != PQ_F16 && dtype != PQ_F32) return set_error(PQ_EDTYPE, "pq_mx_quant: dtype %d", dtype);
  if (M == 0) return PQ_OK;
  if (!x || !codes || !scales) return set_error(PQ_EINVAL, "pq_mx_quant: null pointer");
  const int es = dtype == PQ_F32 ? 4 : 2;
  if ((uintptr_t)codes % 16 || (uintptr_t)q8 % 16 || (uintptr_t)x % es)
    return set_error(PQ_EALIGN, "pq_mx_quant: codes and q8 16-byte aligned, x to its elements");
  const bool vec = (uintptr_t)x % 16 == 0 && ldx * es % 16 == 0;
#define PQ_MXQ(D) (vec ? launch_quant<D, true>(x, M, K, ldx, codes, scales, q8, stream)                                  \
                       : launch_quant<D, false>(x, M, K, ldx, codes, scales, q8, stream))
  return dtype == PQ_BF16 ? PQ_MXQ(PQ_BF16) : dtype == PQ_F16 ? PQ_MXQ(PQ_F16) : PQ_MXQ(PQ_F32);
#undef PQ_MXQ
}

extern "C" int pq_mx_values(const void* codes, const uint8_t* scales, int32_t bits, int64_t M, int64_t K, void* out,
                            int32_t dtype, int64_t ldo, hipStream_t stream) {
  if (M < 0 || K < 32 || K % 32 || ldo < K || K > (1 << 30))
    return set_error(PQ_ESHAPE, "pq_mx_values: M=%lld K=%lld ldo=%lld (K %% 32 == 0, ldo >= K)", (long long)M, (long long)K,
                     (long long)ldo);
  if (bits != 4 && bits != 8) return set_error(PQ_EINVAL, "pq_mx_values: codes of %d bits (4 or 8)", bits);
  if (dtype != PQ_BF16 && dtype != PQ_F16 && dtype != PQ_F32) return set_error(PQ_EDTYPE, "pq_mx_values: dtype %d", dtype);
  if (M == 0) return PQ_OK;
  if (!codes || !scales || !out) return set_error(PQ_EINVAL, "pq_mx_values: null pointer");
  const int es = dtype == PQ_F32 ? 4 : 2;
  if ((uintptr_t)codes % 16 || (uintptr_t)out % 16 || ldo * es % 16)
    return set_error(PQ_EALIGN, "pq_mx_values: codes, out and its rows 16-byte aligned");
  const int KT = stages(K);
  const int64_t units = (M + 15) / 16 * KT;
  if (const int st = check_grid((units + 3) / 4, 256, "mx_values")) return st;
  const dim3 grid((unsigned)((units + 3) / 4)), block(256);
#define PQ_MXV(D, E)                                                                                                      \
  hipLaunchKernelGGL((mx_values_kernel<D, E>), grid, block, 0, stream, static_cast<const uint8_t*>(codes), scales, M, (int)K, \
                     KT, out, ldo, units)
  if (bits == 4) {
    if (dtype == PQ_BF16) PQ_MXV(PQ_BF16, false); else if (dtype == PQ_F16) PQ_MXV(PQ_F16, false); else PQ_MXV(PQ_F32, false);
  } else {
    if (dtype == PQ_BF16) PQ_MXV(PQ_BF16, true); else if (dtype == PQ_F16) PQ_MXV(PQ_F16, true); else PQ_MXV(PQ_F32, true);
  }
#undef PQ_MXV
  return check_launch("mx_values");
}

extern "C" int pq_mx_factors(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t K, int64_t N, int64_t R,
                             int64_t P, void* At, void* Ap, void* Bt, void* Bp, hipStream_t stream) {
  if (K < 1 || N < 1 || R < 1 || R > P || (P != 32 && P != 64) || lda < R || ldb < N || K > (1 << 30) || N > (1 << 30))
    return set_error(PQ_ESHAPE, "pq_mx_factors: K=%lld N=%lld R=%lld P=%lld (R <= P, P 32 or 64)", (long long)K, (long long)N,
                     (long long)R, (long long)P);
  if (!A || !B) return set_error(PQ_EINVAL, "pq_mx_factors: null pointer");
  const int blocks_a = (int)((K + 63) / 64), blocks_b = (int)((N + 63) / 64);
  hipLaunchKernelGGL(mx_factors_kernel, dim3(blocks_a + blocks_b), dim3(256), 0, stream, static_cast<const uint16_t*>(A), lda,
                     static_cast<const uint16_t*>(B), ldb, (int)K, (int)N, (int)R, (int)P, static_cast<uint16_t*>(At),
                     static_cast<uint16_t*>(Ap), static_cast<uint16_t*>(Bt), static_cast<uint16_t*>(Bp), blocks_a);
  return check_launch("mx_factors");
}
