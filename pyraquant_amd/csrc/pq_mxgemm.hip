// Product of two microscaled 4-bit matrices (pq_mx.h), with the low-rank term and the bias in its epilogue:
//   y[m, n] = sum_k xh[m, k] wh[n, k]  (+ sum_r t[m, r] l2t[n, r])  (+ bias[n]),  rounded once to 16 bits.
//
// The matrix instructions take the 4-bit codes and the scale bytes as they are stored (v_mfma_scale_f32_32x32x64_f8f6f4:
// 64 values of k a step, one scale byte per lane and operand) and sum in fp32. The row operand is a weight row n and the
// column operand an activation row m, so each lane holds 4 consecutive n of one output row.
#include "pq_mx.h"

namespace pq {
namespace mx {
namespace {

struct GemmArgs {
  const uint8_t *a, *as, *w, *ws;   // codes and scales of x and of the weight
  const float* bias;
  const uint16_t *t, *l2t;
  uint16_t* c;
  int64_t ldt, ldc;
  int M, N, KT;
};

// One step over 64 values: both operands 4-bit (format code 4), scale byte S of each scale word.
template <int S>
__device__ __forceinline__ v16f mfma4(v4i a, int sa, v4i b, int sb, v16f c) {
  const v8i a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, S, sa, S, sb);
}

template <int DT>
__device__ __forceinline__ v16f mfma16(v4i a, v4i b, v16f c) {
  if constexpr (DT == PQ_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// Four waves, each a 64 x 64 part of a 128 x 128 block, fragments straight from memory into registers.
template <int DT, int R>
__global__ __launch_bounds__(256) void mx_gemm_kernel(const GemmArgs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n0 = blockIdx.x * 128 + (wave & 1) * 64, m0 = blockIdx.y * 128 + (wave >> 1) * 64;
  if (n0 >= p.N || m0 >= p.M) return;
  const int l32 = lane & 31, half = lane >> 5, r16 = lane & 15, sw = k64_swz(r16);
  const int last_n = (p.N - 1) >> 4, last_m = (p.M - 1) >> 4;
  int64_t wb[2], ab[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {   // (row blocks past the end repeat the last one: their outputs are not stored)
    wb[i] = (int64_t)min((n0 + 32 * i + l32) >> 4, last_n) * p.KT;
    ab[i] = (int64_t)min((m0 + 32 * i + l32) >> 4, last_m) * p.KT;
  }
  v16f acc[2][2] = {};
  for (int kt = 0; kt < p.KT; ++kt) {
    int ws[2], as[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      ws[i] = *reinterpret_cast<const uint16_t*>(p.ws + (wb[i] + kt) * 64 + r16 * 4 + 2 * half);
      as[i] = *reinterpret_cast<const uint16_t*>(p.as + (ab[i] + kt) * 64 + r16 * 4 + 2 * half);
    }
    v4i w[2][2], a[2][2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int off = r16 * 64 + (((2 * s + half) ^ sw) << 4);
        w[s][i] = *reinterpret_cast<const v4i*>(p.w + (wb[i] + kt) * 1024 + off);
        a[s][i] = *reinterpret_cast<const v4i*>(p.a + (ab[i] + kt) * 1024 + off);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        acc[i][j] = mfma4<0>(w[0][i], ws[i], a[0][j], as[j], acc[i][j]);
        acc[i][j] = mfma4<1>(w[1][i], ws[i], a[1][j], as[j], acc[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int m = m0 + 32 * j + l32, n = n0 + 32 * i + l32;
      if constexpr (R > 0) {
#pragma unroll
        for (int s = 0; s < R / 16; ++s) {
          const v4i b = *reinterpret_cast<const v4i*>(p.l2t + (int64_t)min(n, p.N - 1) * R + 16 * s + 8 * half);
          const v4i t = *reinterpret_cast<const v4i*>(p.t + (int64_t)min(m, p.M - 1) * p.ldt + 16 * s + 8 * half);
          acc[i][j] = mfma16<DT>(b, t, acc[i][j]);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int nq = n0 + 32 * i + 8 * q + 4 * half;
        if (m < p.M && nq < p.N) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = acc[i][j][4 * q + e] + (p.bias ? p.bias[nq + e] : 0.0f);
          *reinterpret_cast<v2u*>(p.c + (int64_t)m * p.ldc + nq) = v2u{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
        }
      }
    }
}

}  // namespace
}  // namespace mx
}  // namespace pq

using namespace pq;

extern "C" int pq_mx_gemm(const uint8_t* a, const uint8_t* a_scales, const uint8_t* w, const uint8_t* w_scales,
                          const float* bias, const void* t, int64_t ldt, const void* l2t, int64_t R, void* c, int64_t ldc,
                          int32_t dtype, int64_t M, int64_t N, int64_t K, hipStream_t stream) {
  if (M < 0 || N < 16 || N % 16 || K < 32 || K % 32 || ldc < N || ldc >= (1LL << 31) || M > (1 << 30) ||
      N > (1 << 30) || K > (1 << 22))
    return set_error(PQ_ESHAPE, "pq_mx_gemm: M=%lld N=%lld K=%lld ldc=%lld (N %% 16 == 0, K %% 32 == 0)", (long long)M,
                     (long long)N, (long long)K, (long long)ldc);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_mx_gemm: dtype %d", dtype);
  if (t ? (R != 32 && R != 64) || ldt < R || ldt > (1 << 22) : false)
    return set_error(PQ_ESHAPE, "pq_mx_gemm: rank %lld (32 or 64), ldt=%lld", (long long)R, (long long)ldt);
  if (M == 0) return PQ_OK;
  if (!a || !a_scales || !w || !w_scales || !c || (t && !l2t)) return set_error(PQ_EINVAL, "pq_mx_gemm: null pointer");
  if ((uintptr_t)a % 16 || (uintptr_t)w % 16 || (uintptr_t)a_scales % 16 || (uintptr_t)w_scales % 16 || (uintptr_t)c % 16 ||
      ldc % 8 || (uintptr_t)bias % 16 || (t && ((uintptr_t)t % 16 || (uintptr_t)l2t % 16 || ldt % 8)))
    return set_error(PQ_EALIGN, "pq_mx_gemm: operands 16-byte aligned, ldc and ldt multiples of 8");
  mx::GemmArgs p{a, a_scales, w, w_scales, bias, static_cast<const uint16_t*>(t), static_cast<const uint16_t*>(l2t),
                 static_cast<uint16_t*>(c), ldt, ldc, (int)M, (int)N, mx::stages(K)};
  const int64_t bn = (N + 127) / 128, bm = (M + 127) / 128;
  if (bm > 65535) return set_error(PQ_ESHAPE, "pq_mx_gemm: M=%lld too large", (long long)M);
  const dim3 grid((unsigned)bn, (unsigned)bm), block(256);
  const int r = t ? (int)R : 0;
#define PQ_MXG(D, RR) hipLaunchKernelGGL((mx::mx_gemm_kernel<D, RR>), grid, block, 0, stream, p)
  if (dtype == PQ_BF16) {
    if (r == 0) PQ_MXG(PQ_BF16, 0); else if (r == 32) PQ_MXG(PQ_BF16, 32); else PQ_MXG(PQ_BF16, 64);
  } else {
    if (r == 0) PQ_MXG(PQ_F16, 0); else if (r == 32) PQ_MXG(PQ_F16, 32); else PQ_MXG(PQ_F16, 64);
  }
#undef PQ_MXG
  return check_launch("mx_gemm");
}
