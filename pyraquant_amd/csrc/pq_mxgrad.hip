// Gradients of a layer over frozen microscaled 4-bit weights (pq_mx.h) with a low-rank branch:
//   y  = xh wh^T + t B + b,  t = x A
//   dt = dy B^T,  dB = t^T dy,  db = sum_m dy,  dA = xt^T dt,  dx = dy wh + dt A^T
// xt: the values of the 8-bit codes the forward pass kept of x. The rounding of x to 4 bits counts as the identity.
#include "pq_mx.h"

#include <algorithm>

namespace pq {
namespace mx {
namespace {

template <int DT>
__device__ __forceinline__ v16f mfma16(v4i a, v4i b, v16f c) {
  if constexpr (DT == PQ_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s_t;

// Matrix operand from a tile held row-major along the other axis: lane l gets, of column c0 + l % 32, the 8 rows
// r0 + 8 (l / 32) .. + 7. Each 16 lanes read a 4 x 16 patch (8 bytes a lane) that the transposing read hands back by
// columns. `at(row, chunk)`: address of the 16 bytes holding columns 8 chunk .. of a row.
template <typename At>
__device__ __forceinline__ v4i read_columns(At at, int r0, int c0, int lane) {
  const int i = lane & 15, row = r0 + 8 * (lane >> 5) + (i >> 2), col = c0 + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
  union { v4s h[2]; v4i v; } u;
  u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(at(row, col >> 3) + (col & 4) * 2));
  u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(at(row + 4, col >> 3) + (col & 4) * 2));
  return u.v;
}

// ---- dx = dy wh + dt A^T ---------------------------------------------------------------------------------------------
struct DxArgs {
  const uint16_t* dy;
  const uint8_t *w, *ws;
  const uint16_t *dt, *ap;   // [M, R], [K, R]
  uint16_t* dx;
  int64_t lddy, lddx;
  int M, N, K, KT;
};

// A workgroup of four waves: 128 rows m x 128 columns k (one stage of the packed weight), 64 n a step. The 4-bit weights are
// widened to 16 bits on their way into LDS, and read back by columns.
template <int DT, int R>
__global__ __launch_bounds__(256) void mx_dx_kernel(const DxArgs p) {
  __shared__ __attribute__((aligned(16))) uint8_t sa[128 * 128];   // [m][64 n]
  __shared__ __attribute__((aligned(16))) uint8_t sw[64 * 256];    // [n][128 k]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int kt = blockIdx.x, k0 = kt * 128, m0 = blockIdx.y * 128;
  const int wk = (wave & 1) * 64, wm = (wave >> 1) * 64;
  const int l32 = lane & 31, half = lane >> 5;
  auto a_at = [&](int row, int chunk) { return sa + row * 128 + ((chunk ^ (row & 7)) << 4); };
  auto w_at = [&](int row, int chunk) { return sw + row * 256 + ((chunk ^ ((row & 3) << 2)) << 4); };
  v16f acc[2][2] = {};   // [k tile][m tile]
  for (int n0 = 0; n0 < p.N; n0 += 64) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // dy: 8 chunks of 8 n a row, 32 rows a pass
      const int row = i * 32 + (tid >> 3), chunk = tid & 7, n = n0 + chunk * 8;
      v4u v = v4u{0, 0, 0, 0};
      if (m0 + row < p.M && n < p.N) v = *reinterpret_cast<const v4u*>(p.dy + (int64_t)(m0 + row) * p.lddy + n);
      *reinterpret_cast<v4u*>(a_at(row, chunk)) = v;
    }
    {   // weights: a thread widens one block of 32 k of one n
      const int row = tid >> 2, b = tid & 3, n = n0 + row;
      const bool in = n < p.N && k0 + b * 32 < p.K;
      v4u c = v4u{0, 0, 0, 0};
      int byte = 0;
      if (in) {
        c = *reinterpret_cast<const v4u*>(p.w + code_offset(n, kt, b, p.KT));
        byte = p.ws[scale_offset(n, kt, b, p.KT)];
      }
      const float s = scale_value(byte);
      constexpr uint32_t nn = nan2<DT>();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<v4u*>(w_at(row, b * 4 + i)) = byte == kNaN ? v4u{nn, nn, nn, nn} : widen8<DT>(c[i], s);
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      v4i w[2], a[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        w[i] = read_columns(w_at, 16 * s, wk + 32 * i, lane);
        a[i] = *reinterpret_cast<const v4i*>(a_at(wm + 32 * i + l32, 2 * s + half));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma16<DT>(w[i], a[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int m = m0 + wm + 32 * j + l32, kk = k0 + wk + 32 * i;
      if constexpr (R > 0) {
#pragma unroll
        for (int s = 0; s < R / 16; ++s) {
          const v4i b = *reinterpret_cast<const v4i*>(p.ap + (int64_t)min(kk + l32, p.K - 1) * R + 16 * s + 8 * half);
          const v4i t = *reinterpret_cast<const v4i*>(p.dt + (int64_t)min(m, p.M - 1) * R + 16 * s + 8 * half);
          acc[i][j] = mfma16<DT>(b, t, acc[i][j]);
        }
      }
      if (m < p.M && kk < p.K) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<v2u*>(p.dx + (int64_t)m * p.lddx + kk + 8 * q + 4 * half) =
              v2u{pack2<DT>(acc[i][j][4 * q], acc[i][j][4 * q + 1]), pack2<DT>(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3])};
      }
    }
}

// ---- sums over rows: part[s][r][c] = sum over the rows of slice s of v[m, r] z[m, c] -------------------------------------
// z is dy (EIGHT false) or the 8-bit codes of x with their scales; v is t or dt, [M, R]. Column sums of z too (COLS). A
// workgroup of four waves takes 128 columns and a slice of the rows, 64 rows a step; the order of the sums is fixed.
struct SumArgs {
  const void* z;
  const uint8_t* scales;
  const uint16_t* v;
  float *part, *part_cols;
  int64_t ldz;
  int M, C, KT, rows;   // rows a slice, a multiple of 64
};

template <int DT, int R, bool EIGHT, bool COLS>
__global__ __launch_bounds__(256) void mx_rowsum_kernel(const SumArgs p) {
  __shared__ __attribute__((aligned(16))) uint8_t sz[64 * 256];      // [m][128 c]
  __shared__ __attribute__((aligned(16))) uint8_t sv[64 * R * 2];    // [m][R]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c0 = blockIdx.x * 128, s0 = blockIdx.y * p.rows;
  const int end = min(p.M, s0 + p.rows);
  auto z_at = [&](int row, int chunk) { return sz + row * 256 + ((chunk ^ ((row & 3) << 2)) << 4); };
  auto v_at = [&](int row, int chunk) { return sv + row * R * 2 + (chunk << 4); };
  const uint32_t one2 = DT == PQ_BF16 ? 0x3f803f80u : 0x3c003c00u;
  const v4i ones = {(int)one2, (int)one2, (int)one2, (int)one2};
  v16f acc[R / 32] = {}, cols = {};
  for (int m0 = s0; m0 < end; m0 += 64) {
    __syncthreads();
    if constexpr (EIGHT) {
      const int row = tid >> 2, b = tid & 3, m = m0 + row, c = c0 + b * 32;
      const bool in = m < end && c < p.C;
      v4u q[2] = {};
      int byte = 0;
      if (in) {
        const v4u* const src = reinterpret_cast<const v4u*>(static_cast<const int8_t*>(p.z) + (int64_t)m * p.ldz + c);
        q[0] = src[0];
        q[1] = src[1];
        byte = p.scales[scale_offset(m, blockIdx.x, b, p.KT)];
      }
      const float s = in ? restore_scale(byte) : 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v2u lo = restore4<DT>(q[i >> 1][2 * (i & 1)], s), hi = restore4<DT>(q[i >> 1][2 * (i & 1) + 1], s);
        *reinterpret_cast<v4u*>(z_at(row, b * 4 + i)) = v4u{lo[0], lo[1], hi[0], hi[1]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = i * 16 + (tid >> 4), chunk = tid & 15, m = m0 + row, c = c0 + chunk * 8;
        v4u x = v4u{0, 0, 0, 0};
        if (m < end && c < p.C) x = *reinterpret_cast<const v4u*>(static_cast<const uint16_t*>(p.z) + (int64_t)m * p.ldz + c);
        *reinterpret_cast<v4u*>(z_at(row, chunk)) = x;
      }
    }
    for (int i = tid; i < 64 * R / 8; i += 256) {
      const int row = i / (R / 8), chunk = i % (R / 8);
      v4u x = v4u{0, 0, 0, 0};
      if (m0 + row < end) x = *reinterpret_cast<const v4u*>(p.v + (int64_t)(m0 + row) * R + chunk * 8);
      *reinterpret_cast<v4u*>(v_at(row, chunk)) = x;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const v4i z = read_columns(z_at, 16 * s, wave * 32, lane);
#pragma unroll
      for (int j = 0; j < R / 32; ++j) acc[j] = mfma16<DT>(z, read_columns(v_at, 16 * s, 32 * j, lane), acc[j]);
      if constexpr (COLS) cols = mfma16<DT>(z, ones, cols);
    }
  }
  // lane: r = 32 j + lane % 32, columns c0 + 32 wave + 8 q + 4 (lane / 32) + e
  const int c = c0 + wave * 32 + 4 * (lane >> 5);
  if (c0 + wave * 32 >= p.C) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (c + 8 * q >= p.C) break;
#pragma unroll
    for (int j = 0; j < R / 32; ++j)
      *reinterpret_cast<v4f*>(p.part + ((int64_t)blockIdx.y * R + 32 * j + (lane & 31)) * p.C + c + 8 * q) =
          v4f{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
    if (COLS && (lane & 31) == 0)
      *reinterpret_cast<v4f*>(p.part_cols + (int64_t)blockIdx.y * p.C + c + 8 * q) =
          v4f{cols[4 * q], cols[4 * q + 1], cols[4 * q + 2], cols[4 * q + 3]};
  }
}

// The slices' sums added in order: out[r, c] (TRANS: out[c, r]) rounded to 16 bits, and the column sums in 32.
template <int DT, bool TRANS>
__global__ __launch_bounds__(256) void mx_join_kernel(const float* __restrict__ part, const float* __restrict__ part_cols,
                                                      int slices, int P, int R, int C, uint16_t* __restrict__ out,
                                                      float* __restrict__ cols) {
  const int c = blockIdx.x * 64 + (threadIdx.x & 63);
  if (c >= C) return;
  for (int r = threadIdx.x >> 6; out && r < R; r += 4) {
    float s = 0.0f;
    for (int i = 0; i < slices; ++i) s += part[((int64_t)i * P + r) * C + c];
    out[TRANS ? (int64_t)c * R + r : (int64_t)r * C + c] = (uint16_t)f32_to_16_bits<DT>(s);
  }
  if (cols && threadIdx.x < 64) {
    float s = 0.0f;
    for (int i = 0; i < slices; ++i) s += part_cols[(int64_t)i * C + c];
    cols[c] = s;
  }
}

// Row slices of mx_rowsum_kernel: enough workgroups to fill the chip, none of fewer than 64 rows.
int row_slices(int64_t M, int64_t C) {
  const int64_t panels = (C + 127) / 128, steps = (M + 63) / 64;
  const int64_t want = std::max<int64_t>(1, (1024 + panels - 1) / panels);
  return (int)std::min<int64_t>({want, steps, 256});
}

}  // namespace
}  // namespace mx
}  // namespace pq

using namespace pq;

extern "C" int pq_mx_grad_input(const void* dy, int32_t dtype, int64_t lddy, const uint8_t* w, const uint8_t* w_scales,
                                const void* dt, const void* ap, int64_t R, void* dx, int64_t lddx, int64_t M, int64_t N,
                                int64_t K, hipStream_t stream) {
  if (M < 0 || N < 16 || N % 16 || K < 32 || K % 32 || lddy < N || lddx < K || M > (1 << 30) ||
      N > (1 << 30) || K > (1 << 22))
    return set_error(PQ_ESHAPE, "pq_mx_grad_input: M=%lld N=%lld K=%lld (N %% 16 == 0, K %% 32 == 0)", (long long)M,
                     (long long)N, (long long)K);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_mx_grad_input: dtype %d", dtype);
  if (dt && R != 32 && R != 64) return set_error(PQ_ESHAPE, "pq_mx_grad_input: rank %lld (32 or 64)", (long long)R);
  if (M == 0) return PQ_OK;
  if (!dy || !w || !w_scales || !dx || (dt && !ap)) return set_error(PQ_EINVAL, "pq_mx_grad_input: null pointer");
  if ((uintptr_t)dy % 16 || lddy % 8 || (uintptr_t)w % 16 || (uintptr_t)w_scales % 16 || (uintptr_t)dx % 16 || lddx % 8 ||
      (uintptr_t)dt % 16 || (uintptr_t)ap % 16)
    return set_error(PQ_EALIGN, "pq_mx_grad_input: operands 16-byte aligned, lddy and lddx multiples of 8");
  mx::DxArgs p{static_cast<const uint16_t*>(dy), w, w_scales, static_cast<const uint16_t*>(dt), static_cast<const uint16_t*>(ap),
               static_cast<uint16_t*>(dx), lddy, lddx, (int)M, (int)N, (int)K, mx::stages(K)};
  if ((M + 127) / 128 > 65535) return set_error(PQ_ESHAPE, "pq_mx_grad_input: M=%lld too large", (long long)M);
  const dim3 grid((unsigned)p.KT, (unsigned)((M + 127) / 128)), block(256);
  const int r = dt ? (int)R : 0;
#define PQ_MXD(D, RR) hipLaunchKernelGGL((mx::mx_dx_kernel<D, RR>), grid, block, 0, stream, p)
  if (dtype == PQ_BF16) {
    if (r == 0) PQ_MXD(PQ_BF16, 0); else if (r == 32) PQ_MXD(PQ_BF16, 32); else PQ_MXD(PQ_BF16, 64);
  } else {
    if (r == 0) PQ_MXD(PQ_F16, 0); else if (r == 32) PQ_MXD(PQ_F16, 32); else PQ_MXD(PQ_F16, 64);
  }
#undef PQ_MXD
  return check_launch("mx_grad_input");
}

extern "C" int64_t pq_mx_grad_factors_workspace_size(int64_t M, int64_t K, int64_t N, int64_t P) {
  if (M < 1 || K < 32 || N < 16 || (P != 32 && P != 64)) return 0;
  const int64_t b = (int64_t)mx::row_slices(M, N) * (P + 1) * N, a = (int64_t)mx::row_slices(M, K) * P * K;
  return 4 * std::max(a, b);
}

extern "C" int pq_mx_grad_factors(const void* dy, int32_t dtype, int64_t lddy, const void* t, const void* dt, const int8_t* q8,
                                  const uint8_t* x_scales, int64_t M, int64_t K, int64_t N, int64_t R, int64_t P, void* dA,
                                  void* dB, float* dbias, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (M < 1 || N < 16 || N % 16 || K < 32 || K % 32 || lddy < N || R < 1 || R > P || (P != 32 && P != 64) ||
      M > (1 << 30) || N > (1 << 30) || K > (1 << 22))
    return set_error(PQ_ESHAPE, "pq_mx_grad_factors: M=%lld N=%lld K=%lld R=%lld P=%lld", (long long)M, (long long)N,
                     (long long)K, (long long)R, (long long)P);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_mx_grad_factors: dtype %d", dtype);
  if (((dB || dbias) && (!dy || !t)) || (dA && (!dt || !q8 || !x_scales)) || !workspace)
    return set_error(PQ_EINVAL, "pq_mx_grad_factors: null pointer");
  if ((uintptr_t)dy % 16 || lddy % 8 || (uintptr_t)t % 16 || (uintptr_t)dt % 16 || (uintptr_t)q8 % 16 || (uintptr_t)workspace % 16)
    return set_error(PQ_EALIGN, "pq_mx_grad_factors: operands 16-byte aligned, lddy a multiple of 8");
  if (workspace_bytes < pq_mx_grad_factors_workspace_size(M, K, N, P))
    return set_error(PQ_ESHAPE, "pq_mx_grad_factors: workspace of %lld bytes", (long long)workspace_bytes);
  float* const part = static_cast<float*>(workspace);
  const int sb = mx::row_slices(M, N), sk = mx::row_slices(M, K);
  auto rows = [&](int slices) { return (int)(((M + 63) / 64 + slices - 1) / slices * 64); };
  mx::SumArgs b{dy, nullptr, static_cast<const uint16_t*>(t), part, part + (int64_t)sb * P * N, lddy, (int)M, (int)N, 0, rows(sb)};
  mx::SumArgs a{q8, x_scales, static_cast<const uint16_t*>(dt), part, nullptr, K, (int)M, (int)K, mx::stages(K), rows(sk)};
  const dim3 gb((unsigned)((N + 127) / 128), (unsigned)sb), ga((unsigned)((K + 127) / 128), (unsigned)sk), block(256);
  const dim3 jb((unsigned)((N + 63) / 64)), ja((unsigned)((K + 63) / 64));
#define PQ_MXS(D, PP)                                                                                                     \
  do {                                                                                                                   \
    if (dbias) hipLaunchKernelGGL((mx::mx_rowsum_kernel<D, PP, false, true>), gb, block, 0, stream, b);                  \
    else if (dB) hipLaunchKernelGGL((mx::mx_rowsum_kernel<D, PP, false, false>), gb, block, 0, stream, b);               \
    if (dB || dbias)                                                                                                     \
      hipLaunchKernelGGL((mx::mx_join_kernel<D, false>), jb, block, 0, stream, part, b.part_cols, sb, (int)P, (int)R,    \
                         (int)N, static_cast<uint16_t*>(dB), dbias);                                                     \
    if (dA) {                                                                                                            \
      hipLaunchKernelGGL((mx::mx_rowsum_kernel<D, PP, true, false>), ga, block, 0, stream, a);                           \
      hipLaunchKernelGGL((mx::mx_join_kernel<D, true>), ja, block, 0, stream, part, nullptr, sk, (int)P, (int)R, (int)K, \
                         static_cast<uint16_t*>(dA), nullptr);                                                           \
    }                                                                                                                    \
  } while (0)
  if (dtype == PQ_BF16) {
    if (P == 32) PQ_MXS(PQ_BF16, 32); else PQ_MXS(PQ_BF16, 64);
  } else {
    if (P == 32) PQ_MXS(PQ_F16, 32); else PQ_MXS(PQ_F16, 64);
  }
#undef PQ_MXS
  return check_launch("mx_grad_factors");
}
