// Microscaled 4-bit quantization (pq_mx.h): rows to packed codes and scales, with the 8-bit codes of a training layer's
// checkpoint in the same pass, and back to values.
//
// One lane takes one block of 32 values: its largest magnitude, its scale byte and its 16 bytes of codes need no other lane.
// A wave takes 16 rows x 4 blocks, which is one 1 KB block of the packed layout, so its codes go out as one contiguous
// 1 KB store and a row's 4 blocks are whole 128-byte lines of the input. Bound by memory: 2 bytes read per value, 1/2 +
// 1/32 written (and 1 for the 8-bit codes): 65536 x 3072 bf16 in 88 us, 5.8 TB/s, and in 131 us, 5.4 TB/s, with the 8-bit codes
// (a large copy: 5.1 TB/s); 640 x 640 in 3 us, a launch.
#include "pq_mx.h"

#include <algorithm>
#include <type_traits>

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

// t = x l1t^T ([M, R], fp32) and, where QUANT, the codes of x, in one pass over x. A workgroup takes 16 RG rows and its NW
// waves every NW-th stage of 128 values, 16 rows at a time as above: what a lane holds of x for its block is also its operand
// of the 16 x 16 x 32 products (8 consecutive values of a row; the order of k within the sum is free as long as l1t's operand
// has the same), so x is read once and needs no other lane or LDS. l1t comes from the cache in fragment order (1 KB a load, zeros
// past K), once per RG row groups. The waves' sums are added in LDS in a fixed order. dt, of dy, is made here too.
// Bound by reading x and by l1t from the cache: 65536 x 3072 with codes 103 us (the quantizer alone: 88), dy of 16384 x 12288
// to dt in 104-116 us, 3.5-3.9 TB/s.
template <int DT, int R, int RG, int NW, bool QUANT, bool CKPT>
__global__ __launch_bounds__(64 * NW) void mx_lowrank_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t M, int K, int KT,
                                                             const uint16_t* __restrict__ l1f, uint8_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales, int8_t* __restrict__ q8,
                                                             float* __restrict__ t) {
  constexpr int C = R / 16;                                  // column tiles of t
  __shared__ float part[NW][RG * C][64 * 4 + 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, b = lane >> 4;
  const int64_t m0 = (int64_t)blockIdx.x * (16 * RG);
  v4f acc[RG][C] = {};
  for (int kt = blockIdx.y * NW + wave; kt < KT; kt += NW * (int)gridDim.y) {
    const int k = kt * 128 + b * kBlock;
    Block<DT> blk[RG];
#pragma unroll
    for (int g = 0; g < RG; ++g) {
      const int64_t row = m0 + 16 * g + l16;
      const uint16_t* const src = x + row * ldx + k;
      if (QUANT) {   // whole blocks
        if (row < M && k < K) blk[g].template load<true>(src);
        else blk[g].zero();
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v4u v = v4u{0, 0, 0, 0};
          if (row < M && k + 8 * i < K) v = *reinterpret_cast<const v4u*>(src + 8 * i);
#pragma unroll
          for (int e = 0; e < 4; ++e) blk[g].w[4 * i + e] = v[e];
        }
      }
    }
    v4i l[4][C];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < C; ++c)
        l[i][c] = *reinterpret_cast<const v4i*>(l1f + (((int64_t)kt * 4 + i) * C + c) * 512 + lane * 8);
#pragma unroll
    for (int g = 0; g < RG; ++g) {
      const int64_t row = m0 + 16 * g + l16;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v4i xv = {(int)blk[g].w[4 * i], (int)blk[g].w[4 * i + 1], (int)blk[g].w[4 * i + 2], (int)blk[g].w[4 * i + 3]};
#pragma unroll
        for (int c = 0; c < C; ++c) acc[g][c] = mfma16_16<DT>(l[i][c], xv, acc[g][c]);
      }
      if (QUANT && row < ((M + 15) & ~15LL)) {
        const int byte = blk[g].scale_byte();
        scales[scale_offset(row, kt, b, KT)] = (uint8_t)byte;
        *reinterpret_cast<v4i*>(codes + code_offset(row, kt, b, KT)) = blk[g].codes(byte);
        if (CKPT && row < M && k < K) {
          v4i q[2];
          blk[g].codes8(byte, q);
          v4i* const o = reinterpret_cast<v4i*>(q8 + row * K + k);
          o[0] = q[0];
          o[1] = q[1];
        }
      }
    }
  }
#pragma unroll
  for (int g = 0; g < RG; ++g)
#pragma unroll
    for (int c = 0; c < C; ++c) *reinterpret_cast<v4f*>(&part[wave][g * C + c][lane * 4]) = acc[g][c];
  __syncthreads();
  // lane l of tile (g, c): row 16 g + l % 16, columns 16 c + 4 (l / 16) ..
  for (int u = threadIdx.x; u < RG * C * 64; u += 64 * NW) {
    const int tile = u >> 6, l = u & 63;
    v4f sum = {};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const v4f v = *reinterpret_cast<const v4f*>(&part[w][tile][l * 4]);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += v[e];
    }
    const int64_t row = m0 + 16 * (tile / C) + (l & 15);
    if (row >= M) continue;
    *reinterpret_cast<v4f*>(t + (blockIdx.y * M + row) * R + 16 * (tile % C) + 4 * (l >> 4)) = sum;   // (a slice of k each)
  }
}

// t from the sums of workgroups that share rows (`partial` [slices][M R]), in order; a thread takes four.
__global__ __launch_bounds__(256) void mx_lowrank_join_kernel(const float* __restrict__ partial, int slices, int64_t n,
                                                              float* __restrict__ t) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  v4f sum = {};
  for (int z = 0; z < slices; ++z) {
    const v4f v = *reinterpret_cast<const v4f*>(partial + z * n + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += v[e];
  }
  *reinterpret_cast<v4f*>(t + i) = sum;
}

// Values of the 4-bit codes (EIGHT: of the 8-bit ones), one lane a block. ODT: output type. Bound by the store of 2 or 4 bytes a
// value: quantizing 12288 x 3072 and this back to bf16 take 45 us together.
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

// The factors in the orders the layer's kernels read them, zero-padded from rank R to P. A factor is a matrix of C columns c (k of
// lr_A, n of lr_B) by r; a workgroup takes 64 columns of one. Source: [C, R] rows (kByColumn), [R, C] rows (kByRank) or
// fragments. Results, either or none: rows [C, P], and fragments: for each 128 columns, 8-column group i of a block and
// 16 ranks, the 64 lanes' 16 bytes in a row, as mx_lowrank_kernel loads them. A launch and one or two waits for memory: 4 us for
// 2048 + 640 columns of rank 16, 5.9 for 1280 + 5120 of rank 64 (9.9 with one load in flight).
__host__ __device__ __forceinline__ int64_t frag_offset(int c, int r, int P) {
  return ((((int64_t)(c >> 7) * 4 + ((c >> 3) & 3)) * (P >> 4) + (r >> 4)) * 64 + ((c >> 5) & 3) * 16 + (r & 15)) * 8 + (c & 7);
}
struct Factor {
  const uint16_t* src;
  int64_t ld;
  int kind, C;
  uint16_t *rows, *frags;
};
__global__ __launch_bounds__(256) void mx_factors_kernel(const Factor fa, const Factor fb, int R, int P, int blocks_a) {
  __shared__ uint16_t tile[64][66];   // [c][r]; a pitch of 33 words: both directions spread over the banks
  const bool is_a = (int)blockIdx.x < blocks_a;
  const Factor f = is_a ? fa : fb;
  const int c0 = ((int)blockIdx.x - (is_a ? 0 : blocks_a)) * 64, log_p = P == 32 ? 5 : 6;
  if (!f.rows && !f.frags) return;
  auto at = [&](int i, int& c, int& r) {
    if (f.kind == PQ_MX_BY_RANK) { r = i >> 6; c = i & 63; }   // read along c
    else { c = i >> log_p; r = i & (P - 1); }                  // read along r
  };
  for (int i0 = threadIdx.x; i0 < 64 * P; i0 += 8 * 256) {   // eight loads in flight (64 P is a multiple of 8 * 256)
    uint16_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      int c, r;
      at(i0 + e * 256, c, r);
      const bool in = c0 + c < f.C && r < R;
      v[e] = !in ? 0 : f.kind == PQ_MX_BY_COLUMN ? f.src[(int64_t)(c0 + c) * f.ld + r]
                     : f.kind == PQ_MX_BY_RANK   ? f.src[(int64_t)r * f.ld + c0 + c]
                                                 : f.src[frag_offset(c0 + c, r, P)];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      int c, r;
      at(i0 + e * 256, c, r);
      tile[c][r] = v[e];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * P; i += 256) {
    if (f.frags) {   // 8 columns of one rank: 16 bytes
      const int g = i & 7, r = i >> 3;
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = tile[8 * g + 2 * e][r] | ((uint32_t)tile[8 * g + 2 * e + 1][r] << 16);
      *reinterpret_cast<v4u*>(f.frags + frag_offset(c0 + 8 * g, r, P)) = v4u{w[0], w[1], w[2], w[3]};
    }
    if (f.rows) {    // 8 ranks of one column
      const int g = i & (P / 8 - 1), c = i >> (log_p - 3);
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = tile[c][8 * g + 2 * e] | ((uint32_t)tile[c][8 * g + 2 * e + 1] << 16);
      if (c0 + c < f.C) *reinterpret_cast<v4u*>(f.rows + (int64_t)(c0 + c) * P + 8 * g) = v4u{w[0], w[1], w[2], w[3]};
    }
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

// Slices of K for few rows: a compute unit draws 75-150 GB/s, and a group of 16 rows reads all of l1t, so below 128 groups long
// rows are shared by up to eight workgroups (512 x 12288, rank 32: 23.5 us on 32 of them).
int lowrank_slices(int64_t M, int64_t K) {
  const int64_t groups = (M + 15) / 16;
  return groups >= 128 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>({8, 256 / groups, stages(K) / 16}));
}

template <int DT, int R, int RG, int NW>
int launch_lowrank(const uint16_t* x, int64_t M, int64_t K, int64_t ldx, const uint16_t* l1f, uint8_t* codes, uint8_t* scales,
                   int8_t* q8, float* t, int slices, hipStream_t stream) {
  const int64_t blocks = (M + 16 * RG - 1) / (16 * RG);
  if (const int st = check_grid(blocks, 64 * NW, "mx_lowrank")) return st;
  const dim3 grid((unsigned)blocks, (unsigned)slices), block(64 * NW);
  const int KT = stages(K);
#define PQ_MXL(Q, C) \
  hipLaunchKernelGGL((mx_lowrank_kernel<DT, R, RG, NW, Q, C>), grid, block, 0, stream, x, ldx, M, (int)K, KT, l1f, codes, scales, q8, \
                     t)
  if (!codes) PQ_MXL(false, false); else if (q8) PQ_MXL(true, true); else PQ_MXL(true, false);
#undef PQ_MXL
  return check_launch("mx_lowrank");
}

}  // namespace
}  // namespace mx
}  // namespace pq

using namespace pq;
using namespace pq::mx;

int64_t pq::mx::lowrank_workspace(int64_t M, int64_t K, int64_t R) {
  const int slices = lowrank_slices(M, K);
  return slices > 1 ? 4 * slices * M * R : 0;
}

// Rows a workgroup takes, and its waves: 16 and 16, 32 and 8, or 64 and 4 (us, bf16; t alone / with the 4-bit codes / with these and
// the 8-bit ones; quantizer and product of their own, rank 32: 65536 x 3072 161, 16384 x 3072 48, 4096 x 3072 20, 2050 x 1280 12):
//   M x K           rank 32: 16 rows       32 rows          64 rows         rank 64: 16 rows       32 rows          64 rows
//   65536 x 3072     120 / 126 / 179   105 / 107 / 160    95 / 103 / 153    142 / 193 / 241   117 / 130 / 180   103 / 115 / 163
//   16384 x 12288    119 / 132 / 196   104 / 117 / 178   101 / 124 / 182    146 / 169 / 233   118 / 133 / 192   110 / 134 / 193
//   16384 x 3072      23 /  26 /  35    21 /  25 /  35    22 /  30 /  43     33 /  46 /  55    25 /  31 /  40    25 /  32 /  44
//   8192 x 3072       14 /  16 /  20    13 /  15 /  20    19 /  24 /  34     18 /  25 /  30    15 /  18 /  22    22 /  26 /  36
//   4352 x 3072       10 /  14 /  18    11 /  12 /  17    19 /  23 /  32     15 /  20 /  26    12 /  14 /  19    20 /  25 /  34
//   4096 x 3072      6.5 / 9.8 /  12    10 /  12 /  17    16 /  23 /  32    8.5 /  14 /  16    12 /  14 /  19    18 /  25 /  34
//   2050 x 5120      8.9 /  13 /  16    13 /  17 /  25    25 /  36 /  50     12 /  18 /  21    16 /  21 /  28    27 /  38 /  53
//   2050 x 1280      4.0 / 4.8 / 5.7   5.2 / 5.6 / 7.3   8.3 /  11 /  16    4.9 / 6.1 / 7.0   5.9 / 6.4 / 8.0   9.2 /  13 /  17
int pq::mx::lowrank(const void* x, int32_t dtype, int64_t M, int64_t K, int64_t ldx, const void* l1f, int64_t R, uint8_t* codes,
                    uint8_t* scales, int8_t* q8, float* t, void* workspace, hipStream_t stream) {
  const int slices = lowrank_slices(M, K);
  float* const partial = slices > 1 ? static_cast<float*>(workspace) : nullptr;
  auto launch = [&](auto rg, auto nw) {
    constexpr int RG = decltype(rg)::value, NW = decltype(nw)::value;
#define PQ_MXL(D, RR)                                                                                               \
  launch_lowrank<D, RR, RG, NW>(static_cast<const uint16_t*>(x), M, K, ldx, static_cast<const uint16_t*>(l1f), codes, scales, q8, \
                                partial ? partial : t, slices, stream)
    if (dtype == PQ_BF16) return R == 32 ? PQ_MXL(PQ_BF16, 32) : PQ_MXL(PQ_BF16, 64);
    return R == 32 ? PQ_MXL(PQ_F16, 32) : PQ_MXL(PQ_F16, 64);
#undef PQ_MXL
  };
  using std::integral_constant;
  const int st = M <= 16 * 256  ? launch(integral_constant<int, 1>{}, integral_constant<int, 16>{})
                 : M < 32768    ? launch(integral_constant<int, 2>{}, integral_constant<int, 8>{})
                                : launch(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  if (st || !partial) return st;
  const int64_t n = M * R;
  const dim3 grid((unsigned)((n / 4 + 255) / 256)), block(256);
  hipLaunchKernelGGL(mx_lowrank_join_kernel, grid, block, 0, stream, partial, slices, n, t);
  return check_launch("mx_lowrank_join");
}

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

extern "C" int pq_mx_factors(const void* A, int64_t lda, int32_t a_order, const void* B, int64_t ldb, int32_t b_order, int64_t K,
                             int64_t N, int64_t R, int64_t P, void* af, void* ap, void* bt, void* bf, hipStream_t stream) {
  if (K < 1 || N < 1 || R < 1 || R > P || (P != 32 && P != 64) || K > (1 << 30) || N > (1 << 30))
    return set_error(PQ_ESHAPE, "pq_mx_factors: K=%lld N=%lld R=%lld P=%lld (R <= P, P 32 or 64)", (long long)K, (long long)N,
                     (long long)R, (long long)P);
  if (!A || !B) return set_error(PQ_EINVAL, "pq_mx_factors: null pointer");
  for (const int32_t o : {a_order, b_order})
    if (o != PQ_MX_BY_COLUMN && o != PQ_MX_BY_RANK && o != PQ_MX_FRAGMENTS) return set_error(PQ_EINVAL, "pq_mx_factors: order %d", o);
  auto short_rows = [&](int32_t o, int64_t ld, int64_t C) { return (o == PQ_MX_BY_COLUMN && ld < R) || (o == PQ_MX_BY_RANK && ld < C); };
  if (short_rows(a_order, lda, K) || short_rows(b_order, ldb, N))
    return set_error(PQ_ESHAPE, "pq_mx_factors: lda=%lld ldb=%lld", (long long)lda, (long long)ldb);
  for (const void* p : {(const void*)af, (const void*)ap, (const void*)bt, (const void*)bf})
    if ((uintptr_t)p % 16) return set_error(PQ_EALIGN, "pq_mx_factors: results 16-byte aligned");
  auto u16 = [](void* p) { return static_cast<uint16_t*>(p); };
  const Factor fa{static_cast<const uint16_t*>(A), lda, a_order, (int)K, u16(ap), u16(af)};
  const Factor fb{static_cast<const uint16_t*>(B), ldb, b_order, (int)N, u16(bt), u16(bf)};
  const int blocks_a = 2 * stages(K), blocks_b = 2 * stages(N);   // (64 columns each; fragments are whole stages of 128)
  hipLaunchKernelGGL(mx_factors_kernel, dim3(blocks_a + blocks_b), dim3(256), 0, stream, fa, fb, (int)R, (int)P, blocks_a);
  return check_launch("mx_factors");
}

extern "C" int64_t pq_mx_lowrank_workspace_size(int64_t M, int64_t K, int64_t R) {
  return M < 1 || K < 16 || K > (1 << 30) || (R != 32 && R != 64) ? 0 : lowrank_workspace(M, K, R);
}

extern "C" int pq_mx_lowrank_down(const void* x, int32_t dtype, int64_t M, int64_t K, int64_t ldx, const void* l1f, int64_t R,
                                  float* t, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (M < 0 || K < 16 || K % 16 || ldx < K || K > (1 << 30) || (R != 32 && R != 64))
    return set_error(PQ_ESHAPE, "pq_mx_lowrank_down: M=%lld K=%lld ldx=%lld R=%lld (K %% 16 == 0, R 32 or 64)", (long long)M,
                     (long long)K, (long long)ldx, (long long)R);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_mx_lowrank_down: dtype %d", dtype);
  if (M == 0) return PQ_OK;
  if (!x || !l1f || !t) return set_error(PQ_EINVAL, "pq_mx_lowrank_down: null pointer");
  if ((uintptr_t)x % 16 || ldx % 8 || (uintptr_t)l1f % 16 || (uintptr_t)t % 16)
    return set_error(PQ_EALIGN, "pq_mx_lowrank_down: operands 16-byte aligned, ldx a multiple of 8");
  const int64_t need = lowrank_workspace(M, K, R);
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return set_error(PQ_EINVAL, "pq_mx_lowrank_down: a workspace of %lld bytes, 16-byte aligned", (long long)need);
  return lowrank(x, dtype, M, K, ldx, l1f, R, nullptr, nullptr, nullptr, t, workspace, stream);
}
