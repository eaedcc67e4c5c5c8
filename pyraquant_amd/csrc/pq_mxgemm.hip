// Product of two microscaled 4-bit matrices (pq_mx.h), with the low-rank term and the bias in its epilogue:
//   y[m, n] = sum_k xh[m, k] wh[n, k]  (+ sum_r t[m, r] l2t[n, r])  (+ bias[n]),  rounded once to 16 bits.
//
// The matrix instructions take the 4-bit codes and the scale bytes as they are stored (v_mfma_scale_f32_32x32x64_f8f6f4:
// 64 values of k a step, one scale byte per lane and operand) and sum in fp32. The row operand is a weight row n and the
// column operand an activation row m, so each lane holds 4 consecutive n of one output row.
//
// Large products are bound by the matrix units at the power limit (50-62 % busy at 1.7-1.5 GHz; from registers alone the same
// instructions reach 6.5 PFLOP/s): 16384 x 12288 x 12288 in 1070 us, 4.6 PFLOP/s, with rank 32 1126 to 1180; 65536 x 3072 x 12288 with
// rank 32 in 1390 to 1475 us, 3.6 to 3.4, without 1259 (both parts of t: 70 us more than the first alone). With a short K the
// output's bytes bind (8202 x 640 x 5120: 32 us, 84 MB out), with few rows the start of a launch and LDS.
#include "pq_mx.h"

#include <algorithm>
#include <type_traits>

namespace pq {
namespace mx {
namespace {

struct GemmArgs {
  const uint8_t *a, *as, *w, *ws;   // codes and scales of x and of the weight
  const float* bias;
  const float* t;
  const uint16_t* l2t;
  uint16_t* c;
  int ldt, ldc;
  int M, N, KT;
  int tiles_m, tiles_n;
};

// One step over 64 values: both operands 4-bit (format code 4), scale byte S of each scale word.
template <int S>
__device__ __forceinline__ v16f mfma4(v4i a, int sa, v4i b, int sb, v16f c) {
  const v8i a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, S, sa, S, sb);
}

// Sums of one output block, then its epilogue. WMW waves along m times 2 along n; each wave holds TI x TJ tiles of 32 x 32 (n
// x m). K advances in stages of 128 values (64 bytes a row) through a ring of NS stages in LDS, filled by LDS-DMA: NS - 1
// stages in flight, no registers or LDS writes spent on them. A stage is the row blocks of the packed layout as they are (the
// swizzle keeps the ds_read_b128 of 32 rows free of bank conflicts), and after them their scale words, 4 bytes a row.
// KG groups of these waves, each with a ring of its own, take every KG-th stage; their sums are added in LDS in group order.
template <int TI, int TJ, int WMW, int NS>
struct Ring {
  static constexpr int NW = 2 * WMW, BN = 64 * TI, BM = 32 * TJ * WMW;
  static constexpr int CODES = (BN + BM) * 64, SLOTS = (BN + BM) / 64;   // bytes of codes; 256-byte pieces of scales
  static constexpr int STAGE = CODES + NW * 256;                         // (a wave without a piece of scales has a slot too)
  static constexpr int DW = BN / 16 / NW, DA = BM / 16 / NW, DPW = DW + DA + 1;   // DMA instructions a wave and stage
  static_assert(DW * 16 * NW == BN && DA * 16 * NW == BM && SLOTS <= NW, "a stage split over the waves");
  static constexpr int LDS = NS * STAGE;
  static constexpr int PITCH = 144;   // output staging: 64 outputs of a row and 16 bytes of padding
};

template <int TI, int TJ, int WMW, int NS, int OCC, int KG, int DT, int R>
__global__ __attribute__((amdgpu_flat_work_group_size(128 * WMW * KG, 128 * WMW * KG),
                          amdgpu_waves_per_eu(OCC * WMW * KG / 2, OCC * WMW * KG / 2)))
void mx_gemm_kernel(const GemmArgs p) {
  using T = Ring<TI, TJ, WMW, NS>;
  constexpr int NW = T::NW, BN = T::BN, BM = T::BM;
  __shared__ __attribute__((aligned(1024))) uint8_t rings[KG * T::LDS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6) % NW;
  const int group = __builtin_amdgcn_readfirstlane(tid >> 6) / NW;
  uint8_t* const smem = rings + group * T::LDS;
  const int wn = wave & 1, wm = wave >> 1, l32 = lane & 31, half = lane >> 5;
  int tm, tn;
  tile_of(blockIdx.x, gridDim.x, p.tiles_m, p.tiles_n, OCC == 1 ? 6 : 8, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN, KT = p.KT;

  // Row blocks past the end, and stages past the last, lie outside the buffers: their loads read nothing and give zeros.
  const int blk_w = (min(BN, p.N - n0) + 15) >> 4, blk_a = (min(BM, p.M - m0) + 15) >> 4;
  const int64_t wb = (int64_t)(n0 >> 4) * KT, ab = (int64_t)(m0 >> 4) * KT;
  const auto rs_w = __builtin_amdgcn_make_buffer_rsrc((void*)(p.w + wb * 1024), (short)0, blk_w * KT * 1024, kBufferWord3);
  const auto rs_a = __builtin_amdgcn_make_buffer_rsrc((void*)(p.a + ab * 1024), (short)0, blk_a * KT * 1024, kBufferWord3);
  const bool w_scales = wave < BN / 64;
  const auto rs_s = w_scales
      ? __builtin_amdgcn_make_buffer_rsrc((void*)(p.ws + wb * 64), (short)0, blk_w * KT * 64, kBufferWord3)
      : __builtin_amdgcn_make_buffer_rsrc((void*)(p.as + ab * 64), (short)0, wave < T::SLOTS ? blk_a * KT * 64 : 0, kBufferWord3);
  const int vw = wave * T::DW * KT * 1024 + lane * 16, va = wave * T::DA * KT * 1024 + lane * 16;
  const int vs = (((w_scales ? wave : wave - BN / 64) * 4 + (lane >> 4)) * KT) * 64 + (lane & 15) * 4;
  auto dma = [&](int buf, int kt) {
    uint8_t* const sb = smem + buf * T::STAGE;
    const int off = kt < KT ? kt * 1024 : kOOB;
#pragma unroll
    for (int i = 0; i < T::DW; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_w, (lds_void_t*)(sb + (wave * T::DW + i) * 1024), 16, vw + i * KT * 1024 + off, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < T::DA; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_a, (lds_void_t*)(sb + BN * 64 + (wave * T::DA + i) * 1024), 16,
                                               va + i * KT * 1024 + off, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_s, (lds_void_t*)(sb + T::CODES + wave * 256), 4, vs + (kt < KT ? kt * 64 : kOOB), 0, 0, 0);
  };

  const int sw = k64_swz(lane & 15);
  const int fw = (wn * (BN / 2) + l32) * 64, fa = (BN + wm * (BM / WMW) + l32) * 64;
  v4i w0[TI], w1[TI], a0[TJ], a1[TJ];
  int sw_[TI], sa_[TJ];
  auto rd = [&](v4i (&w)[TI], v4i (&a)[TJ], int buf, int s) {
    const uint8_t* const sb = smem + buf * T::STAGE;
    const int c = ((2 * s + half) ^ sw) << 4;
#pragma unroll
    for (int i = 0; i < TI; ++i) w[i] = *reinterpret_cast<const v4i*>(sb + fw + i * 2048 + c);
#pragma unroll
    for (int j = 0; j < TJ; ++j) a[j] = *reinterpret_cast<const v4i*>(sb + fa + j * 2048 + c);
  };
  auto rd_scales = [&](int (&w)[TI], int (&a)[TJ], int buf) {
    const uint8_t* const sb = smem + buf * T::STAGE + T::CODES + 2 * half;
#pragma unroll
    for (int i = 0; i < TI; ++i) w[i] = *reinterpret_cast<const uint16_t*>(sb + (fw >> 4) + i * 128);
#pragma unroll
    for (int j = 0; j < TJ; ++j) a[j] = *reinterpret_cast<const uint16_t*>(sb + (fa >> 4) + j * 128);
  };
  auto settle = [&](int (&w)[TI], int (&a)[TJ]) {
    // (kept here: the compiler would put the masking of the words between the products that use them)
#pragma unroll
    for (int i = 0; i < TI; ++i) asm volatile("" : "+v"(w[i]));
#pragma unroll
    for (int j = 0; j < TJ; ++j) asm volatile("" : "+v"(a[j]));
  };
  v16f acc[TI][TJ] = {};
  auto mm = [&](auto s, const v4i (&w)[TI], const v4i (&a)[TJ], const int (&ws)[TI], const int (&as)[TJ]) {
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[i][j] = mfma4<decltype(s)::value>(w[i], ws[i], a[j], as[j], acc[i][j]);
  };
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;

  if constexpr (NW == 8) {
    // Two groups of four waves, one wave of each per SIMD, take turns: while one issues a stage's products back to back from
    // registers, the other reads the next stage's fragments and issues its part of a DMA. Group B runs one slot behind; a
    // workgroup barrier ends each slot. Stage s + 1 has landed at the barrier that ends slot 2 s + 1 (each group waits for
    // all but its NS - 2 younger stages), and stage s + NS - 1 goes into the buffer of stage s - 1, which both groups have read.
    const bool grp_b = wave >= NW / 2;
#pragma unroll
    for (int st = 0; st < NS - 1; ++st) dma(st, st);
    wait_vmcnt<(NS - 2) * T::DPW>();
    ring_barrier();
    if (grp_b) ring_barrier();
    int b = 0;
    for (int s = 0; s < KT; ++s) {
      rd(w0, a0, b, 0);
      rd(w1, a1, b, 1);
      rd_scales(sw_, sa_, b);
      dma(b == 0 ? NS - 1 : b - 1, s + NS - 1);
      settle(sw_, sa_);
      if (grp_b) wait_vmcnt<(NS - 2) * T::DPW>();
      ring_barrier();
      mm(S0{}, w0, a0, sw_, sa_);
      mm(S1{}, w1, a1, sw_, sa_);
      if (!grp_b) wait_vmcnt<(NS - 2) * T::DPW>();
      ring_barrier();
      b = b + 1 == NS ? 0 : b + 1;
    }
    if (!grp_b) ring_barrier();
  } else {
    // The fragments of the next half stage are read while the products of this one run; one barrier a stage.
#pragma unroll
    for (int st = 0; st < NS; ++st) dma(st, st * KG + group);
    wait_vmcnt<(NS - 1) * T::DPW>();
    ring_barrier();
    rd(w0, a0, 0, 0);
    rd_scales(sw_, sa_, 0);
    int b = 0;
    for (int s = 0; s < KT; s += KG) {
      const int bn = b + 1 == NS ? 0 : b + 1;
      rd(w1, a1, b, 1);
      mm(S0{}, w0, a0, sw_, sa_);
      __builtin_amdgcn_sched_barrier(0);
      wait_vmcnt<(NS - 2) * T::DPW>();   // stage s + 1 has landed
      ring_barrier();                    // for every wave, and buffer b is read
      int nsw[TI], nsa[TJ];
      rd(w0, a0, bn, 0);
      rd_scales(nsw, nsa, bn);
      dma(b, s + NS * KG + group);
      mm(S1{}, w1, a1, sw_, sa_);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < TI; ++i) sw_[i] = nsw[i];
#pragma unroll
      for (int j = 0; j < TJ; ++j) sa_[j] = nsa[j];
      b = bn;
    }
  }
  wait_vmcnt<0>();
  __syncthreads();   // the rings become room for the groups' sums and the output staging
  if constexpr (KG > 1) {
    static_assert((KG - 1) * NW * TI * TJ * 4096 + NW * 32 * T::PITCH <= KG * T::LDS, "sums and staging in the rings");
    auto sums = [&](int g, int i, int j, int q) {
      return reinterpret_cast<v4f*>(rings) + (((((g - 1) * NW + wave) * TI + i) * TJ + j) * 4 + q) * 64 + lane;
    };
    if (group)
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *sums(group, i, j, q) = v4f{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int g = 1; g < KG; ++g)
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const v4f v = *sums(g, i, j, q);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += v[e];
          }
  }

  // Lane l holds, of tile (i, j): row m = 32 j + l % 32, outputs n = 32 i + 8 q + 4 (l / 32) .. + 3 in elements 4 q ... They
  // go through LDS two weight tiles at a time so that whole 128-byte lines are stored.
  const int nb = n0 + wn * (BN / 2), mb = m0 + wm * (BM / WMW);
  uint8_t* const stage = rings + (KG - 1) * NW * TI * TJ * 4096 + wave * 32 * T::PITCH;
#pragma unroll
  for (int j = 0; j < TJ; ++j) {
    if constexpr (R > 0) {
#pragma unroll
      for (int r0 = 0; r0 < R; r0 += 32) {
        RankPiece t[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) t[s].load(p.t + (int64_t)min(mb + 32 * j + l32, p.M - 1) * p.ldt + r0 + 16 * s + 8 * half);
        static_assert(TI == 2, "tiles of a wave");
        rank_products<DT, TI, 2>({&acc[0][j], &acc[1][j]}, t, [&](int i, int s) {
          return *reinterpret_cast<const v4i*>(p.l2t + (int64_t)min(nb + 32 * i + l32, p.N - 1) * R + r0 + 16 * s + 8 * half);
        });
      }
    }
#pragma unroll
    for (int ih = 0; ih < TI / 2; ++ih) {
#pragma unroll
      for (int ii = 0; ii < 2; ++ii) {
        const int i = 2 * ih + ii;
        const v16f& y = acc[i][j];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = nb + 32 * i + 8 * q + 4 * half;
          v4f o = v4f{y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]};
          if (p.bias && n < p.N) {
            const v4f bv = *reinterpret_cast<const v4f*>(p.bias + n);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += bv[e];
          }
          *reinterpret_cast<v2u*>(stage + l32 * T::PITCH + (ii * 32 + 8 * q + 4 * half) * 2) =
              v2u{pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3])};
        }
      }
      wave_sync();
      const int n = nb + ih * 64 + (lane & 7) * 8, row = lane >> 3;
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += 8) {
        const int m = mb + 32 * j + r0 + row;
        const v4u v = *reinterpret_cast<const v4u*>(stage + (r0 + row) * T::PITCH + (lane & 7) * 16);
        if (m < p.M && n < p.N) {
          v4u* const dst = reinterpret_cast<v4u*>(p.c + (int64_t)m * p.ldc + n);
          if constexpr (OCC == 1) __builtin_nontemporal_store(v, dst);
          else *dst = v;
        }
      }
      wave_sync();
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

template <int TI, int TJ, int WMW, int NS, int OCC, int KG>
int launch_ring(GemmArgs p, int dtype, int r, hipStream_t stream) {
  using T = Ring<TI, TJ, WMW, NS>;
  p.tiles_m = (p.M + T::BM - 1) / T::BM;
  p.tiles_n = (p.N + T::BN - 1) / T::BN;
  const int64_t blocks = (int64_t)p.tiles_m * p.tiles_n;
  if (const int st = check_grid(blocks, 128 * WMW * KG, "mx_gemm")) return st;
#define PQ_MXG(D, RR) \
  hipLaunchKernelGGL((mx_gemm_kernel<TI, TJ, WMW, NS, OCC, KG, D, RR>), dim3((unsigned)blocks), dim3(128 * WMW * KG), 0, stream, p)
  if (dtype == PQ_BF16) {
    if (r == 0) PQ_MXG(PQ_BF16, 0); else if (r == 32) PQ_MXG(PQ_BF16, 32); else PQ_MXG(PQ_BF16, 64);
  } else {
    if (r == 0) PQ_MXG(PQ_F16, 0); else if (r == 32) PQ_MXG(PQ_F16, 32); else PQ_MXG(PQ_F16, 64);
  }
#undef PQ_MXG
  return check_launch("mx_gemm");
}

// ---- large products ----------------------------------------------------------------------------------------------------
// 256 x 256 blocks on persistent workgroups of eight waves, one to a compute unit: each takes the blocks b, b + grid, .. of its
// XCD's raster. The same ring and the same turns of two wave groups as above; what a loop over blocks adds is that the next
// block's first stages and bias are on their way while this one's results go out:
//  * the sums start from the bias (through LDS, 1 KB a block), so the epilogue needs no registers for it;
//  * the epilogue's low-rank operands are loaded, then the next block's bias and stages 0 .. NS - 2 are issued into the ring that
//    the last barrier freed, then the results go out through a staging area of their own, 16 rows of 64 outputs at a time;
//  * results are stored with buffer stores, whose bounds replace branches: every wave issues the same 16, and the ring's waits
//    count them (vmcnt completes in order: 16 more may be outstanding until stage NS is waited for).
// Against one block a workgroup (with the first part of t alone): 65536 x 3072 x 12288 1562 -> 1387 us, 4096 x 3072 x 3072 31.1 -> 27.0.
template <int DT, int R>
__global__ __attribute__((amdgpu_flat_work_group_size(512, 512), amdgpu_waves_per_eu(2, 2)))
void mx_gemm_large_kernel(const GemmArgs p) {
  constexpr int TI = 4, TJ = 2, NS = 4;
  using T = Ring<TI, TJ, 4, NS>;
  constexpr int BN = T::BN, BM = T::BM, DPW = T::DPW, PITCH = T::PITCH, STORES = 2 * TI * TJ;
  constexpr int AT_STAGING = T::LDS, AT_BIAS = AT_STAGING + 8 * 16 * PITCH;   // two slots of bias, and one for the idle waves
  __shared__ __attribute__((aligned(1024))) uint8_t smem[AT_BIAS + 3 * 1024];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave & 1, wm = wave >> 1, l32 = lane & 31, half = lane >> 5, KT = p.KT;
  const bool grp_b = wave >= 4, w_scales = wave < BN / 64;
  const int vw = wave * T::DW * KT * 1024 + lane * 16, va = wave * T::DA * KT * 1024 + lane * 16;
  const int vs = ((wave & 3) * 4 + (lane >> 4)) * KT * 64 + (lane & 15) * 4;
  const int tiles = p.tiles_m * p.tiles_n;

  int m0, n0;
  __amdgpu_buffer_rsrc_t rs_w, rs_a, rs_s;
  auto set = [&](int tile) {
    int tm, tn;
    tile_of(tile, tiles, p.tiles_m, p.tiles_n, 6, tm, tn);
    m0 = tm * BM;
    n0 = tn * BN;
    const int blk_w = (min(BN, p.N - n0) + 15) >> 4, blk_a = (min(BM, p.M - m0) + 15) >> 4;
    const int64_t wb = (int64_t)(n0 >> 4) * KT, ab = (int64_t)(m0 >> 4) * KT;
    rs_w = __builtin_amdgcn_make_buffer_rsrc((void*)(p.w + wb * 1024), (short)0, blk_w * KT * 1024, kBufferWord3);
    rs_a = __builtin_amdgcn_make_buffer_rsrc((void*)(p.a + ab * 1024), (short)0, blk_a * KT * 1024, kBufferWord3);
    rs_s = __builtin_amdgcn_make_buffer_rsrc((void*)(w_scales ? p.ws + wb * 64 : p.as + ab * 64), (short)0,
                                             (w_scales ? blk_w : blk_a) * KT * 64, kBufferWord3);
  };
  auto dma = [&](int buf, int kt) {
    uint8_t* const sb = smem + buf * T::STAGE;
    const int off = kt < KT ? kt * 1024 : kOOB;
#pragma unroll
    for (int i = 0; i < T::DW; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_w, (lds_void_t*)(sb + (wave * T::DW + i) * 1024), 16, vw + i * KT * 1024 + off, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < T::DA; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_a, (lds_void_t*)(sb + BN * 64 + (wave * T::DA + i) * 1024), 16,
                                               va + i * KT * 1024 + off, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_s, (lds_void_t*)(sb + T::CODES + wave * 256), 4, vs + (kt < KT ? kt * 64 : kOOB), 0, 0, 0);
  };
  // The bias of a block to slot `slot` (waves 0-3, 64 values each) and its first stages; nothing past the last block (`any`).
  auto start = [&](int slot, bool any) {
    const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)(p.bias ? p.bias + n0 : (const float*)p.ws), (short)0,
                                                      p.bias && any ? (p.N - n0) * 4 : 0, kBufferWord3);
    uint8_t* const dst = smem + AT_BIAS + (wave < 4 ? slot * 1024 + wave * 256 : 2048 + (wave - 4) * 256);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)dst, 4, wave < 4 ? (wave * 64 + lane) * 4 : kOOB, 0, 0, 0);
#pragma unroll
    for (int st = 0; st < NS - 1; ++st) dma(st, any ? st : KT);
  };

  const int sw = k64_swz(lane & 15);
  const int fw = (wn * (BN / 2) + l32) * 64, fa = (BN + wm * (BM / 4) + l32) * 64;
  v16f acc[TI][TJ];
  // one stage: the memory phase, a barrier, the products; `stores`: that many more instructions may be outstanding when the next
  // stage has landed (one loop: the sums stay in their registers)
  auto stage_step = [&](int s, int b, bool stores) {
    auto landed = [&] {
      if (stores) wait_vmcnt<(NS - 2) * DPW + STORES>();
      else wait_vmcnt<(NS - 2) * DPW>();
    };
    const uint8_t* const sb = smem + b * T::STAGE;
    v4i w[2][TI], a[2][TJ];
    int ws[TI], as[TJ];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = ((2 * h + half) ^ sw) << 4;
#pragma unroll
      for (int i = 0; i < TI; ++i) w[h][i] = *reinterpret_cast<const v4i*>(sb + fw + i * 2048 + c);
#pragma unroll
      for (int j = 0; j < TJ; ++j) a[h][j] = *reinterpret_cast<const v4i*>(sb + fa + j * 2048 + c);
    }
#pragma unroll
    for (int i = 0; i < TI; ++i) ws[i] = *reinterpret_cast<const uint16_t*>(sb + T::CODES + (fw >> 4) + i * 128 + 2 * half);
#pragma unroll
    for (int j = 0; j < TJ; ++j) as[j] = *reinterpret_cast<const uint16_t*>(sb + T::CODES + (fa >> 4) + j * 128 + 2 * half);
    dma(b == 0 ? NS - 1 : b - 1, s + NS - 1);
    // (kept here: the compiler would put the masking of the words between the products that use them)
#pragma unroll
    for (int i = 0; i < TI; ++i) asm volatile("" : "+v"(ws[i]));
#pragma unroll
    for (int j = 0; j < TJ; ++j) asm volatile("" : "+v"(as[j]));
    if (grp_b) landed();
    ring_barrier();
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[i][j] = mfma4<0>(w[0][i], ws[i], a[0][j], as[j], acc[i][j]);
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[i][j] = mfma4<1>(w[1][i], ws[i], a[1][j], as[j], acc[i][j]);
    if (!grp_b) landed();
    ring_barrier();
  };

  int tile = blockIdx.x, slot = 0;
  set(tile);
  start(0, true);
  wait_vmcnt<(NS - 2) * DPW>();   // the first block's bias and stage 0
  while (true) {
    ring_barrier();
    {   // the sums start from the bias
      const float* const bs = reinterpret_cast<const float*>(smem + AT_BIAS + slot * 1024) + wn * (BN / 2) + 4 * half;
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v4f v = {};
          if (p.bias) v = *reinterpret_cast<const v4f*>(bs + 32 * i + 8 * q);
#pragma unroll
          for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = v[e];
        }
    }
    if (grp_b) ring_barrier();
    // Stages 1 and 2 are waited for with the previous block's stores still out (the first block has none).
    const int lead = tile != (int)blockIdx.x ? NS - 2 : 0;
    int b = 0;
    for (int s = 0; s < KT; ++s) {
      stage_step(s, b, s < lead);
      b = b + 1 == NS ? 0 : b + 1;
    }
    if (!grp_b) ring_barrier();
    wait_vmcnt<0>();
    ring_barrier();   // every wave is done with the ring

    // Lane l holds, of tile (i, j): row m = 32 j + l % 32, outputs n = 32 i + 8 q + 4 (l / 32) .. + 3 in elements 4 q ..
    const int nb = n0 + wn * (BN / 2), mb = m0 + wm * (BM / 4);
    const int m_out = m0, n_out = n0;
    const int next = tile + (int)gridDim.x;
    const bool more = next < tiles;
    auto go_on = [&] {
      tile = next;
      slot ^= 1;
      if (more) set(tile);
      start(slot, more);
    };
    // The low-rank term, 32 ranks at a time; the next block starts once the last operands are asked for.
    if constexpr (R > 0) {
#pragma unroll
      for (int r0 = 0; r0 < R; r0 += 32) {
        RankPiece tv[TJ][2];
        v4i lv[TI][2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int j = 0; j < TJ; ++j)
            tv[j][x].load(p.t + (int64_t)min(mb + 32 * j + l32, p.M - 1) * p.ldt + r0 + 16 * x + 8 * half);
#pragma unroll
          for (int i = 0; i < TI; ++i)
            lv[i][x] = *reinterpret_cast<const v4i*>(p.l2t + (int64_t)min(nb + 32 * i + l32, p.N - 1) * R + r0 + 16 * x + 8 * half);
        }
        if (r0 + 32 == R) go_on();
#pragma unroll
        for (int j = 0; j < TJ; ++j)
          rank_products<DT, TI, 2>({&acc[0][j], &acc[1][j], &acc[2][j], &acc[3][j]}, tv[j], [&](int i, int x) { return lv[i][x]; });
      }
    } else {
      go_on();
    }
    const int valid_n = p.N - n_out;
    const auto rs_c = __builtin_amdgcn_make_buffer_rsrc((void*)(p.c + (int64_t)m_out * p.ldc + n_out), (short)0,
                                                        ((min(BM, p.M - m_out) - 1) * p.ldc + min(BN, valid_n)) * 2, kBufferWord3);
    uint8_t* const out = smem + AT_STAGING + wave * 16 * PITCH;
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
      for (int ih = 0; ih < TI / 2; ++ih) {
        v2u y[2][4];
#pragma unroll
        for (int ii = 0; ii < 2; ++ii) {
          const v16f& v = acc[2 * ih + ii][j];
#pragma unroll
          for (int q = 0; q < 4; ++q) y[ii][q] = v2u{pack2<DT>(v[4 * q], v[4 * q + 1]), pack2<DT>(v[4 * q + 2], v[4 * q + 3])};
        }
#pragma unroll
        for (int rows = 0; rows < 2; ++rows) {   // 16 of the 32 rows
          if ((l32 >> 4) == rows) {
#pragma unroll
            for (int ii = 0; ii < 2; ++ii)
#pragma unroll
              for (int q = 0; q < 4; ++q)
                *reinterpret_cast<v2u*>(out + (l32 & 15) * PITCH + (ii * 32 + 8 * q + 4 * half) * 2) = y[ii][q];
          }
          wave_sync();
          const int n = wn * (BN / 2) + ih * 64 + (lane & 7) * 8;
#pragma unroll
          for (int r0 = 0; r0 < 16; r0 += 8) {
            const int m = wm * (BM / 4) + 32 * j + 16 * rows + r0 + (lane >> 3);
            const v4u v = *reinterpret_cast<const v4u*>(out + (r0 + (lane >> 3)) * PITCH + (lane & 7) * 16);
            const int off = n < valid_n ? (m * p.ldc + n) * 2 : kOOB;
            __builtin_amdgcn_raw_buffer_store_b128(v, rs_c, off, 0, 2);   // (2: streamed past the L2)
          }
          wave_sync();
        }
      }
    if (!more) break;
    wait_vmcnt<(NS - 2) * DPW + STORES>();   // the next block's bias and stage 0
  }
  wait_vmcnt<0>();   // (no DMA outlives the workgroup's LDS)
}

template <int DT>
int launch_large(GemmArgs p, int r, int cus, hipStream_t stream) {
  p.tiles_m = (p.M + 255) / 256;
  p.tiles_n = (p.N + 255) / 256;
  const int64_t blocks = (int64_t)p.tiles_m * p.tiles_n;
  if (blocks > 0x7fffffff - cus) return set_error(PQ_ESHAPE, "mx_gemm: M=%d N=%d too large", p.M, p.N);
  const dim3 grid((unsigned)std::min<int64_t>(blocks, cus)), block(512);
  if (r == 0) hipLaunchKernelGGL((mx_gemm_large_kernel<DT, 0>), grid, block, 0, stream, p);
  else if (r == 32) hipLaunchKernelGGL((mx_gemm_large_kernel<DT, 32>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((mx_gemm_large_kernel<DT, 64>), grid, block, 0, stream, p);
  return check_launch("mx_gemm");
}

// ---- few blocks --------------------------------------------------------------------------------------------------------
// Where the blocks of the kernel above would leave most compute units idle, a workgroup of NW waves takes a block of 32 TI x 32
// TJ and its waves every NW-th stage of K, each with all of the block's sums; fragments come from memory into registers, D
// stages ahead, and the waves' sums are added in LDS in a fixed order. QUANT: x is 16-bit, and each lane quantizes the very
// blocks its fragments are (32 consecutive values of a row), so few rows need no quantizer of their own before the product.
// Bound by the latency of a launch and of a wave's first loads: 154 x 2048 x 1280 4.3 us; 1 x 12288 x 3072 8.3 us for 20 MB.
struct SplitArgs {
  GemmArgs g;
  const uint16_t* x;   // QUANT
  int64_t ldx;
  int K;
};

template <int TI, int TJ, int NW, int D, int DT, int R, bool QUANT>
__global__ __launch_bounds__(64 * NW) void mx_gemm_split_kernel(const SplitArgs sp) {
  const GemmArgs& p = sp.g;
  __shared__ float part[NW][64 * 17];   // one 32 x 32 tile of each wave, 16 sums a lane (17: spread over the banks)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 32 * TI, m0 = blockIdx.y * 32 * TJ, KT = p.KT;
  const int l32 = lane & 31, half = lane >> 5, r16 = lane & 15, sw = k64_swz(r16);
  int64_t wb[TI], ab[TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)   // (row blocks past the end repeat the last one: their outputs are not stored)
    wb[i] = (int64_t)min((n0 + 32 * i + l32) >> 4, (p.N - 1) >> 4) * KT;
#pragma unroll
  for (int j = 0; j < TJ; ++j)
    ab[j] = QUANT ? (int64_t)(m0 + 32 * j + l32) * sp.ldx : (int64_t)min((m0 + 32 * j + l32) >> 4, (p.M - 1) >> 4) * KT;
  struct Stage {
    v4i w[2][TI], a[2][QUANT ? 1 : TJ];
    Block<DT> x[2][QUANT ? TJ : 1];
    int ws[TI], as[QUANT ? 1 : TJ];
  } st[D];
  auto load = [&](Stage& g, int kt) {
#pragma unroll
    for (int i = 0; i < TI; ++i) g.ws[i] = *reinterpret_cast<const uint16_t*>(p.ws + (wb[i] + kt) * 64 + r16 * 4 + 2 * half);
    if constexpr (!QUANT) {
#pragma unroll
      for (int j = 0; j < TJ; ++j) g.as[j] = *reinterpret_cast<const uint16_t*>(p.as + (ab[j] + kt) * 64 + r16 * 4 + 2 * half);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int off = r16 * 64 + (((2 * s + half) ^ sw) << 4);
#pragma unroll
      for (int i = 0; i < TI; ++i) g.w[s][i] = *reinterpret_cast<const v4i*>(p.w + (wb[i] + kt) * 1024 + off);
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        if constexpr (QUANT) {
          const int k = kt * 128 + (2 * s + half) * kBlock;
          if (m0 + 32 * j + l32 < p.M && k < sp.K) g.x[s][j].template load<true>(sp.x + ab[j] + k);
          else g.x[s][j].zero();
        } else {
          g.a[s][j] = *reinterpret_cast<const v4i*>(p.a + (ab[j] + kt) * 1024 + off);
        }
      }
    }
  };
  v16f acc[TI][TJ] = {};
  auto products = [&](auto s, const Stage& g) {
    constexpr int S = decltype(s)::value;
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      v4i a;
      int as;
      if constexpr (QUANT) {
        as = g.x[S][j].scale_byte();
        a = g.x[S][j].codes(as);
        as = as << (8 * S);
      } else {
        a = g.a[S][j];
        as = g.as[j];
      }
#pragma unroll
      for (int i = 0; i < TI; ++i) acc[i][j] = mfma4<S>(g.w[S][i], g.ws[i], a, as, acc[i][j]);
    }
  };
  const int mine = (KT - wave + NW - 1) / NW;   // stages wave, wave + NW, ..
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < mine) load(st[d], wave + d * NW);
  for (int c = 0; c < mine; c += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (c + d < mine) {
        products(std::integral_constant<int, 0>{}, st[d]);
        products(std::integral_constant<int, 1>{}, st[d]);
        if (c + d + D < mine) load(st[d], wave + (c + d + D) * NW);
      }
    }
  }
  // The waves' sums, a tile at a time: all of them leave theirs in LDS, and one wave adds them up.
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      if (i + j) __syncthreads();
#pragma unroll
      for (int r = 0; r < 16; ++r) part[wave][lane * 17 + r] = acc[i][j][r];
      __syncthreads();
      if (wave == (i * TJ + j) % NW) {   // (its lanes hold the layout the low-rank products have)
        v16f y = {};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float s = 0.0f;
#pragma unroll
          for (int u = 0; u < NW; ++u) s += part[u][lane * 17 + r];
          y[r] = s;
        }
        const int m = m0 + 32 * j + l32;
        if constexpr (R > 0) {
#pragma unroll
          for (int r0 = 0; r0 < R; r0 += 32) {
            RankPiece t[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) t[s].load(p.t + (int64_t)min(m, p.M - 1) * p.ldt + r0 + 16 * s + 8 * half);
            rank_products<DT, 1, 2>({&y}, t, [&](int, int s) {
              return *reinterpret_cast<const v4i*>(p.l2t + (int64_t)min(n0 + 32 * i + l32, p.N - 1) * R + r0 + 16 * s + 8 * half);
            });
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n0 + 32 * i + 8 * q + 4 * half;
          if (m < p.M && n < p.N) {
            v4f o = v4f{y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]};
            if (p.bias) {
              const v4f bv = *reinterpret_cast<const v4f*>(p.bias + n);
#pragma unroll
              for (int e = 0; e < 4; ++e) o[e] += bv[e];
            }
            *reinterpret_cast<v2u*>(p.c + (int64_t)m * p.ldc + n) = v2u{pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3])};
          }
        }
      }
    }
}

template <int TI, int TJ, int NW, int D, bool QUANT>
int launch_split(const SplitArgs& p, int dtype, int r, hipStream_t stream) {
  const int64_t bm = (p.g.M + 32 * TJ - 1) / (32 * TJ), bn = (p.g.N + 32 * TI - 1) / (32 * TI);
  if (bm > 65535) return set_error(PQ_ESHAPE, "mx_gemm: M=%d too large", p.g.M);
  if (const int st = check_grid(bn, 64 * NW, "mx_gemm")) return st;
#define PQ_MXP(D_, RR)                                                                                              \
  hipLaunchKernelGGL((mx_gemm_split_kernel<TI, TJ, NW, D, D_, RR, QUANT>), dim3((unsigned)bn, (unsigned)bm), dim3(64 * NW), \
                     0, stream, p)
  if (dtype == PQ_BF16) {
    if (r == 0) PQ_MXP(PQ_BF16, 0); else if (r == 32) PQ_MXP(PQ_BF16, 32); else PQ_MXP(PQ_BF16, 64);
  } else {
    if (r == 0) PQ_MXP(PQ_F16, 0); else if (r == 32) PQ_MXP(PQ_F16, 32); else PQ_MXP(PQ_F16, 64);
  }
#undef PQ_MXP
  return check_launch("mx_gemm");
}

// The block of a product, by how its blocks fill the chip. us of the kernel (bf16, rank 32, bias):
//   M x K x N            256x256  128x256  128x64  128x64, 3 groups  32x32 split   (n x m; 256x256, 128x256: one workgroup per CU)
//   65536 x 3072 x 12288   1390     1848    2253                                   (256x256: persistent, times the CUs' rounds)
//   4096 x 3072 x 3072     27.2     38.3    38.2         50.4          97.8
//   2050 x 1280 x 5120     15.9     24.2    22.6         37.5          48.2        180 blocks of 256 x 256
//   512 x 3072 x 12288     24.0     20.9    22.0         27.4          50.0        192 blocks of 128 x 256, 384 of 128 x 128
//   1024 x 3072 x 3072     23.7     18.8    12.2         16.6          25.3        384 blocks of 128 x 64
//   512 x 12288 x 3072     68.6     50.7    24.9         21.2          35.0        192 blocks of 128 x 64, one to a CU
//   512 x 3072 x 3072      23.5     18.9     9.6          9.4          14.1        the same, 24 stages of K
//   300 x 640 x 5120       11.8     10.5     5.6          6.9           8.7        5 stages: the groups' join costs more
//   256 x 3072 x 3072      23.6     18.6     9.2          9.1           8.3        768 blocks of 32 x 32
//   154 x 2048 x 1280      18.0     14.2     7.3          7.8           4.4
//   1 x 12288 x 3072       67.4     47.5    22.3         17.5           8.8
// (128 x 128 won nowhere and is not built. What the last column gets fits two of its workgroups per CU at once. A lone
// workgroup of four waves leaves LDS idle between its barriers; three groups of four keep it busy: 96 stages of 12 KB in and 24
// KB out at 128 B a clock are 14 us. Deeper rings alone changed nothing.)
int launch_gemm(const GemmArgs& p, int dtype, int r, hipStream_t stream) {
  auto blocks = [&](int bn, int bm) { return (int64_t)((p.N + bn - 1) / bn) * ((p.M + bm - 1) / bm); };
  int cus = persistent_workgroups(stream);
  if (cus <= 0) cus = 256;
  if (blocks(32, 32) <= 3 * cus) return launch_split<1, 1, 8, 4, false>({p, nullptr, 0, 0}, dtype, r, stream);
  if (blocks(256, 256) > cus / 2) return dtype == PQ_BF16 ? launch_large<PQ_BF16>(p, r, cus, stream) : launch_large<PQ_F16>(p, r, cus, stream);
  if (blocks(128, 128) > cus) return launch_ring<2, 2, 4, 4, 1, 1>(p, dtype, r, stream);
  if (blocks(128, 64) <= cus && p.KT > 24) return launch_ring<2, 1, 2, 4, 1, 3>(p, dtype, r, stream);
  return launch_ring<2, 1, 2, 4, 2, 1>(p, dtype, r, stream);
}

// Few short rows are quantized by the product's own lanes, once per 32 outputs: a launch less. us on the GPU (bf16), quantizer and
// product / the product alone: 1 x 1280 x 1280 5.2 / 4.3, 8 x 1536 x 1536 5.4 / 4.9, 32 x 640 x 640 5.2 / 4.2, 8 x 2048 x 1280
// 5.7 / 5.7 (and 7.6 / 5.9 where the launches bind), but 32 x 2048 x 1280 5.9 / 7.2, 1 x 12288 x 3072 10.2 / 17.4.
inline bool quantized_inside(int64_t M, int64_t K) { return M <= 32 && K <= 2048 && M * K <= 32768; }

}  // namespace
}  // namespace mx
}  // namespace pq

using namespace pq;

extern "C" int pq_mx_gemm(const uint8_t* a, const uint8_t* a_scales, const uint8_t* w, const uint8_t* w_scales,
                          const float* bias, const float* t, int64_t ldt, const void* l2t, int64_t R, void* c, int64_t ldc,
                          int32_t dtype, int64_t M, int64_t N, int64_t K, hipStream_t stream) {
  if (M < 0 || N < 16 || N % 16 || K < 32 || K % 32 || ldc < N || ldc > (1 << 21) || M > (1 << 30) ||
      N > (1 << 30) || K > (1 << 22))
    return set_error(PQ_ESHAPE, "pq_mx_gemm: M=%lld N=%lld K=%lld ldc=%lld (N %% 16 == 0, K %% 32 == 0, ldc <= 2^21)", (long long)M,
                     (long long)N, (long long)K, (long long)ldc);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_mx_gemm: dtype %d", dtype);
  if (t ? (R != 32 && R != 64) || ldt < R || ldt > (1 << 22) : false)
    return set_error(PQ_ESHAPE, "pq_mx_gemm: rank %lld (32 or 64), ldt=%lld", (long long)R, (long long)ldt);
  if (M == 0) return PQ_OK;
  if (!a || !a_scales || !w || !w_scales || !c || (t && !l2t)) return set_error(PQ_EINVAL, "pq_mx_gemm: null pointer");
  if ((uintptr_t)a % 16 || (uintptr_t)w % 16 || (uintptr_t)a_scales % 16 || (uintptr_t)w_scales % 16 || (uintptr_t)c % 16 ||
      ldc % 8 || (uintptr_t)bias % 16 || (t && ((uintptr_t)t % 16 || (uintptr_t)l2t % 16 || ldt % 8)))
    return set_error(PQ_EALIGN, "pq_mx_gemm: operands 16-byte aligned, ldc and ldt multiples of 8");
  mx::GemmArgs p{a, a_scales, w, w_scales, bias, t, static_cast<const uint16_t*>(l2t),
                 static_cast<uint16_t*>(c), (int)ldt, (int)ldc, (int)M, (int)N, mx::stages(K), 0, 0};
  return mx::launch_gemm(p, dtype, t ? (int)R : 0, stream);
}

extern "C" int pq_mx_linear(const void* x, int32_t dtype, int64_t M, int64_t K, int64_t ldx, const uint8_t* w,
                            const uint8_t* w_scales, const float* bias, const void* l1f, const void* l2t, int64_t R, void* y,
                            int64_t ldy, int64_t N, uint8_t* codes, uint8_t* scales, int8_t* q8, float* t, void* workspace,
                            int64_t workspace_bytes, hipStream_t stream) {
  if (M < 0 || N < 16 || N % 16 || K < 32 || K % 32 || ldx < K || ldy < N || ldy > (1 << 21) || M > (1 << 30) ||
      N > (1 << 30) || K > (1 << 22))
    return set_error(PQ_ESHAPE, "pq_mx_linear: M=%lld N=%lld K=%lld ldx=%lld ldy=%lld (N %% 16 == 0, K %% 32 == 0)", (long long)M,
                     (long long)N, (long long)K, (long long)ldx, (long long)ldy);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_mx_linear: dtype %d", dtype);
  if (R != 0 && R != 32 && R != 64) return set_error(PQ_ESHAPE, "pq_mx_linear: rank %lld (0, 32 or 64)", (long long)R);
  if (M == 0) return PQ_OK;
  if (!x || !w || !w_scales || !y || !codes || !scales || (R && (!l1f || !l2t || !t)))
    return set_error(PQ_EINVAL, "pq_mx_linear: null pointer");
  if ((uintptr_t)x % 16 || ldx % 8 || (uintptr_t)w % 16 || (uintptr_t)w_scales % 16 || (uintptr_t)y % 16 || ldy % 8 ||
      (uintptr_t)bias % 16 || (uintptr_t)codes % 16 || (uintptr_t)scales % 16 || (uintptr_t)q8 % 16 ||
      (R && ((uintptr_t)l1f % 16 || (uintptr_t)l2t % 16 || (uintptr_t)t % 16)))
    return set_error(PQ_EALIGN, "pq_mx_linear: operands 16-byte aligned, ldx and ldy multiples of 8");
  mx::GemmArgs p{codes, scales, w, w_scales, bias, R ? t : nullptr, static_cast<const uint16_t*>(l2t),
                 static_cast<uint16_t*>(y), (int)R, (int)ldy, (int)M, (int)N, mx::stages(K), 0, 0};
  const int64_t need = R ? mx::lowrank_workspace(M, K, R) : 0;
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return set_error(PQ_EINVAL, "pq_mx_linear: a workspace of %lld bytes, 16-byte aligned", (long long)need);
  const bool inside = mx::quantized_inside(M, K) && !q8;   // the product quantizes the rows itself
  if (R) {
    if (const int st = mx::lowrank(x, dtype, M, K, ldx, l1f, R, inside ? nullptr : codes, scales, q8, t, workspace, stream))
      return st;
  } else if (!inside) {
    if (const int st = pq_mx_quant(x, dtype, M, K, ldx, codes, scales, q8, stream)) return st;
  }
  if (inside)
    return mx::launch_split<1, 1, 8, 2, true>({p, static_cast<const uint16_t*>(x), ldx, (int)K}, dtype, (int)R, stream);
  return mx::launch_gemm(p, dtype, (int)R, stream);
}
