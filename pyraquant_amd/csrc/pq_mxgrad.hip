// Gradients of a layer over frozen microscaled 4-bit weights (pq_mx.h) with a low-rank branch:
//   y  = xh wh^T + t B + b,  t = x A
//   dt = dy B^T,  dB = t^T dy,  db = sum_m dy,  dA = xt^T dt,  dx = dy wh + dt A^T
// xt: the values of the 8-bit codes the forward pass kept of x. The rounding of x to 4 bits counts as the identity. All sums in
// fp32. t and dt are fp32, and operands of 16-bit matrix instructions in two parts (two_parts).
#include "pq_mx.h"

#include <algorithm>

namespace pq {
namespace mx {
namespace {

typedef __attribute__((address_space(3))) uint8_t lds_u8_t;

// ---- dx = dy wh + dt A^T ---------------------------------------------------------------------------------------------
struct DxArgs {
  const uint16_t* dy;
  const uint8_t *w, *ws;
  const float* dt;           // [M, R]
  const uint16_t* ap;        // [K, R]
  uint16_t* dx;
  int64_t lddy, lddx;
  int M, N, K, KT;
  int tiles_m, tiles_k;
  float* part;   // a split over n: [slices][M][K], `slice` n each
  int slice;
};

// dx += dt A^T for NI tiles of 32 columns k (from kk on) x 32 rows, lane % 32 of which is m
template <int DT, int R, int NI>
__device__ __forceinline__ void add_low_rank(const DxArgs& p, int kk, int m, int lane, v16f* const (&acc)[NI]) {
#pragma unroll
  for (int r0 = 0; r0 < R; r0 += 32) {
    const int r = r0 + 8 * (lane >> 5);
    RankPiece t[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) t[s].load(p.dt + (int64_t)min(m, p.M - 1) * R + r + 16 * s);
    rank_products<DT, NI, 2>(acc, t, [&](int i, int s) {
      return *reinterpret_cast<const v4i*>(p.ap + (int64_t)min(kk + 32 * i + (lane & 31), p.K - 1) * R + r + 16 * s);
    });
  }
}

// Few blocks: a workgroup of four waves takes 64 rows m x 128 columns k (one stage of the packed weight), 64 n a step. dy and
// the 4-bit weights of the next two steps are on their way into registers while the products of this one run, then go to the
// other of two LDS buffers, the weights widened to 16 bits on the way; they are read back by columns. One barrier a step.
// (Blocks of one row of blocks are neighbours in blockIdx.x: a grid's y ends at 65535.)
// SPLIT: blockIdx.y takes a slice of n and leaves its sums in fp32 in p.part [slices][M][K] for mx_dx_join_kernel.
// Bound by the steps' latency, one workgroup to a compute unit or less: 154 x 2048 x 640 9.5 us, 1000 x 1312 x 1040 14.
template <int DT, int R, bool SPLIT>
__global__ __launch_bounds__(256) void mx_dx_kernel(const DxArgs p) {
  constexpr int BM = 64, A = BM * 128, W = 64 * 256, LA = BM / 32, TJ = BM / 64;   // 16-byte loads of dy a thread; m tiles of a wave
  __shared__ __attribute__((aligned(16))) uint8_t smem[2 * (A + W)];      // [m][64 n] and [n][128 k], twice
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int kt = blockIdx.x % p.KT, k0 = kt * 128, m0 = blockIdx.x / p.KT * BM;
  const int wk = (wave & 1) * 64, wm = (wave >> 1) * (BM / 2);
  const int l32 = lane & 31, half = lane >> 5;
  const int first = SPLIT ? blockIdx.y * p.slice : 0, end = SPLIT ? min(p.N, first + p.slice) : p.N;
  const int arow = tid >> 3, achunk = tid & 7, wrow = tid >> 2, wb = tid & 3;
  const bool in_k = k0 + wb * 32 < p.K;
  struct Step {
    v4u dy[LA], c;
    int byte;
  } next[2];
  auto load = [&](Step& g, int n0) {
    const int n = n0 + achunk * 8;
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      const int m = m0 + arow + 32 * i;
      g.dy[i] = v4u{0, 0, 0, 0};
      if (m < p.M && n < end) g.dy[i] = *reinterpret_cast<const v4u*>(p.dy + (int64_t)m * p.lddy + n);
    }
    g.c = v4u{0, 0, 0, 0};
    g.byte = 0;
    if (in_k && n0 + wrow < end) {
      g.c = *reinterpret_cast<const v4u*>(p.w + code_offset(n0 + wrow, kt, wb, p.KT));
      g.byte = p.ws[scale_offset(n0 + wrow, kt, wb, p.KT)];
    }
  };
  auto store = [&](const Step& g, int buf) {
    uint8_t* const sa = smem + buf * (A + W);
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      const int row = arow + 32 * i;
      *reinterpret_cast<v4u*>(sa + row * 128 + ((achunk ^ (row & 7)) << 4)) = g.dy[i];
    }
    const float s = scale_value(g.byte);
    const uint32_t nan = g.byte == kNaN ? nan2<DT>() : 0;   // (such a block's codes are 0: or-ing makes every value NaN)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<v4u*>(sa + A + wrow * 256 + (((wb * 4 + i) ^ spread(wrow)) << 4)) = widen8<DT>(g.c[i], s) | nan;
  };
  v16f acc[2][TJ] = {};   // [k tile][m tile]
  load(next[0], first);
  load(next[1], first + 64);
  store(next[0], 0);
  auto step = [&](Step& coming, Step& after, int n0, int buf) {   // after: the step two ahead; coming: the next
    __syncthreads();
    load(after, n0 + 128);   // (past the end: loads nothing)
    const uint8_t* const sa = smem + buf * (A + W);
    auto w_at = [&](int row, int chunk) { return sa + A + row * 256 + ((chunk ^ spread(row)) << 4); };
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      v4i w[2], a[TJ];
#pragma unroll
      for (int i = 0; i < 2; ++i) w[i] = read_columns(w_at, 16 * s, wk + 32 * i, lane);
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        const int row = wm + 32 * j + l32;
        a[j] = *reinterpret_cast<const v4i*>(sa + row * 128 + (((2 * s + half) ^ (row & 7)) << 4));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = mfma16<DT>(w[i], a[j], acc[i][j]);
    }
    store(coming, buf ^ 1);
  };
  for (int n0 = first; n0 < end; n0 += 128) {
    step(next[1], next[0], n0, 0);
    if (n0 + 64 < end) step(next[0], next[1], n0 + 64, 1);
  }
#pragma unroll
  for (int j = 0; j < TJ; ++j) {
    const int m = m0 + wm + 32 * j + l32;
    if constexpr (!SPLIT) add_low_rank<DT, R, 2>(p, k0 + wk, m, lane, {&acc[0][j], &acc[1][j]});
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int kk = k0 + wk + 32 * i;
      if (SPLIT) {
        if (m < p.M && kk < p.K) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<v4f*>(p.part + ((int64_t)blockIdx.y * p.M + m) * p.K + kk + 8 * q + 4 * half) =
                v4f{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        }
        continue;
      }
      if (m < p.M && kk < p.K) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<v2u*>(p.dx + (int64_t)m * p.lddx + kk + 8 * q + 4 * half) =
              v2u{pack2<DT>(acc[i][j][4 * q], acc[i][j][4 * q + 1]), pack2<DT>(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3])};
      }
    }
  }
}

// dx from the slices' sums, added in order, and the low-rank term. A wave takes 32 rows x 32 columns. Bound by reading the sums:
// five slices of 2050 x 1280 (52 MB) and rank 64 in 17 us.
template <int DT, int R>
__global__ __launch_bounds__(256) void mx_dx_join_kernel(const DxArgs p, int slices) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l32 = lane & 31, half = lane >> 5;
  const int kk = blockIdx.x % p.KT * 128 + wave * 32, m = blockIdx.x / p.KT * 32 + l32;
  if (kk >= p.K) return;
  v16f acc = {};
  if (m < p.M) {
    for (int z = 0; z < slices; ++z) {
      const float* const src = p.part + ((int64_t)z * p.M + m) * p.K + kk + 4 * half;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const v4f v = *reinterpret_cast<const v4f*>(src + 8 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[4 * q + e] += v[e];
      }
    }
  }
  add_low_rank<DT, R, 1>(p, kk, m, lane, {&acc});
  if (m < p.M) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<v2u*>(p.dx + (int64_t)m * p.lddx + kk + 8 * q + 4 * half) =
          v2u{pack2<DT>(acc[4 * q], acc[4 * q + 1]), pack2<DT>(acc[4 * q + 2], acc[4 * q + 3])};
  }
}

// A workgroup of eight waves: 256 rows m x 256 columns k, each wave 64 x 128 of it (2 x 4 tiles). n advances in steps of 32.
//  * dy comes by LDS-DMA in stages of 64 n (whole 128-byte lines of a row) through a ring of three; 16-byte chunk c of a row
//    sits at c ^ (row % 8), so the fragments' ds_read_b128 meet no bank conflicts.
//  * The weight's codes and scales come by LDS-DMA as they are stored, through a ring of five steps; a step ahead of its
//    use each thread widens 16 of them to 16 bits into one of two [32 n][256 k] buffers, whose transposing reads give
//    fragments along n. So a weight is widened once per 256 rows, and memory and cache hold it in 4 bits.
//  * Two groups of four waves, one of each per SIMD, take turns: one issues a step's 16 products back to back while the other
//    reads its fragments, widens its part of the next step's weights and issues its DMA. Group B runs one slot behind.
// In its memory phase of step s a wave issues half of dy stage s / 2 + 2 and its part of codes s + 5. Slot 2 s reads dy step s
// and codes s + 2, all issued by phase s - 3; the barrier before it has every wave wait for all but its two younger phases.
// LDS, per step: fragments 8 waves x 12 KB, dy 16 KB in, weights 16 KB in: as many cycles as the products take (bf16 products
// of 32 x 32 x 16 at 32 cycles, 128 bytes of LDS a cycle), so the kernel is bound by both at once, and by the power limit:
// 16384 x 3072 x 12288 in 1000 us, 1.24 PFLOP/s (a library's product of the weight in bf16: 1.36-1.38); 4352 x 3072 x 3072, 204
// blocks on 256 compute units, in 79.5 us, 1.03. Moving the loads or the reads of codes between the products cost 10 %.
struct DxTile {
  // (64 bytes after each KB of codes: the 128 values that two of them hold of a row are read together)
  static constexpr int DY = 256 * 128, BLOCK = 1024 + 64, CODES = 4 * BLOCK + 1024, W = 32 * 512;
  static constexpr int AT_CODES = 3 * DY, AT_W = AT_CODES + 5 * CODES, LDS = AT_W + 2 * W + 3 * 1024;   // (and room for the three
  static constexpr int PITCH = 144;                                                                     // waves that bring nothing)
};

// SPLIT: a slice of n each, the sums left in fp32 in p.part for mx_dx_join_kernel.
template <int DT, int R, bool SPLIT>
__global__ __attribute__((amdgpu_flat_work_group_size(512, 512), amdgpu_waves_per_eu(2, 2)))
void mx_dx_ring_kernel(const DxArgs p) {
  using T = DxTile;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = wave & 1, wm = wave >> 1, l32 = lane & 31, half = lane >> 5;
  const int tiles = p.tiles_m * p.tiles_k, z = SPLIT ? (int)blockIdx.x / tiles : 0;
  int tm, tk;
  tile_of((int)blockIdx.x - z * tiles, tiles, p.tiles_m, p.tiles_k, 6, tm, tk);
  const int m0 = tm * 256, k0 = tk * 256, kt0 = tk * 2, KT = p.KT;
  const int first = SPLIT ? z * p.slice : 0, N = SPLIT ? min(p.slice, p.N - first) : p.N;   // n of this block (slices: of 64)
  const int rows = min(256, p.M - m0), NB = (N + 15) >> 4, steps = (N + 31) >> 5;

  // Loads outside their buffers give zeros: rows past M and n past N of dy, and n past N or k past K of the weight.
  const auto rs_dy = __builtin_amdgcn_make_buffer_rsrc((void*)(p.dy + (int64_t)m0 * p.lddy + first), (short)0,
                                                       (int)(((rows - 1) * p.lddy + N) * 2), kBufferWord3);
  const int lddy2 = (int)p.lddy * 2;
  const int dchunk = (lane & 7) ^ (lane >> 3);   // row % 8 == lane / 8
  const int vdy = (wave * 32 + (lane >> 3)) * lddy2 + dchunk * 16;
  // Codes: wave w < 4 brings row block w / 2, stage kt0 + w % 2 of a step; wave 4 the scales, 64 bytes for each of the four;
  // the others bring nothing (a step counts the same number of DMA instructions for every wave).
  const int unit = wave < 4 ? 1024 : wave == 4 ? 64 : 0, kb = wave < 4 ? wave & 1 : (lane >> 2) & 1;
  const int vc = kt0 + kb < KT && (wave < 4 || lane < 16)
      ? ((wave < 4 ? wave >> 1 : lane >> 3) * KT + kt0 + kb) * unit + (wave < 4 ? lane : lane & 3) * 16 : kOOB;
  // (the steps go out in order: a pointer, the row blocks left and the ring's slot move along)
  const int64_t cstep = (int64_t)2 * KT * unit;
  const uint8_t* cptr = (wave < 4 ? p.w : p.ws) + (first >> 5) * cstep;
  int cleft = NB, cslot = 0, crec = __builtin_amdgcn_readfirstlane(min(2, NB) * KT * unit);
  const int cdst = wave <= 4 ? T::AT_CODES + wave * T::BLOCK : T::LDS - 1024 * (8 - wave), cmove = wave <= 4 ? T::CODES : 0;
  auto dma_codes = [&]() {
    const uint64_t at = (uint64_t)cptr;   // (the same in every lane: kept in scalar registers)
    const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at) |
                          (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32;
    const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, crec, kBufferWord3);
    uint8_t* const dst = smem + cdst + cslot * cmove;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)dst, 16, vc, 0, 0, 0);
  };
  auto next_codes = [&]() {
    cptr += cstep;
    cleft -= 2;
    cslot = cslot == 4 ? 0 : cslot + 1;
    crec = __builtin_amdgcn_readfirstlane(max(0, min(2, cleft)) * KT * unit);
  };
  // Phase u's part: dy half u % 2 of stage u / 2 + 2, codes u + 5. What it and the reads below need per phase (LDS addresses,
  // offsets) is worked out between the products of the phase before: every instruction of a memory phase counts.
  int dslot = 0, dhalf = 0, dn = dchunk * 8, dat = vdy, doff[2];   // slot and half of the DMA; its n, and offset in the buffer
  auto offsets = [&]() {
    const int inside = (dn - N) >> 31;   // (all ones where n < N: no branch)
    doff[0] = (dat & inside) | (kOOB & ~inside);
    doff[1] = ((dat + 8 * lddy2) & inside) | (kOOB & ~inside);
  };
  auto dma = [&]() {
    uint8_t* const sb = smem + dslot * T::DY + wave * 4096 + dhalf * 2048;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_dy, (lds_void_t*)sb, 16, doff[0], 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_dy, (lds_void_t*)(sb + 1024), 16, doff[1], 0, 0, 0);
    dma_codes();
  };
  auto next_dma = [&]() {
    dat += dhalf ? 128 - 16 * lddy2 : 16 * lddy2;
    dn += dhalf ? 64 : 0;
    dslot = dhalf == 0 ? dslot : dslot == 2 ? 0 : dslot + 1;
    dhalf ^= 1;
    offsets();
    next_codes();
  };
  // 16 values of a step: row n = tid / 16 of 32, columns 16 (tid % 16) .. Read in one phase, widened in the next: neither waits
  // for the other. (Lanes 4-7 of 8 store their second half first: eight lanes' 16-byte stores meet no bank twice.)
  const int wr = tid >> 4, wc = tid & 15, wblk = (wr >> 4) * 2 + (wc >> 3), wb4 = (wc & 7) >> 1, turn = (wc >> 2) & 1;
  v2u wq;
  int wbyte;
  v4u wide[2];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8_t*)smem;
  uint32_t code_at = lds0 + T::AT_CODES + wblk * T::BLOCK + (wr & 15) * 64 + ((wb4 ^ k64_swz(wr & 15)) << 4) + (wc & 1) * 8;
  uint32_t scale_at = lds0 + T::AT_CODES + 4 * T::BLOCK + wblk * 64 + (wr & 15) * 4 + scale_slot(wb4);
  int rslot = 0;   // (read in order too)
  auto rd_codes = [&]() {
    wq = *(const __attribute__((address_space(3))) v2u*)(uintptr_t)code_at;
    wbyte = *(const lds_u8_t*)(uintptr_t)scale_at;
  };
  auto next_rd_codes = [&]() {
    const int move = rslot == 4 ? -4 * T::CODES : T::CODES;
    code_at += move;
    scale_at += move;
    rslot = rslot == 4 ? 0 : rslot + 1;
  };
  auto widen = [&]() {
    const float s = scale_value(wbyte);
    const uint32_t nan = wbyte == kNaN ? nan2<DT>() : 0;   // (such a block's codes are 0: or-ing makes every value NaN)
    wide[0] = widen8<DT>(turn ? wq[1] : wq[0], s) | nan;
    wide[1] = widen8<DT>(turn ? wq[0] : wq[1], s) | nan;
  };
  uint32_t put_at[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) put_at[i] = lds0 + T::AT_W + wr * 512 + (((2 * wc + (turn ^ i)) ^ spread(wr)) << 4);
  auto put = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) *(__attribute__((address_space(3))) v4u*)(uintptr_t)put_at[i] = wide[i];
  };
  // Fragments of the weight (read_columns, in one block of assembly that ends with its own wait: the compiler would wait for
  // every DMA in flight before the builtin's reads). Four tiles of 32 columns, rows 0-15 and 16-31 of the step.
  v4i a[2][2];
  uint32_t wat[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 8 * half + ((lane & 15) >> 2), col = wk * 128 + 32 * i + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    wat[i] = lds0 + T::AT_W + row * 512 + (((col >> 3) ^ spread(row)) << 4) + (col & 4) * 2;
  }
  uint32_t dy_at[2];   // (a half stage on: the same chunks with bit 2 of their number, bit 6 of the address, turned)
#pragma unroll
  for (int h = 0; h < 2; ++h) dy_at[h] = lds0 + (wm * 64 + l32) * 128 + (((2 * h + half) ^ (l32 & 7)) << 4);
  int yslot = 0;
  auto rd_dy = [&]() {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j) a[h][j] = *(const __attribute__((address_space(3))) v4i*)(uintptr_t)(dy_at[h] + j * 4096);
  };
  v16f acc[4][2] = {};
  const bool grp_b = wave >= 4;
  offsets();
  dma_codes();
  next_codes();
#pragma unroll
  for (int u = -4; u < 0; ++u) {
    dma();
    next_dma();
  }
  wait_vmcnt<6>();
  ring_barrier();
  rd_codes();
  next_rd_codes();
  widen();
  put();
  rd_codes();
  next_rd_codes();
  widen();
#pragma unroll
  for (int i = 0; i < 2; ++i) put_at[i] += T::W;
  ring_barrier();
  if (grp_b) ring_barrier();
  for (int s = 0; s < steps; ++s) {
    put();        // step s + 1
    rd_codes();   // of step s + 2
    rd_dy();
    dma();
    v4i w0, w1, w2, w3, w4, w5, w6, w7;
    asm volatile(
        "ds_read_b64_tr_b16 v[220:221], %[p0]\n\tds_read_b64_tr_b16 v[222:223], %[p0] offset:2048\n\t"
        "ds_read_b64_tr_b16 v[224:225], %[p1]\n\tds_read_b64_tr_b16 v[226:227], %[p1] offset:2048\n\t"
        "ds_read_b64_tr_b16 v[228:229], %[p2]\n\tds_read_b64_tr_b16 v[230:231], %[p2] offset:2048\n\t"
        "ds_read_b64_tr_b16 v[232:233], %[p3]\n\tds_read_b64_tr_b16 v[234:235], %[p3] offset:2048\n\t"
        "ds_read_b64_tr_b16 v[236:237], %[p0] offset:8192\n\tds_read_b64_tr_b16 v[238:239], %[p0] offset:10240\n\t"
        "ds_read_b64_tr_b16 v[240:241], %[p1] offset:8192\n\tds_read_b64_tr_b16 v[242:243], %[p1] offset:10240\n\t"
        "ds_read_b64_tr_b16 v[244:245], %[p2] offset:8192\n\tds_read_b64_tr_b16 v[246:247], %[p2] offset:10240\n\t"
        "ds_read_b64_tr_b16 v[248:249], %[p3] offset:8192\n\tds_read_b64_tr_b16 v[250:251], %[p3] offset:10240\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&{v[220:223]}"(w0), "=&{v[224:227]}"(w1), "=&{v[228:231]}"(w2), "=&{v[232:235]}"(w3), "=&{v[236:239]}"(w4),
          "=&{v[240:243]}"(w5), "=&{v[244:247]}"(w6), "=&{v[248:251]}"(w7)
        : [p0] "v"(wat[0]), [p1] "v"(wat[1]), [p2] "v"(wat[2]), [p3] "v"(wat[3])
        : "memory");
    if (grp_b) wait_vmcnt<6>();
    ring_barrier();
    const v4i w[2][4] = {{w0, w1, w2, w3}, {w4, w5, w6, w7}};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma16<DT>(w[h][i], a[h][j], acc[i][j]);
    // Between the products: the next step's weights widened, and the next phase's addresses.
    widen();
    const int up = s & 1 ? -T::W : T::W, along = !(s & 1) ? 0 : yslot == 2 ? -2 * T::DY : T::DY;
    yslot = !(s & 1) ? yslot : yslot == 2 ? 0 : yslot + 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) wat[i] += up;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      put_at[i] -= up;
      dy_at[i] = (dy_at[i] ^ 64) + along;
    }
    next_rd_codes();
    next_dma();
    asm volatile("" : "+v"(wide[0]), "+v"(wide[1]), "+v"(wat[0]), "+v"(wat[1]), "+v"(wat[2]), "+v"(wat[3]), "+v"(put_at[0]),
                 "+v"(put_at[1]), "+v"(dy_at[0]), "+v"(dy_at[1]), "+v"(code_at), "+v"(scale_at), "+v"(doff[0]), "+v"(doff[1]));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
    }
    if (!grp_b) wait_vmcnt<6>();
    ring_barrier();
  }
  if (!grp_b) ring_barrier();
  wait_vmcnt<0>();
  __syncthreads();   // the rings become the output staging

  const int kb0 = k0 + wk * 128, mb = m0 + wm * 64;
  if constexpr (SPLIT) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int m = mb + 32 * j + l32, kk = kb0 + 32 * i;
        if (m >= p.M || kk >= p.K) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<v4f*>(p.part + ((int64_t)z * p.M + m) * p.K + kk + 8 * q + 4 * half) =
              v4f{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
      }
    return;
  }
  uint8_t* const stage = smem + wave * 32 * T::PITCH;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    add_low_rank<DT, R, 4>(p, kb0, mb + 32 * j + l32, lane, {&acc[0][j], &acc[1][j], &acc[2][j], &acc[3][j]});
#pragma unroll
    for (int ih = 0; ih < 2; ++ih) {
#pragma unroll
      for (int ii = 0; ii < 2; ++ii) {
        const int i = 2 * ih + ii;
        const v16f& y = acc[i][j];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<v2u*>(stage + l32 * T::PITCH + (ii * 32 + 8 * q + 4 * half) * 2) =
              v2u{pack2<DT>(y[4 * q], y[4 * q + 1]), pack2<DT>(y[4 * q + 2], y[4 * q + 3])};
      }
      wave_sync();
      const int k = kb0 + ih * 64 + (lane & 7) * 8, row = lane >> 3;
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += 8) {
        const int m = mb + 32 * j + r0 + row;
        const v4u v = *reinterpret_cast<const v4u*>(stage + (r0 + row) * T::PITCH + (lane & 7) * 16);
        if (m < p.M && k < p.K) *reinterpret_cast<v4u*>(p.dx + (int64_t)m * p.lddx + k) = v;
      }
      wave_sync();
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// ---- sums over rows: part[s][r][c] = sum over the rows of slice s of v[m, r] z[m, c] -------------------------------------
// z is dy (EIGHT false) or the 8-bit codes of x with their scales; v is t or dt, [M, R] in fp32. Column sums of z too
// (COLS), and these alone where v is NULL. A workgroup of four waves takes 128 columns and a slice of the rows, 64 rows a step, the
// next step's rows on their way into registers meanwhile; the order of the sums is fixed. Bound by reading z: 460 MB of 16384 x 3072 x
// 12288 in 98 us, 4.7 TB/s. In fp16 a rank's 64 values of a step are taken on a scale of their own, so that small ones keep their bits: both launches
// 133 us instead of 125 at these sizes with rank 32, 21.8 instead of 19.8 at 4352 x 3072 x 3072, nothing with rank 64.
struct SumArgs {
  const void* z;
  const uint8_t* scales;
  const float* v;
  float *part, *part_cols;
  int64_t ldz;
  int M, C, KT, rows;   // rows a slice, a multiple of 64
  int panels, blocks;   // of 128 columns; workgroups (0: this sum is not wanted)
};

template <int DT, int R, bool EIGHT, bool COLS>
__device__ __forceinline__ void row_sums(const SumArgs& p, int block, uint8_t* sz, uint8_t* sv, uint32_t* top, float* back) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slice = block / p.panels, panel = block - slice * p.panels;
  const int c0 = panel * 128, s0 = slice * p.rows;
  const int end = min(p.M, s0 + p.rows);
  auto z_at = [&](int row, int chunk) { return sz + row * 256 + ((chunk ^ spread(row)) << 4); };
  auto hi_at = [&](int row, int chunk) { return sv + row * R * 2 + (chunk << 4); };
  auto lo_at = [&](int row, int chunk) { return sv + (64 + row) * R * 2 + (chunk << 4); };
  const uint32_t one2 = DT == PQ_BF16 ? 0x3f803f80u : 0x3c003c00u;
  const v4i ones = {(int)one2, (int)one2, (int)one2, (int)one2};
  v16f acc[R / 32] = {}, cols = {};
  v4u zr[EIGHT ? 2 : 4];
  v4f vr[R / 16];
  int byte = 0;
  auto load = [&](int m0) {
    if constexpr (EIGHT) {
      const int m = m0 + (tid >> 2), b = tid & 3, c = c0 + b * 32;
      zr[0] = zr[1] = v4u{0, 0, 0, 0};
      byte = 0;
      if (m < end && c < p.C) {
        const v4u* const src = reinterpret_cast<const v4u*>(static_cast<const int8_t*>(p.z) + (int64_t)m * p.ldz + c);
        zr[0] = src[0];
        zr[1] = src[1];
        byte = p.scales[scale_offset(m, panel, b, p.KT)];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = m0 + i * 16 + (tid >> 4), c = c0 + (tid & 15) * 8;
        zr[i] = v4u{0, 0, 0, 0};
        if (m < end && c < p.C) zr[i] = *reinterpret_cast<const v4u*>(static_cast<const uint16_t*>(p.z) + (int64_t)m * p.ldz + c);
      }
    }
#pragma unroll
    for (int i = 0; i < R / 16; ++i) {
      const int at = i * 256 + tid, m = m0 + at / (R / 4);
      vr[i] = v4f{};
      if (p.v && m < end) vr[i] = *reinterpret_cast<const v4f*>(p.v + (int64_t)m * R + at % (R / 4) * 4);
    }
  };
  load(s0);
  for (int m0 = s0; m0 < end; m0 += 64) {
    if constexpr (DT == PQ_F16) tell_largest<R>(vr, top, tid);
    __syncthreads();
    if constexpr (EIGHT) {
      const int row = tid >> 2, b = tid & 3;
      const float s = restore_scale(byte);   // (past the end the codes are zeros)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v2u lo = restore4<DT>(zr[i >> 1][2 * (i & 1)], s), hi = restore4<DT>(zr[i >> 1][2 * (i & 1) + 1], s);
        *reinterpret_cast<v4u*>(z_at(row, b * 4 + i)) = v4u{lo[0], lo[1], hi[0], hi[1]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<v4u*>(z_at(i * 16 + (tid >> 4), tid & 15)) = zr[i];
    }
    if constexpr (DT == PQ_F16) scale_values<R>(vr, top, back, tid);
#pragma unroll
    for (int i = 0; i < R / 16; ++i) {   // 64 rows of the first part, then of the second
      v2u hi, lo;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t h, l;
        two_parts<DT>(vr[i][2 * e], vr[i][2 * e + 1], h, l);
        hi[e] = h;
        lo[e] = l;
      }
      *reinterpret_cast<v2u*>(sv + (i * 256 + tid) * 8) = hi;
      *reinterpret_cast<v2u*>(sv + 64 * R * 2 + (i * 256 + tid) * 8) = lo;
    }
    __syncthreads();
    if (m0 + 64 < end) load(m0 + 64);   // in flight while this step's products run
    if constexpr (DT == PQ_F16) {
      v4i z[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        z[s] = read_columns(z_at, 16 * s, wave * 32, lane);
        if constexpr (COLS) cols = mfma16<DT>(z[s], ones, cols);
      }
      if (p.v) {
#pragma unroll
        for (int j = 0; j < R / 32; ++j) {
          v16f sum = {};   // of a step by themselves, then on no scale
          const float by = back[32 * j + (lane & 31)];
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            sum = mfma16<DT>(z[s], read_columns(hi_at, 16 * s, 32 * j, lane), sum);
            sum = mfma16<DT>(z[s], read_columns(lo_at, 16 * s, 32 * j, lane), sum);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[j][e] = fmaf(sum[e], by, acc[j][e]);
        }
      }
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const v4i z = read_columns(z_at, 16 * s, wave * 32, lane);
        if (p.v) {
#pragma unroll
          for (int j = 0; j < R / 32; ++j) {
            acc[j] = mfma16<DT>(z, read_columns(hi_at, 16 * s, 32 * j, lane), acc[j]);
            acc[j] = mfma16<DT>(z, read_columns(lo_at, 16 * s, 32 * j, lane), acc[j]);
          }
        }
        if constexpr (COLS) cols = mfma16<DT>(z, ones, cols);
      }
    }
  }
  // lane: r = 32 j + lane % 32, columns c0 + 32 wave + 8 q + 4 (lane / 32) + e
  const int c = c0 + wave * 32 + 4 * (lane >> 5);
  if (c0 + wave * 32 >= p.C) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (c + 8 * q >= p.C) break;
    if (p.v) {
#pragma unroll
      for (int j = 0; j < R / 32; ++j)
        *reinterpret_cast<v4f*>(p.part + ((int64_t)slice * R + 32 * j + (lane & 31)) * p.C + c + 8 * q) =
            v4f{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
    }
    if (COLS && (lane & 31) == 0)
      *reinterpret_cast<v4f*>(p.part_cols + (int64_t)slice * p.C + c + 8 * q) =
          v4f{cols[4 * q], cols[4 * q + 1], cols[4 * q + 2], cols[4 * q + 3]};
  }
}

// Both sums in one launch: dB and the column sums of dy (b), then dA (a).
template <int DT, int R, bool COLS>
__global__ __launch_bounds__(256) void mx_rowsum_kernel(const SumArgs b, const SumArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t sz[64 * 256];      // [m][128 c]
  __shared__ __attribute__((aligned(16))) uint8_t sv[2 * 64 * R * 2];   // [2][m][R]
  __shared__ __attribute__((aligned(16))) uint32_t top[DT == PQ_F16 ? 2 * R : 4];
  __shared__ __attribute__((aligned(16))) float back[DT == PQ_F16 ? R : 4];
  if ((int)blockIdx.x < b.blocks) row_sums<DT, R, false, COLS>(b, blockIdx.x, sz, sv, top, back);
  else row_sums<DT, R, true, false>(a, blockIdx.x - b.blocks, sz, sv, top, back);
}

// The slices' sums added in order, rounded to 16 bits: dB [R, N] and dA [K, R]; and the column sums in 32. A thread sums one
// element, eight slices' loads in flight.
__device__ __forceinline__ float sum_slices(const float* at, int slices, int64_t step) {
  float s = 0.0f;
  int i = 0;
  for (; i + 8 <= slices; i += 8) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = at[(i + e) * step];
#pragma unroll
    for (int e = 0; e < 8; ++e) s += v[e];
  }
  for (; i < slices; ++i) s += at[i * step];
  return s;
}
struct JoinArgs {
  const float *part, *part_cols;
  uint16_t* out;
  float* cols;
  int slices, C, groups, blocks;   // groups of 64 columns; workgroups (0: not wanted)
};
template <int DT>
__global__ __launch_bounds__(256) void mx_join_kernel(const JoinArgs b, const JoinArgs a, int P, int R) {
  const bool is_b = (int)blockIdx.x < b.blocks;
  const JoinArgs p = is_b ? b : a;
  const int block = (int)blockIdx.x - (is_b ? 0 : b.blocks);
  const int c = block % p.groups * 64 + (threadIdx.x & 63), r = block / p.groups * 4 + (threadIdx.x >> 6);
  if (c >= p.C) return;
  if (p.out && r < R)
    p.out[is_b ? (int64_t)r * p.C + c : (int64_t)c * R + r] =
        (uint16_t)f32_to_16_bits<DT>(sum_slices(p.part + (int64_t)r * p.C + c, p.slices, (int64_t)P * p.C));
  if (p.cols && r == 0) p.cols[c] = sum_slices(p.part_cols + c, p.slices, p.C);
}

// How dx is computed: in blocks of 256 x 256 (m x k) or 64 x 128, with n cut into `slices` where that ends sooner, by an
// estimate in us for the card's 256 compute units (the workspace's size comes from the same plan, and knows no device). A 256 x 256
// block, one to a compute unit: 9 for its start and end, and for 64 n 1.25 alone to 1.7 with all 256 at work (the clock falls with
// the power they draw). A 64 x 128 block: 0.62 for 64 n, more where a compute unit holds more than one, 1 for the end of each past
// the third, and 4 for the launch. Slices: 4 for another launch; 1.2 for 10^6 values of their sums (fp32, written and read again).
// Measured (bf16, rank 32, * the plan's):
//   M x K x N            256 x 256, slices: 1  2      4      5      8   64 x 128: 1      2      4      8
//   16384 x 3072 x 12288      999*  1160   1259   1344   1580      1730   1936   2052   2322
//   4352 x 3072 x 3072       79.7*   124    169    184    275       132    161    193    308
//   2050 x 5120 x 1280       38.5*  78.4   98.7    117              51.7   80.2    101
//   2050 x 1280 x 5120        113   74.8   55.3   53.0*  73.5      69.6   62.0   67.8   77.8
//   1024 x 3072 x 12288       255    147   95.7   89.8*   114       153    127    133    143
//   1024 x 3072 x 3072       72.0   54.7   45.4   46.3   65.0      43.0*  44.4   50.6   63.9
//   512 x 3072 x 12288        255    142   84.2   73.9   60.2*      127   91.6   70.8   78.7
//   512 x 12288 x 3072       72.6   63.1*  82.3   83.3    107      62.4   79.8   93.5    118
//   5150 x 9248 x 416        74.2*   268    422                    95.9    273    433
//   11734 x 608 x 1680       46.0*  73.6   87.4   93.1             54.9   74.3   89.3
//   13664 x 1344 x 4704       220*   246    303    331    422       290    343    398    511
//   3000 x 2048 x 2048       52.0   52.4   70.9   74.0   97.0      45.6*  63.2   76.5   99.2
//   1000 x 1312 x 1040       30.3   33.8   31.5   30.7             13.9*  20.9   22.5
//   154 x 2048 x 640         21.0   19.3   18.8   18.5              9.5*  10.1   10.1
//   64 x 3072 x 3072         68.3   40.4   27.0   25.3   22.6      30.8   21.8   15.5   14.0*
struct DxPlan {
  bool ring;
  int slices, slice;
};
DxPlan dx_plan(int64_t M, int64_t N, int64_t K) {
  const int64_t large = ((M + 255) / 256) * ((K + 255) / 256), small = ((M + 63) / 64) * stages(K);
  const int steps = (int)((N + 63) / 64);
  auto rounds = [](int64_t blocks, int per) {   // of 256 blocks, and of those left
    auto round = [&](double fill) { return per * (1.25 + 0.45 * fill * fill * fill) + 9; };
    return (double)(blocks / 256) * round(1.0) + (blocks % 256 ? round((double)(blocks % 256) / 256) : 0.0);
  };
  DxPlan best{true, 1, 0};
  double least = 0;
  for (int ring = 1; ring >= 0; --ring)
    for (int s = 1; s <= 8 && s <= steps; ++s) {
      const int per = (steps + s - 1) / s;
      if ((s - 1) * per >= steps) continue;   // (no empty slice)
      const double each = (double)(small * s) / 256;   // 64 x 128 blocks a compute unit
      double t = ring ? rounds(large * s, per) : per * 0.62 * std::max(1.0, 0.45 + 0.58 * each) + 4 + std::max(0.0, each - 3);
      if (s > 1) t += 4 + s * (double)(M * K) * 1.2e-6;
      if ((ring && s == 1) || t < least) least = t, best = {ring == 1, s, s > 1 ? per * 64 : 0};
    }
  return best;
}

int launch_dx(DxArgs p, int dtype, int r, hipStream_t stream) {
#define PQ_MXD()                                                                                           \
  do {                                                                                                     \
    if (dtype == PQ_BF16) {                                                                                \
      if (r == 0) PQ_MXK(PQ_BF16, 0); else if (r == 32) PQ_MXK(PQ_BF16, 32); else PQ_MXK(PQ_BF16, 64);     \
    } else {                                                                                               \
      if (r == 0) PQ_MXK(PQ_F16, 0); else if (r == 32) PQ_MXK(PQ_F16, 32); else PQ_MXK(PQ_F16, 64);        \
    }                                                                                                      \
  } while (0)
  const DxPlan plan = dx_plan(p.M, p.N, p.K);
  p.slice = plan.slice;
  p.tiles_m = (p.M + 255) / 256;
  p.tiles_k = (p.K + 255) / 256;
  const int64_t blocks = plan.ring ? (int64_t)p.tiles_m * p.tiles_k * plan.slices : (int64_t)p.KT * ((p.M + 63) / 64);
  const int64_t join_blocks = plan.slices > 1 ? (int64_t)p.KT * ((p.M + 31) / 32) : 0;
  if (const int st = check_grid(blocks, plan.ring ? 512 : 256, "mx_grad_input")) return st;
  if (const int st = check_grid(join_blocks, 256, "mx_grad_input")) return st;
  const dim3 ring((unsigned)blocks), grid((unsigned)blocks, (unsigned)plan.slices);
  if (plan.slices == 1) {
    if (plan.ring) {
#define PQ_MXK(D, RR) hipLaunchKernelGGL((mx_dx_ring_kernel<D, RR, false>), ring, dim3(512), 0, stream, p)
      PQ_MXD();
#undef PQ_MXK
    } else {
#define PQ_MXK(D, RR) hipLaunchKernelGGL((mx_dx_kernel<D, RR, false>), grid, dim3(256), 0, stream, p)
      PQ_MXD();
#undef PQ_MXK
    }
    return check_launch("mx_grad_input");
  }
  const bool bf16 = dtype == PQ_BF16;
  if (plan.ring) {
    if (bf16) hipLaunchKernelGGL((mx_dx_ring_kernel<PQ_BF16, 0, true>), ring, dim3(512), 0, stream, p);
    else hipLaunchKernelGGL((mx_dx_ring_kernel<PQ_F16, 0, true>), ring, dim3(512), 0, stream, p);
  } else {
    if (bf16) hipLaunchKernelGGL((mx_dx_kernel<PQ_BF16, 0, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((mx_dx_kernel<PQ_F16, 0, true>), grid, dim3(256), 0, stream, p);
  }
  const dim3 join((unsigned)join_blocks);
#define PQ_MXK(D, RR) hipLaunchKernelGGL((mx_dx_join_kernel<D, RR>), join, dim3(256), 0, stream, p, plan.slices)
  PQ_MXD();
#undef PQ_MXK
#undef PQ_MXD
  return check_launch("mx_grad_input");
}

// Row slices of mx_rowsum_kernel: about 384 workgroups a sum. More only add sums to write and join; fewer read too little at once.
// us of both launches, for 256 / 384 / 512 / 1024 workgroups (bf16): 2050 x 1280 x 5120 rank 64 21.8 / 21.9 / 20.5 / 24.5,
// 4352 x 3072 x 3072 rank 32 17.5 / 19.7 / 19.1 / 24.3, 8192 x 3072 x 3072 rank 64 42.1 / 39.1 / 43.6 / 52.9, 16384 x 3072 x 12288
// rank 32 123 / 104 / 111 / 106.
int row_slices(int64_t M, int64_t C) {
  const int64_t panels = (C + 127) / 128, steps = (M + 63) / 64;
  const int64_t want = std::min<int64_t>({(384 + panels - 1) / panels, steps, 256});
  const int64_t each = (steps + want - 1) / want;
  return (int)((steps + each - 1) / each);   // (no empty slice)
}

}  // namespace
}  // namespace mx
}  // namespace pq

using namespace pq;

extern "C" int64_t pq_mx_grad_input_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 16 || K < 32 || M > (1 << 30) || N > (1 << 21) || K > (1 << 22)) return 0;
  const mx::DxPlan plan = mx::dx_plan(M, N, K);
  return plan.slices > 1 ? 4 * plan.slices * M * K : 0;
}

extern "C" int pq_mx_grad_input(const void* dy, int32_t dtype, int64_t lddy, const uint8_t* w, const uint8_t* w_scales,
                                const float* dt, const void* ap, int64_t R, void* dx, int64_t lddx, int64_t M, int64_t N,
                                int64_t K, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (M < 0 || N < 16 || N % 16 || K < 32 || K % 32 || lddy < N || lddx < K || M > (1 << 30) ||
      lddy > (1 << 21) || K > (1 << 22))
    return set_error(PQ_ESHAPE, "pq_mx_grad_input: M=%lld N=%lld K=%lld lddy=%lld (N %% 16 == 0, K %% 32 == 0, lddy <= 2^21)",
                     (long long)M, (long long)N, (long long)K, (long long)lddy);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_mx_grad_input: dtype %d", dtype);
  if (dt && R != 32 && R != 64) return set_error(PQ_ESHAPE, "pq_mx_grad_input: rank %lld (32 or 64)", (long long)R);
  if (M == 0) return PQ_OK;
  if (!dy || !w || !w_scales || !dx || (dt && !ap)) return set_error(PQ_EINVAL, "pq_mx_grad_input: null pointer");
  if ((uintptr_t)dy % 16 || lddy % 8 || (uintptr_t)w % 16 || (uintptr_t)w_scales % 16 || (uintptr_t)dx % 16 || lddx % 8 ||
      (uintptr_t)dt % 16 || (uintptr_t)ap % 16)
    return set_error(PQ_EALIGN, "pq_mx_grad_input: operands 16-byte aligned, lddy and lddx multiples of 8");
  mx::DxArgs p{static_cast<const uint16_t*>(dy), w, w_scales, dt, static_cast<const uint16_t*>(ap),
               static_cast<uint16_t*>(dx), lddy, lddx, (int)M, (int)N, (int)K, mx::stages(K), 0, 0, static_cast<float*>(workspace), 0};
  const int64_t need = pq_mx_grad_input_workspace_size(M, N, K);
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return set_error(PQ_EINVAL, "pq_mx_grad_input: a workspace of %lld bytes, 16-byte aligned", (long long)need);
  return mx::launch_dx(p, dtype, dt ? (int)R : 0, stream);
}

extern "C" int64_t pq_mx_grad_factors_workspace_size(int64_t M, int64_t K, int64_t N, int64_t P) {
  if (M < 1 || K < 32 || N < 16 || (P != 32 && P != 64)) return 0;
  return 4 * ((int64_t)mx::row_slices(M, N) * (P + 1) * N + (int64_t)mx::row_slices(M, K) * P * K);
}

extern "C" int pq_mx_grad_factors(const void* dy, int32_t dtype, int64_t lddy, const float* t, const float* dt, const int8_t* q8,
                                  const uint8_t* x_scales, int64_t M, int64_t K, int64_t N, int64_t R, int64_t P, void* dA,
                                  void* dB, float* dbias, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (M < 1 || N < 16 || N % 16 || K < 32 || K % 32 || lddy < N || R < 1 || R > P || (P != 32 && P != 64) ||
      M > (1 << 30) || N > (1 << 30) || K > (1 << 22))
    return set_error(PQ_ESHAPE, "pq_mx_grad_factors: M=%lld N=%lld K=%lld R=%lld P=%lld", (long long)M, (long long)N,
                     (long long)K, (long long)R, (long long)P);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_mx_grad_factors: dtype %d", dtype);
  if (((dB || dbias) && !dy) || (dB && !t) || (dA && (!dt || !q8 || !x_scales)) || !workspace)
    return set_error(PQ_EINVAL, "pq_mx_grad_factors: null pointer");
  if ((uintptr_t)dy % 16 || lddy % 8 || (uintptr_t)t % 16 || (uintptr_t)dt % 16 || (uintptr_t)q8 % 16 || (uintptr_t)workspace % 16)
    return set_error(PQ_EALIGN, "pq_mx_grad_factors: operands 16-byte aligned, lddy a multiple of 8");
  if (workspace_bytes < pq_mx_grad_factors_workspace_size(M, K, N, P))
    return set_error(PQ_ESHAPE, "pq_mx_grad_factors: workspace of %lld bytes", (long long)workspace_bytes);
  float* const part = static_cast<float*>(workspace);
  const int sb = mx::row_slices(M, N), sk = mx::row_slices(M, K);
  auto rows = [&](int slices) { return (int)(((M + 63) / 64 + slices - 1) / slices * 64); };
  float* const part_a = part + (int64_t)sb * (P + 1) * N;
  const int pb = (int)((N + 127) / 128), pk = (int)((K + 127) / 128);
  const bool want_b = dB || dbias, want_a = dA != nullptr;
  const mx::SumArgs b{dy, nullptr, dB ? t : nullptr, part, part + (int64_t)sb * P * N, lddy, (int)M, (int)N, 0,
                      rows(sb), pb, want_b ? pb * sb : 0};
  const mx::SumArgs a{q8, x_scales, dt, part_a, nullptr, K, (int)M, (int)K, mx::stages(K), rows(sk),
                      pk, want_a ? pk * sk : 0};
  const int quads = (int)((R + 3) / 4), gb = (int)((N + 63) / 64), ga = (int)((K + 63) / 64);
  const mx::JoinArgs jb{part, b.part_cols, static_cast<uint16_t*>(dB), dbias, sb, (int)N, gb, !want_b ? 0 : gb * (dB ? quads : 1)};
  const mx::JoinArgs ja{part_a, nullptr, static_cast<uint16_t*>(dA), nullptr, sk, (int)K, ga, want_a ? ga * quads : 0};
  if (!want_a && !want_b) return PQ_OK;
  const dim3 grid((unsigned)(b.blocks + a.blocks)), join((unsigned)(jb.blocks + ja.blocks)), block(256);
#define PQ_MXS(D, PP)                                                                                       \
  do {                                                                                                     \
    if (dbias) hipLaunchKernelGGL((mx::mx_rowsum_kernel<D, PP, true>), grid, block, 0, stream, b, a);      \
    else hipLaunchKernelGGL((mx::mx_rowsum_kernel<D, PP, false>), grid, block, 0, stream, b, a);           \
    hipLaunchKernelGGL((mx::mx_join_kernel<D>), join, block, 0, stream, jb, ja, (int)P, (int)R);           \
  } while (0)
  if (dtype == PQ_BF16) {
    if (P == 32) PQ_MXS(PQ_BF16, 32); else PQ_MXS(PQ_BF16, 64);
  } else {
    if (P == 32) PQ_MXS(PQ_F16, 32); else PQ_MXS(PQ_F16, 64);
  }
#undef PQ_MXS
  return check_launch("mx_grad_factors");
}
