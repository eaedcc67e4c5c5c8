// Low-rank adapters of many requests beside one shared projection (gfx950): with id = ids[m / each] the adapter of row m (none
// unless 0 <= id < slots), s its scale, A [K, R] and B [R, N] its factors,
//   y[m] = base[m] + t[m] B,  t[m] = s x[m] A
//   dt[m] = s dy[m] B^T,  dx[m] = dt[m] A^T,  dA = sum over its rows of x^T dt,  dB = sum over its rows of t^T dy
// Rows without an adapter keep base's bits (dx: zeros), and no row's result depends on another's values or adapter: the
// adapters of a tile of 64 rows are taken one after the other, each with its own rows packed together (`passes`), so a NaN in one
// request or adapter stays there.
//
//   down  part[s][m][r] = sum over slice s of k of x[m, k] f[id][k, r]          (t and dt without the scale; slices are added where
//                                                                                    they are read)
//   up    out[m, c] = base[m, c] + scale[id] sum_r part[m, r] g[id][c, r], and scale[id] part[m], the slices added, for `sums`
//   sums  the two sums over rows, per adapter, over chunks of the rows, added by `join` in their order
// All sums are fp32. t and dt are taken by the 16-bit matrix instructions in two parts (two_parts), in fp16 on a scale of each row's (`up`) or of each
// rank's in 64 rows (`sums`), so that their rounding shows in no result, however small they are (the scales of `sums` cost a step of tuning 16384 x
// 1280 x 5120 with rank 32 205 -> 206 us). No atomics: the same bits every time. Bound by memory: 2 R operations for each value that is read.
#include "pq_mx.h"

#include <algorithm>
#include <type_traits>

namespace pq {
namespace adapt {
namespace {

using namespace mx;

struct Ids {
  const void* at;
  uint32_t each;   // rows of an id
  int slots, wide; // wide: 64-bit ids
  __device__ __forceinline__ int entry(uint32_t i) const {
    const int64_t v = wide ? static_cast<const int64_t*>(at)[i] : static_cast<const int32_t*>(at)[i];
    return v >= 0 && v < slots ? (int)v : -1;
  }
  __device__ __forceinline__ int of(int m) const { return entry((uint32_t)m / each); }
};

// The rows of a tile that `match` names, packed: lane q holds the q-th of them (and those past their count the others).
__device__ __forceinline__ int packed_rows(uint64_t match, int lane) {
  const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(match >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)match, 0));
  const int to = match >> lane & 1 ? before : __popcll(match) + lane - before;
  return __builtin_amdgcn_ds_permute(to << 2, lane);
}

// f(id, rows) for each adapter among the ids (`mine`: this lane's row's, or -1) of 64 rows: all of them, or, of 64 workgroups that share
// the rows (z of 64), the one whose first row is row z.
template <typename F>
__device__ __forceinline__ void passes(int mine, int z, bool shared, F f) {
  uint64_t left = __ballot(mine >= 0);
  if (shared) {
    if (!(left >> z & 1)) return;
    const int id = __builtin_amdgcn_readlane(mine, z);
    const uint64_t match = __ballot(mine == id);
    if (!(match & ((1ull << z) - 1))) f(id, match);
    return;
  }
  while (left) {
    const int id = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)left) - 1);
    const uint64_t match = __ballot(mine == id);
    left &= ~match;
    f(id, match);
  }
}

// Memory wants neighbouring lanes in neighbouring 16 bytes. With a row a lane (what a matrix operand is), each lane needs a line of its own from
// the first cache, and 65536 x 5120 x rank 64 ran at 3.6 TB/s, bound by that; so x goes through LDS, a result's lane is eight columns
// (`up`), and the factors are kept in the order in which a wave's lanes read them.
//
// The factors' orders, of a factor with columns c (k of A, n of B) and ranks r < P: C rounded up to 128, P values each.
__host__ __device__ __forceinline__ int64_t factor_size(int64_t C, int P) { return (C + 127) / 128 * 128 * P; }
// for `down`: of 32 columns and 16 ranks, lane 16 ((c >> 3) & 3) + (r & 15) holds eight columns
__device__ __forceinline__ int64_t down_at(int c, int r, int P) {
  return ((int64_t)((c >> 5) * (P >> 4) + (r >> 4)) * 64 + (c >> 3 & 3) * 16 + (r & 15)) * 8 + (c & 7);
}
// for `up`: of the 16 columns c with one c & 7 of 128, and 32 ranks (16 with P 16), lane 16 ((r >> 3) & 3) + ((c >> 3) & 15) holds eight ranks
__device__ __forceinline__ int64_t up_at(int c, int r, int P) {
  return ((int64_t)((c >> 7) * 8 + (c & 7)) * (2 * P) + (r >> 3) * 16 + (c >> 3 & 15)) * 8 + (r & 7);
}

// ---- down ----------------------------------------------------------------------------------------------------------------
// A wave takes 16 NS rows and 64 k a step, the next step on its way meanwhile; x goes through its part of LDS (8 lanes a row; chunk c of a
// row at c ^ (row % 8), so that neither direction meets a bank twice). The factor is the first operand, so that a lane's sums are of one row
// and four consecutive ranks. The four waves of a workgroup take 32 rows each and the same slice of k; with few rows (ROWS false) the same 64
// rows, 16 at a time, and every fourth step, and add their sums in LDS. Bound by memory where there are many rows: 65536 x 1280 bf16 with rank
// 64 40 us, 4.2 TB/s of x; 16384 x 5120 with rank 32 39 us, 4.3; 8202 x 640 9.2 us, most of it the start and the end of the launch.
struct DownArgs {
  const uint16_t *x, *f;
  Ids ids;
  float* part;
  int64_t ldx;
  int M, K, slice;
};

template <int DT, int J, int NS, bool ROWS, bool ONE>
__device__ __forceinline__ void down_pass(const DownArgs& p, int id, int row0, int list, int count, uint8_t* lds) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int k0 = (int)blockIdx.y * p.slice, k1 = min(p.K, k0 + p.slice), stride = ROWS ? 64 : 256;
  const int piece = lane & 7;
  uint8_t* const turn = lds + wave * (ROWS ? 4096 : 2048);   // (waves may hold different NS)
  const uint16_t* x[NS * 2];
#pragma unroll
  for (int i = 0; i < NS * 2; ++i) x[i] = p.x + (int64_t)(row0 + __shfl(list, min(8 * i + (lane >> 3), count - 1))) * p.ldx;
  constexpr int SLAB = 2 * J * 64, MINE = SLAB / 256 ? SLAB / 256 : 1;   // 16-byte pieces of 64 k; of a thread
  const v4u* const f = reinterpret_cast<const v4u*>(p.f + id * factor_size(p.K, 16 * J)) + (ONE ? threadIdx.x % SLAB : lane);
  v4u* const slab = reinterpret_cast<v4u*>(lds + 16384);
  v4f acc[J][NS] = {};
  struct Step {
    v4u x[NS * 2], f[ONE ? MINE : 2 * J];
  };
  auto load = [&](Step& b, int k) {
    const int from = min(k + 8 * piece, p.K - 8);
#pragma unroll
    for (int i = 0; i < NS * 2; ++i) b.x[i] = *reinterpret_cast<const v4u*>(x[i] + from);
#pragma unroll
    for (int i = 0; i < (ONE ? MINE : 2 * J); ++i) b.f[i] = f[(int64_t)(k >> 6) * SLAB + i * (ONE ? 256 : 64)];
  };
  auto products = [&](const Step& b, int k, int n) {
    const uint32_t in = k + 8 * piece < k1 ? ~0u : 0u;   // zeros past the end (the factor's are, but an infinity times zero would be NaN)
    wave_sync();
#pragma unroll
    for (int i = 0; i < NS * 2; ++i) {
      const int r = 8 * i + (lane >> 3);
      *reinterpret_cast<v4u*>(turn + r * 128 + ((piece ^ (r & 7)) << 4)) = b.x[i] & in;
    }
    wave_sync();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const v4i xs = *reinterpret_cast<const v4i*>(turn + (16 * s + l16) * 128 + (((4 * h + g) ^ (l16 & 7)) << 4));
#pragma unroll
        for (int j = 0; j < J; ++j)
          acc[j][s] = mfma16_16<DT>(__builtin_bit_cast(v4i, ONE ? slab[n * SLAB + (h * J + j) * 64 + lane] : b.f[ONE ? 0 : h * J + j]), xs, acc[j][s]);
      }
  };
  int k = k0 + (ROWS ? 0 : wave * 64);
  if (k < k1) {   // (past the end the first step is loaded again: no branch between a step's loads and the products that wait for the one before)
    const int first = k;
    Step b[2];
    load(b[0], k);
    for (int n = 0; k < k1; k += stride, n ^= 1) {
      if constexpr (ONE) {   // the workgroup's rows have one adapter: its waves share a step's factor in LDS. Two slabs, one barrier a step
#pragma unroll
        for (int i = 0; i < MINE; ++i) slab[n * SLAB + (i * 256 + threadIdx.x) % SLAB] = b[0].f[i];
      }
      load(b[1], k + stride < k1 ? k + stride : first);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (ONE) ring_barrier();
      products(b[0], k, n);
      b[0] = b[1];
    }
  }
  if constexpr (ROWS) {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int row = row0 + __shfl(list, min(16 * s + l16, count - 1));   // (the last one's sums are written more than once)
      float* const to = p.part + ((int64_t)blockIdx.y * p.M + row) * (16 * J) + 4 * g;
#pragma unroll
      for (int j = 0; j < J; ++j) *reinterpret_cast<v4f*>(to + 16 * j) = acc[j][s];
    }
  } else {   // wave w adds ranks 16 w .. 16 w + 15 of the four waves' sums
    v4f* const sums = reinterpret_cast<v4f*>(lds);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < J; ++j) sums[(wave * J + j) * 64 + lane] = acc[j][0];
    __syncthreads();
    if (wave < J) {
      v4f sum = sums[wave * 64 + lane];
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        const v4f o = sums[(w * J + wave) * 64 + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += o[e];
      }
      const int row = row0 + __shfl(list, min(l16, count - 1));
      *reinterpret_cast<v4f*>(p.part + ((int64_t)blockIdx.y * p.M + row) * (16 * J) + 16 * wave + 4 * g) = sum;
    }
    __syncthreads();
  }
}

template <int DT, int J, bool ROWS>
__global__ __launch_bounds__(256) void adapter_down_kernel(const DownArgs p) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[ROWS ? 16384 + 4096 * J : (J < 2 ? 8192 : 4096 * J)];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int row0 = (int)blockIdx.x * (ROWS ? 128 : 64);
  if constexpr (ROWS) {
    const int a = row0 + lane < p.M ? p.ids.of(row0 + lane) : -1, b = row0 + 64 + lane < p.M ? p.ids.of(row0 + 64 + lane) : -1;
    const int id = __builtin_amdgcn_readfirstlane(a);
    if (id >= 0 && __ballot(a == id && b == id) == ~0ull) {
      if (blockIdx.z == 0) down_pass<DT, J, 2, true, true>(p, id, row0 + wave * 32, lane, 32, lds);
      return;
    }
    row0 += wave * 32;
  }
  const int mine = (!ROWS || lane < 32) && row0 + lane < p.M ? p.ids.of(row0 + lane) : -1;
  passes(mine, blockIdx.z, gridDim.z > 1, [&](int id, uint64_t match) {
    int list = packed_rows(match, lane), count = __popcll(match);
    if constexpr (ROWS) {
      if (count <= 16) down_pass<DT, J, 1, true, false>(p, id, row0, list, count, lds);
      else down_pass<DT, J, 2, true, false>(p, id, row0, list, count, lds);
    } else {
      for (; count > 0; count -= 16, list = __shfl(list, lane + 16)) down_pass<DT, J, 1, false, false>(p, id, row0, list, count, lds);
    }
  });
}

// ---- up ------------------------------------------------------------------------------------------------------------------
// A wave takes 16 rows and 128 columns a step: eight tiles of 16 x 16, tile u of the columns with c % 8 == u, so that a lane's sums are
// eight consecutive columns of four rows, and 16 lanes' 256 bytes of a row. The four waves of a workgroup take 16 rows each and the same `cols`
// columns; with few rows (ROWS false) the same 64 rows, 16 at a time, and every fourth step. PAST: results go past the caches. With rank 16
// one instruction takes both parts of t. Bound by memory where there are many rows: 65536 x 5120 bf16 with rank 64, base read and result
// written, 277 us, 4.8 TB/s; 16384 x 5120 with rank 32 71.5 us, 4.7. 8202 rows whose twenty-odd requests end inside tiles 44 us, 3.8: such a
// tile's passes read the factors of each of its adapters from the second cache.
struct UpArgs {
  const float *part, *scale;
  const uint16_t* g;
  Ids ids;
  const uint16_t* base;   // BASE; zeros without
  uint16_t* out;
  float* joined;          // [M, P]: t with its scale, or NULL
  int ldb, ldo, M, C, R, slices, cols, blocks;   // columns of a workgroup, such blocks of columns
};

template <int DT, int P, bool BASE, int NS, bool ROWS, bool ONE, bool PAST>
__device__ __forceinline__ void up_pass(const UpArgs& p, int id, int row0, int list, int count, int c, int c_end, bool join, uint8_t* lds) {
  constexpr int KS = P == 16 ? 1 : P / 32, PARTS = P == 16 ? 1 : 2, STEP = ROWS ? 128 : 512, LANES = P == 16 ? 32 : 64;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4, gr = P == 16 ? g & 1 : g;
  const float scale = p.scale[id];
  int line[NS][4];   // rows of the sums; past the count the last one, whose results are written more than once
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) line[s][i] = row0 + __shfl(list, min(16 * s + 4 * g + i, count - 1));
  v4i t[NS][KS][PARTS];
  float back[NS][4];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int row = row0 + __shfl(list, min(16 * s + l16, count - 1));
    RankPiece piece[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const float* at = p.part + (int64_t)row * P + 32 * k + 8 * gr;
      const int64_t step = (int64_t)p.M * P;
      piece[k].load(at);
      int i = 1;
      constexpr int AT_ONCE = 4;   // loads in flight
      for (; i + AT_ONCE <= p.slices; i += AT_ONCE) {
        RankPiece more[AT_ONCE];
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) more[n].load(at + (i + n) * step);
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n)
#pragma unroll
          for (int e = 0; e < 8; ++e) piece[k].raw[e >> 2][e & 3] += more[n].raw[e >> 2][e & 3];
      }
      for (; i < p.slices; ++i) {
        RankPiece more;
        more.load(at + i * step);
#pragma unroll
        for (int e = 0; e < 8; ++e) piece[k].raw[e >> 2][e & 3] += more.raw[e >> 2][e & 3];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {   // (ranks past R are sums of zeros times x, and may be NaN)
        const float v = piece[k].raw[e >> 2][e & 3] * scale;
        piece[k].raw[e >> 2][e & 3] = 32 * k + 8 * gr + e < p.R ? v : 0.0f;
      }
      if (join && (P != 16 || g < 2)) {
        v4f* const to = reinterpret_cast<v4f*>(p.joined + (int64_t)row * P + 32 * k + 8 * gr);
        to[0] = piece[k].raw[0];
        to[1] = piece[k].raw[1];
      }
    }
    if constexpr (DT == PQ_F16) {   // a row on a scale of its own, that its largest value gives
      float m = piece[0].largest();
#pragma unroll
      for (int k = 1; k < KS; ++k) m = fmaxf(m, piece[k].largest());
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      const int by = scale_exponent(m);
#pragma unroll
      for (int i = 0; i < 4; ++i) back[s][i] = power(__shfl(by, 4 * g + i));
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) piece[k].raw[e >> 2][e & 3] *= power(-by);
    }
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const RankParts both = parts_of<DT>(piece[k]);
      if constexpr (P == 16) {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[s][0][0][e] = g < 2 ? both.hi[e] : both.lo[e];
      } else {
        t[s][k][0] = both.hi;
        t[s][k][PARTS - 1] = both.lo;
      }
    }
  }
  v4u b[NS][4], ahead[NS][4];   // this step's base, and the next one's
  v4f acc[NS][8];
  auto load = [&](int c0) {
    if constexpr (BASE) {
      const int from = min(c0 + 8 * l16, p.C - 8);
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) ahead[s][i] = *reinterpret_cast<const v4u*>(p.base + (int64_t)line[s][i] * p.ldb + from);
    }
  };
  auto take = [&] {
    if constexpr (BASE) {
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) b[s][i] = ahead[s][i];
    }
  };
  auto products = [&](const v4u* from, int step) {   // from, step: the lane's place in a tile's factor, and from tile to tile
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int u = 0; u < 8; ++u) acc[s][u] = v4f{};
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const v4i fs = __builtin_bit_cast(v4i, from[(u * KS + k) * step]);
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int part = PARTS - 1; part >= 0; --part) acc[s][u] = mfma16_16<DT>(t[s][k][part], fs, acc[s][u]);
      }
  };
  auto result = [&](int s, int i) {
    v4u o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float lo = acc[s][2 * e][i], hi = acc[s][2 * e + 1][i];
      if constexpr (DT == PQ_F16) lo *= back[s][i], hi *= back[s][i];
      if constexpr (BASE) lo += lo16_to_f32<DT>(b[s][i][e]), hi += hi16_to_f32<DT>(b[s][i][e]);
      o[e] = pack2<DT>(lo, hi);
    }
    return o;
  };
  auto place = [&](int s, int i, int c0) { return reinterpret_cast<v4u*>(p.out + (int64_t)line[s][i] * p.ldo + c0 + 8 * l16); };
  const v4u* const factor = reinterpret_cast<const v4u*>(p.g + id * factor_size(p.C, P));
  constexpr int SLAB = 8 * KS * LANES;   // 16-byte pieces of 128 columns
  const int first = c;
  if (c < c_end) load(c);
  if constexpr (ONE) {
    // The workgroup's rows have one adapter: its waves share a step's factor in LDS, where it costs the way from memory a quarter of what
    // it does from the first cache (65536 x 5120 x rank 64: 389 us without). Two slabs, one barrier a step.
    constexpr int MINE = SLAB / 256 ? SLAB / 256 : 1;
    const int tid = threadIdx.x;
    v4u* const slab = reinterpret_cast<v4u*>(lds);
    v4u next[MINE];
    auto fetch = [&](int c0) {
#pragma unroll
      for (int i = 0; i < MINE; ++i) next[i] = factor[(int64_t)(c0 >> 7) * SLAB + i * 256 + tid];
    };
    auto put = [&](int which) {
#pragma unroll
      for (int i = 0; i < MINE; ++i) slab[which * SLAB + i * 256 + tid] = next[i];
    };
    if (c + 128 <= c_end) {
      fetch(c);
      put(0);
      ring_barrier();
      for (int n = 0; c + 128 <= c_end; c += 128, n ^= 1) {   // (past the end the first step again: no branch between loads and what waits for those before)
        take();
        fetch(c + 256 <= c_end ? c + 128 : first);
        load(c + 128 < c_end ? c + 128 : first);
        __builtin_amdgcn_sched_barrier(0);
        products(slab + n * SLAB + (lane & (LANES - 1)), LANES);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (PAST) __builtin_nontemporal_store(result(0, i), place(0, i, c));
          else *place(0, i, c) = result(0, i);
        }
        put(n ^ 1);
        ring_barrier();
      }
    }
  }
  for (; c < c_end; c += STEP) {
    take();
    if (c + STEP < c_end) load(c + STEP);
    products(factor + (int64_t)(c >> 7) * SLAB + (lane & (LANES - 1)), LANES);
    if (c + 8 * l16 < p.C) {
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) *place(s, i, c) = result(s, i);
    }
  }
}

template <int DT, int P, bool BASE, bool ROWS, bool PAST>
__global__ __launch_bounds__(256) void adapter_up_kernel(const UpArgs p) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[ROWS ? 512 * P : 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = (int)blockIdx.x / p.blocks, block = (int)blockIdx.x - tile * p.blocks;
  const int c_begin = block * p.cols + (ROWS ? 0 : wave * 128), c_end = min(p.C, (block + 1) * p.cols);
  const bool join = p.joined && block == 0 && (ROWS || wave == 0);
  int row0 = tile * 64;
  bool mine_in = row0 + lane < p.M;
  int mine = mine_in ? p.ids.of(row0 + lane) : -1;
  if constexpr (ROWS) {
    const int id = __builtin_amdgcn_readfirstlane(mine);
    if (id >= 0 && __ballot(mine == id) == ~0ull) {
      if (blockIdx.z == 0) up_pass<DT, P, BASE, 1, true, true, PAST>(p, id, row0 + wave * 16, lane, 16, c_begin, c_end, join, lds);
      return;
    }
    row0 += wave * 16;
    mine = __shfl(mine, wave * 16 + (lane & 15));
    mine_in = lane < 16 && row0 + lane < p.M;
    if (!mine_in) mine = -1;
  }
  passes(mine, blockIdx.z, gridDim.z > 1, [&](int id, uint64_t match) {
    int list = packed_rows(match, lane), count = __popcll(match);
    for (; count > 0; count -= 16, list = __shfl(list, lane + 16)) up_pass<DT, P, BASE, 1, ROWS, false, false>(p, id, row0, list, count, c_begin, c_end, join, lds);
  });
  if (blockIdx.z || (BASE && p.out == p.base)) return;
  // rows without an adapter, 16 at a time, 16 lanes a row, eight loads in flight
  const uint64_t none = __ballot(mine < 0 && mine_in);
  const int list = packed_rows(none, lane), count = __popcll(none);
  constexpr int STEP = ROWS ? 128 : 512;
  for (int i0 = 0; i0 < count; i0 += 16) {
    int64_t row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) row[i] = row0 + __shfl(list, min(i0 + 4 * i + (lane >> 4), count - 1));   // (the last one more than once)
    for (int c = c_begin + (lane & 15) * 8; c < c_end; c += 2 * STEP) {
      v4u v[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[h][i] = BASE ? *reinterpret_cast<const v4u*>(p.base + row[i] * p.ldb + min(c + h * STEP, p.C - 8)) : v4u{0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (c + h * STEP < c_end) {
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<v4u*>(p.out + row[i] * p.ldo + c + h * STEP) = v[h][i];
        }
    }
  }
}

// ---- a few rows, both products in one launch -----------------------------------------------------------------------------
// A workgroup of eight waves takes a row and `cols` columns: t whole (32 k a wave at a time, lane 16 q + r the product of eight k and rank r,
// added over lanes and waves), then 128 columns of the result a wave. No matrix instructions: of 16 rows they would use one. Bound by the latency of
// three loads that wait for each other (an id, its factor, the launch) and, from some 64 rows on, by the factors' way from the second cache: a row
// reads K P values for each of its column blocks. A row's workgroups are M apart, on one XCD where M is a multiple of 8.
struct RowArgs {
  const uint16_t *x, *f, *g, *base;
  const float* scale;
  uint16_t* out;
  float* joined;
  Ids ids;
  int64_t ldx, ldb, ldo;
  int M, K, C, R, cols;
};

template <int DT>
__device__ __forceinline__ float dot8(v4u a, v4u b, float s) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    s = fmaf(lo16_to_f32<DT>(a[e]), lo16_to_f32<DT>(b[e]), s);
    s = fmaf(hi16_to_f32<DT>(a[e]), hi16_to_f32<DT>(b[e]), s);
  }
  return s;
}
template <int DT>
__device__ __forceinline__ float dot8(v4f t0, v4f t1, v4u b, float s) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const v4f t = e < 2 ? t0 : t1;
    s = fmaf(t[2 * e & 3], lo16_to_f32<DT>(b[e]), s);
    s = fmaf(t[(2 * e & 3) + 1], hi16_to_f32<DT>(b[e]), s);
  }
  return s;
}

template <int DT, int P, bool BASE>
__global__ __launch_bounds__(512) void adapter_rows_kernel(const RowArgs p) {
  constexpr int J = P / 16, G = P / 4, AHEAD = P == 64 ? 2 : 4;   // a wave's loads of 128 columns of g; blocks of 32 k in flight
  __shared__ __attribute__((aligned(16))) float parts[8][P];
  __shared__ __attribute__((aligned(16))) float t[P];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int block = (int)blockIdx.x / p.M, m = (int)blockIdx.x - block * p.M;
  const int c_begin = block * p.cols, c_end = min(p.C, c_begin + p.cols);
  const int id = __builtin_amdgcn_readfirstlane(p.ids.of(m));
  const uint16_t* const base = p.base + (int64_t)m * p.ldb;
  uint16_t* const out = p.out + (int64_t)m * p.ldo;
  if (id < 0) {
    if (BASE && p.out == p.base) return;
    for (int c = c_begin + (int)threadIdx.x * 8; c < c_end; c += 4096)
      *reinterpret_cast<v4u*>(out + c) = BASE ? *reinterpret_cast<const v4u*>(base + c) : v4u{0, 0, 0, 0};
    return;
  }
  v4u gv[G], bv;
  const v4u* const g = reinterpret_cast<const v4u*>(p.g + id * factor_size(p.C, P));
  auto load = [&](int c0) {
#pragma unroll
    for (int i = 0; i < G; ++i) gv[i] = g[(int64_t)(c0 >> 7) * (16 * P) + i * 64 + lane];
    if constexpr (BASE) bv = *reinterpret_cast<const v4u*>(base + min(c0 + 8 * (lane & 15), p.C - 8));
  };
  int c0 = c_begin + wave * 128;
  if (c0 < c_end) load(c0);   // in flight while t is summed

  const uint16_t* const x = p.x + m * p.ldx;
  const v4u* const f = reinterpret_cast<const v4u*>(p.f + id * factor_size(p.K, P));
  const int blocks = (p.K + 31) >> 5;
  float acc[J] = {};
  for (int k0 = wave; k0 < blocks; k0 += 8 * AHEAD) {
    v4u xv[AHEAD], fv[AHEAD][J];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int k = min(k0 + 8 * a, blocks - 1), c = k * 32 + 8 * (lane >> 4);
      xv[a] = *reinterpret_cast<const v4u*>(x + min(c, p.K - 8));
#pragma unroll
      for (int j = 0; j < J; ++j) fv[a][j] = f[((int64_t)k * J + j) * 64 + lane];
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const bool in = (k0 + 8 * a) * 32 + 8 * (lane >> 4) < p.K;   // zeros on both sides past K: an infinity times zero is none of the sum's
      if (!in) xv[a] = v4u{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < J; ++j) acc[j] = dot8<DT>(xv[a], in ? fv[a][j] : v4u{0, 0, 0, 0}, acc[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    acc[j] += __shfl_xor(acc[j], 16);
    acc[j] += __shfl_xor(acc[j], 32);
    if (lane < 16) parts[wave][16 * j + lane] = acc[j];
  }
  __syncthreads();
  if (threadIdx.x < P) {
    const int r = threadIdx.x;
    float sum = parts[0][r];
#pragma unroll
    for (int w = 1; w < 8; ++w) sum += parts[w][r];
    sum = r < p.R ? sum * p.scale[id] : 0.0f;
    t[r] = sum;
    if (p.joined && block == 0) p.joined[(int64_t)m * P + r] = sum;
  }
  __syncthreads();
  while (c0 < c_end) {
    float sum[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {   // column 8 (lane % 16) + u: the ranks of lane / 16, added over the lanes
      const int at = P == 16 ? (lane >> 4 & 1) * 8 : (lane >> 4) * 8;
      const v4f t0 = *reinterpret_cast<const v4f*>(t + at), t1 = *reinterpret_cast<const v4f*>(t + at + 4);
      if constexpr (P == 16) {      // (two columns a load, lanes 0-31 and 32-63)
        if (u & 1) continue;
        float one = dot8<DT>(t0, t1, gv[u / 2], 0.0f);
        one += __shfl_xor(one, 16);
        const float other = __shfl_xor(one, 32);
        sum[u] = lane < 32 ? one : other;
        sum[u + 1] = lane < 32 ? other : one;
      } else {
        float one = dot8<DT>(t0, t1, gv[u * (P / 32)], 0.0f);
        if constexpr (P == 64) {
          const v4f t2 = *reinterpret_cast<const v4f*>(t + at + 32), t3 = *reinterpret_cast<const v4f*>(t + at + 36);
          one = dot8<DT>(t2, t3, gv[2 * u + 1], one);
        }
        one += __shfl_xor(one, 16);
        sum[u] = one + __shfl_xor(one, 32);
      }
    }
    v4u o;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = BASE ? pack2<DT>(sum[2 * e] + lo16_to_f32<DT>(bv[e]), sum[2 * e + 1] + hi16_to_f32<DT>(bv[e])) : pack2<DT>(sum[2 * e], sum[2 * e + 1]);
    const int c = c0 + 8 * (lane & 15);
    if (lane < 16 && c < c_end) *reinterpret_cast<v4u*>(out + c) = o;
    c0 += 1024;
    if (c0 < c_end) load(c0);
  }
}

// ---- sums over the rows of an adapter ------------------------------------------------------------------------------------
// part[chunk][slot][r][c] = sum over the chunk's rows m of that adapter of v[m, r] z[m, c], v: t or dt with its scale (`joined`). A
// workgroup of four waves takes 128 columns, a chunk of rows and an adapter; of its rows, 64 a step, only steps that hold a row of
// the adapter are read, the next one's on their way into registers meanwhile, with zeros in the place of other adapters' rows. Both sums of
// 16384 x (5120 + 1280) bf16 with rank 32: 53 us, 4.0 TB/s of dy and x; beside them each panel reads t, half as many bytes again, from the
// second cache.
struct SumArgs {
  const uint16_t* z;
  const float* v;
  float* part;
  int32_t* used;          // [chunk][slot]: whether part was written
  int64_t ldz;
  int M, C, panels, blocks;   // panels of 128 columns, blocks: panels * chunks, or 0
  int unit, parts, rows;      // see Chunks
  int by_entry;               // a chunk's rows have at most 64 ids, and gridDim.y workgroups take an adapter of theirs each
};

template <int DT, int P>
__device__ __forceinline__ void row_sums(const SumArgs& p, const Ids& ids, int block, int which, uint8_t* sz, uint8_t* sv, uint32_t* top, float* back) {
  constexpr int TILES = P == 16 ? 1 : P / 32, PITCH = P == 16 ? 64 : P * 2;   // of v's tiles: with P 16, the first part in ranks 0-15, the second in 16-31
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunk = block / p.panels, panel = block - chunk * p.panels;
  const int unit = chunk / p.parts, u0 = unit * p.unit, at0 = (chunk - unit * p.parts) * p.rows;
  const int c0 = panel * 128, s0 = u0 + at0, end = min(p.M, u0 + min(p.unit, at0 + p.rows));
  int slot = p.by_entry ? -1 : which;
  if (p.by_entry) {   // the which-th adapter among the chunk's ids
    const uint32_t e0 = (uint32_t)s0 / ids.each;
    const int mine = (int64_t)(e0 + lane) * ids.each < end ? ids.entry(e0 + lane) : -1;
    uint64_t left = __ballot(mine >= 0);
    if (which == 0 && panel == 0 && wave == 0)
      for (int at = lane; at - lane < ids.slots; at += 64) {
        int has = 0;
        for (uint64_t more = left; more;) {
          const int id = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)more) - 1);
          more &= ~__ballot(mine == id);
          has |= id == at;
        }
        if (at < ids.slots) p.used[chunk * ids.slots + at] = has;
      }
    for (int i = 0; left; ++i) {
      slot = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)left) - 1);
      left &= ~__ballot(mine == slot);
      if (i == which) break;
      slot = -1;
    }
    if (slot < 0) return;
  }
  auto z_at = [&](int row, int at) { return sz + row * 256 + ((at ^ spread(row)) << 4); };
  auto hi_at = [&](int row, int at) { return sv + row * PITCH + (at << 4); };
  auto lo_at = [&](int row, int at) { return sv + (64 + row) * PITCH + (at << 4); };
  // the step (its first row) at or after m that holds a row of the adapter, or `end`
  auto next = [&](int m) {
    for (uint32_t e = (uint32_t)m / ids.each; m < end; e += 64) {
      const int64_t first = (int64_t)(e + lane) * ids.each;
      const uint64_t match = __ballot(first < end && ids.entry(first < end ? e + lane : e) == slot);
      if (match) {
        const int64_t row = (int64_t)(e + __ffsll((unsigned long long)match) - 1) * ids.each;
        return max(m, (int)row) - (max(m, (int)row) - s0) % 64;
      }
      if ((int64_t)(e + 64) * ids.each >= end) break;
    }
    return end;
  };
  v16f acc[TILES] = {};
  v4u zr[4];
  v4f vr[P / 16];
  auto load = [&](int m0) {
    const uint64_t match = __ballot(m0 + lane < end && ids.of(min(m0 + lane, p.M - 1)) == slot);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 16 + (tid >> 4), c = c0 + (tid & 15) * 8;
      zr[i] = v4u{0, 0, 0, 0};
      if ((match >> r & 1) && c < p.C) zr[i] = *reinterpret_cast<const v4u*>(p.z + (int64_t)(m0 + r) * p.ldz + c);
    }
#pragma unroll
    for (int i = 0; i < P / 16; ++i) {
      const int at = i * 256 + tid, r = at / (P / 4);
      vr[i] = v4f{};
      if (match >> r & 1) vr[i] = *reinterpret_cast<const v4f*>(p.v + (int64_t)(m0 + r) * P + at % (P / 4) * 4);
    }
  };
  auto rank = [&](int j) { return P == 16 ? lane & 15 : 32 * j + (lane & 31); };
  int m0 = next(s0);
  if (!p.by_entry && panel == 0 && tid == 0) p.used[chunk * ids.slots + slot] = m0 < end;
  if (m0 >= end) return;
  load(m0);
  while (m0 < end) {
    if constexpr (DT == PQ_F16) tell_largest<P>(vr, top, tid);
    __syncthreads();
    if constexpr (DT == PQ_F16) scale_values<P>(vr, top, back, tid);
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<v4u*>(z_at(i * 16 + (tid >> 4), tid & 15)) = zr[i];
#pragma unroll
    for (int i = 0; i < P / 16; ++i) {
      const int at = i * 256 + tid, r = at / (P / 4), q = at % (P / 4);   // row, and its ranks 4 q ..
      v2u hi, lo;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t h, l;
        two_parts<DT>(vr[i][2 * e], vr[i][2 * e + 1], h, l);
        hi[e] = h;
        lo[e] = l;
      }
      *reinterpret_cast<v2u*>(sv + r * PITCH + q * 8) = hi;
      *reinterpret_cast<v2u*>(sv + (P == 16 ? r * PITCH + 32 : (64 + r) * PITCH) + q * 8) = lo;
    }
    __syncthreads();
    const int m1 = next(m0 + 64);
    if (m1 < end) load(m1);   // in flight while this step's products run
    v4i z[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) z[s] = read_columns(z_at, 16 * s, wave * 32, lane);
#pragma unroll
    for (int j = 0; j < TILES; ++j) {
      v16f sum = DT == PQ_F16 ? v16f{} : acc[j];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        sum = mfma16<DT>(z[s], read_columns(hi_at, 16 * s, 32 * j, lane), sum);
        if constexpr (P != 16) sum = mfma16<DT>(z[s], read_columns(lo_at, 16 * s, 32 * j, lane), sum);
      }
      if constexpr (DT == PQ_F16) {
        const float by = back[rank(j)];
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[j][e] = fmaf(sum[e], by, acc[j][e]);
      } else {
        acc[j] = sum;
      }
    }
    m0 = m1;
  }
  if constexpr (P == 16) {
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[0][e] += __shfl_xor(acc[0][e], 16);
  }
  // lane: r = 32 j + lane % 32, columns c0 + 32 wave + 8 q + 4 (lane / 32) + e
  const int c = c0 + wave * 32 + 4 * (lane >> 5);
  float* const part = p.part + ((int64_t)chunk * ids.slots + slot) * P * p.C;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (c + 8 * q >= p.C) break;
#pragma unroll
    for (int j = 0; j < TILES; ++j)
      if (P != 16 || (lane & 31) < 16)
        *reinterpret_cast<v4f*>(part + (int64_t)rank(j) * p.C + c + 8 * q) =
            v4f{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
  }
}

template <int DT, int P>
__global__ __launch_bounds__(256) void adapter_sums_kernel(const SumArgs b, const SumArgs a, const Ids ids) {
  __shared__ __attribute__((aligned(16))) uint8_t sz[64 * 256];
  __shared__ __attribute__((aligned(16))) uint8_t sv[2 * 64 * (P == 16 ? 32 : P * 2)];
  __shared__ __attribute__((aligned(16))) uint32_t top[DT == PQ_F16 ? 2 * P : 4];
  __shared__ __attribute__((aligned(16))) float back[DT == PQ_F16 ? P : 4];
  const bool is_b = (int)blockIdx.x < b.blocks;
  row_sums<DT, P>(is_b ? b : a, ids, (int)blockIdx.x - (is_b ? 0 : b.blocks), blockIdx.y, sz, sv, top, back);
}

// The chunks' sums in order, rounded: dB [slots, R, N] and dA [slots, K, R]. (8 adapters of 5120 + 1280 columns and rank 32, of 16 and 48 chunks, 8 us.)
struct JoinArgs {
  const float* part;
  const int32_t* used;
  uint16_t* out;
  int chunks, C, groups, blocks;   // groups of 256 columns; workgroups (0: not wanted)
};
template <int DT>
__global__ __launch_bounds__(256) void adapter_join_kernel(const JoinArgs b, const JoinArgs a, int slots, int P, int R) {
  const bool is_b = (int)blockIdx.x < b.blocks;
  const JoinArgs p = is_b ? b : a;
  const int block = (int)blockIdx.x - (is_b ? 0 : b.blocks), slot = blockIdx.y;
  const int lane = threadIdx.x & 63, c = block % p.groups * 256 + 4 * lane, r = block / p.groups * 4 + (threadIdx.x >> 6);
  v4f s = {};
  const float* const at = p.part + ((int64_t)slot * P + min(r, P - 1)) * p.C + min(c, p.C - 4);
  const int64_t step = (int64_t)slots * P * p.C;
  for (int i0 = 0; i0 < p.chunks; i0 += 64) {
    uint64_t used = __ballot(i0 + lane < p.chunks && p.used[min(i0 + lane, p.chunks - 1) * slots + slot]);
    while (used) {   // four loads in flight
      v4f v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = v4f{};
        if (used) v[e] = *reinterpret_cast<const v4f*>(at + (i0 + __ffsll((unsigned long long)used) - 1) * step);
        used &= used - 1;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int n = 0; n < 4; ++n) s[n] += v[e][n];
    }
  }
  if (c >= p.C || r >= R) return;
  uint16_t* const out = p.out + (int64_t)slot * R * p.C;
  if (is_b) {
    *reinterpret_cast<v2u*>(out + (int64_t)r * p.C + c) = v2u{pack2<DT>(s[0], s[1]), pack2<DT>(s[2], s[3])};
  } else {
#pragma unroll
    for (int n = 0; n < 4; ++n) out[(int64_t)(c + n) * R + r] = (uint16_t)f32_to_16_bits<DT>(s[n]);
  }
}

// ---- the factors' orders -------------------------------------------------------------------------------------------------
// A factor of each slot from any of its orders to those of `down` and `up`, with zeros past R and C: 128 columns a workgroup, in LDS between.
struct FactorArgs {
  const uint16_t* from;
  uint16_t *down, *up;
  int C, blocks, order;   // of `from`
};
__global__ __launch_bounds__(256) void adapter_factors_kernel(const FactorArgs a, const FactorArgs b, int R, int P) {
  __shared__ uint16_t tile[128][66];   // [c][r]; a pitch of 33 words: both directions spread over the banks
  const bool is_a = (int)blockIdx.x < a.blocks;
  const FactorArgs p = is_a ? a : b;
  const int c0 = ((int)blockIdx.x - (is_a ? 0 : a.blocks)) * 128, slot = blockIdx.y;
  const bool packed = p.order >= PQ_ADAPTER_DOWN;
  const uint16_t* const from = p.from + slot * (packed ? factor_size(p.C, P) : (int64_t)R * p.C);
  const bool wide = (uintptr_t)p.from % 16 == 0;
  for (int i = threadIdx.x; i < 16 * P; i += 256) {   // eight values: of columns c .. c + 7, or of ranks r .. r + 7
    const bool by_rank = p.order == PQ_ADAPTER_BY_RANK || p.order == PQ_ADAPTER_DOWN;
    int c, r;
    if (p.order == PQ_ADAPTER_DOWN) r = i % P, c = i / P * 8;
    else if (p.order == PQ_ADAPTER_UP) c = i % 16 * 8 + i / 16 % 8, r = i / 128 * 8;
    else if (by_rank) c = i % 16 * 8, r = i / 16;
    else c = i / (P / 8), r = i % (P / 8) * 8;
    uint16_t v[8] = {};
    if (r < R && c0 + c < p.C) {
      const uint16_t* const at = from + (p.order == PQ_ADAPTER_DOWN ? down_at(c0 + c, r, P) : p.order == PQ_ADAPTER_UP ? up_at(c0 + c, r, P)
                                         : by_rank ? (int64_t)r * p.C + c0 + c : (int64_t)(c0 + c) * R + r);
      if (packed || (wide && (by_rank || R % 8 == 0))) {
        const v4u w = *reinterpret_cast<const v4u*>(at);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (by_rank || r + e < R) v[e] = at[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) tile[c + (by_rank ? e : 0)][r + (by_rank ? 0 : e)] = v[e];
  }
  __syncthreads();
  const int64_t to = slot * factor_size(p.C, P);
  for (int i = threadIdx.x; i < 16 * P; i += 256) {
    v4u w;
    if (p.down) {
      const int r = i % 16 + i / 64 % (P / 16) * 16, c = i / 16 % 4 * 8 + i / (4 * P) * 32;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = tile[c + 2 * e][r] | (uint32_t)tile[c + 2 * e + 1][r] << 16;
      *reinterpret_cast<v4u*>(p.down + to + down_at(c0 + c, r, P)) = w;
    }
    if (p.up) {
      const int c = i % 16 * 8 + i / (2 * P) % 8, r = i / 16 % (P / 8) * 8;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = tile[c][r + 2 * e] | (uint32_t)tile[c][r + 2 * e + 1] << 16;
      *reinterpret_cast<v4u*>(p.up + to + up_at(c0 + c, r, P)) = w;
    }
  }
}

// ---- launches --------------------------------------------------------------------------------------------------------------
constexpr int kMostSlices = 16;
bool by_rows(int64_t M) { return M >= 128; }   // the waves of a workgroup take rows of their own (128 of them), else 64 rows together
int64_t tiles_of(int64_t M) { return by_rows(M) ? (M + 127) / 128 : (M + 63) / 64; }
// k of a slice: about 512 workgroups, but four steps of a wave each or more (with few rows one). (With 256, 16384 x 5120 takes 44.5 us for 38.7 and `up`,
// which reads the slices, 16.3 for 18.6; slices of two steps save 1 us at 8202 x 640 and cost `up` 3.)
int slice_of(int64_t M, int64_t K) {
  const int64_t steps = (K + 255) / 256, want = std::min<int64_t>({512 / std::max<int64_t>(tiles_of(M), 1), steps, (int64_t)kMostSlices});
  const int64_t n = std::max<int64_t>(want, 1);
  return (int)((steps + n - 1) / n * 256);
}
int slices_of(int64_t M, int64_t K) { const int s = slice_of(M, K); return (int)((K + s - 1) / s); }
// Workgroups that share a tile's adapters: one for each of its rows where few rows may hold many adapters, else one takes them in turn.
int sharers(int64_t M, int64_t each) { return each < 16 && M <= 1024 ? (by_rows(M) ? 32 : 64) : 1; }

// The rows in units of `unit` and each unit in `parts` of `rows`, a chunk each, so that about 512 workgroups take a sum (us of `sums` for 256, 384,
// 512, 768, with ids of one row: 16384 x 5120 and 1280, rank 32, 71.8, 75.9, 70.1, 68.5; 2051 rows of the same 15.3, 17.2, 16.2, 16.4), and the parts
// have no more than 256 MB. Units are whole requests, so that a chunk's workgroup has all its rows for one adapter where they are long (the first of
// these, requests of 1024 rows: 66 us with chunks of 1280 and 320 rows, which two or three requests share, and 53 with 1024 and 384).
struct Chunks { int64_t unit, parts, rows, count; };
Chunks chunks_of(int64_t M, int64_t C, int64_t slots, int64_t P, int64_t each) {
  if (M < 1) return {64, 1, 64, 1};
  const int64_t steps = (M + 63) / 64, panels = (C + 127) / 128;
  const int64_t room = std::max<int64_t>(((int64_t)128 << 20) / (slots * P * C * 4), 1);   // (units may come out half as long as wanted)
  const int64_t want = std::min<int64_t>({(512 + panels - 1) / panels, steps, (int64_t)256, room});
  const int64_t rows = (steps + want - 1) / want * 64;
  if (each <= rows) {
    const int64_t unit = rows / each * each;
    return {unit, 1, unit, (M + unit - 1) / unit};
  }
  const int64_t of_each = (each + 63) / 64, long_steps = (of_each + each / rows - 1) / (each / rows), parts = (of_each + long_steps - 1) / long_steps;
  return {each, parts, long_steps * 64, M / each * parts};
}

int check_ids(const void* ids, int32_t id_bits, int64_t each, int64_t M, int64_t slots, const char* what) {
  if (id_bits != 32 && id_bits != 64) return set_error(PQ_EDTYPE, "%s: ids of %d bits (32 or 64)", what, id_bits);
  if (slots < 1 || slots > 65535) return set_error(PQ_ESHAPE, "%s: %lld adapters (1 to 65535)", what, (long long)slots);
  if (M > 0 && (each < 1 || M % each)) return set_error(PQ_ESHAPE, "%s: %lld rows are not ids of %lld rows each", what, (long long)M, (long long)each);
  if (M > 0 && !ids) return set_error(PQ_EINVAL, "%s: null pointer", what);
  if ((uintptr_t)ids % (id_bits / 8)) return set_error(PQ_EALIGN, "%s: ids aligned to their size", what);
  return PQ_OK;
}
bool rank_ok(int64_t R, int64_t P) { return (P == 16 || P == 32 || P == 64) && R >= 1 && R <= P; }
bool size_ok(int64_t C) { return C >= 8 && C % 8 == 0 && C <= (1 << 24); }
Ids ids_of(const void* ids, int32_t bits, int64_t each, int64_t slots) { return {ids, (uint32_t)each, (int)slots, bits == 64}; }

}  // namespace
}  // namespace adapt
}  // namespace pq

using namespace pq;
using namespace pq::adapt;

#define PQ_BY_RANK(D, GO)                                                    \
  do {                                                                       \
    if (P == 16) GO(D, 16); else if (P == 32) GO(D, 32); else GO(D, 64);     \
  } while (0)
#define PQ_BY_TYPE(GO)                                                       \
  do {                                                                       \
    if (dtype == PQ_BF16) PQ_BY_RANK(PQ_BF16, GO); else PQ_BY_RANK(PQ_F16, GO); \
  } while (0)

extern "C" int64_t pq_adapter_slices(int64_t M, int64_t K) {
  if (M < 1 || !size_ok(K) || M > (1 << 30)) return 1;
  return slices_of(M, K);
}

extern "C" int pq_adapter_down(const void* x, int32_t dtype, int64_t M, int64_t K, int64_t ldx, const void* f, int64_t slots, int64_t P,
                               const void* ids, int32_t id_bits, int64_t each, float* part, hipStream_t stream) {
  if (M < 0 || M > (1 << 30) || !size_ok(K) || ldx < K || !rank_ok(1, P))
    return set_error(PQ_ESHAPE, "pq_adapter_down: M=%lld K=%lld ldx=%lld P=%lld (K a multiple of 8, P 16, 32 or 64)", (long long)M,
                     (long long)K, (long long)ldx, (long long)P);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_adapter_down: dtype %d", dtype);
  if (const int st = check_ids(ids, id_bits, each, M, slots, "pq_adapter_down")) return st;
  if (M == 0) return PQ_OK;
  if (!x || !f || !part) return set_error(PQ_EINVAL, "pq_adapter_down: null pointer");
  if ((uintptr_t)x % 16 || ldx % 8 || (uintptr_t)f % 16 || (uintptr_t)part % 16)
    return set_error(PQ_EALIGN, "pq_adapter_down: operands 16-byte aligned, ldx a multiple of 8");
  const int slice = slice_of(M, K);
  const DownArgs p{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(f), ids_of(ids, id_bits, each, slots), part, ldx, (int)M, (int)K, slice};
  if (const int st = check_grid(tiles_of(M), 256, "pq_adapter_down")) return st;
  const dim3 grid((unsigned)tiles_of(M), (unsigned)slices_of(M, K), (unsigned)sharers(M, each));
#define PQ_DOWN(D, PP)                                                                                              \
  do {                                                                                                              \
    if (by_rows(M)) hipLaunchKernelGGL((adapter_down_kernel<D, PP / 16, true>), grid, dim3(256), 0, stream, p);     \
    else hipLaunchKernelGGL((adapter_down_kernel<D, PP / 16, false>), grid, dim3(256), 0, stream, p);               \
  } while (0)
  PQ_BY_TYPE(PQ_DOWN);
#undef PQ_DOWN
  return check_launch("pq_adapter_down");
}

extern "C" int pq_adapter_up(const float* part, int64_t slices, const float* scale, const void* g, int64_t slots, int64_t C, int64_t R,
                             int64_t P, const void* ids, int32_t id_bits, int64_t each, const void* base, int64_t ldb, void* out,
                             int64_t ldo, float* joined, int32_t dtype, int64_t M, hipStream_t stream) {
  if (M < 0 || M > (1 << 30) || !size_ok(C) || (out && (ldo < C || ldo > (1 << 30))) || (base && (ldb < C || ldb > (1 << 30))) || !rank_ok(R, P) || slices < 1 || slices > kMostSlices)
    return set_error(PQ_ESHAPE, "pq_adapter_up: M=%lld C=%lld ldb=%lld ldo=%lld R=%lld P=%lld slices=%lld (C a multiple of 8)", (long long)M,
                     (long long)C, (long long)ldb, (long long)ldo, (long long)R, (long long)P, (long long)slices);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_adapter_up: dtype %d", dtype);
  if (const int st = check_ids(ids, id_bits, each, M, slots, "pq_adapter_up")) return st;
  if (M == 0) return PQ_OK;
  if (!part || !scale || (!out && (!joined || base)) || (out && !g)) return set_error(PQ_EINVAL, "pq_adapter_up: null pointer");
  if ((uintptr_t)part % 16 || (uintptr_t)g % 16 || (uintptr_t)base % 16 || (base && ldb % 8) || (uintptr_t)out % 16 || ldo % 8 || (uintptr_t)joined % 16)
    return set_error(PQ_EALIGN, "pq_adapter_up: operands 16-byte aligned, strides multiples of 8");
  if (out && base == out && ldb != ldo) return set_error(PQ_ESHAPE, "pq_adapter_up: out is base, with another stride");
  // About 1024 workgroups; where a tile may hold several adapters, and take so many times as long, 4096 (8202 x 5120 with some twenty requests
  // end to end: 65.7 us with 1024, 51.1 with 2048, 47.6 with 4096; 16384 x 5120 with 16 of them: 62.7, 67.0, 70.4).
  // Results of 64 MB and more go past the caches, where they would only drive out what is read next (8202 x 5120 with `down`: 78 -> 73 us,
  // 65536 x 5120 327 -> 314, 16384 x 5120 and its backward pass 240 -> 227).
  const bool rows = by_rows(M), past = rows && M * C >= 32 << 20;
  const int64_t tiles = (M + 63) / 64, width = rows ? 128 : 512, steps = out ? (C + width - 1) / width : 0;
  const int64_t want = std::max<int64_t>(std::min<int64_t>(steps, (each < 64 ? 4096 : 1024) / tiles), 1), each_steps = (steps + want - 1) / want;
  const int blocks = steps ? (int)((steps + each_steps - 1) / each_steps) : 1;   // (no output: no columns)
  const UpArgs p{part, scale, static_cast<const uint16_t*>(g), ids_of(ids, id_bits, each, slots), static_cast<const uint16_t*>(base),
                 static_cast<uint16_t*>(out), joined, (int)ldb, (int)ldo, (int)M, (int)C, (int)R, (int)slices, (int)(each_steps * width), blocks};
  if (const int st = check_grid(tiles * blocks, 256, "pq_adapter_up")) return st;
  const dim3 grid((unsigned)(tiles * blocks), 1, (unsigned)(rows ? std::min(sharers(M, each), 16) : sharers(M, each)));
#define PQ_UP2(D, PP, B)                                                                                    \
  do {                                                                                                      \
    if (past) hipLaunchKernelGGL((adapter_up_kernel<D, PP, B, true, true>), grid, dim3(256), 0, stream, p);       \
    else if (rows) hipLaunchKernelGGL((adapter_up_kernel<D, PP, B, true, false>), grid, dim3(256), 0, stream, p); \
    else hipLaunchKernelGGL((adapter_up_kernel<D, PP, B, false, false>), grid, dim3(256), 0, stream, p);          \
  } while (0)
#define PQ_UP(D, PP)                                          \
  do {                                                        \
    if (base) PQ_UP2(D, PP, true); else PQ_UP2(D, PP, false); \
  } while (0)
  PQ_BY_TYPE(PQ_UP);
#undef PQ_UP
#undef PQ_UP2
  return check_launch("pq_adapter_up");
}

static int64_t padded_bytes(int64_t n) { return (n + 255) / 256 * 256; }

extern "C" int64_t pq_adapter_grads_workspace_size(int64_t M, int64_t K, int64_t N, int64_t slots, int64_t P, int64_t each) {
  if (M < 0 || M > (1 << 30) || !size_ok(K) || !size_ok(N) || slots < 1 || slots > 65535 || !rank_ok(1, P) || (M && (each < 1 || M % each))) return 0;
  int64_t bytes = 0;
  for (const int64_t C : {N, K}) {
    const int64_t chunks = chunks_of(M, C, slots, P, each).count;
    bytes += padded_bytes(4 * chunks * slots * P * C) + padded_bytes(4 * chunks * slots);
  }
  return bytes;
}

extern "C" int pq_adapter_grads(const void* x, int64_t ldx, const void* dy, int64_t lddy, int32_t dtype, const float* t,
                                const float* dt, const void* ids, int32_t id_bits, int64_t each,
                                int64_t M, int64_t K, int64_t N, int64_t slots, int64_t R, int64_t P, void* dA, void* dB, void* workspace,
                                int64_t workspace_bytes, hipStream_t stream) {
  if (M < 0 || M > (1 << 30) || !size_ok(K) || !size_ok(N) || (dA && ldx < K) || (dB && lddy < N) || !rank_ok(R, P))
    return set_error(PQ_ESHAPE, "pq_adapter_grads: M=%lld K=%lld N=%lld R=%lld P=%lld (K and N multiples of 8)", (long long)M, (long long)K,
                     (long long)N, (long long)R, (long long)P);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_adapter_grads: dtype %d", dtype);
  if (const int st = check_ids(ids, id_bits, each, M, slots, "pq_adapter_grads")) return st;
  if (!dA && !dB) return PQ_OK;
  if (!workspace || (M && ((dB && (!dy || !t)) || (dA && (!x || !dt))))) return set_error(PQ_EINVAL, "pq_adapter_grads: null pointer");
  if ((dA && ((uintptr_t)x % 16 || ldx % 8 || (uintptr_t)dt % 16)) || (dB && ((uintptr_t)dy % 16 || lddy % 8 || (uintptr_t)t % 16)) ||
      (uintptr_t)workspace % 16)
    return set_error(PQ_EALIGN, "pq_adapter_grads: operands 16-byte aligned, strides multiples of 8");
  if (workspace_bytes < pq_adapter_grads_workspace_size(M, K, N, slots, P, each))
    return set_error(PQ_ESHAPE, "pq_adapter_grads: workspace of %lld bytes", (long long)workspace_bytes);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  SumArgs sums[2];
  JoinArgs join[2];
  for (int i = 0; i < 2; ++i) {   // dB, dA
    const bool b = i == 0, wanted = b ? dB != nullptr : dA != nullptr;
    const int64_t C = b ? N : K, panels = (C + 127) / 128, groups = (C + 255) / 256;
    const Chunks of = chunks_of(M, C, slots, P, each);
    const int64_t chunks = of.count;
    float* const part = reinterpret_cast<float*>(at);
    at += padded_bytes(4 * chunks * slots * P * C);
    int32_t* const used = reinterpret_cast<int32_t*>(at);
    at += padded_bytes(4 * chunks * slots);
    sums[i] = {static_cast<const uint16_t*>(b ? dy : x), b ? t : dt, part, used, b ? lddy : ldx, (int)M, (int)C, (int)panels, wanted ? (int)(panels * chunks) : 0,
               (int)of.unit, (int)of.parts, (int)of.rows, 0};
    join[i] = {part, used, static_cast<uint16_t*>(b ? dB : dA), (int)chunks, (int)C, (int)groups, wanted ? (int)(groups * ((R + 3) / 4)) : 0};
  }
  // Adapters that a chunk may have, where that is fewer than there are: workgroups without rows cost a microsecond or two of a place.
  int64_t among[2];
  for (int i = 0; i < 2; ++i) {
    among[i] = M ? std::max<int64_t>(sums[i].unit / each, 1) : 1;
    sums[i].by_entry = M && among[i] <= 64 && among[i] < slots;
  }
  const bool by_entry = (sums[0].by_entry || !dB) && (sums[1].by_entry || !dA);
  for (int i = 0; i < 2; ++i) sums[i].by_entry = by_entry;
  const int64_t ways = !by_entry ? slots : std::max(dB ? among[0] : 1, dA ? among[1] : 1);
  // (no rows: no adapter has any, and the ids are not read)
  const Ids id = ids_of(ids, id_bits, M ? each : 1, slots);
  if (const int st = check_grid((int64_t)sums[0].blocks + sums[1].blocks, 256, "pq_adapter_grads")) return st;
  if (const int st = check_grid((int64_t)join[0].blocks + join[1].blocks, 256, "pq_adapter_grads")) return st;
  const dim3 grid((unsigned)(sums[0].blocks + sums[1].blocks), (unsigned)ways), joins((unsigned)(join[0].blocks + join[1].blocks), (unsigned)slots);
#define PQ_SUMS(D, PP) hipLaunchKernelGGL((adapter_sums_kernel<D, PP>), grid, dim3(256), 0, stream, sums[0], sums[1], id)
  PQ_BY_TYPE(PQ_SUMS);
#undef PQ_SUMS
  if (dtype == PQ_BF16) hipLaunchKernelGGL(adapter_join_kernel<PQ_BF16>, joins, dim3(256), 0, stream, join[0], join[1], (int)slots, (int)P, (int)R);
  else hipLaunchKernelGGL(adapter_join_kernel<PQ_F16>, joins, dim3(256), 0, stream, join[0], join[1], (int)slots, (int)P, (int)R);
  return check_launch("pq_adapter_grads");
}

// One launch for both products (us of two launches and of one in a captured graph, bf16, every row another of up to 32 adapters, P 16: 1280 x 1280,
// 1 row 5.7 and 3.5, 64 rows 6.2 and 3.8; 4096 x 4096, 1 row 7.1 and 4.7, 64 rows 10.4 and 6.8; 5120 x 1280 6.5 and 5.2. P 32: 5120 x 1280,
// 1 row 7.2 and 6.9; 8192 x 8192 8.1 and 9.5; P 64: 5120 x 1280 8.6 and 9.1). A workgroup reads a factor for one row alone, so many rows are for `down`
// and `up`: later where a tile of 64 rows may hold many adapters (1280 x 5120 with 16 adapters in turn, P 16, 1024 rows 47 and 20; P 32, 512 rows 31 and
// 18) than where requests are long (77 rows each: P 16, 308 rows 11.6 and 10.5; P 32, 154 rows 10.7 and 10.4, 308 12.9 and 14.6).
extern "C" int pq_adapter_rows_fit(int64_t M, int64_t K, int64_t C, int64_t P, int64_t each) {
  return M >= 0 && M <= 1 << 16 && size_ok(K) && size_ok(C) && rank_ok(1, P) && K * P <= 160 << 10 && M * P <= (each < 16 ? 16 << 10 : 5 << 10);
}

extern "C" int pq_adapter_rows(const void* x, int32_t dtype, int64_t M, int64_t K, int64_t ldx, const void* f, const float* scale, const void* g,
                               int64_t slots, int64_t C, int64_t R, int64_t P, const void* ids, int32_t id_bits, int64_t each, const void* base,
                               int64_t ldb, void* out, int64_t ldo, float* joined, hipStream_t stream) {
  if (M < 0 || M > (1 << 16) || !size_ok(K) || ldx < K || !size_ok(C) || (out && ldo < C) || (base && ldb < C) || !rank_ok(R, P))
    return set_error(PQ_ESHAPE, "pq_adapter_rows: M=%lld K=%lld C=%lld ldx=%lld ldb=%lld ldo=%lld R=%lld P=%lld (K and C multiples of 8)",
                     (long long)M, (long long)K, (long long)C, (long long)ldx, (long long)ldb, (long long)ldo, (long long)R, (long long)P);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_adapter_rows: dtype %d", dtype);
  if (const int st = check_ids(ids, id_bits, each, M, slots, "pq_adapter_rows")) return st;
  if (M == 0) return PQ_OK;
  if (!x || !f || !scale || (!out && (!joined || base)) || (out && !g)) return set_error(PQ_EINVAL, "pq_adapter_rows: null pointer");
  if ((uintptr_t)x % 16 || ldx % 8 || (uintptr_t)f % 16 || (uintptr_t)g % 16 || (uintptr_t)base % 16 || (base && ldb % 8) || (uintptr_t)out % 16 || (out && ldo % 8) || (uintptr_t)joined % 16)
    return set_error(PQ_EALIGN, "pq_adapter_rows: operands 16-byte aligned, strides multiples of 8");
  if (out && base == out && ldb != ldo) return set_error(PQ_ESHAPE, "pq_adapter_rows: out is base, with another stride");
  const int64_t panels = out ? (C + 127) / 128 : 0, blocks = std::max<int64_t>(std::min<int64_t>(panels, 256 / M), 1), cols = (panels + blocks - 1) / blocks * 128;
  const RowArgs p{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(f), static_cast<const uint16_t*>(g), static_cast<const uint16_t*>(base), scale,
                  static_cast<uint16_t*>(out), joined, ids_of(ids, id_bits, each, slots), ldx, ldb, ldo, (int)M, (int)K, (int)C, (int)R, (int)cols};
  const dim3 grid((unsigned)(M * (out ? (C + cols - 1) / cols : 1)));   // (no result: no columns)
#define PQ_ROWS(D, PP)                                                                                    \
  do {                                                                                                    \
    if (base) hipLaunchKernelGGL((adapter_rows_kernel<D, PP, true>), grid, dim3(512), 0, stream, p);      \
    else hipLaunchKernelGGL((adapter_rows_kernel<D, PP, false>), grid, dim3(512), 0, stream, p);          \
  } while (0)
  PQ_BY_TYPE(PQ_ROWS);
#undef PQ_ROWS
  return check_launch("pq_adapter_rows");
}

extern "C" int64_t pq_adapter_factor_size(int64_t C, int64_t P) { return size_ok(C) && rank_ok(1, P) ? factor_size(C, (int)P) : 0; }

extern "C" int pq_adapter_factors(const void* A, int32_t a_order, const void* B, int32_t b_order, int64_t slots, int64_t K, int64_t N, int64_t R,
                                  int64_t P, void* a_down, void* a_up, void* b_down, void* b_up, hipStream_t stream) {
  if (!size_ok(K) || !size_ok(N) || !rank_ok(R, P) || slots < 1 || slots > 65535)
    return set_error(PQ_ESHAPE, "pq_adapter_factors: %lld adapters, K=%lld N=%lld R=%lld P=%lld", (long long)slots, (long long)K, (long long)N,
                     (long long)R, (long long)P);
  if (a_order < 0 || a_order > PQ_ADAPTER_UP || b_order < 0 || b_order > PQ_ADAPTER_UP)
    return set_error(PQ_EINVAL, "pq_adapter_factors: orders %d and %d", a_order, b_order);
  const bool want_a = a_down || a_up, want_b = b_down || b_up;
  if ((want_a && !A) || (want_b && !B)) return set_error(PQ_EINVAL, "pq_adapter_factors: null pointer");
  for (const void* to : {(const void*)a_down, (const void*)a_up, (const void*)b_down, (const void*)b_up, a_order >= PQ_ADAPTER_DOWN ? A : nullptr, b_order >= PQ_ADAPTER_DOWN ? B : nullptr})
    if ((uintptr_t)to % 16) return set_error(PQ_EALIGN, "pq_adapter_factors: orders of `down` and `up` 16-byte aligned");
  if (!want_a && !want_b) return PQ_OK;
  const FactorArgs a{static_cast<const uint16_t*>(A), static_cast<uint16_t*>(a_down), static_cast<uint16_t*>(a_up), (int)K, want_a ? (int)((K + 127) / 128) : 0, a_order};
  const FactorArgs b{static_cast<const uint16_t*>(B), static_cast<uint16_t*>(b_down), static_cast<uint16_t*>(b_up), (int)N, want_b ? (int)((N + 127) / 128) : 0, b_order};
  hipLaunchKernelGGL(adapter_factors_kernel, dim3((unsigned)(a.blocks + b.blocks), (unsigned)slots), dim3(256), 0, stream, a, b, (int)R, (int)P);
  return check_launch("pq_adapter_factors");
}
