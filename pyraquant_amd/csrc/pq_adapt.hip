// Low-rank adapters of many requests beside one shared projection (gfx950): with id = ids[m / each] the adapter of row m (none
// unless 0 <= id < slots), s its scale, A [K, R] and B [R, N] its factors,
//   y[m] = base[m] + t[m] B,  t[m] = s x[m] A
//   dt[m] = s dy[m] B^T,  dx[m] = dt[m] A^T,  dA = sum over its rows of x^T dt,  dB = sum over its rows of t^T dy
// Rows without an adapter keep base's bits (dx: zeros), and no row's result depends on another's values or adapter: the
// adapters of a tile of 64 rows are taken one after the other, each with its own rows packed together (`passes`), so a NaN in one
// request or adapter stays there.
//
//   down  part[s][m][r] = sum over slice s of k of x[m, k] f[id][r][k]          (t and dt without the scale; slices are added where
//                                                                                    they are read)
//   up    out[m, c] = base[m, c] + scale[id] sum_r part[m, r] g[id][c][r]
//   sums  the two sums over rows, per adapter, over chunks of the rows, added by `join` in their order
// All sums are fp32. t and dt are taken by the 16-bit matrix instructions in two parts (two_parts), so their rounding shows in no
// result. No atomics: the same bits every time. Bound by memory: 2 R operations for each value that is read.
#include "pq_mx.h"

#include <algorithm>

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

// ---- down ----------------------------------------------------------------------------------------------------------------
// A workgroup takes 64 rows and a slice of k, 128 k a step, 32 for each of its four waves, whose sums are added in LDS. The factor is the
// first operand, so that a lane's sums are of one row and four consecutive ranks.
struct DownArgs {
  const uint16_t *x, *f;
  Ids ids;
  float* part;
  int64_t ldx;
  int M, K, slice;
};

template <int DT, int J, int NS>
__device__ __forceinline__ void down_pass(const DownArgs& p, int id, int row0, int list, int count, v4f* lds) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int k0 = (int)blockIdx.y * p.slice, k1 = min(p.K, k0 + p.slice);
  const uint16_t* x[NS];
  int row[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    row[s] = row0 + __shfl(list, 16 * s + l16);
    x[s] = p.x + (int64_t)min(row[s], p.M - 1) * p.ldx;
  }
  const uint16_t* const f = p.f + ((int64_t)id * (16 * J) + l16) * p.K;
  v4f acc[J][NS] = {};
  for (int k = k0 + wave * 32; k < k1; k += 128) {
    const int at = k + 8 * g, from = min(at, p.K - 8);
    const bool in = at < k1;
    v4i xs[NS], fs[J];
#pragma unroll
    for (int s = 0; s < NS; ++s) xs[s] = *reinterpret_cast<const v4i*>(x[s] + from);
#pragma unroll
    for (int j = 0; j < J; ++j) fs[j] = *reinterpret_cast<const v4i*>(f + (int64_t)(16 * j) * p.K + from);
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) xs[s][e] = in ? xs[s][e] : 0;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) fs[j][e] = in ? fs[j][e] : 0;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int j = 0; j < J; ++j) acc[j][s] = mfma16_16<DT>(fs[j], xs[s], acc[j][s]);
  }
  // wave w adds the tiles (j, s) of those with index % 4 == w; the others' go through LDS
#pragma unroll
  for (int i = 0; i < J * NS; ++i)
    if ((i & 3) != wave) lds[(wave * (J * NS) + i) * 64 + lane] = acc[i / NS][i % NS];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < J * NS; ++i) {
    if ((i & 3) != wave) continue;
    v4f sum = acc[i / NS][i % NS];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const v4f o = lds[((wave ^ w) * (J * NS) + i) * 64 + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += o[e];
    }
    const int s = i % NS, j = i / NS;
    if (16 * s + l16 < count)
      *reinterpret_cast<v4f*>(p.part + ((int64_t)blockIdx.y * p.M + row[s]) * (16 * J) + 16 * j + 4 * g) = sum;
  }
  __syncthreads();
}

template <int DT, int J>
__global__ __launch_bounds__(256) void adapter_down_kernel(const DownArgs p) {
  __shared__ v4f lds[4 * J * 4 * 64];
  const int lane = threadIdx.x & 63, row0 = (int)blockIdx.x * 64;
  const int mine = row0 + lane < p.M ? p.ids.of(row0 + lane) : -1;
  passes(mine, blockIdx.z, gridDim.z > 1, [&](int id, uint64_t match) {
    const int list = packed_rows(match, lane), count = __popcll(match);
    if (count <= 16) down_pass<DT, J, 1>(p, id, row0, list, count, lds);
    else if (count <= 32) down_pass<DT, J, 2>(p, id, row0, list, count, lds);
    else down_pass<DT, J, 4>(p, id, row0, list, count, lds);
  });
}

// ---- up ------------------------------------------------------------------------------------------------------------------
// A workgroup takes 64 rows and `cols` columns, a wave 64 columns a step. The factor is the first operand, its rows in an order in
// which a lane's sums over four tiles are 16 consecutive columns of one row. With rank 16 one instruction takes both parts of t.
struct UpArgs {
  const float *part, *scale;
  const uint16_t* g;
  Ids ids;
  const uint16_t* base;   // BASE; zeros without
  uint16_t* out;
  int64_t ldb, ldo;
  int M, C, R, slices, cols, blocks;   // blocks of columns
};

template <int DT, int P, bool BASE, int NS>
__device__ __forceinline__ void up_pass(const UpArgs& p, int id, int row0, int list, int count, int c_begin, int c_end) {
  constexpr int KS = P == 16 ? 1 : P / 32, PARTS = P == 16 ? 1 : 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const float scale = p.scale[id];
  int row[NS];
  v4i t[NS][KS][PARTS];
  float back[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    row[s] = row0 + __shfl(list, 16 * s + l16);
    float m = 0.0f;
    RankPiece piece[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int r = 32 * k + 8 * (P == 16 ? g & 1 : g);
      const float* at = p.part + (int64_t)min(row[s], p.M - 1) * P + r;
      piece[k].load(at);
      for (int i = 1; i < p.slices; ++i) {
        at += (int64_t)p.M * P;
        RankPiece more;
        more.load(at);
#pragma unroll
        for (int e = 0; e < 8; ++e) piece[k].raw[e >> 2][e & 3] += more.raw[e >> 2][e & 3];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {   // (ranks past R are sums of zeros times x, and may be NaN)
        const float v = piece[k].raw[e >> 2][e & 3] * scale;
        piece[k].raw[e >> 2][e & 3] = r + e < p.R ? v : 0.0f;
      }
      m = fmaxf(m, piece[k].largest());
    }
    back[s] = 1.0f;
    if constexpr (DT == PQ_F16) {   // rows past fp16's end are taken times a power of two
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      const float down = scale_down(__float_as_uint(m));
      back[s] = scale_back(down);
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) piece[k].raw[e >> 2][e & 3] *= down;
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
  const uint16_t* const f = p.g + (int64_t)id * p.C * P + 8 * (P == 16 ? g & 1 : g);
  for (int c0 = c_begin + wave * 64; c0 < c_end; c0 += 256) {
    v4i fs[4][KS];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = min(c0 + 16 * (l16 >> 2) + 4 * u + (l16 & 3), p.C - 1);
#pragma unroll
      for (int k = 0; k < KS; ++k) fs[u][k] = *reinterpret_cast<const v4i*>(f + (int64_t)c * P + 32 * k);
    }
    v4u b[NS][2];
    const int c = c0 + 16 * g;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        b[s][h] = BASE ? *reinterpret_cast<const v4u*>(p.base + (int64_t)min(row[s], p.M - 1) * p.ldb + min(c + 8 * h, p.C - 8)) : v4u{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      v4f acc[4] = {};
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
          for (int u = 0; u < 4; ++u) acc[u] = mfma16_16<DT>(fs[u][k], t[s][k][part], acc[u]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v4u o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const v4f& a = acc[2 * h + (e >> 1)];
          float lo = a[2 * (e & 1)], hi = a[2 * (e & 1) + 1];
          if constexpr (DT == PQ_F16) lo *= back[s], hi *= back[s];
          o[e] = BASE ? pack2<DT>(lo + lo16_to_f32<DT>(b[s][h][e]), hi + hi16_to_f32<DT>(b[s][h][e])) : pack2<DT>(lo, hi);
        }
        if (16 * s + l16 < count && c + 8 * h < p.C) *reinterpret_cast<v4u*>(p.out + (int64_t)row[s] * p.ldo + c + 8 * h) = o;
      }
    }
  }
}

template <int DT, int P, bool BASE>
__global__ __launch_bounds__(256) void adapter_up_kernel(const UpArgs p) {
  const int lane = threadIdx.x & 63, tile = (int)blockIdx.x / p.blocks, row0 = tile * 64;
  const int c_begin = ((int)blockIdx.x - tile * p.blocks) * p.cols, c_end = min(p.C, c_begin + p.cols);
  const int mine = row0 + lane < p.M ? p.ids.of(row0 + lane) : -1;
  passes(mine, blockIdx.z, gridDim.z > 1, [&](int id, uint64_t match) {
    const int list = packed_rows(match, lane), count = __popcll(match);
    if (count <= 16) up_pass<DT, P, BASE, 1>(p, id, row0, list, count, c_begin, c_end);
    else if (count <= 32) up_pass<DT, P, BASE, 2>(p, id, row0, list, count, c_begin, c_end);
    else up_pass<DT, P, BASE, 4>(p, id, row0, list, count, c_begin, c_end);
  });
  if (blockIdx.z || (BASE && p.out == p.base)) return;
  const uint64_t none = __ballot(mine < 0 && row0 + lane < p.M);   // rows without an adapter, 16 at a time, 16 lanes a row
  const int list = packed_rows(none, lane), count = __popcll(none);
  for (int i0 = 0; i0 < count; i0 += 16) {
    const int i = i0 + (threadIdx.x >> 4), row = row0 + __shfl(list, i);
    if (i >= count) continue;
    for (int c = c_begin + (threadIdx.x & 15) * 8; c < c_end; c += 128) {
      v4u v = v4u{0, 0, 0, 0};
      if (BASE) v = *reinterpret_cast<const v4u*>(p.base + (int64_t)row * p.ldb + c);
      *reinterpret_cast<v4u*>(p.out + (int64_t)row * p.ldo + c) = v;
    }
  }
}

// ---- sums over the rows of an adapter ------------------------------------------------------------------------------------
// part[chunk][slot][r][c] = sum over the chunk's rows m of that adapter of v[m, r] z[m, c], v = scale (the sum of `slices` parts). A
// workgroup of four waves takes 128 columns, a chunk of rows and an adapter; of its rows, 64 a step, only steps that hold a row of
// the adapter are read, the next one's on their way into registers meanwhile, with zeros in the place of other adapters' rows.
struct SumArgs {
  const uint16_t* z;
  const float *v, *scale;
  float* part;
  int32_t* used;          // [chunk][slot]: whether part was written
  int64_t ldz;
  int M, C, slices, rows, panels, blocks;   // rows of a chunk (a multiple of 64), panels of 128 columns, blocks: panels * chunks, or 0
};

template <int DT, int P>
__device__ __forceinline__ void row_sums(const SumArgs& p, const Ids& ids, int block, int slot, uint8_t* sz, uint8_t* sv, uint32_t* top) {
  constexpr int TILES = P == 16 ? 1 : P / 32, PITCH = P == 16 ? 64 : P * 2;   // of v's tiles: with P 16, the first part in ranks 0-15, the second in 16-31
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunk = block / p.panels, panel = block - chunk * p.panels;
  const int c0 = panel * 128, s0 = chunk * p.rows, end = min(p.M, s0 + p.rows);
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
  const float scale = p.scale[slot];
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
      if (match >> r & 1) {
        const float* from = p.v + (int64_t)(m0 + r) * P + at % (P / 4) * 4;
        vr[i] = *reinterpret_cast<const v4f*>(from);
        for (int s = 1; s < p.slices; ++s) {
          from += (int64_t)p.M * P;
          const v4f more = *reinterpret_cast<const v4f*>(from);
#pragma unroll
          for (int e = 0; e < 4; ++e) vr[i][e] += more[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) vr[i][e] *= scale;
      }
    }
  };
  auto rank = [&](int j) { return P == 16 ? lane & 15 : 32 * j + (lane & 31); };
  int m0 = next(s0);
  if (panel == 0 && tid == 0) p.used[chunk * ids.slots + slot] = m0 < end;
  if (m0 >= end) return;
  load(m0);
  while (m0 < end) {
    bool far = false;   // some value of v is 2^16 or more (fp16: scale_down); the waves tell each other in top[0 .. 3]
    if constexpr (DT == PQ_F16) {
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < P / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(vr[i][e]));
      const bool any = __ballot(m >= 65536.0f) != 0;
      if (lane == 0) top[wave] = any;
    }
    __syncthreads();
    if constexpr (DT == PQ_F16) {
      const v4u all = *reinterpret_cast<const v4u*>(top);
      far = __builtin_amdgcn_readfirstlane((int)(all[0] | all[1] | all[2] | all[3])) != 0;
      if (far) {   // rare: the largest magnitude of each rank's 64 values, in top[4 ..]
        if (tid < P) top[4 + tid] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < P / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) atomicMax(&top[4 + (i * 256 + tid) % (P / 4) * 4 + e], __float_as_uint(vr[i][e]) & 0x7fffffffu);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < P / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) vr[i][e] *= scale_down(top[4 + (i * 256 + tid) % (P / 4) * 4 + e]);
#pragma unroll
        for (int j = 0; j < TILES; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[j][e] *= scale_down(top[4 + rank(j)]);
      }
    }
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
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const v4i z = read_columns(z_at, 16 * s, wave * 32, lane);
#pragma unroll
      for (int j = 0; j < TILES; ++j) {
        acc[j] = mfma16<DT>(z, read_columns(hi_at, 16 * s, 32 * j, lane), acc[j]);
        if constexpr (P != 16) acc[j] = mfma16<DT>(z, read_columns(lo_at, 16 * s, 32 * j, lane), acc[j]);
      }
    }
    if (DT == PQ_F16 && far) {
#pragma unroll
      for (int j = 0; j < TILES; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[j][e] *= scale_back(scale_down(top[4 + rank(j)]));
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
  __shared__ __attribute__((aligned(16))) uint32_t top[4 + P];
  const bool is_b = (int)blockIdx.x < b.blocks;
  row_sums<DT, P>(is_b ? b : a, ids, (int)blockIdx.x - (is_b ? 0 : b.blocks), blockIdx.y, sz, sv, top);
}

// The chunks' sums in order, rounded: dB [slots, R, N] and dA [slots, K, R].
struct JoinArgs {
  const float* part;
  const int32_t* used;
  uint16_t* out;
  int chunks, C, groups, blocks;   // groups of 64 columns; workgroups (0: not wanted)
};
template <int DT>
__global__ __launch_bounds__(256) void adapter_join_kernel(const JoinArgs b, const JoinArgs a, int slots, int P, int R) {
  const bool is_b = (int)blockIdx.x < b.blocks;
  const JoinArgs p = is_b ? b : a;
  const int block = (int)blockIdx.x - (is_b ? 0 : b.blocks), slot = blockIdx.y;
  const int c = block % p.groups * 64 + (threadIdx.x & 63), r = block / p.groups * 4 + (threadIdx.x >> 6);
  if (c >= p.C || r >= R) return;
  float s = 0.0f;
  for (int i = 0; i < p.chunks; ++i)
    if (p.used[i * slots + slot]) s += p.part[(((int64_t)i * slots + slot) * P + r) * p.C + c];
  p.out[(int64_t)slot * R * p.C + (is_b ? (int64_t)r * p.C + c : (int64_t)c * R + r)] = (uint16_t)f32_to_16_bits<DT>(s);
}

// ---- the factors' orders -------------------------------------------------------------------------------------------------
// A [C, R] or [R, C] of each slot, to [P, C] and [C, P] with zeros past R: 64 columns a workgroup, turned in LDS.
struct FactorArgs {
  const uint16_t* from;
  uint16_t *by_rank, *by_column;   // [P, C], [C, P]
  int C, blocks, ranks_first;
};
__global__ __launch_bounds__(256) void adapter_factors_kernel(const FactorArgs a, const FactorArgs b, int R, int P) {
  __shared__ uint16_t tile[64][66];   // [c][r]; a pitch of 33 words: both directions spread over the banks
  const bool is_a = (int)blockIdx.x < a.blocks;
  const FactorArgs p = is_a ? a : b;
  const int c0 = ((int)blockIdx.x - (is_a ? 0 : a.blocks)) * 64, slot = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint16_t* const from = p.from + (int64_t)slot * R * p.C;
  for (int i = threadIdx.x; i < 64 * P; i += 256) {
    const int c = p.ranks_first ? i & 63 : i / P, r = p.ranks_first ? i >> 6 : i % P;
    uint16_t v = 0;
    if (r < R && c0 + c < p.C) v = from[p.ranks_first ? (int64_t)r * p.C + c0 + c : (int64_t)(c0 + c) * R + r];
    tile[c][r] = v;
  }
  __syncthreads();
  if (p.by_rank && c0 + lane < p.C)
    for (int r = wave; r < P; r += 4) p.by_rank[((int64_t)slot * P + r) * p.C + c0 + lane] = tile[lane][r];
  if (p.by_column)
    for (int i = threadIdx.x; i < 64 * P; i += 256)
      if (c0 + i / P < p.C) p.by_column[((int64_t)slot * p.C + c0) * P + i] = tile[i / P][i % P];
}

// ---- launches --------------------------------------------------------------------------------------------------------------
constexpr int kMostSlices = 16;
int64_t tiles_of(int64_t M) { return (M + 63) / 64; }
// k of a slice: about 1024 workgroups, but 256 k each or more
int slice_of(int64_t M, int64_t K) {
  const int64_t steps = (K + 255) / 256, want = std::min<int64_t>({1024 / std::max<int64_t>(tiles_of(M), 1), steps, (int64_t)kMostSlices});
  const int64_t n = std::max<int64_t>(want, 1);
  return (int)((steps + n - 1) / n * 256);
}
int slices_of(int64_t M, int64_t K) { const int s = slice_of(M, K); return (int)((K + s - 1) / s); }
// Workgroups that share a tile's adapters: 64 where few rows may hold many adapters, else each takes them in turn.
int sharers(int64_t M, int64_t each) { return each < 16 && M <= 1024 ? 64 : 1; }

int64_t chunk_rows(int64_t M, int64_t C, int64_t slots, int64_t P) {
  const int64_t steps = std::max<int64_t>((M + 63) / 64, 1), panels = (C + 127) / 128;
  const int64_t room = std::max<int64_t>(((int64_t)256 << 20) / (slots * P * C * 4), 1);
  const int64_t want = std::min<int64_t>({(384 + panels - 1) / panels, steps, (int64_t)256, room});
  return (steps + want - 1) / want * 64;
}
int chunks_of(int64_t M, int64_t rows) { return (int)std::max<int64_t>((M + rows - 1) / rows, 1); }

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
#define PQ_DOWN(D, PP) hipLaunchKernelGGL((adapter_down_kernel<D, PP / 16>), grid, dim3(256), 0, stream, p)
  PQ_BY_TYPE(PQ_DOWN);
#undef PQ_DOWN
  return check_launch("pq_adapter_down");
}

extern "C" int pq_adapter_up(const float* part, int64_t slices, const float* scale, const void* g, int64_t slots, int64_t C, int64_t R,
                             int64_t P, const void* ids, int32_t id_bits, int64_t each, const void* base, int64_t ldb, void* out,
                             int64_t ldo, int32_t dtype, int64_t M, hipStream_t stream) {
  if (M < 0 || M > (1 << 30) || !size_ok(C) || ldo < C || (base && ldb < C) || !rank_ok(R, P) || slices < 1 || slices > kMostSlices)
    return set_error(PQ_ESHAPE, "pq_adapter_up: M=%lld C=%lld ldb=%lld ldo=%lld R=%lld P=%lld slices=%lld (C a multiple of 8)", (long long)M,
                     (long long)C, (long long)ldb, (long long)ldo, (long long)R, (long long)P, (long long)slices);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_adapter_up: dtype %d", dtype);
  if (const int st = check_ids(ids, id_bits, each, M, slots, "pq_adapter_up")) return st;
  if (M == 0) return PQ_OK;
  if (!part || !scale || !g || !out) return set_error(PQ_EINVAL, "pq_adapter_up: null pointer");
  if ((uintptr_t)part % 16 || (uintptr_t)g % 16 || (uintptr_t)base % 16 || (base && ldb % 8) || (uintptr_t)out % 16 || ldo % 8)
    return set_error(PQ_EALIGN, "pq_adapter_up: operands 16-byte aligned, strides multiples of 8");
  if (base == out && ldb != ldo) return set_error(PQ_ESHAPE, "pq_adapter_up: out is base, with another stride");
  const int64_t tiles = tiles_of(M), steps = (C + 255) / 256;
  const int64_t want = std::min<int64_t>(steps, std::max<int64_t>(2048 / tiles, 1)), each_steps = (steps + want - 1) / want;
  const int blocks = (int)((steps + each_steps - 1) / each_steps);
  const UpArgs p{part, scale, static_cast<const uint16_t*>(g), ids_of(ids, id_bits, each, slots), static_cast<const uint16_t*>(base),
                 static_cast<uint16_t*>(out), ldb, ldo, (int)M, (int)C, (int)R, (int)slices, (int)each_steps * 256, blocks};
  if (const int st = check_grid(tiles * blocks, 256, "pq_adapter_up")) return st;
  const dim3 grid((unsigned)(tiles * blocks), 1, (unsigned)sharers(M, each));
#define PQ_UP(D, PP)                                                                                     \
  do {                                                                                                   \
    if (base) hipLaunchKernelGGL((adapter_up_kernel<D, PP, true>), grid, dim3(256), 0, stream, p);       \
    else hipLaunchKernelGGL((adapter_up_kernel<D, PP, false>), grid, dim3(256), 0, stream, p);           \
  } while (0)
  PQ_BY_TYPE(PQ_UP);
#undef PQ_UP
  return check_launch("pq_adapter_up");
}

static int64_t padded_bytes(int64_t n) { return (n + 255) / 256 * 256; }

extern "C" int64_t pq_adapter_grads_workspace_size(int64_t M, int64_t K, int64_t N, int64_t slots, int64_t P) {
  if (M < 0 || M > (1 << 30) || !size_ok(K) || !size_ok(N) || slots < 1 || slots > 65535 || !rank_ok(1, P)) return 0;
  int64_t bytes = 0;
  for (const int64_t C : {N, K}) {
    const int64_t chunks = chunks_of(M, chunk_rows(M, C, slots, P));
    bytes += padded_bytes(4 * chunks * slots * P * C) + padded_bytes(4 * chunks * slots);
  }
  return bytes;
}

extern "C" int pq_adapter_grads(const void* x, int64_t ldx, const void* dy, int64_t lddy, int32_t dtype, const float* t, int64_t t_slices,
                                const float* dt, int64_t dt_slices, const float* scale, const void* ids, int32_t id_bits, int64_t each,
                                int64_t M, int64_t K, int64_t N, int64_t slots, int64_t R, int64_t P, void* dA, void* dB, void* workspace,
                                int64_t workspace_bytes, hipStream_t stream) {
  if (M < 0 || M > (1 << 30) || !size_ok(K) || !size_ok(N) || (dA && ldx < K) || (dB && lddy < N) || !rank_ok(R, P) ||
      (dB && (t_slices < 1 || t_slices > kMostSlices)) || (dA && (dt_slices < 1 || dt_slices > kMostSlices)))
    return set_error(PQ_ESHAPE, "pq_adapter_grads: M=%lld K=%lld N=%lld R=%lld P=%lld (K and N multiples of 8)", (long long)M, (long long)K,
                     (long long)N, (long long)R, (long long)P);
  if (dtype != PQ_BF16 && dtype != PQ_F16) return set_error(PQ_EDTYPE, "pq_adapter_grads: dtype %d", dtype);
  if (const int st = check_ids(ids, id_bits, each, M, slots, "pq_adapter_grads")) return st;
  if (!dA && !dB) return PQ_OK;
  if (!workspace || !scale || (M && ((dB && (!dy || !t)) || (dA && (!x || !dt))))) return set_error(PQ_EINVAL, "pq_adapter_grads: null pointer");
  if ((dA && ((uintptr_t)x % 16 || ldx % 8 || (uintptr_t)dt % 16)) || (dB && ((uintptr_t)dy % 16 || lddy % 8 || (uintptr_t)t % 16)) ||
      (uintptr_t)workspace % 16)
    return set_error(PQ_EALIGN, "pq_adapter_grads: operands 16-byte aligned, strides multiples of 8");
  if (workspace_bytes < pq_adapter_grads_workspace_size(M, K, N, slots, P))
    return set_error(PQ_ESHAPE, "pq_adapter_grads: workspace of %lld bytes", (long long)workspace_bytes);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  SumArgs sums[2];
  JoinArgs join[2];
  for (int i = 0; i < 2; ++i) {   // dB, dA
    const bool b = i == 0, wanted = b ? dB != nullptr : dA != nullptr;
    const int64_t C = b ? N : K, rows = chunk_rows(M, C, slots, P), chunks = chunks_of(M, rows), panels = (C + 127) / 128, groups = (C + 63) / 64;
    float* const part = reinterpret_cast<float*>(at);
    at += padded_bytes(4 * chunks * slots * P * C);
    int32_t* const used = reinterpret_cast<int32_t*>(at);
    at += padded_bytes(4 * chunks * slots);
    sums[i] = {static_cast<const uint16_t*>(b ? dy : x), b ? t : dt, scale, part, used, b ? lddy : ldx, (int)M, (int)C,
               (int)(b ? t_slices : dt_slices), (int)rows, (int)panels, wanted ? (int)(panels * chunks) : 0};
    join[i] = {part, used, static_cast<uint16_t*>(b ? dB : dA), (int)chunks, (int)C, (int)groups, wanted ? (int)(groups * ((R + 3) / 4)) : 0};
  }
  // (no rows: no adapter has any, and the ids are not read)
  const Ids id = ids_of(ids, id_bits, M ? each : 1, slots);
  if (const int st = check_grid((int64_t)sums[0].blocks + sums[1].blocks, 256, "pq_adapter_grads")) return st;
  if (const int st = check_grid((int64_t)join[0].blocks + join[1].blocks, 256, "pq_adapter_grads")) return st;
  const dim3 grid((unsigned)(sums[0].blocks + sums[1].blocks), (unsigned)slots), joins((unsigned)(join[0].blocks + join[1].blocks), (unsigned)slots);
#define PQ_SUMS(D, PP) hipLaunchKernelGGL((adapter_sums_kernel<D, PP>), grid, dim3(256), 0, stream, sums[0], sums[1], id)
  PQ_BY_TYPE(PQ_SUMS);
#undef PQ_SUMS
  if (dtype == PQ_BF16) hipLaunchKernelGGL(adapter_join_kernel<PQ_BF16>, joins, dim3(256), 0, stream, join[0], join[1], (int)slots, (int)P, (int)R);
  else hipLaunchKernelGGL(adapter_join_kernel<PQ_F16>, joins, dim3(256), 0, stream, join[0], join[1], (int)slots, (int)P, (int)R);
  return check_launch("pq_adapter_grads");
}

extern "C" int pq_adapter_factors(const void* A, const void* B, int64_t slots, int64_t K, int64_t N, int64_t R, int64_t P, void* at, void* ap,
                                  void* bt, void* bp, hipStream_t stream) {
  if (!size_ok(K) || !size_ok(N) || !rank_ok(R, P) || slots < 1 || slots > 65535)
    return set_error(PQ_ESHAPE, "pq_adapter_factors: %lld adapters, K=%lld N=%lld R=%lld P=%lld", (long long)slots, (long long)K, (long long)N,
                     (long long)R, (long long)P);
  const bool want_a = at || ap, want_b = bt || bp;
  if ((want_a && !A) || (want_b && !B)) return set_error(PQ_EINVAL, "pq_adapter_factors: null pointer");
  const FactorArgs a{static_cast<const uint16_t*>(A), static_cast<uint16_t*>(at), static_cast<uint16_t*>(ap), (int)K, want_a ? (int)((K + 63) / 64) : 0, 0};
  const FactorArgs b{static_cast<const uint16_t*>(B), static_cast<uint16_t*>(bp), static_cast<uint16_t*>(bt), (int)N, want_b ? (int)((N + 63) / 64) : 0, 1};
  if (!want_a && !want_b) return PQ_OK;
  hipLaunchKernelGGL(adapter_factors_kernel, dim3((unsigned)(a.blocks + b.blocks), (unsigned)slots), dim3(256), 0, stream, a, b, (int)R, (int)P);
  return check_launch("pq_adapter_factors");
}
