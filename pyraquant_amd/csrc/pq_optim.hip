// AdamW over the tensors of a model in one launch (gfx950), with states in 32 bits or in 8, and the norm of all gradients.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = (1 - lr wd) p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// g is the gradient times min(1, max_norm / (norm + 1e-6)) where a limit is given. Everything is computed in fp32 and rounded to
// the parameter's type once, at the end.
//
// A chunk is 1024 values of one tensor, and one wave's work; a table in memory says which tensor each chunk belongs to, so one
// launch serves thousands of tensors of any sizes. The gradients, whose places change from step to step, come as kernel arguments (448
// to a launch), which a captured graph keeps. Each chunk has a step counter of its own, read and written by its wave alone: no
// wave waits for another, and replays of a graph count on.
//
// States in 8 bits. The states of 128 consecutive values share two exponents. With bits(a) the bits of |a| as fp32, a mean is kept as
// R = (bits(m) + u) >> 20, a root (of the mean of squares) as R = (bits(root) + u) >> 19: 3 and 4 mantissa bits. u is uniform in the bits
// that are cut off, so that R rounds up as often as what it loses says: an average that moves by 1 - b2 of its distance a step
// moves by far less than a grid step (2^-4 of the value against 5e-4), and would stand still if it were rounded to nearest. u is a hash of the
// value's place, the step and a seed; no state beside these. The byte is R - 2^bits (E - 15), E the exponent of the block's largest R,
// and 0 stands for zero: what lies below the grid is zero, but a root that is no zero is at least the grid's first value, so
// that no mean is divided by a root that went to zero before it. A block with an infinity or a NaN is NaN (E 255).
//
// A bf16 value with 8-bit states moves 10 bytes, with 32-bit ones 22, an fp32 value with 8-bit states 16. The latter two are bound by memory (88.2 M bf16
// values with 32-bit states 390 us, 5.0 TB/s; 12.7 M fp32 values 43 us, 4.8). The first takes 243 us for 88.2 M values in a graph (three launches, 89 us each alone)
// where its memory would take 169: a wave loads, computes some 68 instructions a value, and stores, one chunk after the other.
#include "pq_common.h"

#include <math.h>

namespace pq {
namespace optim {
namespace {

constexpr int kChunk = PQ_ADAMW_CHUNK, kBlock = PQ_ADAMW_BLOCK;
constexpr int kGrads = 448;            // gradients to a launch: 3584 bytes of arguments
constexpr int kGroups = 1024;          // workgroups at most: 4 to a compute unit, which its registers hold, a chunk to a wave
static_assert(kChunk == 1024 && kBlock == 128, "a lane holds two times eight values, 16 lanes a block");

struct Grads {
  const void* at[kGrads];
};

struct StepArgs {
  const pq_adamw_tensor* tensors;
  const int32_t* chunks;               // the tensor of each
  int32_t* steps;
  void *m, *v;
  uint8_t* exps;
  const float* lr_at;                  // the rate in device memory, or NULL
  const double* partials;              // sums of squares, or NULL
  float* norm_out;
  double lr, log_b1, log_b2, decay;
  float b1, b2, b1c, b2c, b1l, eps, max_norm;   // (b1l: what b1c lacks)
  uint32_t seed_key;
  int n_partials, first_tensor, first_chunk, end_chunk;
};

// ---- eight consecutive values of a parameter or a gradient ---------------------------------------------------------------
template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t at, int left, bool wide, float (&x)[8]) {
  if constexpr (DT == PQ_F32) {
    const float* const p = static_cast<const float*>(base) + at;
    if (wide && left >= 8) {
      const v4f a = reinterpret_cast<const v4f*>(p)[0], b = reinterpret_cast<const v4f*>(p)[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = e < left ? p[e] : 0.0f;
    }
  } else {
    const uint16_t* const p = static_cast<const uint16_t*>(base) + at;
    if (wide && left >= 8) {
      const v4u a = *reinterpret_cast<const v4u*>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[2 * e] = lo16_to_f32<DT>(a[e]), x[2 * e + 1] = hi16_to_f32<DT>(a[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = e < left ? lo16_to_f32<DT>(p[e]) : 0.0f;
    }
  }
}
template <int DT, bool NT = false>
__device__ __forceinline__ void store8(void* base, int64_t at, int left, bool wide, const float (&x)[8]) {
  if constexpr (DT == PQ_F32) {
    float* const p = static_cast<float*>(base) + at;
    if (wide && left >= 8) {
      const v4f a = {x[0], x[1], x[2], x[3]}, b = {x[4], x[5], x[6], x[7]};
      if (NT) __builtin_nontemporal_store(a, reinterpret_cast<v4f*>(p)), __builtin_nontemporal_store(b, reinterpret_cast<v4f*>(p) + 1);
      else reinterpret_cast<v4f*>(p)[0] = a, reinterpret_cast<v4f*>(p)[1] = b;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) p[e] = x[e];
    }
  } else {
    uint16_t* const p = static_cast<uint16_t*>(base) + at;
    if (wide && left >= 8) {
      v4u a;
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = pack2<DT>(x[2 * e], x[2 * e + 1]);
      if (NT) __builtin_nontemporal_store(a, reinterpret_cast<v4u*>(p));
      else *reinterpret_cast<v4u*>(p) = a;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) p[e] = (uint16_t)f32_to_16_bits<DT>(x[e]);
    }
  }
}

// ---- the 8-bit states ----------------------------------------------------------------------------------------------------
constexpr uint32_t kPlace = 0x9E3779B1u;
__device__ __forceinline__ uint32_t mixed(uint32_t z) {   // z: the place times kPlace, and the step's key
  z = (z ^ (z >> 15)) * 0x7FB5D329u;
  z = (z ^ (z >> 13)) * 0x4C957F2Bu;
  return z ^ (z >> 16);
}
// the largest of the 16 lanes of a block
__device__ __forceinline__ int block_max(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, false));   // row_ror 1, 2, 4, 8
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, false));
  return max(x, __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false));
}
// Two values' R, bytes and the like as two 16-bit numbers of a word. R is kept 15 exponents up (R + 15 2^bits): no number falls below zero,
// and a difference that would is 0.
__device__ __forceinline__ us2 two(uint32_t w) { return __builtin_bit_cast(us2, w); }
__device__ __forceinline__ us2 both(uint32_t v) { return two(v | v << 16); }
template <int BITS>
__device__ __forceinline__ us2 rounded2(uint32_t a, uint32_t ua, uint32_t b, uint32_t ub) {   // of magnitudes' bits; at most an infinity's
  constexpr uint32_t up = 15u << 23;
  const uint32_t ra = (a + ua + up) >> (23 - BITS), rb = (b + ub + up) >> (23 - BITS);
  return __builtin_elementwise_max(__builtin_elementwise_min(two(ra | rb << 16), both((255u + 15u) << BITS)), both(15u << BITS));   // (u may be -1)
}
// fp32 bits of two bytes (without signs) of a block of exponent E
template <int BITS>
__device__ __forceinline__ us2 widened2(us2 bytes, int E) {
  return (bytes + both((uint32_t)((E - 15) << BITS) & 0xffffu)) * __builtin_elementwise_min(bytes, both(1));   // (0 is zero)
}
struct Moments8 {
  v2u m, root;
  int exps;   // the mean's exponent, then the root's

  __device__ __forceinline__ void load(const StepArgs& p, int64_t at) {
    m = *reinterpret_cast<const v2u*>(static_cast<const uint8_t*>(p.m) + at);
    root = *reinterpret_cast<const v2u*>(static_cast<const uint8_t*>(p.v) + at);
    exps = *reinterpret_cast<const uint16_t*>(p.exps + at / kBlock * 2);
  }
  __device__ __forceinline__ void values(float (&mean)[8], float (&roots)[8]) const {
    const int em = exps & 0xff, er = exps >> 8;
    const uint32_t nan_m = em == 255 ? 0x7fc00000u : 0u, nan_r = er == 255 ? 0x7fc00000u : 0u;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const uint32_t wm = m[e >> 2] >> (e & 2 ? 16 : 0), wr = root[e >> 2];
      const uint32_t am = __builtin_bit_cast(uint32_t, widened2<3>(two(__builtin_amdgcn_perm(0, wm, 0x0c010c00) & 0x007f007fu), em));
      const uint32_t ar = __builtin_bit_cast(uint32_t, widened2<4>(two(__builtin_amdgcn_perm(0, wr, e & 2 ? 0x0c030c02 : 0x0c010c00)), er));
      mean[e] = __uint_as_float(am << 20 | (wm << 24 & 0x80000000u) | nan_m);
      mean[e + 1] = __uint_as_float((am << 4 & 0xfff00000u) | (wm << 16 & 0x80000000u) | nan_m);
      roots[e] = __uint_as_float(ar << 19 | nan_r);
      roots[e + 1] = __uint_as_float((ar << 3 & 0x7ff80000u) | nan_r);
    }
  }
  // the values as they are kept, from magnitudes of roots; add(e, um, ur): what the rounding adds
  template <typename U>
  __device__ __forceinline__ void keep(const float (&mean)[8], const float (&roots)[8], U add) {
    us2 rm[4], rr[4], tm = both(0), tr = both(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t um[2], ur[2];
      add(2 * i, um[0], ur[0]);
      add(2 * i + 1, um[1], ur[1]);
      rm[i] = rounded2<3>(__float_as_uint(mean[2 * i]) & 0x7fffffffu, um[0], __float_as_uint(mean[2 * i + 1]) & 0x7fffffffu, um[1]);
      rr[i] = rounded2<4>(__float_as_uint(roots[2 * i]), ur[0], __float_as_uint(roots[2 * i + 1]), ur[1]);
      tm = __builtin_elementwise_max(tm, rm[i]);
      tr = __builtin_elementwise_max(tr, rr[i]);
    }
    const int em = (block_max(max((int)tm[0], (int)tm[1])) >> 3) - 15, er = (block_max(max((int)tr[0], (int)tr[1])) >> 4) - 15;
    const us2 zero_m = both((uint32_t)em << 3), zero_r = both((uint32_t)er << 4), none = both(15 << 4);
    uint32_t bm[4], br[4];   // two bytes each, in 16 bits
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bm[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(rm[i], zero_m)) | (__float_as_uint(mean[2 * i]) >> 24 & 0x80u) |
              (__float_as_uint(mean[2 * i + 1]) >> 8 & 0x800000u);
      const us2 some = __builtin_elementwise_min(__builtin_elementwise_sub_sat(rr[i], none), both(1));   // (a root that is no zero: at least 1)
      br[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_elementwise_sub_sat(rr[i], zero_r), some));
    }
    m = v2u{__builtin_amdgcn_perm(bm[1], bm[0], 0x06040200), __builtin_amdgcn_perm(bm[3], bm[2], 0x06040200)};
    root = v2u{__builtin_amdgcn_perm(br[1], br[0], 0x06040200), __builtin_amdgcn_perm(br[3], br[2], 0x06040200)};
    exps = em | er << 8;
  }
  __device__ __forceinline__ void store(void* ms, void* roots, uint8_t* ex, int64_t at) const {
    *reinterpret_cast<v2u*>(static_cast<uint8_t*>(ms) + at) = m;
    *reinterpret_cast<v2u*>(static_cast<uint8_t*>(roots) + at) = root;
    if ((threadIdx.x & 15) == 0) *reinterpret_cast<uint16_t*>(ex + at / kBlock * 2) = (uint16_t)exps;
  }
};

__device__ __forceinline__ double wave_sum(double s) {
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  return s;
}

// ---- the step ------------------------------------------------------------------------------------------------------------
struct Rates {   // of one step count
  float size, unbias, keep;   // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr wd
};

template <int DT, bool EIGHT>
__device__ __forceinline__ void step_chunk(const StepArgs& p, void* param, const void* grad, int64_t n, int64_t c0, int64_t base,
                                           const Rates& r, float clip, uint32_t key, int lane) {
  const bool wide_p = (uintptr_t)param % 16 == 0, wide_g = (uintptr_t)grad % 16 == 0;
  float x[2][8], g[2][8], m[2][8], v[2][8];
  Moments8 s[2];
  int left[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t at = c0 + i * 512 + lane * 8;
    left[i] = (int)max((int64_t)-1024, min(n - at, (int64_t)8));
    if (at - at % kBlock >= n) continue;   // (the whole block is behind the end: 16 lanes as one)
    if constexpr (EIGHT) {
      s[i].load(p, base + at);
    } else {
      load8<PQ_F32>(p.m, base + at, 8, true, m[i]);
      load8<PQ_F32>(p.v, base + at, 8, true, v[i]);
    }
    load8<DT>(param, at, left[i], wide_p, x[i]);
    load8<DT>(grad, at, left[i], wide_g, g[i]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t at = c0 + i * 512 + lane * 8;
    if (at - at % kBlock >= n) continue;
    float root[8];
    if constexpr (EIGHT) {
      s[i].values(m[i], v[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] *= v[i][e];
    }
    uint32_t least = ~0u;   // of the squares that are no zeros (bits - 1)
    int past[8] = {};       // -1 where the exact mean's magnitude lies below m's
    if (EIGHT && p.b1c <= 0.5f && p.b2c <= 0.5f) {
      // b m + (1 - b) d as m + (1 - b) (d - m), in few roundings: b in fp32 is off by as much as half a step itself. What is cut to 8 bits next goes by the
      // exact mean: where this one was rounded up, and that may be to a border of the grid, by the number below it. (The step of 88 M bf16 values 290 ->
      // 300 us, of 12.7 M fp32 values 41 -> 43; a half to a third as many means fall to another step of the grid than the exact one, and fewer than from
      // elementary operations in fp32.)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = g[i][e] * clip, w = fmaf(d, d, -v[i][e]), before = m[i][e], q = d - before;
        m[i][e] = fmaf(q, p.b1c, before);
        float lacks = fmaf(q, p.b1c, before - m[i][e]);
        if constexpr (DT == PQ_F32) lacks = fmaf((d - q) - before, p.b1c, fmaf(q, p.b1l, lacks));   // (and what q and 1 - b lack)
        past[e] = fmaf(m[i][e], 0x1p-27f, lacks) * m[i][e] < 0.0f ? -1 : 0;   // (less than 1 / 16 is what lacks itself may be off; of an infinity it is NaN)
        v[i][e] = fmaf(w, p.b2c, v[i][e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = g[i][e] * clip;
        m[i][e] = fmaf(d, p.b1c, m[i][e] * p.b1);
        v[i][e] = fmaf(d * d, p.b2c, v[i][e] * p.b2);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; e += 2) least = min(least, min(__float_as_uint(v[i][e]) - 1, __float_as_uint(v[i][e + 1]) - 1));
    // The instructions for roots and reciprocals are within 1 of the last place, but take subnormal numbers for zeros: with 8-bit states (the step of 88 M
    // bf16 values, its states' values read out, 488 us with the exact ones, 12 and 10 instructions, and 430 with these) those are taken where a square of
    // the wave's is below 2^-96, or eps is. 32-bit states always take them, so that no value's last bit depends on its neighbours' (88 M bf16 values 390
    // us for 394, 0.1 M 5.7 for 5.2).
    if (!EIGHT || __ballot(least < 0x0f7fffffu) || p.eps < 0x1p-96f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        root[e] = fabsf(sqrtf(v[i][e]));   // (a NaN may have a sign)
        x[i][e] = x[i][e] * r.keep - r.size * m[i][e] / fmaf(root[e], r.unbias, p.eps);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        root[e] = __builtin_amdgcn_sqrtf(fabsf(v[i][e]));
        x[i][e] = fmaf(-r.size * m[i][e], __builtin_amdgcn_rcpf(fmaf(root[e], r.unbias, p.eps)), x[i][e] * r.keep);
      }
    }
    store8<DT>(param, at, left[i], wide_p, x[i]);
    if constexpr (EIGHT) {
      const uint32_t place = (uint32_t)(base + at) * kPlace + key;
      s[i].keep(m[i], root, [&](int e, uint32_t& um, uint32_t& ur) {
        const uint32_t h = mixed(place + e * kPlace);
        um = ((h & 0xffffu) << 4) + (uint32_t)past[e];
        ur = (h >> 16) << 3;
      });
      s[i].store(p.m, p.v, p.exps, base + at);
    } else {
      store8<PQ_F32>(p.m, base + at, 8, true, m[i]);
      store8<PQ_F32>(p.v, base + at, 8, true, v[i]);
    }
  }
}

template <bool EIGHT>
__global__ __launch_bounds__(256) void adamw_step_kernel(const StepArgs p, const Grads grads) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float clip = 1.0f;
  if (p.partials) {
    double sum = 0.0;
    for (int i = lane; i < p.n_partials; i += 64) sum += p.partials[i];
    const float norm = (float)sqrt(wave_sum(sum));
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.norm_out = norm;
    if (!(norm < INFINITY)) return;   // (an infinity or a NaN: no parameter, state or count changes)
    clip = fminf(p.max_norm / (norm + 1e-6f), 1.0f);
  }
  const double lr = p.lr_at ? (double)*p.lr_at : p.lr;
  int last = -1;
  Rates r{};
  for (int c = p.first_chunk + (int)blockIdx.x * 4 + wave; c < p.end_chunk; c += (int)gridDim.x * 4) {
    const int at = __builtin_amdgcn_readfirstlane(p.chunks[c]);
    const void* const grad = grads.at[at - p.first_tensor];
    if (!grad) continue;
    const pq_adamw_tensor t = p.tensors[at];
    const int step = __builtin_amdgcn_readfirstlane(p.steps[c]) + 1;
    if (lane == 0) p.steps[c] = step;
    if (step != last) {
      last = step;
      r.size = (float)(lr / (1.0 - exp(step * p.log_b1)));
      r.unbias = (float)(1.0 / sqrt(1.0 - exp(step * p.log_b2)));
      r.keep = (float)(1.0 - lr * p.decay);
    }
    const int64_t c0 = (int64_t)(c - t.first_chunk) * kChunk;
    const uint32_t key = (uint32_t)step * 0x6C8E9CF5u + p.seed_key;
    if (t.dtype == PQ_F32) step_chunk<PQ_F32, EIGHT>(p, t.p, grad, t.n, c0, t.base, r, clip, key, lane);
    else if (t.dtype == PQ_BF16) step_chunk<PQ_BF16, EIGHT>(p, t.p, grad, t.n, c0, t.base, r, clip, key, lane);
    else step_chunk<PQ_F16, EIGHT>(p, t.p, grad, t.n, c0, t.base, r, clip, key, lane);
  }
}

// ---- the sum of all gradients' squares, in 64 bits: one partial sum a workgroup, the order fixed by the sizes ---------------
template <int DT>
__device__ __forceinline__ double squares(const void* grad, int64_t n, int64_t c0, int lane) {
  const bool wide = (uintptr_t)grad % 16 == 0;
  double s = 0.0;
  float g[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t at = c0 + i * 512 + lane * 8;
    load8<DT>(grad, at, (int)max((int64_t)0, min(n - at, (int64_t)8)), wide, g[i]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (double)g[i][e] * (double)g[i][e];
  return s;
}
// (29.5 M bf16 gradients of 420 tensors a launch: 17 us, 3.4 TB/s; they come from memory, with the stores of what ran before them.)
__global__ __launch_bounds__(256) void grad_squares_kernel(const StepArgs p, const Grads grads, double* out) {
  __shared__ double sums[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double s = 0.0;
  for (int c = p.first_chunk + (int)blockIdx.x * 4 + wave; c < p.end_chunk; c += (int)gridDim.x * 4) {
    const int at = __builtin_amdgcn_readfirstlane(p.chunks[c]);
    const void* const grad = grads.at[at - p.first_tensor];
    if (!grad) continue;
    const pq_adamw_tensor t = p.tensors[at];
    const int64_t c0 = (int64_t)(c - t.first_chunk) * kChunk;
    if (t.dtype == PQ_F32) s += squares<PQ_F32>(grad, t.n, c0, lane);
    else if (t.dtype == PQ_BF16) s += squares<PQ_BF16>(grad, t.n, c0, lane);
    else s += squares<PQ_F16>(grad, t.n, c0, lane);
  }
  s = wave_sum(s);
  if (lane == 0) sums[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) out[blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

// Many partial sums in one, in a fixed order.
__global__ __launch_bounds__(1024) void grad_join_kernel(const double* sums, int n, double* out) {
  __shared__ double part[16];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += sums[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) s += part[i];
    *out = s;
  }
}

// ---- states out and in -----------------------------------------------------------------------------------------------------
// Bound by memory: 88.6 M values of 8-bit states to two bf16 tensors 85 us, 6.2 TB/s, their bytes in part from the caches.
template <int DT, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_moments_kernel(const StepArgs p, int64_t n, void* mean, void* root) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at >= n) return;
  float m[8], w[8];
  if constexpr (EIGHT) {
    Moments8 s;
    s.load(p, at);
    s.values(m, w);
  } else {
    load8<PQ_F32>(p.m, at, 8, true, m);
    load8<PQ_F32>(p.v, at, 8, true, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = sqrtf(w[e]);
  }
  store8<DT, true>(mean, at, 8, true, m);   // (past the caches: what they hold is read again before this is. The next step's sums 21 -> 17 us a launch)
  store8<DT, true>(root, at, 8, true, w);
}
template <bool EIGHT>
__global__ __launch_bounds__(256) void adamw_load_kernel(const StepArgs p, int64_t n, const float* mean, const float* root) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at >= n) return;
  float m[8], w[8];
  load8<PQ_F32>(mean, at, 8, true, m);
  load8<PQ_F32>(root, at, 8, true, w);
  if constexpr (EIGHT) {
    Moments8 s;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = fabsf(w[e]);
    s.keep(m, w, [](int, uint32_t& um, uint32_t& ur) { um = 1u << 19, ur = 1u << 18; });   // to nearest
    s.store(p.m, p.v, p.exps, at);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] *= w[e];
    store8<PQ_F32>(p.m, at, 8, true, m);
    store8<PQ_F32>(p.v, at, 8, true, w);
  }
}

int check_states(const pq_adamw_states* s, const char* what) {
  if (!s || (s->n && (!s->m || !s->v || (s->bits == 8 && !s->exps)))) return set_error(PQ_EINVAL, "%s: null pointer", what);
  if (s->bits != 8 && s->bits != 32) return set_error(PQ_EINVAL, "%s: states of %d bits (8 or 32)", what, s->bits);
  if (s->n < 0 || s->n % kBlock || s->n > ((int64_t)1 << 40)) return set_error(PQ_ESHAPE, "%s: %lld values (a multiple of %d)", what, (long long)s->n, kBlock);
  if ((uintptr_t)s->m % 16 || (uintptr_t)s->v % 16 || (uintptr_t)s->exps % 2) return set_error(PQ_EALIGN, "%s: states 16-byte aligned", what);
  return PQ_OK;
}
int check_list(const pq_adamw_list* l, const char* what) {
  if (!l || l->n_tensors < 0) return set_error(PQ_EINVAL, "%s: no list", what);
  if (l->n_tensors > (1 << 30)) return set_error(PQ_ESHAPE, "%s: %lld tensors", what, (long long)l->n_tensors);
  if (l->n_tensors == 0) return PQ_OK;
  if (!l->tensors || !l->chunks || !l->first_chunk || !l->grads) return set_error(PQ_EINVAL, "%s: null pointer", what);
  if (l->first_chunk[0] != 0 || l->first_chunk[l->n_tensors] > (1 << 30))
    return set_error(PQ_ESHAPE, "%s: %lld chunks (2^30 at most, the first 0)", what, (long long)l->first_chunk[l->n_tensors]);
  for (int64_t i = 0; i < l->n_tensors; ++i)
    if (l->first_chunk[i + 1] < l->first_chunk[i]) return set_error(PQ_ESHAPE, "%s: first_chunk falls at %lld", what, (long long)i);
  return PQ_OK;
}

// Calls f(args, grads, workgroups) for each batch of tensors that a launch takes and that has a gradient.
template <typename F>
int batches(const pq_adamw_list* l, StepArgs p, int most, F f) {
  p.tensors = l->tensors;
  p.chunks = l->chunks;
  for (int64_t t = 0; t < l->n_tensors; t += kGrads) {
    const int64_t end = t + kGrads < l->n_tensors ? t + kGrads : l->n_tensors;
    Grads g;
    bool any = false;
    for (int64_t i = t; i < end; ++i) {
      g.at[i - t] = l->grads[i];
      any |= l->grads[i] != nullptr && l->first_chunk[i + 1] > l->first_chunk[i];
    }
    if (!any) continue;
    for (int64_t i = end - t; i < kGrads; ++i) g.at[i] = nullptr;
    p.first_tensor = (int)t;
    p.first_chunk = (int)l->first_chunk[t];
    p.end_chunk = (int)l->first_chunk[end];
    const int groups = (p.end_chunk - p.first_chunk + 3) / 4;
    if (const int st = f(p, g, groups < most ? groups : most)) return st;
  }
  return PQ_OK;
}
constexpr int kPartials = 2048;   // workgroups of a launch that sums squares
}  // namespace
}  // namespace optim
}  // namespace pq

using namespace pq;
using namespace pq::optim;

extern "C" int64_t pq_grad_squares_partials(const pq_adamw_list* list) {
  int64_t n = 0;
  if (check_list(list, "pq_grad_squares_partials") != PQ_OK) return 0;
  if (list->n_tensors) batches(list, StepArgs{}, kPartials, [&](const StepArgs&, const Grads&, int groups) { return n += groups, PQ_OK; });
  return n;
}

extern "C" int pq_grad_squares(const pq_adamw_list* list, double* partials, int64_t n_partials, hipStream_t stream) {
  if (const int st = check_list(list, "pq_grad_squares")) return st;
  const int64_t need = pq_grad_squares_partials(list);
  if (need && !partials) return set_error(PQ_EINVAL, "pq_grad_squares: null pointer");
  if (need > n_partials) return set_error(PQ_ESHAPE, "pq_grad_squares: room for %lld sums (%lld)", (long long)n_partials, (long long)need);
  if (!need) return PQ_OK;
  return batches(list, StepArgs{}, kPartials, [&](const StepArgs& p, const Grads& g, int groups) {
    hipLaunchKernelGGL(grad_squares_kernel, dim3(groups), dim3(256), 0, stream, p, g, partials);
    partials += groups;
    return check_launch("pq_grad_squares");
  });
}

extern "C" int pq_grad_squares_join(const double* partials, int64_t n_partials, double* sum, hipStream_t stream) {
  if (n_partials < 1 || n_partials > (1 << 30)) return set_error(PQ_ESHAPE, "pq_grad_squares_join: %lld sums", (long long)n_partials);
  if (!partials || !sum) return set_error(PQ_EINVAL, "pq_grad_squares_join: null pointer");
  hipLaunchKernelGGL(grad_join_kernel, dim3(1), dim3(1024), 0, stream, partials, (int)n_partials, sum);
  return check_launch("pq_grad_squares_join");
}

extern "C" int pq_adamw_step(const pq_adamw_list* list, const pq_adamw_states* states, const pq_adamw_rates* rates,
                             const double* partials, int64_t n_partials, float* norm, hipStream_t stream) {
  if (const int st = check_list(list, "pq_adamw_step")) return st;
  if (const int st = check_states(states, "pq_adamw_step")) return st;
  if (!rates || (states->n && !states->steps)) return set_error(PQ_EINVAL, "pq_adamw_step: null pointer");
  if (list->n_tensors && list->first_chunk[list->n_tensors] && !states->n) return set_error(PQ_ESHAPE, "pq_adamw_step: no states for the list's values");
  if (!(rates->beta1 >= 0 && rates->beta1 < 1 && rates->beta2 >= 0 && rates->beta2 < 1 && rates->eps >= 0 && rates->weight_decay >= 0) ||
      (!rates->lr_at && !(rates->lr >= 0)))
    return set_error(PQ_EINVAL, "pq_adamw_step: lr %g, betas %g and %g, eps %g, weight decay %g", rates->lr, rates->beta1, rates->beta2,
                     rates->eps, rates->weight_decay);
  if (n_partials < 0 || n_partials > (1 << 30)) return set_error(PQ_ESHAPE, "pq_adamw_step: %lld sums", (long long)n_partials);
  if (n_partials && (!partials || !norm || !(rates->max_norm > 0)))
    return set_error(PQ_EINVAL, "pq_adamw_step: sums of squares come with a limit above 0 and a place for the norm");
  StepArgs p{};
  p.steps = states->steps, p.m = states->m, p.v = states->v, p.exps = states->exps;
  p.lr_at = rates->lr_at, p.lr = rates->lr;
  p.log_b1 = log(rates->beta1), p.log_b2 = log(rates->beta2), p.decay = rates->weight_decay;
  p.b1 = (float)rates->beta1, p.b1c = (float)(1.0 - rates->beta1), p.b1l = (float)(1.0 - rates->beta1 - (double)p.b1c), p.b2 = (float)rates->beta2, p.b2c = (float)(1.0 - rates->beta2);
  p.eps = (float)rates->eps, p.max_norm = (float)rates->max_norm;
  p.partials = n_partials ? partials : nullptr, p.n_partials = (int)n_partials, p.norm_out = norm;
  p.seed_key = rates->seed * 0x5851F42Du;
  return batches(list, p, kGroups, [&](const StepArgs& a, const Grads& g, int groups) {
    if (states->bits == 8) hipLaunchKernelGGL(adamw_step_kernel<true>, dim3(groups), dim3(256), 0, stream, a, g);
    else hipLaunchKernelGGL(adamw_step_kernel<false>, dim3(groups), dim3(256), 0, stream, a, g);
    return check_launch("pq_adamw_step");
  });
}

static int moments_grid(int64_t n, dim3& grid, const char* what) {
  const int64_t blocks = (n / 8 + 255) / 256;
  if (const int st = check_grid(blocks, 256, what)) return st;
  grid = dim3((unsigned)blocks);
  return PQ_OK;
}

extern "C" int pq_adamw_moments(const pq_adamw_states* states, void* mean, void* root, int32_t dtype, hipStream_t stream) {
  if (const int st = check_states(states, "pq_adamw_moments")) return st;
  if (dtype != PQ_BF16 && dtype != PQ_F16 && dtype != PQ_F32) return set_error(PQ_EDTYPE, "pq_adamw_moments: dtype %d", dtype);
  if (states->n == 0) return PQ_OK;
  if (!mean || !root) return set_error(PQ_EINVAL, "pq_adamw_moments: null pointer");
  if ((uintptr_t)mean % 16 || (uintptr_t)root % 16) return set_error(PQ_EALIGN, "pq_adamw_moments: results 16-byte aligned");
  StepArgs p{};
  p.m = states->m, p.v = states->v, p.exps = states->exps;
  dim3 grid;
  if (const int st = moments_grid(states->n, grid, "pq_adamw_moments")) return st;
#define PQ_MOMENTS(D)                                                                                                              \
  do {                                                                                                                             \
    if (states->bits == 8) hipLaunchKernelGGL((adamw_moments_kernel<D, true>), grid, dim3(256), 0, stream, p, states->n, mean, root);   \
    else hipLaunchKernelGGL((adamw_moments_kernel<D, false>), grid, dim3(256), 0, stream, p, states->n, mean, root);               \
  } while (0)
  if (dtype == PQ_BF16) PQ_MOMENTS(PQ_BF16);
  else if (dtype == PQ_F16) PQ_MOMENTS(PQ_F16);
  else PQ_MOMENTS(PQ_F32);
#undef PQ_MOMENTS
  return check_launch("pq_adamw_moments");
}

extern "C" int pq_adamw_load(const pq_adamw_states* states, const float* mean, const float* root, hipStream_t stream) {
  if (const int st = check_states(states, "pq_adamw_load")) return st;
  if (states->n == 0) return PQ_OK;
  if (!mean || !root) return set_error(PQ_EINVAL, "pq_adamw_load: null pointer");
  if ((uintptr_t)mean % 16 || (uintptr_t)root % 16) return set_error(PQ_EALIGN, "pq_adamw_load: operands 16-byte aligned");
  StepArgs p{};
  p.m = states->m, p.v = states->v, p.exps = states->exps;
  dim3 grid;
  if (const int st = moments_grid(states->n, grid, "pq_adamw_load")) return st;
  if (states->bits == 8) hipLaunchKernelGGL(adamw_load_kernel<true>, grid, dim3(256), 0, stream, p, states->n, mean, root);
  else hipLaunchKernelGGL(adamw_load_kernel<false>, grid, dim3(256), 0, stream, p, states->n, mean, root);
  return check_launch("pq_adamw_load");
}
