// AdamW over every tensor of a model, with moments in 32 or in 8 bits.
//
//   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr wd) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// Parameters are fp32, or bf16 beside an fp32 master that takes the update (a bf16 weight of 1 does not move by less
// than 4e-3).  A bf16 parameter that may have been changed between steps by others is read too (FOLLOW): where it is not what
// the last step left, its master's rounding, the master takes its value.  2 bytes more per parameter (218 M of them: 1112 us instead
// of 1052 with moments of 32 bits, 777 instead of 650 with 8), which a list whose owner changes masters alone does not need.
//
// Moments in 8 bits: blocks of 256 elements of a tensor share an fp32 scale per moment.  The first is e4m3 (largest
// value 448); the second, which is never negative, has the upper byte of a positive fp16 number without its sign: 5
// bits of exponent, 3 of mantissa, largest value 61440.  A rounding, up or down, moves m by less than 12.5 % over a range of 2^14.8
// and sqrt(v) by less than 6.3 % over one of 2^15; below those the codes are evenly spaced.  With beta2 = 0.999 an average moves by a thousandth of itself in a step, which rounding to nearest would
// lose for good, so values are rounded up or down at random in proportion to the distance; 16 random bits each, from a
// hash of (seed, step, tensor, element), so that a run can be repeated.  A second moment never falls to zero in a block
// that holds anything: its smallest code stands for 2^-33 of the block's largest value, and |m| / sqrt(v) stays bounded
// by that of the largest elements (the first moment's smallest code is 2^-17.8 of its largest).  A block with a NaN or an
// infinity gets a scale that is one: all of its moments read as NaN or infinity from then on.
// m and v are computed with one rounding per operation, as the formula reads, so that the codes depend on nothing else;
// the parameters are updated from the moments before they are rounded to 8 bits.
//
// The list of tensors travels in the launch's parameters: nothing is kept on the device that could go stale, and a launch
// can be recorded.
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = GC_ADAMW_BLOCK;          // elements that share a scale: one warp, 8 per lane
constexpr int kChunk = kThreads / 32 * kBlock;  // elements of a CTA's pass
static_assert(kBlock == 256, "a warp holds a block, 8 elements per lane");

using bf16 = __nv_bfloat16;

// What an entry of the list points at: gradient, moments, fp32 parameter; beside bf16 parameters those; scales of 8-bit
// moments.  Launch parameters hold up to 32,764 bytes; most models need far fewer than fit.
enum Role { kG, kM, kV, kMaster };
template <int BITS, bool MIXED>
struct Layout {
  [[maybe_unused]] static constexpr int kP16 = 4, kMs = 4 + MIXED, kVs = 5 + MIXED;
  static constexpr int kArrays = 4 + MIXED + (BITS == 8 ? 2 : 0);
  static constexpr int kMany = 31000 / (8 * kArrays + 13);
};
constexpr int kFew = 48;
template <int ARRAYS, int MAX>
struct List {
  void* at[ARRAYS][MAX];
  int64_t n[MAX];
  int32_t first_chunk[MAX + 1];  // prefix sum of ceil(n / kChunk)
  uint8_t vec[MAX];              // every array is aligned for vector accesses
  int count, first_tensor;       // first_tensor: tensors of earlier launches of the same step
};

struct Hyper {
  double lr, beta1, beta2;
  float b1, w1, b2, w2, eps, keep;  // w = 1 - b, keep = 1 - lr wd, each rounded once from the doubles
  uint32_t seed;
  int advance;  // the step's last launch: counts it
};

// The finalizer of MurmurHash3 (public domain): every input bit reaches every output bit.
__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x85EBCA6Bu;
  x = (x ^ (x >> 13)) * 0xC2B2AE35u;
  return x ^ (x >> 16);
}

// Four elements from `at` on.  FAST: all of them exist, in one access; else those beyond n are zeros.
template <bool FAST, class T>
__device__ __forceinline__ void load4(const void* base, int64_t at, int64_t n, T (&v)[4]) {
  struct alignas(4 * sizeof(T)) V { T v[4]; };
  const T* p = static_cast<const T*>(base) + at;
  if constexpr (FAST) {
    const V t = *reinterpret_cast<const V*>(p);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = t.v[k];
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = at + k < n ? p[k] : T(0.f);
  }
}
// Stores that the L2 gives up first: nothing is read again before the next step (82 M parameters in 394 us, with plain stores
// 402).
template <bool FAST, class T>
__device__ __forceinline__ void store4(void* base, int64_t at, int64_t n, const T (&v)[4]) {
  struct alignas(4 * sizeof(T)) V { T v[4]; };
  T* p = static_cast<T*>(base) + at;
  if constexpr (FAST) {
    V t;
#pragma unroll
    for (int k = 0; k < 4; ++k) t.v[k] = v[k];
    using W = std::conditional_t<sizeof(V) == 16, uint4, uint2>;
    static_assert(sizeof(V) == sizeof(W), "four elements of 4 or 2 bytes");
    __stcs(reinterpret_cast<W*>(p), *reinterpret_cast<const W*>(&t));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at + k < n) p[k] = v[k];
  }
}
// Four codes as one word.
template <bool FAST>
__device__ __forceinline__ uint32_t load_codes(const void* base, int64_t at, int64_t n) {
  const uint8_t* p = static_cast<const uint8_t*>(base) + at;
  if constexpr (FAST) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (at + k < n) w |= uint32_t(p[k]) << (8 * k);
  return w;
}
// (the lowest bytes of q)
template <bool FAST>
__device__ __forceinline__ void store_codes(void* base, int64_t at, int64_t n, const uint32_t (&q)[4]) {
  uint8_t* p = static_cast<uint8_t*>(base) + at;
  if constexpr (FAST) {
    *reinterpret_cast<uint32_t*>(p) = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at + k < n) p[k] = uint8_t(q[k]);
  }
}
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __bfloat162float(x); }

// The scale of a block whose largest |value| has these bits, and what values are multiplied by.  A scale that would be
// subnormal: a block of zeros.
__device__ __forceinline__ float2 scale_of(uint32_t top_bits, float top_code) {
  const float s = __fmul_rn(__uint_as_float(top_bits), top_code);
  if (s < 1.17549435e-38f) return make_float2(0.f, 0.f);
  return make_float2(s, __frcp_rn(s));
}
// To a code of 3 bits of mantissa and an exponent of bias BIAS: u (16 bits) is added below the last kept bit and the rest
// cut off.  Floats and integers are taken from each other's bits here: conversion instructions run at an eighth of the rate.
// Normal numbers: the result, of either sign, is in bits 20 to 26 (30), with the sign in bit 31.  None rounds up beyond the largest
// code: what is left of the largest value's own mantissa is an error of 3 units at most, and 16 would carry.
template <int BIAS>
__device__ __forceinline__ uint32_t round_normal(float t, uint32_t u_by_16) {
  return __float_as_uint(t) + u_by_16 - ((127u - BIAS) << 23);
}
// Any t >= 0.  Below the smallest normal number the grid is even, and the sum is formed in units of it.
template <int BIAS>
constexpr float kLowest = BIAS == 7 ? 0x1p-6f : 0x1p-14f;
template <int BIAS>
__device__ __forceinline__ uint32_t round_code(float t, uint32_t u) {
  constexpr float kUnits = BIAS == 7 ? 0x1p9f : 0x1p17f;
  const uint32_t high = round_normal<BIAS>(t, u << 4) >> 20;
  const float fraction = __uint_as_float(0x3F800000u | (u << 7)) - 1.0f;  // u / 2^16
  const uint32_t low = __float_as_uint(__fadd_rd(__fmaf_rn(t, kUnits, fraction), 0x1p23f)) & 0xFFu;  // towards zero
  return t < kLowest<BIAS> ? low : high;
}

// Four codes of a word as values.
__device__ __forceinline__ void decode_m(uint32_t q, float s, float (&x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(uint16_t(q >> (8 * k)), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    x[k] = __fmul_rn(f.x, s);
    x[k + 1] = __fmul_rn(f.y, s);
  }
}
__device__ __forceinline__ void decode_v(uint32_t q, float s, float (&x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    const uint32_t w = __byte_perm(q, 0, k ? 0x4342 : 0x4140) << 7;  // two fp16 numbers
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    x[k] = __fmul_rn(f.x, s);
    x[k + 1] = __fmul_rn(f.y, s);
  }
}

// The tensor that a chunk belongs to, the last whose first chunk is not beyond it; k is that of an earlier chunk.
template <class L>
__device__ __forceinline__ int tensor_of(const L& tl, int chunk, int k) {
  if (chunk < tl.first_chunk[k + 1]) return k;
  int lo = k + 1, hi = tl.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (tl.first_chunk[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The step's scalars, by two threads while the CTA's first loads are on their way, in double, as Python would form them.
struct Scalars {
  float step_size, inv_bc2;
  uint32_t key;
};
__device__ __forceinline__ void form_scalars(const Hyper& hp, unsigned long long step, Scalars& out) {
  const int warp = threadIdx.x / 32;
  if (threadIdx.x % 32 != 0 || warp >= 2) return;
  const double rest = 1.0 - pow(warp ? hp.beta2 : hp.beta1, double(step + 1ull));
  if (warp) {
    out.inv_bc2 = float(1.0 / sqrt(rest));
  } else {
    out.step_size = float(hp.lr / rest);
    out.key = mix(hp.seed + uint32_t(step + 1ull) * 0x9E3779B9u);
  }
}
// state[0] = steps taken so far (read by every CTA before it counts itself in state[1]); of the step's last launch the
// CTA that arrives last writes the new count and clears the counter.
__device__ __forceinline__ unsigned long long read_step(const unsigned long long* state) {
  return *reinterpret_cast<const volatile unsigned long long*>(state);
}
__device__ __forceinline__ void count_step(const Hyper& hp, unsigned long long step, unsigned long long* state) {
  if (!hp.advance) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const unsigned long long arrived = atomicAdd(state + 1, 1ull);
    if (arrived == gridDim.x - 1) {
      state[1] = 0ull;
      state[0] = step + 1ull;
    }
  }
}

// Masters of four parameters: their own values, or the parameters' where those are no longer what was rounded from them (compared two
// at a time, and nearly always equal).
__device__ __forceinline__ void follow(float (&master)[4], const bf16 (&p)[4]) {
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(master[k], master[k + 1]);
    const uint32_t left = *reinterpret_cast<const uint32_t*>(&t);
    const uint32_t now = __bfloat16_as_ushort(p[k]) | uint32_t(__bfloat16_as_ushort(p[k + 1])) << 16;
    if (left != now) {
      if ((left ^ now) & 0xFFFFu) master[k] = __bfloat162float(p[k]);
      if ((left ^ now) >> 16) master[k + 1] = __bfloat162float(p[k + 1]);
    }
  }
}

// One element: moments as the formula reads, one rounding per operation; the parameter from them.  The quotient may be off
// by 2^-21 of the update (approximate root and division: the exact ones take half of an element's instructions).  What is
// added to v, the smallest normal number, is a root of 1.1e-19: it stands for the subnormal ones, which the fast
// instructions take for zero.
__device__ __forceinline__ void update(const Hyper& hp, const Scalars& sc, float g, float& m, float& v, float& p) {
  m = __fadd_rn(__fmul_rn(m, hp.b1), __fmul_rn(g, hp.w1));
  v = __fadd_rn(__fmul_rn(v, hp.b2), __fmul_rn(__fmul_rn(g, g), hp.w2));
  float root;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"(v + 1.17549435e-38f));
  float inverse;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(root * sc.inv_bc2 + hp.eps));
  p = p * hp.keep - sc.step_size * (m * inverse);
}

// Moments of 32 bits.  Bound by memory: 28 bytes per parameter (82 M of them in 394 us, 5.8 TB/s).  A thread takes 4 elements of
// a pass, all of whose loads are under way before the first is used; 6 CTAs per SM.
template <class TP, bool FOLLOW, int MAX>
__global__ void __launch_bounds__(kThreads, 6)
adamw_kernel(const __grid_constant__ List<Layout<32, sizeof(TP) == 2>::kArrays, MAX> tl, const __grid_constant__ Hyper hp,
             unsigned long long* __restrict__ state) {
  constexpr bool kMixed = sizeof(TP) == 2;
  __shared__ Scalars sc_s;
  const int total = 2 * tl.first_chunk[tl.count];  // half a chunk per pass
  float pv[4], mv[4], vv[4];
  TP gv[4];
  [[maybe_unused]] bf16 old[4];
  int k = 0;
  int64_t at = 0, n = 0;
  bool fast = false;
  auto load = [&](int pass) {
    k = tensor_of(tl, pass / 2, k);
    n = tl.n[k];
    at = int64_t(pass - 2 * tl.first_chunk[k]) * (kChunk / 2) + threadIdx.x * 4;
    fast = tl.vec[k] && at + 4 <= n;
    auto all = [&](auto f) {
      constexpr bool F = decltype(f)::value;
      load4<F>(tl.at[kMaster][k], at, n, pv);
      load4<F>(tl.at[kG][k], at, n, gv);
      load4<F>(tl.at[kM][k], at, n, mv);
      load4<F>(tl.at[kV][k], at, n, vv);
      if constexpr (FOLLOW) load4<F>(tl.at[Layout<32, kMixed>::kP16][k], at, n, old);
    };
    if (fast) all(std::true_type{});
    else all(std::false_type{});
  };
  int pass = blockIdx.x;
  unsigned long long step = read_step(state);
  if (pass < total) load(pass);
  form_scalars(hp, step, sc_s);
  __syncthreads();
  const Scalars sc = sc_s;
  while (pass < total) {
    if constexpr (FOLLOW) follow(pv, old);
#pragma unroll
    for (int e = 0; e < 4; ++e) update(hp, sc, to_f32(gv[e]), mv[e], vv[e], pv[e]);
    auto all = [&](auto f) {
      constexpr bool F = decltype(f)::value;
      store4<F>(tl.at[kMaster][k], at, n, pv);
      store4<F>(tl.at[kM][k], at, n, mv);
      store4<F>(tl.at[kV][k], at, n, vv);
      if constexpr (kMixed) {
        const bf16 p16[4] = {__float2bfloat16_rn(pv[0]), __float2bfloat16_rn(pv[1]), __float2bfloat16_rn(pv[2]),
                             __float2bfloat16_rn(pv[3])};
        store4<F>(tl.at[Layout<32, kMixed>::kP16][k], at, n, p16);
      }
    };
    if (fast) all(std::true_type{});
    else all(std::false_type{});
    pass += gridDim.x;
    if (pass < total) load(pass);
  }
  count_step(hp, step, state);
}

// Moments of 8 bits.  A warp takes a block of 256 elements, a lane two runs of 4.  16 bytes per mixed parameter, of which 218 M
// take 667 us (5.2 TB/s): some 60 instructions to an element share the issue slots with the loads.  4 CTAs per SM hide more of
// these than 3 (694 us) and than 2 that read a chunk ahead (764).
template <class TP, bool FOLLOW, int MAX>
__global__ void __launch_bounds__(kThreads, 4)
adamw_8bit_kernel(const __grid_constant__ List<Layout<8, sizeof(TP) == 2>::kArrays, MAX> tl,
                  const __grid_constant__ Hyper hp, unsigned long long* __restrict__ state) {
  constexpr bool kMixed = sizeof(TP) == 2;
  using L = Layout<8, kMixed>;
  __shared__ Scalars sc_s;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int total = tl.first_chunk[tl.count];
  float pv[2][4];
  TP gv[2][4];
  [[maybe_unused]] bf16 old[2][4];
  uint32_t mq[2], vq[2];
  float ms = 0.f, vs = 0.f;
  int k = 0;
  int64_t at = 0, n = 0;
  bool fast = false;
  auto load = [&](int chunk) {
    k = tensor_of(tl, chunk, k);
    n = tl.n[k];
    const int64_t block = int64_t(chunk - tl.first_chunk[k]) * (kChunk / kBlock) + warp;
    at = block * kBlock + lane * 4;
    fast = tl.vec[k] && (block + 1) * kBlock <= n;
    auto all = [&](auto f) {
      constexpr bool F = decltype(f)::value;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        load4<F>(tl.at[kMaster][k], at + j * 128, n, pv[j]);
        load4<F>(tl.at[kG][k], at + j * 128, n, gv[j]);
        mq[j] = load_codes<F>(tl.at[kM][k], at + j * 128, n);
        vq[j] = load_codes<F>(tl.at[kV][k], at + j * 128, n);
        if constexpr (FOLLOW) load4<F>(tl.at[L::kP16][k], at + j * 128, n, old[j]);
      }
      if (F || block * kBlock < n) {
        ms = static_cast<const float*>(tl.at[L::kMs][k])[block];
        vs = static_cast<const float*>(tl.at[L::kVs][k])[block];
      }
    };
    if (fast) all(std::true_type{});
    else all(std::false_type{});
  };
  int chunk = blockIdx.x;
  const unsigned long long step = read_step(state);
  if (chunk < total) load(chunk);
  form_scalars(hp, step, sc_s);
  __syncthreads();
  const Scalars sc = sc_s;
  while (chunk < total) {
    auto all = [&](auto f) {
      constexpr bool F = decltype(f)::value;
      float m[2][4], v[2][4];
      uint32_t top_m = 0, top_v = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        decode_m(mq[j], ms, m[j]);
        decode_v(vq[j], vs, v[j]);
        if constexpr (FOLLOW) follow(pv[j], old[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          update(hp, sc, to_f32(gv[j][e]), m[j][e], v[j][e], pv[j][e]);
          if (!F && at + j * 128 + e >= n) m[j][e] = v[j][e] = 0.f;  // beyond the tensor
          top_m = max(top_m, __float_as_uint(m[j][e]) & 0x7FFFFFFFu);  // a NaN is above infinity and stays
          top_v = max(top_v, __float_as_uint(v[j][e]));  // never negative
        }
        store4<F>(tl.at[kMaster][k], at + j * 128, n, pv[j]);
        if constexpr (kMixed) {
          const bf16 p16[4] = {__float2bfloat16_rn(pv[j][0]), __float2bfloat16_rn(pv[j][1]), __float2bfloat16_rn(pv[j][2]),
                               __float2bfloat16_rn(pv[j][3])};
          store4<F>(tl.at[L::kP16][k], at + j * 128, n, p16);
        }
      }
      const float2 sm = scale_of(__reduce_max_sync(0xFFFFFFFFu, top_m), 1.0f / 448.0f);
      const float2 sv = scale_of(__reduce_max_sync(0xFFFFFFFFu, top_v), 1.0f / 61440.0f);
      if (lane == 0) {
        static_cast<float*>(tl.at[L::kMs][k])[at / kBlock] = sm.x;
        static_cast<float*>(tl.at[L::kVs][k])[at / kBlock] = sv.x;
      }
      const uint32_t key = mix(sc.key + uint32_t(tl.first_tensor + k)) + uint32_t(at);
      bool normal = true;  // of nearly all blocks: no value below the smallest normal code, no NaN
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          m[j][e] = __fmul_rn(m[j][e], sm.y);
          v[j][e] = __fmul_rn(v[j][e], sv.y);
          normal = normal && fabsf(m[j][e]) >= kLowest<7> && v[j][e] >= kLowest<15>;
        }
      const bool all_normal = __all_sync(0xFFFFFFFFu, normal);
      const uint32_t least = sv.x > 0.f ? 1u : 0u;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t qm[4], qv[4];
        if (all_normal) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t r = mix(key + uint32_t(j * 128 + e));
            const uint32_t c = round_normal<7>(m[j][e], (r << 4) & 0xFFFF0u);
            qm[e] = ((c >> 20) & 0x7Fu) | ((c >> 24) & 0x80u);
            qv[e] = round_normal<15>(v[j][e], (r >> 12) & 0xFFFF0u) >> 20;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t r = mix(key + uint32_t(j * 128 + e));
            qm[e] = min(round_code<7>(fabsf(m[j][e]), r & 0xFFFFu), 0x7Eu) | (__float_as_uint(m[j][e]) >> 31 << 7);
            qv[e] = max(min(round_code<15>(v[j][e], r >> 16), 0xF7u), least);
          }
        }
        store_codes<F>(tl.at[kM][k], at + j * 128, n, qm);
        store_codes<F>(tl.at[kV][k], at + j * 128, n, qv);
      }
    };
    if (fast) all(std::true_type{});
    else if (at - lane * 4 < n) all(std::false_type{});  // uniform in the warp
    chunk += gridDim.x;
    if (chunk < total) load(chunk);
  }
  count_step(hp, step, state);
}

// The values of 8-bit moments, into the fp32 tensors at kG (first) and kMaster (second); scales as for 8 bits and fp32
// parameters.  A chunk per CTA.
template <int MAX>
__global__ void __launch_bounds__(kThreads)
adamw_moments_kernel(const __grid_constant__ List<Layout<8, false>::kArrays, MAX> tl) {
  using L = Layout<8, false>;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, chunk = blockIdx.x;
  const int k = tensor_of(tl, chunk, 0);
  const int64_t n = tl.n[k], block = int64_t(chunk - tl.first_chunk[k]) * (kChunk / kBlock) + warp;
  if (block * kBlock >= n) return;
  const int64_t at = block * kBlock + lane * 4;
  auto all = [&](auto f) {
    constexpr bool F = decltype(f)::value;
    uint32_t qm[2], qv[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      qm[j] = load_codes<F>(tl.at[kM][k], at + j * 128, n);
      qv[j] = load_codes<F>(tl.at[kV][k], at + j * 128, n);
    }
    const float ms = static_cast<const float*>(tl.at[L::kMs][k])[block];
    const float vs = static_cast<const float*>(tl.at[L::kVs][k])[block];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float m[4], v[4];
      decode_m(qm[j], ms, m);
      decode_v(qv[j], vs, v);
      store4<F>(tl.at[kG][k], at + j * 128, n, m);
      store4<F>(tl.at[kMaster][k], at + j * 128, n, v);
    }
  };
  if (tl.vec[k] && (block + 1) * kBlock <= n) all(std::true_type{});
  else all(std::false_type{});
}

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Host arrays in the order of a layout, the bytes that four elements of each take (0: scales, which have no say in whether
// accesses are vectors), and the sizes.
struct Arrays {
  const void* const* at[7];
  int unit[7];
  const int64_t* n;
};
// Fills the list with tensors from `from` on, as many as fit; returns the first that does not.
template <int ARRAYS, int MAX>
int fill(List<ARRAYS, MAX>& tl, const Arrays& a, int from, int n_tensors) {
  tl.count = 0;
  tl.first_tensor = from;
  tl.first_chunk[0] = 0;
  int i = from;
  for (; i < n_tensors && tl.count < MAX; ++i) {
    const int k = tl.count;
    const int64_t chunks = gc::ceil_div(a.n[i], kChunk);
    if (int64_t(tl.first_chunk[k]) + chunks > 0x3F000000) break;
    bool vec = true;
    for (int r = 0; r < ARRAYS; ++r) {
      tl.at[r][k] = const_cast<void*>(a.at[r][i]);
      vec = vec && (a.unit[r] == 0 || aligned(a.at[r][i], a.unit[r]));
    }
    tl.n[k] = a.n[i];
    tl.vec[k] = vec;
    tl.first_chunk[k + 1] = tl.first_chunk[k] + int32_t(chunks);
    ++tl.count;
  }
  return i;
}

template <int BITS, class TP, bool FOLLOW, int MAX>
int step_lists(const Arrays& a, int n_tensors, Hyper hp, void* state, cudaStream_t st) {
  constexpr int kArrays = Layout<BITS, sizeof(TP) == 2>::kArrays;
  static_assert(sizeof(List<kArrays, MAX>) + sizeof(Hyper) <= 32000, "launch parameters");
  unsigned long long* count = static_cast<unsigned long long*>(state);
  int from = 0, launches = 0;
  do {
    List<kArrays, MAX> tl;
    const int next = fill(tl, a, from, n_tensors);
    if (next == from && n_tensors > 0) return gc::fail(GC_ERR_UNSUPPORTED, "gc_adamw_step: tensor %d is too large", from);
    hp.advance = next >= n_tensors;
    const int passes = tl.first_chunk[tl.count] * (BITS == 8 ? 1 : 2);
    // as many CTAs as the SMs hold, each over many passes; an empty model still counts the step
    const int blocks = std::max(1, std::min(passes, gc::kNumSMs * (BITS == 8 ? 4 : 6)));
    if constexpr (BITS == 8) adamw_8bit_kernel<TP, FOLLOW, MAX><<<blocks, kThreads, 0, st>>>(tl, hp, count);
    else adamw_kernel<TP, FOLLOW, MAX><<<blocks, kThreads, 0, st>>>(tl, hp, count);
    ++launches;
    from = next;
  } while (from < n_tensors);
  return gc::check_launch("gc_adamw_step", launches);
}
template <int BITS, class TP, bool FOLLOW>
int step(const Arrays& a, int n_tensors, const Hyper& hp, void* state, cudaStream_t st) {
  return n_tensors <= kFew ? step_lists<BITS, TP, FOLLOW, kFew>(a, n_tensors, hp, state, st)
                           : step_lists<BITS, TP, FOLLOW, Layout<BITS, sizeof(TP) == 2>::kMany>(a, n_tensors, hp, state, st);
}
template <int MAX>
int moments(const Arrays& a, int n_tensors, cudaStream_t st) {
  int launches = 0;
  for (int from = 0; from < n_tensors;) {
    List<Layout<8, false>::kArrays, MAX> tl;
    const int next = fill(tl, a, from, n_tensors);
    if (next == from) return gc::fail(GC_ERR_UNSUPPORTED, "gc_adamw_moments_f32: tensor %d is too large", from);
    from = next;
    const int total = tl.first_chunk[tl.count];
    if (total == 0) continue;
    adamw_moments_kernel<MAX><<<total, kThreads, 0, st>>>(tl);
    ++launches;
  }
  return launches ? gc::check_launch("gc_adamw_moments_f32", launches) : GC_OK;
}

}  // namespace

extern "C" {

int gc_adamw_step(int n_tensors, void* const* params, int param_type, const void* const* grads, float* const* masters,
                  void* const* exp_avg, void* const* exp_avg_sq, float* const* exp_avg_scales,
                  float* const* exp_avg_sq_scales, const int64_t* sizes, int state_bits, double lr, double beta1,
                  double beta2, double eps, double weight_decay, uint32_t seed, void* state, void* stream) {
  GC_REQUIRE(state, "gc_adamw_step: null state");
  GC_REQUIRE(n_tensors >= 0, "gc_adamw_step: negative number of tensors");
  GC_REQUIRE(param_type == GC_TYPE_F32 || param_type == GC_TYPE_BF16 || param_type == (GC_TYPE_BF16 | GC_ADAMW_FOLLOW),
             "gc_adamw_step: parameters are fp32 or bf16, and those beside masters may be followed");
  GC_REQUIRE(state_bits == 8 || state_bits == 32, "gc_adamw_step: moments have 8 or 32 bits");
  const bool mixed = param_type != GC_TYPE_F32, eight = state_bits == 8, followed = param_type & GC_ADAMW_FOLLOW;
  GC_REQUIRE(n_tensors == 0 || (params && grads && exp_avg && exp_avg_sq && sizes), "gc_adamw_step: null list");
  GC_REQUIRE(n_tensors == 0 || !mixed || masters, "gc_adamw_step: bf16 parameters need fp32 masters");
  GC_REQUIRE(n_tensors == 0 || !eight || (exp_avg_scales && exp_avg_sq_scales), "gc_adamw_step: 8-bit moments need scales");
  for (int i = 0; i < n_tensors; ++i) {
    GC_REQUIRE(sizes[i] >= 0, "gc_adamw_step: negative size");
    GC_REQUIRE(sizes[i] == 0 || (params[i] && grads[i] && exp_avg[i] && exp_avg_sq[i] && (!mixed || masters[i]) &&
                                 (!eight || (exp_avg_scales[i] && exp_avg_sq_scales[i]))),
               "gc_adamw_step: null pointer in tensor %d", i);
  }
  Hyper hp{lr, beta1, beta2, float(beta1), float(1.0 - beta1), float(beta2), float(1.0 - beta2), float(eps),
           float(1.0 - lr * weight_decay), seed, 0};
  const auto list = [](auto p) { return reinterpret_cast<const void* const*>(p); };
  const int tp = mixed ? 8 : 16, tm = eight ? 4 : 16;
  Arrays a{{grads, list(exp_avg), list(exp_avg_sq), mixed ? list(masters) : list(params)}, {tp, tm, tm, 16}, sizes};
  int r = kMaster + 1;
  if (mixed) a.unit[r] = tp, a.at[r++] = list(params);
  if (eight) {
    a.at[r++] = list(exp_avg_scales);
    a.at[r++] = list(exp_avg_sq_scales);
  }
  const cudaStream_t st = gc::as_stream(stream);
  if (followed) return eight ? step<8, bf16, true>(a, n_tensors, hp, state, st) : step<32, bf16, true>(a, n_tensors, hp, state, st);
  if (mixed) return eight ? step<8, bf16, false>(a, n_tensors, hp, state, st) : step<32, bf16, false>(a, n_tensors, hp, state, st);
  return eight ? step<8, float, false>(a, n_tensors, hp, state, st) : step<32, float, false>(a, n_tensors, hp, state, st);
}

int gc_adamw_moments_f32(int n_tensors, const uint8_t* const* exp_avg, const uint8_t* const* exp_avg_sq,
                         const float* const* exp_avg_scales, const float* const* exp_avg_sq_scales,
                         const int64_t* sizes, float* const* exp_avg_out, float* const* exp_avg_sq_out, void* stream) {
  GC_REQUIRE(n_tensors >= 0, "gc_adamw_moments_f32: negative number of tensors");
  GC_REQUIRE(n_tensors == 0 || (exp_avg && exp_avg_sq && exp_avg_scales && exp_avg_sq_scales && sizes && exp_avg_out &&
                                exp_avg_sq_out),
             "gc_adamw_moments_f32: null list");
  for (int i = 0; i < n_tensors; ++i) {
    GC_REQUIRE(sizes[i] >= 0, "gc_adamw_moments_f32: negative size");
    GC_REQUIRE(sizes[i] == 0 || (exp_avg[i] && exp_avg_sq[i] && exp_avg_scales[i] && exp_avg_sq_scales[i] &&
                                 exp_avg_out[i] && exp_avg_sq_out[i]),
               "gc_adamw_moments_f32: null pointer in tensor %d", i);
  }
  const auto list = [](auto p) { return reinterpret_cast<const void* const*>(p); };
  const Arrays a{{list(exp_avg_out), list(exp_avg), list(exp_avg_sq), list(exp_avg_sq_out), list(exp_avg_scales),
                  list(exp_avg_sq_scales)},
                 {16, 4, 4, 16},
                 sizes};
  const cudaStream_t st = gc::as_stream(stream);
  return n_tensors <= kFew ? moments<kFew>(a, n_tensors, st) : moments<Layout<8, false>::kMany>(a, n_tensors, st);
}

}  // extern "C"
