// AdamW over every tensor of a model, with moments in 32 or in 8 bits.
//
//   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr wd) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// Parameters are fp32, or bf16 beside an fp32 master that takes the update (a bf16 weight of 1 does not move by less
// than 4e-3).
//
// Moments in 8 bits: blocks of 256 elements of a tensor share an fp32 scale per moment.  The first is e4m3 (largest
// value 448); the second, which is never negative, has the upper byte of a positive fp16 number without its sign: 5
// bits of exponent, 3 of mantissa, largest value 61440.  Both keep 3 to 6 % at most over a range of 2^17 in |m| and in
// sqrt(v).  With beta2 = 0.999 an average moves by a thousandth of itself in a step, which rounding to nearest would
// lose for good, so values are rounded up or down at random in proportion to the distance; 16 random bits each, from a
// hash of (seed, step, tensor, element), so that a run can be repeated.  A second moment never falls to zero in a block
// that holds anything: its smallest code stands for 2^-33 of the block's largest value, and |m| / sqrt(v) stays bounded
// by that of the largest elements (the first moment's smallest code is 2^-17.8 of its largest).  A block with a NaN or an
// infinity gets a scale that is one: all of its moments read as NaN or infinity from then on.
// m and v are computed with one rounding per operation, as the formula reads, so that the codes depend on nothing else;
// the parameters are updated from the moments before they are rounded to 8 bits.
//
// Bound by memory: 28 bytes per parameter (32 bits), 16 and a sixteenth (8 bits).  A CTA takes chunks of 2048
// elements, a warp 256 of them, a thread two runs of 4: accesses of 16 bytes (4 for codes), of which every thread has all in
// flight before it uses the first.  The list of tensors travels in the launch's parameters: nothing is kept on the device that
// could go stale, and a launch can be recorded.
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
// Tensors of one launch: launch parameters hold up to 32,764 bytes, and most models need far fewer.
constexpr int kFew = 48, kMany = 440;

using bf16 = __nv_bfloat16;

template <int MAX>
struct List {
  void* p[MAX];        // bf16 or fp32 parameters
  float* master[MAX];  // fp32 parameters (p itself where it is fp32)
  const void* g[MAX];
  void* m[MAX];
  void* v[MAX];
  float* ms[MAX];  // scales, 8 bits
  float* vs[MAX];
  int64_t n[MAX];
  int32_t first_chunk[MAX + 1];  // prefix sum of ceil(n / kChunk)
  uint8_t vec[MAX];              // every array is aligned for vector accesses
  int count, first_tensor;       // first_tensor: tensors of earlier launches of the same step
};
static_assert(sizeof(List<kMany>) <= 32000, "launch parameters");

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

// The four elements from `at` on; beyond n: zeros.
template <class T>
__device__ __forceinline__ void load4(const T* base, int64_t at, int64_t n, bool vec, T (&v)[4]) {
  struct alignas(4 * sizeof(T)) V { T v[4]; };
  if (vec && at + 4 <= n) {
    const V t = *reinterpret_cast<const V*>(base + at);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = t.v[k];
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = at + k < n ? base[at + k] : T(0.f);
  }
}
template <class T>
__device__ __forceinline__ void store4(T* base, int64_t at, int64_t n, bool vec, const T (&v)[4]) {
  struct alignas(4 * sizeof(T)) V { T v[4]; };
  if (vec && at + 4 <= n) {
    V t;
#pragma unroll
    for (int k = 0; k < 4; ++k) t.v[k] = v[k];
    *reinterpret_cast<V*>(base + at) = t;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at + k < n) base[at + k] = v[k];
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
// t >= 0 to a code of 3 bits of mantissa and an exponent of bias BIAS: u (16 bits) is added below the last kept bit and
// the rest cut off.  Below the smallest normal number the grid is even, and the sum is formed in units of it.
template <int BIAS>
__device__ __forceinline__ uint32_t round_code(float t, uint32_t u) {
  constexpr float kLowest = BIAS == 7 ? 0x1p-6f : 0x1p-14f, kUnits = BIAS == 7 ? 0x1p9f : 0x1p17f;
  const uint32_t high = ((__float_as_uint(t) + (u << 4)) >> 20) - ((127u - BIAS) << 3);
  const uint32_t low = uint32_t(__fadd_rn(t * kUnits, float(u) * 0x1p-16f));  // towards zero
  return t < kLowest ? low : high;
}

// e4m3 and second-moment codes, four at a time
__device__ __forceinline__ void decode_m(const uint8_t (&q)[4], float s, float (&x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(uint16_t(q[k] | q[k + 1] << 8), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    x[k] = __fmul_rn(f.x, s);
    x[k + 1] = __fmul_rn(f.y, s);
  }
}
__device__ __forceinline__ void decode_v(const uint8_t (&q)[4], float s, float (&x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = __fmul_rn(__half2float(__ushort_as_half(uint16_t(q[k] << 7))), s);
}

// The tensor that a chunk belongs to: the last whose first chunk is not beyond it.
template <int MAX>
__device__ __forceinline__ int tensor_of(const List<MAX>& tl, int chunk) {
  int lo = 0, hi = tl.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (tl.first_chunk[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// state[0] = steps taken so far (read by every CTA before it counts itself in state[1]); of the step's last launch the
// CTA that arrives last writes the new count and clears the counter.
// BITS: of the moments.  TP: of the parameters and gradients.
template <int BITS, class TP, int MAX>
__global__ void __launch_bounds__(kThreads)
adamw_kernel(const __grid_constant__ List<MAX> tl, const __grid_constant__ Hyper hp,
             unsigned long long* __restrict__ state) {
  __shared__ float consts_s[2];
  __shared__ uint32_t key_s;
  constexpr bool kMixed = sizeof(TP) == 2;
  using TM = std::conditional_t<BITS == 8, uint8_t, float>;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int total = tl.first_chunk[tl.count];

  float pv[2][4];
  TP gv[2][4];
  TM mv[2][4], vv[2][4];
  float ms = 0.f, vs = 0.f;
  int k = 0;
  int64_t block = 0, n = 0;
  bool vec = false;
  auto load = [&](int chunk) {
    k = tensor_of(tl, chunk);
    n = tl.n[k];
    vec = tl.vec[k];
    block = int64_t(chunk - tl.first_chunk[k]) * (kChunk / kBlock) + warp;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t at = block * kBlock + j * 128 + lane * 4;
      load4(static_cast<const float*>(tl.master[k]), at, n, vec, pv[j]);
      load4(static_cast<const TP*>(tl.g[k]), at, n, vec, gv[j]);
      load4(static_cast<const TM*>(tl.m[k]), at, n, vec, mv[j]);
      load4(static_cast<const TM*>(tl.v[k]), at, n, vec, vv[j]);
    }
    if (BITS == 8 && block * kBlock < n) {
      ms = tl.ms[k][block];
      vs = tl.vs[k][block];
    }
  };

  int chunk = blockIdx.x;
  unsigned long long step = 0;
  if (lane == 0 && warp < 2) step = *reinterpret_cast<volatile unsigned long long*>(state);
  if (chunk < total) load(chunk);
  if (lane == 0 && warp < 2) {
    // the scalars in double, as Python would form them
    const double rest = 1.0 - pow(warp ? hp.beta2 : hp.beta1, double(step + 1ull));
    consts_s[warp] = float(warp ? 1.0 / sqrt(rest) : hp.lr / rest);
    if (warp == 0) key_s = mix(hp.seed + uint32_t(step + 1ull) * 0x9E3779B9u);
  }
  __syncthreads();
  const float step_size = consts_s[0], inv_bc2 = consts_s[1];
  const uint32_t step_key = key_s;

  while (chunk < total) {
    const int64_t at0 = block * kBlock + lane * 4;
    if (block * kBlock < n) {  // uniform in the warp
      float m[2][4], v[2][4];
      if constexpr (BITS == 8) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          decode_m(mv[j], ms, m[j]);
          decode_v(vv[j], vs, v[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) m[j][e] = mv[j][e], v[j][e] = vv[j][e];
      }
      uint32_t top_m = 0, top_v = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float g = to_f32(gv[j][e]);
          m[j][e] = __fadd_rn(__fmul_rn(m[j][e], hp.b1), __fmul_rn(g, hp.w1));
          v[j][e] = __fadd_rn(__fmul_rn(v[j][e], hp.b2), __fmul_rn(__fmul_rn(g, g), hp.w2));
          pv[j][e] = pv[j][e] * hp.keep - step_size * (m[j][e] / (sqrtf(v[j][e]) * inv_bc2 + hp.eps));
          if (BITS == 8) {  // elements beyond the tensor: zeros
            const bool in = at0 + j * 128 + e < n;
            top_m = max(top_m, in ? __float_as_uint(m[j][e]) & 0x7FFFFFFFu : 0u);
            top_v = max(top_v, in ? __float_as_uint(v[j][e]) & 0x7FFFFFFFu : 0u);
          }
        }
        const int64_t at = at0 + j * 128;
        store4(tl.master[k], at, n, vec, pv[j]);
        if constexpr (kMixed) {
          bf16 p16[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) p16[e] = __float2bfloat16_rn(pv[j][e]);
          store4(static_cast<bf16*>(tl.p[k]), at, n, vec, p16);
        }
        if constexpr (BITS == 32) {
          store4(static_cast<float*>(tl.m[k]), at, n, vec, m[j]);
          store4(static_cast<float*>(tl.v[k]), at, n, vec, v[j]);
        }
      }
      if constexpr (BITS == 8) {
        const float2 sm = scale_of(__reduce_max_sync(0xFFFFFFFFu, top_m), 1.0f / 448.0f);
        const float2 sv = scale_of(__reduce_max_sync(0xFFFFFFFFu, top_v), 1.0f / 61440.0f);
        if (lane == 0) {
          tl.ms[k][block] = sm.x;
          tl.vs[k][block] = sv.x;
        }
        const uint32_t key = mix(step_key + uint32_t(tl.first_tensor + k));
        const uint32_t least = sv.x > 0.f ? 1u : 0u;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint8_t qm[4], qv[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t r = mix(key + uint32_t(at0 + j * 128 + e));
            const float tm = __fmul_rn(m[j][e], sm.y), tv = __fmul_rn(v[j][e], sv.y);
            qm[e] = uint8_t(min(round_code<7>(fabsf(tm), r & 0xFFFFu), 0x7Eu) | (__float_as_uint(tm) >> 31 << 7));
            qv[e] = uint8_t(max(min(round_code<15>(tv, r >> 16), 0xF7u), least));
          }
          store4(static_cast<uint8_t*>(tl.m[k]), at0 + j * 128, n, vec, qm);
          store4(static_cast<uint8_t*>(tl.v[k]), at0 + j * 128, n, vec, qv);
        }
      }
    }
    chunk += gridDim.x;
    if (chunk < total) load(chunk);
  }
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

// The values of 8-bit moments.  p, g: where the first and second moments go.
template <int MAX>
__global__ void __launch_bounds__(kThreads)
adamw_moments_kernel(const __grid_constant__ List<MAX> tl, int total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  for (int chunk = blockIdx.x; chunk < total; chunk += gridDim.x) {
    const int k = tensor_of(tl, chunk);
    const int64_t n = tl.n[k], block = int64_t(chunk - tl.first_chunk[k]) * (kChunk / kBlock) + warp;
    const bool vec = tl.vec[k];
    if (block * kBlock >= n) continue;
    const float ms = tl.ms[k][block], vs = tl.vs[k][block];
    uint8_t qm[2][4], qv[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      load4(static_cast<const uint8_t*>(tl.m[k]), block * kBlock + j * 128 + lane * 4, n, vec, qm[j]);
      load4(static_cast<const uint8_t*>(tl.v[k]), block * kBlock + j * 128 + lane * 4, n, vec, qv[j]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float m[4], v[4];
      decode_m(qm[j], ms, m);
      decode_v(qv[j], vs, v);
      store4(static_cast<float*>(tl.p[k]), block * kBlock + j * 128 + lane * 4, n, vec, m);
      store4(tl.master[k], block * kBlock + j * 128 + lane * 4, n, vec, v);
    }
  }
}

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Fills the list with tensors from `from` on, as many as fit; returns the first that does not.
struct Arrays {
  void* const* p;
  float* const* master;
  const void* const* g;
  void* const* m;
  void* const* v;
  float* const* ms;
  float* const* vs;
  const int64_t* n;
  int p_size, m_size;  // bytes of an element
};
template <int MAX>
int fill(List<MAX>& tl, const Arrays& a, int from, int n_tensors) {
  tl.count = 0;
  tl.first_tensor = from;
  tl.first_chunk[0] = 0;
  int i = from;
  for (; i < n_tensors && tl.count < MAX; ++i) {
    const int k = tl.count;
    const int64_t chunks = gc::ceil_div(a.n[i], kChunk);
    if (int64_t(tl.first_chunk[k]) + chunks > 0x40000000) break;
    tl.p[k] = a.p[i];
    tl.master[k] = a.master ? a.master[i] : static_cast<float*>(a.p[i]);
    tl.g[k] = a.g ? a.g[i] : nullptr;
    tl.m[k] = a.m[i];
    tl.v[k] = a.v[i];
    tl.ms[k] = a.ms ? a.ms[i] : nullptr;
    tl.vs[k] = a.vs ? a.vs[i] : nullptr;
    tl.n[k] = a.n[i];
    tl.vec[k] = aligned(tl.p[k], 4 * a.p_size) && aligned(tl.g[k], 4 * a.p_size) && aligned(tl.master[k], 16) &&
                aligned(tl.m[k], 4 * a.m_size) && aligned(tl.v[k], 4 * a.m_size);
    tl.first_chunk[k + 1] = tl.first_chunk[k] + int32_t(chunks);
    ++tl.count;
  }
  return i;
}

template <int MAX, int BITS, class TP>
void launch(const List<MAX>& tl, const Hyper& hp, void* state, cudaStream_t st) {
  const int total = tl.first_chunk[tl.count];
  const int blocks = std::max(1, std::min(total, gc::kNumSMs * (BITS == 8 ? 4 : 4)));
  adamw_kernel<BITS, TP, MAX><<<blocks, kThreads, 0, st>>>(tl, hp, static_cast<unsigned long long*>(state));
}
template <int MAX>
int step(const Arrays& a, int n_tensors, int bits, Hyper hp, void* state, cudaStream_t st) {
  int from = 0, launches = 0;
  do {
    List<MAX> tl;
    const int next = fill(tl, a, from, n_tensors);
    if (next == from && n_tensors > 0) return gc::fail(GC_ERR_UNSUPPORTED, "gc_adamw_step: tensor %d is too large", from);
    hp.advance = next >= n_tensors;
    if (bits == 8) a.p_size == 2 ? launch<MAX, 8, bf16>(tl, hp, state, st) : launch<MAX, 8, float>(tl, hp, state, st);
    else a.p_size == 2 ? launch<MAX, 32, bf16>(tl, hp, state, st) : launch<MAX, 32, float>(tl, hp, state, st);
    ++launches;
    from = next;
  } while (from < n_tensors);
  return gc::check_launch("gc_adamw_step", launches);
}
template <int MAX>
int moments(const Arrays& a, int n_tensors, cudaStream_t st) {
  int launches = 0;
  for (int from = 0; from < n_tensors;) {
    List<MAX> tl;
    const int next = fill(tl, a, from, n_tensors);
    if (next == from) return gc::fail(GC_ERR_UNSUPPORTED, "gc_adamw_moments_f32: tensor %d is too large", from);
    from = next;
    const int total = tl.first_chunk[tl.count];
    if (total == 0) continue;
    adamw_moments_kernel<MAX><<<std::min(total, gc::kNumSMs * 8), kThreads, 0, st>>>(tl, total);
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
  GC_REQUIRE(param_type == GC_TYPE_F32 || param_type == GC_TYPE_BF16, "gc_adamw_step: parameters are fp32 or bf16");
  GC_REQUIRE(state_bits == 8 || state_bits == 32, "gc_adamw_step: moments have 8 or 32 bits");
  const bool mixed = param_type == GC_TYPE_BF16, eight = state_bits == 8;
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
  const Arrays a{params, mixed ? masters : nullptr, grads, exp_avg, exp_avg_sq, eight ? exp_avg_scales : nullptr,
                 eight ? exp_avg_sq_scales : nullptr, sizes, mixed ? 2 : 4, eight ? 1 : 4};
  const cudaStream_t st = gc::as_stream(stream);
  return n_tensors <= kFew ? step<kFew>(a, n_tensors, state_bits, hp, state, st)
                           : step<kMany>(a, n_tensors, state_bits, hp, state, st);
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
  const Arrays a{reinterpret_cast<void* const*>(exp_avg_out), exp_avg_sq_out, nullptr,
                 const_cast<void* const*>(reinterpret_cast<const void* const*>(exp_avg)),
                 const_cast<void* const*>(reinterpret_cast<const void* const*>(exp_avg_sq)),
                 const_cast<float* const*>(exp_avg_scales), const_cast<float* const*>(exp_avg_sq_scales), sizes, 4, 1};
  const cudaStream_t st = gc::as_stream(stream);
  return n_tensors <= kFew ? moments<kFew>(a, n_tensors, st) : moments<kMany>(a, n_tensors, st);
}

}  // extern "C"
