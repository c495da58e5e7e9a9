// Distillation loss of a student's logits against a teacher's top logits, and its gradient with respect to the student's.
//
//   p_j = softmax over the entries of a row's list of t_j / T        q_c = softmax over all C classes of z_c / T
//   loss = scale T^2 sum over selected rows of sum_j p_j (log p_j - log q_{i_j})
//   dZ[r, c] = g scale T (q_c - sum of p_j over the entries with i_j = c)      for rows that count, 0 otherwise
//
// An entry whose index is no class, or whose logit is -inf, is none; a row without entries does not count.  The logits are read
// once forward (a running maximum and sum) and once backward, where the row's four statistics are at hand; probabilities
// come from one exponential each, and nothing but dZ is written.  Sums and statistics are fp32.  With u = (z - max) log2(e) / T the
// subtraction comes before the product, so that neither a row filled with the type's lowest value overflows nor one far from zero loses the
// difference to rounding; where the maximum lies near zero (see near_zero) dZ, and one_pass's sums, take one multiply-add for both.
//
// With a gradient to be asked for, rows of some thousands of classes are read once in all (one_pass): a CTA streams rows through a ring of
// segments in shared memory; one half of its threads goes over a row's segments as they arrive for its statistics, the other
// over the same segments again for dZ, giving them back to the copies of the next row.  That is dZ for g = 1, which is what a loss that is
// differentiated by itself has; the backward call looks at g and, where it is another, computes dZ from the logits as it does for other rows.  Rows that a warp
// or less takes get their gradient in the forward launch too, from logits that are still in the caches.
//
// Otherwise G threads take a row: 8 up to 256 classes (a row is few vectors, and what a row costs beside them is shared by fewer), a warp up to
// 4096, a CTA of 128 threads up to 12,288, of 256 above (forward: 20,000 x 8192 in bf16 88 us with 128 threads, 102 with 256, 237 with 512; 4096 x
// 65,536 99, 92, 109); with fewer rows than SMs a CTA takes a part of a row and another launch puts the parts together.  Rows may start
// anywhere: what lies before the first and behind the last 16-byte vector is read by itself.
#include "common.cuh"
#include "ffn_internal.cuh"
#include "tiles.cuh"

#include <cuda_bf16.h>

#include <algorithm>

namespace {

using gc::ffn::both;
using gc::ffn::each;
using gc::ffn::exp2_approx;
using gc::ffn::F2;
using gc::ffn::fma2;

constexpr int kBlocks = gc::kNumSMs * 64;  // partial sums of the loss, at most
constexpr int kMaxParts = 16;             // of a row
constexpr int kMaxList = 1024;            // entries of a list
constexpr int kWide = 256, kMid = 128;    // threads of a CTA that takes a row
constexpr int kPart = 512;                // of one that takes a part of a row
constexpr int64_t kMidTo = 12288;         // classes up to which kMid threads take a row
constexpr int kShortList = 32;            // entries up to which 8 threads take a row
constexpr float kLn2 = 0.69314718055994531f, kLog2e = 1.4426950408889634f;

struct Problem {
  const void* z;
  const void* top;
  const void* index;
  const uint8_t* mask;  // null: all rows
  int64_t ldz, ldt, ldi, M;
  int C, k, parts;
  bool top16, index64;
  float a;  // log2(e) / T
};

__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------ groups of threads
// Reductions over the G threads of a row, of several values at once; all threads get the results.  For a CTA `sh` holds so many words per
// warp.
template <int G, int N, class F>
__device__ __forceinline__ void over_group(float (&v)[N], float* sh, F&& f) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = f(v[i], __shfl_xor_sync(0xffffffffu, v[i], o));
  if constexpr (G > 32) {
    __syncthreads();  // the words' last readers are done
    if (threadIdx.x % 32 == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) sh[threadIdx.x / 32 * N + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sh[i];
#pragma unroll
    for (int w = 1; w < G / 32; ++w)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = f(v[i], sh[w * N + i]);
  }
}
struct Larger {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Sum {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
template <int G>
__device__ __forceinline__ void group_sync() {
  if constexpr (G > 32) __syncthreads();
  else if constexpr (G == 32) __syncwarp();
  else __syncwarp(((1u << G) - 1) << (threadIdx.x % 32 / G * G));
}

// ------------------------------------------------------------------ logits
template <class T>
__device__ __forceinline__ float as_float(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else return __bfloat162float(v);
}
// A vector of 16 bytes as pairs of floats.
template <class T>
struct Vec {
  static constexpr int N = 16 / sizeof(T), P = N / 2;
};
template <class T>
__device__ __forceinline__ void unpack(const uint4& v, F2 (&f)[Vec<T>::P]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(T) == 4) {
    f[0] = F2(w[0], w[1]);
    f[1] = F2(w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = F2(w[i] << 16, w[i] & 0xFFFF0000u);
  }
}
template <class T>
__device__ __forceinline__ float vec_max(const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else {
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&v);
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3])));
    return fmaxf(m.x, m.y);
  }
}
template <class T>
__device__ __forceinline__ uint4 nothing() {  // a vector of -inf
  const uint32_t w = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
  return make_uint4(w, w, w, w);
}
// Elements before the first 16-byte boundary at or behind p.
template <class T>
__device__ __forceinline__ int before_vectors(const T* p, int n) {
  return min(n, int((16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T)));
}

// A maximum m and the sum of 2^((z - m) a), of nothing at first.  (Of a row of -inf the sum is zero; of one with +inf or a NaN, a NaN.)
struct Running {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
  __device__ __forceinline__ void raise(float to, float a) {
    if (to > m) {
      s *= exp2_approx((m - to) * a);
      m = to;
    }
  }
};

template <class T, int G>
__device__ __forceinline__ Running scan(const T* __restrict__ z, int n, int rank, float a) {
  constexpr int U = G == 8 ? 2 : 4;
  Running r;
  const int head = before_vectors(z, n), vectors = (n - head) / Vec<T>::N, tail = head + vectors * Vec<T>::N;
  const uint4* v = reinterpret_cast<const uint4*>(z + head);
  // what no vector holds, fewer than 8 elements at either end
  float ends[2] = {-INFINITY, -INFINITY};
  if (rank < head) ends[0] = as_float(z[rank]);
  if (rank < n - tail) ends[1] = as_float(z[tail + rank]);
  for (int i = rank; i < vectors; i += G * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = i + u * G < vectors ? __ldg(v + i + u * G) : nothing<T>();
    float top = vec_max<T>(w[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) top = fmaxf(top, vec_max<T>(w[u]));
    r.raise(top, a);
    const F2 base = both(-r.base()), scale = both(a);
    F2 sum = both(0.f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      F2 f[Vec<T>::P];
      unpack<T>(w[u], f);
#pragma unroll
      for (int e = 0; e < Vec<T>::P; ++e) sum = sum + each((f[e] + base) * scale, [](float x) { return exp2_approx(x); });
    }
    float x, y;
    sum.get(x, y);
    r.s += x + y;
  }
  r.raise(fmaxf(ends[0], ends[1]), a);
#pragma unroll
  for (int i = 0; i < 2; ++i) r.s += exp2_approx((ends[i] - r.base()) * a);
  return r;
}
// What a thread's sum is where the maximum is `top`.
__device__ __forceinline__ float rescaled(const Running& r, float top, float a) {
  return r.m == -INFINITY ? r.s : r.s * exp2_approx((r.m - top) * a);
}

// ------------------------------------------------------------------ lists
struct Entry {
  float t;
  int c;  // below zero: none
};
// As it was loaded, so that the loads can go out long before anything looks at it.
struct Loaded {
  int64_t c;
  float t;
};
__device__ __forceinline__ Loaded load_entry(const Problem& p, int64_t r, int j) {
  const int64_t at = r * p.ldi + j, ta = r * p.ldt + j;
  Loaded e;
  e.c = p.index64 ? __ldg(static_cast<const int64_t*>(p.index) + at) : __ldg(static_cast<const int32_t*>(p.index) + at);
  e.t = p.top16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.top)[ta]) : __ldg(static_cast<const float*>(p.top) + ta);
  return e;
}
__device__ __forceinline__ Entry looked_at(const Problem& p, const Loaded& e) {
  return {e.t, e.c >= 0 && e.c < p.C && e.t != -INFINITY ? int(e.c) : -1};
}
__device__ __forceinline__ Entry entry(const Problem& p, int64_t r, int j) { return looked_at(p, load_entry(p, r, j)); }

// Of a row: the student's maximum and the logarithm (base 2) of its sum, and the teacher's.  A row that does not count has +inf
// for the last, which no other has.
struct Stats {
  float zm, zl, tm, tl;
};

// The parts of a row's columns begin at multiples of this.
__device__ __host__ __forceinline__ int part_columns(int C, int parts) { return ((C + parts - 1) / parts + 63) / 64 * 64; }

// Part `blockIdx.x` of row `blockIdx.y`.
template <class T>
__global__ void __launch_bounds__(kPart)
distill_part_kernel(const __grid_constant__ Problem p, float2* __restrict__ out) {
  __shared__ float sh[kPart / 32];
  const int64_t r = blockIdx.y;
  if (p.mask && !p.mask[r]) return;
  const int width = part_columns(p.C, p.parts), from = min(p.C, int(blockIdx.x) * width), n = min(width, p.C - from);
  const Running x = scan<T, kPart>(static_cast<const T*>(p.z) + r * p.ldz + from, n, threadIdx.x, p.a);
  float top[1] = {x.m};
  over_group<kPart>(top, sh, Larger{});
  float sum[1] = {rescaled(x, top[0], p.a)};
  over_group<kPart>(sum, sh, Sum{});
  if (threadIdx.x == 0) out[r * p.parts + blockIdx.x] = make_float2(top[0], sum[0]);
}

__global__ void __launch_bounds__(256)
distill_sum_kernel(const float* __restrict__ partials, int n, float scale, float* __restrict__ loss) {
  __shared__ double sh[256];
  double a = 0.;
  for (int i = threadIdx.x; i < n; i += 256) a += partials[i];
  sh[threadIdx.x] = a;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) *loss = float(sh[0] * scale);
}

// ------------------------------------------------------------------ gradient
template <class T>
__device__ __forceinline__ uint4 pack(const F2 (&f)[Vec<T>::P]) {
  uint32_t w[4];
  float x, y;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[i].get(x, y);
      w[2 * i] = __float_as_uint(x);
      w[2 * i + 1] = __float_as_uint(y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i].get(x, y);
      const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <class T>
__device__ __forceinline__ T rounded(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else return __float2bfloat16_rn(v);
}

// g (q - p) of a logit.  Where the maximum lies near zero the exponent is one multiply-add, z a + (-zm a - zl), as in the vectors: the rounding
// of that sum, half a step of numbers below 64, stays below 2^-19.  It grows with the maximum (at -1e9, a mask's value, it is 64 or so),
// so that other rows subtract first, which is exact beside the difference.
__device__ __forceinline__ bool near_zero(float m, float a) { return fabsf(m * a) < 32.f; }
struct Gradient {
  float zm, zl, a, g;
  __device__ __forceinline__ float operator()(float z, float p) const {
    const float e = near_zero(zm, a) ? fmaf(z, a, -zm * a - zl) : (z - zm) * a - zl;
    return g * (exp2_approx(e) - p);
  }
};
// The probabilities of a class's entries: an index may stand in the list more than once.  kp: a multiple of 4.
__device__ __forceinline__ float sum_at(int c, const int* cls, const float* prob, int kp) {
  float sum = 0.f;
  for (int i = 0; i < kp; i += 4) {
    const int4 ci = *reinterpret_cast<const int4*>(cls + i);
    const float4 pi = *reinterpret_cast<const float4*>(prob + i);
    sum += (ci.x == c ? pi.x : 0.f) + (ci.y == c ? pi.y : 0.f) + (ci.z == c ? pi.z : 0.f) + (ci.w == c ? pi.w : 0.f);
  }
  return sum;
}

// An index's bit among 32 for each of a list's entries.  Of a long list it marks what may stand in it twice, and only those entries look
// the list over (with every entry doing so 200,000 x 300 in fp32 with lists of 256 took 2190 us instead of 819, 60,000 x 1000 with 64 160 and 150).
struct Mark {
  int word;
  uint32_t bit;
};
__device__ __forceinline__ Mark mark_of(int c, int kp) {
  const uint32_t at = __umulhi(uint32_t(c) * 2654435761u, uint32_t(kp) * 32u);
  return {int(at / 32), 1u << at % 32};
}
__host__ __device__ constexpr bool marked(int k) { return k > kShortList; }
__host__ __device__ constexpr int list_words(int k) { return (marked(k) ? 4 : 2) * ((k + 3) / 4 * 4); }

// n columns of a row's gradient, from column `from` on, by G threads: z and d point at the first.  `list`: list_words() of shared memory.  pad:
// columns of zeros behind them.
template <class T, int G>
__device__ __forceinline__ void gradient_of_row(const Problem& p, int64_t r, const T* z, T* d, int from, int n, int pad, const Stats& st, float g,
                                                int rank, int* list) {
  constexpr int U = G == 8 ? 2 : 4;
  const int kp = (p.k + 3) / 4 * 4;
  int* const cls = list;
  float* const prob = reinterpret_cast<float*>(list + kp);
  uint32_t *const once = reinterpret_cast<uint32_t*>(list + 2 * kp), *const again = once + kp;
  const bool counts = !(st.tl == INFINITY), marks = marked(p.k);
  if (rank < pad) d[n + rank] = rounded<T>(0.f);
  if (counts)
    for (int j = rank; j < kp; j += G) {
      Entry e{0.f, -1};
      if (j < p.k) e = entry(p, r, j);
      cls[j] = e.c;
      prob[j] = e.c < 0 ? 0.f : exp2_approx((e.t - st.tm) * p.a - st.tl);
      if (marks) once[j] = again[j] = 0;
    }
  if (counts && marks) {
    group_sync<G>();
    for (int j = rank; j < p.k; j += G) {
      const int c = cls[j];
      if (c < 0) continue;
      const Mark m = mark_of(c, kp);
      if (atomicOr(once + m.word, m.bit) & m.bit) atomicOr(again + m.word, m.bit);
    }
  }
  const Gradient one{st.zm, st.zl, p.a, g};
  const int head = before_vectors(d, n);
  const bool vectors_fit = (reinterpret_cast<uintptr_t>(z) - reinterpret_cast<uintptr_t>(d)) % 16 == 0;
  const int vectors = vectors_fit ? (n - head) / Vec<T>::N : 0, tail = vectors_fit ? head + vectors * Vec<T>::N : head;
  if (rank < head) d[rank] = rounded<T>(counts ? one(as_float(z[rank]), 0.f) : 0.f);
  for (int c = tail + rank; c < n; c += G) d[c] = rounded<T>(counts ? one(as_float(z[c]), 0.f) : 0.f);
  const uint4* v = reinterpret_cast<const uint4*>(z + head);
  uint4* to = reinterpret_cast<uint4*>(d + head);
  const bool plain = near_zero(st.zm, p.a);
  const F2 m = both(-st.zm), a = both(p.a), l = both(-st.zl), gg = both(g), c = both(-st.zm * p.a - st.zl);
  for (int i = rank; i < vectors; i += G * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = counts && i + u * G < vectors ? __ldg(v + i + u * G) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      F2 f[Vec<T>::P];
      unpack<T>(w[u], f);
      if (plain) {
#pragma unroll
        for (int e = 0; e < Vec<T>::P; ++e) f[e] = each(fma2(f[e], a, c), [](float x) { return exp2_approx(x); }) * gg;
      } else {
#pragma unroll
        for (int e = 0; e < Vec<T>::P; ++e) f[e] = each(fma2(f[e] + m, a, l), [](float x) { return exp2_approx(x); }) * gg;
      }
      if (i + u * G < vectors) __stcs(to + i + u * G, counts ? pack<T>(f) : make_uint4(0, 0, 0, 0));
    }
  }
  group_sync<G>();  // the lists, and the columns that the entries below write again
  if (!counts) return;
  for (int j = rank; j < p.k; j += G) {
    const int c = cls[j];
    if (c < from || c >= from + n) continue;
    // all of an index's entries write the same
    const Mark m = mark_of(c, kp);
    const float sum = marks && !(again[m.word] & m.bit) ? prob[j] : sum_at(c, cls, prob, kp);
    d[c - from] = rounded<T>(one(as_float(z[c - from]), sum));
  }
}

// G threads per row; the block's sum of losses goes to partials.  from_parts: what distill_part_kernel left, or null.  GRADIENT: the
// row's gradient too, for a loss that is differentiated by itself.
template <class T, int G, bool GRADIENT>
__global__ void __launch_bounds__(G > 32 ? G : 256)
distill_forward_kernel(const __grid_constant__ Problem p, const float2* __restrict__ from_parts, Stats* __restrict__ stats,
                       float* __restrict__ partials, float factor, T* __restrict__ dz, int64_t lddz, int pad) {
  constexpr int kThreads = G > 32 ? G : 256, R = kThreads / G;  // rows of a CTA at a time
  __shared__ float sh[3 * 32];
  extern __shared__ __align__(16) uint8_t lists[];  // GRADIENT: see distill_backward_kernel
  const int rank = threadIdx.x % G;
  float loss = 0.f;
  for (int64_t r0 = int64_t(blockIdx.x) * R; r0 < p.M; r0 += int64_t(gridDim.x) * R) {  // the same for all of a CTA
    const int64_t mine = r0 + threadIdx.x / G, r = min(mine, p.M - 1);
    const bool chosen = mine < p.M && (!p.mask || p.mask[r]);
    const T* z = static_cast<const T*>(p.z) + r * p.ldz;
    if (G > 32 && !chosen) {
      if (threadIdx.x == 0) stats[r] = {0.f, 0.f, 0.f, INFINITY};
      continue;
    }
    // the thread's first entry is on its way while the row is read
    Loaded own{-1, 0.f};
    if (chosen && rank < p.k) own = load_entry(p, r, rank);
    Running x;
    if (chosen) {
      if (from_parts) {
        for (int i = rank; i < p.parts; i += G) {
          const float2 part = from_parts[r * p.parts + i];
          x.raise(part.x, p.a);
          x.s += part.x == -INFINITY ? part.y : part.y * exp2_approx((part.x - x.m) * p.a);
        }
      } else {
        x = scan<T, G>(z, p.C, rank, p.a);
      }
    }
    const Entry mine_first = looked_at(p, own);
    const float at_first = mine_first.c >= 0 ? as_float(z[mine_first.c]) : 0.f;
    // the maxima; whether the list has entries
    float top[3] = {x.m, mine_first.c >= 0 ? mine_first.t : -INFINITY, mine_first.c >= 0 ? 1.f : 0.f};
    for (int j = rank + G; chosen && j < p.k; j += G) {
      const Entry e = entry(p, r, j);
      if (e.c >= 0) top[1] = fmaxf(top[1], e.t), top[2] = 1.f;
    }
    over_group<G>(top, sh, Larger{});
    const float zm = top[0], tm = top[1];
    const bool counts = chosen && top[2] > 0.f;
    // the sums: of the row's exponentials, of the list's, and of the list's times what the logarithms differ by
    float sum[3] = {rescaled(x, zm, p.a), 0.f, 0.f};
    auto add = [&](const Entry& e, float at) {
      if (e.c < 0) return;
      const float w = exp2_approx((e.t - tm) * p.a);
      sum[1] += w;
      if (!(w == 0.f)) sum[2] += w * (((e.t - tm) - (at - zm)) * p.a);
    };
    if (counts) {
      add(mine_first, at_first);
      for (int j = rank + G; j < p.k; j += G) {
        const Entry e = entry(p, r, j);
        add(e, e.c >= 0 ? as_float(z[e.c]) : 0.f);
      }
    }
    over_group<G>(sum, sh, Sum{});
    const Stats st = counts ? Stats{zm, log2_approx(sum[0]), tm, log2_approx(sum[1])} : Stats{0.f, 0.f, 0.f, INFINITY};
    if (rank == 0 && mine < p.M) {
      stats[r] = st;
      if (counts) loss += kLn2 * (sum[2] / sum[1] - st.tl + st.zl);
    }
    if constexpr (GRADIENT) {
      if (mine < p.M) {
        gradient_of_row<T, G>(p, r, z, dz + r * lddz, 0, p.C, pad, st, factor, rank, reinterpret_cast<int*>(lists) + threadIdx.x / G * list_words(p.k));
      }
      group_sync<G>();  // the lists are read
    }
  }
  float all[1] = {loss};
  over_group<(G > 32 ? G : 256)>(all, sh, Sum{});
  if (threadIdx.x == 0) partials[blockIdx.x] = all[0];
}

// ------------------------------------------------------------------ both in one pass
constexpr int64_t kOnePassFrom = 8192;  // bytes; rows that are longer (30,000 x 4096 in bf16: 161 us, 143 in two passes; 20,000 x 8192: 184 and 412)
constexpr int kLong = 352, kShort = 64;  // threads of either half, for long and short rows
constexpr int kSegments = 10;            // of a ring
constexpr int kEach = 4;                 // vectors per thread of a segment
template <int THREADS>
struct Ring {
  static constexpr int kVectors = THREADS * kEach, kBytes = kVectors * 16;  // of a segment
  static constexpr int kMostBytes = (kSegments - 1) * kBytes;               // of a row
};
// Entries' classes, logits (later probabilities) and the student's logits at them, of a row.
constexpr int kListWords = 3;
constexpr int kOnePassList = 256;  // entries of a list

template <int BARRIER, int THREADS>
__device__ __forceinline__ void sync_threads() { asm volatile("bar.sync %0, %1;" ::"n"(BARRIER), "n"(THREADS) : "memory"); }

// THREADS that make a row's statistics, as many that make the gradient of the row before, a warp whose first lane fetches segments, and
// one that fetches lists a row ahead (two loads after each other, which the row's threads would wait for).  Persistent over rows.  (4096 x 65,536 in bf16, forward and backward: 217 us, 5.0 TB/s
// of the bytes that cannot be avoided; 285 with the same threads doing one after the other, whose exponentials of a row wait for its
// sums; 231 with 256 threads and 13 segments of 16 KB, 220 with 384 and 9.  What is left is issue slots: 16 instructions per logit,
// the special function unit half busy.)
template <class T, int THREADS>
__global__ void __launch_bounds__(2 * THREADS + 64)
distill_one_pass_kernel(const __grid_constant__ Problem p, Stats* __restrict__ stats, float* __restrict__ partials, float g,
                        T* __restrict__ dz, int64_t lddz, int pad, int* __restrict__ word) {
  using namespace gc::tc;
  constexpr int kBytes = Ring<THREADS>::kBytes, kVectors = Ring<THREADS>::kVectors, kWarps = THREADS / 32, N = Vec<T>::N;
  extern __shared__ __align__(128) uint8_t smem[];  // the ring; the lists of two rows: classes, logits (then probabilities), the student's logits
  __shared__ __align__(8) uint64_t bars[2 * kSegments + 6];
  __shared__ float sh[2][kWarps][4];
  __shared__ float info[2][4];  // of two rows: the student's maximum and logarithm of its sum; whether the row counts; the list's largest logit
  __shared__ int abort_s;
  const uint32_t ring = smem_u32(smem);
  auto full = [&](int i) { return smem_u32(&bars[i]); };
  auto empty = [&](int i) { return smem_u32(&bars[kSegments + i]); };
  auto ready = [&](int i) { return smem_u32(&bars[2 * kSegments + i]); };
  auto taken = [&](int i) { return smem_u32(&bars[2 * kSegments + 2 + i]); };
  auto listed = [&](int i) { return smem_u32(&bars[2 * kSegments + 4 + i]); };
  const int kp = (p.k + 3) / 4 * 4;
  auto classes = [&](int i) { return reinterpret_cast<int*>(smem + kSegments * kBytes) + i * kListWords * kp; };
  auto probs = [&](int i) { return reinterpret_cast<float*>(classes(i) + kp); };
  auto at_entries = [&](int i) { return probs(i) + kp; };
  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int i = 0; i < kSegments; ++i) {
      mbar_init(full(i), 1);
      mbar_init(empty(i), kWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(ready(i), 1);
      mbar_init(listed(i), 1);
      mbar_init(taken(i), kWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  __syncthreads();
  volatile int* abort_p = &abort_s;
  const int rank = threadIdx.x % THREADS, lane = threadIdx.x % 32;
  int slot = 0, rows = 0;  // rows: of those that are chosen
  uint32_t phase = 0;
  auto advance = [&]() {
    if (++slot == kSegments) slot = 0, phase ^= 1u;
  };
  bool ok = true;

  if (threadIdx.x >= 2 * THREADS + 32) {
    // ------------------------------------------------------------ fetches lists
    constexpr int kEntries = kOnePassList / 32;  // of a lane
    for (int64_t r = blockIdx.x; r < p.M; r += gridDim.x) {
      if (p.mask && !p.mask[r]) continue;
      const T* z = static_cast<const T*>(p.z) + r * p.ldz;
      const int buf = rows & 1;
      Entry e[kEntries];
      float at[kEntries], tm = -INFINITY;
#pragma unroll
      for (int i = 0; i < kEntries; ++i) e[i] = i * 32 + lane < p.k ? entry(p, r, i * 32 + lane) : Entry{0.f, -1};
#pragma unroll
      for (int i = 0; i < kEntries; ++i) at[i] = e[i].c >= 0 ? as_float(z[e[i].c]) : 0.f;
      bool any = false;
#pragma unroll
      for (int i = 0; i < kEntries; ++i)
        if (e[i].c >= 0) tm = fmaxf(tm, e[i].t), any = true;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, o));
      any = __any_sync(0xffffffffu, any);
      if (ok) ok = gc::tiles::wait(taken(buf), ((rows >> 1) & 1u) ^ 1u, abort_p);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kEntries; ++i) {
        const int j = i * 32 + lane;
        if (j < kp) classes(buf)[j] = e[i].c, probs(buf)[j] = e[i].t, at_entries(buf)[j] = at[i];
      }
      if (lane == 0) info[buf][2] = any ? 1.f : 0.f, info[buf][3] = tm;
      __syncwarp();
      if (lane == 0) mbar_arrive(listed(buf));
      ++rows;
    }
  } else if (threadIdx.x >= 2 * THREADS) {
    // ------------------------------------------------------------ fetches
    if (lane == 0) {
      uint32_t issued = 0;
      for (int64_t r = blockIdx.x; ok && r < p.M; r += gridDim.x) {
        if (p.mask && !p.mask[r]) continue;
        const T* z = static_cast<const T*>(p.z) + r * p.ldz;
        const int head = before_vectors(z, p.C), vectors = (p.C - head) / N;
        for (int v = 0; v < vectors; v += kVectors) {
          if (!gc::tiles::wait(empty(slot), phase ^ 1u, abort_p)) { ok = false; break; }
          const uint32_t bytes = min(kVectors, vectors - v) * 16;
          mbar_expect_tx(full(slot), bytes);
          bulk_load(ring + slot * kBytes, z + head + int64_t(v) * N, bytes, full(slot));
          advance();
          ++issued;
        }
      }
      for (uint32_t j = 0; j < issued && j < uint32_t(kSegments); ++j) {  // what was issued lands before the CTA exits
        if (slot == 0) phase ^= 1u;
        slot = slot == 0 ? kSegments - 1 : slot - 1;
        gc::tiles::drain(full(slot), phase);
      }
    }
  } else if (threadIdx.x < THREADS) {
    // ------------------------------------------------------------ statistics
    const int warp = rank / 32;
    float loss = 0.f;
    int turn = 0;
    auto reduce = [&](auto& v, auto f) {
      constexpr int n = sizeof(v) / sizeof(float);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = f(v[i], __shfl_xor_sync(0xffffffffu, v[i], o));
      turn ^= 1;  // the other place's readers have come past a barrier since
      if (lane == 0)
#pragma unroll
        for (int i = 0; i < n; ++i) sh[turn][warp][i] = v[i];
      sync_threads<1, THREADS>();
#pragma unroll
      for (int i = 0; i < n; ++i) v[i] = sh[turn][0][i];
#pragma unroll
      for (int w = 1; w < kWarps; ++w)
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = f(v[i], sh[turn][w][i]);
    };
    for (int64_t r = blockIdx.x; r < p.M; r += gridDim.x) {
      if (p.mask && !p.mask[r]) {
        if (rank == 0) stats[r] = {0.f, 0.f, 0.f, INFINITY};
        continue;
      }
      const T* z = static_cast<const T*>(p.z) + r * p.ldz;
      const int head = before_vectors(z, p.C), vectors = (p.C - head) / N, tail = head + vectors * N;
      const int buf = rows & 1;
      const int* cls = classes(buf);
      float* prob = probs(buf);
      const float* at_entry = at_entries(buf);
      Running x;
      const float ends[2] = {rank < head ? as_float(z[rank]) : -INFINITY, rank < p.C - tail ? as_float(z[tail + rank]) : -INFINITY};
      for (int v = 0; v < vectors; v += kVectors) {
        if (ok) ok = gc::tiles::wait(full(slot), phase, abort_p);
        const uint4* seg = reinterpret_cast<const uint4*>(smem + slot * kBytes);
        uint4 w[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) w[u] = v + rank + u * THREADS < vectors ? seg[rank + u * THREADS] : nothing<T>();
        x.raise(fmaxf(fmaxf(vec_max<T>(w[0]), vec_max<T>(w[1])), fmaxf(vec_max<T>(w[2]), vec_max<T>(w[3]))), p.a);
        const F2 scale = both(p.a);
        F2 sum = both(0.f);
        if (near_zero(x.base(), p.a)) {
          const F2 base = both(-x.base() * p.a);
#pragma unroll
          for (int u = 0; u < kEach; ++u) {
            F2 f[Vec<T>::P];
            unpack<T>(w[u], f);
#pragma unroll
            for (int e = 0; e < Vec<T>::P; ++e) sum = sum + each(fma2(f[e], scale, base), [](float t) { return exp2_approx(t); });
          }
        } else {
          const F2 base = both(-x.base());
#pragma unroll
          for (int u = 0; u < kEach; ++u) {
            F2 f[Vec<T>::P];
            unpack<T>(w[u], f);
#pragma unroll
            for (int e = 0; e < Vec<T>::P; ++e) sum = sum + each((f[e] + base) * scale, [](float t) { return exp2_approx(t); });
          }
        }
        float a, b;
        sum.get(a, b);
        x.s += a + b;
        advance();
      }
      x.raise(fmaxf(ends[0], ends[1]), p.a);
#pragma unroll
      for (int i = 0; i < 2; ++i) x.s += exp2_approx((ends[i] - x.base()) * p.a);
      float top[1] = {x.m};
      reduce(top, [](float a, float b) { return fmaxf(a, b); });
      if (ok) ok = gc::tiles::wait(listed(buf), (rows >> 1) & 1u, abort_p);
      const bool counts = info[buf][2] > 0.f;
      const float zm = top[0], tm = info[buf][3];
      float sums[3] = {x.m == -INFINITY ? x.s : x.s * exp2_approx((x.m - zm) * p.a), 0.f, 0.f};
      for (int j = rank; counts && j < p.k; j += THREADS) {
        if (cls[j] < 0) continue;
        const float w = exp2_approx((prob[j] - tm) * p.a);
        sums[1] += w;
        if (!(w == 0.f)) sums[2] += w * (((prob[j] - tm) - (at_entry[j] - zm)) * p.a);
      }
      reduce(sums, [](float a, float b) { return a + b; });
      const float zl = log2_approx(sums[0]), tl = log2_approx(sums[1]);
      for (int j = rank; counts && j < p.k; j += THREADS) prob[j] = exp2_approx((prob[j] - tm) * p.a - tl);
      if (rank == 0) {
        stats[r] = counts ? Stats{zm, zl, tm, tl} : Stats{0.f, 0.f, 0.f, INFINITY};
        if (counts) loss += kLn2 * (sums[2] / sums[1] - tl + zl);
        info[buf][0] = zm, info[buf][1] = zl;
      }
      sync_threads<1, THREADS>();  // all of the list is written
      if (rank == 0) mbar_arrive(ready(buf));
      ++rows;
    }
    if (rank == 0) partials[blockIdx.x] = loss;
  } else {
    // ------------------------------------------------------------ gradient
    for (int64_t r = blockIdx.x; r < p.M; r += gridDim.x) {
      const T* z = static_cast<const T*>(p.z) + r * p.ldz;
      T* d = dz + r * lddz;
      const int head = before_vectors(z, p.C), vectors = (p.C - head) / N, tail = head + vectors * N;
      uint4* to = reinterpret_cast<uint4*>(d + head);
      if (rank < pad) d[p.C + rank] = rounded<T>(0.f);
      const bool chosen = !p.mask || p.mask[r];
      const int buf = rows & 1;
      if (chosen && ok) ok = gc::tiles::wait(ready(buf), (rows >> 1) & 1u, abort_p);
      const float zm = info[buf][0], zl = info[buf][1];
      const bool counts = chosen && info[buf][2] > 0.f;
      if (!counts) {
        if (rank < head) d[rank] = rounded<T>(0.f);
        if (rank < p.C - tail) d[tail + rank] = rounded<T>(0.f);
        for (int i = rank; i < vectors; i += THREADS) to[i] = make_uint4(0, 0, 0, 0);
        if (!chosen) continue;
      }
      const Gradient one{zm, zl, p.a, g};
      if (counts) {
        if (rank < head) d[rank] = rounded<T>(one(as_float(z[rank]), 0.f));
        if (rank < p.C - tail) d[tail + rank] = rounded<T>(one(as_float(z[tail + rank]), 0.f));
      }
      const bool plain = near_zero(zm, p.a);
      const F2 a = both(p.a), gg = both(g), c = both(-zm * p.a - zl), m = both(-zm), l = both(-zl);
      for (int v = 0; v < vectors; v += kVectors) {
        if (ok) ok = gc::tiles::wait(full(slot), phase, abort_p);
        const uint4* seg = reinterpret_cast<const uint4*>(smem + slot * kBytes);
        uint4 w[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) w[u] = seg[rank + u * THREADS];  // (in a last segment's rest: what a row before left)
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(slot));
        advance();
        if (!counts) continue;
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
          const int i = v + rank + u * THREADS;
          F2 f[Vec<T>::P];
          unpack<T>(w[u], f);
          if (plain) {
#pragma unroll
            for (int e = 0; e < Vec<T>::P; ++e) f[e] = each(fma2(f[e], a, c), [](float t) { return exp2_approx(t); }) * gg;
          } else {
#pragma unroll
            for (int e = 0; e < Vec<T>::P; ++e) f[e] = each(fma2(f[e] + m, a, l), [](float t) { return exp2_approx(t); }) * gg;
          }
          if (i < vectors) to[i] = pack<T>(f);
        }
      }
      // The columns that the entries write again.  (Of every row that is chosen: when a wait has run out, lists change under their readers and
      // not all threads find the same `counts`, but all come here; and what they then find for a class may be anything.)
      sync_threads<2, THREADS>();
      if (counts) {
        const int* cls = classes(buf);
        const float* at_entry = at_entries(buf);
        for (int j = rank; j < p.k; j += THREADS) {
          const int at = cls[j];
          if (uint32_t(at) < uint32_t(p.C)) d[at] = rounded<T>(one(at_entry[j], sum_at(at, cls, probs(buf), kp)));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(taken(buf));
      ++rows;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && abort_s) atomicExch(word, 1);
}

// G threads per row, or per part of one.  Rows are taken from the last to the first: the forward pass, which has mostly
// just run, left the last ones in the L2.  `pad`: columns of zeros behind a row of dZ.
template <class T, int G>
__global__ void __launch_bounds__(G > 32 ? G : 256)
distill_backward_kernel(const __grid_constant__ Problem p, const Stats* __restrict__ stats, const float* __restrict__ grad, float factor,
                        T* __restrict__ dz, int64_t lddz, int pad, bool has_one) {
  constexpr int kThreads = G > 32 ? G : 256, R = kThreads / G;
  if (has_one && __ldg(grad) == 1.f) return;  // dZ holds that gradient
  extern __shared__ __align__(16) uint8_t lists[];  // of each of the CTA's rows: the entries' classes, their probabilities, marks
  const int rank = threadIdx.x % G;
  int* const list = reinterpret_cast<int*>(lists) + threadIdx.x / G * list_words(p.k);
  const float g = factor * __ldg(grad);
  const int width = p.parts > 1 ? part_columns(p.C, p.parts) : p.C;
  const int64_t items = p.M * p.parts;
  for (int64_t i0 = int64_t(blockIdx.x) * R; i0 < items; i0 += int64_t(gridDim.x) * R) {
    const int64_t item = items - 1 - (i0 + threadIdx.x / G);
    group_sync<G>();  // the lists of the row before are read
    if (item < 0) continue;  // only in groups of a warp or less, whose other rows exist
    const int64_t r = item / p.parts;
    const int from = min(p.C, int(item - r * p.parts) * width), n = min(width, p.C - from);
    const bool last = int(item - r * p.parts) == p.parts - 1;
    const T* z = static_cast<const T*>(p.z) + r * p.ldz + from;
    T* d = dz + r * lddz + from;
    gradient_of_row<T, G>(p, r, z, d, from, n, last ? pad : 0, stats[r], g, rank, list);
  }
}

// ------------------------------------------------------------------ host
int threads_per_row(int64_t C, int64_t k) { return C > kMidTo ? kWide : C > 4096 ? kMid : C <= 256 && k <= kShortList ? 8 : 32; }
// Whether one pass makes statistics and gradient: rows that both start as far behind a 16-byte boundary, enough of them, and of a length
// that keeps the CTA's barriers small beside it.  Returns the CTA's computing threads, or 0.
int one_pass_threads(const void* Z, int type, int64_t ldz, const void* dZ, int64_t lddz, int64_t M, int64_t C, int64_t k) {
  const int64_t size = type == GC_TYPE_F32 ? 4 : 2, bytes = C * size;
  const bool same = (reinterpret_cast<uintptr_t>(Z) - reinterpret_cast<uintptr_t>(dZ)) % 16 == 0 && (ldz - lddz) * size % 16 == 0;
  if (!same || M < gc::kNumSMs || k > kOnePassList) return 0;
  return bytes <= kOnePassFrom || bytes > Ring<kLong>::kMostBytes ? 0 : bytes <= Ring<kShort>::kMostBytes ? kShort : kLong;
}
// Whether a forward call makes the gradient: in one pass, or where a warp or less takes a row, which is still near when the row's
// statistics are there.  169,343 x 47 in fp32: 41 us in all, 52 with a launch of its own for the gradient; 60,000 x 1000 in bf16 87 and 102, in
// fp32 127 and 142; 20,000 x 4096 in bf16 96 and 111, in fp32 175 and 175.
bool makes_gradient(const void* Z, int type, int64_t ldz, const void* dZ, int64_t lddz, int64_t M, int64_t C, int64_t k) {
  return one_pass_threads(Z, type, ldz, dZ, lddz, M, C, k) || threads_per_row(C, k) <= 32;
}
// Rows above 8192 columns of which there are fewer than SMs are cut, into parts of 4096 or more.
int parts_of(int64_t M, int64_t C) {
  if (M >= gc::kNumSMs || C <= 8192) return 1;
  return int(std::max<int64_t>(1, std::min<int64_t>({2 * gc::kNumSMs / std::max<int64_t>(M, 1), C / 4096, kMaxParts})));
}
// Forward.  A CTA for a row is done with it, up to 64 to an SM: they balance out by themselves (20,000 x 8192 in bf16: 66 us, 78 with 8 to an SM
// that take several rows each).  Warps and less take several rows, as many CTAs as an SM holds (60,000 x 1000 in fp32: 49 us, 58).
unsigned grid_of(int64_t M, int G) {
  if (G > 32) return unsigned(std::min<int64_t>(M, kBlocks));
  return unsigned(std::min<int64_t>(gc::ceil_div(M, 256 / G), gc::kNumSMs * (G == 32 ? 6 : 8)));
}

int fill(Problem& p, const char* what, const void* Z, int type, int64_t ldz, const void* top, int top_type, int64_t ldt,
         const void* index, int index_bits, int64_t ldi, int64_t M, int64_t C, int64_t k, float temperature) {
  GC_REQUIRE(M >= 0 && C >= 1 && k >= 0, "%s: bad size", what);
  GC_REQUIRE((type == GC_TYPE_F32 || type == GC_TYPE_BF16) && (top_type == GC_TYPE_F32 || top_type == GC_TYPE_BF16),
             "%s: logits are float32 or bfloat16", what);
  GC_REQUIRE(index_bits == 32 || index_bits == 64, "%s: indices have 32 or 64 bits", what);
  GC_REQUIRE(temperature > 0.f && temperature < INFINITY && kLog2e / temperature < INFINITY,
             "%s: the temperature must be positive and finite, and so its reciprocal", what);
  GC_REQUIRE(ldz >= C && ldt >= k && ldi >= k, "%s: leading dimension below the row length", what);
  if (C > (1 << 30) || k > kMaxList) return gc::fail(GC_ERR_UNSUPPORTED, "%s: more than %d entries to a list, or too many classes", what, kMaxList);
  GC_REQUIRE(M == 0 || (Z && (k == 0 || (top && index))), "%s: null pointer", what);
  p = Problem{Z, top, index, nullptr, ldz, ldt, ldi, M, int(C), int(k), parts_of(M, C), top_type == GC_TYPE_BF16, index_bits == 64,
              kLog2e / temperature};
  return GC_OK;
}
// Shared memory of a launch: the ring and two rows' lists; the lists of a CTA's rows.
constexpr int one_pass_bytes(int threads, int k) { return kSegments * threads * kEach * 16 + 2 * kListWords * ((k + 3) / 4 * 4) * 4; }
constexpr int list_bytes(int G, int k) { return (G > 32 ? 1 : 256 / G) * list_words(k) * 4; }
// The attribute belongs to all threads of the process: a call sets it to the longest list's, so that a launch that another thread has
// just allowed stays allowed.
template <class Kernel>
cudaError_t allow_lists(Kernel kern, int G, int smem) {
  return smem > 47 * 1024 ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, list_bytes(G, kMaxList)) : cudaSuccess;
}
template <class F>
void with_group(int G, bool parts, F&& f) {
  if (G == 8) f(std::integral_constant<int, 8>{});
  else if (G == 32) f(std::integral_constant<int, 32>{});
  else if (G == kMid && !parts) f(std::integral_constant<int, kMid>{});
  else f(std::integral_constant<int, kWide>{});
}
template <class F>
void with_type(int type, F&& f) {
  if (type == GC_TYPE_F32) f(float{});
  else f(__nv_bfloat16{});
}

}  // namespace

extern "C" {

size_t gc_distill_workspace_bytes(int64_t M, int64_t C) {
  if (M < 0 || C < 1) return 0;
  return size_t(kBlocks) * sizeof(float) + (parts_of(M, C) > 1 ? size_t(M) * kMaxParts * sizeof(float2) : 0);
}

int gc_distill_one_pass(const void* Z, int type, int64_t ldz, int64_t lddz, int64_t M, int64_t C, int64_t k) {
  return (type == GC_TYPE_F32 || type == GC_TYPE_BF16) && M >= 0 && C >= 1 && k >= 0 && k <= kMaxList &&
         makes_gradient(Z, type, ldz, nullptr, lddz, M, C, k);
}

int gc_distill_forward(const void* Z, int type, int64_t ldz, const void* top, int top_type, int64_t ldt, const void* index,
                       int index_bits, int64_t ldi, const uint8_t* row_mask, int64_t M, int64_t C, int64_t k, float temperature,
                       float scale, float* loss, float* stats, void* dZ, int64_t lddz, int64_t pad, void* workspace,
                       size_t workspace_bytes, void* stream) {
  Problem p;
  int rc = fill(p, "gc_distill_forward", Z, type, ldz, top, top_type, ldt, index, index_bits, ldi, M, C, k, temperature);
  if (rc != GC_OK) return rc;
  GC_REQUIRE(loss && (M == 0 || stats), "gc_distill_forward: null pointer");
  GC_REQUIRE(gc::aligned16(stats), "gc_distill_forward: the statistics must be 16-byte aligned");
  GC_REQUIRE(!dZ || (pad >= 0 && pad < 8 && lddz >= C + pad), "gc_distill_forward: leading dimension below the row length");
  GC_REQUIRE(!dZ || makes_gradient(Z, type, ldz, dZ, lddz, M, C, k), "gc_distill_forward: no gradient for rows like these");
  const cudaStream_t st = gc::as_stream(stream);
  if (M == 0) {
    const cudaError_t e = cudaMemsetAsync(loss, 0, sizeof(float), st);
    return e == cudaSuccess ? GC_OK : gc::fail(GC_ERR_CUDA, "gc_distill_forward: %s", cudaGetErrorString(e));
  }
  if (!workspace || workspace_bytes < gc_distill_workspace_bytes(M, C))
    return gc::fail(GC_ERR_WORKSPACE, "gc_distill_forward: workspace missing or smaller than its query says");
  GC_REQUIRE(gc::aligned16(workspace), "gc_distill_forward: workspace must be 16-byte aligned");
  p.mask = row_mask;
  float* partials = static_cast<float*>(workspace);
  float2* parts = p.parts > 1 ? reinterpret_cast<float2*>(partials + kBlocks) : nullptr;
  const int G = parts ? 32 : threads_per_row(C, k);
  const int whole = dZ ? one_pass_threads(Z, type, ldz, dZ, lddz, M, C, k) : 0;
  if (whole) {
    int* word = nullptr;
    rc = gc::tiles::error_word(&word);
    if (rc != GC_OK) return rc;
    const int smem = one_pass_bytes(whole, int(k));
    const unsigned ctas = unsigned(std::min<int64_t>(M, gc::kNumSMs * (whole == kLong ? 1 : std::min(4, 222 * 1024 / (smem + 2048)))));
    with_type(type, [&](auto t) {
      using T = decltype(t);
      auto run = [&](auto threads) {
        constexpr int kThreads = decltype(threads)::value;
        auto kern = distill_one_pass_kernel<T, kThreads>;
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, one_pass_bytes(kThreads, kOnePassList));
        if (e != cudaSuccess) rc = gc::fail(GC_ERR_CUDA, "gc_distill_forward: %s", cudaGetErrorString(e));
        else
          kern<<<ctas, 2 * kThreads + 64, smem, st>>>(p, reinterpret_cast<Stats*>(stats), partials, scale * temperature, static_cast<T*>(dZ), lddz,
                                                  int(pad), word);
      };
      if (whole == kLong) run(std::integral_constant<int, kLong>{});
      else run(std::integral_constant<int, kShort>{});
    });
    if (rc != GC_OK) return rc;
    distill_sum_kernel<<<1, 256, 0, st>>>(partials, int(ctas), scale * temperature * temperature, loss);
    return gc::check_launch("gc_distill_forward", 2);
  }
  const unsigned grid = grid_of(M, G);
  with_type(type, [&](auto t) {
    using T = decltype(t);
    if (parts) distill_part_kernel<T><<<dim3(unsigned(p.parts), unsigned(M)), kPart, 0, st>>>(p, parts);
    with_group(G, p.parts > 1, [&](auto gt) {
      constexpr int kG = decltype(gt)::value;
      Stats* const to = reinterpret_cast<Stats*>(stats);
      if constexpr (kG <= 32) {
        if (dZ) {
          const int smem = list_bytes(kG, int(k));
          auto kern = distill_forward_kernel<T, kG, true>;
          const cudaError_t e = allow_lists(kern, kG, smem);
          if (e != cudaSuccess) rc = gc::fail(GC_ERR_CUDA, "gc_distill_forward: %s", cudaGetErrorString(e));
          else kern<<<grid, 256, smem, st>>>(p, parts, to, partials, scale * temperature, static_cast<T*>(dZ), lddz, int(pad));
          return;
        }
      }
      distill_forward_kernel<T, kG, false><<<grid, kG > 32 ? kG : 256, 0, st>>>(p, parts, to, partials, 0.f, nullptr, 0, 0);
    });
  });
  if (rc != GC_OK) return rc;
  distill_sum_kernel<<<1, 256, 0, st>>>(partials, int(grid), scale * temperature * temperature, loss);
  return gc::check_launch("gc_distill_forward", parts ? 3 : 2);
}

int gc_distill_backward(const void* Z, int type, int64_t ldz, const void* top, int top_type, int64_t ldt, const void* index,
                        int index_bits, int64_t ldi, const float* stats, int64_t M, int64_t C, int64_t k, float temperature,
                        float scale, const float* grad_loss, void* dZ, int64_t lddz, int64_t pad, int dz_made, void* stream) {
  Problem p;
  const int rc = fill(p, "gc_distill_backward", Z, type, ldz, top, top_type, ldt, index, index_bits, ldi, M, C, k, temperature);
  if (rc != GC_OK) return rc;
  GC_REQUIRE(pad >= 0 && pad < 8 && lddz >= C + pad, "gc_distill_backward: leading dimension below the row length");
  if (M == 0) return GC_OK;
  GC_REQUIRE(stats && grad_loss && dZ, "gc_distill_backward: null pointer");
  GC_REQUIRE(gc::aligned16(stats), "gc_distill_backward: the statistics must be 16-byte aligned");
  const int G = p.parts > 1 ? kWide : threads_per_row(C, k);
  const int rows = G > 32 ? 1 : 256 / G;
  const int smem = list_bytes(G, int(k));
  // where dZ is mostly there already, as many CTAs as run at one time
  const unsigned grid = unsigned(std::min<int64_t>(gc::ceil_div(M * p.parts, rows), dz_made ? gc::kNumSMs * 4 : int64_t(1) << 30));
  int bad = GC_OK;
  with_type(type, [&](auto t) {
    using T = decltype(t);
    with_group(G, p.parts > 1, [&](auto gt) {
      constexpr int kG = decltype(gt)::value;
      auto kern = distill_backward_kernel<T, kG>;
      const cudaError_t e = allow_lists(kern, kG, smem);
      if (e != cudaSuccess) bad = gc::fail(GC_ERR_CUDA, "gc_distill_backward: %s", cudaGetErrorString(e));
      else
        kern<<<grid, kG > 32 ? kG : 256, smem, gc::as_stream(stream)>>>(p, reinterpret_cast<const Stats*>(stats), grad_loss,
                                                                         scale * temperature, static_cast<T*>(dZ), lddz, int(pad), dz_made != 0);
    });
  });
  return bad != GC_OK ? bad : gc::check_launch("gc_distill_backward");
}

}  // extern "C"
