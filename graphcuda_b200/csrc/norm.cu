// Root-mean-square norm with the residual's addition, forward and backward.
//
//   h = x + r,  c = 1 / sqrt(mean(h^2) + eps),  y = h c w           (the new residual stream is h)
//   dh = c (dy w - hat mean(dy w hat)) + dstream,  hat = h c,  dx = dr = dh,  dw = sum over the rows of dy hat
//
// and, for y in 8 bits, one scale per row: s = max|y| / 448, q = e4m3(y / s).
//
// Bound by memory: every element is read once and written once and a handful of operations is done on it.  A row is
// held in the registers of a group of 8, 32 or 256 threads between the pass that sums its squares and the pass that
// scales it, 8 consecutive elements (16 or 32 bytes) per thread and load; rows whose length, pitch or base do not allow that
// are read 4 elements at a time, or element by element, in the same kernels.  A group that has several rows reads the next
// one before it works on this one, where registers allow: without that a row's loads, its sum and its stores follow each
// other, and wide rows came to 4.3 TB/s.  Rows of more than 8192 elements are read twice instead.  Sums and statistics are
// fp32; h enters the statistics, y and the gradients unrounded, also where the stream that is stored has 16 bits (the backward
// pass then adds x and r again: from a stream rounded to bf16 the weight gradient would be off by 2e-3).
//
// 169,343 x 256, bf16 beside an fp32 stream: forward 75 us (6.9 TB/s), backward 111 (6.2 TB/s; reading ahead by asynchronous copies
// into shared memory 157, vectors of 4 that lie side by side in fp32 too 115).  8192 x 4096 to 8 bits: 39 us (6.0 TB/s).
//
// dw: a thread keeps the same columns for all rows of its group and sums them in registers; groups are added through
// shared memory, CTAs by a second kernel, both in a fixed order.
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>

namespace {

constexpr int kThreads = 256;
constexpr int kMaxHeld = 8192;  // widest row that is held in registers

using bf16 = __nv_bfloat16;

// VEC (8, 4 or 1) elements as they lie in memory, read in accesses of up to 16 bytes
template <class T, int VEC>
struct alignas(VEC * sizeof(T) > 16 ? 16 : VEC * sizeof(T)) Raw {
  T v[VEC];
};
template <class T, int VEC>
__device__ __forceinline__ void widen(const Raw<T, VEC>& r, float (&v)[VEC]) {
#pragma unroll
  for (int k = 0; k < VEC; ++k) v[k] = float(r.v[k]);
}
template <class T, int VEC>
__device__ __forceinline__ void load(const T* p, Raw<T, VEC>& r) {
  constexpr int kBytes = VEC * sizeof(T);
  if constexpr (kBytes >= 16) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(&r)[i] = reinterpret_cast<const uint4*>(p)[i];
  } else if constexpr (kBytes == 8) {
    *reinterpret_cast<uint2*>(&r) = *reinterpret_cast<const uint2*>(p);
  } else {
    r.v[0] = *p;
  }
}
template <int VEC, class T>
__device__ __forceinline__ void load(const T* p, float (&v)[VEC]) {
  Raw<T, VEC> r;
  load(p, r);
  widen(r, v);
}
template <int VEC>
__device__ __forceinline__ void store_f32(float* p, const float (&v)[VEC]) {
  if constexpr (VEC > 1) {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) *reinterpret_cast<float4*>(p + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
  } else {
    *p = v[0];
  }
}
template <int VEC>
__device__ __forceinline__ void store_bf16(bf16* p, const float (&v)[VEC]) {
  if constexpr (VEC > 1) {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k) {
      const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
      w[k] = *reinterpret_cast<const uint32_t*>(&t);
    }
    if constexpr (VEC == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
    *p = __float2bfloat16_rn(v[0]);
  }
}
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&v)[VEC]) {
  if constexpr (VEC > 1) {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k)
      w[k] = uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(v[4 * k], v[4 * k + 1]), __NV_SATFINITE, __NV_E4M3)) |
             uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(v[4 * k + 2], v[4 * k + 3]), __NV_SATFINITE, __NV_E4M3)) << 16;
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  } else {
    *p = __nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
  }
}
template <int VEC>
__device__ __forceinline__ void store_as(void* base, int type, int64_t at, const float (&v)[VEC]) {
  if (type == GC_TYPE_F32) store_f32<VEC>(static_cast<float*>(base) + at, v);
  else if (type == GC_TYPE_BF16) store_bf16<VEC>(static_cast<bf16*>(base) + at, v);
  else store_e4m3<VEC>(static_cast<uint8_t*>(base) + at, v);
}

struct Sum {
  using T = float;
  static __device__ T of(T a, T b) { return a + b; }
};
// The largest of |v| by its bits: a NaN is above infinity and stays.
struct MaxBits {
  using T = uint32_t;
  static __device__ T of(T a, T b) { return max(a, b); }
};
// Over a group of G threads; every thread gets the result.  `sm`: one word per warp, for groups of whole CTAs; two uses of the
// same words have a barrier between them (another reduction's).
template <int G, class Op>
__device__ __forceinline__ typename Op::T reduce(typename Op::T v, typename Op::T* sm) {
  constexpr int kIn = G < 32 ? G : 32;
#pragma unroll
  for (int d = kIn / 2; d > 0; d /= 2) v = Op::of(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
  if constexpr (G > 32) {
    static_assert(G == kThreads, "a group is part of a warp, a warp, or the CTA");
    if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = v;
    __syncthreads();
    v = sm[0];
#pragma unroll
    for (int w = 1; w < G / 32; ++w) v = Op::of(v, sm[w]);
  }
  return v;
}

// The scale of a row in 8 bits and what its elements are multiplied by: products with rounded reciprocals, which put no more codes on
// the wrong side of a boundary than a quotient's own rounding (28 against 25 of the 34 M of 8192 x 4096, PyTorch's quotients 28), where
// dividing every element takes 60 us instead of 41.  A row whose scale would be subnormal is stored
// as zeros; one with a NaN has a NaN for its scale, one with an infinity an infinity.
__device__ __forceinline__ float2 scale_of(uint32_t top_bits) {
  const float s = __uint_as_float(top_bits) * (1.0f / 448.0f);
  if (s < 1.17549435e-38f) return make_float2(0.f, 0.f);
  return make_float2(s, 1.0f / s);
}

struct Forward {
  const void* x;
  const void* r;  // null: no residual
  const float* w;
  void* y;
  void* stream_out;  // null: not written
  float* rstd;       // null: not written
  float* scale;      // for y in 8 bits
  int64_t ldx, ldr, ldy, lds;
  int64_t M;
  int N, y_type;
  float eps;
};

// A row at a time per group of G threads, held in ITEMS vectors of VEC elements per thread.
template <class TX, class TS, int G, int VEC, int ITEMS>
__global__ void __launch_bounds__(kThreads)
rms_norm_kernel(Forward f) {
  __shared__ float sum_s[2][kThreads / 32];
  __shared__ uint32_t top_s[2][kThreads / 32];
  // bytes per thread that are read ahead; groups within a warp have enough rows in flight without
  constexpr bool kAhead = G == kThreads && ITEMS * VEC * (sizeof(TX) + sizeof(TS)) <= 128;
  const int in_group = threadIdx.x % G;
  auto column = [&](int i) { return (i * G + in_group) * VEC; };
  Raw<TX, VEC> xr[ITEMS];
  Raw<TS, VEC> rr[ITEMS];
  auto read = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (row < f.M && column(i) < f.N) {
        load(static_cast<const TX*>(f.x) + row * f.ldx + column(i), xr[i]);
        if (f.r) load(static_cast<const TS*>(f.r) + row * f.ldr + column(i), rr[i]);
      }
  };
  const int64_t step = int64_t(gridDim.x) * (kThreads / G);
  int64_t first = int64_t(blockIdx.x) * (kThreads / G);
  if (kAhead) read(first + threadIdx.x / G);
  for (int turn = 0; first < f.M; first += step, turn ^= 1) {  // the same count for all of a CTA
    const int64_t row = first + threadIdx.x / G;
    if (!kAhead) read(row);
    const bool live = row < f.M;  // a group of the last CTA may have none, and takes part in the shuffles
    float h[ITEMS][VEC];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const bool ok = live && column(i) < f.N;
      float add[VEC];
      widen(xr[i], h[i]);
      if (f.r) widen(rr[i], add);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        h[i][k] = !ok ? 0.f : f.r ? h[i][k] + add[k] : h[i][k];
        s += h[i][k] * h[i][k];
      }
    }
    if (kAhead) read(row + step);
    if (f.stream_out && live) {
      TS* out = static_cast<TS*>(f.stream_out) + row * f.lds;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (column(i) < f.N) {
          if constexpr (sizeof(TS) == 4) store_f32<VEC>(out + column(i), h[i]);
          else store_bf16<VEC>(out + column(i), h[i]);
        }
    }
    s = reduce<G, Sum>(s, sum_s[turn]);
    const float c = rsqrtf(s / float(f.N) + f.eps);
    if (f.rstd && live && in_group == 0) f.rstd[row] = c;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (column(i) < f.N) {
        float w[VEC];
        load<VEC>(f.w + column(i), w);
#pragma unroll
        for (int k = 0; k < VEC; ++k) h[i][k] = h[i][k] * c * w[k];
      }
    if (f.y_type == GC_TYPE_E4M3) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          if (column(i) < f.N) top = max(top, __float_as_uint(h[i][k]) & 0x7FFFFFFFu);
      const float2 sc = scale_of(reduce<G, MaxBits>(top, top_s[turn]));
      if (live && in_group == 0) f.scale[row] = sc.x;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) h[i][k] *= sc.y;
    }
    if (live)
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (column(i) < f.N) store_as<VEC>(f.y, f.y_type, row * f.ldy + column(i), h[i]);
    if (G < kThreads) break;  // the grid has a group for every row: see launch_forward
  }
}

// Rows of more than kMaxHeld elements: a CTA reads the row for its sum, and again to scale it (three times in 8 bits).
template <class TX, class TS>
__global__ void __launch_bounds__(kThreads)
rms_norm_long_kernel(Forward f) {
  __shared__ float sum_s[kThreads / 32];
  __shared__ uint32_t top_s[kThreads / 32];
  const int64_t row = blockIdx.x;
  const TX* x = static_cast<const TX*>(f.x) + row * f.ldx;
  const TS* r = f.r ? static_cast<const TS*>(f.r) + row * f.ldr : nullptr;
  auto at = [&](int n) {
    float v[1], a[1] = {0.f};
    load<1>(x + n, v);
    if (r) load<1>(r + n, a);
    return r ? v[0] + a[0] : v[0];
  };
  float s = 0.f;
  for (int n = threadIdx.x; n < f.N; n += kThreads) {
    const float h[1] = {at(n)};
    s += h[0] * h[0];
  }
  s = reduce<kThreads, Sum>(s, sum_s);
  const float c = rsqrtf(s / float(f.N) + f.eps);
  if (f.rstd && threadIdx.x == 0) f.rstd[row] = c;
  float up = 1.f;
  if (f.y_type == GC_TYPE_E4M3) {
    uint32_t top = 0;
    for (int n = threadIdx.x; n < f.N; n += kThreads) top = max(top, __float_as_uint(at(n) * c * f.w[n]) & 0x7FFFFFFFu);
    const float2 sc = scale_of(reduce<kThreads, MaxBits>(top, top_s));
    if (threadIdx.x == 0) f.scale[row] = sc.x;
    up = sc.y;
  }
  for (int n = threadIdx.x; n < f.N; n += kThreads) {
    const float h[1] = {at(n)};  // before the stream is written, which may be the residual itself
    if (f.stream_out) {
      if constexpr (sizeof(TS) == 4) store_f32<1>(static_cast<float*>(f.stream_out) + row * f.lds + n, h);
      else store_bf16<1>(static_cast<bf16*>(f.stream_out) + row * f.lds + n, h);
    }
    float y[1] = {h[0] * c * f.w[n]};
    if (f.y_type == GC_TYPE_E4M3) y[0] *= up;
    store_as<1>(f.y, f.y_type, row * f.ldy + n, y);
  }
}

struct Backward {
  const void* dy;
  const void* dstream;  // null: none; of h's type
  const void* h;        // the stream, or x where the stream's rounding would show
  const void* r;        // then the residual; null: none
  const float* w;
  const float* rstd;
  void* dx;    // null: not wanted
  void* dres;  // null: dx serves
  float* dw;   // partial sums [CTA][N], or the gradient itself when there is one CTA; null: not wanted
  int64_t lddy, ldds, ldh, ldr, lddx, lddr;
  int64_t M;
  int N, dx_type;
};

// CTAs of the backward kernel per SM that its registers have to allow, by the elements that a thread holds; and how many are
// launched per SM, a multiple of what is resident then (a grid of one and a third times that leaves most of the GPU idle
// at the end: 169,343 x 256 with 3 resident of 4 142 us, 2 of 4 109).
constexpr int least_resident(int held) { return held <= 4 ? 4 : held <= 8 ? 1 : held <= 16 ? 2 : 1; }
constexpr int ctas_per_sm(int held) { return held <= 8 ? 4 : held <= 16 ? 2 : 1; }

// RES: r is there.  Rows are dealt to the groups of a grid of at most some CTAs per SM.
template <class TH, bool RES, class TY, int G, int VEC, int ITEMS>
__global__ void __launch_bounds__(kThreads, least_resident(ITEMS * VEC))
rms_norm_backward_kernel(Backward b) {
  constexpr int kGroups = kThreads / G;
  constexpr bool kAhead = ITEMS * VEC * (sizeof(TH) * (RES ? 2 : 1) + sizeof(TY)) <= 128;  // as above
  // dstream is used last: where registers are short (two vectors a thread, two CTAs an SM) its loads go out with the row's own
  // work instead (8192 x 4096: 60 us against 85 in bf16, 96 against 126 in fp32; 20,000 x 2048, which has the registers: 110 against 132)
  constexpr bool kStreamAhead = kAhead && ITEMS * VEC <= 8;
  __shared__ float sum_s[2][kThreads / 32];
  __shared__ float dw_s[G < kThreads ? kThreads * VEC : 1];
  const int in_group = threadIdx.x % G, group = threadIdx.x / G;
  auto column = [&](int i) { return (i * G + in_group) * VEC; };
  float dw[ITEMS][VEC];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int k = 0; k < VEC; ++k) dw[i][k] = 0.f;
  Raw<TH, VEC> hr[ITEMS], rr[ITEMS], dr[ITEMS];
  Raw<TY, VEC> yr[ITEMS];
  float cr = 0.f;
  auto read = [&](int64_t row) {
    if (row >= b.M) return;
    cr = b.rstd[row];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int n = column(i);
      if (n < b.N) {
        load(static_cast<const TH*>(b.h) + row * b.ldh + n, hr[i]);
        load(static_cast<const TY*>(b.dy) + row * b.lddy + n, yr[i]);
        if (kStreamAhead && b.dstream) load(static_cast<const TH*>(b.dstream) + row * b.ldds + n, dr[i]);
        if constexpr (RES) load(static_cast<const TH*>(b.r) + row * b.ldr + n, rr[i]);
      }
    }
  };
  const int64_t step = int64_t(gridDim.x) * kGroups;
  int64_t first = int64_t(blockIdx.x) * kGroups;
  if (kAhead) read(first + group);
  for (int turn = 0; first < b.M; first += step, turn ^= 1) {  // the same count for all of a CTA
    const int64_t row = first + group;
    if (!kAhead) read(row);
    const bool live = row < b.M;
    float ds[ITEMS][VEC];
    Raw<TH, VEC> late[ITEMS];
    if (!kStreamAhead && b.dstream && live)
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (column(i) < b.N) load(static_cast<const TH*>(b.dstream) + row * b.ldds + column(i), late[i]);
    float h[ITEMS][VEC], g[ITEMS][VEC];
    const float c = live ? cr : 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const bool ok = live && column(i) < b.N;
      float add[VEC];
      widen(hr[i], h[i]);
      widen(yr[i], g[i]);
      if constexpr (RES) widen(rr[i], add);
      if (kStreamAhead && b.dstream) widen(dr[i], ds[i]);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        if (RES) h[i][k] += add[k];
        if (!ok) h[i][k] = g[i][k] = 0.f;
        if (kStreamAhead && !b.dstream) ds[i][k] = 0.f;
      }
    }
    if (kAhead) read(row + step);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      float w[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) w[k] = 0.f;
      if (column(i) < b.N) load<VEC>(b.w + column(i), w);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float hat = h[i][k] * c;
        dw[i][k] += g[i][k] * hat;
        g[i][k] *= w[k];
        s += g[i][k] * hat;
        h[i][k] = hat;
      }
    }
    s = reduce<G, Sum>(s, sum_s[turn]);
    const float mean = s / float(b.N);
    if (live && b.dx)
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (column(i) < b.N) {
          float d[VEC];
#pragma unroll
          for (int k = 0; k < VEC; ++k)
            if (!kStreamAhead) ds[i][k] = 0.f;
          if (!kStreamAhead && b.dstream) widen(late[i], ds[i]);
#pragma unroll
          for (int k = 0; k < VEC; ++k) d[k] = c * (g[i][k] - h[i][k] * mean) + ds[i][k];
          store_as<VEC>(b.dx, b.dx_type, row * b.lddx + column(i), d);
          if (b.dres) store_as<VEC>(b.dres, sizeof(TH) == 4 ? GC_TYPE_F32 : GC_TYPE_BF16, row * b.lddr + column(i), d);
        }
  }
  if (!b.dw) return;
  float* out = b.dw + int64_t(blockIdx.x) * b.N;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if constexpr (G < kThreads) {  // the CTA's groups, in their order
      __syncthreads();
#pragma unroll
      for (int k = 0; k < VEC; ++k) dw_s[(group * VEC + k) * G + in_group] = dw[i][k];
      __syncthreads();
      for (int e = threadIdx.x; e < G * VEC; e += kThreads) {  // element e: vector e % G, place e / G
        float t = 0.f;
#pragma unroll 8
        for (int q = 0; q < kGroups; ++q) t += dw_s[q * VEC * G + e];
        const int n = (i * G + e % G) * VEC + e / G;
        if (n < b.N) out[n] = t;
      }
    } else if (column(i) < b.N) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) out[column(i) + k] = dw[i][k];
    }
  }
}

// dw = the sum of the CTAs' partial rows: 32 columns per CTA, 32 rows side by side, added in a fixed order.
__global__ void __launch_bounds__(1024)
rms_norm_dw_kernel(const float* __restrict__ partial, int parts, int N, float* __restrict__ dw) {
  __shared__ float sm[32][33];
  const int lane = threadIdx.x % 32, q = threadIdx.x / 32, n = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (n < N) {
#pragma unroll 8
    for (int p = q; p < parts; p += 32) s += partial[int64_t(p) * N + n];
  }
  sm[lane][q] = s;
  __syncthreads();
  s = sm[q][lane];  // column q, part `lane`
#pragma unroll
  for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
  if (lane == 0 && blockIdx.x * 32 + q < N) dw[blockIdx.x * 32 + q] = s;
}

// Rows of more than kMaxHeld elements, read twice; the weight gradient by columns in a kernel of its own.
template <class TH, bool RES, class TY>
__global__ void __launch_bounds__(kThreads)
rms_norm_backward_long_kernel(Backward b) {
  __shared__ float sum_s[kThreads / 32];
  const int64_t row = blockIdx.x;
  const float c = b.rstd[row];
  auto at = [&](int n, float& hat, float& g) {
    float v[1], r[1] = {0.f};
    load<1>(static_cast<const TH*>(b.h) + row * b.ldh + n, v);
    if constexpr (RES) load<1>(static_cast<const TH*>(b.r) + row * b.ldr + n, r);
    hat = (RES ? v[0] + r[0] : v[0]) * c;
    load<1>(static_cast<const TY*>(b.dy) + row * b.lddy + n, v);
    g = v[0] * b.w[n];
  };
  float s = 0.f, hat, g;
  for (int n = threadIdx.x; n < b.N; n += kThreads) {
    at(n, hat, g);
    s += g * hat;
  }
  const float mean = reduce<kThreads, Sum>(s, sum_s) / float(b.N);
  for (int n = threadIdx.x; n < b.N; n += kThreads) {
    at(n, hat, g);
    float d[1] = {0.f};
    if (b.dstream) load<1>(static_cast<const TH*>(b.dstream) + row * b.ldds + n, d);
    d[0] += c * (g - hat * mean);
    store_as<1>(b.dx, b.dx_type, row * b.lddx + n, d);
    if (b.dres) store_as<1>(b.dres, sizeof(TH) == 4 ? GC_TYPE_F32 : GC_TYPE_BF16, row * b.lddr + n, d);
  }
}
template <class TH, bool RES, class TY>
__global__ void __launch_bounds__(kThreads)
rms_norm_dw_long_kernel(Backward b) {
  const int n = blockIdx.x * kThreads + threadIdx.x;
  if (n >= b.N) return;
  const int64_t per = (b.M + gridDim.y - 1) / gridDim.y;
  float s = 0.f;
  for (int64_t row = blockIdx.y * per; row < min(b.M, (blockIdx.y + 1) * per); ++row) {
    float v[1], r[1] = {0.f}, g[1];
    load<1>(static_cast<const TH*>(b.h) + row * b.ldh + n, v);
    if constexpr (RES) load<1>(static_cast<const TH*>(b.r) + row * b.ldr + n, r);
    load<1>(static_cast<const TY*>(b.dy) + row * b.lddy + n, g);
    s += g[0] * ((RES ? v[0] + r[0] : v[0]) * b.rstd[row]);
  }
  b.dw[int64_t(blockIdx.y) * b.N + n] = s;
}

// ------------------------------------------------------------------ host
bool known(int type, bool eight) { return type == GC_TYPE_F32 || type == GC_TYPE_BF16 || (eight && type == GC_TYPE_E4M3); }
size_t size_of(int type) { return type == GC_TYPE_F32 ? 4 : type == GC_TYPE_BF16 ? 2 : 1; }

// How many elements at a time rows of this matrix can be read in: 8, 4 or 1.
int vector_of(const void* p, int type, int64_t ld) {
  if (!p) return 8;
  for (int vec = 8; vec > 1; vec /= 2) {
    const size_t unit = std::min<size_t>(16, vec * size_of(type));
    if (reinterpret_cast<uintptr_t>(p) % unit == 0 && size_t(ld) * size_of(type) % unit == 0) return vec;
  }
  return 1;
}
int vector_of(int64_t N) { return N % 8 == 0 ? 8 : N % 4 == 0 ? 4 : 1; }

// The group that holds a row, and how many vectors each of its threads has.  Smallest that fits: a row of 64 elements
// takes 8 threads of a warp, one of up to 1024 a warp, beyond that the CTA.
template <class F>
void with_shape(int vec, int N, F&& go) {
#define GC_SHAPE(G, V, I) go(std::integral_constant<int, G>{}, std::integral_constant<int, V>{}, std::integral_constant<int, I>{})
  if (vec == 4) {
    if (N <= 32) GC_SHAPE(8, 4, 1);
    else if (N <= 128) GC_SHAPE(32, 4, 1);
    else if (N <= 512) GC_SHAPE(32, 4, 4);
    else if (N <= 1024) GC_SHAPE(32, 4, 8);
    else if (N <= 4096) GC_SHAPE(256, 4, 4);
    else GC_SHAPE(256, 4, 8);
  } else if (vec == 8) {
    if (N <= 64) GC_SHAPE(8, 8, 1);
    else if (N <= 256) GC_SHAPE(32, 8, 1);
    else if (N <= 512) GC_SHAPE(32, 8, 2);
    else if (N <= 1024) GC_SHAPE(32, 8, 4);
    else if (N <= 2048) GC_SHAPE(256, 8, 1);
    else if (N <= 4096) GC_SHAPE(256, 8, 2);
    else GC_SHAPE(256, 8, 4);
  } else {
    if (N <= 64) GC_SHAPE(8, 1, 8);
    else if (N <= 256) GC_SHAPE(32, 1, 8);
    else if (N <= 1024) GC_SHAPE(32, 1, 32);
    else if (N <= 2048) GC_SHAPE(256, 1, 8);
    else GC_SHAPE(256, 1, 32);
  }
#undef GC_SHAPE
}

template <class TX, class TS>
int launch_forward(const Forward& f, int vec, cudaStream_t st) {
  if (f.N > kMaxHeld) {
    if (f.M > 0x7FFFFFFF) return gc::fail(GC_ERR_UNSUPPORTED, "gc_rms_norm_forward: too many rows");
    rms_norm_long_kernel<TX, TS><<<unsigned(f.M), kThreads, 0, st>>>(f);
  } else {
    with_shape(vec, f.N, [&](auto g, auto v, auto items) {
      constexpr int G = decltype(g)::value;
      // A CTA per row: a grid that the SMs hold, which reads ahead.  Smaller groups have enough in flight as it is, with one
      // row each (169,343 x 256, bf16 + fp32 -> bf16: 76 us, 86 as a loop).
      const int64_t most = G == kThreads ? gc::kNumSMs * 8 : 0x7FFFFFFF;
      const unsigned blocks = unsigned(std::min<int64_t>(gc::ceil_div(f.M, kThreads / G), most));
      rms_norm_kernel<TX, TS, G, decltype(v)::value, decltype(items)::value><<<blocks, kThreads, 0, st>>>(f);
    });
  }
  return gc::check_launch("gc_rms_norm_forward");
}

// Partial rows of the weight gradient that a backward launch leaves, at most.
int64_t most_parts(int64_t M, int64_t N) {
  return N > kMaxHeld ? std::min<int64_t>(gc::ceil_div(M, 64), 64) : std::min<int64_t>(M, gc::kNumSMs * 4);
}

template <class TH, bool RES, class TY>
int launch_backward(Backward b, int vec, float* dw, float* partial, cudaStream_t st) {
  int64_t ctas = most_parts(b.M, b.N);
  b.dw = !dw ? nullptr : ctas == 1 ? dw : partial;
  int launches = 0;
  if (b.N > kMaxHeld) {
    if (b.M > 0x7FFFFFFF) return gc::fail(GC_ERR_UNSUPPORTED, "gc_rms_norm_backward: too many rows");
    if (b.dx) {
      rms_norm_backward_long_kernel<TH, RES, TY><<<unsigned(b.M), kThreads, 0, st>>>(b);
      ++launches;
    }
    if (dw) {
      rms_norm_dw_long_kernel<TH, RES, TY><<<dim3(unsigned(gc::ceil_div(b.N, kThreads)), unsigned(ctas)), kThreads, 0, st>>>(b);
      ++launches;
    }
  } else {
    with_shape(vec, b.N, [&](auto g, auto v, auto items) {
      constexpr int G = decltype(g)::value, V = decltype(v)::value, I = decltype(items)::value;
      ctas = std::min<int64_t>(gc::ceil_div(b.M, kThreads / G), gc::kNumSMs * ctas_per_sm(V * I));
      b.dw = !dw ? nullptr : ctas == 1 ? dw : partial;
      rms_norm_backward_kernel<TH, RES, TY, G, V, I><<<unsigned(ctas), kThreads, 0, st>>>(b);
    });
    ++launches;
  }
  if (dw && ctas > 1) {
    rms_norm_dw_kernel<<<unsigned(gc::ceil_div(b.N, 32)), 1024, 0, st>>>(partial, int(ctas), b.N, dw);
    ++launches;
  }
  return gc::check_launch("gc_rms_norm_backward", launches);
}

}  // namespace

extern "C" {

int gc_rms_norm_forward(const void* x, int x_type, int64_t ldx, const void* residual, int64_t ldr, int stream_type,
                        const float* weight, int64_t M, int64_t N, double eps, void* y, int y_type, int64_t ldy,
                        void* stream_out, int64_t lds, float* rstd, float* scale, void* stream) {
  GC_REQUIRE(M >= 0 && N >= 0, "gc_rms_norm_forward: negative size");
  GC_REQUIRE(known(x_type, false) && known(stream_type, false) && known(y_type, true), "gc_rms_norm_forward: unknown type");
  GC_REQUIRE(x_type == stream_type || (residual && x_type == GC_TYPE_BF16),
             "gc_rms_norm_forward: x has the stream's type, or is bf16 beside an fp32 stream");
  if (M == 0 || N == 0) return GC_OK;
  GC_REQUIRE(N < (int64_t(1) << 31) - 8192, "gc_rms_norm_forward: rows of 2^31 elements and more are not served");
  GC_REQUIRE(x && weight && y, "gc_rms_norm_forward: null pointer");
  GC_REQUIRE(y_type != GC_TYPE_E4M3 || scale, "gc_rms_norm_forward: 8-bit rows need room for their scales");
  GC_REQUIRE(ldx >= N && ldy >= N && (!residual || ldr >= N) && (!stream_out || lds >= N),
             "gc_rms_norm_forward: leading dimension below the row length");
  Forward f{x, residual, weight, y, stream_out, rstd, scale, ldx, ldr, ldy, lds, M, int(N), y_type, float(eps)};
  const int vec = std::min({vector_of(N), vector_of(x, x_type, ldx), vector_of(residual, stream_type, ldr),
                            vector_of(y, y_type, ldy), vector_of(stream_out, stream_type, lds), vector_of(weight, GC_TYPE_F32, 8)});
  const cudaStream_t st = gc::as_stream(stream);
  if (x_type == GC_TYPE_F32) return launch_forward<float, float>(f, vec, st);
  if (stream_type == GC_TYPE_F32) return launch_forward<bf16, float>(f, vec, st);
  return launch_forward<bf16, bf16>(f, vec, st);
}

size_t gc_rms_norm_backward_workspace_bytes(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0) return 0;
  const int64_t ctas = most_parts(M, N);
  return ctas > 1 ? size_t(ctas) * size_t(N) * sizeof(float) : 0;
}

int gc_rms_norm_backward(const void* dy, int dy_type, int64_t lddy, const void* dstream, int64_t ldds, const void* h,
                         int64_t ldh, const void* residual, int64_t ldr, int stream_type, const float* weight,
                         const float* rstd, int64_t M, int64_t N, void* dx, int dx_type, int64_t lddx, void* dresidual,
                         int64_t lddr, float* dweight, void* workspace, size_t workspace_bytes, void* stream) {
  GC_REQUIRE(M >= 0 && N >= 0, "gc_rms_norm_backward: negative size");
  GC_REQUIRE(known(dy_type, false) && known(stream_type, false) && known(dx_type, false),
             "gc_rms_norm_backward: unknown type");
  const cudaStream_t st = gc::as_stream(stream);
  if (N == 0) return GC_OK;
  GC_REQUIRE(N < (int64_t(1) << 31) - 8192, "gc_rms_norm_backward: rows of 2^31 elements and more are not served");
  if (M == 0) {
    if (dweight && cudaMemsetAsync(dweight, 0, size_t(N) * sizeof(float), st) != cudaSuccess)
      return gc::fail(GC_ERR_CUDA, "gc_rms_norm_backward: %s", cudaGetErrorString(cudaGetLastError()));
    return GC_OK;
  }
  GC_REQUIRE(dy && h && weight && rstd, "gc_rms_norm_backward: null pointer");
  GC_REQUIRE(!residual || stream_type == GC_TYPE_BF16,
             "gc_rms_norm_backward: an fp32 stream is exact, and taken instead of x and the residual");
  GC_REQUIRE(dx || !dresidual, "gc_rms_norm_backward: dresidual alone is what dx of that type would be");
  GC_REQUIRE(lddy >= N && ldh >= N && (!dstream || ldds >= N) && (!residual || ldr >= N) && (!dx || lddx >= N) &&
                 (!dresidual || lddr >= N),
             "gc_rms_norm_backward: leading dimension below the row length");
  if (!dx && !dweight) return GC_OK;
  const size_t need = dweight ? gc_rms_norm_backward_workspace_bytes(M, N) : 0;
  if (need && (!workspace || workspace_bytes < need))
    return gc::fail(GC_ERR_WORKSPACE, "gc_rms_norm_backward: workspace missing or smaller than its query says");
  GC_REQUIRE(!need || reinterpret_cast<uintptr_t>(workspace) % 4 == 0, "gc_rms_norm_backward: workspace is not aligned");
  Backward b{dy, dstream, h, residual, weight, rstd, dx, dresidual, nullptr, lddy, ldds, ldh, ldr, lddx, lddr, M, int(N),
             dx_type};
  const int vec = std::min({vector_of(N), vector_of(dy, dy_type, lddy), vector_of(dstream, stream_type, ldds),
                            vector_of(h, stream_type, ldh), vector_of(residual, stream_type, ldr),
                            vector_of(dx, dx_type, lddx), vector_of(dresidual, stream_type, lddr),
                            vector_of(weight, GC_TYPE_F32, 8)});
  float* partial = static_cast<float*>(workspace);
  const bool y32 = dy_type == GC_TYPE_F32;
  if (stream_type == GC_TYPE_F32)
    return y32 ? launch_backward<float, false, float>(b, vec, dweight, partial, st)
               : launch_backward<float, false, bf16>(b, vec, dweight, partial, st);
  if (residual)
    return y32 ? launch_backward<bf16, true, float>(b, vec, dweight, partial, st)
               : launch_backward<bf16, true, bf16>(b, vec, dweight, partial, st);
  return y32 ? launch_backward<bf16, false, float>(b, vec, dweight, partial, st)
             : launch_backward<bf16, false, bf16>(b, vec, dweight, partial, st);
}

}  // extern "C"
