// What the two kernels of the gated feed-forward block share: activations, and the entry to the form for few rows.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>

namespace gc {
namespace ffn {

// 2^x and 1 / x to 2^-22, one instruction each; results below 2^-126 are zero.
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats at a time: the packed instructions do both in one issue slot.
struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ F2(uint32_t a, uint32_t b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(a), "r"(b)); }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ F2 both(float x) { return F2(x, x); }
template <class F>
__device__ __forceinline__ F2 each(F2 a, F&& f) {
  float x, y;
  a.get(x, y);
  return F2(f(x), f(y));
}

// act(g) and, for the backward pass, its derivative.
template <int ACT>
__device__ __forceinline__ F2 activate(F2 g, F2& slope) {
  if constexpr (ACT == GC_ACT_SILU) {
    const F2 e = each(g * both(-1.4426950408889634f), [](float x) { return exp2_approx(x); });
    const F2 s = each(e + both(1.f), [](float x) { return rcp_approx(x); });
    const F2 a = g * s;
    slope = fma2(a, fma2(s, both(-1.f), both(1.f)), s);
    return a;
  } else if constexpr (ACT == GC_ACT_GELU) {
    // The normal distribution's tail beyond |g| is e^(-g^2/2) / 2 times erfcx(|g| / sqrt 2), and for erfcx a polynomial in t =
    // 1 / (1 + 0.44 x) was fitted here, the relative error made even over 0 <= x <= 13: 6e-6, and 9e-6 as evaluated in fp32, in the
    // far tail too, where 1 + erf would cancel.  The exponential is the one that the derivative needs.  (With erff the epilogue of the backward product set
    // its time: tensor cores 59 % active at K = 2048.)
    const F2 x = each(g, [](float v) { return fabsf(v); }) * both(0.70710678118654752f);
    const F2 t = each(fma2(x, both(0.44f), both(1.f)), [](float v) { return rcp_approx(v); });
    const F2 pdf = each(g * g * both(-0.72134752044448170f), [](float v) { return exp2_approx(v); });
    F2 q = both(-0.14544761f);
    q = fma2(q, t, both(0.34884202f));
    q = fma2(q, t, both(0.04260680f));
    q = fma2(q, t, both(0.26268032f));
    q = fma2(q, t, both(0.24277152f));
    q = fma2(q, t, both(0.24854454f));
    q = q * (t * (pdf * both(0.5f)));
    float g0, g1, q0, q1;
    g.get(g0, g1);
    q.get(q0, q1);
    const F2 cdf(g0 < 0.f ? q0 : 1.f - q0, g1 < 0.f ? q1 : 1.f - q1);
    slope = fma2(g * pdf, both(0.39894228040143268f), cdf);
    return g * cdf;
  } else {
    slope = each(g, [](float x) { return x > 0.f ? 1.f : 0.f; });
    return each(g, [](float x) { return x <= 0.f ? 0.f : x; });  // a NaN stays
  }
}
template <class F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  if (act == GC_ACT_SILU) f(std::integral_constant<int, GC_ACT_SILU>{});
  else if (act == GC_ACT_GELU) f(std::integral_constant<int, GC_ACT_GELU>{});
  else f(std::integral_constant<int, GC_ACT_RELU>{});
}

// What a forward pass leaves for the backward pass, in one buffer: G and U are kept as fp16 numbers with an exponent for every
// 32 columns of a row: eight times as exact as bf16 in as many bits, over the same range.
struct Saved {
  uint16_t* hidden;   // M x P bf16, P = H rounded up to a multiple of 8; for few rows what its rounding left follows, M x P
  uint16_t* gate_up;  // M x 2P
  int8_t* exps;       // [2][ceil(P / 32)][M]
};
// A magnitude as a float's bits; 0 for an infinity or a NaN, which any exponent keeps and which has no say in its neighbours'.
__device__ __forceinline__ uint32_t finite_bits(uint32_t v) { return (v & 0x7FFFFFFFu) < 0x7F800000u ? v & 0x7FFFFFFFu : 0u; }
// The exponent that 32 values with the largest magnitude `bits` (as a float's) take where `most`, the largest fp16 number they
// would be, overflows or falls below 2^-10, from where fp16 loses bits: it brings the largest to 2^14.  0 where it does not.
__device__ __forceinline__ int shared_exponent(uint32_t bits) {
  if (bits == 0) return 0;
  return max(int(bits >> 23) - 127 - 14, -126);
}
__device__ __forceinline__ bool fits_fp16(uint32_t most) { return most >= 0x1400u && most < 0x7C00u; }
// What is positive stays so: the smallest fp16 number stands for less.  relu's slope hangs on it, and a value of G below 2^-25
// beside one above 2^-10 would come back as zero.
__device__ __forceinline__ float stay_positive(float v) { return v > 0.f ? fmaxf(v, 0x1p-24f) : v; }
// 2^-e as two factors: alone it may not be a number.
__device__ __forceinline__ float2 unscale(int e) {
  return make_float2(__uint_as_float(uint32_t(127 - e / 2) << 23), __uint_as_float(uint32_t(127 - (e - e / 2)) << 23));
}

// Forward passes of up to 8 rows, which read every weight once and hardly compute, may run on CUDA cores (ffn_rows.cu); whether
// they do: few_rows().
constexpr int kFewRows = 8;
struct Rows {
  const void* x;  // M x D: bf16, or e4m3 with scales
  const void* w;  // bf16: D x 2H; e4m3: 2H x D
  const uint16_t* w_out;  // H x O
  const float* x_scale;
  const float* w_scale;
  float* hidden;     // M x H scratch, pitch `ldh` = P
  uint16_t* y;
  int64_t ldx, ldw, ldwout, ldh, ldy;
  int M, D, H, O, act;
  Saved saved;  // all null where nothing is kept (e4m3 keeps nothing)
};
int forward_few_rows(const Rows& r, bool e4m3, cudaStream_t st);

// On the tensor cores, with weights whose inputs run along their rows (16-byte aligned ones): Y (M x N) = X W^T with W N x K, all
// bf16; X and Y may lie as they like.
size_t rows_workspace(int64_t M, int64_t K, int64_t N);
int rows_times(const uint16_t* X, int64_t ldx, const uint16_t* W, int64_t ldw, int64_t M, int64_t K, int64_t N, uint16_t* Y,
               int64_t ldy, void* workspace, cudaStream_t st);
// The block with fp16 operands that are so times powers of two (exponents -126 to 127): X row by row, the weights output by output, and
// the hidden row, whose exponents have to bring it below 2^16.  X is M x D, Win 2H x D, Wout O x H, all of them in rows that
// are a multiple of 8 long; Y is bf16.
struct BlockFp16 {
  const uint16_t *x, *w_in, *w_out;
  const int *ex, *eh, *ein, *eout;  // value = stored * 2^exponent
};
size_t block_fp16_workspace(int64_t M, int64_t D, int64_t H, int64_t O);
int block_fp16(const BlockFp16& b, int64_t M, int64_t D, int64_t H, int64_t O, int act, uint16_t* Y, int64_t ldy, void* workspace,
               cudaStream_t st);

}  // namespace ffn
}  // namespace gc
