// The gated feed-forward block for a few rows: what a server runs for single vertices.
//
// Bound by memory: with up to 8 rows every weight is read once and used for a handful of multiply-adds, so the products run on
// CUDA cores, in fp32 (the product between the launches too: it is small, and no tensor core asks for 16 bits), with as many
// loads in flight as the SMs hold; a tile of the tensor cores would be empty.  Two launches: G, U and their product; then Y.
// The second starts while the first still runs, brings its weights into the L2, which do not depend on it, and waits.
// One row through 2048 -> 8192 -> 2048, 100 MB of weights that are not in the L2: 23.6 us by the call, 4.3 TB/s.
//
// Weights with K down the rows (bf16): a CTA has 64 output columns (of G and of U), its warps take blocks of 8 rows in turn, and a
// lane holds 8 columns of 8 rows: 16-byte loads, whole 128-byte lines per row, and the 8 values of x in one load too.
// Blocks are also dealt to the CTAs of a cluster, up to 8, where the columns alone would not fill the GPU; their sums meet
// in shared memory across the cluster, in a fixed order.
// Weights with K along the rows (e4m3): a warp per column of G and of U.
#include "ffn_internal.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

namespace {

using namespace gc::ffn;
using bf16 = __nv_bfloat16;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kCols = 64;  // output columns of a CTA

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Lets the next launch begin; waits until the one before has ended and its results can be read.
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A float of the CTA of that rank in the cluster, at the place that `p` has in this one.
__device__ __forceinline__ float peer_load(const float* p, uint32_t rank) {
  uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(p)), there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
  return v;
}
// One value per lane to fp16 with a power of two for the warp, which is returned.  sign: see stay_positive.
__device__ __forceinline__ int pack_fp16(float v, bool sign, __half& out) {
  out = __float2half_rn(sign ? stay_positive(v) : v);
  const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, uint32_t(__half_as_ushort(out)) & 0x7FFFu);
  if (fits_fp16(most)) return 0;
  const int e = shared_exponent(__reduce_max_sync(0xFFFFFFFFu, finite_bits(__float_as_uint(v))));
  const float2 f = unscale(e);
  v = v * f.x * f.y;
  out = __float2half_rn(sign ? stay_positive(v) : v);
  return e;
}
__device__ __forceinline__ float gated(float g, float u, int act) {
  float a = 0.f, unused;
  with_activation(act, [&](auto t) {
    F2 slope;
    activate<decltype(t)::value>(F2(g, g), slope).get(a, unused);
  });
  return a * u;
}

// GATED: hidden (M x N, fp32) = act(x Wg) * (x Wu) with W = [Wg | Wu], x in bf16, and what `keep` asks for; else out (M x N, bf16)
// = hidden W.  VEC: rows of W in 16-byte accesses, N a multiple of 8.
template <bool GATED, int MR, bool VEC>
__global__ void __launch_bounds__(kThreads)
ffn_rows_kernel(const std::conditional_t<GATED, bf16, float>* __restrict__ x, int64_t ldx, const bf16* __restrict__ w,
                int64_t ldw, std::conditional_t<GATED, float, bf16>* __restrict__ out, int64_t ldo, int M, int K, int N, int act, int ctas, int x_vec, Saved keep) {
  constexpr int kLanes = GATED ? 16 : 8;   // to a row of W
  constexpr int kSubs = 32 / kLanes;       // blocks of 8 rows that a warp reads at once
  constexpr int kWidth = GATED ? 2 * kCols : kCols;
  __shared__ float sums_s[kWarps][MR][kWidth];
  __shared__ float part_s[MR][kWidth];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t rank = ctas > 1 ? cluster_rank() : 0;
  const int col0 = int(blockIdx.x / ctas) * kCols;
  const int place = lane % kLanes, col = col0 + place % 8 * 8;
  const bf16* base = w + (GATED && place >= 8 ? N : 0) + col;
  const int blocks = (K + 7) / 8;
  const int b_from = int(int64_t(blocks) * rank / ctas), b_to = int(int64_t(blocks) * (rank + 1) / ctas);
  if (GATED) {
    let_next_begin();
  } else {
    if (VEC)  // a line per row of the CTA's
      for (int k = b_from * 8 + threadIdx.x; k < min(K, b_to * 8); k += kThreads)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(w + int64_t(k) * ldw + col0));
    wait_for_last();
  }
  F2 acc[MR][4];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[m][j] = both(0.f);

#pragma unroll 1
  for (int b = b_from + warp * kSubs + lane / kLanes; b < b_to; b += kWarps * kSubs) {
    const int k0 = b * 8;
    uint4 wv[8];
    float xv[MR][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = k0 + i;
      wv[i] = make_uint4(0, 0, 0, 0);
      if (VEC) {
        if (k < K && col < N) wv[i] = __ldcs(reinterpret_cast<const uint4*>(base + int64_t(k) * ldw));
      } else if (k < K) {
        uint32_t* words = &wv[i].x;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (col + e < N) words[e / 2] |= uint32_t(__bfloat16_as_ushort(base[int64_t(k) * ldw + e])) << (e % 2 * 16);
      }
    }
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const auto* row = x + int64_t(min(m, M - 1)) * ldx + k0;
      if (x_vec && k0 + 8 <= K) {
        if constexpr (GATED) {
          const uint4 t = *reinterpret_cast<const uint4*>(row);
          const uint32_t words[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) xv[m][e] = __uint_as_float(e % 2 ? words[e / 2] & 0xFFFF0000u : words[e / 2] << 16);
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 t = *reinterpret_cast<const float4*>(row + 4 * h);
            xv[m][4 * h] = t.x, xv[m][4 * h + 1] = t.y, xv[m][4 * h + 2] = t.z, xv[m][4 * h + 3] = t.w;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) xv[m][e] = k0 + e < K ? float(row[e]) : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t words[4] = {wv[i].x, wv[i].y, wv[i].z, wv[i].w};
      F2 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = F2(words[j] << 16, words[j] & 0xFFFF0000u);
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const F2 xm = both(xv[m][i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[m][j] = fma2(xm, v[j], acc[m][j]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      acc[m][j].get(a, b);
#pragma unroll
      for (int d = kLanes; d < 32; d *= 2) {
        a += __shfl_xor_sync(0xFFFFFFFFu, a, d);
        b += __shfl_xor_sync(0xFFFFFFFFu, b, d);
      }
      if (lane < kLanes) {
        sums_s[warp][m][place * 8 + 2 * j] = a;
        sums_s[warp][m][place * 8 + 2 * j + 1] = b;
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < MR * kWidth; i += kThreads) {
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) s += sums_s[v][i / kWidth][i % kWidth];
    part_s[i / kWidth][i % kWidth] = s;
  }
  if (ctas > 1) cluster_sync();
  else __syncthreads();
  // the cluster's CTAs share the outputs out among them
  for (int i = int(rank) * kThreads + threadIdx.x; i < MR * kCols; i += ctas * kThreads) {
    const int m = i / kCols, c = i % kCols;
    float a = 0.f, u = 0.f;
    for (int r = 0; r < ctas; ++r) {
      a += ctas > 1 ? peer_load(&part_s[m][c], r) : part_s[m][c];
      if (GATED) u += ctas > 1 ? peer_load(&part_s[m][kCols + c], r) : part_s[m][kCols + c];
    }
    const int col = col0 + c;
    if (m < M && col < N) {
      if constexpr (GATED) {
        const float h = gated(a, u, act);
        out[int64_t(m) * ldo + col] = h;
        if (keep.hidden) {  // [hi; lo]; nothing is left of what is not finite
          bf16* at = reinterpret_cast<bf16*>(keep.hidden) + int64_t(m) * ldo + col;
          const bf16 hi = __float2bfloat16_rn(h);
          at[0] = hi;
          at[int64_t(M) * ldo] = __float2bfloat16_rn(isfinite(__bfloat162float(hi)) ? h - __bfloat162float(hi) : 0.f);
        }
      } else {
        out[int64_t(m) * ldo + col] = __float2bfloat16_rn(a);
      }
    }
    if (GATED && keep.gate_up && m < M) {  // a warp has 32 columns of one row
      const int pitch = (N + 7) / 8 * 8;
      if (col >= N) a = u = 0.f;  // the pad columns take part in the backward pass as zeros
      __half hg, hu;
      const int eg = pack_fp16(a, act == GC_ACT_RELU, hg), eu = pack_fp16(u, false, hu);
      if (col < pitch) {
        __half* row = reinterpret_cast<__half*>(keep.gate_up) + int64_t(m) * 2 * pitch;
        row[col] = hg;
        row[pitch + col] = hu;
        if (c % 32 == 0) {
          const int64_t at = int64_t(col / 32) * M + m;
          keep.exps[at] = int8_t(eg);
          keep.exps[at + int64_t((pitch + 31) / 32) * M] = int8_t(eu);
        }
      }
    }
  }
  if (ctas > 1) cluster_sync();  // a CTA's shared memory is read by the others until here
}

// hidden (M x H, fp32) = act(G) U from e4m3 operands, K along the rows of both: a warp per column.
template <int MR, bool VEC>
__global__ void __launch_bounds__(kThreads)
ffn_rows_e4m3_kernel(const uint8_t* __restrict__ x, int64_t ldx, const float* __restrict__ x_scale,
                     const uint8_t* __restrict__ w, int64_t ldw, const float* __restrict__ w_scale,
                     float* __restrict__ out, int64_t ldo, int M, int K, int H, int act) {
  const int lane = threadIdx.x % 32, h = int(blockIdx.x) * kWarps + threadIdx.x / 32;
  let_next_begin();
  if (h >= H) return;
  const uint8_t* rows[2] = {w + int64_t(h) * ldw, w + (int64_t(h) + H) * ldw};
  F2 acc[2][MR];
#pragma unroll
  for (int m = 0; m < MR; ++m) acc[0][m] = acc[1][m] = both(0.f);
  auto load = [&](const uint8_t* p, int k) {
    if (VEC && k < K) return *reinterpret_cast<const uint4*>(p + k);
    uint4 v = make_uint4(0, 0, 0, 0);
    uint32_t* words = &v.x;
    if (!VEC)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (k + e < K) words[e / 4] |= uint32_t(p[k + e]) << (e % 4 * 8);
    return v;
  };
  auto two = [](uint32_t word, int j) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(uint16_t(word >> (16 * j)), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
    return F2(f.x, f.y);
  };
  constexpr int kUnroll = MR > 2 ? 2 : 4;
  for (int k0 = lane * 16; k0 < K; k0 += kUnroll * 512) {
    uint4 wv[kUnroll][2], xv[kUnroll][MR];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      wv[i][0] = load(rows[0], k0 + i * 512);
      wv[i][1] = load(rows[1], k0 + i * 512);
#pragma unroll
      for (int m = 0; m < MR; ++m) xv[i][m] = load(x + int64_t(min(m, M - 1)) * ldx, k0 + i * 512);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const F2 a = two((&wv[i][0].x)[q / 2], q % 2), b = two((&wv[i][1].x)[q / 2], q % 2);
#pragma unroll
        for (int m = 0; m < MR; ++m) {
          const F2 v = two((&xv[i][m].x)[q / 2], q % 2);
          acc[0][m] = fma2(v, a, acc[0][m]);
          acc[1][m] = fma2(v, b, acc[1][m]);
        }
      }
  }
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    float s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float a, b;
      acc[t][m].get(a, b);
      s[t] = a + b;
#pragma unroll
      for (int d = 16; d > 0; d /= 2) s[t] += __shfl_xor_sync(0xFFFFFFFFu, s[t], d);
    }
    if (lane == 0 && m < M) {
      const float sx = x_scale[m];
      out[int64_t(m) * ldo + h] = gated(s[0] * (sx * w_scale[h]), s[1] * (sx * w_scale[H + h]), act);
    }
  }
}

bool aligned_rows(const void* p, int64_t ld_bytes) { return gc::aligned16(p) && ld_bytes % 16 == 0; }

// CTAs of a cluster: as many as leave each some rows of W and no more than fill the GPU twice.
int cluster_of(int N, int K) {
  const int64_t groups = gc::ceil_div(N, kCols);
  int c = 1;
  while (c < 8 && groups * c < 2 * gc::kNumSMs && K / (2 * c) >= 64) c *= 2;
  return c;
}

template <bool GATED>
using In = std::conditional_t<GATED, bf16, float>;
template <bool GATED>
using Out = std::conditional_t<GATED, float, bf16>;

template <bool GATED, int MR, bool VEC>
int launch_rows(const In<GATED>* x, int64_t ldx, const bf16* w, int64_t ldw, Out<GATED>* out, int64_t ldo, int M, int K, int N, int act,
                const Saved& keep, cudaStream_t st) {
  const int ctas = cluster_of(N, K);
  const int64_t blocks = gc::ceil_div(N, kCols) * ctas;
  if (blocks > 0x7FFFFFFF) return gc::fail(GC_ERR_UNSUPPORTED, "gated feed-forward: too many columns");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  if (!GATED) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (ctas > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = unsigned(ctas);
    at[cfg.numAttrs].val.clusterDim.y = 1;
    at[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  cudaLaunchKernelEx(&cfg, ffn_rows_kernel<GATED, MR, VEC>, x, ldx, w, ldw, out, ldo, M, K, N, act, ctas, int(aligned_rows(x, ldx * int64_t(sizeof(*x)))), keep);
  return gc::check_launch("ffn_rows_kernel");
}
template <bool GATED, bool VEC>
int rows_of(const In<GATED>* x, int64_t ldx, const bf16* w, int64_t ldw, Out<GATED>* out, int64_t ldo, int M, int K, int N, int act,
            const Saved& keep, cudaStream_t st) {
  if (M == 1) return launch_rows<GATED, 1, VEC>(x, ldx, w, ldw, out, ldo, M, K, N, act, keep, st);
  if (M == 2) return launch_rows<GATED, 2, VEC>(x, ldx, w, ldw, out, ldo, M, K, N, act, keep, st);
  if (M <= 4) return launch_rows<GATED, 4, VEC>(x, ldx, w, ldw, out, ldo, M, K, N, act, keep, st);
  return launch_rows<GATED, 8, VEC>(x, ldx, w, ldw, out, ldo, M, K, N, act, keep, st);
}
template <bool GATED>
int product(const In<GATED>* x, int64_t ldx, const bf16* w, int64_t ldw, Out<GATED>* out, int64_t ldo, int M, int K, int N, int act,
            const Saved& keep, cudaStream_t st) {
  return N % 8 == 0 && aligned_rows(w, ldw * 2) ? rows_of<GATED, true>(x, ldx, w, ldw, out, ldo, M, K, N, act, keep, st)
                                                : rows_of<GATED, false>(x, ldx, w, ldw, out, ldo, M, K, N, act, keep, st);
}
template <int MR>
int product_e4m3(const Rows& r, cudaStream_t st) {
  const unsigned blocks = unsigned(gc::ceil_div(r.H, kWarps));
  const uint8_t *x = static_cast<const uint8_t*>(r.x), *w = static_cast<const uint8_t*>(r.w);
  if (r.D % 16 == 0 && aligned_rows(x, r.ldx) && aligned_rows(w, r.ldw))
    ffn_rows_e4m3_kernel<MR, true><<<blocks, kThreads, 0, st>>>(x, r.ldx, r.x_scale, w, r.ldw, r.w_scale, r.hidden, r.ldh, r.M, r.D, r.H, r.act);
  else
    ffn_rows_e4m3_kernel<MR, false><<<blocks, kThreads, 0, st>>>(x, r.ldx, r.x_scale, w, r.ldw, r.w_scale, r.hidden, r.ldh, r.M, r.D, r.H, r.act);
  return gc::check_launch("ffn_rows_e4m3_kernel");
}

}  // namespace

namespace gc {
namespace ffn {

int forward_few_rows(const Rows& r, bool e4m3, cudaStream_t st) {
  int rc;
  if (e4m3)
    rc = r.M == 1 ? product_e4m3<1>(r, st) : r.M == 2 ? product_e4m3<2>(r, st) : r.M <= 4 ? product_e4m3<4>(r, st) : product_e4m3<8>(r, st);
  else
    rc = product<true>(static_cast<const bf16*>(r.x), r.ldx, static_cast<const bf16*>(r.w), r.ldw, r.hidden, r.ldh, r.M, r.D, r.H,
                       r.act, r.saved, st);
  if (rc != GC_OK) return rc;
  return product<false>(r.hidden, r.ldh, reinterpret_cast<const bf16*>(r.w_out), r.ldwout, reinterpret_cast<bf16*>(r.y), r.ldy,
                        r.M, r.H, r.O, r.act, Saved{}, st);
}

}  // namespace ffn
}  // namespace gc
