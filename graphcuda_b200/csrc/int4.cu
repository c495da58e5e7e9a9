// Products with weights of 4 bits, for serving: Y = X W, and the gated feed-forward block with both of its weights so.
//
//   W[k, n] = (code[k, n] - zero[k / group, n]) * scale[k / group, n]      codes 0 to 15, zero 8 where none is given, scale bf16
//
// Up to kFewRows rows every code is read once and the time is that of reading them.  A warp turns 16 outputs x 32 inputs of codes into
// the bf16 operand of mma.sync -- code - zero is a whole number below 16 and exact there -- multiplies it by up to 64 rows of X, and
// adds the fp32 sums of a group times its scale to the outputs' fp32 sums: no weight is ever rounded.  (The 5th-generation tensor
// core takes its operands from shared memory and TMEM, through which every unpacked weight would have to go first; a
// product that waits for memory gains nothing from its rate.)  Codes are laid out so that a lane's 16 bytes are what it
// multiplies: see gc_linear_int4_bf16 in the header.
//
// A CTA has 16 or 32 outputs, whose chunks of 128 inputs its warps take in turn; where the outputs alone do not fill the GPU, those of a
// cluster do.  Sums meet in a fixed order.  In the block, the hidden row between the
// two launches goes as two bf16 numbers, hi and lo, in twice the rows of X; the second launch starts while the first runs, and its
// first codes are in registers when it has ended.
//
// More rows than that: the weights are unpacked once into bf16 in the workspace (rounded: 2^-9 at most, as an operand of the tensor
// cores has to be), 2.5 bytes of traffic per weight, and the tensor-core product of the gated block runs on them.
#include "common.cuh"
#include "ffn_internal.cuh"
#include "tiles.cuh"

#include <cuda_bf16.h>

#include <algorithm>

namespace {

using namespace gc::ffn;
using bf16 = __nv_bfloat16;

constexpr int kMostThreads = 256;
constexpr int kChunk = 128;       // inputs of a chunk
constexpr int kTile = 1024;       // bytes of 16 outputs' codes of a chunk
constexpr int kMostColumns = 64;  // rows of X (of hi and lo: twice) that a launch takes

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer_load(const float* p, uint32_t rank) {
  uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(p)), there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
  return v;
}
// c = A B, or c + A B.
template <bool FIRST>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  float d[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) d[i] = FIRST ? 0.f : c[i];
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(d[0]), "f"(d[1]), "f"(d[2]), "f"(d[3]));
}
// Eight codes as four pairs of bf16 numbers less `zero`, a pair of 128 + zero point: 0x4300 is 128 and its last bits count ones.
__device__ __forceinline__ void unpack(uint32_t w, __nv_bfloat162 zero, uint32_t (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&t), zero);
    o[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}
__device__ __forceinline__ __nv_bfloat162 zero_pair(uint32_t zeros, int byte) {
  const uint32_t t = __byte_perm(zeros, 0x43u, 0x4040u + 0x0101u * byte);
  return *reinterpret_cast<const __nv_bfloat162*>(&t);
}
__device__ __forceinline__ float gated(float g, float u, int act) {
  float a = 0.f, unused;
  with_activation(act, [&](auto t) {
    F2 slope;
    activate<decltype(t)::value>(F2(g, g), slope).get(a, unused);
  });
  return a * u;
}

struct Params {
  const uint16_t* x;  // rows in 16-byte accesses, zeros up to the next multiple of 8 inputs
  const uint8_t* codes;
  const uint16_t* scale;
  const uint8_t* zero;  // null: 8
  uint16_t* out;
  int64_t ldx, ldo;
  int rows, out_rows;  // of X; of the output: half of them where X is hi and lo
  int K, N;            // N: outputs, of either half of a gated product
  int ctas;            // of a cluster
  int act;
  int wait;  // X comes from the launch before
  const uint8_t* next;  // gated: the codes of the launch behind
  int64_t next_bytes;
};

// Of one chunk what a lane needs: codes of its outputs lane / 4 and lane / 4 + 8 of MT blocks, and their groups' scales and zero
// points, packed as they lie.
template <int MT, int GPC>
struct Fetched {
  uint4 codes[MT][2];
  uint32_t scale[MT][2][GPC == 4 ? 2 : 1];
  uint32_t zero[MT][2];
};

// NT: 8 rows of X each.  MT: blocks of 16 outputs of a CTA (GATED: the same ones of G and of U).  GPC: groups in a chunk.  DEPTH: chunks
// that a warp has on their way to its registers.  The CTA's warps, and those of the cluster's other CTAs, take chunks in turn.
template <int NT, int MT, bool GATED, int GPC, int DEPTH>
__global__ void __launch_bounds__(kMostThreads, NT == 1 ? 2 : 1)
int4_rows_kernel(const __grid_constant__ Params p) {
  extern __shared__ float sums[];  // [warp][MT * 16][NT * 8]
  constexpr int kCols = NT * 8, kOuts = MT * 16, kBlocks = 4 / GPC;  // kBlocks: 32s of inputs in a group
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32, g = lane / 4, t = lane % 4;
  const uint32_t rank = p.ctas > 1 ? cluster_rank() : 0;
  const int chunks = (p.K + kChunk - 1) / kChunk, total_n = GATED ? 2 * p.N : p.N;
  const int out0 = int(blockIdx.x / p.ctas) * (GATED ? 16 : kOuts);  // the CTA's first output
  // Where the lane's outputs begin: rows g and g + 8 of a block, but for U's of a gated product, which need not begin one.  The
  // second lies `codes_on` and `groups_on` behind the first.
  constexpr int kCodesOn = 8 * 64, kGroupsOn = 8 * GPC;
  const int step = p.ctas * warps;
  const uint8_t* codes_at[MT];
  const uint16_t* scale_at[MT];
  const uint8_t* zero_at[MT];
  int codes_on = kCodesOn, groups_on = kGroupsOn;  // U's
  int c = int(rank) * warps + warp;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    auto place = [&](int n, int64_t& codes, int64_t& groups) {
      const int64_t tile = int64_t(n / 16) * chunks + c;
      codes = tile * kTile + n % 16 * 64 + t * 16;
      groups = (tile * 16 + n % 16) * GPC;
    };
    int64_t codes, groups;
    if (GATED && m == 1) {
      const int n0 = min(out0 + g + p.N, total_n - 1), n1 = min(out0 + 8 + g + p.N, total_n - 1);
      int64_t codes1, groups1;
      place(n0, codes, groups);
      place(n1, codes1, groups1);
      codes_on = int(codes1 - codes);
      groups_on = int(groups1 - groups);
    } else {
      place(min(out0 / 16 + m, (total_n - 1) / 16) * 16 + g, codes, groups);
    }
    codes_at[m] = p.codes + codes;
    scale_at[m] = p.scale + groups;
    zero_at[m] = p.zero ? p.zero + groups : nullptr;
  }
  // The next chunk of the warp's.
  auto fetch = [&]() {
    Fetched<MT, GPC> f;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const bool any = GATED && m == 1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f.codes[m][h] = __ldcs(reinterpret_cast<const uint4*>(codes_at[m] + (h == 0 ? 0 : any ? codes_on : kCodesOn)));
        const uint16_t* scale = scale_at[m] + (h == 0 ? 0 : any ? groups_on : kGroupsOn);
        const uint8_t* zero = zero_at[m] + (h == 0 ? 0 : any ? groups_on : kGroupsOn);
        if constexpr (GPC == 4) {
          const uint2 v = __ldg(reinterpret_cast<const uint2*>(scale));
          f.scale[m][h][0] = v.x, f.scale[m][h][1] = v.y;
          f.zero[m][h] = p.zero ? __ldg(reinterpret_cast<const uint32_t*>(zero)) : 0x08080808u;
        } else if constexpr (GPC == 2) {
          f.scale[m][h][0] = __ldg(reinterpret_cast<const uint32_t*>(scale));
          f.zero[m][h] = p.zero ? __ldg(reinterpret_cast<const uint16_t*>(zero)) : 0x0808u;
        } else {
          f.scale[m][h][0] = __ldg(scale);
          f.zero[m][h] = p.zero ? __ldg(zero) : 8;
        }
      }
      codes_at[m] += int64_t(step) * kTile;
      scale_at[m] += int64_t(step) * 16 * GPC;
      zero_at[m] += int64_t(step) * 16 * GPC;
    }
    return f;
  };
  // Eight inputs of a row of X.  What columns beyond the last row hold, nobody reads: they take that row's once more.
  const uint16_t* x_at[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x_at[n] = p.x + int64_t(min(n * 8 + g, p.rows - 1)) * p.ldx + t * 8;
  auto fetch_x = [&](int n, int k, bool all) {  // all: of the chunk, or some beyond the last input, where zeros go
    if (all || k + t * 8 < p.K) return __ldg(reinterpret_cast<const uint4*>(x_at[n] + k));
    return make_uint4(0, 0, 0, 0);
  };

  float tot[MT][NT][4], acc[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) tot[m][n][e] = 0.f;
  Fetched<MT, GPC> ring[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (c + d * step < chunks) ring[d] = fetch();
  if (GATED) {
    let_next_begin();
    // the next launch's codes, a line per thread, on their way to the L2
    for (int64_t at = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) * 128; at < p.next_bytes; at += int64_t(gridDim.x) * blockDim.x * 128)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.next + at));
  }
  if (p.wait) wait_for_last();
  // X of a chunk: for up to 16 rows all at once, and of up to 8 rows a chunk ahead
  constexpr bool kWhole = NT <= 2, kAhead = NT == 1;
  uint4 xs[kWhole ? NT : 1][4], xn[kAhead ? NT : 1][4];
  auto fetch_chunk = [&](uint4 (&to)[kWhole ? NT : 1][4], int at) {
    if ((at + 1) * kChunk <= p.K) {
#pragma unroll
      for (int n = 0; n < (kWhole ? NT : 1); ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) to[n][j] = fetch_x(n, at * kChunk + j * 32, true);
    } else {
#pragma unroll
      for (int n = 0; n < (kWhole ? NT : 1); ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) to[n][j] = fetch_x(n, at * kChunk + j * 32, false);
    }
  };
  if constexpr (kAhead)
    if (c < chunks) fetch_chunk(xs, c);
  for (; c < chunks;) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d, c += step) {
      if (c >= chunks) break;
      const Fetched<MT, GPC>& now = ring[d];
      if constexpr (kAhead) {
        if (c + step < chunks) fetch_chunk(xn, c + step);
      } else if constexpr (kWhole) {
        fetch_chunk(xs, c);
      }
      const bool all = (c + 1) * kChunk <= p.K;
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // 32 inputs
        uint4 xj[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (kWhole) xj[n] = xs[n][j];
          else xj[n] = fetch_x(n, c * kChunk + j * 32, all);
        }
        uint32_t a[MT][2][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) unpack((&now.codes[m][h].x)[j], zero_pair(now.zero[m][h], j / kBlocks), a[m][h]);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (j % kBlocks == 0) mma<true>(acc[m][n], a[m][0][0], a[m][1][0], a[m][0][1], a[m][1][1], xj[n].x, xj[n].y);
            else mma<false>(acc[m][n], a[m][0][0], a[m][1][0], a[m][0][1], a[m][1][1], xj[n].x, xj[n].y);
            mma<false>(acc[m][n], a[m][0][2], a[m][1][2], a[m][0][3], a[m][1][3], xj[n].z, xj[n].w);
          }
        if (j % kBlocks == kBlocks - 1) {
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            auto scale = [&](int h) {
              const uint32_t w = now.scale[m][h][j / kBlocks / 2];
              return __uint_as_float(j / kBlocks % 2 ? w & 0xFFFF0000u : w << 16);
            };
            const float s0 = scale(0), s1 = scale(1);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              tot[m][n][0] = fmaf(s0, acc[m][n][0], tot[m][n][0]);
              tot[m][n][1] = fmaf(s0, acc[m][n][1], tot[m][n][1]);
              tot[m][n][2] = fmaf(s1, acc[m][n][2], tot[m][n][2]);
              tot[m][n][3] = fmaf(s1, acc[m][n][3], tot[m][n][3]);
            }
          }
        }
      }
      if (c + DEPTH * step < chunks) ring[d] = fetch();
      if constexpr (kAhead) {
#pragma unroll
        for (int j = 0; j < 4; ++j) xs[0][j] = xn[0][j];
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sums[(warp * kOuts + m * 16 + g + e / 2 * 8) * kCols + n * 8 + 2 * t + e % 2] = tot[m][n][e];
  __syncthreads();
  for (int i = threadIdx.x; i < kOuts * kCols; i += blockDim.x) {
    float s = sums[i];
    for (int w = 1; w < warps; ++w) s += sums[w * kOuts * kCols + i];
    sums[i] = s;
  }
  if (p.ctas > 1) cluster_sync();
  else __syncthreads();
  auto whole = [&](int out, int row) {  // over the cluster; hi and lo
    float s = 0.f;
    for (int r = row; r < p.rows; r += p.out_rows)
      for (int q = 0; q < p.ctas; ++q) {
        const float* v = sums + out * kCols + r;
        s += p.ctas > 1 ? peer_load(v, q) : *v;
      }
    return s;
  };
  constexpr int kWidth = GATED ? 16 : kOuts;  // outputs of the CTA, which the cluster shares out among its CTAs
  for (int i = int(rank) * blockDim.x + threadIdx.x; i < kWidth * p.out_rows; i += p.ctas * blockDim.x) {
    const int r = i / kWidth, o = i % kWidth, n = out0 + o;
    bf16* to = reinterpret_cast<bf16*>(p.out) + r * p.ldo + n;
    if constexpr (GATED) {
      const float h = n < p.N ? gated(whole(o, r), whole(o + 16, r), p.act) : 0.f;
      const bf16 hi = __float2bfloat16_rn(h);
      if (n < (p.N + 7) / 8 * 8) {  // zeros up to there
        to[0] = hi;
        to[p.out_rows * p.ldo] = __float2bfloat16_rn(isfinite(__bfloat162float(hi)) ? h - __bfloat162float(hi) : 0.f);  // of inf nothing is left
      }
    } else if (n < p.N) {
      to[0] = __float2bfloat16_rn(whole(o, r));
    }
  }
  if (p.ctas > 1) cluster_sync();  // a CTA's shared memory is read by the others until here
}

// Weights as bf16, an output's inputs in a row: eight of them per thread.
__global__ void __launch_bounds__(256)
int4_unpack_kernel(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scale, const uint8_t* __restrict__ zero, int K, int N,
                   int gpc, uint16_t* __restrict__ w, int64_t ldw) {
  const int chunks = (K + kChunk - 1) / kChunk;
  const int64_t total = int64_t(N) * chunks * 16;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int piece = int(i % 16), j = piece / 4, t = piece % 4;
    const int c = int(i / 16 % chunks), n = int(i / 16 / chunks), k = c * kChunk + piece * 8;
    if (k >= K) continue;
    const int64_t tile = int64_t(n / 16) * chunks + c;
    const uint32_t word = __ldg(reinterpret_cast<const uint32_t*>(codes + tile * kTile + n % 16 * 64 + t * 16) + j);
    const int64_t at = (tile * 16 + n % 16) * gpc + j * gpc / 4;
    const float s = __uint_as_float(uint32_t(__ldg(scale + at)) << 16);
    uint32_t o[4];
    unpack(word, zero_pair(zero ? __ldg(zero + at) : 8, 0), o);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(s * __uint_as_float(o[e] << 16), s * __uint_as_float(o[e] & 0xFFFF0000u));
      o[e] = *reinterpret_cast<const uint32_t*>(&v);
    }
    *reinterpret_cast<uint4*>(w + n * ldw + k) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ------------------------------------------------------------------ host
struct Weights {
  const uint8_t* codes;
  const uint16_t* scale;
  const uint8_t* zero;
  int group;
};
using gc::tiles::align256;
using gc::tiles::up8;

template <int NT, int MT, bool GATED, int GPC, int DEPTH>
int launch_rows(Params p, cudaStream_t st) {
  const int64_t blocks = gc::ceil_div(p.N, GATED ? 16 : 16 * MT);
  const int chunks = int(gc::ceil_div(p.K, kChunk));
  const int warps = chunks >= 32 ? 8 : 4;
  // All warps at once, 16 to an SM
  p.ctas = 1;
  while (p.ctas < 8 && blocks * 2 * p.ctas * warps <= 16 * gc::kNumSMs && 2 * p.ctas * warps <= chunks) p.ctas *= 2;
  if (blocks * p.ctas > 0x7FFFFFFF) return gc::fail(GC_ERR_UNSUPPORTED, "4-bit product: too many outputs");
  const size_t smem = size_t(warps) * MT * 16 * NT * 8 * sizeof(float);
  auto kern = int4_rows_kernel<NT, MT, GATED, GPC, DEPTH>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return gc::fail(GC_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(blocks * p.ctas));
  cfg.blockDim = dim3(unsigned(32 * warps));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  if (p.wait) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.ctas > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = unsigned(p.ctas);
    at[cfg.numAttrs].val.clusterDim.y = 1;
    at[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  cudaLaunchKernelEx(&cfg, kern, p);
  return gc::check_launch("int4_rows_kernel");
}
template <bool GATED>
int product(const Weights& w, Params p, cudaStream_t st) {
  p.codes = w.codes;
  p.scale = w.scale;
  p.zero = w.zero;
  auto sized = [&](auto gpc) {
    constexpr int kGpc = decltype(gpc)::value;
    if (p.rows <= 8) return launch_rows<1, GATED ? 2 : 1, GATED, kGpc, GATED ? 2 : 4>(p, st);
    if (p.rows <= 16) return launch_rows<2, 2, GATED, kGpc, 2>(p, st);
    if (p.rows <= 32) return launch_rows<4, 2, GATED, kGpc, 2>(p, st);
    return launch_rows<8, 2, GATED, kGpc, 1>(p, st);
  };
  return w.group == 32    ? sized(std::integral_constant<int, 4>{})
         : w.group == 64 ? sized(std::integral_constant<int, 2>{})
                         : sized(std::integral_constant<int, 1>{});
}
// X as the kernel takes it: itself, or a copy in the workspace.
bool rows_ready(const uint16_t* X, int64_t ldx, int64_t K) { return gc::aligned16(X) && ldx % 8 == 0 && K % 8 == 0; }
size_t rows_bytes(int64_t M, int64_t K) { return align256(size_t(M) * up8(K) * 2); }
int ready_rows(Params& p, const uint16_t* X, int64_t ldx, int64_t M, int64_t K, char*& ws, cudaStream_t st) {
  p.x = X;
  p.ldx = ldx;
  if (rows_ready(X, ldx, K)) return GC_OK;
  gc::tiles::Copies copies{};
  gc::tiles::add_copy(copies, gc::tiles::Matrix{X, M, K, ldx, 2}, ws, up8(K), up8(K));
  p.x = reinterpret_cast<const uint16_t*>(ws);
  p.ldx = up8(K);
  ws += rows_bytes(M, K);
  return gc::tiles::run_copies(copies, st);
}
int unpack_to(const Weights& w, int64_t K, int64_t N, void* to, cudaStream_t st) {
  const int64_t pieces = N * gc::ceil_div(K, kChunk) * 16;
  int4_unpack_kernel<<<unsigned(std::min<int64_t>(gc::ceil_div(pieces, 256), gc::kNumSMs * 32)), 256, 0, st>>>(
      w.codes, w.scale, w.zero, int(K), int(N), kChunk / w.group, static_cast<uint16_t*>(to), up8(K));
  return gc::check_launch("int4_unpack_kernel");
}
size_t unpacked_bytes(int64_t K, int64_t N) { return align256(size_t(N) * up8(K) * 2); }

bool sizes_ok(int64_t M, int64_t K, int64_t N) {
  const int64_t top = (int64_t(1) << 30) - 512;  // coordinates are 32-bit, and so is the way from a block's codes to the next one's
  return M <= top && K <= top / 8 && N <= top;
}
int weights_ok(const Weights& w, const char* what) {
  GC_REQUIRE(w.group == 32 || w.group == 64 || w.group == 128, "%s: a group is 32, 64 or 128 inputs", what);
  GC_REQUIRE(w.codes && w.scale, "%s: null pointer", what);
  GC_REQUIRE(gc::aligned16(w.codes) && gc::aligned16(w.scale) && gc::aligned16(w.zero), "%s: weights must be 16-byte aligned", what);
  return GC_OK;
}
int zeros(uint16_t* Y, int64_t ldy, int64_t M, int64_t N, cudaStream_t st, const char* what) {
  const cudaError_t e = cudaMemset2DAsync(Y, size_t(ldy) * 2, 0, size_t(N) * 2, size_t(M), st);
  return e == cudaSuccess ? GC_OK : gc::fail(GC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
constexpr int64_t kLinearRows = kMostColumns, kBlockRows = kMostColumns / 2;

}  // namespace

extern "C" {

size_t gc_linear_int4_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (M <= 0 || K <= 0 || N <= 0 || !sizes_ok(M, K, N)) return 0;
  if (M <= kLinearRows) return rows_bytes(M, K);
  return unpacked_bytes(K, N) + gc::ffn::rows_workspace(M, K, N);
}

int gc_linear_int4_bf16(const uint16_t* X, int64_t ldx, const uint8_t* codes, const uint16_t* scale, const uint8_t* zero, int group,
                        int64_t M, int64_t K, int64_t N, uint16_t* Y, int64_t ldy, void* workspace, size_t workspace_bytes,
                        void* stream) {
  GC_REQUIRE(M >= 0 && K >= 0 && N >= 0, "gc_linear_int4_bf16: negative size");
  GC_REQUIRE(ldx >= K && ldy >= N, "gc_linear_int4_bf16: leading dimension below the row length");
  if (!sizes_ok(M, K, N)) return gc::fail(GC_ERR_UNSUPPORTED, "gc_linear_int4_bf16: rows or outputs beyond 2^30, or inputs beyond 2^27");
  const cudaStream_t st = gc::as_stream(stream);
  if (M == 0 || N == 0) return GC_OK;
  GC_REQUIRE(Y, "gc_linear_int4_bf16: null pointer");
  if (K == 0) return zeros(Y, ldy, M, N, st, "gc_linear_int4_bf16");
  GC_REQUIRE(X, "gc_linear_int4_bf16: null pointer");
  const Weights w{codes, scale, zero, group};
  int rc = weights_ok(w, "gc_linear_int4_bf16");
  if (rc != GC_OK) return rc;
  if (!workspace || workspace_bytes < gc_linear_int4_workspace_bytes(M, K, N))
    return gc::fail(GC_ERR_WORKSPACE, "gc_linear_int4_bf16: workspace missing or smaller than its query says");
  GC_REQUIRE(gc::aligned16(workspace), "gc_linear_int4_bf16: workspace must be 16-byte aligned");
  if (M <= kLinearRows) {
    Params p{};
    char* ws = static_cast<char*>(workspace);
    rc = ready_rows(p, X, ldx, M, K, ws, st);
    if (rc != GC_OK) return rc;
    p.out = Y; p.ldo = ldy;
    p.rows = p.out_rows = int(M);
    p.K = int(K); p.N = int(N);
    return product<false>(w, p, st);
  }
  rc = unpack_to(w, K, N, workspace, st);
  if (rc != GC_OK) return rc;
  return gc::ffn::rows_times(X, ldx, static_cast<const uint16_t*>(workspace), up8(K), M, K, N, Y, ldy,
                             static_cast<char*>(workspace) + unpacked_bytes(K, N), st);
}

size_t gc_gated_ffn_int4_workspace_bytes(int64_t M, int64_t D, int64_t H, int64_t O) {
  if (M <= 0 || D <= 0 || H <= 0 || O <= 0 || !sizes_ok(M, std::max(D, H), O) || !sizes_ok(2 * H, 0, 0)) return 0;
  if (M <= kBlockRows) return rows_bytes(M, D) + rows_bytes(2 * M, H);
  return unpacked_bytes(D, 2 * H) + unpacked_bytes(H, O) + gc::ffn::block_workspace(M, D, H, O);
}

int gc_gated_ffn_int4_bf16(const uint16_t* X, int64_t ldx, const uint8_t* codes_in, const uint16_t* scale_in, const uint8_t* zero_in,
                           int group_in, const uint8_t* codes_out, const uint16_t* scale_out, const uint8_t* zero_out, int group_out,
                           int64_t M, int64_t D, int64_t H, int64_t O, int act, uint16_t* Y, int64_t ldy, void* workspace,
                           size_t workspace_bytes, void* stream) {
  GC_REQUIRE(M >= 0 && D >= 0 && H >= 0 && O >= 0, "gc_gated_ffn_int4_bf16: negative size");
  GC_REQUIRE(act >= GC_ACT_SILU && act <= GC_ACT_RELU, "gc_gated_ffn_int4_bf16: unknown activation");
  GC_REQUIRE(ldx >= D && ldy >= O, "gc_gated_ffn_int4_bf16: leading dimension below the row length");
  if (!sizes_ok(M, std::max(D, H), O) || !sizes_ok(2 * H, 0, 0)) return gc::fail(GC_ERR_UNSUPPORTED, "gc_gated_ffn_int4_bf16: rows or outputs beyond 2^30, or inputs beyond 2^27");
  const cudaStream_t st = gc::as_stream(stream);
  if (M == 0 || O == 0) return GC_OK;
  GC_REQUIRE(Y, "gc_gated_ffn_int4_bf16: null pointer");
  if (D == 0 || H == 0) return zeros(Y, ldy, M, O, st, "gc_gated_ffn_int4_bf16");
  GC_REQUIRE(X, "gc_gated_ffn_int4_bf16: null pointer");
  const Weights in{codes_in, scale_in, zero_in, group_in}, out{codes_out, scale_out, zero_out, group_out};
  int rc = weights_ok(in, "gc_gated_ffn_int4_bf16");
  if (rc == GC_OK) rc = weights_ok(out, "gc_gated_ffn_int4_bf16");
  if (rc != GC_OK) return rc;
  if (!workspace || workspace_bytes < gc_gated_ffn_int4_workspace_bytes(M, D, H, O))
    return gc::fail(GC_ERR_WORKSPACE, "gc_gated_ffn_int4_bf16: workspace missing or smaller than its query says");
  GC_REQUIRE(gc::aligned16(workspace), "gc_gated_ffn_int4_bf16: workspace must be 16-byte aligned");
  char* ws = static_cast<char*>(workspace);
  if (M <= kBlockRows) {
    Params p{};
    rc = ready_rows(p, X, ldx, M, D, ws, st);
    if (rc != GC_OK) return rc;
    p.out = reinterpret_cast<uint16_t*>(ws); p.ldo = up8(H);
    p.rows = p.out_rows = int(M);
    p.K = int(D); p.N = int(H);
    p.act = act;
    p.next = codes_out;
    p.next_bytes = gc::ceil_div(O, 16) * gc::ceil_div(H, kChunk) * kTile;
    rc = product<true>(in, p, st);
    if (rc != GC_OK) return rc;
    Params q{};
    q.x = p.out; q.ldx = p.ldo;
    q.out = Y; q.ldo = ldy;
    q.rows = int(2 * M); q.out_rows = int(M);
    q.K = int(H); q.N = int(O);
    q.wait = 1;
    return product<false>(out, q, st);
  }
  uint16_t* w_in = reinterpret_cast<uint16_t*>(ws);
  uint16_t* w_out = reinterpret_cast<uint16_t*>(ws + unpacked_bytes(D, 2 * H));
  ws += unpacked_bytes(D, 2 * H) + unpacked_bytes(H, O);
  rc = unpack_to(in, D, 2 * H, w_in, st);
  if (rc == GC_OK) rc = unpack_to(out, H, O, w_out, st);
  if (rc != GC_OK) return rc;
  return gc::ffn::block_times(X, ldx, w_in, up8(D), w_out, up8(H), M, D, H, O, act, Y, ldy, ws, st);
}

}  // extern "C"
