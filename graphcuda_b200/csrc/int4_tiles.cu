// Products with 4-bit weights for some tens of rows: 17 to 128, in the gated block 9 to 64.
//
// The arithmetic is that of the form for few rows (int4.cu): codes less their zero points are bf16 operands of mma.sync, which multiplies
// 16 outputs x 16 inputs by 8 rows, groups' fp32 sums are scaled in fp32, and no weight is rounded.  But X is no longer
// small beside the codes: with every warp fetching its own rows from the L2, 32 rows took twice the time of 16.  Here the 8
// warps of a CTA have 16 or 32 outputs each and the same chunk of 128 inputs at a time, so that X comes to the CTA once per chunk; a
// ninth warp keeps a ring of chunks -- X and the warps' records -- filled with bulk copies.  CTAs of a cluster share an output's chunks out
// and add their sums in a fixed order.
//
// A first launch brings X into the order of the operand's fragments, so that a lane's 16 bytes of 8 rows x 32 inputs lie where its bulk
// copy needs no address of its own and its load from shared memory has no conflict; zeros go beyond the last row and input.  In the block
// the hidden row is stored in that order by the first product, as two bf16 numbers, hi and lo, in rows of their own.
//
// What bounds it is mma.sync and the unpacking before it, which share the warps' issue slots: 16,384 inputs x 8192 outputs, groups of 64,
// take 43 us for 32 rows, 68 for 64 and 126 for 128, at which 273 TFLOP/s are reached; for 17 rows they are as many as for 32.
// The form for few rows took 58 us for 32, unpacking into bf16 and the tensor-core product 144 and 146 for 64 and 128, and 149
// for 129, so that beyond 128 rows they take over; at 2048 x 8192 the three are 11.9 against 13.2, 15.6 against 23 and 22 against 26.  The
// block with 2048, 8192 and 2048 takes 28 us for 16 rows, 47 for 64, and 69 for 65 unpacked.
#include "int4_internal.cuh"

#include <algorithm>

namespace {

using namespace gc::int4;
using gc::int4::unpack;

constexpr int kWarps = 8, kThreads = 32 * (kWarps + 1);
// Products of fewer tiles than this take smaller ones: those of 8192 inputs x 2048 outputs, 17 us for 33 rows and 15 for 17, took 29 and 18
// (with clusters of 8, which do not all find their SMs at a time when a CTA has one to itself; so there they are of 4).
constexpr int kFewTiles = 24;
constexpr int kFragments = 2048;  // bytes of 8 rows x 128 inputs

// Rows in fragments: [chunk][block of 8 rows][32 inputs][lane][8 inputs].  Lane 4 g + t has row g, inputs 8 t to 8 t + 7.
__host__ __device__ __forceinline__ int64_t fragment_at(int row, int k, int blocks) {
  return ((int64_t(k / kChunk) * blocks + row / 8) * 4 + k % kChunk / 32) * 256 + (row % 8 * 4 + k % 32 / 8) * 8 + k % 8;
}
// Hidden rows of the block: of every 8 * nt rows of fragments the first half are hi of so many rows, the second half their lo.
__host__ __device__ __forceinline__ int hi_row(int m, int nt) { return m / (4 * nt) * 8 * nt + m % (4 * nt); }

__device__ __forceinline__ float4 peer_load4(const float* p, uint32_t rank) {
  uint32_t at = smem_u32(p), there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(there) : "memory");
  return v;
}

struct Params {
  const uint16_t* x;  // fragments
  const uint8_t* w;   // records
  uint16_t* out;      // rows, or (gated) fragments
  int64_t ldo;
  int blocks;       // of 8 rows in the fragments
  int out_rows;     // of the output
  int halves;       // 2: X is hi and lo
  int K, N;         // N: outputs, of either half of a gated product
  int ctas;         // of a cluster
  int stages;
  int vec;  // the output in 8-byte accesses
  int act;
  int next_nt, next_blocks;  // gated: of the fragments that are written
  int* word;                 // the device's error word
};

// NT: 8 rows each.  MT: blocks of 16 outputs of a warp (GATED: one of G and the same of U, whose outputs lie in two records where SPLIT).
template <int NT, int MT, bool GATED, bool SPLIT, int GPC, bool ZEROS>
struct Shape {
  static constexpr int kRecord = record_bytes(GPC, ZEROS);
  static constexpr int kRecords = GATED ? 2 * kWarps + SPLIT : MT * kWarps;  // of a stage
  static constexpr int kX = NT * kFragments, kStage = (kX + kRecords * kRecord + 127) / 128 * 128;
  static constexpr int kOuts = kWarps * MT * 16, kCols = NT * 8;  // G and U count as two
  static constexpr int kPitch = kOuts + 4, kSums = kPitch * kCols * 4;  // [row][output], so that 8 outputs x 4 rows meet no bank twice
  static constexpr int kWidth = GATED ? kWarps * 16 : kOuts;                                // outputs of a CTA
};

// CTAs of an SM: two where the sums leave room for it in registers.
constexpr int per_sm(int nt, int mt) { return nt * mt <= 4 ? 2 : 1; }

template <int NT, int MT, bool GATED, bool SPLIT, int GPC, bool ZEROS>
__global__ void __launch_bounds__(kThreads, per_sm(NT, MT))
int4_tiles_kernel(const __grid_constant__ Params p) {
  using S_ = Shape<NT, MT, GATED, SPLIT, GPC, ZEROS>;
  constexpr int kRecord = S_::kRecord, kCols = S_::kCols, kBlocks = 4 / GPC;  // kBlocks: 32s of inputs in a group
  extern __shared__ __align__(128) uint8_t shared[];  // barriers; stages, and then the sums in their place
  __shared__ int abort_s;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const int rank = blockIdx.y, out0 = blockIdx.x * S_::kWidth, z = blockIdx.z;
  const int chunks = (p.K + kChunk - 1) / kChunk;
  const int from = int(int64_t(chunks) * rank / p.ctas), to = int(int64_t(chunks) * (rank + 1) / p.ctas);
  const uint32_t bars = smem_u32(shared), ring = bars + 128;
  auto full = [&](int i) { return bars + 8 * i; };
  auto empty = [&](int i) { return bars + 8 * (p.stages + i); };
  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(full(i), 1);
      mbar_init(empty(i), kWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  __syncthreads();
  let_next_begin();
  volatile int* abort_p = &abort_s;
  int slot = 0;
  uint32_t phase = 0;
  auto advance = [&]() {
    if (++slot == p.stages) slot = 0, phase ^= 1u;
  };
  float tot[MT][NT][4], acc[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) tot[m][n][e] = 0.f;

  if (warp == kWarps) {
    // ------------------------------------------------------------ fetches: a record per lane, and X
    const int last_block = ((GATED ? 2 * p.N : p.N) + 15) / 16 - 1;
    const int block = GATED && lane >= kWarps ? (out0 + p.N) / 16 + lane - kWarps : out0 / 16 + lane;
    const uint8_t* record = p.w + (int64_t(min(block, last_block)) * chunks + from) * kRecord;
    const uint16_t* x = p.x + (int64_t(from) * p.blocks + z * NT) * (kFragments / 2);
    auto fetch_records = [&]() {
      if (lane == 0) mbar_expect_tx(full(slot), S_::kX + S_::kRecords * kRecord);
      __syncwarp();
      if (lane < S_::kRecords) bulk_load(ring + slot * S_::kStage + S_::kX + lane * kRecord, record, kRecord, full(slot));
      record += kRecord;
    };
    auto fetch_x = [&](int s) {
      if (lane == 0) bulk_load(ring + s * S_::kStage, x, S_::kX, full(s));
      x += int64_t(p.blocks) * (kFragments / 2);
    };
    // the first records, while X may still be written
    const int ahead = min(to - from, p.stages);
    for (int i = 0; i < ahead; ++i) {
      fetch_records();
      advance();
    }
    wait_for_last();
    for (int i = 0; i < ahead; ++i) fetch_x(i);
    int issued = ahead;
    for (int c = from + ahead; c < to; ++c) {
      if (!__all_sync(0xFFFFFFFFu, gc::tiles::wait(empty(slot), phase ^ 1u, abort_p))) break;
      fetch_records();
      fetch_x(slot);
      advance();
      ++issued;
    }
    if (lane == 0)  // what was issued lands before its place becomes the sums'
      for (int j = 0; j < issued && j < p.stages; ++j) {
        if (slot == 0) phase ^= 1u;
        slot = slot == 0 ? p.stages - 1 : slot - 1;
        drain(full(slot), phase);
      }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ multiplies
    // Where in a stage the lane's outputs lie: rows g and g + 8 of a record, U's from row N % 16 on.
    auto record_at = [&](int m, int h) {
      if (!GATED) return (warp * MT + m) * kRecord;
      return (m == 0 ? warp : kWarps + warp + (SPLIT ? (g + h * 8 + p.N % 16) / 16 : 0)) * kRecord;
    };
    auto row_at = [&](int m, int h) { return SPLIT && m == 1 ? (g + h * 8 + p.N % 16) % 16 : g + h * 8; };
    uint32_t codes_at[MT][2], scales_at[MT][2], zeros_of[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        codes_at[m][h] = S_::kX + record_at(m, h) + row_at(m, h) * 64 + t * 16;
        scales_at[m][h] = S_::kX + record_at(m, h) + kScales + row_at(m, h) * (GPC * 2);
        zeros_of[m][h] = S_::kX + record_at(m, h) + zeros_at(GPC) + row_at(m, h) * GPC;
      }
    bool ok = true;
    for (int c = from; c < to; ++c) {
      if (ok) ok = __all_sync(0xFFFFFFFFu, gc::tiles::wait(full(slot), phase, abort_p));
      const uint32_t stage = ring + slot * S_::kStage, xs = stage + lane * 16;
      uint4 codes[MT][2];
      uint32_t scale[MT][2][GPC == 4 ? 2 : 1], zero[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          codes[m][h] = shared_16(stage + codes_at[m][h]);
          const uint32_t s = stage + scales_at[m][h], zs = stage + zeros_of[m][h];
          if constexpr (GPC == 4) {
            const uint2 v = shared_8(s);
            scale[m][h][0] = v.x, scale[m][h][1] = v.y;
          } else {
            scale[m][h][0] = GPC == 2 ? shared_4(s) : shared_2(s);
          }
          zero[m][h] = !ZEROS ? 0x08080808u : GPC == 4 ? shared_4(zs) : GPC == 2 ? shared_2(zs) : shared_1(zs);
        }
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // 32 inputs
        uint32_t a[MT][2][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) unpack((&codes[m][h].x)[j], zero_pair(zero[m][h], j / kBlocks), a[m][h]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 x = shared_16(xs + n * kFragments + j * 512);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (j % kBlocks == 0) mma<true>(acc[m][n], a[m][0][0], a[m][1][0], a[m][0][1], a[m][1][1], x.x, x.y);
            else mma<false>(acc[m][n], a[m][0][0], a[m][1][0], a[m][0][1], a[m][1][1], x.x, x.y);
            mma<false>(acc[m][n], a[m][0][2], a[m][1][2], a[m][0][3], a[m][1][3], x.z, x.w);
          }
        }
        if (j == 3) {  // all of the stage is in registers
          __syncwarp();
          if (lane == 0) mbar_arrive(empty(slot));
        }
        if (j % kBlocks == kBlocks - 1) {
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            auto value = [&](int h) {
              const uint32_t w = scale[m][h][j / kBlocks / 2];
              return __uint_as_float(j / kBlocks % 2 ? w & 0xFFFF0000u : w << 16);
            };
            const float s0 = value(0), s1 = value(1);
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
      advance();
    }
  }
  // ---------------------------------------------------------------- the sums, in the stages' place
  __syncthreads();
  float* sums = reinterpret_cast<float*>(shared + 128);
  if (warp < kWarps) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sums[(n * 8 + 2 * t + e % 2) * S_::kPitch + (warp * MT + m) * 16 + g + e / 2 * 8] = tot[m][n][e];
  }
  if (p.ctas > 1) cluster_sync();
  else __syncthreads();
  const int rows = kCols / p.halves;  // of the output, of this CTA
  auto each_four = [&](auto cluster) {  // outputs of a row
    constexpr int C = decltype(cluster)::value;
    auto whole = [&](int out, int row) {  // over the cluster
      float4 v[C];
#pragma unroll
      for (int q = 0; q < C; ++q) {
        const float* at = sums + row * S_::kPitch + out;
        v[q] = C > 1 ? peer_load4(at, q) : *reinterpret_cast<const float4*>(at);
      }
#pragma unroll
      for (int q = 1; q < C; ++q) v[0].x += v[q].x, v[0].y += v[q].y, v[0].z += v[q].z, v[0].w += v[q].w;
      return v[0];
    };
    for (int i = rank * kThreads + threadIdx.x; i < S_::kWidth / 4 * rows; i += C * kThreads) {
      const int r = i / (S_::kWidth / 4), o = i % (S_::kWidth / 4) * 4, n = out0 + o, m = z * rows + r;
      if (n >= p.N || m >= p.out_rows) continue;
      if constexpr (GATED) {
        const int place = o / 16 * 32 + o % 16;
        const float4 vg = whole(place, r), vu = whole(place + 16, r);
        const float gs[4] = {vg.x, vg.y, vg.z, vg.w}, us[4] = {vu.x, vu.y, vu.z, vu.w};
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float h = n + e < p.N ? gated(gs[e], us[e], p.act) : 0.f;
          const bf16 b = __float2bfloat16_rn(h);
          hi[e] = __bfloat16_as_ushort(b);  // nothing is left of what is not finite
          lo[e] = __bfloat16_as_ushort(__float2bfloat16_rn(isfinite(__bfloat162float(b)) ? h - __bfloat162float(b) : 0.f));
        }
        const int row = hi_row(m, p.next_nt);
        *reinterpret_cast<uint2*>(p.out + fragment_at(row, n, p.next_blocks)) = make_uint2(hi[0] | hi[1] << 16, hi[2] | hi[3] << 16);
        *reinterpret_cast<uint2*>(p.out + fragment_at(row + 4 * p.next_nt, n, p.next_blocks)) =
            make_uint2(lo[0] | lo[1] << 16, lo[2] | lo[3] << 16);
      } else {
        float4 v = whole(o, r);
        if (p.halves > 1) {
          const float4 lo = whole(o, r + rows);
          v.x += lo.x, v.y += lo.y, v.z += lo.z, v.w += lo.w;
        }
        const float vs[4] = {v.x, v.y, v.z, v.w};
        bf16* out = reinterpret_cast<bf16*>(p.out) + m * p.ldo + n;
        if (p.vec) {
          *reinterpret_cast<uint2*>(out) = make_uint2(gc::tiles::pack2(v.x, v.y), gc::tiles::pack2(v.z, v.w));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < p.N) out[e] = __float2bfloat16_rn(vs[e]);
        }
      }
    }
  };
  if (p.ctas == 1) each_four(std::integral_constant<int, 1>{});
  else if (p.ctas == 2) each_four(std::integral_constant<int, 2>{});
  else if (p.ctas == 4) each_four(std::integral_constant<int, 4>{});
  else each_four(std::integral_constant<int, 8>{});
  if (p.ctas > 1) cluster_sync();  // a CTA's shared memory is read by the others until here
  if (threadIdx.x == 0 && abort_s) atomicExch(p.word, 1);
}

// X as fragments, zeros beyond its last row and input; `zeros`: 16-byte units behind them that become zero too (the hidden rows').
__global__ void __launch_bounds__(256)
int4_arrange_kernel(const uint16_t* __restrict__ x, int64_t ldx, int M, int K, int blocks, int vec, uint4* __restrict__ out, int64_t zeros) {
  let_next_begin();
  const int64_t total = int64_t((K + kChunk - 1) / kChunk) * blocks * 128;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total + zeros; i += int64_t(gridDim.x) * 256) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (i < total) {
      const int lane = int(i % 32), j = int(i / 32 % 4);
      const int64_t tile = i / 128;
      const int row = int(tile % blocks) * 8 + lane / 4, k = int(tile / blocks) * kChunk + j * 32 + lane % 4 * 8;
      if (row < M && k < K) {
        const uint16_t* from = x + row * ldx + k;
        if (vec && k + 8 <= K) {
          v = __ldg(reinterpret_cast<const uint4*>(from));
        } else {
          uint32_t w[4] = {};
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (k + e < K) w[e / 2] |= uint32_t(from[e]) << (e % 2 * 16);
          v = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    out[i] = v;
  }
}

// ------------------------------------------------------------------ host
// 8-row blocks of X in the workspace: what every form below rounds up to.
int64_t blocks_of(int64_t rows) { return rows <= 16 ? 2 : rows <= 32 ? 4 : gc::ceil_div(rows, 64) * 8; }
// 8-row blocks of a CTA: up to 8, for which the codes are unpacked once; 4 and two CTAs took 10 percent longer (75 us instead of 68 above),
// but are the faster where CTAs of 8 would be too few, and in the block, whose two sums per output spill at 8 (54 us instead of 47).
int nt_of(int64_t rows, int64_t N, bool is_gated) {
  if (rows <= 16) return 2;
  if (rows <= 32) return 4;
  return is_gated || gc::ceil_div(N, kWarps * 16) * gc::ceil_div(rows, 64) <= kFewTiles ? 4 : 8;
}
int64_t fragment_bytes(int64_t rows, int64_t K) { return gc::ceil_div(K, kChunk) * blocks_of(rows) * kFragments; }

template <int NT, int MT, bool GATED, bool SPLIT, int GPC, bool ZEROS>
int launch(Params p, int64_t z, cudaStream_t st) {
  using S_ = Shape<NT, MT, GATED, SPLIT, GPC, ZEROS>;
  static_assert(S_::kRecords <= 32, "a lane for every record");
  const int64_t ctas = gc::ceil_div(p.N, S_::kWidth) * z;
  const int chunks = int(gc::ceil_div(p.K, kChunk));
  constexpr int kPerSm = per_sm(NT, MT);
  p.ctas = 1;
  while (p.ctas < 4 * kPerSm && ctas * 2 * p.ctas <= kPerSm * gc::kNumSMs && 2 * p.ctas <= chunks) p.ctas *= 2;
  constexpr int kRoom = 222 * 1024 / kPerSm - 1024 - 128 - 16;
  static_assert(2 * S_::kStage <= kRoom && S_::kSums <= kRoom, "room for two stages and for the sums");
  p.stages = int(std::min<int64_t>({gc::ceil_div(chunks, p.ctas), 8, kRoom / S_::kStage}));
  const int smem = 128 + std::max(p.stages * S_::kStage, S_::kSums);
  auto kern = int4_tiles_kernel<NT, MT, GATED, SPLIT, GPC, ZEROS>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 + kRoom);  // any call's: see int4.cu
  if (e != cudaSuccess) return gc::fail(GC_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  const int rc = gc::tiles::error_word(&p.word);
  if (rc != GC_OK) return rc;
  if (gc::ceil_div(p.N, S_::kWidth) > 0x7FFFFFFF) return gc::fail(GC_ERR_UNSUPPORTED, "4-bit product: too many outputs");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(gc::ceil_div(p.N, S_::kWidth)), unsigned(p.ctas), unsigned(z));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  if (p.ctas > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = 1;
    at[cfg.numAttrs].val.clusterDim.y = unsigned(p.ctas);
    at[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  cudaLaunchKernelEx(&cfg, kern, p);
  return gc::check_launch("int4_tiles_kernel");
}
template <bool GATED, bool SPLIT, int GPC, bool ZEROS>
int for_rows(const Params& p, int nt, int64_t z, cudaStream_t st) {
  if constexpr (GATED) {
    if (nt == 2) return launch<2, 2, GATED, SPLIT, GPC, ZEROS>(p, z, st);
    return launch<4, 2, GATED, SPLIT, GPC, ZEROS>(p, z, st);
  } else {
    if (nt == 8) return launch<8, 1, GATED, SPLIT, GPC, ZEROS>(p, z, st);
    if (gc::ceil_div(p.N, kWarps * 32) * z <= kFewTiles) return launch<4, 1, GATED, SPLIT, GPC, ZEROS>(p, z, st);
    return launch<4, 2, GATED, SPLIT, GPC, ZEROS>(p, z, st);
  }
}
// `rows`: of the fragments in use.
template <bool GATED>
int product(const Weights& w, Params p, int64_t rows, cudaStream_t st) {
  p.w = w.records;
  p.vec = p.N % 4 == 0 && p.ldo % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % 8 == 0;
  p.blocks = int(blocks_of(rows));
  const int nt = nt_of(rows, p.N, GATED);
  const int64_t z = gc::ceil_div(rows, 8 * nt);
  auto with = [&](auto gpc, auto zeros) {
    constexpr int kGpc = decltype(gpc)::value;
    constexpr bool kZeros = decltype(zeros)::value;
    if constexpr (GATED)
      if (p.N % 16) return for_rows<true, true, kGpc, kZeros>(p, nt, z, st);
    return for_rows<GATED, false, kGpc, kZeros>(p, nt, z, st);
  };
  auto grouped = [&](auto zeros) {
    return w.group == 32    ? with(std::integral_constant<int, 4>{}, zeros)
           : w.group == 64 ? with(std::integral_constant<int, 2>{}, zeros)
                           : with(std::integral_constant<int, 1>{}, zeros);
  };
  return w.zeros ? grouped(std::true_type{}) : grouped(std::false_type{});
}
int arrange(const uint16_t* X, int64_t ldx, int64_t M, int64_t K, void* to, int64_t zero_bytes, cudaStream_t st) {
  const int64_t units = (fragment_bytes(M, K) + zero_bytes) / 16;
  const int vec = gc::aligned16(X) && ldx % 8 == 0;
  int4_arrange_kernel<<<unsigned(std::min<int64_t>(gc::ceil_div(units, 256), gc::kNumSMs * 8)), 256, 0, st>>>(
      X, ldx, int(M), int(K), int(blocks_of(M)), vec, static_cast<uint4*>(to), zero_bytes / 16);
  return gc::check_launch("int4_arrange_kernel");
}
// hi and lo of M rows: in every 8 nt rows of fragments half as many rows of the block
int64_t hidden_rows(int64_t M, int64_t O) {
  const int nt = nt_of(2 * M, O, false);
  return gc::ceil_div(M, 4 * nt) * 8 * nt;
}

}  // namespace

namespace gc {
namespace int4 {

size_t linear_tiles_workspace(int64_t M, int64_t K, int64_t) { return align256(size_t(fragment_bytes(M, K))); }
int linear_tiles(const uint16_t* X, int64_t ldx, const Weights& w, int64_t M, int64_t K, int64_t N, uint16_t* Y, int64_t ldy, void* workspace,
                 cudaStream_t st) {
  const int rc = arrange(X, ldx, M, K, workspace, 0, st);
  if (rc != GC_OK) return rc;
  Params p{};
  p.x = static_cast<const uint16_t*>(workspace);
  p.out = Y; p.ldo = ldy;
  p.out_rows = int(M);
  p.halves = 1;
  p.K = int(K); p.N = int(N);
  return product<false>(w, p, M, st);
}

size_t block_tiles_workspace(int64_t M, int64_t D, int64_t H, int64_t O) {
  return align256(size_t(fragment_bytes(M, D) + fragment_bytes(hidden_rows(M, O), H)));
}
int block_tiles(const uint16_t* X, int64_t ldx, const Weights& in, const Weights& out, int64_t M, int64_t D, int64_t H, int64_t O, int act,
                uint16_t* Y, int64_t ldy, void* workspace, cudaStream_t st) {
  const int64_t rows = hidden_rows(M, O), x_bytes = fragment_bytes(M, D);
  int rc = arrange(X, ldx, M, D, workspace, fragment_bytes(rows, H), st);
  if (rc != GC_OK) return rc;
  Params p{};
  p.x = static_cast<const uint16_t*>(workspace);
  p.out = reinterpret_cast<uint16_t*>(static_cast<char*>(workspace) + x_bytes);
  p.out_rows = int(M);
  p.halves = 1;
  p.K = int(D); p.N = int(H);
  p.act = act;
  p.next_nt = nt_of(rows, O, false); p.next_blocks = int(blocks_of(rows));
  rc = product<true>(in, p, M, st);
  if (rc != GC_OK) return rc;
  Params q{};
  q.x = p.out;
  q.out = Y; q.ldo = ldy;
  q.out_rows = int(M);
  q.halves = 2;
  q.K = int(H); q.N = int(O);
  return product<false>(out, q, rows, st);
}

}  // namespace int4
}  // namespace gc
