// Products with weights of 4 bits, for serving: Y = X W, and the gated feed-forward block with both of its weights so.
//
//   W[k, n] = (code[k, n] - zero[k / group, n]) * scale[k / group, n]      codes 0 to 15, zero 8 where none is given, scale bf16
//
// Up to 16 rows (8 in the block) every code is read once and the time is that of reading them.  A warp turns 16 outputs x 32 inputs of codes into
// the bf16 operand of mma.sync -- code - zero is a whole number below 16 and exact there -- multiplies it by up to 16 rows of X, and
// adds the fp32 sums of a group times its scale to the outputs' fp32 sums: no weight is ever rounded.  (The 5th-generation tensor
// core takes its operands from shared memory and TMEM, through which every unpacked weight would have to go first; a
// product that waits for memory gains nothing from its rate.)
//
// Weights are records: of 16 outputs and 128 inputs the codes, scales and zero points (see gc_linear_int4_bf16 in the header), laid out so
// that a lane's 16 bytes are what it multiplies.  A warp has a ring of records in shared memory, which one lane keeps filled
// with bulk copies: some 100 KB have to be on their way to an SM at any time (64 KB in registers, as loads of 16 warps: 4.0 TB/s
// without any arithmetic), and no instructions are spent on them.  A CTA takes 16 or 32 outputs at a time, whose records its warps take in
// turn; where the outputs alone do not fill the GPU, those of a cluster do.  Sums meet in a fixed order.  In the block, the hidden row between the
// two launches goes as two bf16 numbers, hi and lo, in twice the rows of X; the second launch starts while the first runs, and its
// first codes are in registers when it has ended.
//
// One row of 8192 x 32,768 takes 38.8 us, 3.67 TB/s of codes and scales; of 2048 x 8192, whose floor is 1.4 us, 5.2, which are launch,
// first fetch and the cluster's sum; 16 rows of 16,384 x 8192 with zero points 34.1 (floor 11.9), where unpacking (151 instructions a warp for
// 2048 codes at one row) takes half of the issue slots and warps wait for X, twice as many bytes from the L2 as codes; the next chunk's X in
// registers ahead spills (47.6).  Loads into registers instead of rings took 10.2 and 89.5 us for the last two.
//
// Up to 128 rows (64 in the block): int4_tiles.cu.  More than that: the weights are unpacked once into the workspace, 2.5 bytes of traffic per
// weight, and the tensor-core products of the gated block run on them.  For Y = X W they are bf16 (rounded: 2^-8 of a weight at most, as
// much as the result's own rounding; fp16 as in the block would need X's copy too, 35 us beside 34 for all of 169,343 rows through 256 and
// 256).  In the block, where two weights and the hidden row would be rounded so, they are fp16, 2^-11,
// with a power of two per output, row of X, hidden row and hidden column that keeps fp16's range from mattering; X is copied into fp16, exactly
// down to 2^-28 of a row's largest.  A hidden row's power is what its largest value asks for, whatever that is: the one that it starts with
// is a guess from norms, 32 columns that do not fit it take another, and a launch after the first product brings a row's columns to the
// largest's (ffn_level_kernel).  So its values have their 11 bits down to 2^-13 of the largest, and large columns are taken down first, see
// column_shift.  (With a power from a bound,
// |x|^2 and the weights' norms, nothing was left of them where channels of X differ by thousands and the weights even that out: it lies
// that far above.)  169,343 rows through 256, 1024 and 256 take 290 us (280
// with the bound; bf16 took 243, with twice the error of a plain form in fp32): 36 for X and the second weight, 6 for the first, 155 for the first
// product, 6 to bring rows together and 77 for the second product.
#include "int4_internal.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace {

using namespace gc::int4;
using gc::int4::unpack;

constexpr int kMostThreads = 256;
constexpr int kRun = 2;  // records that are fetched, waited for and given back together: of a block of outputs they follow each other

struct Params {
  const uint16_t* x;  // rows in 16-byte accesses, zeros up to the next multiple of 8 inputs
  const uint8_t* w;   // records
  uint16_t* out;
  int64_t ldx, ldo;
  int rows, out_rows;  // of X; of the output: half of them where X is hi and lo
  int K, N;            // N: outputs, of either half of a gated product
  int ctas;            // of a cluster
  int ring;            // places in a warp's ring
  int act;
  int wait;  // X comes from the launch before
  const uint8_t* next;  // gated: the records of the launch behind
  int64_t next_bytes;
  int* word;  // the device's error word
};

// NT: 8 rows of X each.  MT: blocks of 16 outputs that a CTA takes at a time (GATED: the same ones of G and of U, whose outputs lie in two
// blocks where SPLIT).  GPC: groups in a record.  ZEROS: whether records have zero points.
template <int NT, int MT, bool GATED, bool SPLIT, int GPC, bool ZEROS>
__global__ void __launch_bounds__(kMostThreads, NT == 1 && MT == 1 ? 3 : 2)
int4_rows_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t shared[];  // sums of two turns, [warp][MT * 16][NT * 8]; barriers; rings
  constexpr int kCols = NT * 8, kOuts = MT * 16, kBlocks = 4 / GPC;  // kBlocks: 32s of inputs in a group
  constexpr int kWidth = GATED ? 16 : kOuts;                         // outputs at a time
  constexpr int kRecord = record_bytes(GPC, ZEROS), kCopies = SPLIT ? 3 : MT, kPlace = kCopies * kRun * kRecord;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32, g = lane / 4, t = lane % 4;
  const int rank = blockIdx.y;  // in the cluster
  const int chunks = (p.K + kChunk - 1) / kChunk;
  const int step = p.ctas * warps * kRun, first = (rank * warps + warp) * kRun;
  float* const sums_of_two = reinterpret_cast<float*>(shared);
  const uint32_t bars = smem_u32(shared) + 2 * warps * kOuts * kCols * 4 + warp * p.ring * 8;
  const uint32_t ring = smem_u32(shared) + 2 * warps * kOuts * kCols * 4 + (warps * p.ring * 8 + 127) / 128 * 128 + warp * p.ring * kPlace;

  // One lane fetches: the run of records from `ahead` on of the outputs from ahead_out on.
  int ahead_out = blockIdx.x * kWidth, ahead = first;
  const uint8_t* from[kCopies];
  auto begin = [&]() {
    const int last_block = ((GATED ? 2 * p.N : p.N) + 15) / 16 - 1;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int b = GATED && i > 0 ? (ahead_out + p.N) / 16 + i - 1 : ahead_out / 16 + i;
      from[i] = p.w + (int64_t(min(b, last_block)) * chunks + first) * kRecord;
    }
  };
  auto fetch = [&](uint32_t bar, uint32_t to) {
    if (ahead >= chunks) {  // on to the CTA's next outputs
      ahead_out += gridDim.x * kWidth;
      ahead = first;
      begin();
    }
    if (ahead_out >= p.N) return false;
    const uint32_t bytes = min(kRun, chunks - ahead) * kRecord;
    mbar_expect_tx(bar, kCopies * bytes);
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      bulk_load(to + i * (kRun * kRecord), from[i], bytes, bar);
      from[i] += step * kRecord;
    }
    ahead += step;
    return true;
  };
  int on_their_way = 0;  // copies, as lane 0 counts them
  if (lane == 0 && first < chunks) {
    for (int i = 0; i < p.ring; ++i) mbar_init(bars + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
    begin();
    while (on_their_way < p.ring && fetch(bars + 8 * on_their_way, ring + on_their_way * kPlace)) ++on_their_way;
  }
  __syncwarp();
  uint32_t bar = bars, place = ring, parity = 0;  // what is used next, and the phase of its barrier
  const uint32_t bar_end = bars + 8 * p.ring;
  // Where in a place the lane's outputs lie, rows g and g + 8 of a block: its codes 16 bytes a lane, then 16 bytes a lane.  But for U's
  // where they lie in two blocks.
  auto row_of = [&](int h) { return g + h * 8 + p.N % 16; };
  auto of_row = [&](int row) { return row / 16 * (kRun * kRecord); };
  auto codes_at = [&](int m, int h) {
    if (SPLIT && m == 1) return (kRun * kRecord) + of_row(row_of(h)) + row_of(h) % 16 * 64 + t * 16;
    return m * (kRun * kRecord) + lane * 16 + h * 512;
  };
  auto groups_at = [&](int m, int h, int bytes) {  // `bytes` for each of the output's groups
    if (SPLIT && m == 1) return (kRun * kRecord) + of_row(row_of(h)) + row_of(h) % 16 * (GPC * bytes);
    return m * (kRun * kRecord) + (g + h * 8) * (GPC * bytes);
  };
  // Eight inputs of a row of X.  What columns beyond the last row hold, nobody reads: they take that row's once more.
  const uint16_t* x_at[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x_at[n] = p.x + int64_t(min(n * 8 + g, p.rows - 1)) * p.ldx + t * 8;
  auto fetch_x = [&](int n, int c, int j, bool all) {  // all: of the chunk, or some beyond the last input, where zeros go
    if (all || c * kChunk + j * 32 + t * 8 < p.K) return __ldg(reinterpret_cast<const uint4*>(x_at[n] + c * kChunk + j * 32));
    return make_uint4(0, 0, 0, 0);
  };

  if (GATED) {
    let_next_begin();
    // the next launch's records, a line per thread, on their way to the L2
    for (int64_t i = ((int64_t(blockIdx.x) * p.ctas + rank) * blockDim.x + threadIdx.x) * 128; i < p.next_bytes;
         i += int64_t(gridDim.x) * p.ctas * blockDim.x * 128)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.next + i));
  }
  if (p.wait) wait_for_last();

  float tot[MT][NT][4], acc[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) tot[m][n][e] = 0.f;
  float* sums = sums_of_two;
  bool ok = true;
  for (int out0 = blockIdx.x * kWidth; out0 < p.N; out0 += gridDim.x * kWidth) {
    for (int c0 = first; c0 < chunks; c0 += step) {
#pragma unroll
      for (int u = 0; u < kRun; ++u) {
        const int c = c0 + u;
        if (u > 0 && c >= chunks) break;
        const bool all = (c + 1) * kChunk <= p.K;
        uint4 xs[NT][4];
        if (all) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) xs[n][j] = fetch_x(n, c, j, true);
        } else {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) xs[n][j] = fetch_x(n, c, j, false);
        }
        if (u == 0 && ok) ok = arrived(bar, parity);
        uint4 codes[MT][2];
        uint32_t scale[MT][2][GPC == 4 ? 2 : 1], zero[MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            codes[m][h] = shared_16(place + u * kRecord + codes_at(m, h));
            const uint32_t s = place + u * kRecord + kScales + groups_at(m, h, 2), z = place + u * kRecord + zeros_at(GPC) + groups_at(m, h, 1);
            if constexpr (GPC == 4) {
              const uint2 v = shared_8(s);
              scale[m][h][0] = v.x, scale[m][h][1] = v.y;
            } else {
              scale[m][h][0] = GPC == 2 ? shared_4(s) : shared_2(s);
            }
            zero[m][h] = !ZEROS ? 0x08080808u : GPC == 4 ? shared_4(z) : GPC == 2 ? shared_2(z) : shared_1(z);
          }
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // 32 inputs
          uint32_t a[MT][2][4];
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) unpack((&codes[m][h].x)[j], zero_pair(zero[m][h], j / kBlocks), a[m][h]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const uint4 x = xs[n][j];
              if (j % kBlocks == 0) mma<true>(acc[m][n], a[m][0][0], a[m][1][0], a[m][0][1], a[m][1][1], x.x, x.y);
              else mma<false>(acc[m][n], a[m][0][0], a[m][1][0], a[m][0][1], a[m][1][1], x.x, x.y);
              mma<false>(acc[m][n], a[m][0][2], a[m][1][2], a[m][0][3], a[m][1][3], x.z, x.w);
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
      }
      __syncwarp();  // all have read
      if (ok) {
        if (lane == 0 && !fetch(bar, place)) --on_their_way;
        bar += 8;
        place += kPlace;
        if (bar == bar_end) bar = bars, place = ring, parity ^= 1;
      }
    }
    // ---- the outputs' sums: over the warps, over the cluster, of hi and lo
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float2* to = reinterpret_cast<float2*>(sums + (warp * kOuts + m * 16 + g + h * 8) * kCols + n * 8 + 2 * t);
          *to = make_float2(tot[m][n][2 * h], tot[m][n][2 * h + 1]);
          tot[m][n][2 * h] = tot[m][n][2 * h + 1] = 0.f;
        }
    __syncthreads();
    if (p.ctas > 1) {
      for (int i = threadIdx.x; i < kOuts * kCols; i += blockDim.x) {
        float s = sums[i];
        for (int w = 1; w < warps; ++w) s += sums[w * kOuts * kCols + i];
        sums[i] = s;
      }
      cluster_sync();
    }
    auto whole = [&](int out, int row) {
      float s = 0.f;
      for (int r = row; r < p.rows; r += p.out_rows) {
        const float* v = sums + out * kCols + r;
        if (p.ctas > 1)
          for (int q = 0; q < p.ctas; ++q) s += peer_load(v, q);
        else
          for (int w = 0; w < warps; ++w) s += v[w * kOuts * kCols];
      }
      return s;
    };
    // a cluster shares the outputs out among its CTAs
    for (int i = rank * blockDim.x + threadIdx.x; i < kWidth * p.out_rows; i += p.ctas * blockDim.x) {
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
    // the other half of the shared memory: the one before's readers have all come past the barrier since
    sums = sums == sums_of_two ? sums_of_two + warps * kOuts * kCols : sums_of_two;
  }
  // what was fetched has all been waited for, unless a wait ran out
  if (!ok && lane == 0) {
    for (; on_their_way > 0; --on_their_way) {
      drain(bar, parity);
      bar += 8;
      if (bar == bar_end) bar = bars, parity ^= 1;
    }
    atomicExch(p.word, 1);
  }
}

// Weights as bf16, an output's inputs in a row: eight of them per thread.
__global__ void __launch_bounds__(256)
int4_unpack_kernel(const uint8_t* __restrict__ records, int zeros, int K, int N, int gpc, uint16_t* __restrict__ w, int64_t ldw) {
  const int chunks = (K + kChunk - 1) / kChunk, size = record_bytes(gpc, zeros != 0);
  const int64_t total = int64_t(N) * chunks * 16;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int piece = int(i % 16), j = piece / 4, t = piece % 4;
    const int c = int(i / 16 % chunks), n = int(i / 16 / chunks), k = c * kChunk + piece * 8;
    if (k >= K) continue;
    const uint8_t* r = records + (int64_t(n / 16) * chunks + c) * size;
    const uint32_t word = __ldg(reinterpret_cast<const uint32_t*>(r + n % 16 * 64 + t * 16) + j);
    const int group = n % 16 * gpc + j * gpc / 4;
    const float s = __uint_as_float(uint32_t(__ldg(reinterpret_cast<const uint16_t*>(r + kScales) + group)) << 16);
    uint32_t o[4];
    unpack(word, zero_pair(zeros ? __ldg(r + zeros_at(gpc) + group) : 8, 0), o);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(s * __uint_as_float(o[e] << 16), s * __uint_as_float(o[e] & 0xFFFF0000u));
      o[e] = *reinterpret_cast<const uint32_t*>(&v);
    }
    *reinterpret_cast<uint4*>(w + n * ldw + k) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// The exponent whose power of two brings numbers up to `most` below 2^14, and half of that at least; not so small that a power is no fp32
// number.
__device__ __forceinline__ int fp16_exponent(float most) { return max(int(__float_as_uint(most) >> 23) - 127 - 13, -100); }

// Weights as fp16, every output's times a power of two, an output's inputs in a row.  A CTA takes a part of 16 outputs' chunks.  Exponents
// are multiples of 16, which brings the largest weight to 2^-2 at least: the outputs of a layer mostly share one, which the products'
// epilogues apply in a multiplication.  An output whose smallest group would come below fp16's normal numbers so has one of its own, which brings
// the largest to 2^13 (groups 2^-20 of the largest, whose inputs make up for it, left an error of up to 3e-2 otherwise).
struct ToFp16 {
  const uint8_t* records;
  uint16_t* w;
  int* exps;
  int64_t ldw;
  int zeros, K, N, gpc, parts;
};
// The block's hidden columns, as the first weight's outputs say: G's are the first H of them, U's follow.
struct Columns {
  int* norms;   // of an output, the exponent of a power of two that its weights, as a vector, are shorter than
  int2* range;  // the largest and the smallest norm of 16 outputs
  int* eup;     // U's exponents, which take up what a column is divided by
  int H;
};
constexpr int kNoNorm = -(1 << 20);  // of zeros
__device__ __forceinline__ int common_exponent(int e) { return min((e + 111) / 16 * 16 - 96, 115); }  // from -100 to 115: one as large at least

// Columns by the product of their two norms: where these differ, the largest columns are divided by 2^14, those below 2^-7 of the largest
// by 2^7, those below 2^-14 not, and the second weight's rows of them are multiplied by that: a large column has so much less of a say in the
// others' rounding.  In steps of 7, so that the columns of a layer mostly share one, for which the first product's epilogue has a short form; two
// of them, for which fp16's range has room in the second weight.
constexpr int kMostShift = 14;
__device__ __forceinline__ int column_shift(const Columns& c, int k, int top) {
  const int bound = __ldg(c.norms + k) + __ldg(c.norms + c.H + k);
  return bound > kNoNorm / 2 ? max(kMostShift - (top - bound) / 7 * 7, 0) : 0;
}
struct Bounds {
  int g, u;    // the largest norms of either half
  bool mixed;  // whether columns may differ in how they are stored
};
__device__ __forceinline__ Bounds bounds_of(const Columns& c) {  // by a whole CTA of 256 threads
  __shared__ int found[8][4];
  int v[4] = {kNoNorm, kNoNorm, kNoNorm, kNoNorm};  // the largest, and less the smallest, of G's and of U's
  for (int i = threadIdx.x; i * 16 < 2 * c.H; i += 256) {  // a block on the border is of both halves
    const int2 r = __ldg(c.range + i);
    if (i * 16 < c.H) v[0] = max(v[0], r.x), v[1] = max(v[1], -r.y);
    if (i * 16 + 16 > c.H) v[2] = max(v[2], r.x), v[3] = max(v[3], -r.y);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    v[q] = __reduce_max_sync(0xFFFFFFFFu, v[q]);
    if (threadIdx.x % 32 == 0) found[threadIdx.x / 32][q] = v[q];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = max(v[q], found[i][q]);
  return {v[0], v[2], v[0] + v[1] + v[2] + v[3] >= 7};
}

// FIRST: the weight of G and U, whose norms go to `columns`; otherwise the second one, whose inputs are the columns.
template <bool FIRST>
__device__ __forceinline__ void unpack_fp16(const ToFp16& p, int cta, const Columns& columns, bool mixed, int top) {
  __shared__ uint32_t most_s[16], least_s[16];
  __shared__ int norms_s[16];
  __shared__ __align__(8) uint8_t shift_s[kChunk];
  const int block = cta / p.parts, part = cta % p.parts;
  const int zeros = p.zeros, K = p.K, N = p.N, gpc = p.gpc;
  const int chunks = (K + kChunk - 1) / kChunk, size = record_bytes(gpc, zeros != 0);
  const uint8_t* r = p.records + int64_t(block) * chunks * size;
  if (threadIdx.x < 16) most_s[threadIdx.x] = 0, least_s[threadIdx.x] = 0x7F800000u;
  __syncthreads();
  const int out = threadIdx.x / 16, piece = threadIdx.x % 16, j = piece / 4, t = piece % 4;  // output, of 16; 8 inputs of a chunk
  const bool exists = block * 16 + out < N;
  uint32_t most = 0, least = 0x7F800000u;  // as a float's bits
  double squares = 0.;
  for (int c = piece; c < chunks && exists; c += 16)
    for (int g = 0; g < gpc && c * kChunk + g * (kChunk / gpc) < K; ++g) {
      const uint32_t bits = gc::ffn::finite_bits(uint32_t(__ldg(reinterpret_cast<const uint16_t*>(r + int64_t(c) * size + kScales) + out * gpc + g)) << 16);
      most = max(most, bits);
      if (bits) least = min(least, bits);
      if (FIRST && part == 0) {
        const double s = __uint_as_float(bits);
        squares += s * s * min(kChunk / gpc, K - c * kChunk - g * (kChunk / gpc));
      }
    }
  atomicMax(&most_s[out], most);
  atomicMin(&least_s[out], least);
  if (FIRST && part == 0) {
    squares *= zeros ? 225. : 64.;  // codes less zero points: -15 to 15, or -8 to 7
    for (int o = 8; o > 0; o >>= 1) squares += __shfl_xor_sync(0xFFFFFFFFu, squares, o);
    const int above = int(__double_as_longlong(squares) >> 52) - 1022;  // squares < 2^above
    const int norm = squares > 0. ? (above + 1) >> 1 : kNoNorm;
    if (piece == 0) {
      norms_s[out] = norm;
      if (exists) columns.norms[block * 16 + out] = norm;
    }
  }
  __syncthreads();
  // (where inputs are multiplied by as much as 2^14, outputs' exponents are their own, so that the other inputs keep fp16's 11 bits)
  const int own = fp16_exponent(__uint_as_float(most_s[out]) * 15.f), common = common_exponent(own);
  const int e = mixed ? min(own + kMostShift, 126) : int(least_s[out] >> 23) - 127 - common < -14 ? own : common;
  const float f = __uint_as_float(uint32_t(127 - e) << 23);
  if (part == 0 && piece == 0) {
    if (exists) p.exps[block * 16 + out] = e;
    if (FIRST && out == 0) {
      int2 range = make_int2(kNoNorm, -kNoNorm);
      for (int i = 0; i < 16; ++i)
        if (norms_s[i] != kNoNorm) range.x = max(range.x, norms_s[i]), range.y = min(range.y, norms_s[i]);
      columns.range[block] = range;
    }
  }
  const int from = int(int64_t(chunks) * part / p.parts), to = int(int64_t(chunks) * (part + 1) / p.parts);
  for (int c = from; c < to; ++c) {
    if (mixed) {  // the same for all of the CTA
      __syncthreads();
      const int k = c * kChunk + threadIdx.x;
      if (threadIdx.x < kChunk) shift_s[threadIdx.x] = k < K ? uint8_t(column_shift(columns, k, top)) : 0;
      __syncthreads();
    }
    const int k = c * kChunk + piece * 8;
    if (k >= K || !exists) continue;
    const uint8_t* at = r + int64_t(c) * size;
    const uint32_t word = __ldg(reinterpret_cast<const uint32_t*>(at + out * 64 + t * 16) + j);
    const int group = out * gpc + j * gpc / 4;
    const float s = __uint_as_float(uint32_t(__ldg(reinterpret_cast<const uint16_t*>(at + kScales) + group)) << 16) * f;
    uint32_t o[4];
    unpack(word, zero_pair(zeros ? __ldg(at + zeros_at(gpc) + group) : 8, 0), o);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float a = s * __uint_as_float(o[q] << 16), b = s * __uint_as_float(o[q] & 0xFFFF0000u);
      if (mixed) {
        a *= __uint_as_float((127u + shift_s[piece * 8 + 2 * q]) << 23);
        b *= __uint_as_float((127u + shift_s[piece * 8 + 2 * q + 1]) << 23);
      }
      const __half2 v = __floats2half2_rn(a, b);
      o[q] = *reinterpret_cast<const uint32_t*>(&v);
    }
    *reinterpret_cast<uint4*>(p.w + (int64_t(block) * 16 + out) * p.ldw + k) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}
__global__ void __launch_bounds__(256)
int4_unpack_fp16_kernel(const ToFp16 p, const Columns columns) {
  unpack_fp16<true>(p, blockIdx.x, columns, false, 0);
}

// What follows from the columns: U's exponents, the second weight, and X as fp16, every row times a power of two, zeros up to a multiple of
// 8.  The first `row_ctas` CTAs take rows, a warp each; then 256 columns to a CTA; then the weight.
// eh: where the hidden row's values are to lie, from |x| and the largest norms of G's and of U's outputs.  |act(G) U| is at most |x|^2
// |Wg| |Wu| and mostly, as sums of products that do not know of each other, a K-th of that or less: the largest of 32 such come to some 2^5.
// (Where they do not, the first product's epilogue sees it and takes another exponent.)
// SHORT: rows of up to 256 inputs in 16-byte accesses, each a load and a store.  169,343 rows of 256 take 34 us so, and 40 with the loops
// that other rows need.
template <bool SHORT>
__global__ void __launch_bounds__(256)
int4_rows_fp16_kernel(const uint16_t* __restrict__ x, int64_t ldx, int M, int K, int vec, const Columns columns, const ToFp16 second,
                      int row_ctas, int column_ctas, uint16_t* __restrict__ out, int64_t ldo, int* __restrict__ exps, int* __restrict__ eh) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const Bounds most_of = bounds_of(columns);
  const int behind = int(blockIdx.x) - row_ctas;
  if (behind >= column_ctas) return unpack_fp16<false>(second, behind - column_ctas, columns, most_of.mixed, most_of.g + most_of.u);
  if (behind >= 0) {
    const int k = behind * 256 + threadIdx.x;
    if (most_of.mixed && k < columns.H) columns.eup[k] -= column_shift(columns, k, most_of.g + most_of.u);
    return;
  }
  const int log_k = 32 - __clz(K);  // 2^log_k > K
  const float unit = __uint_as_float(uint32_t(130 - log_k) << 23);  // sums of squares in 2^(log_k - 3): what is finite stays below 2^14 each
  const int64_t step = int64_t(row_ctas) * 8;
  uint4 following = make_uint4(0, 0, 0, 0);  // the first 256 inputs of a row are on their way while the one before is written
  for (int64_t m = int64_t(blockIdx.x) * 8 + warp - step; m < M; m += step) {
    auto load_of = [&](const uint16_t* row, int k) {
      if (SHORT || (vec && k + 8 <= K)) return __ldg(reinterpret_cast<const uint4*>(row + k));
      uint32_t w[4] = {};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k + e < K) w[e / 2] |= uint32_t(row[k + e]) << (e % 2 * 16);
      return make_uint4(w[0], w[1], w[2], w[3]);
    };
    auto load = [&](int k) { return load_of(x + m * ldx, k); };
    const uint4 first = following;
    if (m + step < M && lane * 8 < K) following = load_of(x + (m + step) * ldx, lane * 8);
    if (m < 0) continue;
    __nv_bfloat162 tops = __float2bfloat162_rn(0.f);
    for (int k = lane * 8; k < K; k += SHORT ? 1 << 30 : 256) {
      const uint4 v = SHORT || k < 256 ? first : load(k);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // a NaN is passed over
        const uint32_t a = w[q] & 0x7FFF7FFFu;
        tops = __hmax2(tops, *reinterpret_cast<const __nv_bfloat162*>(&a));
      }
    }
    const uint32_t both_tops = *reinterpret_cast<const uint32_t*>(&tops);
    uint32_t most = __reduce_max_sync(0xFFFFFFFFu, max(both_tops << 16, both_tops & 0xFFFF0000u));
    if (most == 0x7F800000u) {  // an infinity has no say in its row's exponent either
      most = 0;
      for (int k = lane * 8; k < K; k += 256) {
        const uint4 v = load(k);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) most = max(most, max(gc::ffn::finite_bits(w[q] << 16), gc::ffn::finite_bits(w[q] & 0xFFFF0000u)));
      }
      most = __reduce_max_sync(0xFFFFFFFFu, most);
    }
    const int e = fp16_exponent(__uint_as_float(most));
    const F2 f = gc::ffn::both(__uint_as_float(uint32_t(127 - e) << 23));
    F2 squares2(0.f, 0.f);
    for (int k = lane * 8; k < K; k += SHORT ? 1 << 30 : 256) {
      const uint4 v = SHORT || k < 256 ? first : load(k);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t o[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const F2 v2 = F2(w[q] << 16, w[q] & 0xFFFF0000u) * f;
        squares2 = gc::ffn::fma2(v2, v2, squares2);
        float a, b;
        v2.get(a, b);
        const __half2 h = __floats2half2_rn(a, b);
        o[q] = *reinterpret_cast<const uint32_t*>(&h);
      }
      *reinterpret_cast<uint4*>(out + m * ldo + k) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    float squares, odd;
    squares2.get(squares, odd);
    squares += odd;
    const bool finite = squares < INFINITY;  // which a NaN is not either
    uint32_t sum = __reduce_add_sync(0xFFFFFFFFu, finite ? __float2uint_ru(squares * unit) : 0u);
    if (!__all_sync(0xFFFFFFFFu, finite)) sum = 1u << 31;
    if (lane == 0) {
      exps[m] = e;
      const int row = 2 * e + 32 - __clz(sum) + log_k - 3;  // |x|^2 < 2^row
      // (U times 2^-eh has to be a number by itself: the second term, for G below 2^-90 or so)
      const int bound = row + most_of.g + most_of.u - (most_of.mixed ? kMostShift + 3 : 0);  // (columns are then spread over 7 powers below it)
      const int h = max(bound - log_k - 10, max(((row + 1) >> 1) + most_of.u - 112, -126));
      eh[m] = sum > 0 && most_of.g > kNoNorm / 2 && most_of.u > kNoNorm / 2 ? min(h, 126) : 0;
    }
  }
}

// ------------------------------------------------------------------ host
template <int NT, int MT, bool GATED, bool SPLIT, int GPC, bool ZEROS>
int launch_rows(Params p, cudaStream_t st) {
  const int64_t blocks = gc::ceil_div(p.N, GATED ? 16 : 16 * MT);
  const int runs = int(gc::ceil_div(gc::ceil_div(p.K, kChunk), kRun));
  constexpr int kPerSm = NT == 1 && MT == 1 ? 24 : 16;  // warps
  const int warps = runs >= 16 ? 8 : 4;
  // All warps at once: outputs beyond those follow in the same CTAs.
  const int64_t slots = kPerSm / warps * gc::kNumSMs;
  p.ctas = 1;
  while (p.ctas < 8 && blocks * 2 * p.ctas <= slots && 2 * p.ctas * warps <= runs) p.ctas *= 2;
  const int64_t ctas = std::min(blocks, slots);
  // As many places in a ring as a warp has runs of records, up to what the SM's shared memory holds.
  constexpr int kPlace = (SPLIT ? 3 : MT) * kRun * record_bytes(GPC, ZEROS);
  const int64_t mine = gc::ceil_div(runs, p.ctas * warps) * gc::ceil_div(blocks, ctas);
  const int sums = 2 * warps * MT * 16 * NT * 8 * int(sizeof(float));
  const int room = (220 * 1024 / (kPerSm / warps) - 1024 - 256 - sums) / warps;
  static_assert((220 * 1024 / (kPerSm / 4) - 1280) / 4 - 2 * MT * 16 * NT * 8 * 4 >= kPlace + 8, "room for a place");
  p.ring = int(std::min<int64_t>({mine, 16, room / (kPlace + 8)}));
  const int smem = sums + (warps * p.ring * 8 + 127) / 128 * 128 + warps * p.ring * kPlace;
  auto kern = int4_rows_kernel<NT, MT, GATED, SPLIT, GPC, ZEROS>;
  // what any call of this form may take: the attribute is every thread's of the process, and one that calls with less must not lower it
  // between another's two calls
  constexpr int kMostBytes = 220 * 1024 / (kPerSm / 8) - 1024;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostBytes);
  if (e != cudaSuccess) return gc::fail(GC_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  const int rc = gc::tiles::error_word(&p.word);
  if (rc != GC_OK) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(ctas), unsigned(p.ctas));
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
    at[cfg.numAttrs].val.clusterDim.x = 1;
    at[cfg.numAttrs].val.clusterDim.y = unsigned(p.ctas);
    at[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  cudaLaunchKernelEx(&cfg, kern, p);
  return gc::check_launch("int4_rows_kernel");
}
// Records from which on a warp takes two blocks of outputs at a time, with half of the instructions around them: a row of 4096 x 8192 takes
// 8.3 us so and 9.0 with one block, 8192 x 32,768 38.1 and 39.9; 2048 x 8192 5.6 and 5.1, for it is short of warps.
constexpr int64_t kWideFrom = 16384;
template <bool GATED, int GPC, bool ZEROS>
int launch_for(const Params& p, cudaStream_t st) {
  auto sized = [&](auto split) {
    constexpr bool kSplit = decltype(split)::value;
    if (p.rows > 8) return launch_rows<2, 2, GATED, kSplit, GPC, ZEROS>(p, st);
    if constexpr (!GATED)
      if (gc::ceil_div(p.N, 16) * gc::ceil_div(p.K, kChunk) < kWideFrom) return launch_rows<1, 1, GATED, kSplit, GPC, ZEROS>(p, st);
    return launch_rows<1, 2, GATED, kSplit, GPC, ZEROS>(p, st);
  };
  if constexpr (GATED)
    if (p.N % 16) return sized(std::true_type{});
  return sized(std::false_type{});
}
template <bool GATED>
int product(const Weights& w, Params p, cudaStream_t st) {
  p.w = w.records;
  auto zeros = [&](auto gpc) {
    constexpr int kGpc = decltype(gpc)::value;
    return w.zeros ? launch_for<GATED, kGpc, true>(p, st) : launch_for<GATED, kGpc, false>(p, st);
  };
  return w.group == 32    ? zeros(std::integral_constant<int, 4>{})
         : w.group == 64 ? zeros(std::integral_constant<int, 2>{})
                         : zeros(std::integral_constant<int, 1>{});
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
      w.records, w.zeros, int(K), int(N), w.gpc(), static_cast<uint16_t*>(to), up8(K));
  return gc::check_launch("int4_unpack_kernel");
}
ToFp16 to_fp16(const Weights& w, int64_t K, int64_t N, uint16_t* to, int* exps) {
  const int64_t parts = std::min(gc::ceil_div(K, kChunk), gc::ceil_div(gc::kNumSMs * 8, gc::ceil_div(N, 16)));
  return ToFp16{w.records, to, exps, up8(K), w.zeros, int(K), int(N), w.gpc(), int(parts)};
}
int64_t ctas_of(const ToFp16& p) { return gc::ceil_div(p.N, 16) * p.parts; }
size_t unpacked_bytes(int64_t K, int64_t N) { return align256(size_t(N) * up8(K) * 2); }

// The block's operands in the workspace, and what follows them.
struct Unpacked {
  uint16_t *x, *w_in, *w_out;
  int *ex, *eh, *ein, *eout, *norms;
  int2* range;
  void* rest;
  size_t bytes;
};
Unpacked unpacked_block(char* ws, int64_t M, int64_t D, int64_t H, int64_t O) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* p = ws ? ws + at : nullptr;
    at += align256(bytes);
    return static_cast<void*>(p);
  };
  auto ints = [&](int64_t n) { return static_cast<int*>(take(size_t(n) * 4)); };
  Unpacked u;
  u.x = static_cast<uint16_t*>(take(size_t(M) * up8(D) * 2));
  u.w_in = static_cast<uint16_t*>(take(unpacked_bytes(D, 2 * H)));
  u.w_out = static_cast<uint16_t*>(take(unpacked_bytes(H, O)));
  u.ex = ints(M), u.eh = ints(M), u.ein = ints(2 * H), u.eout = ints(O);
  u.norms = ints(2 * H);
  u.range = static_cast<int2*>(take(size_t(gc::ceil_div(2 * H, 16)) * sizeof(int2)));
  u.rest = ws ? ws + at : nullptr;
  u.bytes = at;
  return u;
}

bool sizes_ok(int64_t M, int64_t K, int64_t N) {
  const int64_t top = (int64_t(1) << 30) - 512;  // coordinates are 32-bit
  return M <= top && K <= top / 8 && N <= top;
}
int weights_ok(const Weights& w, const char* what) {
  GC_REQUIRE(w.group == 32 || w.group == 64 || w.group == 128, "%s: a group is 32, 64 or 128 inputs", what);
  GC_REQUIRE(w.records, "%s: null pointer", what);
  GC_REQUIRE(gc::aligned16(w.records), "%s: weights must be 16-byte aligned", what);
  return GC_OK;
}
int zeros(uint16_t* Y, int64_t ldy, int64_t M, int64_t N, cudaStream_t st, const char* what) {
  const cudaError_t e = cudaMemset2DAsync(Y, size_t(ldy) * 2, 0, size_t(N) * 2, size_t(M), st);
  return e == cudaSuccess ? GC_OK : gc::fail(GC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
constexpr int64_t kLinearRows = 16, kBlockRows = 8;  // in the block the hidden rows are twice as many

}  // namespace

extern "C" {

size_t gc_linear_int4_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (M <= 0 || K <= 0 || N <= 0 || !sizes_ok(M, K, N)) return 0;
  if (M <= kLinearRows) return rows_bytes(M, K);
  if (M <= kLinearTileRows) return linear_tiles_workspace(M, K, N);
  return unpacked_bytes(K, N) + gc::ffn::rows_workspace(M, K, N);
}

int gc_linear_int4_bf16(const uint16_t* X, int64_t ldx, const uint8_t* W, int group, int zero_points, int64_t M, int64_t K, int64_t N,
                        uint16_t* Y, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
  GC_REQUIRE(M >= 0 && K >= 0 && N >= 0, "gc_linear_int4_bf16: negative size");
  GC_REQUIRE(ldx >= K && ldy >= N, "gc_linear_int4_bf16: leading dimension below the row length");
  if (!sizes_ok(M, K, N)) return gc::fail(GC_ERR_UNSUPPORTED, "gc_linear_int4_bf16: rows or outputs beyond 2^30, or inputs beyond 2^27");
  const cudaStream_t st = gc::as_stream(stream);
  if (M == 0 || N == 0) return GC_OK;
  GC_REQUIRE(Y, "gc_linear_int4_bf16: null pointer");
  if (K == 0) return zeros(Y, ldy, M, N, st, "gc_linear_int4_bf16");
  GC_REQUIRE(X, "gc_linear_int4_bf16: null pointer");
  const Weights w{W, group, zero_points != 0};
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
  if (M <= kLinearTileRows) return linear_tiles(X, ldx, w, M, K, N, Y, ldy, workspace, st);
  rc = unpack_to(w, K, N, workspace, st);
  if (rc != GC_OK) return rc;
  return gc::ffn::rows_times(X, ldx, static_cast<const uint16_t*>(workspace), up8(K), M, K, N, Y, ldy,
                             static_cast<char*>(workspace) + unpacked_bytes(K, N), st);
}

size_t gc_gated_ffn_int4_workspace_bytes(int64_t M, int64_t D, int64_t H, int64_t O) {
  if (M <= 0 || D <= 0 || H <= 0 || O <= 0 || !sizes_ok(M, std::max(D, H), O) || !sizes_ok(2 * H, 0, 0)) return 0;
  if (M <= kBlockRows) return rows_bytes(M, D) + rows_bytes(2 * M, H);
  if (M <= kBlockTileRows) return block_tiles_workspace(M, D, H, O);
  return unpacked_block(nullptr, M, D, H, O).bytes + gc::ffn::block_fp16_workspace(M, D, H, O);
}

int gc_gated_ffn_int4_bf16(const uint16_t* X, int64_t ldx, const uint8_t* Win, int group_in, int zero_points_in, const uint8_t* Wout,
                           int group_out, int zero_points_out, int64_t M, int64_t D, int64_t H, int64_t O, int act, uint16_t* Y,
                           int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
  GC_REQUIRE(M >= 0 && D >= 0 && H >= 0 && O >= 0, "gc_gated_ffn_int4_bf16: negative size");
  GC_REQUIRE(act >= GC_ACT_SILU && act <= GC_ACT_RELU, "gc_gated_ffn_int4_bf16: unknown activation");
  GC_REQUIRE(ldx >= D && ldy >= O, "gc_gated_ffn_int4_bf16: leading dimension below the row length");
  if (!sizes_ok(M, std::max(D, H), O) || !sizes_ok(2 * H, 0, 0)) return gc::fail(GC_ERR_UNSUPPORTED, "gc_gated_ffn_int4_bf16: rows or outputs beyond 2^30, or inputs beyond 2^27");
  const cudaStream_t st = gc::as_stream(stream);
  if (M == 0 || O == 0) return GC_OK;
  GC_REQUIRE(Y, "gc_gated_ffn_int4_bf16: null pointer");
  if (D == 0 || H == 0) return zeros(Y, ldy, M, O, st, "gc_gated_ffn_int4_bf16");
  GC_REQUIRE(X, "gc_gated_ffn_int4_bf16: null pointer");
  const Weights in{Win, group_in, zero_points_in != 0}, out{Wout, group_out, zero_points_out != 0};
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
    p.next = Wout;
    p.next_bytes = out.bytes(H, O);
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
  if (M <= kBlockTileRows) return block_tiles(X, ldx, in, out, M, D, H, O, act, Y, ldy, workspace, st);
  const Unpacked u = unpacked_block(ws, M, D, H, O);
  const ToFp16 first = to_fp16(in, D, 2 * H, u.w_in, u.ein), second = to_fp16(out, H, O, u.w_out, u.eout);
  const Columns columns{u.norms, u.range, u.ein + H, int(H)};
  int4_unpack_fp16_kernel<<<unsigned(ctas_of(first)), 256, 0, st>>>(first, columns);
  rc = gc::check_launch("int4_unpack_fp16_kernel");
  if (rc != GC_OK) return rc;
  const bool vec = gc::aligned16(X) && ldx % 8 == 0;
  auto rows = vec && D <= 256 && D % 8 == 0 ? int4_rows_fp16_kernel<true> : int4_rows_fp16_kernel<false>;
  const int row_ctas = int(std::min<int64_t>(gc::ceil_div(M, 8), gc::kNumSMs * 8)), column_ctas = int(gc::ceil_div(H, 256));
  rows<<<unsigned(row_ctas + column_ctas + ctas_of(second)), 256, 0, st>>>(X, ldx, int(M), int(D), vec, columns, second, row_ctas, column_ctas, u.x,
                                                                           up8(D), u.ex, u.eh);
  rc = gc::check_launch("int4_rows_fp16_kernel");
  if (rc != GC_OK) return rc;
  return gc::ffn::block_fp16(gc::ffn::BlockFp16{u.x, u.w_in, u.w_out, u.ex, u.eh, u.ein, u.eout}, M, D, H, O, act, Y, ldy, u.rest, st);
}

}  // extern "C"
