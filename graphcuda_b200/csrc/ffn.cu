// Gated feed-forward block on the 5th-generation tensor cores, forward and backward, bf16 (or e4m3 into the first product).
//
//   forward    G = X Wg, U = X Wu, A = act(G) * U, Y = A Wo                   [Wg | Wu] is one matrix, D x 2H
//   backward   dA = dY Wo^T, dU = dA act(G), dG = dA U act'(G)
//              dX = [dG | dU] [Wg | Wu]^T, d[Wg | Wu] = X^T [dG | dU], dWo = A^T dY
//
// One kernel, three epilogues:
//   Gated      the accumulators of a tile hold as many columns of G as of U (the same ones), so the epilogue has both and stores A
//              alone; for a backward pass G and U are stored beside it
//   GatedBack  the accumulator is a tile of dA, which is never stored: the epilogue reads G and U and stores dG and dU
//   Plain      a bf16 product: Y, dX and the weight gradients
// Operands are read where they lie: K-major or MN-major tiles (matrices whose rows run along the product's K or across it),
// so nothing is transposed in memory.  Sums are fp32 in TMEM.  A, dG and dU are rounded to bf16 where they are stored
// between kernels: they are the next product's operands, which the tensor core takes in 16 bits; that adds as much noise
// as the output's own rounding does.  G and U are no operands, and three times their rounding on top would show in dX and
// dWin: they are kept as fp16 numbers with an exponent for every 32 columns of a row, eight times as exact in as many bits.
//
// CTA = 20 warps, persistent over tiles of 128 x BN accumulators (or a pair of CTAs over 256 x BN):
//   warp 0       TMA producer of A (one lane)
//   warp 1       MMA issuer (one lane)
//   warp 2       TMEM allocator
//   warp 3       TMA producer of B (one lane)
// The three single lanes share their schedulers with the epilogue, so an instruction takes them some eight clocks and a k-block only
// 512: what they do per k-block and per tile is kept to a minimum (stages and coordinates are counted on, never divided;
// one producer for both operands and divisions per tile left the tensor cores idle half of the time at K = 256).
//   warps 4-19   epilogue: four warps per TMEM lane quarter, which take the 32-column chunks of a tile in turn; a chunk
//                leaves through swizzled 32 x 32 tiles in shared memory and TMA stores.  (Two warps to a tile of 64
//                columns, with a barrier between them: 265 us instead of 245 for A, G and U of 169,343 rows at K =
//                256, H = 1024; half of the warps on every other tile: 259; G and U in blocks that warps store and load
//                from registers: 238, but GatedBack 350 instead of 277.)
// Two accumulators in TMEM let the epilogue of a tile overlap the main loop of the next.  The epilogues are chains of
// dependent loads and special functions: with 8 warps on chunks of 64 columns they, not memory or the tensor cores, set the
// time of products with a short K.  Products with few tiles and a long K are split along K into fp32 parts that a second
// kernel adds in a fixed order.
//
// Measured, us (profiled one by one, clocks near their maximum):
//   169,343 x 256 -> 1024 -> 256, SiLU: Gated with G and U 245 (1.14 GB, 4.7 TB/s), Y 83 (1070 TFLOP/s, 5.2 TB/s), GatedBack 277 (1.48
//   GB, 5.3 TB/s), dX 139 (1280 TFLOP/s, 5.6 TB/s), dWin 129 + 4, dWout 77 + 5: memory, and in the first and third the
//   epilogue's chains.  The e4m3 first product: 149, epilogue.
//   8192 x 2048 -> 8192 -> 2048, GELU: 375, 206, 231, 402, 341, 204 = 1190 to 1610 TFLOP/s: the tensor cores, under the power limit.
//
// Up to 64 rows (kStacked) the roundings of A, dG and dU, few and dominated by the largest values, do not average out, and rows
// cost nothing there, the tiles having 128: those matrices are stored with what their rounding left as as many rows more,
// [hi; lo].  Products over their rows' columns (Y, dX) have twice the rows, whose fp32 halves are added on the way to the
// output; products along their rows (the weight gradients) take the other operand twice.  (Relative errors of the outputs of a step
// of 3 rows, 25 -> 68 -> 2336: 1.6e-3, which is the output's own rounding, against 2.8e-3.)
//
// Every wait on a barrier is bounded, as in the other tensor-core kernel: a wait that ran out raises the device's error
// word, all roles leave, copies in flight are drained and TMEM is released.
#include "common.cuh"
#include "ffn_internal.cuh"
#include "gemm_internal.cuh"
#include "tcgen05.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

namespace {

using namespace gc::tc;
using namespace gc::ffn;
using bf16 = __nv_bfloat16;

constexpr int BM = 128;
constexpr int kEpiWarps = 16, kEpiGroups = kEpiWarps / 4;
constexpr int kThreads = 128 + 32 * kEpiWarps;
constexpr int kTileBytes = 32 * 64;  // what an epilogue warp stores at once: 32 rows of 64 bytes
constexpr int kResident = 4;         // k-blocks of A that stay in shared memory, where that is all of K

enum Kind { kPlain, kGated, kGatedBack };

// RES: A stays in shared memory while the CTA goes through all columns of its rows, and only B is loaded for every tile.
template <int KIND, int BN, bool F8, bool PAIR, bool RES>
struct Cfg {
  static constexpr int BNC = PAIR ? BN / 2 : BN;  // rows of B that a CTA holds
  static constexpr int kABytes = BM * 128, kBBytes = BNC * 128;  // of a k-block: 128 bytes of K
  static constexpr int kStageBytes = (RES ? 0 : kABytes) + kBBytes;
  static constexpr int kHeldBytes = RES ? kResident * kABytes : 0;
  // tiles in shared memory per epilogue warp: two, filled in turn; GatedBack works in place on a tile of G and one of U, and
  // with a short K, where memory is the limit, on two pairs in turn
  static constexpr int kTiles = KIND == kGatedBack && RES ? 4 : 2;
  static constexpr int kScaleBytes = F8 ? kEpiWarps * 64 * 4 : 0;  // of a warp's columns of G and of U
  static constexpr int kStaging = kEpiWarps * kTiles * kTileBytes + kScaleBytes;
  static constexpr int kStages = std::min(8, (227 * 1024 - 1024 - 512 - kStaging - kHeldBytes) / kStageBytes);
  static constexpr int kSmemBytes = kHeldBytes + kStages * kStageBytes + kStaging + 512 /*barriers*/ + 1024 /*alignment*/;
  static constexpr uint32_t kTmemCols = 2 * BN;
  static_assert(kSmemBytes <= 227 * 1024 && kStages >= 2, "shared memory budget");
  static_assert(kTmemCols >= 32 && kTmemCols <= 512, "two accumulators in TMEM");
};

struct Params {
  int M, N, K;  // of the product; Gated: N = H, the columns of G and of U
  int a_bytes;  // of a k-block of A that are loaded: fewer than a tile's where M is below its rows
  int b_up;     // Gated: where U's columns start in B
  int act;
  int8_t* exps;     // G's and U's exponents, [2][ceil(N / 32)][M] (Gated: null where G and U are not stored)
  const float* sa;  // e4m3: scales of A's rows and B's columns
  const float* sb;
  bf16* C;  // Plain: the output, for rows that TMA cannot store; else what the rounding of A, or of dG | dU, left; or null
  int64_t ldc;
  int tma_store, parts;  // parts: Plain stores fp32 parts
  // columns of the product -> the c_cols columns of C: those from `gap_from` on move down by `gap`, over the ones in between
  int gap_from, gap, c_cols;
  int splits, kb_per_split;
  int* word;  // the device's error word
};

// One MMA of 32 bytes of K.
template <bool PAIR, bool F8>
__device__ __forceinline__ void umma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
#define GC_UMMA(GROUP, KIND)                                                                    \
  asm volatile(                                                                                 \
      "{\n\t.reg .pred p;\n\t"                                                                  \
      "setp.ne.b32 p, %4, 0;\n\t"                                                               \
      "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), \
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)                                       \
      : "memory")
  if constexpr (PAIR && F8) GC_UMMA("2", "f8f6f4");
  else if constexpr (PAIR) GC_UMMA("2", "f16");
  else if constexpr (F8) GC_UMMA("1", "f8f6f4");
  else GC_UMMA("1", "f16");
#undef GC_UMMA
}

// Instruction descriptor, fp32 accumulation.  Operand formats: kind::f16 1 = bf16; kind::f8f6f4 0 = e4m3.
__host__ __device__ constexpr uint32_t make_idesc(int bm, int bn, bool a_mn, bool b_mn, bool f8) {
  return (1u << 4) | (uint32_t(f8 ? 0 : 1) << 7) | (uint32_t(f8 ? 0 : 1) << 10) | (uint32_t(a_mn) << 15) |
         (uint32_t(b_mn) << 16) | (uint32_t(bn >> 3) << 17) | (uint32_t(bm >> 4) << 24);
}

// Tiles in shared memory are rows of 128 bytes under the 128-byte swizzle (16-byte atoms).  K-major: a row is 128 bytes of K
// of one index, 8-row groups 1024 bytes apart, one MMA takes 32 bytes of every row.  MN-major (bf16): a row is 64
// consecutive indices at one k, 8-k groups 1024 bytes apart, 64-index blocks 64 rows (8192 bytes) apart, one MMA
// takes 16 rows.
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, bool mn_major) {
  return mn_major ? smem_desc(saddr, 64 * 128, 1024, 2u) : smem_desc(saddr, 0, 1024, 2u);
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
               "r"(src)
               : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y),
               "r"(z), "r"(src)
               : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// At most N of this thread's stores still read shared memory.
template <int N>
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Waits for a phase of a barrier, bounded.  The thread sleeps in the barrier unit between tries (a microsecond at most): twenty
// warps that poll take issue slots from the lanes that feed the tensor cores, and power from all.  Returns false when the CTA is
// aborting (this wait or another ran out).
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort_s) {
  constexpr uint32_t kTries = 1u << 21;
  for (uint32_t i = 0; i < kTries; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if (*abort_s) return false;
  }
  *abort_s = 1;
  return false;
}
// Waits for a copy in flight whatever else has failed (bounded): it must have landed before the CTA may exit.
__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < kWaitLimit; ++i) {
    if (mbar_test(bar, parity)) break;
    __nanosleep(64);
  }
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}

__device__ __forceinline__ uint32_t pack2(F2 a) {
  float x, y;
  a.get(x, y);
  return pack2(x, y);
}
// What that left of a, rounded in its turn; nothing where it is not finite.
__device__ __forceinline__ uint32_t pack_rest(F2 a, uint32_t packed) {
  float x, y;
  a.get(x, y);
  const uint32_t lo = packed << 16, hi = packed & 0xFFFF0000u;
  return pack2((lo & 0x7F800000u) == 0x7F800000u ? 0.f : x - __uint_as_float(lo),
               (hi & 0x7F800000u) == 0x7F800000u ? 0.f : y - __uint_as_float(hi));
}

// A tile in shared memory: 32 rows of 64 bytes, their 16-byte units swizzled as TMA does it.  row_at is the address of unit
// 0 of a row; unit j is where its bits 4 and 5 are XORed with j.
__device__ __forceinline__ uint32_t row_at(uint32_t tile, int row) { return tile + row * 64 + (((row >> 1) & 3) << 4); }
__device__ __forceinline__ void store_unit(uint32_t lane_at, int j, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(lane_at ^ (j << 4)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 load_unit(uint32_t lane_at, int j) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(lane_at ^ (j << 4))
               : "memory");
  return v;
}

__device__ __forceinline__ uint16_t load_column(uint32_t tile, int row, int column) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"((row_at(tile, row) ^ (column / 8 << 4)) + column % 8 * 2) : "memory");
  return v;
}

// Eight floats from shared memory, the same for all lanes.
__device__ __forceinline__ void load_8(uint32_t at, F2 (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
    asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(v[2 * j].v), "=l"(v[2 * j + 1].v) : "r"(at + 16 * j) : "memory");
}

// 32 values to a row of a tile as fp16 with a common power of two, which is returned.  SIGN: see stay_positive.
template <bool SIGN>
__device__ __forceinline__ int pack_fp16(const uint32_t (&v)[32], uint32_t lane_at) {
  __half2 top[2] = {__float2half2_rn(0.f), __float2half2_rn(0.f)};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = __uint_as_float(v[j * 8 + 2 * e]), y = __uint_as_float(v[j * 8 + 2 * e + 1]);
      const __half2 h = SIGN ? __floats2half2_rn(stay_positive(x), stay_positive(y)) : __floats2half2_rn(x, y);
      top[e & 1] = __hmax2(top[e & 1], __habs2(h));
      w[e] = *reinterpret_cast<const uint32_t*>(&h);
    }
    store_unit(lane_at, j, w[0], w[1], w[2], w[3]);
  }
  top[0] = __hmax2(top[0], top[1]);
  const uint32_t t = *reinterpret_cast<const uint32_t*>(&top[0]), most = max(t & 0xFFFFu, t >> 16);
  if (fits_fp16(most)) return 0;
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) bits = max(bits, finite_bits(v[j]));
  const int e = shared_exponent(bits);
  const float2 f = unscale(e);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = j * 8 + 2 * k;
      const float x = __uint_as_float(v[i]) * f.x * f.y, y = __uint_as_float(v[i + 1]) * f.x * f.y;
      const __half2 h = SIGN ? __floats2half2_rn(stay_positive(x), stay_positive(y)) : __floats2half2_rn(x, y);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    store_unit(lane_at, j, w[0], w[1], w[2], w[3]);
  }
  return e;
}
__device__ __forceinline__ F2 unpack_fp16(uint32_t w, F2 scale) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return F2(f.x, f.y) * scale;
}

// Where a column of the product goes (see Params); one that is dropped goes beyond the last.
__device__ __forceinline__ int out_column(int n, int gap_from, int gap) {
  return n < gap_from ? n : n < gap_from + gap ? 0x7FFFFFFF : n - gap;
}

struct Maps {
  CUtensorMap a, b;
  CUtensorMap out;      // Plain: C, or the fp32 parts; Gated: A; GatedBack: dG
  CUtensorMap out2;     // Gated: G; GatedBack: dU
  CUtensorMap out3;     // Gated: U
  CUtensorMap in1, in2;  // GatedBack: G, U
};

// A_MN / B_MN: the operand is MN-major.  F8: e4m3 operands (K-major).  PAIR: two CTAs of a cluster work on a tile of 256 rows,
// each with its 128 rows of A and half of B's (Gated: rank 0 has G's columns, rank 1 U's).  RES: see Cfg.  LO: what roundings left is
// stored too.
template <int KIND, int BN, bool A_MN, bool B_MN, bool F8, bool PAIR, bool RES, bool LO>
__global__ void __launch_bounds__(kThreads, 1)
ffn_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  using C_ = Cfg<KIND, BN, F8, PAIR, RES>;
  constexpr int S = C_::kStages, BNC = C_::BNC;
  constexpr int KE = F8 ? 128 : 64;  // K elements per k-block
  constexpr int TM = PAIR ? 2 * BM : BM;
  constexpr int NT = KIND == kGated ? BN / 2 : BN;  // output columns of a tile
  static_assert(!F8 || (!A_MN && !B_MN && KIND == kGated), "e4m3 operands are K-major");
  static_assert(!RES || (!A_MN && KIND != kPlain), "A is held K-major, for short products");
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  const int unit = PAIR ? int(blockIdx.x / 2) : int(blockIdx.x), units = PAIR ? int(gridDim.x / 2) : int(gridDim.x);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  auto sHeld = [&](int kb) { return base + kb * C_::kABytes; };
  auto sA = [&](int s) { return base + C_::kHeldBytes + s * C_::kStageBytes; };
  auto sB = [&](int s) { return sA(s) + (RES ? 0 : C_::kABytes); };
  const uint32_t staging = base + C_::kHeldBytes + S * C_::kStageBytes;
  const uint32_t bars = staging + C_::kStaging;
  auto bar_full = [&](int s) { return bars + 8 * s; };
  auto bar_empty = [&](int s) { return bars + 8 * (S + s); };
  auto bar_tfull = [&](int b) { return bars + 8 * (2 * S + b); };
  auto bar_tempty = [&](int b) { return bars + 8 * (2 * S + 2 + b); };
  auto bar_afull = [&](int kb) { return bars + 8 * (2 * S + 4 + kb); };  // RES: a k-block of A
  auto bar_aempty = [&](int kb) { return bars + 8 * (2 * S + 4 + kResident + kb); };
  auto bar_in = [&](int i) { return bars + 8 * (2 * S + 4 + 2 * kResident + i); };  // GatedBack: G and U have landed
  constexpr int kPlaces = KIND == kGatedBack ? C_::kTiles / 2 : 1;  // for a tile of G and one of U, per warp
  static_assert(8 * (2 * S + 4 + 2 * kResident + kPlaces * kEpiWarps) <= 512, "room for the barriers");
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int tiles_n = (p.N + NT - 1) / NT;
  const int tiles_m = (p.M + TM - 1) / TM;
  const int nkb_total = (p.K + KE - 1) / KE;
  const int splits = KIND == kPlain ? p.splits : 1;
  const int kb_per = splits > 1 ? p.kb_per_split : nkb_total;
  const int num_items = tiles_m * tiles_n * splits;  // (split, m, n), n fastest
  // This CTA's items: every units-th, or (RES) a run of them, so that A changes once per row of tiles.
  const int first_item = RES ? int(int64_t(num_items) * unit / units) : unit;
  const int my_tiles = RES ? int(int64_t(num_items) * (unit + 1) / units) - first_item
                           : unit < num_items ? (num_items - unit + units - 1) / units : 0;
  // Tile t = from, from + by, .. of this CTA.  RES: n fastest, in coordinates that are divided once and counted on from there.
  // Otherwise (split, group of 8 rows of tiles, n, m within the group): the tiles that run at one time are a square of the
  // product, not a strip of it, so that what they read stays in the L2 and near (8192 x 2048 -> 8192 -> 2048, a step back to
  // back with the card at its power limit: 2232 us with groups of 1, 2159 with 4, 2125 with 8, 2123 with 16).
  struct Tile {
    int t, m, n, split, by, dm, dn;
  };
  constexpr int kGroup = 8;
  auto place = [&](Tile& x) {
    int i = first_item + x.t * units;
    if (splits > 1) x.split = i / (tiles_m * tiles_n), i -= x.split * (tiles_m * tiles_n);
    const int g = i / (kGroup * tiles_n), r = i - g * (kGroup * tiles_n), high = min(kGroup, tiles_m - g * kGroup);
    x.n = r / high;
    x.m = g * kGroup + r - x.n * high;
  };
  auto tile_at = [&](int from, int by) {
    Tile x{from, 0, 0, 0, by, 0, 0};
    if (RES) {
      x.m = (first_item + from) / tiles_n, x.n = (first_item + from) % tiles_n;
      x.dm = by / tiles_n, x.dn = by % tiles_n;
    } else {
      place(x);
    }
    return x;
  };
  auto next = [&](Tile& x) {
    x.t += x.by;
    if (RES) {
      x.n += x.dn;
      x.m += x.dm;
      if (x.n >= tiles_n) x.n -= tiles_n, ++x.m;
    } else if (x.t < my_tiles) {
      place(x);
    }
  };
  auto row_of = [&](const Tile& x) { return x.m * TM + int(rank) * BM; };  // first row of this CTA's half
  auto first_kb = [&](const Tile& x) { return x.split * kb_per; };
  auto last_kb = [&](const Tile& x) { return min(nkb_total, x.split * kb_per + kb_per); };

  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int s = 0; s < S; ++s) {
      mbar_init(bar_full(s), RES ? 1 : 2);  // B's producer, and A's
      mbar_init(bar_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_tfull(b), 1);
      mbar_init(bar_tempty(b), kEpiWarps * (PAIR ? 2 : 1));
    }
    for (int kb = 0; kb < kResident; ++kb) {
      mbar_init(bar_afull(kb), 1);
      mbar_init(bar_aempty(kb), 1);
    }
    for (int i = 0; i < kPlaces * kEpiWarps; ++i) mbar_init(bar_in(i), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (PAIR) {
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers exist before either is signalled
  }
  if (warp == 2) tmem_alloc<PAIR>(smem_u32(&tmem_base_s), C_::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_s;
  volatile int* abort_p = &abort_s;

  if ((warp == 0 || warp == 3) && lane == 0) {
    // ------------------------------------------------------------ TMA producers: A, B
    const bool is_a = warp == 0;
    // a pair's copies are all counted at the leader
    auto expect = [&](uint32_t bar, uint32_t bytes) {
      if (!PAIR) mbar_expect_tx(bar, bytes);
      else if (rank == 0) mbar_expect_tx(bar, 2 * bytes);
    };
    auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
      if (PAIR) tma_load_2d_leader(dst, map, x, y, bar);
      else tma_load_2d(dst, map, x, y, bar);
    };
    bool ok = true;
    if (RES && is_a) {
      uint32_t rows = 0, held = 0;  // whole A's fetched; k-blocks of the one that is being fetched
      for (Tile x = tile_at(0, 1); x.t < my_tiles && ok; next(x)) {
        if (x.t > 0 && x.n > 0) continue;  // the A of the tile before
        for (int kb = 0; kb < nkb_total; ++kb) {
          if (!wait(bar_aempty(kb), (rows & 1u) ^ 1u, abort_p)) { ok = false; break; }
          expect(bar_afull(kb), C_::kABytes);
          load(sHeld(kb), &maps.a, kb * KE, row_of(x), bar_afull(kb));
          ++held;
        }
        if (ok) ++rows, held = 0;
      }
      // every copy issued must have landed before the CTA may exit (counted at the leader, for whom the peer waits)
      for (uint32_t kb = 0; kb < uint32_t(nkb_total) && (!PAIR || rank == 0); ++kb) {
        const uint32_t fetched = rows + (kb < held ? 1u : 0u);
        if (fetched) drain(bar_afull(kb), (fetched - 1) & 1u);
      }
    } else {
      uint32_t s = 0, phase = 0, issued = 0;
      for (Tile x = tile_at(0, 1); x.t < my_tiles && ok; next(x)) {
        const int m0 = row_of(x), kb1 = last_kb(x);
        // Gated takes the tile's columns of G, then the same of U
        const int n0 = KIND == kGated ? x.n * NT + (PAIR && rank ? p.b_up : 0) : x.n * NT + int(rank) * BNC;
        for (int kb = first_kb(x); kb < kb1; ++kb) {
          if (!wait(bar_empty(s), phase ^ 1u, abort_p)) { ok = false; break; }
          const uint32_t bar = bar_full(s);
          if (is_a) {
            expect(bar, p.a_bytes);
            if (A_MN) {
#pragma unroll
              for (int c = 0; c < BM / 64; ++c) load(sA(s) + c * (64 * 128), &maps.a, m0 + c * 64, kb * KE, bar);
            } else {
              load(sA(s), &maps.a, kb * KE, m0, bar);
            }
          } else {
            expect(bar, C_::kBBytes);
            constexpr int kRows = KIND == kGated && !PAIR ? BNC / 2 : BNC;
#pragma unroll
            for (int part = 0; part < BNC / kRows; ++part) {
              const int n = n0 + part * p.b_up;
              const uint32_t dst = sB(s) + part * kRows * 128;
              if (B_MN) {
#pragma unroll
                for (int c = 0; c < kRows / 64; ++c) load(dst + c * (64 * 128), &maps.b, n + c * 64, kb * KE, bar);
              } else {
                load(dst, &maps.b, kb * KE, n, bar);
              }
            }
          }
          ++issued;
          if (++s == uint32_t(S)) s = 0, phase ^= 1u;
        }
      }
      if (!PAIR || rank == 0)
        for (uint32_t j = 0; j < issued && j < uint32_t(S); ++j) {  // as above
          if (s == 0) phase ^= 1u;
          s = s == 0 ? S - 1 : s - 1;
          drain(bar_full(s), phase);
        }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = make_idesc(TM, BN, A_MN, B_MN, F8);
      constexpr uint32_t kAStep = A_MN ? 16 * 128 : 32, kBStep = B_MN ? 16 * 128 : 32;  // bytes per MMA
      const uint64_t da0 = operand_desc(RES ? sHeld(0) : sA(0), A_MN), db0 = operand_desc(sB(0), B_MN);
      uint32_t s = 0, phase = 0, rows = 0;
      bool ok = true;
      for (Tile x = tile_at(0, 1); x.t < my_tiles && ok;) {
        const int b = x.t & 1, kb0 = first_kb(x), kb1 = last_kb(x);
        const uint32_t turn = (x.t >> 1) & 1u;
        const bool new_a = RES && (x.t == 0 || x.n == 0);
        next(x);
        const bool last_of_a = RES && (x.t >= my_tiles || x.n == 0);
        if (!wait(bar_tempty(b), turn ^ 1u, abort_p)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + uint32_t(b * BN);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (new_a && !wait(bar_afull(kb), rows & 1u, abort_p)) { ok = false; break; }
          if (!wait(bar_full(s), phase, abort_p)) { ok = false; break; }
          tc_fence_after();
          const uint64_t da = da0 + (RES ? uint32_t(kb) * (C_::kABytes >> 4) : s * (C_::kStageBytes >> 4));
          const uint64_t db = db0 + s * (C_::kStageBytes >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma<PAIR, F8>(d_tmem, da + ((k * kAStep) >> 4), db + ((k * kBStep) >> 4), idesc, (kb > kb0 || k > 0) ? 1u : 0u);
          umma_commit<PAIR>(bar_empty(s));  // frees the stage once these MMAs have read it
          if (last_of_a) umma_commit<PAIR>(bar_aempty(kb));
          if (++s == uint32_t(S)) s = 0, phase ^= 1u;
        }
        if (new_a) ++rows;
        if (ok) umma_commit<PAIR>(bar_tfull(b));
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int q = warp % 4;  // TMEM lane quarter
    const int grp = (warp - 4) / 4;  // which of the 32-column chunks: grp, grp + 4, ..
    const uint32_t tiles = staging + (warp - 4) * (C_::kTiles * kTileBytes);
    const uint32_t lane_at = row_at(tiles, lane);
    const int64_t exps_u = int64_t((p.N + 31) / 32) * p.M;  // from G's table of exponents to U's
    uint32_t buf = 0;  // byte offset of the tile that was filled last
    bool ok = true;
    // The same answer for all of a warp.
    auto wait_warp = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, wait(bar, parity, abort_p)) != 0; };
    // The next of the warp's tiles, once the store that read it last has done so.
    auto acquire = [&]() {
      if (lane == 0) store_wait_read<1>();
      __syncwarp();
      buf ^= kTileBytes;
      return buf;
    };
    // Hands a filled tile to the TMA store.
    auto put = [&](const CUtensorMap* map, uint32_t at, int col, int row) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(map, tiles + at, col, row);
        store_commit();
      }
    };

    // GatedBack: the warp's chunks in their order, and the copies of G and U for them.
    Tile ahead = tile_at(0, 1);
    int ahead_c = grp;
    auto find_chunk = [&]() {  // the next that exists, from there on
      for (; ahead.t < my_tiles; next(ahead), ahead_c = grp)
        if (row_of(ahead) + q * 32 < p.M && ahead_c < NT / 32 && ahead.n * NT + ahead_c * 32 < p.N) return true;
      return false;
    };
    uint32_t asked = 0, used = 0;  // copies
    auto request = [&]() {
      if (lane == 0) {
        const int col = ahead.n * NT + ahead_c * 32, row = row_of(ahead) + q * 32;
        const uint32_t at = asked % kPlaces, bar = bar_in((warp - 4) * kPlaces + at), dst = tiles + at * 2 * kTileBytes;
        store_wait_read<0>();  // what was put from these tiles has left them
        mbar_expect_tx(bar, 2 * kTileBytes);
        tma_load_2d(dst, &maps.in1, col, row, bar);
        tma_load_2d(dst + kTileBytes, &maps.in2, col, row, bar);
      }
      ++asked;
      ahead_c += kEpiGroups;
    };
    if (KIND == kGatedBack && find_chunk()) request();

    for (Tile x = tile_at(0, 1); x.t < my_tiles && ok; next(x)) {
      const int b = x.t & 1, n0 = x.n * NT;
      const int row0 = row_of(x) + q * 32, row = row0 + lane;  // the warp's first row, the lane's
      const uint32_t taddr = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(b * BN);
      if (!wait_warp(bar_tfull(b), (x.t >> 1) & 1u)) {
        ok = false;
        break;
      }
      tc_fence_after();
      // Gives the accumulator back as soon as the warp's last chunk is in registers.
      bool held = true;
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_leader(bar_tempty(b));
          else mbar_arrive(bar_tempty(b));
        }
        held = false;
      };
      auto loaded = [&](int c) {
        tmem_ld_wait();
        if (c + kEpiGroups >= NT / 32 || n0 + (c + kEpiGroups) * 32 >= p.N) release();
      };
      for (int c = grp; c < NT / 32; c += kEpiGroups) {
        const int col = n0 + c * 32;
        if (col >= p.N || row0 >= p.M) break;
        const uint32_t acc_at = taddr + uint32_t(c * 32);
        if constexpr (KIND == kGatedBack) {
          // the next chunk's copies go out before this one is worked on, where there are tiles for them
          if (kPlaces > 1 && find_chunk()) request();
          const int64_t at = int64_t(col / 32) * p.M + min(row, p.M - 1);
          const float sg = __uint_as_float(uint32_t(127 + p.exps[at]) << 23);
          const float su = __uint_as_float(uint32_t(127 + p.exps[at + exps_u]) << 23);
          const uint32_t place = used % kPlaces, at_g = lane_at + place * 2 * kTileBytes, at_u = at_g + kTileBytes;
          uint32_t acc[32];
          tmem_ld32(acc_at, acc);
          if (!wait_warp(bar_in((warp - 4) * kPlaces + place), (used / kPlaces) & 1u)) {
            ok = false;
            break;
          }
          ++used;
          loaded(c);
          with_activation(p.act, [&](auto act) {
            const F2 fg = both(sg), fu = both(su);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint4 g4 = load_unit(at_g, j), u4 = load_unit(at_u, j);
              uint32_t* gw = &g4.x;
              uint32_t* uw = &u4.x;
              uint32_t rest_g[4], rest_u[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const F2 d(acc[j * 8 + 2 * e], acc[j * 8 + 2 * e + 1]);
                const F2 u = unpack_fp16(uw[e], fu);
                F2 slope;
                const F2 a = activate<decltype(act)::value>(unpack_fp16(gw[e], fg), slope);
                const F2 dg = d * u * slope, du = d * a;
                gw[e] = pack2(dg);
                uw[e] = pack2(du);
                if (LO) {
                  rest_g[e] = pack_rest(dg, gw[e]);
                  rest_u[e] = pack_rest(du, uw[e]);
                }
              }
              if (LO && row < p.M && col + 8 * j < p.N) {
                bf16* to = p.C + row * p.ldc + col + 8 * j;
                *reinterpret_cast<uint4*>(to) = make_uint4(rest_g[0], rest_g[1], rest_g[2], rest_g[3]);
                *reinterpret_cast<uint4*>(to + p.N) = make_uint4(rest_u[0], rest_u[1], rest_u[2], rest_u[3]);
              }
              store_unit(at_g, j, g4.x, g4.y, g4.z, g4.w);
              store_unit(at_u, j, u4.x, u4.y, u4.z, u4.w);
            }
          });
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&maps.out, tiles + place * 2 * kTileBytes, col, row0);
            tma_store_2d(&maps.out2, tiles + place * 2 * kTileBytes + kTileBytes, col, row0);
            store_commit();
          }
          if (kPlaces == 1 && find_chunk()) request();
        } else if constexpr (KIND == kGated) {
          const float sa = F8 ? p.sa[min(row, p.M - 1)] : 1.f;
          const uint32_t scales = staging + C_::kStaging - C_::kScaleBytes + (warp - 4) * 256;
          if (F8) {
            const int n = min(col + lane, p.N - 1);
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(scales + 4 * lane), "f"(__ldg(p.sb + n)) : "memory");
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(scales + 128 + 4 * lane), "f"(__ldg(p.sb + p.b_up + n)) : "memory");
          }
          uint32_t g[32], u[32];
          tmem_ld32(acc_at, g);
          tmem_ld32(acc_at + uint32_t(NT), u);
          loaded(c);
          if (!F8 && p.exps) {
            const int64_t at = int64_t(col / 32) * p.M + row;
            if (col + 32 > p.N) {  // what lies beyond has no say in the exponents
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (col + i >= p.N) g[i] = u[i] = 0;
            }
            const uint32_t bg = acquire();
            const int eg = p.act == GC_ACT_RELU ? pack_fp16<true>(g, lane_at + bg) : pack_fp16<false>(g, lane_at + bg);
            put(&maps.out2, bg, col, row0);
            const uint32_t bu = acquire();
            const int eu = pack_fp16<false>(u, lane_at + bu);
            put(&maps.out3, bu, col, row0);
            if (row < p.M) {
              p.exps[at] = int8_t(eg);
              p.exps[at + exps_u] = int8_t(eu);
            }
          }
          const uint32_t bo = acquire();
          if (F8) __syncwarp();  // the scales are written
          with_activation(p.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t w[4], rest[4];
              F2 sg[4], su[4];
              if (F8) {
                load_8(scales + 32 * j, sg);
                load_8(scales + 128 + 32 * j, su);
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int i = j * 8 + 2 * e;
                F2 vg(g[i], g[i + 1]), vu(u[i], u[i + 1]), unused;
                if (F8) vg = vg * (both(sa) * sg[e]), vu = vu * (both(sa) * su[e]);
                const F2 a = activate<decltype(act)::value>(vg, unused) * vu;
                w[e] = pack2(a);
                if (LO) rest[e] = pack_rest(a, w[e]);
              }
              if (LO && row < p.M && col + 8 * j < p.N)
                *reinterpret_cast<uint4*>(p.C + row * p.ldc + col + 8 * j) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
              store_unit(lane_at + bo, j, w[0], w[1], w[2], w[3]);
            }
          });
          put(&maps.out, bo, col, row0);
        } else {
          uint32_t acc[32];
          tmem_ld32(acc_at, acc);
          loaded(c);
          if (p.parts) {
            // fp32 parts, 16 columns to a tile
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t bo = acquire();
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int i = half * 16 + 4 * j;
                store_unit(lane_at + bo, j, acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
              }
              fence_async_smem();
              __syncwarp();
              if (lane == 0) {
                if (col + half * 16 < p.N) tma_store_3d(&maps.out, tiles + bo, col + half * 16, row0, x.split);
                store_commit();
              }
            }
          } else {
            const uint32_t bo = acquire();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = pack2(F2(acc[j * 8 + 2 * e], acc[j * 8 + 2 * e + 1]));
              store_unit(lane_at + bo, j, w[0], w[1], w[2], w[3]);
            }
            if (p.tma_store) {
              put(&maps.out, bo, col, row0);
            } else {
              // rows of an odd pitch: a row at a time, a column per lane
              __syncwarp();
              const int n = out_column(col + lane, p.gap_from, p.gap), rows = min(32, p.M - row0);
              if (n < p.c_cols)
                for (int r = 0; r < rows; ++r)
                  p.C[int64_t(row0 + r) * p.ldc + n] = __ushort_as_bfloat16(load_column(tiles + bo, r, lane));
            }
          }
        }
      }
      if (held) release();
    }
    if (KIND == kGatedBack && lane == 0)  // copies that were asked for and not waited for have to land all the same
      for (; used != asked; ++used) drain(bar_in((warp - 4) * kPlaces + used % kPlaces), (used / kPlaces) & 1u);
    if (lane == 0) store_wait_all();  // shared memory is read until then
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // the peer's MMAs read this CTA's shared memory and write its TMEM until here
  tc_fence_after();
  if (warp == 2) tmem_dealloc<PAIR>(tmem_base, C_::kTmemCols);
  if (threadIdx.x == 0 && abort_s) atomicExch(p.word, 1);
}

// C (bf16) = the sum of the fp32 parts [split][M][pitch] in their order, four columns per thread.
__global__ void __launch_bounds__(256)
ffn_sum_kernel(const float* __restrict__ parts, int splits, int M, int pitch, bf16* __restrict__ C, int64_t ldc, int c_cols,
               int gap_from, int gap) {
  const int64_t quads = int64_t(M) * (pitch / 4);
  const bool vec = gap == 0 && c_cols % 4 == 0 && ldc % 4 == 0 && reinterpret_cast<uintptr_t>(C) % 8 == 0;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < quads; i += int64_t(gridDim.x) * 256) {
    const int64_t m = i / (pitch / 4);
    const int n = int(i % (pitch / 4)) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int z = 0; z < splits; ++z) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(parts + (int64_t(z) * M + m) * pitch + n));
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    if (vec) {
      *reinterpret_cast<uint2*>(C + m * ldc + n) = make_uint2(pack2(s.x, s.y), pack2(s.z, s.w));
    } else {
      const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = out_column(n + e, gap_from, gap);
        if (c < c_cols) C[m * ldc + c] = __float2bfloat16_rn(v[e]);
      }
    }
  }
}

// Copies of matrices whose rows TMA cannot read, all of a call in one launch: dst[r, c] = src[r, c] for c < cols, 0 up to
// `width`, a multiple of 4 bytes in rows that are 4-byte aligned.  A warp takes runs of kRun words of a row in turn, a lane a
// word of the copy (whole rows: 15 us for 16 of 2048 columns, four times).
struct Copies {
  static constexpr int kMost = 7, kRun = 128;
  struct Job {
    const void* src;
    void* dst;
    int64_t lds, ldd, rows;
    int cols, width, size;  // size: bytes of an element, 1 or 2
  } job[kMost];
  int first_block[kMost + 1];  // prefix sum of the CTAs that a job gets
  int count;
};
__global__ void __launch_bounds__(256)
repitch_kernel(const __grid_constant__ Copies c) {
  int j = 0;
  while (j + 1 < c.count && int(blockIdx.x) >= c.first_block[j + 1]) ++j;
  const Copies::Job& job = c.job[j];
  const int lane = threadIdx.x % 32, blocks = c.first_block[j + 1] - c.first_block[j];
  const int per = 4 / job.size;  // elements of a word
  const int words = job.width / per, runs = (words + Copies::kRun - 1) / Copies::kRun;
  for (int64_t i = int64_t(blockIdx.x - c.first_block[j]) * 8 + threadIdx.x / 32; i < job.rows * runs; i += int64_t(blocks) * 8) {
    const int64_t r = i / runs;
    const int from = int(i - r * runs) * Copies::kRun, to = min(words, from + Copies::kRun);
    const uint8_t* src = static_cast<const uint8_t*>(job.src) + r * job.lds * job.size;
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(job.dst) + r * job.ldd * job.size);
#pragma unroll 4
    for (int w = from + lane; w < to; w += 32) {
      uint32_t word = 0;
      if (job.size == 2) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (2 * w + e < job.cols) word |= uint32_t(reinterpret_cast<const uint16_t*>(src)[2 * w + e]) << (16 * e);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * w + e < job.cols) word |= uint32_t(src[4 * w + e]) << (8 * e);
      }
      dst[w] = word;
    }
  }
}

// ------------------------------------------------------------------ host
struct Matrix {  // row-major, `size` bytes per element
  const void* p;
  int64_t rows, cols, ld;
  int size;
};

// Boxes with rows of 128 bytes are operands; the epilogues' have 64.
int make_map(CUtensorMap* map, const Matrix& m, int box_cols, int box_rows, int64_t planes = 0) {
  EncodeFn enc = get_encode();
  if (!enc) return gc::fail(GC_ERR_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const cuuint64_t dims[3] = {cuuint64_t(m.cols), cuuint64_t(m.rows), cuuint64_t(planes)};
  const cuuint64_t strides[2] = {cuuint64_t(m.ld) * m.size, cuuint64_t(m.ld) * m.size * m.rows};
  const cuuint32_t box[3] = {cuuint32_t(box_cols), cuuint32_t(box_rows), 1u};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType type = m.size == 4   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : m.size == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const CUresult r = enc(map, type, planes ? 3 : 2, const_cast<void*>(m.p), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE,
                         box_cols * m.size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return gc::fail(GC_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", int(r));
  return GC_OK;
}

inline int64_t up8(int64_t x) { return (x + 7) & ~int64_t(7); }
inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// A launch's tile: accumulator columns, and whether CTAs work in pairs.
struct Tile {
  int bn;
  bool pair;
};
// Pairs of CTAs on 256 x 256 where that gives every pair a tile; 128 x 128 below, and 128 x 64 where even those are fewer
// than the SMs (a product with few rows is bound by reading B, which more CTAs do faster).
Tile pick_tile(Kind kind, int64_t M, int64_t N, int64_t splits_possible) {
  const int64_t n_acc = kind == kGated ? 2 * N : N;
  const int64_t big = gc::ceil_div(M, 256) * gc::ceil_div(n_acc, 256) * splits_possible;
  if (M > BM && n_acc > 128 && big >= gc::kNumSMs / 2) return {256, true};
  if (kind == kGated) return {128, false};
  const int64_t mid = gc::ceil_div(M, BM) * gc::ceil_div(n_acc, 128) * splits_possible;
  return {n_acc > 64 && mid >= gc::kNumSMs ? 128 : 64, false};
}
// Plain products with at most half as many tiles as CTAs and a long K are cut along K, into at least 4 k-blocks each.  The
// launch that adds the parts costs 2 to 3 us, as much as some ten k-blocks: from 16 k-blocks on (steps of seven sizes, 40 x
// 1024 to 9000 x 300: from 8 on 1 to 5 % slower on the small ones, from 24 or 32 on and into 8 the same or up to 5 %).
struct Split {
  Tile tile;
  int splits, per;
};
Split plan_plain(int64_t M, int64_t N, int64_t K) {
  const int64_t nkb = gc::ceil_div(K, 64);
  Split s;
  s.tile = pick_tile(kPlain, M, N, std::max<int64_t>(1, nkb / 8));
  const int64_t tm = s.tile.pair ? 256 : BM, units = s.tile.pair ? gc::kNumSMs / 2 : gc::kNumSMs;
  const int64_t tiles = gc::ceil_div(M, tm) * gc::ceil_div(N, s.tile.bn);
  int64_t splits = 1;
  if (tiles * 2 <= units && nkb >= 16) splits = std::min<int64_t>(units / tiles, nkb / 4);
  s.per = int(gc::ceil_div(nkb, std::max<int64_t>(1, splits)));
  s.splits = int(gc::ceil_div(nkb, s.per));
  return s;
}
inline int64_t part_pitch(int64_t N) { return (N + 3) & ~int64_t(3); }
// Rows of which A, dG and dU are kept in two bf16 numbers each, [hi; lo].
constexpr int64_t kStacked = BM / 2;
int64_t stack(int64_t M) { return M <= kStacked ? 2 : 1; }
size_t plain_workspace(int64_t M, int64_t N, int64_t K, int64_t halves = 1) {
  M *= halves;
  const Split s = plan_plain(M, N, K);
  return s.splits > 1 || halves > 1 ? align256(size_t(s.splits) * size_t(M) * size_t(part_pitch(N)) * 4) : 0;
}

int error_word(int** word) {
  static std::atomic<int*> cached[64] = {};  // by device; the address does not change
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return gc::fail(GC_ERR_CUDA, "no current device");
  if (dev < 64 && (*word = cached[dev].load(std::memory_order_relaxed))) return GC_OK;
  int32_t* w = nullptr;
  const int rc = gc::wait_error_word(&w);
  if (rc != GC_OK) return rc;
  if (dev < 64) cached[dev].store(w, std::memory_order_relaxed);
  *word = w;
  return GC_OK;
}

template <int KIND, int BN, bool A_MN, bool B_MN, bool F8, bool PAIR, bool RES, bool LO = false>
int launch_kernel(const Maps& maps, const Params& p, cudaStream_t st) {
  using C_ = Cfg<KIND, BN, F8, PAIR, RES>;
  auto kern = ffn_kernel<KIND, BN, A_MN, B_MN, F8, PAIR, RES, LO>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C_::kSmemBytes);
  if (e != cudaSuccess) return gc::fail(GC_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  constexpr int kCtas = PAIR ? 2 : 1;
  constexpr int NT = KIND == kGated ? BN / 2 : BN;
  const int64_t items = gc::ceil_div(p.M, BM * kCtas) * gc::ceil_div(p.N, NT) * (KIND == kPlain ? p.splits : 1);
  if (items > 0x7FFFFFFF) return gc::fail(GC_ERR_UNSUPPORTED, "gated feed-forward: too many tiles");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(std::min<int64_t>(items, gc::kNumSMs / kCtas)) * kCtas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C_::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = PAIR ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kern, maps, p);
  return gc::check_launch("ffn_kernel");
}
template <int KIND, bool A_MN, bool B_MN, bool F8>
int launch_tile(const Tile& t, const Maps& maps, const Params& p, cudaStream_t st) {
  if constexpr (KIND != kPlain)
    if (t.pair && gc::ceil_div(p.K, F8 ? 128 : 64) <= kResident)
      return launch_kernel<KIND, 256, A_MN, B_MN, F8, true, true>(maps, p, st);
  if (t.pair) return launch_kernel<KIND, 256, A_MN, B_MN, F8, true, false>(maps, p, st);
  auto single = [&](auto bn, auto lo) {
    return launch_kernel<KIND, decltype(bn)::value, A_MN, B_MN, F8, false, false, decltype(lo)::value>(maps, p, st);
  };
  auto width = [&](auto lo) {
    if constexpr (KIND != kGated)
      if (t.bn == 64) return single(std::integral_constant<int, 64>{}, lo);
    return single(std::integral_constant<int, 128>{}, lo);
  };
  if constexpr (KIND != kPlain)
    if (p.C) return width(std::true_type{});
  return width(std::false_type{});
}

// The maps of the operands.  A and B: matrices as they lie; K-major ones have K in their rows.
int operand_maps(Maps& maps, Params& p, const Matrix& A, bool a_mn, const Matrix& B, bool b_mn, int b_rows) {
  const int ke = 128 / A.size;  // K elements of a stage
  // Of a tile that M does not fill only the rows that exist are loaded: the TMA unit takes as long for a row of zeros, and
  // what the others hold stays in accumulators that nobody reads.
  const int rows = int(std::min<int64_t>(BM, (A.rows + 7) / 8 * 8));
  p.a_bytes = (a_mn ? BM : rows) * 128;
  int rc = a_mn ? make_map(&maps.a, A, 64, 64) : make_map(&maps.a, A, ke, rows);
  if (rc == GC_OK) rc = b_mn ? make_map(&maps.b, B, 64, 64) : make_map(&maps.b, B, ke, b_rows);
  return rc;
}

// C (M x N, bf16) = A B, fp32 sums; `halves`: A has that many times M rows, and M apart are added.
int plain(const Matrix& A, bool a_mn, const Matrix& B, bool b_mn, int64_t M, int64_t N, int64_t K, bf16* C, int64_t ldc,
          int64_t gap_from, int64_t gap, void* workspace, cudaStream_t st, int64_t halves = 1) {
  if (M == 0 || N == 0) return GC_OK;
  const int64_t out_rows = M;
  M *= halves;
  const Split s = plan_plain(M, N, K);
  Maps maps;
  Params p{};
  p.M = int(M); p.N = int(N); p.K = int(K);
  p.C = C; p.ldc = ldc;
  p.gap_from = gap ? int(gap_from) : int(N);
  p.gap = int(gap);
  p.c_cols = int(N - 2 * gap);  // [G | U] with the pads behind both
  p.splits = s.splits; p.kb_per_split = s.per;
  p.parts = s.splits > 1 || halves > 1;
  p.tma_store = gap == 0 && ldc % 8 == 0 && gc::aligned16(C);
  int rc = error_word(&p.word);
  if (rc == GC_OK) rc = operand_maps(maps, p, A, a_mn, B, b_mn, s.tile.pair ? s.tile.bn / 2 : s.tile.bn);
  const int64_t pitch = part_pitch(N);
  if (rc == GC_OK && p.parts) rc = make_map(&maps.out, Matrix{workspace, M, N, pitch, 4}, 16, 32, s.splits);
  else if (rc == GC_OK && p.tma_store) rc = make_map(&maps.out, Matrix{C, M, N, ldc, 2}, 32, 32);
  if (rc != GC_OK) return rc;
  if (a_mn) rc = launch_tile<kPlain, true, true, false>(s.tile, maps, p, st);
  else if (b_mn) rc = launch_tile<kPlain, false, true, false>(s.tile, maps, p, st);
  else rc = launch_tile<kPlain, false, false, false>(s.tile, maps, p, st);
  if (rc != GC_OK || !p.parts) return rc;
  const int64_t quads = out_rows * (pitch / 4);
  ffn_sum_kernel<<<unsigned(std::min<int64_t>(gc::ceil_div(quads, 256), gc::kNumSMs * 8)), 256, 0, st>>>(
      static_cast<const float*>(workspace), int(s.splits * halves), int(out_rows), int(pitch), C, ldc, p.c_cols, p.gap_from, p.gap);
  return gc::check_launch("ffn_sum_kernel");
}

// A matrix that TMA can read: itself, or a copy with a pitch of 16 bytes in the workspace, which moves on.
bool readable(const Matrix& m) { return gc::aligned16(m.p) && m.ld * m.size % 16 == 0; }
int64_t readable_ld(const Matrix& m) { return (m.cols * m.size + 15) / 16 * 16 / m.size; }
size_t copy_bytes(const Matrix& m) { return readable(m) ? 0 : align256(size_t(m.rows) * size_t(readable_ld(m)) * m.size); }
void add_copy(Copies& c, const Matrix& m, void* dst, int64_t ldd, int64_t width) {
  const int j = c.count++;
  c.job[j] = {m.p, dst, m.ld, ldd, m.rows, int(m.cols), int(width), m.size};
  const int64_t runs = gc::ceil_div(width * m.size / 4, Copies::kRun);
  const int64_t blocks = std::min<int64_t>(gc::ceil_div(m.rows * runs, 8), gc::kNumSMs * 8);
  c.first_block[0] = 0;
  c.first_block[j + 1] = c.first_block[j] + int(blocks);
}
void make_readable(Matrix& m, char*& ws, Copies& c) {
  if (readable(m)) return;
  const size_t bytes = copy_bytes(m);
  const int64_t ld = readable_ld(m);
  add_copy(c, m, ws, ld, ld);
  m.p = ws;
  m.ld = ld;
  ws += bytes;
}
// A copy of m on top of itself.
Matrix stacked(const Matrix& m, char*& ws, Copies& c) {
  const int64_t ld = readable_ld(m);
  const Matrix two{ws, 2 * m.rows, m.cols, ld, m.size};
  for (int i = 0; i < 2; ++i) add_copy(c, m, ws + i * m.rows * ld * m.size, ld, ld);
  ws += align256(size_t(two.rows) * size_t(ld) * m.size);
  return two;
}
// [Wg | Wu]: where H is not a multiple of 8, U's columns are moved to the next one, and the columns between are zeros -- as are
// then those of G, U, A and their gradients.
size_t gate_up_bytes(const Matrix& w, int64_t H) {
  return H % 8 == 0 ? copy_bytes(w) : align256(size_t(w.rows) * size_t(2 * up8(H)) * 2);
}
void make_gate_up(Matrix& w, int64_t H, char*& ws, Copies& c) {
  if (H % 8 == 0) return make_readable(w, ws, c);
  const int64_t hp = up8(H);
  uint16_t* to = reinterpret_cast<uint16_t*>(ws);
  add_copy(c, Matrix{w.p, w.rows, H, w.ld, 2}, to, 2 * hp, hp);
  add_copy(c, Matrix{static_cast<const uint16_t*>(w.p) + H, w.rows, H, w.ld, 2}, to + hp, 2 * hp, hp);
  ws += gate_up_bytes(w, H);
  w = Matrix{to, w.rows, 2 * hp, 2 * hp, 2};
}
int run_copies(const Copies& c, cudaStream_t st) {
  if (c.count == 0) return GC_OK;
  repitch_kernel<<<unsigned(c.first_block[c.count]), 256, 0, st>>>(c);
  return gc::check_launch("repitch_kernel");
}

Saved saved_at(void* p, int64_t M, int64_t H) {
  const int64_t hp = up8(H);
  char* c = static_cast<char*>(p);
  Saved s;
  s.hidden = reinterpret_cast<uint16_t*>(c);
  c += align256(size_t(stack(M) * M) * hp * 2);
  s.gate_up = reinterpret_cast<uint16_t*>(c);
  s.exps = reinterpret_cast<int8_t*>(c + align256(size_t(M) * hp * 4));
  return s;
}

// Whether a forward pass takes the form for few rows, of which its time depends as on the weights' bytes, while this file's
// hardly depends on the rows.  Measured, that form / this file's, us by the call:
//   bf16 in place      12 MB  10 / 21 at two rows, 12 / 21 at four, 31 / 21 at eight;   3 MB  19 / 19 at eight
//                      48 MB  21 / 31            , 25 / 31        , 70 / 31         ;  96 MB  33 / 35, 39 / 36, 94 / 36
//   odd widths, which  12 MB  16 / 33            , 19 / 33        , 47 / 33         ;   4 MB  20 / 29 at eight
//   this file copies   47 MB  55 / 66            , 58 / 66        , 176 / 66
//   e4m3               12 MB  10 / 19            , 10 / 19        , 19 / 19         ;   6 MB  14 / 18 at eight
//                      48 MB  14 / 27            , 19 / 27        , 39 / 27         ;  96 MB  24 / 32, 30 / 32, 62 / 32
//   e4m3 in rows that  3 MB  12 / 25 at one row, 17 / 25 at two, 14 / 25 at four, 21 / 25 at eight;   6 MB  41 / 28 at eight
//   16-byte accesses   12 MB  17 / 29           , 21 / 29       , 29 / 29       , 64 / 29
//   cannot take        24 MB  23 / 35           , 33 / 35       , 46 / 35       ;  47 MB  31 / 43, 40 / 44, 56 / 44
//                      96 MB  72 / 61           , 107 / 61      (with H and O odd too 24 MB 33 / 39, 45 / 39; 47 MB 43 / 54, 53 / 54)
// (weights of e4m3 counted at two bytes here.)
enum class Reading { kBf16InPlace, kOther, kOddE4m3 };
bool few_rows(int64_t M, int64_t D, int64_t H, int64_t O, Reading how) {
  const double weights = 2.0 * double(H) * (2.0 * double(D) + double(O)), mb = 1 << 20;
  if (how == Reading::kOddE4m3)
    return M <= kFewRows && weights <= (M == 1 ? 64 : M == 2 ? 16 : M <= 4 ? 6 : 3) * mb;
  return M <= 2 || (M <= 4 && weights <= 64 * mb) || (M <= kFewRows && weights <= (how == Reading::kBf16InPlace ? 3 : 6) * mb);
}

// Room for the product between the two launches: fp32, or [hi; lo], up to kStacked rows.
size_t hidden_bytes(int64_t M, int64_t hp) { return align256(size_t(stack(M) * M) * hp * 2); }
static_assert(kFewRows <= kStacked, "the form for few rows has room for fp32");

bool sizes_ok(int64_t M, int64_t D, int64_t H, int64_t O) {
  const int64_t top = (int64_t(1) << 31) - 512;  // coordinates and tile counts are 32-bit
  return M <= top && D <= top && 2 * up8(H) <= top && O <= top;
}

}  // namespace

extern "C" {

size_t gc_gated_ffn_saved_bytes(int64_t M, int64_t H) {
  if (M <= 0 || H <= 0) return 0;
  const int64_t hp = up8(H);
  return align256(size_t(stack(M) * M) * hp * 2) + align256(size_t(M) * hp * 4) + align256(2 * size_t(gc::ceil_div(hp, 32)) * size_t(M));
}

size_t gc_gated_ffn_workspace_bytes(int64_t M, int64_t D, int64_t H, int64_t O, int backward) {
  if (M <= 0 || D <= 0 || H <= 0 || O <= 0 || !sizes_ok(M, D, H, O)) return 0;
  const int64_t hp = up8(H);
  // copies of every operand, should none be readable in place
  const int64_t halves = stack(M), rows = halves * M;
  size_t b = align256(size_t(rows) * up8(D) * 2) + align256(size_t(D) * 2 * hp * 2) + align256(size_t(H) * up8(O) * 2);
  if (!backward) return b + hidden_bytes(M, hp) + plain_workspace(M, O, H, halves);
  b += align256(size_t(rows) * up8(O) * 2) + align256(size_t(rows) * 2 * hp * 2);  // dY, dG | dU
  return b + std::max({plain_workspace(M, D, 2 * hp, halves), plain_workspace(D, 2 * hp, rows), plain_workspace(H, O, rows)});
}

int gc_gated_ffn_forward_bf16(const uint16_t* X, int64_t ldx, const uint16_t* Win, int64_t ldwin, const uint16_t* Wout,
                              int64_t ldwout, int64_t M, int64_t D, int64_t H, int64_t O, int act, uint16_t* Y, int64_t ldy,
                              void* saved, void* workspace, size_t workspace_bytes, void* stream) {
  GC_REQUIRE(M >= 0 && D >= 0 && H >= 0 && O >= 0, "gc_gated_ffn_forward_bf16: negative size");
  GC_REQUIRE(act >= GC_ACT_SILU && act <= GC_ACT_RELU, "gc_gated_ffn_forward_bf16: unknown activation");
  GC_REQUIRE(ldx >= D && ldwin >= 2 * H && ldwout >= O && ldy >= O,
             "gc_gated_ffn_forward_bf16: leading dimension below the row length");
  if (!sizes_ok(M, D, H, O)) return gc::fail(GC_ERR_UNSUPPORTED, "gc_gated_ffn_forward_bf16: a size beyond 2^31");
  const cudaStream_t st = gc::as_stream(stream);
  if (M == 0 || O == 0) return GC_OK;
  GC_REQUIRE(Y, "gc_gated_ffn_forward_bf16: null pointer");
  const int64_t hp = up8(H);
  if (D == 0 || H == 0) {  // G = U = 0, or no hidden columns: Y = 0
    const cudaError_t e = cudaMemset2DAsync(Y, size_t(ldy) * 2, 0, size_t(O) * 2, size_t(M), st);
    return e == cudaSuccess ? GC_OK : gc::fail(GC_ERR_CUDA, "gc_gated_ffn_forward_bf16: %s", cudaGetErrorString(e));
  }
  GC_REQUIRE(X && Win && Wout, "gc_gated_ffn_forward_bf16: null pointer");
  GC_REQUIRE(gc::aligned16(saved), "gc_gated_ffn_forward_bf16: the saved buffer must be 16-byte aligned");
  if (!workspace || workspace_bytes < gc_gated_ffn_workspace_bytes(M, D, H, O, 0))
    return gc::fail(GC_ERR_WORKSPACE, "gc_gated_ffn_forward_bf16: workspace missing or smaller than its query says");
  GC_REQUIRE(gc::aligned16(workspace), "gc_gated_ffn_forward_bf16: workspace must be 16-byte aligned");
  char* ws = static_cast<char*>(workspace);
  Matrix x{X, M, D, ldx, 2}, win{Win, D, 2 * H, ldwin, 2}, wout{Wout, H, O, ldwout, 2};
  if (few_rows(M, D, H, O, readable(win) && H % 8 == 0 && readable(wout) ? Reading::kBf16InPlace : Reading::kOther)) {
    const Saved keep = saved ? saved_at(saved, M, H) : Saved{};
    const Rows r{X, Win, Wout, nullptr, nullptr, reinterpret_cast<float*>(ws), Y, ldx, ldwin, ldwout,
                 hp, ldy, int(M), int(D), int(H), int(O), act, keep};
    return forward_few_rows(r, false, st);
  }
  Copies copies{};
  make_readable(x, ws, copies);
  make_gate_up(win, H, ws, copies);
  make_readable(wout, ws, copies);
  int rc = run_copies(copies, st);
  if (rc != GC_OK) return rc;
  uint16_t* hidden = reinterpret_cast<uint16_t*>(ws);
  Saved keep{};
  if (saved) {
    keep = saved_at(saved, M, H);
    hidden = keep.hidden;
  } else {
    ws += hidden_bytes(M, hp);
  }
  const int64_t halves = stack(M);
  const Tile t = pick_tile(kGated, M, hp, 1);
  Maps maps;
  Params p{};
  p.M = int(M); p.N = int(hp); p.K = int(D);
  p.b_up = int(hp);
  p.act = act;
  p.exps = keep.exps;
  p.C = halves > 1 ? reinterpret_cast<bf16*>(hidden) + M * hp : nullptr;
  p.ldc = hp;
  rc = error_word(&p.word);
  if (rc == GC_OK) rc = operand_maps(maps, p, x, false, win, true, 0);
  if (rc == GC_OK) rc = make_map(&maps.out, Matrix{hidden, M, hp, hp, 2}, 32, 32);
  if (rc == GC_OK && saved) rc = make_map(&maps.out2, Matrix{keep.gate_up, M, hp, 2 * hp, 2}, 32, 32);
  if (rc == GC_OK && saved) rc = make_map(&maps.out3, Matrix{keep.gate_up + hp, M, hp, 2 * hp, 2}, 32, 32);
  if (rc == GC_OK) rc = launch_tile<kGated, false, true, false>(t, maps, p, st);
  if (rc != GC_OK) return rc;
  return plain(Matrix{hidden, halves * M, H, hp, 2}, false, wout, true, M, O, H, reinterpret_cast<bf16*>(Y), ldy, 0, 0, ws, st, halves);
}

int gc_gated_ffn_backward_bf16(const uint16_t* dY, int64_t lddy, const uint16_t* X, int64_t ldx, const uint16_t* Win,
                               int64_t ldwin, const uint16_t* Wout, int64_t ldwout, const void* saved,
                               int64_t M, int64_t D, int64_t H, int64_t O, int act, uint16_t* dX,
                               int64_t lddx, uint16_t* dWin, int64_t lddwin, uint16_t* dWout, int64_t lddwout,
                               void* workspace, size_t workspace_bytes, void* stream) {
  GC_REQUIRE(M >= 0 && D >= 0 && H >= 0 && O >= 0, "gc_gated_ffn_backward_bf16: negative size");
  GC_REQUIRE(act >= GC_ACT_SILU && act <= GC_ACT_RELU, "gc_gated_ffn_backward_bf16: unknown activation");
  GC_REQUIRE(lddy >= O && ldx >= D && ldwin >= 2 * H && ldwout >= O && (!dX || lddx >= D) && (!dWin || lddwin >= 2 * H) &&
                 (!dWout || lddwout >= O),
             "gc_gated_ffn_backward_bf16: leading dimension below the row length");
  if (!sizes_ok(M, D, H, O)) return gc::fail(GC_ERR_UNSUPPORTED, "gc_gated_ffn_backward_bf16: a size beyond 2^31");
  const cudaStream_t st = gc::as_stream(stream);
  const int64_t hp = up8(H);
  if (M == 0 || D == 0 || H == 0 || O == 0) {  // sums of nothing
    cudaError_t e = cudaSuccess;
    auto zero = [&](uint16_t* p, int64_t ld, int64_t rows, int64_t cols) {
      if (p && rows && cols && e == cudaSuccess) e = cudaMemset2DAsync(p, size_t(ld) * 2, 0, size_t(cols) * 2, size_t(rows), st);
    };
    zero(dX, lddx, M, D);
    zero(dWin, lddwin, D, 2 * H);
    zero(dWout, lddwout, H, O);
    return e == cudaSuccess ? GC_OK : gc::fail(GC_ERR_CUDA, "gc_gated_ffn_backward_bf16: %s", cudaGetErrorString(e));
  }
  if (!dX && !dWin && !dWout) return GC_OK;
  GC_REQUIRE(dY && X && Win && Wout && saved, "gc_gated_ffn_backward_bf16: null pointer");
  GC_REQUIRE(gc::aligned16(saved), "gc_gated_ffn_backward_bf16: the saved buffer must be 16-byte aligned");
  if (!workspace || workspace_bytes < gc_gated_ffn_workspace_bytes(M, D, H, O, 1))
    return gc::fail(GC_ERR_WORKSPACE, "gc_gated_ffn_backward_bf16: workspace missing or smaller than its query says");
  GC_REQUIRE(gc::aligned16(workspace), "gc_gated_ffn_backward_bf16: workspace must be 16-byte aligned");
  char* ws = static_cast<char*>(workspace);
  Matrix dy{dY, M, O, lddy, 2}, x{X, M, D, ldx, 2}, win{Win, D, 2 * H, ldwin, 2}, wout{Wout, H, O, ldwout, 2};
  Copies copies{};
  const int64_t halves = stack(M), rows = halves * M;
  Matrix dy_rows = dy;  // as the weight gradients take it and x
  if (halves > 1) {
    dy_rows = stacked(dy, ws, copies);
    dy = Matrix{dy_rows.p, M, O, dy_rows.ld, 2};
    if (dWin) x = stacked(x, ws, copies);
  } else {
    make_readable(dy, ws, copies);
    dy_rows = dy;
    if (dWin) make_readable(x, ws, copies);
  }
  if (dX) make_gate_up(win, H, ws, copies);
  if (dX || dWin) make_readable(wout, ws, copies);
  int rc = run_copies(copies, st);
  if (rc != GC_OK) return rc;
  const Saved kept = saved_at(const_cast<void*>(saved), M, H);
  const Matrix dgu{ws, rows, 2 * hp, 2 * hp, 2};
  if (dX || dWin) {
    uint16_t* out = reinterpret_cast<uint16_t*>(ws);
    ws += align256(size_t(rows) * 2 * hp * 2);
    const Tile t = pick_tile(kGatedBack, M, hp, 1);
    Maps maps;
    Params p{};
    p.M = int(M); p.N = int(hp); p.K = int(O);
    p.act = act;
    p.exps = kept.exps;
    p.C = halves > 1 ? reinterpret_cast<bf16*>(out) + M * 2 * hp : nullptr;
    p.ldc = 2 * hp;
    rc = error_word(&p.word);
    if (rc == GC_OK) rc = operand_maps(maps, p, dy, false, wout, false, t.pair ? t.bn / 2 : t.bn);
    if (rc == GC_OK) rc = make_map(&maps.in1, Matrix{kept.gate_up, M, hp, 2 * hp, 2}, 32, 32);
    if (rc == GC_OK) rc = make_map(&maps.in2, Matrix{kept.gate_up + hp, M, hp, 2 * hp, 2}, 32, 32);
    if (rc == GC_OK) rc = make_map(&maps.out, Matrix{out, M, hp, 2 * hp, 2}, 32, 32);
    if (rc == GC_OK) rc = make_map(&maps.out2, Matrix{out + hp, M, hp, 2 * hp, 2}, 32, 32);
    if (rc == GC_OK) rc = launch_tile<kGatedBack, false, false, false>(t, maps, p, st);
    if (rc != GC_OK) return rc;
  }
  if (dX) rc = plain(dgu, false, win, false, M, D, 2 * hp, reinterpret_cast<bf16*>(dX), lddx, 0, 0, ws, st, halves);
  if (rc == GC_OK && dWin)
    rc = plain(x, true, dgu, true, D, 2 * hp, rows, reinterpret_cast<bf16*>(dWin), lddwin, H, hp - H, ws, st);
  if (rc == GC_OK && dWout)
    rc = plain(Matrix{kept.hidden, rows, H, hp, 2}, true, dy_rows, true, H, O, rows, reinterpret_cast<bf16*>(dWout), lddwout, 0, 0, ws, st);
  return rc;
}

size_t gc_gated_ffn_e4m3_workspace_bytes(int64_t M, int64_t D, int64_t H, int64_t O) {
  if (M <= 0 || D <= 0 || H <= 0 || O <= 0 || !sizes_ok(M, D, H, O)) return 0;
  const int64_t d16 = (D + 15) / 16 * 16;
  return align256(size_t(M) * d16) + align256(size_t(2 * H) * d16) + align256(size_t(H) * up8(O) * 2) +
         hidden_bytes(M, up8(H)) + plain_workspace(M, O, H, stack(M));
}

int gc_gated_ffn_forward_e4m3(const uint8_t* X8, int64_t ldx, const float* x_scale, const uint8_t* W8, int64_t ldw,
                              const float* w_scale, const uint16_t* Wout, int64_t ldwout, int64_t M, int64_t D, int64_t H,
                              int64_t O, int act, uint16_t* Y, int64_t ldy, void* workspace, size_t workspace_bytes,
                              void* stream) {
  GC_REQUIRE(M >= 0 && D >= 0 && H >= 0 && O >= 0, "gc_gated_ffn_forward_e4m3: negative size");
  GC_REQUIRE(act >= GC_ACT_SILU && act <= GC_ACT_RELU, "gc_gated_ffn_forward_e4m3: unknown activation");
  GC_REQUIRE(ldx >= D && ldw >= D && ldwout >= O && ldy >= O,
             "gc_gated_ffn_forward_e4m3: leading dimension below the row length");
  if (!sizes_ok(M, D, H, O)) return gc::fail(GC_ERR_UNSUPPORTED, "gc_gated_ffn_forward_e4m3: a size beyond 2^31");
  const cudaStream_t st = gc::as_stream(stream);
  if (M == 0 || O == 0) return GC_OK;
  GC_REQUIRE(Y, "gc_gated_ffn_forward_e4m3: null pointer");
  if (D == 0 || H == 0) {
    const cudaError_t e = cudaMemset2DAsync(Y, size_t(ldy) * 2, 0, size_t(O) * 2, size_t(M), st);
    return e == cudaSuccess ? GC_OK : gc::fail(GC_ERR_CUDA, "gc_gated_ffn_forward_e4m3: %s", cudaGetErrorString(e));
  }
  GC_REQUIRE(X8 && x_scale && W8 && w_scale && Wout, "gc_gated_ffn_forward_e4m3: null pointer");
  if (!workspace || workspace_bytes < gc_gated_ffn_e4m3_workspace_bytes(M, D, H, O))
    return gc::fail(GC_ERR_WORKSPACE, "gc_gated_ffn_forward_e4m3: workspace missing or smaller than its query says");
  GC_REQUIRE(gc::aligned16(workspace), "gc_gated_ffn_forward_e4m3: workspace must be 16-byte aligned");
  char* ws = static_cast<char*>(workspace);
  Matrix x{X8, M, D, ldx, 1}, w{W8, 2 * H, D, ldw, 1}, wout{Wout, H, O, ldwout, 2};
  if (few_rows(M, D, H, O, D % 16 == 0 && readable(x) && readable(w) ? Reading::kOther : Reading::kOddE4m3)) {
    const Rows r{X8, W8, Wout, x_scale, w_scale, reinterpret_cast<float*>(ws), Y, ldx, ldw, ldwout, up8(H), ldy, int(M), int(D),
                 int(H), int(O), act, Saved{}};
    return forward_few_rows(r, true, st);
  }
  Copies copies{};
  make_readable(x, ws, copies);
  make_readable(w, ws, copies);
  make_readable(wout, ws, copies);
  int rc = run_copies(copies, st);
  if (rc != GC_OK) return rc;
  const int64_t hp = up8(H);
  uint16_t* hidden = reinterpret_cast<uint16_t*>(ws);
  ws += hidden_bytes(M, hp);
  const int64_t halves = stack(M);
  const Tile t = pick_tile(kGated, M, H, 1);
  Maps maps;
  Params p{};
  p.M = int(M); p.N = int(H); p.K = int(D);
  p.b_up = int(H);  // rows of W8: no alignment to keep
  p.act = act;
  p.sa = x_scale;
  p.sb = w_scale;
  p.C = halves > 1 ? reinterpret_cast<bf16*>(hidden) + M * hp : nullptr;
  p.ldc = hp;
  rc = error_word(&p.word);
  if (rc == GC_OK) rc = operand_maps(maps, p, x, false, w, false, t.bn / 2);
  if (rc == GC_OK) rc = make_map(&maps.out, Matrix{hidden, M, H, hp, 2}, 32, 32);
  if (rc == GC_OK) rc = launch_tile<kGated, false, false, true>(t, maps, p, st);
  if (rc != GC_OK) return rc;
  return plain(Matrix{hidden, halves * M, H, hp, 2}, false, wout, true, M, O, H, reinterpret_cast<bf16*>(Y), ldy, 0, 0, ws, st, halves);
}

}  // extern "C"
