// Products of rows that are sorted by group with a weight per group, on the 5th-generation tensor cores, bf16.
//
//   forward    Y[r] = X[r] W[g]              for rows r of group g, offsets[g] <= r < offsets[g + 1]
//   backward   dX[r] = dY[r] W[g]^T,  dW[g] = X_g^T dY_g
//
// Groups are as large as they are: the offsets lie on the device, and nothing here asks the host for them.  One persistent kernel, in
// which one warp of a CTA walks the groups, 32 at a time (a scan over their tiles), as far as the CTA's next tile is, and hands tiles
// to the other warps through a ring in shared memory.  (With every warp walking for itself the MMA issuer spent 3300 clocks on it
// where neighbouring tiles lie in different groups: half of the time at K = 256.)  Tiles begin at a group's first row, wherever that is.  A tile's rows beyond the group's end are multiplied like the others -- rows of a
// product do not mix -- and not stored: blocks of 32 rows that are the group's own leave by TMA, the one that it ends in row by
// row.  In dW the rows are what is summed over, and none of the next group's may come in (zeros would not keep out its
// infinities): a first launch copies what a group has beyond whole blocks of 64 rows into blocks filled up with zeros, from
// which the last block of a sum is loaded.
//
// Operands are read where they lie, K-major or MN-major; sums are fp32 in TMEM, rounded to bf16 once.  dW of many rows is cut along
// them into parts of `part` rows, whose fp32 sums a last launch adds in their order: for parallelism where a weight has few tiles, and
// because a chain of additions in the tensor core truncates (16,384 rows: 1e-4 relative, below the result's rounding).
//
// CTA = 20 warps, as in the gated block's kernel: TMA producers of A and of B, MMA issuer, the warp that deals tiles, 16 epilogue warps
// on the 32 x 32 blocks of a tile in turn; two accumulators; CTAs in pairs on 256 x 256 where there are rows for it.  Waits are bounded
// as there.
//
// Rows of no group (before the first offset, behind the last) get zeros.  Offsets that are no offsets (outside the rows, or
// decreasing) are read as the nearest that are.
#include "tiles.cuh"

namespace {

using namespace gc::tiles;
using bf16 = __nv_bfloat16;

constexpr int BM = 128, KE = 64;  // rows of A per CTA, K elements per k-block
constexpr int kEpiWarps = 16, kEpiGroups = kEpiWarps / 4;
constexpr int kThreads = 128 + 32 * kEpiWarps;
constexpr int kTileBytes = 32 * 64;  // what an epilogue warp stores at once
constexpr uint32_t kAll = 0xFFFFFFFFu;

enum Mode { kForward, kBack, kWeights };  // Y; dX; dW

template <int BN, bool PAIR>
struct Cfg {
  static constexpr int BNC = PAIR ? BN / 2 : BN;  // rows of B that a CTA holds
  static constexpr int kABytes = BM * 128, kBBytes = BNC * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStaging = kEpiWarps * 2 * kTileBytes;
  static constexpr int kStages = std::min(8, (227 * 1024 - 1024 - 512 - kStaging) / kStageBytes);
  static constexpr int kSmemBytes = kStages * kStageBytes + kStaging + 512 /*barriers*/ + 1024 /*alignment*/;
  static constexpr uint32_t kTmemCols = 2 * BN;
  static_assert(kSmemBytes <= 227 * 1024 && kStages >= 2 && kTmemCols <= 512, "shared memory and TMEM");
};

struct Params {
  const int32_t* offsets;
  int groups, rows;
  int K;        // forward, backward: what is summed over (inputs; outputs)
  int m, n;     // dW: the weight's rows;  columns of the product
  int a_bytes;  // of a k-block of A that are loaded
  int part;     // dW: rows of a part, a multiple of 64
  bf16* C;      // Y, dX, or dW
  int64_t ldc;
  int tma_store;
  float* parts;  // dW: [part][m][n rounded up to 4]
  int* word;     // the device's error word
};
struct Maps {
  CUtensorMap a, b;            // forward, backward: rows, weights (3-D); dW: rows, rows
  CUtensorMap a_tail, b_tail;  // dW: the blocks filled up with zeros, 64 rows per group
  CUtensorMap out, out_parts;
};

// The group that holds an item, found by a whole warp.  Items are tiles (dW: parts of tiles), numbered group after group.
struct Group {
  int g, start, end;  // its rows
  int first, count;   // its items
};
__device__ __forceinline__ int clamped(const Params& p, int i) { return min(max(__ldg(p.offsets + i), 0), p.rows); }
template <class Count>
__device__ __forceinline__ bool seek(const Params& p, Group& x, int item, Count&& count) {
  const int lane = threadIdx.x % 32;
  while (true) {
    if (item < x.first + x.count) return true;
    const int base = x.g + 1, from = x.first + x.count;
    if (base >= p.groups) return false;
    int end = base + lane < p.groups ? clamped(p, base + lane + 1) : 0;
    end = max(end, x.end);
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int t = __shfl_up_sync(kAll, end, d);
      if (lane >= d) end = max(end, t);
    }
    int start = __shfl_up_sync(kAll, end, 1);
    if (lane == 0) start = x.end;
    const int mine = base + lane < p.groups ? count(end - start) : 0;
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int t = __shfl_up_sync(kAll, sum, d);
      if (lane >= d) sum += t;
    }
    const uint32_t hit = __ballot_sync(kAll, item < from + sum);
    const int at = hit ? __ffs(hit) - 1 : min(31, p.groups - 1 - base);
    x.g = base + at;
    x.start = __shfl_sync(kAll, start, at);
    x.end = __shfl_sync(kAll, end, at);
    x.first = from + __shfl_sync(kAll, sum - mine, at);
    x.count = __shfl_sync(kAll, mine, at);
  }
}
__device__ __forceinline__ Group before_all(const Params& p) {
  const int first = clamped(p, 0);
  return {-1, first, first, 0, 0};
}

// A tile as one warp deals it to the others.
struct __align__(16) Tile {
  int row, col;        // of the product, where the CTA's half begins
  int row_end, group;  // the group's last row, or the weight's; of the last tile, which is none, the last group's
  int from, blocks;    // dW: first row that is summed over; k-blocks, below zero for the last
  int over, part;      // dW: rows of the last k-block, where that is not whole; number of the part, below zero where it is the only one
};
constexpr int kDealt = 4;

template <int MODE, int BN, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
grouped_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  using C_ = Cfg<BN, PAIR>;
  constexpr int S = C_::kStages, BNC = C_::BNC;
  constexpr int TM = PAIR ? 2 * BM : BM;
  constexpr bool A_MN = MODE == kWeights, B_MN = MODE != kBack;
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  const int unit = PAIR ? int(blockIdx.x / 2) : int(blockIdx.x), units = PAIR ? int(gridDim.x / 2) : int(gridDim.x);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  auto sA = [&](int s) { return base + s * C_::kStageBytes; };
  auto sB = [&](int s) { return sA(s) + C_::kABytes; };
  const uint32_t staging = base + S * C_::kStageBytes;
  const uint32_t bars = staging + C_::kStaging;
  auto bar_full = [&](int s) { return bars + 8 * s; };
  auto bar_empty = [&](int s) { return bars + 8 * (S + s); };
  auto bar_tfull = [&](int b) { return bars + 8 * (2 * S + b); };
  auto bar_tempty = [&](int b) { return bars + 8 * (2 * S + 2 + b); };
  auto bar_dealt = [&](int i) { return bars + 8 * (2 * S + 4 + i); };
  auto bar_taken = [&](int i) { return bars + 8 * (2 * S + 4 + kDealt + i); };
  static_assert(8 * (2 * S + 4 + 2 * kDealt) <= 512, "room for the barriers");
  __shared__ Tile dealt[kDealt];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int tiles_n = (p.n + BN - 1) / BN;
  const int weight_tiles = (p.m + TM - 1) / TM * tiles_n;  // dW
  // This CTA's (or pair's) items are every units-th.  Of a part: groups of 8 rows of tiles, so that tiles that run at one time
  // are a square of the product.
  Group in = before_all(p);
  int item = unit;
  auto find = [&](Tile& x) {  // by a whole warp
    constexpr int kSquare = 8;
    const bool there = seek(p, in, item, [&](int rows) {
      if (MODE == kWeights) return max(1, (rows + p.part - 1) / p.part) * weight_tiles;
      return (rows + TM - 1) / TM * tiles_n;
    });
    x.group = in.g;
    x.row_end = MODE == kWeights && there ? p.m : in.end;
    x.blocks = -1;
    if (!there) return false;
    int i = item - in.first;
    const int tiles_m = MODE == kWeights ? (p.m + TM - 1) / TM : (in.end - in.start + TM - 1) / TM;
    if (MODE == kWeights) {
      const int part = i / weight_tiles;
      i -= part * weight_tiles;
      x.from = in.start + part * p.part;
      const int rows = min(p.part, in.end - x.from);
      x.blocks = (rows + KE - 1) / KE;
      x.over = rows % KE;
      x.part = in.count > weight_tiles ? in.first / weight_tiles + part : -1;
    } else {
      x.blocks = (p.K + KE - 1) / KE;
    }
    const int g = i / (kSquare * tiles_n), r = i - g * (kSquare * tiles_n), high = min(kSquare, tiles_m - g * kSquare);
    const int n = r / high;
    x.row = (MODE == kWeights ? 0 : in.start) + (g * kSquare + r - n * high) * TM + int(rank) * BM;
    x.col = n * BN;
    item += units;
    return true;
  };
  Tile ahead;
  if (warp == 2) find(ahead);  // while the barriers are made and TMEM is allocated

  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int s = 0; s < S; ++s) {
      mbar_init(bar_full(s), 2);  // A's producer, and B's
      mbar_init(bar_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_tfull(b), 1);
      mbar_init(bar_tempty(b), kEpiWarps * (PAIR ? 2 : 1));
    }
    for (int i = 0; i < kDealt; ++i) {
      mbar_init(bar_dealt(i), 1);
      mbar_init(bar_taken(i), 2 + kEpiWarps + (rank == 0));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (PAIR) {
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers exist before either is signalled
  }
  if (warp == 1) tmem_alloc<PAIR>(smem_u32(&tmem_base_s), C_::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_s;
  volatile int* abort_p = &abort_s;
  // The t-th tile, for one lane or a whole warp; false when there is none.
  auto take = [&](int t, Tile& x, bool all) {
    const int i = t % kDealt;
    bool ok = wait(bar_dealt(i), (t / kDealt) & 1u, abort_p);
    if (all) ok = __all_sync(kAll, ok);
    if (!ok) return false;
    x = dealt[i];
    if (all) __syncwarp();
    if (!all || lane == 0) mbar_arrive(bar_taken(i));
    return x.blocks >= 0;
  };

  if (warp == 2) {
    // ------------------------------------------------------------ deals the tiles
    for (int t = 0;; ++t) {
      const int i = t % kDealt;
      if (!__all_sync(kAll, wait(bar_taken(i), ((t / kDealt) & 1u) ^ 1u, abort_p))) break;
      if (lane == 0) {
        dealt[i] = ahead;
        mbar_arrive(bar_dealt(i));
      }
      if (ahead.blocks < 0) break;
      find(ahead);
    }
  } else if ((warp == 0 || warp == 3) && lane == 0) {
    // ------------------------------------------------------------ TMA producers: A, B
    const bool is_a = warp == 0;
    auto expect = [&](uint32_t bar, uint32_t bytes) {  // a pair's copies are all counted at the leader
      if (!PAIR) mbar_expect_tx(bar, bytes);
      else if (rank == 0) mbar_expect_tx(bar, 2 * bytes);
    };
    auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
      if (PAIR) tma_load_2d_leader(dst, map, x, y, bar);
      else tma_load_2d(dst, map, x, y, bar);
    };
    auto load_weight = [&](uint32_t dst, int x, int y, int g, uint32_t bar) {
      if (PAIR) tma_load_3d_leader(dst, &maps.b, x, y, g, bar);
      else tma_load_3d(dst, &maps.b, x, y, g, bar);
    };
    uint32_t s = 0, phase = 0, issued = 0;
    Tile x;
    bool ok = true;
    for (int t = 0; ok && take(t, x, false); ++t) {
      const int n0 = x.col + int(rank) * BNC;
      for (int kb = 0; kb < x.blocks; ++kb) {
        if (!wait(bar_empty(s), phase ^ 1u, abort_p)) { ok = false; break; }
        const uint32_t bar = bar_full(s);
        const bool tail = MODE == kWeights && x.over && kb == x.blocks - 1;
        const int row = tail ? x.group * KE : x.from + kb * KE;  // dW
        if (is_a) {
          expect(bar, p.a_bytes);
          if (A_MN) {
#pragma unroll
            for (int c = 0; c < BM / 64; ++c) load(sA(s) + c * (64 * 128), tail ? &maps.a_tail : &maps.a, x.row + c * 64, row, bar);
          } else {
            load(sA(s), &maps.a, kb * KE, x.row, bar);
          }
        } else {
          expect(bar, C_::kBBytes);
          if (MODE == kBack) {
            load_weight(sB(s), kb * KE, n0, x.group, bar);
          } else {
#pragma unroll
            for (int c = 0; c < BNC / 64; ++c) {
              if (MODE == kForward) load_weight(sB(s) + c * (64 * 128), n0 + c * 64, kb * KE, x.group, bar);
              else load(sB(s) + c * (64 * 128), tail ? &maps.b_tail : &maps.b, n0 + c * 64, row, bar);
            }
          }
        }
        ++issued;
        if (++s == uint32_t(S)) s = 0, phase ^= 1u;
      }
    }
    if (!PAIR || rank == 0)  // every copy issued must have landed before the CTA may exit
      for (uint32_t j = 0; j < issued && j < uint32_t(S); ++j) {
        if (s == 0) phase ^= 1u;
        s = s == 0 ? S - 1 : s - 1;
        drain(bar_full(s), phase);
      }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc = make_idesc(TM, BN, A_MN, B_MN, false);
    constexpr uint32_t kAStep = A_MN ? 16 * 128 : 32, kBStep = B_MN ? 16 * 128 : 32;  // bytes per MMA
    const uint64_t da0 = operand_desc(sA(0), A_MN), db0 = operand_desc(sB(0), B_MN);
    uint32_t s = 0, phase = 0;
    Tile x;
    bool ok = true;
    for (int t = 0; ok && take(t, x, false); ++t) {
      const int b = t & 1;
      if (!wait(bar_tempty(b), ((t >> 1) & 1u) ^ 1u, abort_p)) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + uint32_t(b * BN);
      for (int kb = 0; kb < x.blocks; ++kb) {
        if (!wait(bar_full(s), phase, abort_p)) { ok = false; break; }
        tc_fence_after();
        const uint64_t da = da0 + s * (C_::kStageBytes >> 4), db = db0 + s * (C_::kStageBytes >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma<PAIR, false>(d_tmem, da + ((k * kAStep) >> 4), db + ((k * kBStep) >> 4), idesc, (kb > 0 || k > 0) ? 1u : 0u);
        umma_commit<PAIR>(bar_empty(s));  // frees the stage once these MMAs have read it
        if (++s == uint32_t(S)) s = 0, phase ^= 1u;
      }
      if (ok) umma_commit<PAIR>(bar_tfull(b));
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int q = warp % 4;  // TMEM lane quarter
    const int grp = (warp - 4) / 4;  // which of the 32-column chunks: grp, grp + 4, ..
    const uint32_t tiles = staging + (warp - 4) * (2 * kTileBytes);
    const uint32_t lane_at = row_at(tiles, lane);
    const int pitch = (p.n + 3) / 4 * 4;  // of a part's rows
    uint32_t buf = 0;
    // The next of the warp's tiles, once the store that read it last has done so.
    auto acquire = [&]() {
      if (lane == 0) store_wait_read<1>();
      __syncwarp();
      buf ^= kTileBytes;
      return buf;
    };
    Tile x;
    x.blocks = 0;
    for (int t = 0; take(t, x, true); ++t) {
      const int b = t & 1;
      if (!__all_sync(kAll, wait(bar_tfull(b), (t >> 1) & 1u, abort_p))) break;
      tc_fence_after();
      bool held = true;
      auto release = [&]() {  // the accumulator goes back as soon as the warp's last chunk is in registers
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_leader(bar_tempty(b));
          else mbar_arrive(bar_tempty(b));
        }
        held = false;
      };
      const int row0 = x.row + q * 32, rows = min(32, x.row_end - row0);  // of the product
      const uint32_t taddr = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(b * BN);
      for (int c = grp; c < BN / 32 && rows > 0; c += kEpiGroups) {
        const int col = x.col + c * 32;
        if (col >= p.n) break;
        uint32_t acc[32];
        tmem_ld32(taddr + uint32_t(c * 32), acc);
        tmem_ld_wait();
        if (c + kEpiGroups >= BN / 32 || col + kEpiGroups * 32 >= p.n) release();
        if (MODE == kWeights && x.blocks == 0) {  // a group without rows
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[i] = 0;
        }
        if (MODE == kWeights && x.part >= 0) {
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
              if (col + half * 16 < pitch) tma_store_3d(&maps.out_parts, tiles + bo, col + half * 16, row0, x.part);
              store_commit();
            }
          }
        } else {
          const uint32_t bo = acquire();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = pack2(__uint_as_float(acc[j * 8 + 2 * e]), __uint_as_float(acc[j * 8 + 2 * e + 1]));
            store_unit(lane_at + bo, j, w[0], w[1], w[2], w[3]);
          }
          if (p.tma_store && (MODE == kWeights || rows == 32)) {  // the map ends where the matrix, or a group's weight, does
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (MODE == kWeights) tma_store_3d(&maps.out, tiles + bo, col, row0, x.group);
              else tma_store_2d(&maps.out, tiles + bo, col, row0);
              store_commit();
            }
          } else {
            // rows of an odd pitch, or the last of a group: a row at a time, a column per lane
            __syncwarp();
            bf16* to = p.C + (MODE == kWeights ? int64_t(x.group) * p.m + row0 : int64_t(row0)) * p.ldc + col + lane;
            if (col + lane < p.n)
              for (int r = 0; r < rows; ++r) to[r * p.ldc] = __ushort_as_bfloat16(load_column(tiles + bo, r, lane));
            if (lane == 0) store_commit();  // nothing: the tiles' turns are counted in groups of stores
            __syncwarp();  // before the tile is filled again
          }
        }
      }
      if (held) release();
    }
    if (MODE != kWeights && x.blocks < 0) {  // all tiles are done; rows of no group
      const int head = clamped(p, 0), spare = p.rows - x.row_end;
      const int64_t total = int64_t(head + spare) * p.n, step = int64_t(gridDim.x) * kEpiWarps * 32;
      for (int64_t i = (int64_t(blockIdx.x) * kEpiWarps + warp - 4) * 32 + lane; i < total; i += step) {
        const int64_t r = i / p.n;
        p.C[(r < head ? r : x.row_end + r - head) * p.ldc + (i - r * p.n)] = __ushort_as_bfloat16(0);
      }
    }
    if (lane == 0) store_wait_all();  // shared memory is read until then
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // the peer's MMAs read this CTA's shared memory and write its TMEM until here
  tc_fence_after();
  if (warp == 1) tmem_dealloc<PAIR>(tmem_base, C_::kTmemCols);
  if (threadIdx.x == 0 && abort_s) atomicExch(p.word, 1);
}

// A group's rows, and for dW the number of parts before it, found by a whole CTA of 256 threads.
struct Bounds {
  int start, end, parts_before;
};
__device__ __forceinline__ Bounds bounds_of(const Params& p, int g) {
  __shared__ Bounds found;
  if (threadIdx.x < 32) {
    Group x = before_all(p);
    // an item is a part here, and the walk goes on to group g: it ends at the first item of those behind
    int before = 0, end = x.end, start = x.end;
    const int lane = threadIdx.x;
    for (int base = 0; base <= g; base += 32) {
      const int i = base + lane;
      int e = i <= g ? clamped(p, i + 1) : 0;
      e = max(e, end);
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int t = __shfl_up_sync(kAll, e, d);
        if (lane >= d) e = max(e, t);
      }
      int s = __shfl_up_sync(kAll, e, 1);
      if (lane == 0) s = end;
      int n = i < g ? max(1, (e - s + p.part - 1) / p.part) : 0;
#pragma unroll
      for (int d = 16; d > 0; d /= 2) n += __shfl_xor_sync(kAll, n, d);
      before += n;
      const int last = min(31, g - base);
      start = __shfl_sync(kAll, s, last);
      end = __shfl_sync(kAll, e, last);
    }
    if (lane == 0) found = {start, end, before};
  }
  __syncthreads();
  return found;
}

// The rows of group blockIdx.x beyond its whole blocks of 64, of X and of dY, with zeros up to 64; 16 bytes per thread.
__global__ void __launch_bounds__(256)
grouped_tail_kernel(const __grid_constant__ Params p, const uint16_t* __restrict__ x, int64_t ldx, const uint16_t* __restrict__ dy,
                    int64_t lddy, uint4* __restrict__ x_tail, uint4* __restrict__ dy_tail) {
  const Bounds b = bounds_of(p, blockIdx.x);
  const int over = (b.end - b.start) % KE;
  if (over == 0) return;
  const int x_width = (p.m + 7) / 8, dy_width = (p.n + 7) / 8, width = x_width + dy_width;
  for (int64_t i = blockIdx.y * 256 + threadIdx.x; i < int64_t(KE) * width; i += gridDim.y * 256) {
    const int r = int(i / width);
    int c = int(i - int64_t(r) * width);
    const bool of_x = c < x_width;
    if (!of_x) c -= x_width;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < over) {
      const uint16_t* row = (of_x ? x + int64_t(b.end - over + r) * ldx : dy + int64_t(b.end - over + r) * lddy) + c * 8;
      const int columns = (of_x ? p.m : p.n) - c * 8;
      if (columns >= 8) {
        v = __ldg(reinterpret_cast<const uint4*>(row));
      } else {
        uint32_t* w = &v.x;
        for (int e = 0; e < columns; ++e) w[e / 2] |= uint32_t(row[e]) << (e % 2 * 16);
      }
    }
    (of_x ? x_tail : dy_tail)[(int64_t(blockIdx.x) * KE + r) * (of_x ? x_width : dy_width) + c] = v;
  }
}

// dW of the groups that have more than one part: the sum of the parts in their order.
__global__ void __launch_bounds__(256)
grouped_sum_kernel(const __grid_constant__ Params p) {
  const Bounds b = bounds_of(p, blockIdx.x);
  const int parts = max(1, (b.end - b.start + p.part - 1) / p.part);
  if (parts == 1) return;
  const int pitch = (p.n + 3) / 4 * 4;
  const int64_t quads = int64_t(p.m) * (pitch / 4), size = int64_t(p.m) * pitch;
  const bool vec = p.n % 4 == 0 && p.ldc % 4 == 0 && reinterpret_cast<uintptr_t>(p.C) % 8 == 0;
  const float* from = p.parts + b.parts_before * size;
  for (int64_t i = int64_t(blockIdx.y) * 256 + threadIdx.x; i < quads; i += int64_t(gridDim.y) * 256) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int z = 0; z < parts; ++z) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(from + z * size) + i);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const int64_t m = i / (pitch / 4);
    const int n = int(i - m * (pitch / 4)) * 4;
    bf16* to = p.C + (int64_t(blockIdx.x) * p.m + m) * p.ldc + n;
    if (vec) {
      *reinterpret_cast<uint2*>(to) = make_uint2(pack2(s.x, s.y), pack2(s.z, s.w));
    } else {
      const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.n) to[e] = __float2bfloat16_rn(v[e]);
    }
  }
}

// ------------------------------------------------------------------ host
struct Shape {
  int bn;
  bool pair;
};
// Rows times weights: pairs on 256 x 256, 128 columns or 64, whichever takes least of (rounds of tiles over the SMs) x (rows of A and of B
// that a CTA loads for a k-block), with groups taken to be equally large.  4096 rows of 8 groups, 1024 -> 1024: 64 pairs' tiles in one round 13.6
// us, 64 columns in four 26; 600 of 2, 4096 -> 4096: 29 and 65; a row to each of 8, 4096 -> 4096: 128 columns in two rounds 50, 64 in four 84.
Shape shape_of_rows(int64_t M, int64_t n, int64_t G) {
  const int64_t with_rows = std::min(G, M), rows = gc::ceil_div(M, with_rows), a = std::min<int64_t>(BM, M);
  auto cost = [&](int64_t bm, int64_t bn, int64_t units, int64_t loads) {
    return gc::ceil_div(with_rows * gc::ceil_div(rows, bm) * gc::ceil_div(n, bn), units) * (a + loads);
  };
  const int64_t pair = cost(256, 256, gc::kNumSMs / 2, 128), wide = cost(BM, 128, gc::kNumSMs, 128), narrow = cost(BM, 64, gc::kNumSMs, 64);
  if (n > 128 && rows > BM && pair <= std::min(wide, narrow)) return {256, true};
  return {n > 64 && wide <= narrow ? 128 : 64, false};
}
Shape shape_of_weights(int64_t m, int64_t n) {
  if (m > 128 && n > 128) return {256, true};
  return {n > 64 ? 128 : 64, false};
}
// Rows of a part of dW.  Few tiles: so many that the parts' tiles, one more per group than the rows alone would make, fill the GPU once
// (8 groups of 169,343 rows, 256 x 256: 36 us; with half as many rows in a part, whose last round is nearly empty, 44 and twice the
// sums).  More: the number of parts of an average group that takes least, where a part's fp32 sums cost as much as kSums rows to write and
// add, and the launch that adds as half of that; a group that stays whole may be a quarter
// larger, or half an SM's share of the work (4096 rows of 8 groups, 1024 x 1024: 19 us, 41 where every part is such a share; 60,000 of 8 102 and
// 144; 20,000 of 8, 512 x 512, 27 and 38).  At least 4 k-blocks, and at most kChain rows, beyond which truncation would show.
constexpr int64_t kChain = 16384;
constexpr int64_t kSums = 1280;
int64_t part_rows(int64_t M, int64_t m, int64_t n, int64_t G, const Shape& s) {
  const int64_t tiles = gc::ceil_div(m, s.pair ? 256 : BM) * gc::ceil_div(n, s.bn), units = s.pair ? gc::kNumSMs / 2 : gc::kNumSMs;
  const int64_t groups = std::min(G, M), rows = gc::ceil_div(M, groups), all = groups * tiles;
  int64_t part;
  if (units > 4 * all) {
    part = gc::ceil_div(M * tiles, units - all);
  } else {
    int64_t parts = 1, least = gc::ceil_div(all, units) * (rows + kSums / 4);
    for (int64_t i = 2; i <= 8; ++i) {
      const int64_t cost = gc::ceil_div(all * i, units) * (gc::ceil_div(rows, i) + kSums) + kSums / 2;
      if (cost < least) least = cost, parts = i;
    }
    part = parts > 1 ? gc::ceil_div(rows, parts) : std::max({rows + rows / 4, kSums, gc::ceil_div(M * tiles, 2 * units)});
  }
  return std::min(kChain, std::max<int64_t>(4 * KE, gc::ceil_div(part, KE) * KE));
}
int64_t parts_most(int64_t M, int64_t G, int64_t part) { return M / part + G; }  // that exist, at most

template <int MODE, int BN, bool PAIR>
int launch(const Maps& maps, const Params& p, int64_t items, cudaStream_t st) {
  using C_ = Cfg<BN, PAIR>;
  auto kern = grouped_kernel<MODE, BN, PAIR>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C_::kSmemBytes);
  if (e != cudaSuccess) return gc::fail(GC_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  constexpr int kCtas = PAIR ? 2 : 1;
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
  return gc::check_launch("grouped_kernel");
}
template <int MODE>
int launch_shape(const Shape& s, const Maps& maps, const Params& p, int64_t items, cudaStream_t st) {
  if (items > 0x7FFF0000) return gc::fail(GC_ERR_UNSUPPORTED, "grouped product: too many tiles");
  if (s.pair) return launch<MODE, 256, true>(maps, p, items, st);
  if (s.bn == 128) return launch<MODE, 128, false>(maps, p, items, st);
  return launch<MODE, 64, false>(maps, p, items, st);
}

// C (M x n) = A (M x K) W[g] (K x n), or W[g]^T with W[g] n x K: `w` is all weights, one below the other.
template <int MODE>
int rows_product(const Matrix& A, const Matrix& w, const int32_t* offsets, int64_t M, int64_t K, int64_t n, int64_t G, bf16* C, int64_t ldc,
                 cudaStream_t st) {
  const Shape s = shape_of_rows(M, n, G);
  Maps maps{};
  Params p{};
  p.offsets = offsets;
  p.groups = int(G); p.rows = int(M);
  p.K = int(K); p.n = int(n);
  p.C = C; p.ldc = ldc;
  p.tma_store = ldc % 8 == 0 && gc::aligned16(C);
  const int a_rows = int(std::min<int64_t>(BM, (M + 7) / 8 * 8));
  p.a_bytes = a_rows * 128;
  const int bnc = s.pair ? s.bn / 2 : s.bn;
  int rc = error_word(&p.word);
  if (rc == GC_OK) rc = make_map(&maps.a, A, KE, a_rows);
  const Matrix one{w.p, w.rows / G, w.cols, w.ld, 2};
  if (rc == GC_OK) rc = MODE == kBack ? make_map(&maps.b, one, KE, bnc, G) : make_map(&maps.b, one, 64, 64, G);
  if (rc == GC_OK && p.tma_store) rc = make_map(&maps.out, Matrix{C, M, n, ldc, 2}, 32, 32);
  if (rc != GC_OK) return rc;
  const int64_t items = (M / (s.pair ? 256 : BM) + std::min(G, M)) * gc::ceil_div(n, s.bn);
  return launch_shape<MODE>(s, maps, p, items, st);
}

size_t weights_workspace(int64_t M, int64_t K, int64_t N, int64_t G) {
  const int64_t part = part_rows(M, K, N, G, shape_of_weights(K, N));
  const size_t parts = M > part ? align256(size_t(parts_most(M, G, part)) * size_t(K) * size_t((N + 3) / 4 * 4) * 4) : 0;
  return align256(size_t(G) * KE * up8(K) * 2) + align256(size_t(G) * KE * up8(N) * 2) + parts;
}
int weights_product(const Matrix& x, const Matrix& dy, const int32_t* offsets, int64_t M, int64_t K, int64_t N, int64_t G, bf16* C,
                    char* ws, cudaStream_t st) {
  const Shape s = shape_of_weights(K, N);
  Maps maps{};
  Params p{};
  p.offsets = offsets;
  p.groups = int(G); p.rows = int(M);
  p.m = int(K); p.n = int(N);
  p.part = int(part_rows(M, K, N, G, s));
  p.C = C; p.ldc = N;
  p.tma_store = N % 8 == 0 && gc::aligned16(C);
  p.a_bytes = BM * 128;
  // the rows that fill up no block of 64
  uint4* x_tail = reinterpret_cast<uint4*>(ws);
  ws += align256(size_t(G) * KE * up8(K) * 2);
  uint4* dy_tail = reinterpret_cast<uint4*>(ws);
  ws += align256(size_t(G) * KE * up8(N) * 2);
  p.parts = reinterpret_cast<float*>(ws);
  const unsigned across = unsigned(std::min<int64_t>(gc::ceil_div(int64_t(KE) * (up8(K) + up8(N)) / 8, 4 * 256), 64));
  grouped_tail_kernel<<<dim3(unsigned(G), across), 256, 0, st>>>(p, static_cast<const uint16_t*>(x.p), x.ld,
                                                                 static_cast<const uint16_t*>(dy.p), dy.ld, x_tail, dy_tail);
  int rc = gc::check_launch("grouped_tail_kernel");
  if (rc == GC_OK) rc = error_word(&p.word);
  if (rc == GC_OK) rc = make_map(&maps.a, x, 64, 64);
  if (rc == GC_OK) rc = make_map(&maps.b, dy, 64, 64);
  if (rc == GC_OK) rc = make_map(&maps.a_tail, Matrix{x_tail, G * KE, K, up8(K), 2}, 64, 64);
  if (rc == GC_OK) rc = make_map(&maps.b_tail, Matrix{dy_tail, G * KE, N, up8(N), 2}, 64, 64);
  if (rc == GC_OK && p.tma_store) rc = make_map(&maps.out, Matrix{C, K, N, N, 2}, 32, 32, G);
  const bool cut = M > p.part;
  const int64_t pitch = (N + 3) / 4 * 4;
  if (rc == GC_OK && cut) rc = make_map(&maps.out_parts, Matrix{p.parts, K, pitch, pitch, 4}, 16, 32, parts_most(M, G, p.part));
  if (rc != GC_OK) return rc;
  const int64_t tiles = gc::ceil_div(K, s.pair ? 256 : BM) * gc::ceil_div(N, s.bn);
  rc = launch_shape<kWeights>(s, maps, p, parts_most(M, G, p.part) * tiles, st);
  if (rc != GC_OK || !cut) return rc;
  const unsigned blocks = unsigned(std::min<int64_t>(gc::ceil_div(K * (pitch / 4), 256), gc::ceil_div(gc::kNumSMs * 8, G)));
  grouped_sum_kernel<<<dim3(unsigned(G), blocks), 256, 0, st>>>(p);
  return gc::check_launch("grouped_sum_kernel");
}

// A call's operands, of which it copies those that cannot be read in place.
struct Operands {
  Matrix dy, x, w;
  bool needs_dy, needs_x, needs_w;
};
Operands operands(const uint16_t* dY, int64_t lddy, const uint16_t* X, int64_t ldx, const uint16_t* W, int64_t ldw, int64_t M, int64_t K,
                  int64_t N, int64_t G, bool backward, bool dx, bool dw) {
  return {Matrix{dY, M, N, lddy, 2}, Matrix{X, M, K, ldx, 2}, Matrix{W, G * K, N, ldw, 2}, backward, !backward || dw, !backward || dx};
}
// Up to here room for every copy is asked for whatever the operands are, so that a buffer that is kept does not change its size with them.
constexpr size_t kSmallWorkspace = size_t(1) << 20;
size_t workspace_of_all(int64_t M, int64_t K, int64_t N, int64_t G, bool backward, size_t weights) {
  const size_t x = align256(size_t(M) * up8(K) * 2), dy = align256(size_t(M) * up8(N) * 2), w = align256(size_t(G) * K * up8(N) * 2);
  return backward ? x + dy + w + weights : x + w;
}
size_t workspace_of(const Operands& o, int64_t M, int64_t K, int64_t N, int64_t G, bool backward, bool dw) {
  const size_t weights = backward ? weights_workspace(M, K, N, G) : 0, all = workspace_of_all(M, K, N, G, backward, weights);
  if (all <= kSmallWorkspace) return all;
  size_t b = 256;  // a workspace there is
  if (o.needs_dy) b += copy_bytes(o.dy);
  if (o.needs_x) b += copy_bytes(o.x);
  if (o.needs_w) b += copy_bytes(o.w);
  if (dw) b += weights;
  return std::min(all, b);
}

int check_sizes(const char* what, int64_t M, int64_t K, int64_t N, int64_t G, int64_t ldw, const int32_t* offsets) {
  GC_REQUIRE(M >= 0 && K >= 0 && N >= 0 && G >= 0, "%s: negative size", what);
  GC_REQUIRE(ldw >= N, "%s: leading dimension below the row length", what);
  const int64_t top = (int64_t(1) << 31) - 1024;
  if (M > top || K > top || N > top || G > (1 << 20)) return gc::fail(GC_ERR_UNSUPPORTED, "%s: a size beyond 2^31, or groups beyond 2^20", what);
  GC_REQUIRE(offsets, "%s: null pointer", what);
  return GC_OK;
}
int zero(uint16_t* p, int64_t ld, int64_t rows, int64_t cols, cudaStream_t st, const char* what) {
  if (!p || rows == 0 || cols == 0) return GC_OK;
  const cudaError_t e = cudaMemset2DAsync(p, size_t(ld) * 2, 0, size_t(cols) * 2, size_t(rows), st);
  return e == cudaSuccess ? GC_OK : gc::fail(GC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace

extern "C" {

size_t gc_grouped_linear_workspace_bytes(int64_t M, int64_t K, int64_t N, int64_t G, int backward) {
  if (M <= 0 || K <= 0 || N <= 0 || G <= 0) return 0;
  // copies of every operand, should none be readable in place
  return workspace_of_all(M, K, N, G, backward, backward ? weights_workspace(M, K, N, G) : 0);
}

size_t gc_grouped_linear_workspace_bytes_for(const uint16_t* dY, int64_t lddy, const uint16_t* X, int64_t ldx, const uint16_t* W, int64_t ldw,
                                             int64_t M, int64_t K, int64_t N, int64_t G, int dx, int dw) {
  if (M <= 0 || K <= 0 || N <= 0 || G <= 0) return 0;
  const bool backward = dx || dw;
  return workspace_of(operands(dY, lddy, X, ldx, W, ldw, M, K, N, G, backward, dx, dw), M, K, N, G, backward, dw);
}

int gc_grouped_linear_forward_bf16(const uint16_t* X, int64_t ldx, const uint16_t* W, int64_t ldw, const int32_t* offsets, int64_t M,
                                   int64_t K, int64_t N, int64_t G, uint16_t* Y, int64_t ldy, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  const char* what = "gc_grouped_linear_forward_bf16";
  int rc = check_sizes(what, M, K, N, G, ldw, offsets);
  if (rc != GC_OK) return rc;
  GC_REQUIRE(ldx >= K && ldy >= N, "%s: leading dimension below the row length", what);
  const cudaStream_t st = gc::as_stream(stream);
  if (M == 0 || N == 0) return GC_OK;
  GC_REQUIRE(Y, "%s: null pointer", what);
  if (K == 0 || G == 0) return zero(Y, ldy, M, N, st, what);
  GC_REQUIRE(X && W, "%s: null pointer", what);
  Operands o = operands(nullptr, 0, X, ldx, W, ldw, M, K, N, G, false, false, false);
  if (!workspace || workspace_bytes < workspace_of(o, M, K, N, G, false, false))
    return gc::fail(GC_ERR_WORKSPACE, "%s: workspace missing or smaller than its query says", what);
  GC_REQUIRE(gc::aligned16(workspace), "%s: workspace must be 16-byte aligned", what);
  char* ws = static_cast<char*>(workspace);
  Copies copies{};
  make_readable(o.x, ws, copies);
  make_readable(o.w, ws, copies);
  rc = run_copies(copies, st);
  if (rc != GC_OK) return rc;
  return rows_product<kForward>(o.x, o.w, offsets, M, K, N, G, reinterpret_cast<bf16*>(Y), ldy, st);
}

int gc_grouped_linear_backward_bf16(const uint16_t* dY, int64_t lddy, const uint16_t* X, int64_t ldx, const uint16_t* W, int64_t ldw,
                                    const int32_t* offsets, int64_t M, int64_t K, int64_t N, int64_t G, uint16_t* dX, int64_t lddx,
                                    uint16_t* dW, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "gc_grouped_linear_backward_bf16";
  int rc = check_sizes(what, M, K, N, G, ldw, offsets);
  if (rc != GC_OK) return rc;
  GC_REQUIRE(lddy >= N && ldx >= K && (!dX || lddx >= K), "%s: leading dimension below the row length", what);
  const cudaStream_t st = gc::as_stream(stream);
  if (M == 0 || K == 0 || N == 0 || G == 0) {  // sums of nothing
    rc = zero(dX, lddx, M, K, st, what);
    return rc == GC_OK ? zero(dW, N, G * K, N, st, what) : rc;
  }
  if (!dX && !dW) return GC_OK;
  GC_REQUIRE(dY && X && W, "%s: null pointer", what);
  Operands o = operands(dY, lddy, X, ldx, W, ldw, M, K, N, G, true, dX, dW);
  if (!workspace || workspace_bytes < workspace_of(o, M, K, N, G, true, dW))
    return gc::fail(GC_ERR_WORKSPACE, "%s: workspace missing or smaller than its query says", what);
  GC_REQUIRE(gc::aligned16(workspace), "%s: workspace must be 16-byte aligned", what);
  char* ws = static_cast<char*>(workspace);
  Copies copies{};
  make_readable(o.dy, ws, copies);
  if (o.needs_x) make_readable(o.x, ws, copies);
  if (o.needs_w) make_readable(o.w, ws, copies);
  rc = run_copies(copies, st);
  if (rc == GC_OK && dX) rc = rows_product<kBack>(o.dy, o.w, offsets, M, N, K, G, reinterpret_cast<bf16*>(dX), lddx, st);
  if (rc == GC_OK && dW) rc = weights_product(o.x, o.dy, offsets, M, K, N, G, reinterpret_cast<bf16*>(dW), ws, st);
  return rc;
}

}  // extern "C"
