// What the kernels that multiply bf16 (or e4m3) tiles with tcgen05.mma share: instruction and operand descriptors, bounded waits, tiles
// in shared memory on their way out, tensor maps, and copies of matrices whose rows TMA cannot read.
#pragma once

#include "common.cuh"
#include "gemm_internal.cuh"
#include "tcgen05.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

namespace gc {
namespace tiles {

using namespace gc::tc;

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
static __global__ void __launch_bounds__(256)
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
inline int make_map(CUtensorMap* map, const Matrix& m, int box_cols, int box_rows, int64_t planes = 0) {
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

// A matrix that TMA can read: itself, or a copy with a pitch of 16 bytes in the workspace, which moves on.
inline bool readable(const Matrix& m) { return gc::aligned16(m.p) && m.ld * m.size % 16 == 0; }
inline int64_t readable_ld(const Matrix& m) { return (m.cols * m.size + 15) / 16 * 16 / m.size; }
inline size_t copy_bytes(const Matrix& m) { return readable(m) ? 0 : align256(size_t(m.rows) * size_t(readable_ld(m)) * m.size); }
inline void add_copy(Copies& c, const Matrix& m, void* dst, int64_t ldd, int64_t width) {
  const int j = c.count++;
  c.job[j] = {m.p, dst, m.ld, ldd, m.rows, int(m.cols), int(width), m.size};
  const int64_t runs = gc::ceil_div(width * m.size / 4, Copies::kRun);
  const int64_t blocks = std::min<int64_t>(gc::ceil_div(m.rows * runs, 8), gc::kNumSMs * 8);
  c.first_block[0] = 0;
  c.first_block[j + 1] = c.first_block[j] + int(blocks);
}
inline void make_readable(Matrix& m, char*& ws, Copies& c) {
  if (readable(m)) return;
  const size_t bytes = copy_bytes(m);
  const int64_t ld = readable_ld(m);
  add_copy(c, m, ws, ld, ld);
  m.p = ws;
  m.ld = ld;
  ws += bytes;
}
inline int error_word(int** word) {
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

inline int run_copies(const Copies& c, cudaStream_t st) {
  if (c.count == 0) return GC_OK;
  repitch_kernel<<<unsigned(c.first_block[c.count]), 256, 0, st>>>(c);
  return gc::check_launch("repitch_kernel");
}

}  // namespace tiles
}  // namespace gc
