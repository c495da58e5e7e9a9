// What the kernels of products with 4-bit weights share: records, their unpacking, the tensor-core instruction that takes registers, bulk
// copies.
#pragma once

#include "common.cuh"
#include "ffn_internal.cuh"
#include "tiles.cuh"

#include <cuda_bf16.h>

namespace gc {
namespace int4 {

using namespace gc::ffn;
using namespace gc::tc;
using gc::tiles::align256;
using gc::tiles::drain;
using gc::tiles::up8;
using bf16 = __nv_bfloat16;

constexpr int kChunk = 128;       // inputs of a chunk

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
// Waits for a copy, a bounded time (tries of a microsecond at most); the same answer for all of a warp.
__device__ __forceinline__ bool arrived(uint32_t bar, uint32_t parity) {
  uint32_t tries = 1u << 21;
  bool done;
  do {
    uint32_t now;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(now)
        : "r"(bar), "r"(parity)
        : "memory");
    done = now != 0;
  } while (!done && --tries);
  return __all_sync(0xFFFFFFFFu, done);
}
// Eight codes as four pairs of bf16 numbers less their zero points; 0x4300 is 128 and its last bits count ones, and `zero` is a pair of
// -(128 + zero point).  (A multiply-add, by one: a subtraction would go to the pipe of the shifts and masks, which is the busy one.)
__device__ __forceinline__ void unpack(uint32_t w, __nv_bfloat162 zero, uint32_t (&o)[4]) {
  const __nv_bfloat162 one = __float2bfloat162_rn(1.f);
  uint32_t mask;
  asm("mov.b32 %0, 0x000F000F;" : "=r"(mask));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t t;  // (w >> 4 i & mask) | 128s, in one instruction but for the shift: the mask waits in a register
    asm("lop3.b32 %0, %1, %2, 0x43004300, 0xEA;" : "=r"(t) : "r"(w >> (4 * i)), "r"(mask));
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&t), one, zero);
    o[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}
__device__ __forceinline__ __nv_bfloat162 zero_pair(uint32_t zeros, int byte) {
  const uint32_t t = __byte_perm(zeros, 0xC3u, 0x4040u + 0x0101u * byte);
  return *reinterpret_cast<const __nv_bfloat162*>(&t);
}
__device__ __forceinline__ uint4 shared_16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint2 shared_8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t shared_4(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t shared_2(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t shared_1(uint32_t at) {
  uint16_t v;
  asm volatile("{\n\t.reg .u8 b;\n\tld.shared.u8 b, [%1];\n\tcvt.u16.u8 %0, b;\n\t}" : "=h"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float gated(float g, float u, int act) {
  float a = 0.f, unused;
  with_activation(act, [&](auto t) {
    F2 slope;
    activate<decltype(t)::value>(F2(g, g), slope).get(a, unused);
  });
  return a * u;
}

// A record: 64 bytes of codes for each of 16 outputs, their scales, their zero points.
constexpr int kScales = 16 * 64;
__host__ __device__ constexpr int zeros_at(int gpc) { return kScales + 16 * gpc * 2; }
__host__ __device__ constexpr int record_bytes(int gpc, bool zeros) { return zeros_at(gpc) + (zeros ? 16 * gpc : 0); }

// ------------------------------------------------------------------ host
struct Weights {
  const uint8_t* records;
  int group, zeros;
  int gpc() const { return kChunk / group; }
  int64_t bytes(int64_t K, int64_t N) const { return gc::ceil_div(N, 16) * gc::ceil_div(K, kChunk) * record_bytes(gpc(), zeros); }
};

// For some tens of rows (int4_tiles.cu).
constexpr int64_t kLinearTileRows = 128, kBlockTileRows = 64;
size_t linear_tiles_workspace(int64_t M, int64_t K, int64_t N);
int linear_tiles(const uint16_t* X, int64_t ldx, const Weights& w, int64_t M, int64_t K, int64_t N, uint16_t* Y, int64_t ldy, void* workspace,
                 cudaStream_t st);
size_t block_tiles_workspace(int64_t M, int64_t D, int64_t H, int64_t O);
int block_tiles(const uint16_t* X, int64_t ldx, const Weights& in, const Weights& out, int64_t M, int64_t D, int64_t H, int64_t O, int act,
                uint16_t* Y, int64_t ldy, void* workspace, cudaStream_t st);

}  // namespace int4
}  // namespace gc
