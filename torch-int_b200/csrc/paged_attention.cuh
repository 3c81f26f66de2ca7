// What the kernels of attention over a paged cache share: parameters, the division of the keys, the store.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "paged_device.cuh"
#include "paged_plan.h"

namespace ti {

struct PagedAttnParams {
  PagedView view;
  const int8_t* q;
  long long ld_q;
  int q_heads, group;
  int max_kv_len;
  float scale_log2;   // alpha_qk * log2(e): scores are kept in the log2 domain
  float alpha_pv;
  void* out;
  int out_kind;       // 1 fp16, 2 bf16, 3 int8
  int row_tiles;      // of the largest sequence
  int first_tile;     // of the launch, counted over the sequences
  int chunk;          // keys of a split, a multiple of 32
  int max_splits;     // stride of the partial results
  int cluster;        // the splits of the rows kernel are a cluster and need no partial results
  int rows_below;     // sequences with at most this many rows belong to the rows kernel, the others to the tile kernel
  int beside_tiles;   // the rows kernel follows the tile kernel of the same call without waiting for it
  float* part_o;      // [tokens * q_heads][max_splits][head_dim], unnormalised
  float2* part_ml;    // [tokens * q_heads][max_splits]: maximum (log2 domain) and sum
};

// Runs a kernel's set-up (function attributes) the first time it is launched on a device: a call of its own costs
// about as much as a launch.
class PagedOncePerDevice {
 public:
  template <typename F>
  cudaError_t run(F&& f) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && (done_.load(std::memory_order_acquire) >> dev & 1))) return e;
    e = f();
    if (e == cudaSuccess && dev < 64) done_.fetch_or(1ull << dev, std::memory_order_release);
    return e;
  }

 private:
  std::atomic<unsigned long long> done_{0};
};

int launch_paged_tiles(const PagedBatch& b, const PagedAttnParams& p, const PagedTilePlan& plan, cudaStream_t stream);

struct PagedSplits {
  int keys;  // keys visible to some row of the tile
  int n;     // splits they are divided into, at least one
};
__device__ __forceinline__ PagedSplits paged_splits(int keys, int chunk) {
  PagedSplits s;
  s.keys = max(keys, 0);
  s.n = max(1, (s.keys + chunk - 1) / chunk);
  return s;
}

// Context values rounded once to the output type: two to fp16 or bf16, four to int8 (rne, saturated).
__device__ __forceinline__ uint32_t paged_pack2(int out_kind, float a, float b) {
  uint32_t r;
  if (out_kind == 2)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ uint32_t paged_pack4_s8(float a, float b, float c, float d) {
  uint32_t lo, w;
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(lo) : "r"(__float2int_rn(d)), "r"(__float2int_rn(c)));
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(w) : "r"(__float2int_rn(b)), "r"(__float2int_rn(a)), "r"(lo));
  return w;
}

// Four neighbouring context values times `scale`.
__device__ __forceinline__ void paged_store4(const PagedAttnParams& p, long long at, float4 x, float scale) {
  x.x *= scale;
  x.y *= scale;
  x.z *= scale;
  x.w *= scale;
  if (p.out_kind == 3)
    *reinterpret_cast<uint32_t*>(static_cast<int8_t*>(p.out) + at) = paged_pack4_s8(x.x, x.y, x.z, x.w);
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
        make_uint2(paged_pack2(p.out_kind, x.x, x.y), paged_pack2(p.out_kind, x.z, x.w));
}

}  // namespace ti
