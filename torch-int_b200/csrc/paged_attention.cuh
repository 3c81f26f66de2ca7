// What the kernels of attention over a paged cache share: parameters, the division of the keys, the store.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "paged_device.cuh"

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
  int chunk;          // keys of a split, a multiple of 16
  int max_splits;
  int rows_below;     // sequences with at most this many rows belong to the rows kernel, the others to the tile kernel
  float* part_o;      // [tokens * q_heads][max_splits][head_dim], unnormalised
  float2* part_ml;    // [tokens * q_heads][max_splits]: maximum (log2 domain) and sum
};

constexpr int PAGED_SMS = 148;

// How the tile kernel (paged_attention_sm100.cu) cuts the work.
struct PagedTilePlan {
  int tokens_per_tile;  // of 128 rows: 128 / group
  int pairs;            // pairs of row tiles of the largest sequence
  int chunk;            // keys of a split, a multiple of 128
  int splits;
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

// Four neighbouring context values times `scale`, rounded once to the output type.
__device__ __forceinline__ void paged_store4(const PagedAttnParams& p, long long at, float4 x, float scale) {
  x.x *= scale;
  x.y *= scale;
  x.z *= scale;
  x.w *= scale;
  if (p.out_kind == 3) {
    uint32_t lo, w;
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(lo) : "r"(__float2int_rn(x.w)), "r"(__float2int_rn(x.z)));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(w) : "r"(__float2int_rn(x.y)), "r"(__float2int_rn(x.x)), "r"(lo));
    *reinterpret_cast<uint32_t*>(static_cast<int8_t*>(p.out) + at) = w;
  } else if (p.out_kind == 2) {
    const __nv_bfloat162 u = __floats2bfloat162_rn(x.x, x.y), w = __floats2bfloat162_rn(x.z, x.w);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&w));
  } else {
    const __half2 u = __floats2half2_rn(x.x, x.y), w = __floats2half2_rn(x.z, x.w);
    *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + at) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&w));
  }
}

// Sixteen neighbouring context values (fp32 bits) as `width` 16-byte pieces: 4 as they are (a partial result), 2 and
// 1 times `scale` and rounded once to fp16 / bf16 and int8.
__device__ __forceinline__ void paged_convert16(int width, int out_kind, const uint32_t (&o)[16], float scale, uint4 (&piece)[4]) {
  if (width == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) piece[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    return;
  }
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(o[i]) * scale;
  uint32_t w[8];
  if (width == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t lo;
      asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(lo) : "r"(__float2int_rn(x[4 * i + 3])), "r"(__float2int_rn(x[4 * i + 2])));
      asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;"
          : "=r"(w[i]) : "r"(__float2int_rn(x[4 * i + 1])), "r"(__float2int_rn(x[4 * i])), "r"(lo));
    }
  } else if (out_kind == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __nv_bfloat162 u = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __half2 u = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&u);
    }
  }
  piece[0] = make_uint4(w[0], w[1], w[2], w[3]);
  if (width == 2) piece[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

}  // namespace ti
