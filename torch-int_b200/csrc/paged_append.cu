// Appends the keys and values of a ragged batch of new tokens to a paged int8 cache, with the position
// rotation and the quantisation applied on the way (and, if given, the queries rotated and quantised too):
//   y1 = x1 * c - x2 * s,  y2 = x2 * c + x1 * s      pairs of the first rotary_dim columns of q and k
//   int8 = sat(rne(alpha * y))
// Every product, sum and difference is rounded to fp32 by itself (no contraction), so that the int8 results
// are defined bit by bit whatever the compiler does; int8 -> int8 with alpha = 1 and no rotation is a copy.
//
// Bound by bytes: (q_heads + 2 kv_heads) * head_dim * (size of the input + 1) per token, each touched once.  A unit is
// 16 columns of one head of one token: two runs of 8 (the two halves of 8 rotated pairs, or 16 neighbours), so that
// every access is 8 to 32 contiguous bytes and a pool row of a head is written by neighbouring lanes.  A block takes a
// range of a sequence's units, cut so that few tokens still spread over many blocks and many tokens do not pay a
// block's fixed latency (lengths, then pages, then data) too often; the page lookups of its tokens go through shared
// memory.  What hides the latencies is occupancy: two units in flight per thread at 64 registers move more than four
// at 93 did.  Measured: 8 x 512 int8 tokens of 56 heads x 128 22.5 us (5.2 TB/s), 4 x 2048 fp32 tokens of 40 heads x 128
// with 64 columns rotated 65 us (5.6 TB/s), 8 decoded tokens 2.3 us (a launch and three latencies).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "gemm_i8.h"
#include "grid_dependency.cuh"
#include "paged.h"
#include "paged_device.cuh"

namespace ti {
namespace {

constexpr int APPEND_THREADS = 256;
constexpr int PAGED_APPEND_BLOCKS = 4 * 148;
constexpr int APPEND_MAX_UNITS = 2048;                          // of a block
constexpr int APPEND_MAX_TOKENS = APPEND_MAX_UNITS / (2 * 4) + 2;  // it can touch: a token has at least 8 units

struct AppendParams {
  PagedView view;
  const void* src[3];      // q, k, v
  long long ld[3];         // elements between tokens
  float alpha[3];
  const float* rotary;
  int rotary_rows, rotary_dim, interleaved;
  int8_t* q_out;
  int q_heads;
  int units_per_token;     // (q_heads + 2 kv_heads) * D / 16
  int units_per_block;
};

// Four floats -> four int8 in one word: rne, saturated; NaN -> 0.
__device__ __forceinline__ uint32_t quantise4(float a, float b, float c, float d) {
  uint32_t lo, out;
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(lo) : "r"(__float2int_rn(d)), "r"(__float2int_rn(c)));
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(out) : "r"(__float2int_rn(b)), "r"(__float2int_rn(a)), "r"(lo));
  return out;
}

// Eight elements as they lie in memory.
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ void get(float (&x)[8]) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
};
template <>
struct Raw8<__half> {
  uint4 a;
  __device__ void load(const __half* p) { a = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};
template <>
struct Raw8<__nv_bfloat16> {
  uint4 a;
  __device__ void load(const __nv_bfloat16* p) { a = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
};
template <>
struct Raw8<int8_t> {
  uint2 a;
  __device__ void load(const int8_t* p) { a = __ldg(reinterpret_cast<const uint2*>(p)); }
  __device__ void get(float (&x)[8]) const {
    const uint32_t w[2] = {a.x, a.y};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w[i >> 2] >> (8 * (i & 3))));
  }
};

// COPY: int8 rows stored as they are.
template <typename T, int D, bool COPY>
__global__ void __launch_bounds__(APPEND_THREADS, COPY ? 6 : 4) paged_append_kernel(const AppendParams p) {
  constexpr int PIECES = D / 16;
  constexpr int UNITS = COPY ? 4 : 2;             // units a thread has in flight
  __shared__ int s_row[APPEND_MAX_TOKENS];        // page * page_size + row, -1: nothing to store
  const PagedView& v = p.view;
  const int b = blockIdx.y, tid = threadIdx.x;
  grid_dep_launch();
  grid_dep_wait();
  PagedSeq s;
  if (!paged_sequence(v, b, INT_MAX, &s)) return;
  if (s.L < s.T) {  // the new tokens are part of the keys
    if (tid == 0) atomicCAS(v.status, 0, static_cast<int>(TI_ERR_PAGED_LENGTHS));
    return;
  }
  const int upt = p.units_per_token;
  const long long u0 = static_cast<long long>(blockIdx.x) * p.units_per_block;
  if (u0 >= static_cast<long long>(s.T) * upt) return;
  const int t0 = static_cast<int>(u0 / upt), skip = static_cast<int>(u0 - static_cast<long long>(t0) * upt);
  const int nt = min((skip + p.units_per_block + upt - 1) / upt, s.T - t0);
  const int pos0 = s.L - s.T + t0;
  for (int i = tid; i < nt; i += APPEND_THREADS) {
    const int pos = pos0 + i;
    const int page = paged_page(v, b, pos >> v.page_shift);
    int row = page < 0 ? -1 : (page << v.page_shift) + (pos & ((1 << v.page_shift) - 1));
    if (p.rotary != nullptr && pos >= p.rotary_rows) {
      atomicCAS(v.status, 0, static_cast<int>(TI_ERR_PAGED_LENGTHS));
      row = -1;
    }
    s_row[i] = row;
  }
  __syncthreads();
  const int end = min(skip + p.units_per_block, nt * upt);
  const int hk = v.kv_heads, rd = p.rotary_dim;
  const long long token0 = s.q0 + t0;
  for (int base = skip + tid; base < end; base += APPEND_THREADS * UNITS) {
    Raw8<T> lo[UNITS], hi[UNITS];
    uint4 whole[UNITS];
    int8_t* dst[UNITS];
    int tok[UNITS], piece[UNITS], cls[UNITS];  // cls: 0 q, 1 k, 2 v, -1 none
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int idx = base + u * APPEND_THREADS;
      cls[u] = -1;
      if (idx >= end) continue;
      const int t = idx / upt, rest = idx - t * upt, row = s_row[t];
      if (row < 0) continue;
      const int hh = rest / PIECES;
      piece[u] = rest - hh * PIECES;
      tok[u] = t;
      int head;
      if (hh < p.q_heads) {
        cls[u] = 0;
        head = hh;
        dst[u] = p.q_out + ((token0 + t) * p.q_heads + head) * D;
      } else {
        cls[u] = hh < p.q_heads + hk ? 1 : 2;
        head = hh - p.q_heads - (cls[u] == 2 ? hk : 0);
        const long long page = row >> v.page_shift;
        const int in_page = row & ((1 << v.page_shift) - 1);
        dst[u] = (cls[u] == 1 ? v.k_pages : v.v_pages) + ((((page * hk) + head) << v.page_shift) + in_page) * D;
      }
      const T* src = static_cast<const T*>(p.src[cls[u]]) + (token0 + t) * p.ld[cls[u]] + head * D;
      if constexpr (COPY) {
        whole[u] = __ldg(reinterpret_cast<const uint4*>(src + piece[u] * 16));
      } else {
        const bool halves = cls[u] < 2 && piece[u] * 16 < rd && !p.interleaved;
        lo[u].load(src + (halves ? piece[u] * 8 : piece[u] * 16));
        hi[u].load(src + (halves ? rd / 2 + piece[u] * 8 : piece[u] * 16 + 8));
      }
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      if (cls[u] < 0) continue;
      if constexpr (COPY) {
        *reinterpret_cast<uint4*>(dst[u] + piece[u] * 16) = whole[u];
      } else {
        float x[8], y[8];
        lo[u].get(x);
        hi[u].get(y);
        const bool rotated = cls[u] < 2 && piece[u] * 16 < rd;
        if (rotated) {
          const float* c = p.rotary + static_cast<long long>(pos0 + tok[u]) * rd + piece[u] * 8;
          const float* sn = c + rd / 2;
          auto turn = [](float& a, float& d, float co, float si) {
            const float a1 = __fsub_rn(__fmul_rn(a, co), __fmul_rn(d, si));
            d = __fadd_rn(__fmul_rn(d, co), __fmul_rn(a, si));
            a = a1;
          };
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float4 cs = __ldg(reinterpret_cast<const float4*>(c) + q), ss = __ldg(reinterpret_cast<const float4*>(sn) + q);
            if (p.interleaved) {
              float(&z)[8] = q == 0 ? x : y;
              turn(z[0], z[1], cs.x, ss.x);
              turn(z[2], z[3], cs.y, ss.y);
              turn(z[4], z[5], cs.z, ss.z);
              turn(z[6], z[7], cs.w, ss.w);
            } else {
              turn(x[4 * q], y[4 * q], cs.x, ss.x);
              turn(x[4 * q + 1], y[4 * q + 1], cs.y, ss.y);
              turn(x[4 * q + 2], y[4 * q + 2], cs.z, ss.z);
              turn(x[4 * q + 3], y[4 * q + 3], cs.w, ss.w);
            }
          }
        }
        const float al = p.alpha[cls[u]];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = __fmul_rn(x[i], al);
          y[i] = __fmul_rn(y[i], al);
        }
        const uint2 a = make_uint2(quantise4(x[0], x[1], x[2], x[3]), quantise4(x[4], x[5], x[6], x[7]));
        const uint2 d = make_uint2(quantise4(y[0], y[1], y[2], y[3]), quantise4(y[4], y[5], y[6], y[7]));
        if (rotated && !p.interleaved) {
          *reinterpret_cast<uint2*>(dst[u] + piece[u] * 8) = a;
          *reinterpret_cast<uint2*>(dst[u] + rd / 2 + piece[u] * 8) = d;
        } else {
          *reinterpret_cast<uint4*>(dst[u] + piece[u] * 16) = make_uint4(a.x, a.y, d.x, d.y);
        }
      }
    }
  }
}

// Launched as a programmatic dependent: the launch overlaps the end of the kernel before it, which it waits for.
template <typename T, bool COPY>
cudaError_t launch_append(int head_dim, dim3 grid, const AppendParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(APPEND_THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (head_dim == 128) return cudaLaunchKernelEx(&cfg, paged_append_kernel<T, 128, COPY>, p);
  if (head_dim == 80) return cudaLaunchKernelEx(&cfg, paged_append_kernel<T, 80, COPY>, p);
  return cudaLaunchKernelEx(&cfg, paged_append_kernel<T, 64, COPY>, p);
}

}  // namespace

int check_paged_batch(const PagedBatch& b, const char* name) {
  if (b.head_dim != 64 && b.head_dim != 80 && b.head_dim != 128) {
    set_error("%s: head_dim must be 64, 80 or 128 (got %lld)", name, (long long)b.head_dim);
    return TI_E_INVALID;
  }
  if (b.page_size != 16 && b.page_size != 32 && b.page_size != 64 && b.page_size != 128 && b.page_size != 256) {
    set_error("%s: page_size must be 16, 32, 64, 128 or 256 (got %lld)", name, (long long)b.page_size);
    return TI_E_INVALID;
  }
  const int64_t most_pages = 0x7FFFFFFF / b.page_size;
  if (b.kv_heads <= 0 || b.kv_heads > 65535 || b.batch < 0 || b.batch > 65535 || b.tokens < 0 || b.tokens > 0x7FFFFFFF ||
      b.max_query_len < 0 || b.num_pages <= 0 || b.num_pages > most_pages || b.table_width <= 0 || b.table_width > most_pages ||
      b.table_ld < b.table_width) {
    set_error("%s: sizes out of range (batch %lld, tokens %lld, kv_heads %lld, %lld pages of %lld, block table %lld wide)",
              name, (long long)b.batch, (long long)b.tokens, (long long)b.kv_heads, (long long)b.num_pages,
              (long long)b.page_size, (long long)b.table_width);
    return TI_E_INVALID;
  }
  if (b.batch == 0 || b.tokens == 0) return TI_OK;
  if (!b.k_pages || !b.v_pages || !b.block_table || !b.query_starts || !b.kv_lens) {
    set_error("%s: null pointer", name);
    return TI_E_INVALID;
  }
  if (((reinterpret_cast<uintptr_t>(b.k_pages) | reinterpret_cast<uintptr_t>(b.v_pages)) & 15) != 0 ||
      ((reinterpret_cast<uintptr_t>(b.block_table) | reinterpret_cast<uintptr_t>(b.query_starts) |
        reinterpret_cast<uintptr_t>(b.kv_lens)) & 3) != 0) {
    set_error("%s: the pools must be 16-byte aligned and the index arrays 4-byte aligned", name);
    return TI_E_INVALID;
  }
  return TI_OK;
}

int paged_append(const PagedBatch& b, const PagedAppend& a, cudaStream_t stream) {
  const int rc = check_paged_batch(b, "paged_append");
  if (rc != TI_OK) return rc;
  if (a.dtype < 0 || a.dtype > 3) {
    set_error("paged_append: unknown input type %d", a.dtype);
    return TI_E_INVALID;
  }
  if (a.rotary != nullptr && (a.rotary_dim <= 0 || a.rotary_dim > b.head_dim || a.rotary_dim % 16 != 0 ||
                              a.rotary_rows <= 0 || a.rotary_rows > 0x7FFFFFFF ||
                              (reinterpret_cast<uintptr_t>(a.rotary) & 15) != 0)) {
    set_error("paged_append: the rotary table must be 16-byte aligned [positions, rotary_dim] with rotary_dim a multiple "
              "of 16 of at most head_dim (got %lld)", (long long)a.rotary_dim);
    return TI_E_INVALID;
  }
  if (b.batch == 0 || b.tokens == 0 || b.max_query_len == 0) return TI_OK;
  const int size = a.dtype == 0 ? 4 : a.dtype == 3 ? 1 : 2;
  const int64_t q_heads = a.q != nullptr ? a.q_heads : 0;
  if (!a.k || !a.v || (a.q != nullptr && (!a.q_out || a.q_heads <= 0 || a.q_heads > 65535))) {
    set_error("paged_append: null pointer or no query heads");
    return TI_E_INVALID;
  }
  const int64_t ld_min[3] = {q_heads * b.head_dim, b.kv_heads * b.head_dim, b.kv_heads * b.head_dim};
  const void* src[3] = {a.q, a.k, a.v};
  const int64_t ld[3] = {a.ld_q, a.ld_k, a.ld_v};
  for (int i = a.q != nullptr ? 0 : 1; i < 3; ++i) {
    if ((reinterpret_cast<uintptr_t>(src[i]) & 15) != 0 || (b.tokens > 1 && ((ld[i] * size) % 16 != 0 || ld[i] < ld_min[i]))) {
      set_error("paged_append: q, k and v rows must be 16-byte aligned and hold their heads side by side");
      return TI_E_INVALID;
    }
  }
  if (a.q_out && (reinterpret_cast<uintptr_t>(a.q_out) & 15) != 0) {
    set_error("paged_append: the output of the queries must be 16-byte aligned");
    return TI_E_INVALID;
  }
  int* status = status_word_ptr();
  if (!status) {
    set_error("paged_append: cannot resolve the device status word");
    return TI_E_CUDA;
  }
  AppendParams p;
  p.view = make_paged_view(b, status);
  const float alpha[3] = {a.q_alpha, a.k_alpha, a.v_alpha};
  for (int i = 0; i < 3; ++i) {
    p.src[i] = src[i];
    p.ld[i] = ld[i];
    p.alpha[i] = alpha[i];
  }
  p.rotary = a.rotary;
  p.rotary_rows = static_cast<int>(a.rotary_rows);
  p.rotary_dim = a.rotary != nullptr ? static_cast<int>(a.rotary_dim) : 0;
  p.interleaved = a.interleaved;
  p.q_out = a.q_out;
  p.q_heads = static_cast<int>(q_heads);
  p.units_per_token = static_cast<int>((q_heads + 2 * b.kv_heads) * (b.head_dim / 16));
  // Blocks of up to APPEND_MAX_UNITS units, smaller ones where the tokens would not fill four blocks per SM.
  const int64_t max_q = b.max_query_len < b.tokens ? b.max_query_len : b.tokens;
  int64_t units = b.tokens * p.units_per_token / (PAGED_APPEND_BLOCKS * APPEND_THREADS) * APPEND_THREADS;
  units = units < APPEND_THREADS ? APPEND_THREADS : units > APPEND_MAX_UNITS ? APPEND_MAX_UNITS : units;
  p.units_per_block = static_cast<int>(units);
  const int64_t blocks = (max_q * p.units_per_token + units - 1) / units;
  if (blocks > 0x7FFFFFFF) {
    set_error("paged_append: too many new tokens for one call");
    return TI_E_INVALID;
  }
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(b.batch));
  const int d = static_cast<int>(b.head_dim);
  const bool copy = a.dtype == 3 && a.rotary == nullptr && a.k_alpha == 1.f && a.v_alpha == 1.f && (!a.q || a.q_alpha == 1.f);
  const cudaError_t e = a.dtype == 0   ? launch_append<float, false>(d, grid, p, stream)
                        : a.dtype == 1 ? launch_append<__half, false>(d, grid, p, stream)
                        : a.dtype == 2 ? launch_append<__nv_bfloat16, false>(d, grid, p, stream)
                        : copy         ? launch_append<int8_t, true>(d, grid, p, stream)
                                       : launch_append<int8_t, false>(d, grid, p, stream);
  if (e != cudaSuccess) {
    set_error("paged_append launch failed: %s", cudaGetErrorString(e));
    return TI_E_CUDA;
  }
  return TI_OK;
}

}  // namespace ti
