// Appends the keys and values of a ragged batch of new tokens to a paged int8 cache, with the position
// rotation and the quantisation applied on the way (and, if given, the queries rotated and quantised too):
//   y1 = x1 * c - x2 * s,  y2 = x2 * c + x1 * s      pairs of the first rotary_dim columns of q and k
//   int8 = sat(rne(alpha * y))
// Every product, sum and difference is rounded to fp32 by itself (no contraction), so that the int8 results
// are defined bit by bit whatever the compiler does; int8 -> int8 with alpha = 1 and no rotation is a copy.
//
// Bound by bytes: (q_heads + 2 kv_heads) * head_dim * (size of the input + 1) per token, each touched once.
// A thread owns 16 columns of one head of one token: two runs of 8 (the two halves of 8 rotated pairs, or
// 16 neighbours), so that every access is 8 to 32 contiguous bytes and a pool row of a head is written by
// neighbouring lanes.  UNITS of them are loaded before the first is used.  The page lookup of a token is
// done once per block, into shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "gemm_i8.h"
#include "paged.h"
#include "paged_device.cuh"

namespace ti {
namespace {

constexpr int APPEND_THREADS = 256;
constexpr int APPEND_MAX_TOKENS = 32;  // tokens of a block at most (page lookups in shared memory)

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
  int tokens_per_block;
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

template <typename T, int D>
__global__ void __launch_bounds__(APPEND_THREADS) paged_append_kernel(const AppendParams p) {
  constexpr int PIECES = D / 16;
  constexpr int UNITS = sizeof(T) == 4 ? 2 : 4;  // units a thread has in flight
  __shared__ int s_row[APPEND_MAX_TOKENS];       // page * page_size + row, -1: nothing to store
  __shared__ int s_pos[APPEND_MAX_TOKENS];
  const PagedView& v = p.view;
  const int b = blockIdx.y, t0 = blockIdx.x * p.tokens_per_block;
  PagedSeq s;
  if (!paged_sequence(v, b, INT_MAX, &s)) return;
  if (s.L < s.T) {  // the new tokens are part of the keys
    if (threadIdx.x == 0) atomicCAS(v.status, 0, static_cast<int>(TI_ERR_PAGED_LENGTHS));
    return;
  }
  const int nt = min(p.tokens_per_block, s.T - t0);
  if (nt <= 0) return;
  if (static_cast<int>(threadIdx.x) < nt) {
    const int pos = s.L - s.T + t0 + threadIdx.x;
    const int page = paged_page(v, b, pos >> v.page_shift);
    int row = page < 0 ? -1 : (page << v.page_shift) + (pos & ((1 << v.page_shift) - 1));
    if (p.rotary != nullptr && pos >= p.rotary_rows) {
      atomicCAS(v.status, 0, static_cast<int>(TI_ERR_PAGED_LENGTHS));
      row = -1;
    }
    s_row[threadIdx.x] = row;
    s_pos[threadIdx.x] = pos;
  }
  __syncthreads();
  const int total = nt * p.units_per_token;
  const int hk = v.kv_heads, rd = p.rotary_dim;
  const long long token0 = s.q0 + t0;
  for (int base = threadIdx.x; base < total; base += APPEND_THREADS * UNITS) {
    Raw8<T> lo[UNITS], hi[UNITS];
    int tok[UNITS], which[UNITS], head[UNITS], off0[UNITS], off1[UNITS], pair0[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int idx = base + u * APPEND_THREADS;
      which[u] = -1;
      if (idx >= total) continue;
      const int t = idx / p.units_per_token;
      const int rest = idx - t * p.units_per_token;
      if (s_row[t] < 0) continue;
      const int hh = rest / PIECES, piece = rest - hh * PIECES;
      which[u] = hh < p.q_heads ? 0 : hh < p.q_heads + hk ? 1 : 2;
      head[u] = hh - (which[u] == 0 ? 0 : which[u] == 1 ? p.q_heads : p.q_heads + hk);
      tok[u] = t;
      const bool rotated = which[u] < 2 && piece * 16 < rd;
      pair0[u] = rotated ? piece * 8 : -1;
      const bool halves = rotated && !p.interleaved;
      off0[u] = halves ? piece * 8 : piece * 16;
      off1[u] = halves ? rd / 2 + piece * 8 : piece * 16 + 8;
      const T* src = static_cast<const T*>(p.src[which[u]]) + (token0 + t) * p.ld[which[u]] + head[u] * D;
      lo[u].load(src + off0[u]);
      hi[u].load(src + off1[u]);
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      if (which[u] < 0) continue;
      float x[8], y[8];
      lo[u].get(x);
      hi[u].get(y);
      if (pair0[u] >= 0) {
        const float* c = p.rotary + static_cast<long long>(s_pos[tok[u]]) * rd + pair0[u];
        const float* sn = c + rd / 2;
        float cs[8], ss[8];
        *reinterpret_cast<float4*>(cs) = __ldg(reinterpret_cast<const float4*>(c));
        *reinterpret_cast<float4*>(cs + 4) = __ldg(reinterpret_cast<const float4*>(c) + 1);
        *reinterpret_cast<float4*>(ss) = __ldg(reinterpret_cast<const float4*>(sn));
        *reinterpret_cast<float4*>(ss + 4) = __ldg(reinterpret_cast<const float4*>(sn) + 1);
        auto turn = [](float& a, float& d, float co, float si) {
          const float a1 = __fsub_rn(__fmul_rn(a, co), __fmul_rn(d, si));
          d = __fadd_rn(__fmul_rn(d, co), __fmul_rn(a, si));
          a = a1;
        };
        if (p.interleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            turn(x[2 * i], x[2 * i + 1], cs[i], ss[i]);
            turn(y[2 * i], y[2 * i + 1], cs[4 + i], ss[4 + i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) turn(x[i], y[i], cs[i], ss[i]);
        }
      }
      const float al = p.alpha[which[u]];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = __fmul_rn(x[i], al);
        y[i] = __fmul_rn(y[i], al);
      }
      const uint2 a = make_uint2(quantise4(x[0], x[1], x[2], x[3]), quantise4(x[4], x[5], x[6], x[7]));
      const uint2 d = make_uint2(quantise4(y[0], y[1], y[2], y[3]), quantise4(y[4], y[5], y[6], y[7]));
      int8_t* dst;
      if (which[u] == 0) {
        dst = p.q_out + ((token0 + tok[u]) * p.q_heads + head[u]) * D;
      } else {
        const int row = s_row[tok[u]];
        const long long page = row >> v.page_shift;
        const int in_page = row & ((1 << v.page_shift) - 1);
        dst = (which[u] == 1 ? v.k_pages : v.v_pages) + ((((page * hk) + head[u]) << v.page_shift) + in_page) * D;
      }
      if (off1[u] == off0[u] + 8) {
        *reinterpret_cast<uint4*>(dst + off0[u]) = make_uint4(a.x, a.y, d.x, d.y);
      } else {
        *reinterpret_cast<uint2*>(dst + off0[u]) = a;
        *reinterpret_cast<uint2*>(dst + off1[u]) = d;
      }
    }
  }
}

template <typename T>
void launch_append(int head_dim, dim3 grid, const AppendParams& p, cudaStream_t stream) {
  if (head_dim == 128)
    paged_append_kernel<T, 128><<<grid, APPEND_THREADS, 0, stream>>>(p);
  else if (head_dim == 80)
    paged_append_kernel<T, 80><<<grid, APPEND_THREADS, 0, stream>>>(p);
  else
    paged_append_kernel<T, 64><<<grid, APPEND_THREADS, 0, stream>>>(p);
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
  if (b.kv_heads <= 0 || b.kv_heads > 65535 || b.batch < 0 || b.batch > 65535 || b.tokens < 0 || b.tokens > 0x7FFFFFFF ||
      b.max_query_len < 0 || b.num_pages <= 0 || b.num_pages * b.page_size > 0x7FFFFFFF || b.table_width <= 0 ||
      b.table_width * b.page_size > 0x7FFFFFFF || b.table_ld < b.table_width) {
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
  // about two rounds of the loop per block, at most APPEND_MAX_TOKENS page lookups
  const int64_t max_q = b.max_query_len < b.tokens ? b.max_query_len : b.tokens;
  int64_t per_block = 2048 / p.units_per_token;
  per_block = per_block < 1 ? 1 : per_block > APPEND_MAX_TOKENS ? APPEND_MAX_TOKENS : per_block;
  p.tokens_per_block = static_cast<int>(per_block < max_q ? per_block : max_q);
  const dim3 grid(static_cast<unsigned>((max_q + p.tokens_per_block - 1) / p.tokens_per_block),
                  static_cast<unsigned>(b.batch));
  const int d = static_cast<int>(b.head_dim);
  switch (a.dtype) {
    case 0: launch_append<float>(d, grid, p, stream); break;
    case 1: launch_append<__half>(d, grid, p, stream); break;
    case 2: launch_append<__nv_bfloat16>(d, grid, p, stream); break;
    default: launch_append<int8_t>(d, grid, p, stream); break;
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error("paged_append launch failed: %s", cudaGetErrorString(e));
    return TI_E_CUDA;
  }
  return TI_OK;
}

}  // namespace ti
