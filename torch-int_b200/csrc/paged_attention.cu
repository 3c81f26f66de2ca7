// Attention of a ragged batch of new tokens over a paged int8 cache:
//   s_j = alpha_qk * float(q . k_j)   for keys j <= position of the token     (int8 products, int32 sums)
//   ctx = alpha_pv * sum_j softmax(s)_j * v_j                                 -> int8 (sat rne), fp16 or bf16
// query head h reads key head h / group, group = q_heads / kv_heads.  A row that sees no key gives 0.
//
// paged_rows_kernel serves sequences with few query rows per key head (rows = new tokens x group), decode
// above all: it is bound by the bytes of the cache, 2 * head_dim per key and key head, each read once.
//   * A CTA owns one key head, 8 * NT query rows and `chunk` keys; each of its 4 warps (3, 6 or 8 where make_plan says why)
//     takes 32 keys at a time, as two groups of 16 (a group lies in one page, in consecutive bytes).
//   * Scores transposed, S^T = K . Q^T (m16n8k32 s8, keys as rows, queries as the 8 columns), so that a single
//     query row wastes 7 of 8 columns and not 15 of 16 rows; the context likewise, O^T = V^T . P^T (m16n8k16
//     fp16).  The columns of a dot product may be taken in any order as long as both operands agree, and so may
//     the rows of O^T: the order is chosen so that a lane's fragments are 16-byte pieces of a row (V of 64- and
//     80-wide heads: 8).
//   * Groups come through a queue of the warp in shared memory (cp.async, whole lines, no registers and no barrier of
//     the block), in an order of pieces that makes the fragments' reads free of bank conflicts.  The loop is bound
//     by the latency of its own instructions, not by the depth of the queue (2, 3 and 4 groups in flight: the same):
//     hence 32 keys a step, whose two halves overlap.
//   * int8 values become fp16 exactly (byte + 1152 as the low bits of 1024.., minus 1152).
//   * Running maximum in the log2 domain per warp, raised only when an exponent s + (7 - max) passes 15 (a vote,
//     no reduction, in the common case); probabilities are 2^(s + (7 - max)) <= 2^15, split into two fp16 numbers
//     (p = hi + lo, 22 bits) whose products are summed in fp32: the tensor cores have room for the second
//     product because the loop waits for memory.
// Measured: 64 contexts of 8192 keys, 8 key heads x 128, 168 us (6.4 TB/s); 128 of 2048 83 us; 2 of 131072 88 us; 8 of 640,
// 56 heads, 14.7 us (one round of CTAs: latency).
// The keys are split over CTAs.  Up to MAX_CLUSTER splits are a cluster, whose CTAs join their partial results
// through distributed shared memory: one launch, no workspace.  More splits write them in fp32 to a workspace and
// paged_combine_kernel joins them.  Both in a fixed order, without atomics: results do not depend on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "gemm_i8.h"
#include "grid_dependency.cuh"
#include "paged.h"
#include "paged_attention.cuh"
#include "paged_plan.h"
#define TI_PTX_EXTERNAL_STATUS 1
#include "sm100_ptx.cuh"

namespace ti {
namespace {

constexpr int STAGES = 2;           // steps of a warp in shared memory: one in flight, one in use

__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 8 x 8 matrix of 16-bit elements, rows over lanes / 4 and two columns per lane, transposed across the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void copy_async16(uint32_t dst, const int8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 2^x to about 2 ulp.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// The columns of a row that lane `a` (= lane % 4) holds for a dot product: 16 bytes of each 64, and 4 bytes of
// the last 16 of an 80-wide row.
template <int D>
struct DotRow {
  static constexpr int STEPS = (D + 31) / 32;
  uint32_t w[2 * STEPS];
  __device__ __forceinline__ void put(const uint4& x, int i) { w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w; }
  __device__ __forceinline__ void load(const int8_t* row, int a) {
    put(__ldg(reinterpret_cast<const uint4*>(row + a * 16)), 0);
    if constexpr (D == 128) put(__ldg(reinterpret_cast<const uint4*>(row + 64 + a * 16)), 1);
    if constexpr (D == 80) w[4] = __ldg(reinterpret_cast<const uint32_t*>(row + 64 + a * 4)), w[5] = 0;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 2 * STEPS; ++i) w[i] = 0;
  }
};

// The columns of a value row that lane group `g` (= lane / 4) holds: D / 8 neighbours (128, 64), or 8 of the
// first 64 and 2 of the last 16 (80).  Words of four bytes; the last one of an 80-wide row has two.
template <int D>
struct ValueRow {
  static constexpr int WORDS = D == 128 ? 4 : D == 80 ? 3 : 2;
  uint32_t w[WORDS];
};
// Column of the even row of output tile i (its other row is the next column).
template <int D>
__device__ __forceinline__ int value_column(int g, int i) {
  if (D == 128) return g * 16 + 2 * i;
  return i < 4 ? g * 8 + 2 * i : 64 + 2 * g;
}

// A group of 16 keys in shared memory: rows of D bytes as in the pools, K then V.  The 16-byte pieces of a 128-byte
// row are stored in another order, so that the eight lanes that read at a time find their pieces in different banks:
// K (rows g, g + 1, pieces a) exchanges the halves of odd rows, V (rows 2a, pieces g) xors with the row's bits 1, 2;
// of the 64-byte rows of V four lanes share two rows' banks.
template <int D>
struct Group {
  static constexpr int V = 16 * D, BYTES = 2 * V;
  static __device__ __forceinline__ int key_piece(int row, int c) { return D == 128 ? c ^ ((row & 1) << 2) : c; }
  static __device__ __forceinline__ int value_piece(int row, int c) {
    return D == 128 ? c ^ (row & 6) : D == 64 ? c ^ ((row >> 1) & 3) : c;
  }
  // kp, vp: first key's row in the pools
  static __device__ __forceinline__ void fetch(uint32_t at, const int8_t* kp, const int8_t* vp, int lane) {
    constexpr int PIECES = D / 16;  // of a row
#pragma unroll
    for (int i = 0; i < (D + 31) / 32; ++i) {
      const int n = i * 32 + lane;  // 16 * PIECES in all
      if (D % 32 != 0 && n >= D) continue;
      const int row = n / PIECES, c = n - row * PIECES;
      copy_async16(at + row * D + key_piece(row, c) * 16, kp + n * 16);
      copy_async16(at + V + row * D + value_piece(row, c) * 16, vp + n * 16);
    }
  }
  static __device__ __forceinline__ void keys(const uint8_t* s, int lane, DotRow<D> (&kr)[2]) {
    const int a = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = (lane >> 2) + 8 * i;
      kr[i].put(*reinterpret_cast<const uint4*>(s + row * D + key_piece(row, a) * 16), 0);
      if constexpr (D == 128) kr[i].put(*reinterpret_cast<const uint4*>(s + row * D + key_piece(row, 4 + a) * 16), 1);
      if constexpr (D == 80) kr[i].w[4] = *reinterpret_cast<const uint32_t*>(s + row * D + 64 + a * 4), kr[i].w[5] = 0;
    }
  }
  static __device__ __forceinline__ void values(const uint8_t* s, int lane, ValueRow<D> (&vr)[4]) {
    const int g = lane >> 2;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = 2 * (lane & 3) + (j & 1) + 8 * (j >> 1);
      const uint8_t* r = s + V + row * D;
      if constexpr (D == 128) {
        const uint4 x = *reinterpret_cast<const uint4*>(r + value_piece(row, g) * 16);
        vr[j].w[0] = x.x, vr[j].w[1] = x.y, vr[j].w[2] = x.z, vr[j].w[3] = x.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(r + value_piece(row, g >> 1) * 16 + (g & 1) * 8);
        vr[j].w[0] = x.x, vr[j].w[1] = x.y;
        if constexpr (D == 80) vr[j].w[2] = *reinterpret_cast<const uint16_t*>(r + 64 + g * 2);
      }
    }
  }
};

// Bytes (lo, hi byte pairs of two rows) -> fp16 pairs, exactly.
__device__ __forceinline__ uint32_t halves_of(uint32_t x, uint32_t sel) {
  const uint32_t h = __byte_perm(x, 0x64646464u, sel);  // 1024 + (byte ^ 0x80)
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Shared memory of a rows CTA: the warps' queues; when they are empty, the warps' contexts and what they join to.
template <int D, int NT, int WARPS>
struct RowsSmem {
  static constexpr int R = 8 * NT, LDO = D + 4;
  static constexpr int STAGE = 2 * Group<D>::BYTES, QUEUE = WARPS * STAGES * STAGE;
  static constexpr int JOINED = WARPS * R * LDO * 4;          // fp32 [R][D]
  static constexpr int BYTES = QUEUE > JOINED + R * D * 4 ? QUEUE : JOINED + R * D * 4;
};

__device__ __forceinline__ float4 ld_cluster16(uint32_t addr) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ float2 ld_cluster8(uint32_t addr) {
  float2 x;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(addr) : "memory");
  return x;
}

template <int D, int NT, int WARPS>
__device__ __forceinline__ void rows_of_a_cta(const PagedAttnParams& p) {
  using SM = RowsSmem<D, NT, WARPS>;
  constexpr int R = SM::R, LDO = SM::LDO;
  constexpr int MT = D / 16;  // 16-row tiles of O^T
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float s_m[WARPS][R], s_l[WARPS][R];
  __shared__ float2 s_ml[R];
  float(*s_o)[R][LDO] = reinterpret_cast<float(*)[R][LDO]>(smem);
  float* s_join = reinterpret_cast<float*>(smem + SM::JOINED);
  const PagedView& v = p.view;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, a = lane & 3;
  const int tile = p.first_tile + blockIdx.z, b = tile / p.row_tiles, rt = tile % p.row_tiles, h = blockIdx.y, split = blockIdx.x;
  // the first entries of the block table are loaded beside the lengths, not behind them (one latency less)
  const unsigned first_page = static_cast<unsigned>(split * p.chunk + (warp + WARPS * (lane >> 1)) * STEP + (lane & 1) * 16) >> v.page_shift;
  const int first_entry = first_page < static_cast<unsigned>(v.table_width) ? v.table[b * v.table_ld + first_page] : -1;
  PagedSeq s;
  if (!paged_sequence(v, b, p.max_kv_len, &s)) return;  // (returns before the keys are looked at: a whole cluster's)
  const int G = p.group, rows = s.T * G, r0 = rt * R;
  if (r0 >= rows || rows > p.rows_below) return;
  const int past = s.L - s.T;
  const PagedSplits sp = paged_splits(past + (min(r0 + R, rows) - 1) / G + 1, p.chunk);
  if (split >= sp.n && (!p.cluster || sp.n == 1)) return;
  const int k0 = min(split * p.chunk, sp.keys), k1 = min(k0 + p.chunk, sp.keys);

  // this warp's steps: keys k0 + (warp + WARPS * i) * STEP, i < cnt; lane n knows the page of group n of 32
  const int steps = (k1 - k0 + STEP - 1) / STEP;
  const int cnt = steps > warp ? (steps - warp + WARPS - 1) / WARPS : 0;
  const uint32_t queue = smem_u32(smem) + warp * STAGES * SM::STAGE;
  int my_page = 0;
  auto fetch = [&](int i) {  // in order, every i < cnt once
    if (i < cnt) {
      if ((i & 15) == 0) {
        const int key = k0 + (warp + WARPS * (i + (lane >> 1))) * STEP + (lane & 1) * 16;
        my_page = 0;
        if (key < k1) my_page = max(0, i == 0 ? paged_checked(v, first_entry) : paged_page(v, b, key >> v.page_shift));
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int key = k0 + (warp + WARPS * i) * STEP + n * 16;
        const long long page = __shfl_sync(0xffffffffu, my_page, (i & 15) * 2 + n);
        const long long at = (((page * v.kv_heads + h) << v.page_shift) + (key & ((1 << v.page_shift) - 1))) * D;
        if (key < k1)
          Group<D>::fetch(queue + (i % STAGES) * SM::STAGE + n * Group<D>::BYTES, v.k_pages + at, v.v_pages + at, lane);
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(i);

  // query fragments and limits
  DotRow<D> qf[NT];
  int lim[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + n * 8 + g;
    qf[n].zero();
    if (r < rows) qf[n].load(p.q + static_cast<long long>(s.q0 + r / G) * p.ld_q + (h * G + r % G) * D, a);
#pragma unroll
    for (int i = 0; i < 2; ++i) lim[n][i] = past + min(r0 + n * 8 + 2 * a + i, rows - 1) / G;
  }
  const int lim_min = past + r0 / G;

  float o[NT][MT][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[n][i][c] = 0.f;
    m[n][0] = m[n][1] = -1e30f;
    l[n][0] = l[n][1] = 0.f;
  }
#pragma unroll 1
  for (int i = 0; i < cnt; ++i) {
    const int key = k0 + (warp + WARPS * i) * STEP;
    const uint8_t* stage = smem + (warp * STAGES + i % STAGES) * SM::STAGE;
    copy_wait<STAGES - 2>();
    __syncwarp();  // step i has landed, and every lane is done with the one whose place the next fetch takes
    fetch(i + STAGES - 1);
    // scores (log2 domain): columns 2a, 2a + 1 are queries, rows g, g + 8 keys of a group
    float sc[2][NT][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      DotRow<D> kr[2];
      Group<D>::keys(stage + u * Group<D>::BYTES, lane, kr);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        int acc[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < DotRow<D>::STEPS; ++k) {
          const uint32_t fa[4] = {kr[0].w[2 * k], kr[1].w[2 * k], kr[0].w[2 * k + 1], kr[1].w[2 * k + 1]};
          mma_s8(acc, fa, qf[n].w[2 * k], qf[n].w[2 * k + 1]);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) sc[u][n][c] = __fmul_rn(static_cast<float>(acc[c]), p.scale_log2);  // (not contracted: `raise` relies on it)
      }
    }
    if (key + STEP - 1 > lim_min) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (key + u * 16 + g + (c >> 1) * 8 > lim[n][c & 1]) sc[u][n][c] = -INFINITY;
    }
    float top[NT][2];
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[n][c] = fmaxf(fmaxf(sc[0][n][c], sc[0][n][c + 2]), fmaxf(sc[1][n][c], sc[1][n][c + 2]));
        raise |= top[n][c] + (7.f - m[n][c]) > 15.f;  // the sum that the exponents below are, rounded alike
      }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(m[n][c], top[n][c]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float corr = ex2(m[n][c] - mx);
          m[n][c] = mx;
          l[n][c] *= corr;
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            o[n][t][c] *= corr;
            o[n][t][c + 2] *= corr;
          }
        }
      }
    }
    uint32_t ph[2][NT][2], pl[2][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float base[2] = {7.f - m[n][0], 7.f - m[n][1]};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float e[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          e[c] = ex2(sc[u][n][c] + base[c & 1]);
          l[n][c & 1] += e[c];
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const __half2 hi = __floats2half2_rn(e[2 * c], e[2 * c + 1]);
          const float2 back = __half22float2(hi);
          const __half2 lo = __floats2half2_rn(e[2 * c] - back.x, e[2 * c + 1] - back.y);
          ph[u][n][c] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hi));
          pl[u][n][c] = transpose8x8(*reinterpret_cast<const uint32_t*>(&lo));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      ValueRow<D> vc[4];
      Group<D>::values(stage + u * Group<D>::BYTES, lane, vc);
#pragma unroll
      for (int w = 0; w < ValueRow<D>::WORDS; ++w) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int t = 2 * w + half;
          if (t >= MT) continue;
          const uint32_t pick = half ? 0x7362u : 0x5140u;
          const uint32_t x01 = __byte_perm(vc[0].w[w], vc[1].w[w], pick) ^ 0x80808080u;
          const uint32_t x23 = __byte_perm(vc[2].w[w], vc[3].w[w], pick) ^ 0x80808080u;
          const uint32_t fa[4] = {halves_of(x01, 0x4140), halves_of(x01, 0x4342), halves_of(x23, 0x4140),
                                  halves_of(x23, 0x4342)};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_f16(o[n][t], fa, ph[u][n][0], ph[u][n][1]);
            mma_f16(o[n][t], fa, pl[u][n][0], pl[u][n][1]);
          }
        }
      }
    }
  }
  // ---- join the warps: each had its own maximum
  copy_wait<0>();
  __syncthreads();  // the queues are empty: their memory is used again
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], d);
      const int r = n * 8 + 2 * a + c;
      if (g == 0) {
        s_m[warp][r] = m[n][c];
        s_l[warp][r] = l[n][c];
      }
      if (r0 + r < rows) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
          *reinterpret_cast<float2*>(&s_o[warp][r][value_column<D>(g, t)]) = make_float2(o[n][t][c], o[n][t][c + 2]);
      }
    }
  }
  __syncthreads();
  const int work = min(R, rows - r0) * (D / 4);
  for (int i = threadIdx.x; i < work; i += WARPS * 32) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4, row = r0 + r;
    float mx = s_m[0][r];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) mx = fmaxf(mx, s_m[w][r]);
    float sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = exp2f(s_m[w][r] - mx);
      const float4 y = *reinterpret_cast<const float4*>(&s_o[w][r][d]);
      sum += f * s_l[w][r];
      x.x += f * y.x;
      x.y += f * y.y;
      x.z += f * y.z;
      x.w += f * y.w;
    }
    const long long at = static_cast<long long>(s.q0 + row / G) * p.q_heads + h * G + row % G;
    if (sp.n == 1) {
      paged_store4(p, at * D + d, x, sum > 0.f ? p.alpha_pv / sum : 0.f);
    } else if (p.cluster) {
      *reinterpret_cast<float4*>(s_join + r * D + d) = x;
      if (d == 0) s_ml[r] = make_float2(mx, sum);
    } else {
      *reinterpret_cast<float4*>(p.part_o + (at * p.max_splits + split) * D + d) = x;
      if (d == 0) p.part_ml[at * p.max_splits + split] = make_float2(mx, sum);
    }
  }
  if (sp.n == 1 || !p.cluster) return;
  // ---- join the splits of the cluster (rank = split), each CTA a part of the rows and columns
  cluster_sync_all();
  const uint32_t join_at = smem_u32(s_join), ml_at = smem_u32(s_ml);
  for (int i = split * WARPS * 32 + threadIdx.x; i < work; i += static_cast<int>(gridDim.x) * WARPS * 32) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4, row = r0 + r;
    float mx = -1e30f, sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    float2 ml[MAX_CLUSTER];
    float4 y[MAX_CLUSTER];
#pragma unroll
    for (int c = 0; c < MAX_CLUSTER; ++c) {
      if (c >= sp.n) continue;
      ml[c] = ld_cluster8(mapa_shared(ml_at + r * 8, c));
      y[c] = ld_cluster16(mapa_shared(join_at + (r * D + d) * 4, c));
      mx = fmaxf(mx, ml[c].x);
    }
#pragma unroll
    for (int c = 0; c < MAX_CLUSTER; ++c) {
      if (c >= sp.n) continue;
      const float f = exp2f(ml[c].x - mx);
      sum += f * ml[c].y;
      x.x += f * y[c].x;
      x.y += f * y[c].y;
      x.z += f * y[c].z;
      x.w += f * y[c].w;
    }
    const long long at = static_cast<long long>(s.q0 + row / G) * p.q_heads + h * G + row % G;
    paged_store4(p, at * D + d, x, sum > 0.f ? p.alpha_pv / sum : 0.f);
  }
  cluster_sync_all();  // the others may still read this CTA's part
}

// Launched as a programmatic dependent: of whatever comes before, which it waits for; or of the tile kernel of the
// same call, beside which it runs on the SMs that kernel leaves free (their rows are different sequences').  Then only
// its last CTA waits, at its end: the call is complete when this kernel is.
template <int D, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, rows_ctas_per_sm(D, NT, WARPS)) paged_rows_kernel(const PagedAttnParams p) {
  grid_dep_launch();
  if (!p.beside_tiles) grid_dep_wait();
  rows_of_a_cta<D, NT, WARPS>(p);
  if (p.beside_tiles && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1)
    grid_dep_wait();
}

// Joins the partial contexts of the splits of a row = (token, query head).  A block has 4 / W rows; W = 4 warps share a
// row's splits where there are many (a single warp took 14 us for 56 splits, most of it waiting for its loads), W = 1
// has one warp for each row (16384 rows of two splits: 39 us -> 12).  blockIdx.y is the sequence and the row one of
// it, or - by_token - the row is one of the call and the warp looks its sequence up.
template <int D, int W>
__global__ void __launch_bounds__(128) paged_combine_kernel(const PagedAttnParams p, int few_rows, int many_rows,
                                                            int many_chunk, bool by_token) {
  __shared__ float4 s_x[4][32];
  __shared__ float s_m[4], s_l[4];
  const PagedView& v = p.view;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = W == 1 ? 0 : warp;
  const unsigned row = W == 1 ? blockIdx.x * 4 + warp : blockIdx.x;
  const int head = row % p.q_heads;
  int t = row / p.q_heads, b = blockIdx.y;
  // The lengths too are read behind the wait: the rows kernel lets this one start before it has itself waited for whoever
  // wrote them.
  grid_dep_wait();
  if (by_token) {
    b = -1;
    for (int i = lane; i < v.batch; i += 32) {
      const int q0 = v.query_starts[i], q1 = v.query_starts[i + 1];
      if (q0 >= 0 && q0 <= t && t < q1 && q1 <= v.tokens && q1 - q0 <= v.max_query_len) b = i;
    }
    b = __reduce_max_sync(0xffffffffu, b);
  }
  PagedSeq s;
  if (b < 0 || !paged_sequence(v, b, p.max_kv_len, &s)) return;
  if (by_token) t -= s.q0;
  if (t >= s.T) return;
  // the row tile this row belonged to decides how many keys, hence splits, were visited
  const int G = p.group, rows = s.T * G;
  const bool many = rows > p.rows_below;
  const int R = many ? many_rows : few_rows;
  const int r = t * G + head % G;
  const PagedSplits sp = paged_splits(s.L - s.T + (min((r / R + 1) * R, rows) - 1) / G + 1, many ? many_chunk : p.chunk);
  if (sp.n == 1 || (!many && p.cluster)) return;  // written by the attention kernel
  const long long at = static_cast<long long>(s.q0 + t) * p.q_heads + head;
  const float2* ml = p.part_ml + at * p.max_splits;
  const int d = lane * 4;
  const bool mine = d < D;
  const float* po = p.part_o + at * p.max_splits * D + (mine ? d : 0);
  float mx = -1e30f, sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int BATCH = 8;  // splits whose loads are in flight together
  for (int i0 = part; i0 < sp.n; i0 += W * BATCH) {
    float2 e[BATCH];
    float4 y[BATCH];
    float top = mx;
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int i = min(i0 + W * k, sp.n - 1);
      const bool there = i0 + W * k < sp.n;
      y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (W > 1 || there) {  // (with many splits a load too many costs less than a branch)
        e[k] = ml[i];
        y[k] = *reinterpret_cast<const float4*>(po + static_cast<long long>(i) * D);
      }
      if (!there) e[k] = make_float2(-1e30f, 0.f);
    }
#pragma unroll
    for (int k = 0; k < BATCH; ++k) top = fmaxf(top, e[k].x);
    const float corr = exp2f(mx - top);
    mx = top;
    sum *= corr;
    x.x *= corr;
    x.y *= corr;
    x.z *= corr;
    x.w *= corr;
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const float f = i0 + W * k < sp.n ? exp2f(e[k].x - mx) : 0.f;
      sum += f * e[k].y;
      x.x += f * y[k].x;
      x.y += f * y[k].y;
      x.z += f * y[k].z;
      x.w += f * y[k].w;
    }
  }
  if constexpr (W > 1) {
    s_x[warp][lane] = x;
    if (lane == 0) {
      s_m[warp] = mx;
      s_l[warp] = sum;
    }
    __syncthreads();
    if (warp != 0) return;
    mx = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    sum = 0.f;
    x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2f(s_m[w] - mx);
      const float4 y = s_x[w][lane];
      sum += f * s_l[w];
      x.x += f * y.x;
      x.y += f * y.y;
      x.z += f * y.z;
      x.w += f * y.w;
    }
  }
  if (mine) paged_store4(p, at * D + d, x, sum > 0.f ? p.alpha_pv / sum : 0.f);
}

constexpr int64_t MAX_GRID_Z = 65535;

template <int D, int NT, int WARPS>
cudaError_t launch_rows(const PagedBatch& b, PagedAttnParams p, const PagedPlan& pl, cudaStream_t stream) {
  auto kernel = paged_rows_kernel<D, NT, WARPS>;
  constexpr int smem = RowsSmem<D, NT, WARPS>::BYTES;
  static PagedOncePerDevice once;
  cudaError_t e = once.run([kernel] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(pl.row_splits);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pl.cluster ? 2 : 1;
  const int64_t tiles = b.batch * pl.row_tiles;
  for (int64_t first = 0; first < tiles && e == cudaSuccess; first += MAX_GRID_Z) {
    p.first_tile = static_cast<int>(first);
    cfg.gridDim = dim3(static_cast<unsigned>(pl.row_splits), static_cast<unsigned>(b.kv_heads),
                       static_cast<unsigned>(tiles - first < MAX_GRID_Z ? tiles - first : MAX_GRID_Z));
    e = cudaLaunchKernelEx(&cfg, kernel, p);
  }
  return e;
}

template <int D>
int launch(const PagedBatch& b, const PagedAttnParams& p, const PagedPlan& pl, cudaStream_t stream) {
  if (pl.tiles) {
    const int rc = launch_paged_tiles(b, p, pl.tile, stream);
    if (rc != TI_OK) return rc;
  }
  cudaError_t e = cudaSuccess;
  if (pl.rows)
    e = pl.warps == 3   ? launch_rows<D, 1, 3>(b, p, pl, stream)
        : pl.warps == 6 ? launch_rows<D, 1, D == 128 ? 6 : 8>(b, p, pl, stream)
        : pl.warps == 8 ? (pl.nt == 1 ? launch_rows<D, 1, 8>(b, p, pl, stream) : launch_rows<D, 2, 8>(b, p, pl, stream))
        : pl.nt == 1    ? launch_rows<D, 1, 4>(b, p, pl, stream)
                        : launch_rows<D, 2, 4>(b, p, pl, stream);
  if (e == cudaSuccess && pl.splits > 1) {
    cudaLaunchConfig_t cfg = {};
    const PagedJoin join = plan_join(pl, b.batch, b.tokens, p.q_heads, p.group, b.max_query_len);
    cfg.gridDim = dim3(static_cast<unsigned>(join.blocks), static_cast<unsigned>(join.by_token ? 1 : b.batch));
    cfg.blockDim = dim3(128);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, join.many ? paged_combine_kernel<D, 4> : paged_combine_kernel<D, 1>, p, 8 * pl.nt,
                           2 * pl.tile.tokens_per_tile * p.group, pl.tile.chunk, join.by_token);
  }
  if (e != cudaSuccess) {
    set_error("paged_attention launch failed: %s", cudaGetErrorString(e));
    return TI_E_CUDA;
  }
  return TI_OK;
}

}  // namespace

int64_t paged_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                                        int64_t head_dim, int64_t max_query_len, int64_t max_kv_len) {
  // none for calls without tokens or keys, and for sizes that paged_attention refuses
  if (batch <= 0 || batch > 65535 || tokens <= 0 || tokens > 0x7FFFFFFF || kv_heads <= 0 || q_heads <= 0 || q_heads > 65535 ||
      q_heads % kv_heads != 0 || (head_dim != 64 && head_dim != 80 && head_dim != 128) || max_query_len <= 0 ||
      max_kv_len <= 0 || max_kv_len > MAX_KEYS)
    return 0;
  if (max_query_len > tokens) max_query_len = tokens;
  const PagedPlan pl = make_plan(batch, tokens, q_heads / kv_heads, kv_heads, static_cast<int>(head_dim), max_query_len, max_kv_len);
  return partial_bytes(pl, tokens, q_heads, head_dim);
}

int paged_attention(const PagedBatch& b0, const PagedAttention& a, cudaStream_t stream) {
  int rc = check_paged_batch(b0, "paged_attention");
  if (rc != TI_OK) return rc;
  PagedBatch b = b0;
  if (b.max_query_len > b.tokens) b.max_query_len = b.tokens;
  if (a.q_heads <= 0 || a.q_heads > 65535 || a.q_heads % b.kv_heads != 0) {
    set_error("paged_attention: the query heads (%lld) must be a multiple of the key heads (%lld)", (long long)a.q_heads,
              (long long)b.kv_heads);
    return TI_E_INVALID;
  }
  if (a.out_kind < 1 || a.out_kind > 3) {
    set_error("paged_attention: the output must be int8, fp16 or bf16");
    return TI_E_INVALID;
  }
  if (a.max_kv_len < 0 || a.max_kv_len > MAX_KEYS) {
    set_error("paged_attention: max_kv_len must be from 0 to %lld (got %lld)", (long long)MAX_KEYS, (long long)a.max_kv_len);
    return TI_E_INVALID;
  }
  if (!(fabsf(a.alpha_qk) <= 1e20f) || !(fabsf(a.alpha_pv) <= 1e20f)) {  // the running maximum starts at -1e30
    set_error("paged_attention: alpha_qk and alpha_pv must be finite, of at most 1e20");
    return TI_E_INVALID;
  }
  if (b.batch == 0 || b.tokens == 0 || b.max_query_len == 0) return TI_OK;
  if (!a.q || !a.out) {
    set_error("paged_attention: null pointer");
    return TI_E_INVALID;
  }
  if (((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) & 15) != 0 ||
      (b.tokens > 1 && (a.ld_q % 16 != 0 || a.ld_q < a.q_heads * b.head_dim))) {
    set_error("paged_attention: query rows must be 16-byte aligned and hold their heads side by side");
    return TI_E_INVALID;
  }
  const int64_t group = a.q_heads / b.kv_heads;
  const float scale_log2 = static_cast<float>(static_cast<double>(a.alpha_qk) * 1.4426950408889634);
  const PagedPlan pl = make_plan_for_scale(b.batch, b.tokens, group, b.kv_heads, static_cast<int>(b.head_dim), b.max_query_len,
                                           a.max_kv_len, scale_log2);
  if (b.batch * static_cast<int64_t>(pl.row_tiles) > 0x7FFFFFFF - MAX_GRID_Z || b.max_query_len * a.q_heads > 0x7FFFFFFF) {
    set_error("paged_attention: batch %lld x %lld new tokens is too large for one call", (long long)b.batch,
              (long long)b.max_query_len);
    return TI_E_INVALID;
  }
  const int64_t need = partial_bytes(pl, b.tokens, a.q_heads, b.head_dim);
  if (need > a.workspace_bytes || (need > 0 && (a.workspace == nullptr || (reinterpret_cast<uintptr_t>(a.workspace) & 15) != 0))) {
    set_error("paged_attention: needs a 16-byte aligned workspace of %lld bytes (got %lld)", (long long)need,
              (long long)a.workspace_bytes);
    return TI_E_WORKSPACE;
  }
  int* status = status_word_ptr();
  if (!status) {
    set_error("paged_attention: cannot resolve the device status word");
    return TI_E_CUDA;
  }
  PagedAttnParams p;
  p.view = make_paged_view(b, status);
  p.q = a.q;
  p.ld_q = b.tokens > 1 ? a.ld_q : a.q_heads * b.head_dim;  // (of one token no stride is read, but the tensor map has one)
  p.q_heads = static_cast<int>(a.q_heads);
  p.group = static_cast<int>(group);
  p.max_kv_len = static_cast<int>(a.max_kv_len);
  p.scale_log2 = scale_log2;
  p.alpha_pv = a.alpha_pv;
  p.out = a.out;
  p.out_kind = a.out_kind;
  p.row_tiles = pl.row_tiles;
  p.chunk = pl.chunk;
  p.max_splits = pl.splits;
  p.cluster = pl.cluster;
  p.beside_tiles = pl.tiles && pl.rows;
  p.rows_below = pl.tiles ? pl.few : 0x7FFFFFFF;
  if (!pl.rows) p.rows_below = 0;
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + b.tokens * a.q_heads * pl.splits * b.head_dim);
  switch (b.head_dim) {
    case 128: return launch<128>(b, p, pl, stream);
    case 80: return launch<80>(b, p, pl, stream);
    default: return launch<64>(b, p, pl, stream);
  }
}

}  // namespace ti
