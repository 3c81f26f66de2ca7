// Attention of a ragged batch of new tokens over a paged int8 cache:
//   s_j = alpha_qk * float(q . k_j)   for keys j <= position of the token     (int8 products, int32 sums)
//   ctx = alpha_pv * sum_j softmax(s)_j * v_j                                 -> int8 (sat rne), fp16 or bf16
// query head h reads key head h / group, group = q_heads / kv_heads.  A row that sees no key gives 0.
//
// paged_rows_kernel serves sequences with few query rows per key head (rows = new tokens x group), decode
// above all: it is bound by the bytes of the cache, 2 * head_dim per key and key head, each read once.
//   * A CTA owns one key head, 8 * NT query rows and `chunk` keys; its warps take 16 keys at a time.
//   * Scores transposed, S^T = K . Q^T (m16n8k32 s8, keys as rows, queries as the 8 columns), so that a single
//     query row wastes 7 of 8 columns and not 15 of 16 rows; the context likewise, O^T = V^T . P^T (m16n8k16
//     fp16).  The columns of a dot product may be taken in any order as long as both operands agree, and so may
//     the rows of O^T: the order is chosen so that each lane loads its fragments straight from the pools with
//     16-byte (V of 64- and 80-wide heads: 8-byte) loads that use every sector they touch; no shared memory
//     and no barrier in the loop, one group of keys is in flight while the one before is multiplied.
//   * int8 values become fp16 exactly (byte + 1152 as the low bits of 1024.., minus 1152).
//   * Running maximum in the log2 domain per warp, raised only when a score exceeds it by more than 8 (a vote,
//     no reduction, in the common case); probabilities are 2^(s - max + 7) <= 2^15, split into two fp16 numbers
//     (p = hi + lo, 22 bits) whose products are summed in fp32: the tensor cores have room for the second
//     product because the loop waits for memory.
// The keys are split over CTAs; each writes its unnormalised context, maximum and sum in fp32, and
// paged_combine_kernel joins them in a fixed order (no atomics: results do not depend on timing).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "gemm_i8.h"
#include "grid_dependency.cuh"
#include "paged.h"
#include "paged_attention.cuh"

namespace ti {
namespace {

constexpr int ROWS_WARPS = 4;
constexpr int ROWS_THREADS = ROWS_WARPS * 32;
constexpr int MAX_CHUNK = 32 * ROWS_WARPS * 16;  // a lane holds the page of one of its warp's key groups

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
// Streaming loads: every byte of the cache is read by one warp only.
__device__ __forceinline__ uint4 ld_stream16(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_stream8(const int8_t* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_stream4(const int8_t* p) {
  uint32_t v;
  asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

// The columns of a row that lane `a` (= lane % 4) holds for a dot product: 16 bytes of each 64, and 4 bytes of
// the last 16 of an 80-wide row.
template <int D>
struct DotRow {
  static constexpr int WORDS = D / 16;
  static constexpr int STEPS = (D + 31) / 32;
  uint32_t w[2 * STEPS];
  __device__ __forceinline__ void load(const int8_t* row, int a) {
    const uint4 x = ld_stream16(row + a * 16);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    if constexpr (D == 128) {
      const uint4 y = ld_stream16(row + 64 + a * 16);
      w[4] = y.x, w[5] = y.y, w[6] = y.z, w[7] = y.w;
    } else if constexpr (D == 80) {
      w[4] = ld_stream4(row + 64 + a * 4);
      w[5] = 0;
    }
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
  __device__ __forceinline__ void load(const int8_t* row, int g) {
    if constexpr (D == 128) {
      const uint4 x = ld_stream16(row + g * 16);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
      const uint2 x = ld_stream8(row + g * 8);
      w[0] = x.x, w[1] = x.y;
      if constexpr (D == 80) w[2] = __ldg(reinterpret_cast<const uint16_t*>(row + 64 + g * 2));
    }
  }
};
// Column of the even row of output tile i (its other row is the next column).
template <int D>
__device__ __forceinline__ int value_column(int g, int i) {
  if (D == 128) return g * 16 + 2 * i;
  return i < 4 ? g * 8 + 2 * i : 64 + 2 * g;
}

// Bytes (lo, hi byte pairs of two rows) -> fp16 pairs, exactly.
__device__ __forceinline__ uint32_t halves_of(uint32_t x, uint32_t sel) {
  const uint32_t h = __byte_perm(x, 0x64646464u, sel);  // 1024 + (byte ^ 0x80)
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <int D, int NT>
__global__ void __launch_bounds__(ROWS_THREADS, NT == 1 ? 4 : 2) paged_rows_kernel(const PagedAttnParams p) {
  constexpr int R = 8 * NT;
  constexpr int MT = D / 16;  // 16-row tiles of O^T
  constexpr int LDO = D + 4;
  __shared__ __align__(16) float s_o[ROWS_WARPS][R][LDO];
  __shared__ float s_m[ROWS_WARPS][R], s_l[ROWS_WARPS][R];
  const PagedView& v = p.view;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, a = lane & 3;
  const int b = blockIdx.z / p.row_tiles, rt = blockIdx.z % p.row_tiles, h = blockIdx.y, split = blockIdx.x;
  PagedSeq s;
  grid_dep_launch();
  if (!paged_sequence(v, b, p.max_kv_len, &s)) return;
  const int G = p.group, rows = s.T * G, r0 = rt * R;
  if (r0 >= rows || rows > p.rows_below) return;
  const int past = s.L - s.T;
  const PagedSplits sp = paged_splits(past + (min(r0 + R, rows) - 1) / G + 1, p.chunk);
  if (split >= sp.n) return;
  const int k0 = split * p.chunk, k1 = min(k0 + p.chunk, sp.keys);

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

  // this warp's key groups: k0 + (warp + ROWS_WARPS * i) * 16, i < cnt; lane i knows the page of group i
  const int groups = (k1 - k0 + 15) >> 4;
  const int cnt = groups > warp ? (groups - warp + ROWS_WARPS - 1) / ROWS_WARPS : 0;
  int my_page = 0;
  if (lane < cnt) my_page = max(0, paged_page(v, b, (k0 + (warp + ROWS_WARPS * lane) * 16) >> v.page_shift));

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
  DotRow<D> kr[2];
  ValueRow<D> vr[4];
  auto fetch = [&](int i) {
    const int key = k0 + (warp + ROWS_WARPS * i) * 16;
    const long long page = __shfl_sync(0xffffffffu, my_page, i);
    const long long at = (((page * v.kv_heads + h) << v.page_shift) + (key & ((1 << v.page_shift) - 1))) * D;
    const int8_t* kp = v.k_pages + at;
    const int8_t* vp = v.v_pages + at;
    kr[0].load(kp + g * D, a);
    kr[1].load(kp + (g + 8) * D, a);
    vr[0].load(vp + (2 * a) * D, g);
    vr[1].load(vp + (2 * a + 1) * D, g);
    vr[2].load(vp + (2 * a + 8) * D, g);
    vr[3].load(vp + (2 * a + 9) * D, g);
  };
  if (cnt > 0) fetch(0);
#pragma unroll 1
  for (int i = 0; i < cnt; ++i) {
    const int key = k0 + (warp + ROWS_WARPS * i) * 16;
    int acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0;
#pragma unroll
      for (int k = 0; k < DotRow<D>::STEPS; ++k) {
        const uint32_t fa[4] = {kr[0].w[2 * k], kr[1].w[2 * k], kr[0].w[2 * k + 1], kr[1].w[2 * k + 1]};
        mma_s8(acc[n], fa, qf[n].w[2 * k], qf[n].w[2 * k + 1]);
      }
    }
    ValueRow<D> vc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) vc[j] = vr[j];
    if (i + 1 < cnt) fetch(i + 1);
    // scores (log2 domain): columns 2a, 2a + 1 are queries, rows g, g + 8 keys
    float sc[NT][4];
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 4; ++c) sc[n][c] = static_cast<float>(acc[n][c]) * p.scale_log2;
      if (key + 15 > lim_min) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (key + g + (c >> 1) * 8 > lim[n][c & 1]) sc[n][c] = -INFINITY;
      }
      raise |= fmaxf(sc[n][0], sc[n][2]) > m[n][0] + 8.f || fmaxf(sc[n][1], sc[n][3]) > m[n][1] + 8.f;
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(m[n][c], fmaxf(sc[n][c], sc[n][c + 2]));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float corr = exp2f(m[n][c] - mx);
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
    uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float e[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        e[c] = exp2f(sc[n][c] - m[n][c & 1] + 7.f);
        l[n][c & 1] += e[c];
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const __half2 hi = __floats2half2_rn(e[2 * c], e[2 * c + 1]);
        const float2 back = __half22float2(hi);
        const __half2 lo = __floats2half2_rn(e[2 * c] - back.x, e[2 * c + 1] - back.y);
        ph[n][c] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hi));
        pl[n][c] = transpose8x8(*reinterpret_cast<const uint32_t*>(&lo));
      }
    }
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
          mma_f16(o[n][t], fa, ph[n][0], ph[n][1]);
          mma_f16(o[n][t], fa, pl[n][0], pl[n][1]);
        }
      }
    }
  }
  // ---- join the warps: each had its own maximum
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
#pragma unroll
      for (int t = 0; t < MT; ++t)
        *reinterpret_cast<float2*>(&s_o[warp][r][value_column<D>(g, t)]) = make_float2(o[n][t][c], o[n][t][c + 2]);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * (D / 4); i += ROWS_THREADS) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4, row = r0 + r;
    if (row >= rows) break;
    float mx = s_m[0][r];
#pragma unroll
    for (int w = 1; w < ROWS_WARPS; ++w) mx = fmaxf(mx, s_m[w][r]);
    float sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < ROWS_WARPS; ++w) {
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
    } else {
      *reinterpret_cast<float4*>(p.part_o + (at * p.max_splits + split) * D + d) = x;
      if (d == 0) p.part_ml[at * p.max_splits + split] = make_float2(mx, sum);
    }
  }
}

// One warp per (token, query head): joins the partial contexts of the row's splits, in order.
template <int D>
__global__ void __launch_bounds__(128) paged_combine_kernel(const PagedAttnParams p, int few_rows, int many_rows,
                                                            int many_chunk) {
  const PagedView& v = p.view;
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5);  // (token, head) of the sequence
  PagedSeq s;
  const bool ok = paged_sequence(v, b, p.max_kv_len, &s);
  grid_dep_wait();
  const int t = row / p.q_heads, head = row % p.q_heads;
  if (!ok || t >= s.T) return;
  // the row tile this row belonged to decides how many keys, hence splits, were visited
  const int G = p.group, rows = s.T * G;
  const bool many = rows > p.rows_below;
  const int R = many ? many_rows : few_rows;
  const int r = t * G + head % G;
  const PagedSplits sp = paged_splits(s.L - s.T + (min((r / R + 1) * R, rows) - 1) / G + 1, many ? many_chunk : p.chunk);
  if (sp.n == 1) return;  // written by the attention kernel
  const long long at = static_cast<long long>(s.q0 + t) * p.q_heads + head;
  const float2* ml = p.part_ml + at * p.max_splits;
  float mx = -1e30f;
  for (int i = lane; i < sp.n; i += 32) mx = fmaxf(mx, ml[i].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  const int d = lane * 4;
  const bool mine = d < D;
  const float* po = p.part_o + at * p.max_splits * D + d;
  float sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = 0; i < sp.n; ++i) {
    const float2 e = ml[i];
    const float f = exp2f(e.x - mx);
    const float4 y = mine ? *reinterpret_cast<const float4*>(po + static_cast<long long>(i) * D) : x;
    sum += f * e.y;
    x.x += f * y.x;
    x.y += f * y.y;
    x.z += f * y.z;
    x.w += f * y.w;
  }
  if (mine) paged_store4(p, at * D + d, x, sum > 0.f ? p.alpha_pv / sum : 0.f);
}

constexpr int TILE_ROWS = 128;  // rows of a row tile of paged_tiles_kernel
constexpr int FEW_ROWS = 16;    // rows up to which a sequence is served by paged_rows_kernel

// How a call is cut.  Sequences with at most `few` rows per key head are served by paged_rows_kernel, the others by
// paged_tiles_kernel; a kernel is left out where the bounds show that no sequence needs it.
struct Plan {
  bool rows, tiles;
  int few;
  int nt, row_tiles, chunk, row_splits;  // rows kernel: 8-row tiles of a CTA, CTAs of a sequence, keys of a split
  PagedTilePlan tile;
  int splits;                            // the larger number of splits: stride of the partial results
};

int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
int64_t div_up(int64_t x, int64_t m) { return (x + m - 1) / m; }

Plan make_plan(int64_t batch, int64_t tokens, int64_t group, int64_t kv_heads, int64_t max_query_len, int64_t max_kv_len) {
  Plan pl = {};
  const int64_t rows = max_query_len * group;
  pl.few = group > TILE_ROWS ? 0x7FFFFFFF : FEW_ROWS;
  pl.tiles = rows > pl.few;
  // the shortest sequence brings at least the tokens that the others cannot hold
  const int64_t shortest = tokens - (batch - 1) * max_query_len;
  pl.rows = !pl.tiles || shortest * group <= pl.few;
  pl.splits = 1;
  if (pl.rows) {
    // Enough CTAs for about two rounds on all SMs when every sequence has the maximum length, so that shorter ones
    // still fill them, but not below 128 keys (a CTA's fixed costs) nor above MAX_CHUNK.
    const int64_t most = rows < pl.few ? rows : pl.few;
    pl.nt = most <= 8 ? 1 : 2;
    pl.row_tiles = static_cast<int>(div_up(most, 8 * pl.nt));
    const int64_t units = batch * kv_heads * pl.row_tiles, want = PAGED_SMS * (pl.nt == 1 ? 4 : 2) * 2;
    int64_t chunk = round_up(div_up(max_kv_len, units >= want ? 1 : div_up(want, units)), 16);
    chunk = chunk < 128 ? 128 : chunk > MAX_CHUNK ? MAX_CHUNK : chunk;
    pl.chunk = static_cast<int>(chunk);
    pl.row_splits = static_cast<int>(max_kv_len > chunk ? div_up(max_kv_len, chunk) : 1);
    pl.splits = pl.row_splits;
  }
  if (pl.tiles) {
    pl.tile.tokens_per_tile = static_cast<int>(TILE_ROWS / group);
    pl.tile.pairs = static_cast<int>(div_up(max_query_len, 2 * pl.tile.tokens_per_tile));
    const int64_t units = batch * kv_heads * pl.tile.pairs;
    int64_t chunk = round_up(div_up(max_kv_len, units >= PAGED_SMS ? 1 : div_up(PAGED_SMS, units)), 128);
    if (chunk < 512) chunk = 512;
    pl.tile.chunk = static_cast<int>(chunk);
    pl.tile.splits = static_cast<int>(max_kv_len > chunk ? div_up(max_kv_len, chunk) : 1);
    if (pl.tile.splits > pl.splits) pl.splits = pl.tile.splits;
  }
  return pl;
}

template <int D>
int launch(const PagedBatch& b, const PagedAttnParams& p, const Plan& pl, cudaStream_t stream) {
  if (pl.rows) {
    const dim3 grid(static_cast<unsigned>(pl.row_splits), static_cast<unsigned>(b.kv_heads),
                    static_cast<unsigned>(b.batch * pl.row_tiles));
    if (pl.nt == 1)
      paged_rows_kernel<D, 1><<<grid, ROWS_THREADS, 0, stream>>>(p);
    else
      paged_rows_kernel<D, 2><<<grid, ROWS_THREADS, 0, stream>>>(p);
  }
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && pl.tiles) {
    const int rc = launch_paged_tiles(b, p, pl.tile, stream);
    if (rc != TI_OK) return rc;
  }
  if (e == cudaSuccess && pl.splits > 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(div_up(b.max_query_len * p.q_heads, 4)), static_cast<unsigned>(b.batch));
    cfg.blockDim = dim3(128);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, paged_combine_kernel<D>, p, 8 * pl.nt, 2 * pl.tile.tokens_per_tile * p.group, pl.tile.chunk);
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
  if (batch <= 0 || tokens <= 0 || kv_heads <= 0 || q_heads < kv_heads || max_query_len <= 0 || max_kv_len <= 0) return 0;
  if (max_query_len > tokens) max_query_len = tokens;
  const Plan pl = make_plan(batch, tokens, q_heads / kv_heads, kv_heads, max_query_len, max_kv_len);
  return pl.splits == 1 ? 0 : tokens * q_heads * pl.splits * (head_dim * 4 + 8);
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
  if (a.max_kv_len < 0 || a.max_kv_len > 0x7FFFFFFF) {
    set_error("paged_attention: max_kv_len out of range");
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
  const Plan pl = make_plan(b.batch, b.tokens, group, b.kv_heads, b.max_query_len, a.max_kv_len);
  if (b.batch * static_cast<int64_t>(pl.row_tiles) > 65535 || b.max_query_len * a.q_heads > 0x7FFFFFFF) {
    set_error("paged_attention: batch %lld x %lld new tokens is too large for one call", (long long)b.batch,
              (long long)b.max_query_len);
    return TI_E_INVALID;
  }
  const int64_t need = paged_attention_workspace_bytes(b.batch, b.tokens, a.q_heads, b.kv_heads, b.head_dim,
                                                       b.max_query_len, a.max_kv_len);
  if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need || (reinterpret_cast<uintptr_t>(a.workspace) & 15) != 0)) {
    set_error("paged_attention: needs a 16-byte aligned workspace of %lld bytes (got %lld)", (long long)need,
              (long long)a.workspace_bytes);
    return TI_E_INVALID;
  }
  int* status = status_word_ptr();
  if (!status) {
    set_error("paged_attention: cannot resolve the device status word");
    return TI_E_CUDA;
  }
  PagedAttnParams p;
  p.view = make_paged_view(b, status);
  p.q = a.q;
  p.ld_q = a.ld_q;
  p.q_heads = static_cast<int>(a.q_heads);
  p.group = static_cast<int>(group);
  p.max_kv_len = static_cast<int>(a.max_kv_len);
  p.scale_log2 = static_cast<float>(static_cast<double>(a.alpha_qk) * 1.4426950408889634);
  p.alpha_pv = a.alpha_pv;
  p.out = a.out;
  p.out_kind = a.out_kind;
  p.row_tiles = pl.row_tiles;
  p.chunk = pl.chunk;
  p.max_splits = pl.splits;
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
