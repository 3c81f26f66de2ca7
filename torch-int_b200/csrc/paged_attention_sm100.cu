// Attention over a paged int8 cache for sequences with many query rows per key head (chunks of prompts), on the
// fifth-generation tensor cores.  Same operator as paged_rows_kernel (paged_attention.cu), same partial results.
//
// A CTA owns one key head of one sequence and two tiles of 128 query rows (a row is a token and one of the query
// heads that share the key head) and walks over 128-key tiles:
//   S = Q . K^T      tcgen05 kind::i8, Q and K as TMA stores them (128-byte swizzle), int32 in TMEM;
//   p = 2^(s - off)  two threads per row, S read from TMEM once; p goes as fp16 to columns of its own (S is free by then);
//   O += P . V       tcgen05 kind::f16, A = P from TMEM, B = V from shared memory, fp32 in TMEM.
// V arrives as int8 rows (keys) and one warpgroup turns it into fp16, exactly, in the layout in which the head
// dimension is the contiguous one: no transpose, and 256 query rows share one conversion.
//
// Why this division: per 256 x 128 scores the exponentials take 2048 clocks of an SM (16 per clock), the two
// products 512 + 1024 and everything the softmax threads issue about 1300 slots per scheduler, so the exponentials
// must never wait.  S is one buffer of TMEM that both row tiles use in turn: a thread copies its row to registers
// and hands S back, so the products of one tile run under the softmax of the other, and neither product is on the
// path from one tile's exponentials to the next.  TMEM: S 128 columns, P 2 x 64, O 2 x 128.
//   warps 0-7, 8-15  softmax and epilogue of row tile 0, 1: two threads per row, 64 keys each     96 registers
//   warps 16-19      int8 -> fp16 conversion of V                                                  48
//   warps 20-22      TMA producer, issuer of the scores, issuer of the contexts                    48
// Two threads per row, not one: with one the chain from the scores to P (load 400 clocks, exponents and maximum 700,
// exponentials 1400, store 200) was longer than the 2048 clocks it had to stay under; four warps per scheduler
// overlap their chains.  The two threads agree on `off` through a barrier of their two warps that also carries the
// vote; they exchange maxima only where off is raised.
// The two products have an issuing thread each: one thread for both was the slowest part of the pipeline (a product
// of 128 x 128 takes 64 clocks and about 100 to issue and commit).
// The grid is persistent (one CTA per SM): copies and products of the next work item start while the last one's
// context is still being written.
// The score is formed without a conversion instruction: the bits of 1.5 * 2^23 + acc are acc + constant (|acc| <=
// 2^21), and one fused multiply-add with off = c * (1.5 * 2^23 + max) - 7 gives the exponent; whatever off was
// rounded to, it is the same for the whole row and cancels in the division by the sum (as long as the rounding leaves the
// exponents within fp16: MAX_TILE_SCALE in paged_plan.h).  off is raised only when an exponent passes 15 (p <= 2^15 fits fp16 and, against the maximum's 2^7 or more, keeps weights down to 2^-31);
// then O in TMEM is rescaled by the row's threads.  p is rounded to fp16 (2^-11) for the product, the row sum uses
// it unrounded in fp32.  Every wait is bounded (2 s) and reports through the status word.
// Measured: 2048 tokens behind 14336, 32 query heads on 8 of 128: 446 us, 1155 TFLOP/s, 3400 clocks per 256 x 128 scores
// (the exponentials and their conversion keep their pipe busy for 2300 of them, issue for 2500); 8 prompts of 512, 56
// heads: 64 us, of which per item of 2 to 4 key tiles 6500 of about 20000 clocks are outside the loop.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#define TI_PTX_EXTERNAL_STATUS 1
#include "gemm_i8.h"
#include "grid_dependency.cuh"
#include "paged_attention.cuh"
#include "sm100_ptx.cuh"

namespace ti {
namespace {

constexpr int TILE = 128;                 // rows of a row tile, keys of a key tile
constexpr int TILE_BYTES = TILE * 128;    // an int8 tile: 128 rows of 128 bytes
constexpr int NK = 3;                     // stages of K
constexpr int NV = 2;                     // stages of V as int8
constexpr int NH = 2;                     // stages of V as fp16
constexpr int NQ = 2;                     // stages of the queries of a work item
constexpr int MAX_SEQS = 512;             // sequences of a launch
constexpr int THREADS = 768;
constexpr int TMEM_COLS = 512;
constexpr int REGS_SOFTMAX = 96, REGS_CONVERT = 48, REGS_OTHER = 48;  // per thread, of 768 x 80 at launch

constexpr uint32_t TMEM_S = 0, TMEM_P = 128, TMEM_O = 256;  // P + 64, O + 128 for row tile 1

template <int D>
struct Smem {
  static constexpr int HALF_BYTES = ((D + 63) / 64) * TILE_BYTES;  // fp16 V: 64 columns x 128 keys per 16 KB
  static constexpr int Q = 0;
  static constexpr int K = Q + NQ * 2 * TILE_BYTES;
  static constexpr int V = K + NK * TILE_BYTES;
  static constexpr int H = V + NV * TILE_BYTES;
  static constexpr int SEQ = H + NH * HALF_BYTES;
  static constexpr int XCHG = SEQ + MAX_SEQS * 20;  // [row tile][half][row]: maxima, then sums
  static constexpr int ITEM = XCHG + 2 * 2 * 2 * TILE * 4;
  static constexpr int BARS = ITEM + NQ * 48;
  static constexpr int BYTES = 1024 + BARS + 512;
  static_assert(BYTES <= 232448, "227 KB of shared memory");
};

enum : int {
  TI_ERR_PT_Q = 221,         // MMA warp waited for the queries
  TI_ERR_PT_K_EMPTY = 222,   // producer waited for a stage of K
  TI_ERR_PT_K_FULL = 223,    // MMA warp waited for K
  TI_ERR_PT_V_EMPTY = 224,   // producer waited for a stage of V
  TI_ERR_PT_V_FULL = 225,    // conversion waited for V
  TI_ERR_PT_H_EMPTY = 226,   // conversion waited for a stage of fp16 V
  TI_ERR_PT_H_FULL = 227,    // MMA warp waited for fp16 V
  TI_ERR_PT_S_FULL = 228,    // softmax waited for scores
  TI_ERR_PT_P_FULL = 229,    // MMA warp waited for probabilities
  TI_ERR_PT_PV = 230,        // MMA warp waited for a product with V
  TI_ERR_PT_O_FULL = 231,    // epilogue waited for the context
  TI_ERR_PT_Q_EMPTY = 232,   // producer waited for a stage of the queries
  TI_ERR_PT_S_EMPTY = 233,   // MMA warp waited for the scores to be read
  TI_ERR_PT_ITEM = 234,      // a warp waited for the next work item
};

// Bounded wait (2 s), written for few instructions: the loops of the warps of a scheduler share an instruction cache
// of about 12 KB, and misses in it were the largest stall of this kernel.
__device__ __forceinline__ uint32_t timer_ns() {
  uint32_t t;
  asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
  return t;
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint32_t t0 = timer_ns();
#pragma unroll 1
  do {
    if (mbar_try_wait(bar, parity)) return true;
  } while (*abort_flag == 0 && timer_ns() - t0 < static_cast<uint32_t>(TI_WAIT_LIMIT_NS));
  *abort_flag = 1;
  atomicCAS(status, 0, code);
  return false;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)),
        "l"(*reinterpret_cast<const uint64_t*>(&c)));
  return *reinterpret_cast<const float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)));
  return *reinterpret_cast<const float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)));
  return *reinterpret_cast<const float2*>(&d);
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Four int8 -> four fp16, exactly: 1024 + (byte ^ 0x80) as bits, minus 1152.
__device__ __forceinline__ uint2 halves4(uint32_t w) {
  w ^= 0x80808080u;
  const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
  const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// Barrier of `threads` threads that returns whether any of them passed true.
__device__ __forceinline__ bool barrier_or(int id, int threads, bool mine) {
  int any;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.s32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred.aligned q, %1, %2, p;\n\t"
      "selp.s32 %0, 1, 0, q;\n\t"
      "}\n"
      : "=r"(any)
      : "r"(id), "r"(threads), "r"(static_cast<int>(mine))
      : "memory");
  return any != 0;
}

struct TileParams {
  PagedAttnParams a;
  int tokens_per_tile;  // 128 / group
  int chunk;            // keys of a split, a multiple of 128
  int seq0, seqs;       // sequences of this launch
};

// Sequences of the launch in shared memory; `first` = work items (per key head) of the sequences before it.
struct SeqInfo {
  int q0, T, L, first, pairs;
};

// One work item: two row tiles of a sequence, one key head, one split of the keys.  The TMA producer posts them in
// shared memory, in the order of the stages of the queries, for all other warps.
struct __align__(16) Item {
  int nt0, nt1;     // key tiles of the two row tiles; nt0 < 0: no more items
  int q0, T, L;
  int t0, k0;       // first token of the row tiles, first key of the split
  int h, split, n_splits;
  int b, unused;
};

__device__ __forceinline__ int splits_of(int L, int chunk) { return max(1, (L + chunk - 1) / chunk); }

// The work items of a CTA: every gridDim.x-th of (entry, key head), heads fastest; without a division per item.
struct Walk {
  int e, h, de, dh, hkv, entries;
  __device__ __forceinline__ Walk(int kv_heads, int n_entries) : hkv(kv_heads), entries(n_entries) {
    e = static_cast<int>(blockIdx.x) / hkv;
    h = static_cast<int>(blockIdx.x) - e * hkv;
    de = static_cast<int>(gridDim.x) / hkv;
    dh = static_cast<int>(gridDim.x) - de * hkv;
  }
  __device__ __forceinline__ bool more() const { return e < entries; }
  __device__ __forceinline__ void next() {
    e += de;
    h += dh;
    if (h >= hkv) {
      h -= hkv;
      ++e;
    }
  }
};

// Entry e: sequences in order, in each the row tiles that see most keys first, then splits.
__device__ __forceinline__ Item item_at(const TileParams& tp, const SeqInfo* seq, const Walk& walk) {
  Item w;
  const int e = walk.e;
  w.h = walk.h;
  int lo = 0, hi = tp.seqs - 1;
  while (lo < hi) {  // last sequence with first <= e
    const int mid = (lo + hi + 1) >> 1;
    if (seq[mid].first <= e) lo = mid;
    else hi = mid - 1;
  }
  const SeqInfo s = seq[lo];
  const int TPT = tp.tokens_per_tile;
  const int ns = s.L > tp.chunk ? splits_of(s.L, tp.chunk) : 1;
  const int at = ns > 1 ? (e - s.first) / ns : e - s.first;
  w.b = tp.seq0 + lo;
  w.q0 = s.q0;
  w.T = s.T;
  w.L = s.L;
  w.split = e - s.first - at * ns;
  w.t0 = (s.pairs - 1 - at) * 2 * TPT;
  w.k0 = w.split * tp.chunk;
  const int past = s.L - s.T;
  w.n_splits = ns > 1 ? paged_splits(past + min(w.t0 + 2 * TPT, s.T), tp.chunk).n : 1;
  const int end0 = min(w.k0 + tp.chunk, past + min(w.t0 + TPT, s.T));
  const int end1 = min(w.k0 + tp.chunk, past + min(w.t0 + 2 * TPT, s.T));
  w.nt0 = end0 > w.k0 ? (end0 - w.k0 + TILE - 1) / TILE : 0;
  w.nt1 = w.t0 + TPT < s.T && end1 > w.k0 ? (end1 - w.k0 + TILE - 1) / TILE : 0;
  return w;
}

// A ring position: stage and the parity of its current use.
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++stage == n) {
      stage = 0;
      phase ^= 1;
    }
  }
};

template <int D>
__global__ void __launch_bounds__(THREADS, 1)
paged_tiles_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                   const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ TileParams tp) {
  const PagedAttnParams& p = tp.a;
  const PagedView& v = p.view;
  using SM = Smem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  SeqInfo* seq = reinterpret_cast<SeqInfo*>(smem + SM::SEQ);
  volatile Item* item = reinterpret_cast<volatile Item*>(smem + SM::ITEM);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::BARS);
  uint64_t* q_full = bars;
  uint64_t* q_empty = q_full + NQ;
  uint64_t* i_full = q_empty + NQ;
  uint64_t* k_full = i_full + NQ;
  uint64_t* k_empty = k_full + NK;
  uint64_t* v_full = k_empty + NK;
  uint64_t* v_empty = v_full + NV;
  uint64_t* h_full = v_empty + NV;
  uint64_t* h_empty = h_full + NH;
  uint64_t* s_full = h_empty + NH;
  uint64_t* s_empty = s_full + 2;
  uint64_t* p_full = s_empty + 1;
  uint64_t* pv_done = p_full + 2;
  uint64_t* o_full = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* warp_sum = reinterpret_cast<int*>(tmem_slot + 2);  // [24]
  float* s_top = reinterpret_cast<float*>(smem + SM::XCHG);
  float* s_sum = s_top + 2 * 2 * TILE;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dep_launch();
  if (threadIdx.x == 0) {
    for (int i = 0; i < NQ; ++i) {
      mbar_init(smem_u32(&q_full[i]), 1);
      mbar_init(smem_u32(&q_empty[i]), 16 + 4 + 2);  // every warp that reads the item
      mbar_init(smem_u32(&i_full[i]), 1);
    }
    for (int i = 0; i < NK; ++i) {
      mbar_init(smem_u32(&k_full[i]), 1);
      mbar_init(smem_u32(&k_empty[i]), 1);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(smem_u32(&v_full[i]), 1);
      mbar_init(smem_u32(&v_empty[i]), 128);
    }
    for (int i = 0; i < NH; ++i) {
      mbar_init(smem_u32(&h_full[i]), 128);
      mbar_init(smem_u32(&h_empty[i]), 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(smem_u32(&s_full[x]), 1);
      mbar_init(smem_u32(&p_full[x]), 256);
      mbar_init(smem_u32(&pv_done[x]), 1);
      mbar_init(smem_u32(&o_full[x]), 1);
    }
    mbar_init(smem_u32(s_empty), 256);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == 21) {
    tmem_alloc<1>(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish<1>();
  }
  // ---- the sequences of this launch: one per thread, work items counted by a prefix sum
  int entries;
  {
    PagedSeq s = {0, 0, 0};
    int n = 0, pairs = 0;
    const int i = threadIdx.x;
    if (i < tp.seqs && paged_sequence(v, tp.seq0 + i, p.max_kv_len, &s) && s.T * p.group > p.rows_below) {
      pairs = (s.T + 2 * tp.tokens_per_tile - 1) / (2 * tp.tokens_per_tile);
      n = pairs * splits_of(s.L, tp.chunk);
    }
    int sum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += up;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    int before = 0;
    entries = 0;
    for (int k = 0; k < THREADS / 32; ++k) {
      if (k < warp) before += warp_sum[k];
      entries += warp_sum[k];
    }
    if (i < MAX_SEQS) seq[i] = SeqInfo{s.q0, s.T, s.L, before + sum - n, pairs};
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int G = p.group, TPT = tp.tokens_per_tile;

  if (warp >= 20) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OTHER));
    if (warp == 20) {
      // ------------------------------------------------------------ TMA producer: one lane per page of a tile
      const int P = 1 << v.page_shift;
      const int box = min(P, TILE), boxes = TILE / box;  // a 256-key page holds two tiles
      Ring rk, rv, rq;
      bool ok = true;
      for (Walk walk(v.kv_heads, entries); ok; walk.next()) {
        ok = wait_for(smem_u32(&q_empty[rq.stage]), rq.phase ^ 1, abort_flag, v.status, TI_ERR_PT_Q_EMPTY);
        if (!__all_sync(0xffffffffu, ok)) break;
        Item w;
        w.nt0 = -1;
        if (walk.more()) w = item_at(tp, seq, walk);
        if (lane == 0) {
          *const_cast<Item*>(&item[rq.stage]) = w;
          mbar_arrive(smem_u32(&i_full[rq.stage]));
        }
        if (w.nt0 < 0) break;
        const int n_tiles = max(w.nt0, w.nt1);
        const int pages_used = (w.L + P - 1) >> v.page_shift;
        auto page_at = [&](int j) {  // page of this lane's rows of tile j; one past the pool (zeros) behind the last key
          const int i = (w.k0 + j * TILE + lane * box) >> v.page_shift;
          if (lane >= boxes || i >= pages_used) return v.num_pages;
          const int page = paged_page(v, w.b, i);
          return page < 0 ? 0 : page;
        };
        int next = n_tiles > 0 ? page_at(0) : 0;
        if (lane == 0) {
          const uint32_t bar = smem_u32(&q_full[rq.stage]);
          mbar_expect_tx(bar, ((w.nt0 > 0) + (w.nt1 > 0)) * G * TPT * 128);
          const uint32_t dst = smem_u32(smem + SM::Q + rq.stage * 2 * TILE_BYTES);
          if (w.nt0 > 0) tma_load_4d(dst, &tmap_q, bar, 0, 0, w.h, w.q0 + w.t0);
          if (w.nt1 > 0) tma_load_4d(dst + TILE_BYTES, &tmap_q, bar, 0, 0, w.h, w.q0 + w.t0 + TPT);
        }
        __syncwarp();
        rq.next(NQ);
        for (int j = 0; j < n_tiles; ++j) {
          const int page = next;
          if (j + 1 < n_tiles) next = page_at(j + 1);
          const int row = (w.k0 + j * TILE + lane * box) & (P - 1);
          ok = wait_for(smem_u32(&k_empty[rk.stage]), rk.phase ^ 1, abort_flag, v.status, TI_ERR_PT_K_EMPTY);
          if (!__all_sync(0xffffffffu, ok)) break;
          if (lane == 0) mbar_expect_tx(smem_u32(&k_full[rk.stage]), TILE_BYTES);
          __syncwarp();
          if (lane < boxes)
            tma_load_4d(smem_u32(smem + SM::K + rk.stage * TILE_BYTES + lane * box * 128), &tmap_k,
                        smem_u32(&k_full[rk.stage]), 0, row, w.h, page);
          rk.next(NK);
          ok = wait_for(smem_u32(&v_empty[rv.stage]), rv.phase ^ 1, abort_flag, v.status, TI_ERR_PT_V_EMPTY);
          if (!__all_sync(0xffffffffu, ok)) break;
          if (lane == 0) mbar_expect_tx(smem_u32(&v_full[rv.stage]), TILE_BYTES);
          __syncwarp();
          if (lane < boxes)
            tma_load_4d(smem_u32(smem + SM::V + rv.stage * TILE_BYTES + lane * box * 128), &tmap_v,
                        smem_u32(&v_full[rv.stage]), 0, row, w.h, page);
          rv.next(NV);
        }
        ok = __all_sync(0xffffffffu, ok);
      }
    } else if (warp == 21 && lane == 0) {
      // ------------------------------------------------------------------------- issuer of the scores S = Q . K
      constexpr uint32_t idesc = make_idesc_s8s8s32(TILE, TILE);
      const uint64_t desc = make_smem_desc_sw128(0);
      const uint32_t hi = static_cast<uint32_t>(desc >> 32), lo0 = static_cast<uint32_t>(desc);
      const uint32_t q_lo = lo0 + (smem_u32(smem + SM::Q) >> 4), k_lo = lo0 + (smem_u32(smem + SM::K) >> 4);
      Ring rq, rk;
      uint32_t s_parity = 1;  // the first wait passes at once
      bool ok = true;
      while (ok) {
        ok = wait_for(smem_u32(&i_full[rq.stage]), rq.phase, abort_flag, v.status, TI_ERR_PT_ITEM);
        const int nt0 = item[rq.stage].nt0, nt1 = item[rq.stage].nt1, n_tiles = max(nt0, nt1);
        if (!ok || nt0 < 0) break;
        mbar_arrive(smem_u32(&q_empty[rq.stage]));  // the item is read; its queries are kept by the softmax warps' arrivals
        ok = wait_for(smem_u32(&q_full[rq.stage]), rq.phase, abort_flag, v.status, TI_ERR_PT_Q);
        for (int j = 0; j < n_tiles && ok; ++j) {
          ok = wait_for(smem_u32(&k_full[rk.stage]), rk.phase, abort_flag, v.status, TI_ERR_PT_K_FULL);
          const uint32_t b_lo = k_lo + rk.stage * (TILE_BYTES >> 4);
#pragma unroll 1
          for (int x = 0; x < 2; ++x) {
            if (!ok || j >= (x ? nt1 : nt0)) continue;
            ok = wait_for(smem_u32(s_empty), s_parity, abort_flag, v.status, TI_ERR_PT_S_EMPTY);
            if (!ok) continue;
            s_parity ^= 1;
            tc_fence_after();
            const uint32_t a_lo = q_lo + (rq.stage * 2 + x) * (TILE_BYTES >> 4);
#pragma unroll
            for (int k = 0; k < (D + 31) / 32; ++k) umma_i8_lo(tmem + TMEM_S, a_lo + 2 * k, b_lo + 2 * k, hi, idesc, k != 0);
            umma_commit(smem_u32(&s_full[x]));
          }
          if (!ok) break;
          umma_commit(smem_u32(&k_empty[rk.stage]));
          rk.next(NK);
        }
        rq.next(NQ);
      }
    } else if (warp == 22 && lane == 0) {
      // -------------------------------------------------------------------- issuer of the contexts O += P . V
      constexpr uint32_t idesc = make_idesc_f16_b_mn(TILE, D);
      const uint64_t desc = make_smem_desc_mn_sw128(0, TILE_BYTES);
      const uint32_t hi = static_cast<uint32_t>(desc >> 32);
      const uint32_t v_lo = static_cast<uint32_t>(desc) + (smem_u32(smem + SM::H) >> 4);
      Ring rq, rh;
      bool ok = true;
      uint32_t p_phase = 0;  // one bit per row tile
      while (ok) {
        ok = wait_for(smem_u32(&i_full[rq.stage]), rq.phase, abort_flag, v.status, TI_ERR_PT_ITEM);
        const int nt0 = item[rq.stage].nt0, nt1 = item[rq.stage].nt1, n_tiles = max(nt0, nt1);
        if (!ok || nt0 < 0) break;
        mbar_arrive(smem_u32(&q_empty[rq.stage]));
        rq.next(NQ);
        for (int j = 0; j < n_tiles && ok; ++j) {
          ok = wait_for(smem_u32(&h_full[rh.stage]), rh.phase, abort_flag, v.status, TI_ERR_PT_H_FULL);
          const uint32_t b_lo = v_lo + rh.stage * (SM::HALF_BYTES >> 4);
#pragma unroll 1
          for (int x = 0; x < 2; ++x) {
            const int nt = x ? nt1 : nt0;
            if (!ok || j >= nt) continue;
            ok = wait_for(smem_u32(&p_full[x]), (p_phase >> x) & 1, abort_flag, v.status, TI_ERR_PT_P_FULL);
            if (!ok) continue;
            p_phase ^= 1u << x;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < TILE / 16; ++k)  // 16 keys of V are 2048 bytes
              umma_f16_a_tmem(tmem + TMEM_O + x * TILE, tmem + TMEM_P + x * 64 + 8 * k, b_lo + k * (2048 >> 4), hi, idesc,
                              j != 0 || k != 0);
            umma_commit(smem_u32(j + 1 < nt ? &pv_done[x] : &o_full[x]));
          }
          if (!ok) break;
          umma_commit(smem_u32(&h_empty[rh.stage]));
          rh.next(NH);
        }
      }
    }
  } else if (warp >= 16) {
    // ------------------------------------------------------------------------------- conversion of V to fp16
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CONVERT));
    const int wv = warp - 16;
    // A quarter warp takes four 16-byte chunks of the keys k and k ^ 5: with the swizzle (chunk ^ key % 8) their
    // 16-byte reads and writes fall into different banks.
    const int sub = lane >> 3, c = lane & 3;
    const int key8 = (lane >> 2) & 1 ? sub ^ 5 : sub;  // of a group of 8 keys
    Ring rq, rv, rh;
    bool ok = true;
    while (ok) {
      ok = wait_for(smem_u32(&i_full[rq.stage]), rq.phase, abort_flag, v.status, TI_ERR_PT_ITEM);
      const int nt0 = item[rq.stage].nt0, n_tiles = max(nt0, item[rq.stage].nt1);
      if (!ok || nt0 < 0) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&q_empty[rq.stage]));
      rq.next(NQ);
      for (int j = 0; j < n_tiles; ++j) {
        ok = wait_for(smem_u32(&v_full[rv.stage]), rv.phase, abort_flag, v.status, TI_ERR_PT_V_FULL);
        if (ok) ok = wait_for(smem_u32(&h_empty[rh.stage]), rh.phase ^ 1, abort_flag, v.status, TI_ERR_PT_H_EMPTY);
        if (!ok) break;
        const uint8_t* src = smem + SM::V + rv.stage * TILE_BYTES;
        uint8_t* dst = smem + SM::H + rh.stage * SM::HALF_BYTES;
        auto convert = [&](int key, int chunk) {
          const uint4 in = *reinterpret_cast<const uint4*>(src + key * 128 + ((chunk ^ (key & 7)) << 4));
          const uint2 h0 = halves4(in.x), h1 = halves4(in.y), h2 = halves4(in.z), h3 = halves4(in.w);
          uint8_t* row = dst + (chunk >> 2) * TILE_BYTES + key * 128;
          const int o = (chunk & 3) * 2;
          *reinterpret_cast<uint4*>(row + ((o ^ (key & 7)) << 4)) = make_uint4(h0.x, h0.y, h1.x, h1.y);
          *reinterpret_cast<uint4*>(row + (((o + 1) ^ (key & 7)) << 4)) = make_uint4(h2.x, h2.y, h3.x, h3.y);
        };
#pragma unroll 2
        for (int i = 0; i < 4; ++i) {
          const int key = (wv * 4 + i) * 8 + key8;
          convert(key, c);
          if (D == 128) convert(key, 4 + c);
        }
        if (D == 80) convert(wv * 32 + lane, 4);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(smem_u32(&h_full[rh.stage]));
        mbar_arrive(smem_u32(&v_empty[rv.stage]));
        rv.next(NV);
        rh.next(NH);
      }
    }
  } else {
    // ----------------------------------------------------------------------------------- softmax and epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    const int x = warp >> 3, half = (warp >> 2) & 1;   // row tile, 64 keys of a key tile
    const int r = (warp & 3) * 32 + lane;              // row of the tile = TMEM lane
    const int r_token = r / G;
    const int pair_bar = 1 + x * 4 + (warp & 3);       // barrier of the two warps that share 32 rows
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + TMEM_S + half * 64 + lane_off, tpp = tmem + TMEM_P + x * 64 + half * 32 + lane_off;
    // this thread's columns of O: half of them (48 and 32 of 80)
    const int col0 = half * (D == 80 ? 48 : D / 2), cols = D == 80 ? 48 - 16 * half : D / 2;
    const uint32_t to = tmem + TMEM_O + x * TILE + col0 + lane_off;
    float* my_top = s_top + (x * 2 + half) * TILE + r;
    const float* other_top = s_top + (x * 2 + (half ^ 1)) * TILE + r;
    constexpr uint32_t kMagic = 0x4B400000u;           // bits of 1.5 * 2^23
    const float c = p.scale_log2;
    uint32_t s_phase = 0, pv_phase = 0, o_phase = 0;
    Ring rq;
    // A wait that gives up (all later ones then return at once) does not leave an item: the barriers of two warps have
    // no limit, so both warps pass every one of them and only the results are not stored.
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
      if (!wait_for(smem_u32(bar), parity, abort_flag, v.status, code)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
    };
    while (true) {
      wait(&i_full[rq.stage], rq.phase, TI_ERR_PT_ITEM);
      const int nt0 = item[rq.stage].nt0;
      // both warps of a pair leave together (the sums of the item before have been read by now, too)
      if (barrier_or(pair_bar, 64, !ok || nt0 < 0)) break;
      const int nt1 = item[rq.stage].nt1;
      const int tiles = x ? nt1 : nt0;
      const int k0 = item[rq.stage].k0, T = item[rq.stage].T;
      const int tile_t0 = item[rq.stage].t0 + x * TPT;
      const int lim_min = item[rq.stage].L - T + tile_t0;                                            // last key of the first row
      const int lim = lim_min + min(r_token, T - 1 - tile_t0) - half * 64;  // of this row, counted from this thread's columns
      float off = c * 12582912.f;
      float l = 0.f;
      for (int j = 0; j < tiles; ++j) {
        wait(&s_full[x], s_phase, TI_ERR_PT_S_FULL);
        s_phase ^= 1;
        tc_fence_after();
        const int kt = k0 + j * TILE;
        uint32_t a[2][32];                             // scores, then their exponents
        tmem_ld_32x32(ts, a[0]);
        tmem_ld_32x32(ts + 32, a[1]);
        tmem_ld_wait();
        tc_fence_before();
        mbar_arrive(smem_u32(s_empty));
        const float2 cc = make_float2(c, c), oo = make_float2(-off, -off);
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 e = fma2(make_float2(__uint_as_float(a[q][i] + kMagic), __uint_as_float(a[q][i + 1] + kMagic)), cc, oo);
            a[q][i] = __float_as_uint(e.x);
            a[q][i + 1] = __float_as_uint(e.y);
          }
        if (kt + TILE - 1 > lim_min) {                 // some row does not see all keys of the tile
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (kt + 32 * q + i > lim) a[q][i] = 0xFF800000u;
        }
        float mx[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          mx[q] = __uint_as_float(a[q][0]);
#pragma unroll
          for (int i = 1; i < 31; i += 2) mx[q] = max3(mx[q], __uint_as_float(a[q][i]), __uint_as_float(a[q][i + 1]));
        }
        float top = max3(max3(mx[0], mx[1], __uint_as_float(a[0][31])), __uint_as_float(a[1][31]), -INFINITY);
        if (barrier_or(pair_bar, 64, j == 0 || top > 15.f)) {
          *my_top = top;
          asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
          top = fmaxf(top, *other_top);
          const float old = off;
          if ((j == 0 || top > 15.f) && top > -INFINITY) off += top - 7.f;
          const float by = old - off;
          const float corr = j > 0 ? ex2(by) : 1.f;    // in the first tile nothing is there to rescale, and 2^by may be infinite
          l *= corr;
          const float2 by2 = make_float2(by, by);
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 e = add2(make_float2(__uint_as_float(a[q][i]), __uint_as_float(a[q][i + 1])), by2);
              a[q][i] = __float_as_uint(e.x);
              a[q][i + 1] = __float_as_uint(e.y);
            }
          if (j > 0) {                                 // the product that last wrote O is done
            wait(&pv_done[x], pv_phase, TI_ERR_PT_PV);
            tc_fence_after();
#pragma unroll 1
            for (int col = 0; col < cols; col += 8) {
              uint32_t o[8];
              tmem_ld_32x8(to + col, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
              tmem_st_32x8(to + col, o);
            }
          }
        }
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 e = make_float2(ex2(__uint_as_float(a[q][i])), ex2(__uint_as_float(a[q][i + 1])));
            sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], e);
            pk[i / 2] = pack_half2(e.x, e.y);
          }
          if (q == 0 && j > 0) {                       // the product that last read P is done
            wait(&pv_done[x], pv_phase, TI_ERR_PT_PV);
            pv_phase ^= 1;
            tc_fence_after();
          }
          tmem_st_32x16(tpp + 16 * q, pk);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(smem_u32(&p_full[x]));
      }
      // What the epilogue needs, while the last product runs.  The item is read again and `row` is opaque, so that
      // nothing of this is carried through the loop above.
      s_sum[(x * 2 + half) * TILE + r] = l;
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
      l = s_sum[x * 2 * TILE + r] + s_sum[(x * 2 + 1) * TILE + r];
      int row = r;
      asm volatile("" : "+r"(row));
      const int split = item[rq.stage].split, n_splits = item[rq.stage].n_splits;
      const int t = item[rq.stage].t0 + x * TPT + r_token;
      // beyond the keys of this pair of row tiles there is nothing to write
      const bool valid = row < G * TPT && t < item[rq.stage].T && split < n_splits;
      const bool whole = n_splits == 1;
      long long at = static_cast<long long>(item[rq.stage].q0 + t) * p.q_heads + item[rq.stage].h * G + (row - r_token * G);
      if (!whole) at = at * p.max_splits + split;
      const float scale = !whole ? 1.f : l > 0.f ? p.alpha_pv / l : 0.f;
      if (ok && valid && !whole && half == 0) p.part_ml[at] = make_float2(l > 0.f ? off : -1e30f, l);
      // Context rows.  A thread holds a row; stored from there, a warp would touch 32 rows with every instruction.  So
      // 64 bytes of each row at a time pass through shared memory - the item's query tile, which nobody reads any more -
      // and every group of four lanes stores one row's.  A loop of few instructions: this code is cold each time it is
      // reached, and fetching it unrolled took longer (4200 clocks) than the stores.
      const int width = !whole ? 4 : p.out_kind == 3 ? 1 : 2;  // bytes of an element
      const int c16 = (lane & 3) * 16, swz = (lane >> 1) & 3, swz_out = (lane >> 3) & 3;
      const long long row_bytes = valid ? (at * D + col0) * width : -1;
      uint8_t* dst[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long to_row = __shfl_sync(0xffffffffu, row_bytes, 8 * i + (lane >> 2));
        dst[i] = to_row < 0 ? nullptr : (whole ? static_cast<uint8_t*>(p.out) : reinterpret_cast<uint8_t*>(p.part_o)) + to_row + c16;
      }
      uint8_t* stage = smem + SM::Q + (rq.stage * 2 + x) * TILE_BYTES + (half * 4 + (warp & 3)) * 2048;
      if (tiles > 0) {
        wait(&o_full[x], o_phase, TI_ERR_PT_O_FULL);
        o_phase ^= 1;
        tc_fence_after();
      }
#pragma unroll 1
      for (int col = 0; col < cols; col += 16) {
        uint32_t o[16];
        tmem_ld_32x16(to + col, o);
        tmem_ld_wait();
        if (tiles == 0) {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = 0;
        }
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float2 y = mul2(make_float2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), make_float2(scale, scale));
          o[i] = __float_as_uint(y.x);
          o[i + 1] = __float_as_uint(y.y);
        }
        const int byte = (col * width) & 63, filled = byte + 16 * width;
        uint8_t* mine = stage + lane * 64;
        auto put = [&](int piece, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
          *reinterpret_cast<uint4*>(mine + ((((byte >> 4) + piece) ^ swz) << 4)) = make_uint4(a, b, c, d);
        };
        auto y = [&](int i) { return __uint_as_float(o[i]); };
        if (width == 4) {
#pragma unroll
          for (int i = 0; i < 4; ++i) put(i, o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        } else if (width == 2) {
          uint32_t h[8];
          if (p.out_kind == 2) {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = paged_pack2(2, y(2 * i), y(2 * i + 1));
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = paged_pack2(1, y(2 * i), y(2 * i + 1));
          }
          put(0, h[0], h[1], h[2], h[3]);
          put(1, h[4], h[5], h[6], h[7]);
        } else {
          put(0, paged_pack4_s8(y(0), y(1), y(2), y(3)), paged_pack4_s8(y(4), y(5), y(6), y(7)),
              paged_pack4_s8(y(8), y(9), y(10), y(11)), paged_pack4_s8(y(12), y(13), y(14), y(15)));
        }
        if (filled == 64 || col + 16 == cols) {
          __syncwarp();
          const uint8_t* src = stage + (lane >> 2) * 64 + (c16 ^ (swz_out << 4));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (ok && dst[i] && c16 < filled) *reinterpret_cast<uint4*>(dst[i]) = *reinterpret_cast<const uint4*>(src + 512 * i);
            if (dst[i]) dst[i] += 64;
          }
          __syncwarp();
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&q_empty[rq.stage]));
      rq.next(NQ);
      tc_fence_before();  // the next item's products overwrite O only after this thread's next arrival on p_full
    }
  }

  // ---------------------------------------------------------------------------------------------------- teardown
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // a wait gave up: copies and products in flight get a bounded grace period before TMEM is released
    const uint64_t t_start = global_timer_ns();
    while (global_timer_ns() - t_start < 200000ull) {
    }
  }
  __syncthreads();
  if (warp == 21) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, TMEM_COLS);
  }
}

template <int D>
int launch(const PagedBatch& b, const PagedAttnParams& a, const PagedTilePlan& plan, cudaStream_t stream) {
  TileParams tp;
  tp.a = a;
  tp.tokens_per_tile = plan.tokens_per_tile;
  tp.chunk = plan.chunk;
  CUtensorMap tq, tk, tv;
  const int64_t page_bytes = b.page_size * D;
  const int box = static_cast<int>(b.page_size < TILE ? b.page_size : TILE);
  if (!make_operand_map(&tq, a.q, D, a.group, b.kv_heads, b.tokens, D, a.group * D, a.ld_q, a.group, plan.tokens_per_tile) ||
      !make_operand_map(&tk, b.k_pages, D, b.page_size, b.kv_heads, b.num_pages, D, page_bytes, b.kv_heads * page_bytes, box) ||
      !make_operand_map(&tv, b.v_pages, D, b.page_size, b.kv_heads, b.num_pages, D, page_bytes, b.kv_heads * page_bytes, box))
    return TI_E_CUDA;
  auto kernel = paged_tiles_kernel<D>;
  static PagedOncePerDevice once;
  cudaError_t e = once.run([kernel] {
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::BYTES);
    if (err != cudaSuccess) return err;
    // the warpgroups' register split has to fit what the block is launched with, or the kernel would wait for good
    cudaFuncAttributes fa;
    const cudaError_t got = cudaFuncGetAttributes(&fa, kernel);
    if (got != cudaSuccess) return got;
    return fa.numRegs * THREADS < REGS_SOFTMAX * 512 + REGS_CONVERT * 128 + REGS_OTHER * 128 ? cudaErrorLaunchOutOfResources
                                                                                            : cudaSuccess;
  });
  if (e == cudaSuccess) {
    // persistent: one CTA per SM, or per work item where the bounds allow fewer
    const int64_t most = (b.batch < MAX_SEQS ? b.batch : MAX_SEQS) * static_cast<int64_t>(plan.pairs) * plan.splits * b.kv_heads;
    const unsigned grid = static_cast<unsigned>(most < PAGED_SMS ? most : PAGED_SMS);
    for (int64_t b0 = 0; b0 < b.batch && e == cudaSuccess; b0 += MAX_SEQS) {
      tp.seq0 = static_cast<int>(b0);
      tp.seqs = static_cast<int>(b.batch - b0 < MAX_SEQS ? b.batch - b0 : MAX_SEQS);
      kernel<<<grid, THREADS, Smem<D>::BYTES, stream>>>(tq, tk, tv, tp);
      e = cudaGetLastError();
    }
  }
  if (e != cudaSuccess) {
    set_error("paged_attention launch failed: %s", cudaGetErrorString(e));
    return TI_E_CUDA;
  }
  return TI_OK;
}

}  // namespace

int launch_paged_tiles(const PagedBatch& b, const PagedAttnParams& p, const PagedTilePlan& plan, cudaStream_t stream) {
  switch (b.head_dim) {
    case 128: return launch<128>(b, p, plan, stream);
    case 80: return launch<80>(b, p, plan, stream);
    default: return launch<64>(b, p, plan, stream);
  }
}

}  // namespace ti
