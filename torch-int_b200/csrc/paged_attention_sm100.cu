// Attention over a paged int8 cache for sequences with many query rows per key head (chunks of prompts), on the
// fifth-generation tensor cores.  Same operator as paged_rows_kernel (paged_attention.cu), same partial results.
//
// A CTA owns one key head of one sequence and two tiles of 128 query rows (a row is a token and one of the query
// heads that share the key head) and walks over 128-key tiles:
//   S = Q . K^T      tcgen05 kind::i8, Q and K as TMA stores them (128-byte swizzle), int32 in TMEM;
//   p = 2^(s - off)  one thread per row, S read from TMEM once; p is written back over S as fp16;
//   O += P . V       tcgen05 kind::f16, A = P from TMEM, B = V from shared memory, fp32 in TMEM.
// V arrives as int8 rows (keys) and one warpgroup turns it into fp16, exactly, in the layout in which the head
// dimension is the contiguous one: no transpose, and 256 query rows share one conversion.
//
// Why this division: per 256 x 128 scores the exponentials take 2048 clocks of an SM (16 per clock), the two
// products 512 + 1024 and everything the softmax threads issue about 1300 slots per scheduler, so the exponentials
// must never wait: two row tiles alternate, the products of one run under the softmax of the other.
//   warps 0-3, 4-7  softmax and epilogue of row tile 0, 1      184 registers
//   warps 8-11      int8 -> fp16 conversion of V               104
//   warp 12, 13     TMA producer, MMA issuer                    40
// The score is formed without a conversion instruction: the bits of 1.5 * 2^23 + acc are acc + constant (|acc| <=
// 2^21), and one fused multiply-add with off = c * (1.5 * 2^23 + max) - 7 gives the exponent; whatever off was
// rounded to, it is the same for the whole row and cancels in the division by the sum.  off is raised only when an
// exponent passes 15 (p <= 2^15 fits fp16 and, against the maximum's 2^7 or more, keeps weights down to 2^-31);
// then O in TMEM is rescaled by the row's thread.  p is rounded to fp16 (2^-11) for the product, the row sum uses
// it unrounded in fp32.
//
// S(j+1) of a row tile overwrites P(j) in TMEM: it is issued only after the commit of P(j) . V(j) has arrived.
// Every wait is bounded (2 s) and reports through the status word.
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
constexpr int THREADS = 512;
constexpr int TMEM_COLS = 512;
constexpr int REGS_SOFTMAX = 184, REGS_CONVERT = 104, REGS_OTHER = 40;  // per thread, of 512 x 128 at launch
constexpr uint32_t TMEM_S = 0, TMEM_O = 256;  // + 128 * row tile

template <int D>
struct Smem {
  static constexpr int HALF_BYTES = ((D + 63) / 64) * TILE_BYTES;  // fp16 V: 64 columns x 128 keys per 16 KB
  static constexpr int Q = 0;
  static constexpr int K = Q + 2 * TILE_BYTES;
  static constexpr int V = K + NK * TILE_BYTES;
  static constexpr int H = V + NV * TILE_BYTES;
  static constexpr int BARS = H + NH * HALF_BYTES;
  static constexpr int BYTES = 1024 + BARS + 512;
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
};

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

struct TileParams {
  PagedAttnParams a;
  int tokens_per_tile;  // 128 / group
  int pairs;            // row tile pairs of the largest sequence
  int chunk;            // keys of a split, a multiple of 128
};

template <int D>
__global__ void __launch_bounds__(THREADS, 1)
paged_tiles_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                   const __grid_constant__ CUtensorMap tmap_v, const TileParams tp) {
  const PagedAttnParams& p = tp.a;
  const PagedView& v = p.view;
  const int b = blockIdx.z, h = blockIdx.y;
  // the last rows of a sequence see most keys: they go first
  const int pair = tp.pairs - 1 - static_cast<int>(blockIdx.x) / p.max_splits, split = blockIdx.x % p.max_splits;
  grid_dep_launch();
  PagedSeq s;
  if (!paged_sequence(v, b, p.max_kv_len, &s)) return;
  const int G = p.group, TPT = tp.tokens_per_tile;
  const int t0 = pair * 2 * TPT;
  if (t0 >= s.T || s.T * G <= p.rows_below) return;
  const int past = s.L - s.T;
  const PagedSplits sp = paged_splits(past + min(t0 + 2 * TPT, s.T), tp.chunk);
  if (split >= sp.n) return;
  const int k0 = split * tp.chunk;
  int nt[2];  // key tiles of the two row tiles
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const bool any = t0 + x * TPT < s.T;
    const int end = min(k0 + tp.chunk, past + min(t0 + (x + 1) * TPT, s.T));
    nt[x] = any && end > k0 ? (end - k0 + TILE - 1) / TILE : 0;
  }
  const int n_tiles = max(nt[0], nt[1]);

  using SM = Smem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::BARS);
  uint64_t* q_full = bars;
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + NK;
  uint64_t* v_full = k_empty + NK;
  uint64_t* v_empty = v_full + NV;
  uint64_t* h_full = v_empty + NV;
  uint64_t* h_empty = h_full + NH;
  uint64_t* s_full = h_empty + NH;
  uint64_t* p_full = s_full + 2;
  uint64_t* pv_done = p_full + 2;
  uint64_t* o_full = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(q_full), 1);
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
      mbar_init(smem_u32(&p_full[x]), 128);
      mbar_init(smem_u32(&pv_done[x]), 1);
      mbar_init(smem_u32(&o_full[x]), 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == 13) {
    tmem_alloc<1>(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OTHER));
    if (warp == 12) {
      // ------------------------------------------------------------ TMA producer: one lane per page of a tile
      const int P = 1 << v.page_shift;
      const int box = min(P, TILE), boxes = TILE / box;  // a 256-key page holds two tiles
      const int pages_used = (s.L + P - 1) >> v.page_shift;
      auto page_at = [&](int j) {  // page of this lane's rows of tile j; one past the pool (zeros) behind the last key
        const int i = (k0 + j * TILE + lane * box) >> v.page_shift;
        if (lane >= boxes || i >= pages_used) return v.num_pages;
        const int page = paged_page(v, b, i);
        return page < 0 ? 0 : page;
      };
      if (lane == 0) {
        const uint32_t rows = G * TPT;
        const int tiles = (nt[0] > 0) + (nt[1] > 0);
        mbar_expect_tx(smem_u32(q_full), tiles * rows * 128);
        for (int x = 0; x < 2; ++x)
          if (nt[x] > 0)
            tma_load_4d(smem_u32(smem + SM::Q + x * TILE_BYTES), &tmap_q, smem_u32(q_full), 0, 0, h, s.q0 + t0 + x * TPT);
      }
      __syncwarp();
      bool ok = true;
      int next = page_at(0);
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int page = next;
        if (j + 1 < n_tiles) next = page_at(j + 1);
        const int row = (k0 + j * TILE + lane * box) & (P - 1);
        const int ks = j % NK, vs = j % NV;
        ok = mbar_wait_status(smem_u32(&k_empty[ks]), ((j / NK) & 1) ^ 1, abort_flag, v.status, TI_ERR_PT_K_EMPTY);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) mbar_expect_tx(smem_u32(&k_full[ks]), TILE_BYTES);
        __syncwarp();
        if (lane < boxes)
          tma_load_4d(smem_u32(smem + SM::K + ks * TILE_BYTES + lane * box * 128), &tmap_k, smem_u32(&k_full[ks]), 0, row, h, page);
        ok = mbar_wait_status(smem_u32(&v_empty[vs]), ((j / NV) & 1) ^ 1, abort_flag, v.status, TI_ERR_PT_V_EMPTY);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) mbar_expect_tx(smem_u32(&v_full[vs]), TILE_BYTES);
        __syncwarp();
        if (lane < boxes)
          tma_load_4d(smem_u32(smem + SM::V + vs * TILE_BYTES + lane * box * 128), &tmap_v, smem_u32(&v_full[vs]), 0, row, h, page);
      }
    } else if (warp == 13 && lane == 0) {
      // ------------------------------------------------------------------------------------------- MMA issuer
      constexpr uint32_t idesc_s = make_idesc_s8s8s32(TILE, TILE);
      constexpr uint32_t idesc_o = make_idesc_f16_b_mn(TILE, D);
      bool ok = n_tiles > 0 && mbar_wait_status(smem_u32(q_full), 0, abort_flag, v.status, TI_ERR_PT_Q);
      auto scores = [&](int x, int j) {  // S_x = Q_x . K_j
        const int ks = j % NK;
        ok = mbar_wait_status(smem_u32(&k_full[ks]), (j / NK) & 1, abort_flag, v.status, TI_ERR_PT_K_FULL);
        if (!ok) return;
        tc_fence_after();
        const uint64_t dq = make_smem_desc_sw128(smem_u32(smem + SM::Q + x * TILE_BYTES));
        const uint64_t dk = make_smem_desc_sw128(smem_u32(smem + SM::K + ks * TILE_BYTES));
#pragma unroll
        for (int k = 0; k < (D + 31) / 32; ++k) umma_i8<1>(tmem + TMEM_S + x * TILE, dq + 2 * k, dk + 2 * k, idesc_s, k != 0);
        umma_commit(smem_u32(&s_full[x]));
        if (x == 1 || j >= nt[1]) umma_commit(smem_u32(&k_empty[ks]));  // the last row tile that reads K_j
      };
      for (int x = 0; x < 2 && ok; ++x)
        if (nt[x] > 0) scores(x, 0);
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int hs = j % NH;
        ok = mbar_wait_status(smem_u32(&h_full[hs]), (j / NH) & 1, abort_flag, v.status, TI_ERR_PT_H_FULL);
        const uint64_t dv = make_smem_desc_mn_sw128(smem_u32(smem + SM::H + hs * SM::HALF_BYTES), TILE_BYTES);
        for (int x = 0; x < 2 && ok; ++x) {
          if (j >= nt[x]) continue;
          ok = mbar_wait_status(smem_u32(&p_full[x]), j & 1, abort_flag, v.status, TI_ERR_PT_P_FULL);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < TILE / 16; ++k)
            umma_f16_a_tmem(tmem + TMEM_O + x * TILE, tmem + TMEM_S + x * TILE + 8 * k, dv + k * (2048 >> 4), idesc_o,
                            j != 0 || k != 0);
          if (x == 1 || j >= nt[1]) umma_commit(smem_u32(&h_empty[hs]));
          if (j + 1 < nt[x]) {
            umma_commit(smem_u32(&pv_done[x]));
            ok = mbar_wait_status(smem_u32(&pv_done[x]), j & 1, abort_flag, v.status, TI_ERR_PT_PV);
            if (ok) scores(x, j + 1);
          } else {
            umma_commit(smem_u32(&o_full[x]));
          }
        }
      }
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------------------------- conversion of V to fp16
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CONVERT));
    const int w = warp - 8;
    // A quarter warp takes four 16-byte chunks of the keys k and k ^ 5: with the swizzle (chunk ^ key % 8) their
    // 16-byte reads and writes fall into different banks.
    const int sub = lane >> 3, c = lane & 3;
    const int key8 = (lane >> 2) & 1 ? sub ^ 5 : sub;  // of a group of 8 keys
    bool ok = true;
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int vs = j % NV, hs = j % NH;
      ok = mbar_wait_status(smem_u32(&v_full[vs]), (j / NV) & 1, abort_flag, v.status, TI_ERR_PT_V_FULL);
      if (!ok) break;
      ok = mbar_wait_status(smem_u32(&h_empty[hs]), ((j / NH) & 1) ^ 1, abort_flag, v.status, TI_ERR_PT_H_EMPTY);
      if (!ok) break;
      const uint8_t* src = smem + SM::V + vs * TILE_BYTES;
      uint8_t* dst = smem + SM::H + hs * SM::HALF_BYTES;
      auto convert = [&](int key, int chunk) {
        const uint4 in = *reinterpret_cast<const uint4*>(src + key * 128 + ((chunk ^ (key & 7)) << 4));
        const uint2 h0 = halves4(in.x), h1 = halves4(in.y), h2 = halves4(in.z), h3 = halves4(in.w);
        uint8_t* row = dst + (chunk >> 2) * TILE_BYTES + key * 128;
        const int o = (chunk & 3) * 2;
        *reinterpret_cast<uint4*>(row + ((o ^ (key & 7)) << 4)) = make_uint4(h0.x, h0.y, h1.x, h1.y);
        *reinterpret_cast<uint4*>(row + (((o + 1) ^ (key & 7)) << 4)) = make_uint4(h2.x, h2.y, h3.x, h3.y);
      };
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = (w * 4 + i) * 8 + key8;
        convert(key, c);
        if (D == 128) convert(key, 4 + c);
      }
      if (D == 80) convert(w * 32 + lane, 4);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(smem_u32(&h_full[hs]));
      mbar_arrive(smem_u32(&v_empty[vs]));
    }
  } else {
    // ----------------------------------------------------------------------------------- softmax and epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    const int x = warp >> 2;                       // row tile
    const int r = (warp & 3) * 32 + lane;          // row of it = TMEM lane
    const int tile_t0 = t0 + x * TPT;
    const int t = tile_t0 + r / G;
    const bool valid = r < G * TPT && t < s.T;
    const int lim = past + min(t, s.T - 1);        // last visible key
    const int lim_min = past + tile_t0;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + TMEM_S + x * TILE + lane_off, to = tmem + TMEM_O + x * TILE + lane_off;
    constexpr uint32_t kMagic = 0x4B400000u;       // bits of 1.5 * 2^23
    const float c = p.scale_log2;
    const int tiles = nt[x];
    float off = c * 12582912.f;
    float l = 0.f;
    bool ok = true;
    for (int j = 0; j < tiles && ok; ++j) {
      ok = mbar_wait_status(smem_u32(&s_full[x]), j & 1, abort_flag, v.status, TI_ERR_PT_S_FULL);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const int kt = k0 + j * TILE;
      const bool edge = kt + TILE - 1 > lim_min;   // some row does not see all keys of the tile
      uint32_t a[4][32];
      auto exponents = [&]() {                     // a = exponent of every score, -inf where hidden
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld_32x32(ts + 32 * q, a[q]);
        tmem_ld_wait();
        const float2 cc = make_float2(c, c), oo = make_float2(-off, -off);
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 e = fma2(make_float2(__uint_as_float(a[q][i] + kMagic), __uint_as_float(a[q][i + 1] + kMagic)), cc, oo);
            a[q][i] = __float_as_uint(e.x);
            a[q][i + 1] = __float_as_uint(e.y);
          }
        if (edge) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (kt + 32 * q + i > lim) a[q][i] = 0xFF800000u;
        }
      };
      exponents();
      float mx[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        mx[q] = __uint_as_float(a[q][0]);
#pragma unroll
        for (int i = 1; i < 31; i += 2) mx[q] = max3(mx[q], __uint_as_float(a[q][i]), __uint_as_float(a[q][i + 1]));
        mx[q] = fmaxf(mx[q], __uint_as_float(a[q][31]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool raise = j == 0 || top > 15.f;
      if (__any_sync(0xffffffffu, raise)) {
        const float old = off;
        if (raise && top > -INFINITY) off += top - 7.f;
        const float corr = ex2(old - off);
        l *= corr;
        if (j > 0) {
#pragma unroll
          for (int q = 0; q < (D + 31) / 32; ++q) {  // columns beyond an 80-wide context hold nothing that is used
            tmem_ld_32x32(to + 32 * q, a[0]);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) a[0][i] = __float_as_uint(__uint_as_float(a[0][i]) * corr);
            tmem_st_32x32(to + 32 * q, a[0]);
          }
          tmem_st_wait();
        }
        exponents();
      }
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t pk[32];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 e = make_float2(ex2(__uint_as_float(a[half * 2 + q][i])), ex2(__uint_as_float(a[half * 2 + q][i + 1])));
            sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], e);
            pk[q * 16 + i / 2] = pack_half2(e.x, e.y);
          }
        tmem_st_32x32(ts + 32 * half, pk);
      }
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(smem_u32(&p_full[x]));
    }
    if (ok && tiles > 0) ok = mbar_wait_status(smem_u32(&o_full[x]), 0, abort_flag, v.status, TI_ERR_PT_O_FULL);
    if (__all_sync(0xffffffffu, ok) && tile_t0 < s.T) {
      tc_fence_after();
      const long long at = static_cast<long long>(s.q0 + t) * p.q_heads + h * G + r % G;
      const bool whole = sp.n == 1;
      const float scale = l > 0.f ? p.alpha_pv / l : 0.f;
      float* po = p.part_o + (at * p.max_splits + split) * D;
      if (valid && !whole) p.part_ml[at * p.max_splits + split] = make_float2(l > 0.f ? off : -1e30f, l);
#pragma unroll
      for (int q = 0; q < (D + 31) / 32; ++q) {
        uint32_t a[32];
        if (tiles > 0) {
          tmem_ld_32x32(to + 32 * q, a);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) a[i] = 0;
        }
        if (valid) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            if (32 * q + i >= D) break;
            const float4 y = make_float4(__uint_as_float(a[i]), __uint_as_float(a[i + 1]), __uint_as_float(a[i + 2]),
                                         __uint_as_float(a[i + 3]));
            if (whole)
              paged_store4(p, at * D + 32 * q + i, y, scale);
            else
              *reinterpret_cast<float4*>(po + 32 * q + i) = y;
          }
        }
        __syncwarp();
      }
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
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, TMEM_COLS);
  }
}

template <int D>
int launch(const PagedBatch& b, const PagedAttnParams& a, const PagedTilePlan& plan, cudaStream_t stream) {
  TileParams tp;
  tp.a = a;
  tp.tokens_per_tile = plan.tokens_per_tile;
  tp.pairs = plan.pairs;
  tp.chunk = plan.chunk;
  CUtensorMap tq, tk, tv;
  const int64_t page_bytes = b.page_size * D;
  const int box = static_cast<int>(b.page_size < TILE ? b.page_size : TILE);
  if (!make_operand_map(&tq, a.q, D, a.group, b.kv_heads, b.tokens, D, a.group * D, a.ld_q, a.group, plan.tokens_per_tile) ||
      !make_operand_map(&tk, b.k_pages, D, b.page_size, b.kv_heads, b.num_pages, D, page_bytes, b.kv_heads * page_bytes, box) ||
      !make_operand_map(&tv, b.v_pages, D, b.page_size, b.kv_heads, b.num_pages, D, page_bytes, b.kv_heads * page_bytes, box))
    return TI_E_CUDA;
  auto kernel = paged_tiles_kernel<D>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::BYTES);
  if (e == cudaSuccess) {
    // the warpgroups' register split has to fit what the block is launched with, or the kernel would wait for good
    static const int regs = [kernel] {
      cudaFuncAttributes fa;
      return cudaFuncGetAttributes(&fa, kernel) == cudaSuccess ? fa.numRegs : 0;
    }();
    if (regs * THREADS < REGS_SOFTMAX * 256 + REGS_CONVERT * 128 + REGS_OTHER * 128) {
      set_error("paged_attention: the kernel was built with %d registers per thread, too few for its warpgroups", regs);
      return TI_E_CUDA;
    }
    const dim3 grid(static_cast<unsigned>(plan.pairs * a.max_splits), static_cast<unsigned>(b.kv_heads),
                    static_cast<unsigned>(b.batch));
    kernel<<<grid, THREADS, Smem<D>::BYTES, stream>>>(tq, tk, tv, tp);
    e = cudaGetLastError();
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
