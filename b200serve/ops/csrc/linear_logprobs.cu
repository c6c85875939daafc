// Log probability of a given token and entropy of the next-token distribution for every row of
// hidden states, straight from the LM head: the logits x w^T (softcap * tanh(. / softcap) where
// the model caps them) never reach memory.
//
//   linear_logprobs: a persistent tcgen05 GEMM. The hidden states are the MMA's A operand (128
//   rows = the 128 TMEM lanes), up to 256 rows of the vocabulary its B operand (TMEM columns), so a
//   thread of the epilogue owns a row and sums up a slice's maximum and exponential sums in
//   registers, with no exchange between threads. Per (row, 128 columns) 16 bytes are written
//   instead of 512 of logits.
//   linear_logprob_rows: joins the slices of every row, with the token's own logit computed once more.
//
// With more than 128 rows two CTAs of a cluster work on one tile of 256 rows (cta_group::2): each
// loads its 128 rows of x and half of the tile's columns of w, so an SM reads 32 KB for 64 elements of H
// instead of 48 KB. One CTA per tile reads 64 bytes a clock there, which is what the L2 gives an SM.
//
// Roles (384 threads): warp 0 TMA producer, warp 1 MMA issuer, warps 4..11 epilogue (two per TMEM
// lane quarter, 128 of the tile's columns each). The epilogue's sums need more than the 168
// registers that 384 threads can have: the first warpgroup gives up 112 of its own to the other two.
//
// Sums over H. The tensor cores cut the bits that do not fit when they add to an fp32 accumulator, so
// the error of one long sum grows with H and has a sign: 5.5e-6 of the result's norm at H = 4096, five
// times a rounded fp32 sum's. So only 128 or 512 elements are summed up in TMEM; the epilogue adds these
// parts to the 128 sums that each of its threads keeps in registers, rounding to nearest. The two TMEM
// buffers alternate between parts, and the MMAs run on under the epilogue.
//
// Bound by the tensor cores for a prompt (2 T V H operations) and by the read of w (2 V H bytes)
// for at most 128 rows.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <algorithm>
#include "logprobs.cuh"
#include "tc_primitives.cuh"
#include "tma_host.h"

namespace b200 {

constexpr int kLlBM = 128, kLlBN = 256, kLlBK = 64, kLlMaxStages = 12, kLlThreads = 384;
// registers per thread: at launch, of the producer's and the MMA issuer's warpgroup, of the epilogue's two
constexpr int kLlRegs = 168, kLlRegsLow = 56, kLlRegsHigh = 224;
static_assert(128 * kLlRegsLow + 256 * kLlRegsHigh == kLlThreads * kLlRegs, "the split must use what the block has");
constexpr int kLlCols = kLlBN / 2;       // columns of an epilogue thread = of a slice
constexpr int kLlA = kLlBM * kLlBK * 2;  // a full tile of x; the MMA reads this much from a stage's start
constexpr int kLlRing = 196608;          // bytes of all stages
// The last stages' x windows may reach past the ring (into memory whose contents do not matter).
constexpr size_t kLlSmem = 1024 + kLlRing + kLlA + 512;
constexpr float kLlFloor = -1e30f;       // lower bound of x - m in products with e^(x - m) = 0, which stay 0
constexpr int64_t kLlRows = 8192;        // rows per pass: bounds the partial results (16 bytes per row and slice)

// First error code of the bounded waits, one word per device. A kernel whose wait ran out leaves partial results
// unwritten, so the rows come back as NaN until the word has been read and reset (linear_logprobs_error).
static __device__ int g_ll_err;

// Work units: row tiles x vocabulary tiles of tile_n columns, the row tiles of one vocabulary tile in a row.
struct LlArgs {
  int T, V, kb_total, m_tiles, v_tiles, tile_m, tile_n;
  // A stage holds x_rows rows of x (128, or with one row tile just T rounded up to 16) and then tile_n of
  // w. The MMA always takes 128 rows of x: with fewer, the others are w's bytes, and their results go nowhere.
  int x_rows, stages, stage_bytes;
  int part_kb;                           // 64-element blocks of H summed up in TMEM
  int packed;                            // w: tile-packed [n_tile][k_block][128][64], else plain [V, H]
  float softcap, inv_softcap;
  TokenIds tokens;
  int per_tile;                          // slices of up to 128 columns in a tile: 1 or 2
  int H;
  const __nv_bfloat16* x;                // [T, H], row stride ldx; with w the token's own logit is computed again
  const __nv_bfloat16* w;
  long long ldx;
  float4* part;                          // [v_tiles * per_tile][T] (m, r, t, the token's logit where the slice has it)
};

// TMA maps of w with boxes of 16, 32, 48, ... 128 rows: a tile of a packed weight takes one box per 128-row
// weight tile that it touches. Plain weights take a tile in one box (map 0).
struct LlMaps {
  CUtensorMap m[8];
};

struct LlUnit {
  int m0, v0, v_tile;                    // first row, first column
};

__device__ __forceinline__ LlUnit ll_unit(const LlArgs& a, int u) {
  LlUnit x;
  x.v_tile = u / a.m_tiles;
  x.m0 = (u - x.v_tile * a.m_tiles) * a.tile_m;
  x.v0 = x.v_tile * a.tile_n;
  return x;
}

// ex2 in program order: the compiler would otherwise start many of a row's 128 exponentials at once and spill
__device__ __forceinline__ float ex2_in_order(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// tanh(y) = 1 - 2r, r = 1 / (1 + e^2y), off by less than 2^-21: 2r times e^2y / (1 + e^2y) of the exponential's error
// (2^-22, and |2y| 2^-24 for its argument) and 2^-23 + 2^-24 of the reciprocal and the sum, at most 1.8 * 2^-22 in all.
// Near zero, where that is not small beside the value, the Taylor series to y^9 (the next term,
// 1382 / 155925 y^11, is below 2^-26 of y for |y| < 1/4)
__device__ __forceinline__ float ll_tanh(float y) {
  const float y2 = y * y;
  const float p = y * fmaf(y2, fmaf(y2, fmaf(y2, fmaf(y2, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2(y * 2.8853900817779268f)));
  return y2 < 0.0625f ? p : fmaf(-2.f, r, 1.f);
}

// ---- two-CTA forms of the tensor-core instructions (CG = 2), one-CTA forms otherwise
template <int CG>
__device__ __forceinline__ void ll_tma(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, uint64_t hint) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "l"(hint)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "l"(hint)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void ll_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    tc::mma_bf16(d, da, db, idesc, accumulate);
}
// arrives on `bar` (of both CTAs) once the MMAs issued so far are complete
template <int CG>
__device__ __forceinline__ void ll_commit(uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            tc::smem_u32(bar)), "h"((unsigned short)3)
        : "memory");
  else
    tc::mma_commit(bar);
}
template <int CG>
__device__ __forceinline__ void ll_tmem_alloc(uint32_t* slot) {
  if constexpr (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(slot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tc::tmem_alloc(slot, 512);
    tc::tmem_relinquish();
  }
}
template <int CG>
__device__ __forceinline__ void ll_tmem_free(uint32_t base) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(512) : "memory");
  else
    tc::tmem_dealloc(base, 512);
}

// CG: CTAs per tile. Rank 0 of a pair issues the MMAs of both; the barriers that it waits on are its own.
template <bool CAP, int CG>
__global__ void __launch_bounds__(kLlThreads, 1)
    linear_logprobs_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ LlMaps tm_w,
                           const LlArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kLlRing + kLlA);
  uint64_t* empty = full + kLlMaxStages;
  uint64_t* tfull = empty + kLlMaxStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* mma_done = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = a.m_tiles * a.v_tiles;
  const int rank = CG == 2 ? (int)tc::cluster_ctarank() : 0, first = blockIdx.x / CG, step = gridDim.x / CG;
  int* err = &g_ll_err;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 1); }
    for (int i = 0; i < 2; ++i) { tc::mbar_init(&tfull[i], 1); tc::mbar_init(&tempty[i], 8 * CG); }
    tc::mbar_init(mma_done, 1);
    *abort_flag = 0;
    tc::fence_barrier_init();
    tc::fence_proxy_async_smem();
    tc::prefetch_tmap(&tm_x);
    for (int i = 0; i < (a.packed ? 8 : 1); ++i) tc::prefetch_tmap(&tm_w.m[i]);
  }
  __syncwarp();
  if (warp == 1) {
    ll_tmem_alloc<CG>(tmem_slot);
  }
  tc::tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) tc::cluster_sync();               // the peer's barriers are ready
  tc::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLlRegsLow));
    if (warp == 0 && lane == 0) {
      // ---------------- TMA producer ----------------
      const uint64_t pol_w = tc::policy_evict_first(), pol_x = tc::policy_evict_last();
      int stage = 0;
      uint32_t phase = 0;
      for (int u = first; u < units && !*abort_flag; u += step) {
        const LlUnit x = ll_unit(a, u);
        for (int kb = 0; kb < a.kb_total; ++kb) {
          if (!tc::mbar_wait_bounded(&empty[stage], phase ^ 1, abort_flag, err, 11)) break;
          uint8_t* dst = smem + stage * a.stage_bytes;
          uint32_t bar = tc::smem_u32(&full[stage]);
          if constexpr (CG == 2) bar = tc::map_shared_rank(bar, 0);
          if (rank == 0) tc::mbar_arrive_expect_tx(&full[stage], CG * a.stage_bytes);
          ll_tma<CG>(dst, &tm_x, bar, kb * kLlBK, x.m0 + rank * kLlBM, pol_x);
          dst += a.x_rows * 128;
          const int w_rows = a.tile_n / CG, v0 = x.v0 + rank * w_rows;
          if (!a.packed) {
            ll_tma<CG>(dst, &tm_w.m[0], bar, kb * kLlBK, v0, pol_w);
          } else {
            for (int r = 0; r < w_rows;) {                 // all of it in multiples of 16 rows
              const int v = v0 + r, rows = min(128 - (v & 127), w_rows - r);
              ll_tma<CG>(dst + r * 128, &tm_w.m[rows / 16 - 1], bar, 0, ((v >> 7) * a.kb_total + kb) * 128 + (v & 127),
                         pol_w);
              r += rows;
            }
          }
          if (++stage == a.stages) { stage = 0; phase ^= 1; }
        }
      }
    }
    if (warp == 1 && lane == 0 && rank == 0) {
      // ---------------- MMA issuer ----------------
      const uint32_t idesc = tc::idesc_bf16_f32(CG * kLlBM, a.tile_n);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      for (int u = first; u < units && !*abort_flag; u += step) {
        for (int k0 = 0; k0 < a.kb_total; k0 += a.part_kb) {
          if (!tc::mbar_wait_bounded(&tempty[acc], acc_phase ^ 1, abort_flag, err, 12)) break;
          tc::tc_fence_after();
          const uint32_t d = tmem_base + acc * kLlBN;
          const int kn = min(a.part_kb, a.kb_total - k0);
          for (int kb = 0; kb < kn; ++kb) {
            if (!tc::mbar_wait_bounded(&full[stage], phase, abort_flag, err, 13)) break;
            tc::tc_fence_after();
            const uint32_t at = tc::smem_u32(smem + stage * a.stage_bytes);
            const uint64_t da = tc::sw128_kmajor_desc(at), db = tc::sw128_kmajor_desc(at + a.x_rows * 128);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) ll_mma<CG>(d, da + 2 * kk, db + 2 * kk, idesc, (kb | kk) ? 1u : 0u);
            ll_commit<CG>(&empty[stage]);
            if (++stage == a.stages) { stage = 0; phase ^= 1; }
          }
          ll_commit<CG>(&tfull[acc]);
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1;
        }
      }
      // no tcgen05.mma may still be running when TMEM is released below
      ll_commit<CG>(mma_done);
      volatile int never = 0;
      tc::mbar_wait_bounded(mma_done, 0, &never, err, 15);
    }
    __syncwarp();
  } else {
    // ---------------- epilogue (warps 4..11) ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLlRegsHigh));
    const int quad = warp & 3, half = (warp - 4) >> 2;
    const float L2E = 1.4426950408889634f;
    int acc = 0;
    uint32_t acc_phase = 0;
    uint32_t drained[2] = {tc::smem_u32(&tempty[0]), tc::smem_u32(&tempty[1])};
    if constexpr (CG == 2) {
      drained[0] = tc::map_shared_rank(drained[0], 0);
      drained[1] = tc::map_shared_rank(drained[1], 0);
    }
    for (int u = first; u < units; u += step) {
      const LlUnit x = ll_unit(a, u);
      const int row = x.m0 + rank * kLlBM + quad * 32 + lane;
      const int cols = min(a.tile_n - half * kLlCols, kLlCols); // <= 0: this half of a narrow tile has none
      float v[kLlCols];
#pragma unroll
      for (int j = 0; j < kLlCols; ++j) v[j] = 0.f;
      bool live = true;
      for (int k0 = 0; k0 < a.kb_total; k0 += a.part_kb) {
        live = __all_sync(0xffffffffu, tc::mbar_wait_bounded(&tfull[acc], acc_phase, abort_flag, err, 14));
        if (!live) break;
        tc::tc_fence_after();
        const uint32_t t_row = tmem_base + ((uint32_t)(quad * 32) << 16) + acc * kLlBN + half * kLlCols;
#pragma unroll
        for (int c = 0; c < kLlCols; c += 16) {
          float r[16];                                     // columns past a narrow tile: masked below
          tc::tmem_ld16(t_row + c, r);
#pragma unroll
          for (int j = 0; j < 16; ++j) v[c + j] += r[j];
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2)
            asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(acc ? drained[1] : drained[0])
                         : "memory");
          else
            tc::mbar_arrive(&tempty[acc]);
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      if (!live) break;
      if (cols <= 0) continue;
      const int c0 = x.v0 + half * kLlCols;                // first column; `in` of them are of the vocabulary
      const int in = min(cols, a.V - c0);
      if constexpr (CAP) {
#pragma unroll
        for (int j = 0; j < kLlCols; ++j) v[j] = a.softcap * ll_tanh(v[j] * a.inv_softcap);
      }
      if (in < kLlCols) {
#pragma unroll
        for (int j = 0; j < kLlCols; ++j)
          if (j >= in) v[j] = -INFINITY;                   // past the vocabulary: counts for nothing
      }
      float xt = 0.f;
      const int at = row < a.T ? token_id(a.tokens, row, a.V) - c0 : -1;
      if ((unsigned)at < (unsigned)in) {
#pragma unroll
        for (int j = 0; j < kLlCols; ++j) xt = j == at ? v[j] : xt;
      }
      float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < kLlCols; ++j) m[j & 3] = fmaxf(m[j & 3], v[j]);
      m[0] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
      const float mm = m[0] == -INFINITY ? 0.f : m[0];     // nothing above -inf: all terms are 0
      float s[4] = {0.f, 0.f, 0.f, 0.f}, t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kLlCols; ++j) {
        const float d = v[j] - mm;
        const float e = ex2_in_order(d * L2E);
        s[j & 3] += e;
        t[j & 3] = fmaf(e, fmaxf(d, kLlFloor), t[j & 3]);  // a logit of -inf: 0 * -1e30
      }
      const float ss = (s[0] + s[1]) + (s[2] + s[3]), tt = (t[0] + t[1]) + (t[2] + t[3]);
      // the maximum's own term leaves the sum: by subtraction, or, where that would cost the others' bits, by another
      // sum of the others
      float rest = ss - 1.f;
      if (ss < 2.f && in > 0) {
        float o[2] = {0.f, -1.f};                          // the others' terms; how many are 1, but for one
#pragma unroll
        for (int j = 0; j < kLlCols; ++j) {
          const float e = ex2_in_order((v[j] - mm) * L2E);
          if (e == 1.f) o[1] += 1.f;
          else o[0] += e;
        }
        rest = o[0] + o[1];
      }
      if (row < a.T)
        a.part[(size_t)(x.v_tile * a.per_tile + half) * a.T + row] = make_float4(ss == ss ? m[0] : INFINITY, rest, tt, xt);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // error path: give TMA copies that may still be landing in shared memory time to finish
    const uint64_t until = globaltimer_ns() + 100000ull;
    while (globaltimer_ns() < until) {
    }
  }
  // no CTA of a pair leaves while the other may still signal its barriers or multiply from its memory
  if constexpr (CG == 2) {
    volatile int never = 0;
    if (rank == 1 && threadIdx.x == 32) tc::mbar_wait_bounded(mma_done, 0, &never, err, 16);
    __syncwarp();
    tc::cluster_sync();
  }
  if (warp == 1) {
    tc::tc_fence_after();
    ll_tmem_free<CG>(tmem_base);
  }
}

// This thread's share (one of G) of the product of row `row` of x with the token's row of w, rounded to nearest.
template <int G>
__device__ __forceinline__ float ll_token_dot(const LlArgs& a, int row, int tok, int g) {
  const __nv_bfloat16* x = a.x + row * a.ldx;
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = 0.f;
  constexpr int U = 4;                                 // pieces on the way at a time
  for (int k0 = g * 8; k0 < a.H; k0 += U * G * 8) {
    bf16x8 xv[U], wv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * G * 8;
      xv[u] = wv[u] = bf16x8{};
      if (k < a.H) {
        xv[u] = *reinterpret_cast<const bf16x8*>(x + k);
        wv[u] = *reinterpret_cast<const bf16x8*>(
            a.packed ? a.w + (((size_t)(tok >> 7) * a.kb_total + (k >> 6)) * 128 + (tok & 127)) * 64 + (k & 63)
                     : a.w + (size_t)tok * a.H + k);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float xf[8], wf[8];
      unpack8(xv[u], xf);
      unpack8(wv[u], wf);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = fmaf(xf[i], wf[i], s[i]);
    }
  }
  return ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

// 256 threads per CTA on R rows, neighbouring threads on neighbouring rows. A thread takes its slices eight at
// a time: one maximum for the eight and the running sum, so the chain of rescalings is short.
//
// The token's own logit is computed once more, by rounded additions in a tree, and takes the place of the tensor cores'
// one in the statistics: where the token is likely, its products are mostly positive, all cuts go the same way (a logit of 13
// is off by 1.7e-6 with parts of 128 elements, by 6.6e-6 with 512) and every bit of log p hangs on that logit. It
// takes 9 of the 2000 us of 2048 rows of H = 4096, and 2 of the 200 of one row.
constexpr int kLlRowThreads = 256;
template <int R>
__global__ void __launch_bounds__(kLlRowThreads) linear_logprob_rows_kernel(const LlArgs a, float* __restrict__ logprob,
                                                                            float* __restrict__ entropy) {
  constexpr int G = kLlRowThreads / R;                 // threads per row
  __shared__ RowStat st[G][R];
  __shared__ float dots[G][R];
  pdl_wait();
  pdl_trigger();
  const int r = threadIdx.x % R, g = threadIdx.x / R;
  const int row = blockIdx.x * R + r, S = a.v_tiles * a.per_tile;
  const int tok = row < a.T ? token_id(a.tokens, row, a.V) : -1;
  float dot = tok >= 0 ? ll_token_dot<G>(a, row, tok, g) : 0.f;
  RowStat acc{-INFINITY, 0.f, 0.f};
  if (row < a.T) {
    for (int i0 = g; i0 < S; i0 += 8 * G) {
      float4 p[8];
      float M = acc.m;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = i0 + j * G;
        p[j] = i < S ? __ldcg(a.part + (size_t)i * a.T + row) : make_float4(-INFINITY, 0.f, 0.f, 0.f);
        M = fmaxf(M, p[j].x);
      }
      if (M == -INFINITY) continue;                    // nothing yet
      float d = fmaxf(acc.m - M, kLlFloor), e = __expf(d), rest = e * acc.r, t = e * (acc.t + d * (1.f + acc.r));
      int ones = 0;                                    // slices whose maximum is M
      if (acc.m == M) ++ones;
      else rest += e;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        d = fmaxf(p[j].x - M, kLlFloor);               // an empty slice: e = 0
        e = __expf(d);
        rest += e * p[j].y;
        if (p[j].x == M) ++ones;
        else rest += e;
        t += e * (p[j].z + d * (1.f + p[j].y));
      }
      acc = RowStat{M, rest + (float)(ones - 1), t};
    }
  }
  st[g][r] = acc;
  dots[g][r] = dot;
  __syncthreads();
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    if (g < o) {
      stat_merge(acc, st[g + o][r]);
      st[g][r] = acc;
      dots[g][r] = dot += dots[g + o][r];
    }
    __syncthreads();
  }
  if (g != 0 || row >= a.T) return;
  const bool ok = stat_valid(acc) && __ldcg(&g_ll_err) == 0;
  float xt = NAN;
  if (tok >= 0) {
    const int v_tile = tok / a.tile_n, half = (tok - v_tile * a.tile_n) / kLlCols;
    xt = __ldcg(&a.part[(size_t)(v_tile * a.per_tile + half) * a.T + row].w);
    if (a.softcap > 0.f) dot = a.softcap * tanhf(dot * a.inv_softcap);
    const float delta = dot - xt;                      // not finite where the logit is not: the first one stays then
    if (fabsf(delta) <= 1.f) {
      if (xt == acc.m) {                               // the token leads: all others move by -delta
        const float q = expm1f(-delta);
        acc.t = (1.f + q) * (acc.t - delta * acc.r);
        acc.r += q * acc.r;
        acc.m = dot;
      } else {
        const float p = __expf(xt - acc.m), q = expm1f(delta);
        acc.t += p * ((1.f + q) * (dot - acc.m) - (xt - acc.m));
        acc.r += p * q;
      }
      xt = dot;
    }
  }
  logprob[row] = ok ? (xt - acc.m) - stat_log(acc) : NAN;
  entropy[row] = ok ? stat_entropy(acc) : NAN;
}

}  // namespace b200

using namespace b200;

// x [T, H] bf16 (rows may be strided), w [V, H] bf16 plain or tile-packed (packed_v = V), tokens [T]
// int32 or int64 -> (logprob [T], entropy [T]) fp32.
std::vector<torch::Tensor> linear_logprobs(torch::Tensor x, torch::Tensor w, int64_t packed_v, torch::Tensor tokens,
                                           double softcap) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.scalar_type() == at::kBFloat16 && x.stride(1) == 1,
              "linear_logprobs: x must be a CUDA bf16 tensor [T, H] with unit stride along H");
  TORCH_CHECK(w.dim() == 2 && w.scalar_type() == at::kBFloat16 && w.is_contiguous() && w.device() == x.device(),
              "linear_logprobs: w must be a contiguous bf16 tensor on x's device");
  const bool packed = packed_v > 0;
  const int64_t T = x.size(0), H = x.size(1), V = packed ? packed_v : w.size(0);
  const int kb = (int)((H + 63) / 64);
  B200_REQUIRE(H >= 8 && H % 8 == 0, "linear_logprobs: H must be a multiple of 8, got " + std::to_string(H));
  B200_REQUIRE(V >= 1 && V <= (1 << 20), "linear_logprobs: vocabulary of 1 to 1048576 tokens, got " + std::to_string(V));
  TORCH_CHECK(w.size(0) < (1ll << 31), "linear_logprobs: weight too large");
  TORCH_CHECK(packed ? w.size(1) == 64 && w.size(0) == (V + 127) / 128 * kb * 128 : w.size(1) == H,
              "linear_logprobs: w must be [V, H], or the tile-packed form of it, with x's H");
  TORCH_CHECK(tokens.dim() == 1 && tokens.size(0) == T && tokens.device() == x.device() && tokens.is_contiguous() &&
                  (tokens.scalar_type() == at::kInt || tokens.scalar_type() == at::kLong),
              "linear_logprobs: tokens must be contiguous int32 or int64 [T] on x's device");
  TORCH_CHECK(softcap >= 0.0, "linear_logprobs: softcap must not be negative");
  const c10::cuda::CUDAGuard guard(x.device());
  auto logprob = torch::empty({T}, x.options().dtype(at::kFloat)), entropy = torch::empty_like(logprob);
  if (T == 0) return {logprob, entropy};
  // rows that lie on one another (an expanded or windowed tensor) are copied out: TMA takes rows side by side
  if (T > 1 && x.stride(0) < H) x = x.contiguous();
  const int64_t ldx = T > 1 ? x.stride(0) : H;
  TORCH_CHECK(ldx % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0,
              "linear_logprobs: rows of x must start on 16-byte boundaries");

  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  auto stream = at::cuda::getCurrentCUDAStream();
  torch::Tensor part;
  for (int64_t t0 = 0; t0 < T; t0 += kLlRows) {
    LlArgs a{};
    a.T = (int)std::min(kLlRows, T - t0); a.V = (int)V; a.kb_total = kb; a.packed = packed;
    const int cg = a.T > kLlBM ? 2 : 1;
    a.tile_m = cg * kLlBM;
    a.m_tiles = (a.T + a.tile_m - 1) / a.tile_m;
    auto kernel = cg == 2 ? (softcap > 0.0 ? linear_logprobs_kernel<true, 2> : linear_logprobs_kernel<false, 2>)
                          : (softcap > 0.0 ? linear_logprobs_kernel<true, 1> : linear_logprobs_kernel<false, 1>);
    cudaFuncAttributes attr;
    B200_REQUIRE_CUDA(cudaFuncGetAttributes(&attr, kernel));
    B200_REQUIRE(attr.numRegs == kLlRegs, "linear_logprobs: the register split does not fit this build");
    B200_REQUIRE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kLlSmem));
    const int slots = sms / cg;                          // CTAs, or pairs of them, at a time
    // columns per tile: of the multiples of 16 the one whose waves take the least time. 32 more columns stand
    // for what a tile costs at any width: the rows of x, and the start of its sums.
    int64_t best = INT64_MAX;
    for (int n = kLlBN; n >= 32; n -= 16 * cg) {
      const int64_t cost = ((int64_t)a.m_tiles * ((V + n - 1) / n) + slots - 1) / slots * (n + 32);
      if (cost < best) { best = cost; a.tile_n = n; }
    }
    a.v_tiles = (int)((V + a.tile_n - 1) / a.tile_n);
    a.per_tile = a.tile_n > kLlCols ? 2 : 1;
    const int64_t slices = (int64_t)a.v_tiles * a.per_tile;
    a.inv_softcap = softcap > 0.0 ? (float)(1.0 / softcap) : 0.f;
    // 128 elements per part where the read of w is the bound, else 512 (the epilogue's additions then stay under the
    // MMAs: 2048 rows of H = 4096 take 2.00 ms, parts of 256 2.18). Root-mean-square error of a log probability beside
    // the logits', H = 4096: 3.6e-7 for 128, 5.4e-7 for 256, 1.1e-6 for 512 elements, before the token's own logit
    // is computed again; below 128 the roundings of the many additions take over. One row of 151936 x 4096: 201 us,
    // with parts of 256 195, of 64 228.
    a.part_kb = cg == 1 ? 2 : 8;
    a.softcap = (float)softcap;
    const bool is64 = tokens.scalar_type() == at::kLong;
    a.tokens = TokenIds{static_cast<const char*>(tokens.data_ptr()) + t0 * (is64 ? 8 : 4), is64};
    const int64_t need = slices * a.T * 4;
    if (!part.defined() || part.numel() < need) part = torch::empty({need}, logprob.options());
    a.part = reinterpret_cast<float4*>(part.data_ptr());
    const __nv_bfloat16* xp = static_cast<const __nv_bfloat16*>(x.data_ptr()) + t0 * ldx;
    a.H = (int)H; a.x = xp; a.w = static_cast<const __nv_bfloat16*>(w.data_ptr()); a.ldx = ldx;
    const uint64_t xd[2] = {(uint64_t)H, (uint64_t)a.T}, xs[1] = {(uint64_t)ldx * 2};
    a.x_rows = cg == 2 ? kLlBM : (a.T + 15) / 16 * 16;
    a.stage_bytes = (a.x_rows + a.tile_n / cg) * 128;
    a.stages = std::min(kLlMaxStages, kLlRing / a.stage_bytes);
    const uint32_t xb[2] = {64, (uint32_t)a.x_rows};
    const uint64_t wd[2] = {packed ? 64ull : (uint64_t)H, (uint64_t)w.size(0)}, ws[1] = {(packed ? 64 : H) * 2ull};
    const CUtensorMap tx = tma_bf16(xp, 2, xd, xs, xb);
    LlMaps tw;
    for (int i = 0; i < 8; ++i) {
      const uint32_t wb[2] = {64, (uint32_t)(packed ? 16 * (i + 1) : a.tile_n / cg)};
      tw.m[i] = i == 0 || packed ? tma_bf16(w.data_ptr(), 2, wd, ws, wb) : tw.m[0];
    }
    const int64_t units = (int64_t)a.m_tiles * a.v_tiles;
    const unsigned grid = (unsigned)(std::min<int64_t>(units, slots) * cg);
    if (cg == 2)
      launch_pdl_cluster(kernel, dim3(grid), dim3(kLlThreads), kLlSmem, stream, 2, tx, tw, a);
    else
      launch_pdl(kernel, dim3(grid), dim3(kLlThreads), kLlSmem, stream, tx, tw, a);
    float* lp = logprob.data_ptr<float>() + t0;
    float* en = entropy.data_ptr<float>() + t0;
    // one row per CTA while that is at most four CTAs an SM, then eight (whole 128-byte lines of the partial results)
    if (a.T > 4 * sms)
      launch_pdl(linear_logprob_rows_kernel<8>, dim3((unsigned)((a.T + 7) / 8)), dim3(kLlRowThreads), 0, stream, a, lp,
                 en);
    else
      launch_pdl(linear_logprob_rows_kernel<1>, dim3((unsigned)a.T), dim3(kLlRowThreads), 0, stream, a, lp, en);
  }
  return {logprob, entropy};
}

// The device's error word; `set` >= 0 is stored in it afterwards.
int64_t linear_logprobs_error(int64_t set) {
  int v = 0;
  B200_REQUIRE_CUDA(cudaMemcpyFromSymbol(&v, g_ll_err, sizeof(int)));
  if (set >= 0) {
    const int z = (int)set;
    B200_REQUIRE_CUDA(cudaMemcpyToSymbol(g_ll_err, &z, sizeof(int)));
  }
  return v;
}
