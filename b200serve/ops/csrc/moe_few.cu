// A whole mixture-of-experts feed-forward layer for a few tokens (1 to 16 rows) in two kernels:
//   p = softmax(x R^T), S = the k most likely experts (ties: the lowest id), w = p_S (/ sum w),
//   out = sum over e in S of D_e (w_e silu(G_e x) * (U_e x)).
//
// With so few rows the layer is the read of the chosen experts' weights, 6 H I bytes each, and
// what costs besides is every wait between dependent steps. So:
//   * moe_router: one CTA per expert row of R computes its logit for every token.
//   * moe_few: one CTA per SM. Every CTA repeats the tiny routing step for itself, then takes units
//     of work from one counter: first all gate/up units (8 inner columns of one expert: 8
//     gate and 8 up rows), then all down units (16 output rows over every chosen expert). Its
//     producer thread runs up to 24 stages (192 KB) ahead with TMA, across units and from the
//     gate/up part into the down part, so the memory pipe does not drain where the
//     down products wait for the activations. Units are handed out in order and a gate/up unit
//     waits for nothing but memory, so the down units' wait ends however few CTAs run at a time.
//
// Products: mma.sync m16n8k16 with the weight rows as M and the tokens as N (8 per group). The
// tensor pipe is a few percent busy; tcgen05 tiles of 128 weight rows would only coarsen the units
// that balance the SMs. Lane (g, t) of a fragment takes 16 bytes of row g at element 16 t + 8 h
// of a 64-element block: the sum over k may run in any order as long as weights and activations
// agree on it, and with the TMA's 128-byte swizzle these reads have no bank conflicts.
//
// Numerics: fp32 accumulation; the routing weight is folded into the activation in fp32, and the
// activation is kept as the sum of two bf16 (high part and remainder, 16 bits of mantissa), so
// the only rounding at bf16 precision is that of the output. Stage s of a unit always goes through
// the same partial sum and partial sums join in the order of s, whichever CTA or warp ran it:
// equal inputs give equal bits.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <algorithm>
#include "tc_primitives.cuh"
#include "tma_host.h"

namespace b200 {

constexpr int kMfMaxT = 16, kMfMaxK = 16, kMfMaxE = 256;
constexpr int kMfWarps = 8;                      // consumer warps; warp 8 is the producer
constexpr int kMfThreads = (kMfWarps + 1) * 32;
constexpr int kMfStages = 24;                    // a multiple of kMfWarps: a slot is always the same warp's
constexpr int kMfKb = 4;                         // 64-element blocks per stage
constexpr int kMfStage = 16 * kMfKb * 128;       // 16 rows: 8 KB
constexpr int kMfUnits = 16;                     // units announced ahead of the consumers
constexpr int kMfRed = 2;                        // buffers of partial sums
constexpr int kMfRouterThreads = 256;

static __device__ int g_mf_err;                  // first error code of the bounded waits, one word per device

struct MfArgs {
  const __nv_bfloat16* x;                        // [T, H], row stride ldx
  long long ldx;
  int T, H, E, k, renorm;
  int first, local;                              // this rank's experts: [first, first + local)
  int I;                                         // inner size, padded to 64
  int h_kb, i_kb;                                // 64-element blocks of H and I
  int h_tiles;                                   // 128-row tiles of the down weight
  const float* logits;                           // [T][E]
  int* counters;                                 // [0] next unit, [1] finished gate/up units
  __nv_bfloat16* act;                            // [2][T * k][I] high parts, remainders
  __nv_bfloat16* out;                            // [T, H], row stride ldo
  long long ldo;
};

// ---------------------------------------------------------------- router logits
template <int TT>
__global__ void __launch_bounds__(kMfRouterThreads) moe_router_kernel(const __nv_bfloat16* __restrict__ router, const MfArgs a,
                                                         float* __restrict__ logits, int* __restrict__ counters) {
  __shared__ float red[kMfRouterThreads / 32][TT];
  const int e = blockIdx.x, tid = threadIdx.x;
  const __nv_bfloat16* w = router + (size_t)e * a.H;
  bf16x8 first{};                                // a weight: does not depend on the previous kernel
  if (tid * 8 < a.H) first = *reinterpret_cast<const bf16x8*>(w + tid * 8);
  pdl_trigger();
  pdl_wait();
  if (e == 0 && tid < 2) counters[tid] = 0;
  float acc[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) acc[t] = 0.f;
  for (int i = tid * 8; i < a.H; i += kMfRouterThreads * 8) {
    const bf16x8 wv = i == tid * 8 ? first : *reinterpret_cast<const bf16x8*>(w + i);
    bf16x8 xv[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t)                 // rows past T repeat the last one: loads without branches
      xv[t] = *reinterpret_cast<const bf16x8*>(a.x + min(t, a.T - 1) * a.ldx + i);
    float wf[8];
    unpack8(wv, wf);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      float xf[8];
      unpack8(xv[t], xf);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[t] = fmaf(wf[j], xf[j], acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const float s = warp_sum(acc[t]);
    if ((tid & 31) == 0) red[tid >> 5][t] = s;
  }
  __syncthreads();
  if (tid < a.T) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kMfRouterThreads / 32; ++i) s += red[i][tid];
    logits[(size_t)tid * a.E + e] = s;
  }
}

// ---------------------------------------------------------------- experts
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                            int c3, uint64_t hint) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(tc::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(tc::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "l"(hint)
      : "memory");
}

__device__ __forceinline__ void mma_16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 rows x 8 k-elements a lane (lo: row g, hi: row g + 8) times 8 tokens
__device__ __forceinline__ void mma_piece(float* d, const uint4& lo, const uint4& hi, const uint4& b) {
  mma_16816(d, lo.x, hi.x, lo.y, hi.y, b.x, b.y);
  mma_16816(d, lo.z, hi.z, lo.w, hi.w, b.z, b.w);
}

struct MfShared {
  uint64_t full[kMfStages], empty[kMfStages];
  uint64_t ufull[kMfUnits], uempty[kMfUnits];
  uint64_t rfull[kMfRed], rempty[kMfRed];
  int unit[kMfUnits];
  int abort_flag;
  int warp_slots[8], warp_pairs[8];              // active experts and pairs among each 32 local experts
  float pair_w[kMfMaxT * kMfMaxK];               // routing weight of an (expert, token) pair
  unsigned char pair_t[kMfMaxT * kMfMaxK];       // its token
  int slot_off[kMfMaxE];                         // first pair of an active expert
  unsigned short slot_e[kMfMaxE], slot_mask[kMfMaxE];   // its local id, its tokens
  unsigned int mask[kMfMaxE];                    // tokens of every local expert
};

// One warp: the k most likely experts of token t; those on this rank get their bit in sh.mask and their
// weight in wtab[expert]. EPL: experts per lane.
template <int EPL>
__device__ __forceinline__ void route_token(const MfArgs& a, MfShared& sh, float* wtab, int t, int lane) {
  const float* row = a.logits + (size_t)t * a.E;
  float p[EPL];
  uint32_t key[EPL];                             // order-preserving bits, 0 = absent or taken
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    p[i] = e < a.E ? __ldcg(row + e) : -INFINITY;
    mx = fmaxf(mx, p[i]);
    const uint32_t u = __float_as_uint(p[i] + 0.f);
    key[i] = e < a.E ? u ^ ((uint32_t)((int)u >> 31) | 0x80000000u) : 0u;
  }
  mx = warp_max(mx);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    p[i] = lane + 32 * i < a.E ? __expf(p[i] - mx) : 0.f;
    sum += p[i];
  }
  unsigned taken = 0;                            // bit i: this lane's expert i is chosen
  for (int j = 0; j < a.k; ++j) {
    uint32_t best = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < EPL; ++i)
      if (key[i] > best) { best = key[i]; at = i; }
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const unsigned e = __reduce_min_sync(0xffffffffu, best == top ? (unsigned)(lane + 32 * at) : 0xffffffffu);
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if ((unsigned)(lane + 32 * i) == e) { key[i] = 0u; taken |= 1u << i; }
  }
  if (a.renorm) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) sum += taken >> i & 1u ? p[i] : 0.f;
  }
  const float scale = 1.f / warp_sum(sum);
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i - a.first;
    if ((taken >> i & 1u) && e >= 0 && e < a.local) {
      wtab[t * a.local + e] = p[i] * scale;
      atomicOr(&sh.mask[e], 1u << t);
    }
  }
}

// NG: groups of 8 tokens
template <int NG>
__global__ void __launch_bounds__(kMfThreads, 1)
    moe_few_kernel(const __grid_constant__ CUtensorMap tm_gu, const __grid_constant__ CUtensorMap tm_dn,
                   const MfArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* red = reinterpret_cast<float*>(ring + kMfStages * kMfStage);      // [kMfRed][warps][NG * 128]
  MfShared& sh = *reinterpret_cast<MfShared*>(red + kMfRed * kMfWarps * NG * 128);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &sh.abort_flag;
  int* err = &g_mf_err;

  if (tid == 0) {
    for (int s = 0; s < kMfStages; ++s) { tc::mbar_init(&sh.full[s], 1); tc::mbar_init(&sh.empty[s], 1); }
    for (int s = 0; s < kMfUnits; ++s) { tc::mbar_init(&sh.ufull[s], 1); tc::mbar_init(&sh.uempty[s], kMfWarps); }
    for (int s = 0; s < kMfRed; ++s) { tc::mbar_init(&sh.rfull[s], kMfWarps); tc::mbar_init(&sh.rempty[s], 1); }
    sh.abort_flag = 0;
    tc::fence_barrier_init();
    tc::fence_proxy_async_smem();
    tc::prefetch_tmap(&tm_gu);
    tc::prefetch_tmap(&tm_dn);
  }
  for (int e = tid; e < a.local; e += kMfThreads) sh.mask[e] = 0u;
  __syncthreads();
  pdl_wait();

  // ---- routing, the same in every CTA (the weights of the pairs pass through the partial sums' memory)
  float* wtab = red;
  for (int t = warp; t < a.T; t += kMfWarps + 1) {
    if (a.E <= 32) route_token<1>(a, sh, wtab, t, lane);
    else if (a.E <= 128) route_token<4>(a, sh, wtab, t, lane);
    else route_token<8>(a, sh, wtab, t, lane);
  }
  __syncthreads();
  // active experts in the order of their id, and their pairs in the order of the tokens
  const unsigned my_mask = tid < a.local ? sh.mask[tid] : 0u;
  const unsigned some = __ballot_sync(0xffffffffu, my_mask != 0u);
  const int mine_n = __popc(my_mask);
  int run = mine_n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += v;
  }
  if (warp < 8 && lane == 31) { sh.warp_slots[warp] = __popc(some); sh.warp_pairs[warp] = run; }
  __syncthreads();
  int n_active = 0, slot = 0, off = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i == warp) { slot = n_active; }
    if (i < warp) off += sh.warp_pairs[i];
    n_active += sh.warp_slots[i];
  }
  if (my_mask) {
    slot += __popc(some & ((1u << lane) - 1u));
    off += run - mine_n;
    sh.slot_e[slot] = (unsigned short)tid;
    sh.slot_mask[slot] = (unsigned short)my_mask;
    sh.slot_off[slot] = off;
    for (unsigned m = my_mask; m; m &= m - 1u, ++off) {
      const int t = __ffs(m) - 1;
      sh.pair_w[off] = wtab[t * a.local + tid];
      sh.pair_t[off] = (unsigned char)t;
    }
  }
  __syncthreads();

  const int col_blocks = a.I / 8;                          // gate/up units per expert
  const int n_up = n_active * col_blocks;
  const int total = n_up + (a.H + 15) / 16;
  const int up_stages = (a.h_kb + kMfKb - 1) / kMfKb, dn_stages = (a.i_kb + kMfKb - 1) / kMfKb;

  if (warp == kMfWarps) {
    if (lane == 0) {
      // ---------------- producer ----------------
      const uint64_t pol = tc::policy_evict_first();
      int slot = 0;
      uint32_t par = 1;
      bool live = true;
      // next free stage: waits for it, announces its bytes, returns its memory
      auto stage = [&](uint64_t*& bar) -> uint8_t* {
        live = tc::mbar_wait_bounded(&sh.empty[slot], par, abort_flag, err, 22);
        bar = &sh.full[slot];
        uint8_t* dst = ring + slot * kMfStage;
        if (live) tc::mbar_arrive_expect_tx(bar, kMfStage);
        if (++slot == kMfStages) { slot = 0; par ^= 1u; }
        return dst;
      };
      int u = atomicAdd(a.counters, 1);
      for (int n = 0; live; ++n) {
        const int us = n % kMfUnits;
        if (!tc::mbar_wait_bounded(&sh.uempty[us], ((n / kMfUnits) & 1) ^ 1, abort_flag, err, 21)) break;
        sh.unit[us] = u < total ? u : -1;
        tc::mbar_arrive(&sh.ufull[us]);
        if (u >= total) break;
        const int next = atomicAdd(a.counters, 1);         // needed only at the next unit
        uint64_t* bar;
        if (u < n_up) {
          // a tile of the gate/up weight: 64 gate rows, then the 64 up rows of the same columns
          const int sl = u / col_blocks, cb = u - sl * col_blocks;
          const int tile = sh.slot_e[sl] * (a.I / 64) + cb / 8, r = (cb % 8) * 8;
          for (int kb = 0; kb < a.h_kb && live; kb += kMfKb) {
            uint8_t* dst = stage(bar);
            if (!live) break;
            tma_load_4d(dst, &tm_gu, bar, 0, r, kb, tile, pol);
            tma_load_4d(dst + kMfStage / 2, &tm_gu, bar, 0, 64 + r, kb, tile, pol);
          }
        } else {
          const int hb = u - n_up, r = (hb % 8) * 16;
          for (int sl = 0; sl < n_active && live; ++sl) {
            const int tile = sh.slot_e[sl] * a.h_tiles + hb / 8;
            for (int kb = 0; kb < a.i_kb && live; kb += kMfKb) {
              uint8_t* dst = stage(bar);
              if (!live) break;
              tma_load_4d(dst, &tm_dn, bar, 0, r, kb, tile, pol);
            }
          }
        }
        u = next;
      }
    }
    __syncwarp();
  } else {
    // ---------------- consumers ----------------
    const int g = lane >> 2, t4 = lane & 3;
    const size_t act_rows = (size_t)a.T * a.k;
    int w0 = 0;                                            // the warp that takes the unit's first stage
    int slot = warp;                                       // this warp's stages use slots warp, warp + 8, ...
    uint32_t par = 0;
    bool ready = false;
    for (int n = 0;; ++n) {
      const int us = n % kMfUnits;
      if (!tc::mbar_wait_bounded(&sh.ufull[us], (n / kMfUnits) & 1, abort_flag, err, 23)) break;
      const int u = *(volatile int*)&sh.unit[us];
      if (u < 0) break;
      const bool up = u < n_up;
      const int stages = up ? up_stages : n_active * dn_stages;
      const int us_slot = up ? u / col_blocks : 0;
      const int ntok = up ? __popc(sh.slot_mask[us_slot]) : a.T;
      float acc[NG][4];
#pragma unroll
      for (int q = 0; q < NG; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[q][i] = 0.f;

      if (!up && !ready && stages > 0) {
        // the activations of every gate/up unit (one counter: by the time a down unit comes up the
        // gate/up units are done or in flight)
        if (lane == 0) {
          const uint64_t deadline = globaltimer_ns() + 2000000000ull;
          for (uint32_t it = 1;; ++it) {
            int done;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(done) : "l"(a.counters + 1) : "memory");
            if (done >= n_up || *abort_flag) break;
            if ((it & 63u) == 0 && globaltimer_ns() > deadline) {
              atomicExch(err, 24);
              *abort_flag = 1;
              break;
            }
          }
        }
        __syncwarp();
        if (*abort_flag) break;
        ready = true;
      }

      // the token of this lane's column in the gate/up part: the g-th of the expert's tokens
      const __nv_bfloat16* xrow[NG];
      if (up) {
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          const int c = q * 8 + g;
          xrow[q] = c < ntok ? a.x + sh.pair_t[sh.slot_off[us_slot] + c] * a.ldx : nullptr;
        }
      }
      bool live = true;
      int s = (warp - w0) & (kMfWarps - 1);
      int sl = up ? 0 : s / dn_stages, ks = up ? s : s - sl * dn_stages;
      for (; s < stages; s += kMfWarps) {
        const uint8_t* w = ring + slot * kMfStage;
        const int kend = up ? a.H : a.I;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        if (up) {
          uint4 b[NG][2 * kMfKb];                          // activations do not wait for the weights
#pragma unroll
          for (int q = 0; q < NG; ++q)
#pragma unroll
            for (int i = 0; i < 2 * kMfKb; ++i) {
              const int k0 = (ks * kMfKb + i / 2) * 64 + 16 * t4 + 8 * (i & 1);
              b[q][i] = xrow[q] != nullptr && k0 < kend ? *reinterpret_cast<const uint4*>(xrow[q] + k0) : zero;
            }
          live = tc::mbar_wait_bounded(&sh.full[slot], par, abort_flag, err, 25);
          if (!live) break;
#pragma unroll
          for (int i = 0; i < 2 * kMfKb; ++i) {
            const uint8_t* p = w + (i / 2) * 1024 + g * 128 + (((2 * t4 + (i & 1)) ^ g) << 4);
            const uint4 lo = *reinterpret_cast<const uint4*>(p);
            const uint4 hi = *reinterpret_cast<const uint4*>(p + kMfStage / 2);
#pragma unroll
            for (int q = 0; q < NG; ++q) mma_piece(acc[q], lo, hi, b[q][i]);
          }
        } else {
          const unsigned m = sh.slot_mask[sl];
          const __nv_bfloat16* arow[NG];
#pragma unroll
          for (int q = 0; q < NG; ++q) {
            const int t = q * 8 + g;
            arow[q] = m >> t & 1u
                          ? a.act + (size_t)(sh.slot_off[sl] + __popc(m & ((1u << t) - 1u))) * a.I
                          : nullptr;
          }
          constexpr int HALF = kMfKb / NG;                 // blocks whose activations are loaded at a time
#pragma unroll
          for (int part = 0; part < NG; ++part) {
            uint4 b[NG][2][2 * HALF];
#pragma unroll
            for (int q = 0; q < NG; ++q)
#pragma unroll
              for (int i = 0; i < 2 * HALF; ++i) {
                const int k0 = (ks * kMfKb + part * HALF + i / 2) * 64 + 16 * t4 + 8 * (i & 1);
                const bool in = arow[q] != nullptr && k0 < kend;
                b[q][0][i] = in ? *reinterpret_cast<const uint4*>(arow[q] + k0) : zero;
                b[q][1][i] = in ? *reinterpret_cast<const uint4*>(arow[q] + act_rows * a.I + k0) : zero;
              }
            if (part == 0) {
              live = tc::mbar_wait_bounded(&sh.full[slot], par, abort_flag, err, 25);
              if (!live) break;
            }
#pragma unroll
            for (int i = 0; i < 2 * HALF; ++i) {
              const uint8_t* p = w + (part * HALF + i / 2) * 2048 + g * 128 + (((2 * t4 + (i & 1)) ^ g) << 4);
              const uint4 lo = *reinterpret_cast<const uint4*>(p);
              const uint4 hi = *reinterpret_cast<const uint4*>(p + 1024);
#pragma unroll
              for (int q = 0; q < NG; ++q) {
                mma_piece(acc[q], lo, hi, b[q][0][i]);
                mma_piece(acc[q], lo, hi, b[q][1][i]);
              }
            }
          }
          if (!live) break;
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sh.empty[slot]);
        slot += kMfWarps;
        if (slot >= kMfStages) { slot = warp; par ^= 1u; }
        ks += kMfWarps;
        if (!up)
          while (ks >= dn_stages) { ks -= dn_stages; ++sl; }
      }
      if (!live) break;

      // ---- join the warps' partial sums; one warp in turn finishes the unit
      const int rb = n % kMfRed;
      const uint32_t rpar = (uint32_t)((n / kMfRed) & 1);
      if (!tc::mbar_wait_bounded(&sh.rempty[rb], rpar ^ 1u, abort_flag, err, 26)) break;
      float* mine = red + (rb * kMfWarps + warp) * NG * 128;
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        *reinterpret_cast<float2*>(mine + q * 128 + g * 8 + 2 * t4) = make_float2(acc[q][0], acc[q][1]);
        *reinterpret_cast<float2*>(mine + q * 128 + (g + 8) * 8 + 2 * t4) = make_float2(acc[q][2], acc[q][3]);
      }
      __syncwarp();
      if (lane == 0) {
        tc::mbar_arrive(&sh.rfull[rb]);
        tc::mbar_arrive(&sh.uempty[us]);
      }
      if (warp == n % kMfWarps) {
        if (!tc::mbar_wait_bounded(&sh.rfull[rb], rpar, abort_flag, err, 27)) break;
        const float* part = red + rb * kMfWarps * NG * 128;
        const int nw = min(stages, kMfWarps);
        auto total_of = [&](int idx) {                     // partial sums in stage order
          float v = 0.f;
          for (int i = 0; i < nw; ++i) v += part[((w0 + i) & (kMfWarps - 1)) * NG * 128 + idx];
          return v;
        };
        if (up) {
          const int cb = u % col_blocks, off = sh.slot_off[us_slot];
          for (int i = lane; i < ntok * 8; i += 32) {
            const int c = i & 7, p = i >> 3;               // inner column, token of the expert
            const int idx = (p >> 3) * 128 + c * 8 + (p & 7);
            const float gate = total_of(idx), upv = total_of(idx + 64);
            const float v = gate / (1.f + __expf(-gate)) * upv * sh.pair_w[off + p];
            const __nv_bfloat16 h = __float2bfloat16_rn(v);
            __nv_bfloat16* dst = a.act + (size_t)(off + p) * a.I + cb * 8 + c;
            dst[0] = h;
            dst[act_rows * a.I] = __float2bfloat16_rn(v - __bfloat162float(h));
          }
          __threadfence();
          __syncwarp();
          if (lane == 0) atomicAdd(a.counters + 1, 1);
        } else {
          const int h0 = (u - n_up) * 16;
          for (int i = lane; i < a.T * 16; i += 32) {
            const int r = i & 15, t = i >> 4;
            if (h0 + r < a.H)
              a.out[t * a.ldo + h0 + r] = __float2bfloat16_rn(total_of((t >> 3) * 128 + r * 8 + (t & 7)));
          }
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sh.rempty[rb]);
      }
      w0 = (w0 + stages) & (kMfWarps - 1);
    }
  }
  __syncthreads();
  if (*abort_flag) {
    // error path: give TMA copies that may still be landing in shared memory time to finish
    const uint64_t until = globaltimer_ns() + 100000ull;
    while (globaltimer_ns() < until) {
    }
  }
}

}  // namespace b200

using namespace b200;

// x [T, H] bf16 (rows may be strided), router [E, H], experts packed as pack_experts() lays them out:
// gate_up [local * (n_gate_up / 128) * h_kb * 128, 64], down [local * h_tiles * i_kb * 128, 64];
// out [T, H] (rows may be strided).
void moe_layer(torch::Tensor x, torch::Tensor router, torch::Tensor gate_up, int64_t n_gate_up, torch::Tensor down,
               int64_t n_down, int64_t k, bool renormalize, int64_t first_expert, torch::Tensor out) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.scalar_type() == at::kBFloat16 && (x.size(0) <= 1 || x.stride(0) % 8 == 0) &&
                  x.stride(1) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0,
              "moe_layer: x must be a CUDA bf16 tensor [T, H] whose rows start on 16-byte boundaries");
  const int64_t T = x.size(0), H = x.size(1), E = router.size(0);
  B200_REQUIRE(T <= kMfMaxT, "moe_layer: at most 16 rows, got " + std::to_string(T));
  B200_REQUIRE(H >= 8 && H % 8 == 0, "moe_layer: H must be a multiple of 8, got " + std::to_string(H));
  TORCH_CHECK(router.dim() == 2 && router.size(1) == H && router.scalar_type() == at::kBFloat16 &&
                  router.is_contiguous() && router.device() == x.device() &&
                  reinterpret_cast<uintptr_t>(router.data_ptr()) % 16 == 0,
              "moe_layer: router must be a contiguous bf16 tensor [E, H] on x's device");
  B200_REQUIRE(E >= 1 && E <= kMfMaxE && k >= 1 && k <= kMfMaxK && k <= E,
               "moe_layer: 1 to 256 experts and 1 to 16 of them per token, got " + std::to_string(E) + " and " +
                   std::to_string(k));
  TORCH_CHECK(n_gate_up > 0 && n_gate_up % 128 == 0 && n_down == H,
              "moe_layer: gate/up rows must be a multiple of 128 and the down rows H");
  const int64_t I = n_gate_up / 2, h_kb = (H + 63) / 64, i_kb = I / 64, h_tiles = (H + 127) / 128;
  const int64_t gu_rows = n_gate_up / 128 * h_kb * 128, dn_rows = h_tiles * i_kb * 128;
  for (const auto& w : {gate_up, down})
    TORCH_CHECK(w.dim() == 2 && w.size(1) == 64 && w.scalar_type() == at::kBFloat16 && w.is_contiguous() &&
                    w.device() == x.device(),
                "moe_layer: expert weights must be packed bf16 tensors [*, 64] on x's device");
  const int64_t local = gate_up.size(0) / gu_rows;
  TORCH_CHECK(local >= 1 && gate_up.size(0) == local * gu_rows && down.size(0) == local * dn_rows,
              "moe_layer: packed expert weights have the wrong shape");
  B200_REQUIRE(first_expert >= 0 && first_expert + local <= E,
               "moe_layer: experts [" + std::to_string(first_expert) + ", " + std::to_string(first_expert + local) +
                   ") are not among the router's " + std::to_string(E));
  TORCH_CHECK(out.dim() == 2 && out.size(0) == T && out.size(1) == H && out.scalar_type() == at::kBFloat16 &&
                  out.stride(1) == 1 && out.device() == x.device(),
              "moe_layer: out must be a bf16 tensor [T, H] on x's device");
  if (T == 0) return;
  const c10::cuda::CUDAGuard guard(x.device());
  // this call's scratch: router logits, two counters, the activations of T * k pairs
  const int64_t head = (T * E * 4 + 8 + 15) / 16 * 16;
  auto ws = torch::empty({head + 2 * T * k * I * 2}, x.options().dtype(at::kByte));
  uint8_t* base = ws.data_ptr<uint8_t>();
  MfArgs a{};
  a.x = reinterpret_cast<const __nv_bfloat16*>(x.data_ptr());
  a.ldx = T > 1 ? x.stride(0) : H;
  a.T = (int)T; a.H = (int)H; a.E = (int)E; a.k = (int)k; a.renorm = renormalize;
  a.first = (int)first_expert; a.local = (int)local; a.I = (int)I;
  a.h_kb = (int)h_kb; a.i_kb = (int)i_kb; a.h_tiles = (int)h_tiles;
  float* logits = reinterpret_cast<float*>(base);
  a.logits = logits;
  a.counters = reinterpret_cast<int*>(base + T * E * 4);
  a.act = reinterpret_cast<__nv_bfloat16*>(base + head);
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.ldo = T > 1 ? out.stride(0) : H;
  const uint32_t gu_box[4] = {64, 8, kMfKb, 1}, dn_box[4] = {64, 16, kMfKb, 1};
  const uint64_t gu_dims[4] = {64, 128, (uint64_t)h_kb, (uint64_t)(local * (n_gate_up / 128))};
  const uint64_t gu_str[3] = {128, 128 * 128, (uint64_t)h_kb * 128 * 128};
  const uint64_t dn_dims[4] = {64, 128, (uint64_t)i_kb, (uint64_t)(local * h_tiles)};
  const uint64_t dn_str[3] = {128, 128 * 128, (uint64_t)i_kb * 128 * 128};
  const CUtensorMap tg = tma_bf16(gate_up.data_ptr(), 4, gu_dims, gu_str, gu_box);
  const CUtensorMap td = tma_bf16(down.data_ptr(), 4, dn_dims, dn_str, dn_box);
  auto stream = at::cuda::getCurrentCUDAStream();
  const __nv_bfloat16* rp = reinterpret_cast<const __nv_bfloat16*>(router.data_ptr());
  const dim3 rg((unsigned)E), rb(kMfRouterThreads);
  if (T <= 1) launch_pdl(moe_router_kernel<1>, rg, rb, 0, stream, rp, a, logits, a.counters);
  else if (T <= 4) launch_pdl(moe_router_kernel<4>, rg, rb, 0, stream, rp, a, logits, a.counters);
  else if (T <= 8) launch_pdl(moe_router_kernel<8>, rg, rb, 0, stream, rp, a, logits, a.counters);
  else launch_pdl(moe_router_kernel<16>, rg, rb, 0, stream, rp, a, logits, a.counters);
  const int ng = T <= 8 ? 1 : 2;
  auto kernel = ng == 1 ? moe_few_kernel<1> : moe_few_kernel<2>;
  const size_t smem = 1024 + (size_t)kMfStages * kMfStage + (size_t)kMfRed * kMfWarps * ng * 128 * 4 + sizeof(MfShared);
  B200_REQUIRE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const int64_t units = std::min<int64_t>(T * k, local) * (I / 8) + (H + 15) / 16;
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  launch_pdl(kernel, dim3((unsigned)std::min<int64_t>(units, sms)), dim3(kMfThreads), smem, stream, tg, td, a);
}

int64_t moe_layer_error(bool reset) {
  int v = 0;
  B200_REQUIRE_CUDA(cudaMemcpyFromSymbol(&v, g_mf_err, sizeof(int)));
  if (reset) {
    const int z = 0;
    B200_REQUIRE_CUDA(cudaMemcpyToSymbol(g_mf_err, &z, sizeof(int)));
  }
  return v;
}
