// A whole mixture-of-experts feed-forward layer for a few tokens (1 to 16 rows) in two kernels:
//   p = softmax(x R^T), S = the k most likely experts (ties: the lowest id), w = p_S (/ sum w),
//   out = sum over e in S of D_e (w_e silu(G_e x) * (U_e x)).
//
// With so few rows the layer is the read of the chosen experts' weights, 6 H I bytes each, and
// what costs besides is every wait between dependent steps. So:
//   * moe_router: one CTA per expert row of R and four tokens computes their logits.
//   * moe_few: two CTAs of eight warps per SM. Every CTA repeats the tiny routing step for itself,
//     then takes units of work from one counter: first all gate/up units (8 inner columns of one
//     expert: 8 gate and 8 up rows), then all down units (16 output rows over every chosen
//     expert). The warps share a unit's sum over k, 128 elements (a chunk, 4 KB of weights) at a
//     time, and keep the weights of their next chunks on the way with cp.async, across units and from
//     the gate/up part into the down part, so the memory pipe does not drain while the down
//     products wait for the activations. Units are handed out in order and a gate/up unit waits for
//     nothing but memory, so the down units' wait ends however few CTAs run at a time.
//
// Products: mma.sync m16n8k16 with the weight rows as M and the tokens as N (8 per group). A lane copies
// into shared memory just the bytes that it reads back itself, so a ring of chunks takes neither
// barriers nor registers: lane (g, t) takes 16 bytes of rows g and g + 8 at element
// 32 h + 8 t of a 64-element block (the sum over k may run in any order that weights and activations
// agree on), so a warp's load covers eight whole 64-byte pieces. The tensor pipe is a few percent
// busy; tcgen05 tiles of 128 weight rows would only coarsen the units that balance the SMs. TMA
// into shared memory was slower here: boxes of 8 rows and the waits on 24 stages took 0.25 us per
// 8 KB and SM, 218 us where this takes 148 (16 rows, 128 experts of 768, top 8, 2048 wide).
//
// Numerics: fp32 accumulation; the routing weight is folded into the activation in fp32, and the
// activation is kept as the sum of two bf16 (high part and remainder, 16 bits of mantissa), so
// the only rounding at bf16 precision is that of the output. Chunk c of a unit always goes to warp c mod 8,
// a warp adds its chunks in their order and the warps' sums join in the order of the warps, whichever CTA
// took the unit: equal inputs give equal bits.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <algorithm>
#include <atomic>
#include <cstring>
#include <mutex>
#include "tma_host.h"

namespace b200 {

constexpr int kMfMaxT = 16, kMfMaxK = 16, kMfMaxE = 256;
constexpr int kMfWarps = 8;
constexpr int kMfThreads = kMfWarps * 32;
constexpr int kMfRouterThreads = 256;

constexpr int kMfWaitCode = 24;                  // error code: the wait for the gate/up units ran out
constexpr int kMfMaxDevices = 64;

// One host-mapped error word per device: a kernel whose wait runs out stores its code there, and the host reads it
// without waiting for the GPU.
static std::atomic<int*> g_mf_words{nullptr};
static int* mf_error_words() {
  static std::once_flag once;
  std::call_once(once, [] {
    // allowed while a graph is captured: the allocation is not part of it
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    B200_REQUIRE_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
    void* p = nullptr;
    const cudaError_t e = cudaHostAlloc(&p, kMfMaxDevices * sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
    B200_REQUIRE_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
    B200_REQUIRE_CUDA(e);
    memset(p, 0, kMfMaxDevices * sizeof(int));
    g_mf_words = static_cast<int*>(p);           // the same address on the host and on every device
  });
  return g_mf_words;
}

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
  int* err;                                      // this device's error word
  uint64_t wait_ns;                              // limit of the wait for the gate/up units
};

// ---------------------------------------------------------------- router logits
template <int TT>
__global__ void __launch_bounds__(kMfRouterThreads) moe_router_kernel(const __nv_bfloat16* __restrict__ router, const MfArgs a,
                                                         float* __restrict__ logits, int* __restrict__ counters) {
  __shared__ float red[kMfRouterThreads / 32][TT];
  const int e = blockIdx.x, tid = threadIdx.x, t0 = blockIdx.y * TT;
  const __nv_bfloat16* w = router + (size_t)e * a.H;
  pdl_trigger();
  pdl_wait();                                    // the previous kernel may have written the router itself
  if (e == 0 && t0 == 0 && tid < 2) counters[tid] = 0;
  float acc[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) acc[t] = 0.f;
  for (int i = tid * 8; i < a.H; i += kMfRouterThreads * 8) {
    const bf16x8 wv = *reinterpret_cast<const bf16x8*>(w + i);
    bf16x8 xv[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t)                 // rows past T repeat the last one: loads without branches
      xv[t] = *reinterpret_cast<const bf16x8*>(a.x + min(t0 + t, a.T - 1) * a.ldx + i);
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
  if (tid < TT && t0 + tid < a.T) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kMfRouterThreads / 32; ++i) s += red[i][tid];
    logits[(size_t)(t0 + tid) * a.E + e] = s;
  }
}

// ---------------------------------------------------------------- experts
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

template <int NG>
struct MfShared {
  static constexpr int kDepth = NG == 1 ? 3 : 2;  // chunks on the way per warp; two CTAs share 227 KB
  uint4 ring[kDepth][8][kMfThreads];             // [chunk][block, half, rows g or g + 8][thread]
  float red[2][kMfWarps][NG * 128];              // partial sums: two units' worth
  int unit[4];                                   // the CTA's units, a ring
  int gave_up;                                   // the wait for the gate/up units ran out
  int warp_slots[kMfWarps], warp_pairs[kMfWarps];  // active experts and pairs among each 32 local experts
  float pair_w[kMfMaxT * kMfMaxK];               // routing weight of an (expert, token) pair
  unsigned char pair_t[kMfMaxT * kMfMaxK];       // its token
  int slot_off[kMfMaxE];                         // first pair of an active expert
  unsigned short slot_e[kMfMaxE], slot_mask[kMfMaxE];   // its local id, its tokens
  unsigned int mask[kMfMaxE];                    // tokens of every local expert
};

// One warp: the k most likely experts of token t; those on this rank get their bit in mask[expert] and their
// weight in wtab[t][expert]. EPL: experts per lane.
template <int EPL>
__device__ __forceinline__ void route_token(const MfArgs& a, unsigned int* mask, float* wtab, int t, int lane) {
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
      atomicOr(&mask[e], 1u << t);
    }
  }
}

// NG: groups of 8 tokens. PAIR (at most 4 tokens): the down products take the activations' high parts in
// columns 0..3 and their remainders in columns 4..7 of the one group.
template <int NG, bool PAIR>
__global__ void __launch_bounds__(kMfThreads, 2)
    moe_few_kernel(const __nv_bfloat16* __restrict__ gate_up, const __nv_bfloat16* __restrict__ down, const MfArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  MfShared<NG>& sh = *reinterpret_cast<MfShared<NG>*>(smem_raw);
  constexpr int DEPTH = MfShared<NG>::kDepth;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  for (int e = tid; e < a.local; e += kMfThreads) sh.mask[e] = 0u;
  __syncthreads();
  pdl_wait();
  if (tid == 0) {
    sh.gave_up = 0;
    sh.unit[0] = atomicAdd(a.counters, 1);
    sh.unit[1] = atomicAdd(a.counters, 1);
  }

  // ---- routing, the same in every CTA (the weights of the pairs pass through the partial sums' memory)
  static_assert(sizeof(sh.red) >= (NG == 1 ? 8 : 16) * kMfMaxE * 4, "the routing weights must fit");
  float* wtab = &sh.red[0][0][0];
  for (int t = warp; t < a.T; t += kMfWarps) {
    if (a.E <= 32) route_token<1>(a, sh.mask, wtab, t, lane);
    else if (a.E <= 128) route_token<4>(a, sh.mask, wtab, t, lane);
    else route_token<8>(a, sh.mask, wtab, t, lane);
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
  if (lane == 31) { sh.warp_slots[warp] = __popc(some); sh.warp_pairs[warp] = run; }
  __syncthreads();
  int n_active = 0, first_slot = 0, off = 0;
#pragma unroll
  for (int i = 0; i < kMfWarps; ++i) {
    if (i == warp) first_slot = n_active;
    if (i < warp) off += sh.warp_pairs[i];
    n_active += sh.warp_slots[i];
  }
  if (my_mask) {
    const int sl = first_slot + __popc(some & ((1u << lane) - 1u));
    off += run - mine_n;
    sh.slot_e[sl] = (unsigned short)tid;
    sh.slot_mask[sl] = (unsigned short)my_mask;
    sh.slot_off[sl] = off;
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
  const int up_chunks = (a.h_kb + 1) / 2, dn_chunks = (a.i_kb + 1) / 2;   // per unit; per unit and expert
  const size_t act_rows = (size_t)a.T * a.k;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  // Offsets in 16-byte words: a 64-element row of a weight tile has 8, a tile 1024.
  const int lane_off = g * 8 + t4;

  // ---- the next chunk that this warp copies: chunk `nc` of unit `nu`, which is the CTA's `nn`-th; `ahead` chunks
  // are copied and not consumed
  int nn = 0, nu = sh.unit[0], nc = warp, nsl = 0, nks = 0, n_chunks = 0, in_slot = 0, out_slot = 0, ahead = 0;
  const uint4* n_base = nullptr;                           // tile of the unit (down: of expert 0, row block included)
  int n_hi = 0, n_kb = 0;
  auto enter = [&]() {                                     // sets up unit nu
    nc = warp;
    if (nu < n_up) {
      const int sl = nu / col_blocks, cb = nu - sl * col_blocks;
      n_base = reinterpret_cast<const uint4*>(gate_up) +
               ((size_t)(sh.slot_e[sl] * (a.I / 64) + cb / 8) * a.h_kb * 128 + (cb % 8) * 8) * 8 + lane_off;
      n_hi = 64 * 8;                                       // a tile: 64 gate rows, then the 64 up rows of the same columns
      n_kb = a.h_kb;
      n_chunks = up_chunks;
      nsl = 0;
      nks = warp;
    } else if (nu < total) {
      const int hb = nu - n_up;
      n_base = reinterpret_cast<const uint4*>(down) + ((size_t)(hb / 8) * a.i_kb * 128 + (hb % 8) * 16) * 8 + lane_off;
      n_hi = 8 * 8;
      n_kb = a.i_kb;
      n_chunks = n_active * dn_chunks;
      nsl = warp / dn_chunks;
      nks = warp - nsl * dn_chunks;
    } else {
      n_chunks = 0;
    }
  };
  // copies until DEPTH chunks are ahead or the units known (up to the CTA's `known`-th) hold no more
  auto fill = [&](int known) {
    while (ahead < DEPTH) {
      if (nc >= n_chunks) {
        if (nn == known) return;
        ++nn;
        nu = sh.unit[nn & 3];
        enter();
        continue;
      }
      const uint4* base = n_base;
      if (nu >= n_up) base += (size_t)sh.slot_e[nsl] * a.h_tiles * a.i_kb * 1024;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int kb = nks * 2 + (i >> 2);
        const uint4* src = base + (size_t)min(kb, n_kb - 1) * 1024 + (i >> 1 & 1) * 4 + ((i & 1) ? n_hi : 0);
        const int bytes = kb < n_kb ? 16 : 0;              // past the last block: zeros
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         (uint32_t)__cvta_generic_to_shared(&sh.ring[in_slot][i][tid])), "l"(src), "r"(bytes)
                     : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      in_slot = in_slot + 1 == DEPTH ? 0 : in_slot + 1;
      ++ahead;
      nc += kMfWarps;
      nks += kMfWarps;
      if (nu >= n_up)
        while (nks >= dn_chunks) { nks -= dn_chunks; ++nsl; }
    }
  };
  enter();
  fill(1);

  bool ready = false, dead = false;                        // dead: the outputs of this CTA are NaN
  int done_units = 0;                                      // gate/up units of this CTA
  for (int n = 0;; ++n) {
    const int u = sh.unit[n & 3];
    const bool up = u < n_up;
    if (!up && !ready) {
      // every warp's activations are written: publish the CTA's units, then wait for everybody's
      __syncthreads();
      if (tid == 0) {
        __threadfence();
        if (done_units) atomicAdd(a.counters + 1, done_units);
        if (u < total && n_active > 0) {
          const uint64_t deadline = globaltimer_ns() + a.wait_ns;
          for (uint32_t it = 1;; ++it) {
            int done;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(done) : "l"(a.counters + 1) : "memory");
            if (done >= n_up) break;
            if ((it & 63u) == 0 && globaltimer_ns() > deadline) {
              sh.gave_up = 1;
              *static_cast<volatile int*>(a.err) = kMfWaitCode;   // read by moe_layer_error()
              __threadfence_system();
              break;
            }
          }
        }
      }
      __syncthreads();
      dead = sh.gave_up != 0;
      ready = true;
    }
    if (u >= total) break;
    // the unit after next: asked for now, needed at the end of this one
    int ticket = 0;
    if (tid == 0) ticket = atomicAdd(a.counters, 1);

    const int us = up ? u / col_blocks : 0;
    const int ntok = up ? __popc(sh.slot_mask[us]) : a.T;
    const int chunks = up ? up_chunks : n_active * dn_chunks;
    const __nv_bfloat16* xrow[NG];                         // the token of this lane's column: the g-th of the expert's
    if (up) {
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        const int c = q * 8 + g;
        xrow[q] = c < ntok ? a.x + sh.pair_t[sh.slot_off[us] + c] * a.ldx : nullptr;
      }
    }
    // two accumulators per group keep the chain of dependent MMAs short
    float acc[NG][2][4];
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[q][i >> 2][i & 3] = 0.f;

    int sl = up ? 0 : warp / dn_chunks, ks = warp - sl * dn_chunks;
    for (int c = warp; c < chunks; c += kMfWarps) {
      uint4 w[2][2][2];
      bool have_w = false;
      auto take_w = [&]() {                                // starts further copies, waits for the oldest chunk
        fill(n + 1);
        // it has landed once at most ahead - 1 groups are on the way
        if (ahead >= 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
        else if (ahead == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i >> 2][i >> 1 & 1][i & 1] = sh.ring[out_slot][i][tid];
        have_w = true;
      };
      // activations first: their way from L2 passes under the copies and the wait
      const int k0 = ks * 128 + 8 * t4;
      if (up) {
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          if (q * 8 >= ntok) break;
          uint4 b[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            b[i] = xrow[q] != nullptr && k0 + 32 * i < a.H ? *reinterpret_cast<const uint4*>(xrow[q] + k0 + 32 * i)
                                                           : zero;
          if (!have_w) take_w();
#pragma unroll
          for (int i = 0; i < 4; ++i) mma_piece(acc[q][i & 1], w[i >> 1][i & 1][0], w[i >> 1][i & 1][1], b[i]);
        }
      } else {
        const unsigned m = sh.slot_mask[sl];
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          if (!(m >> (8 * q) & 0xffu)) continue;           // none of this group's tokens
          const int t = PAIR ? g & 3 : q * 8 + g;
          const __nv_bfloat16* arow = a.act + (size_t)(sh.slot_off[sl] + __popc(m & ((1u << t) - 1u))) * a.I + k0;
          if (PAIR && g >= 4) arow += act_rows * a.I;
          const bool in = m >> t & 1u;
          constexpr int PARTS = PAIR ? 1 : 2;              // high parts, remainders
          uint4 b[PARTS][4];
#pragma unroll
          for (int j = 0; j < PARTS; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              b[j][i] = in && k0 + 32 * i < a.I ? *reinterpret_cast<const uint4*>(arow + j * act_rows * a.I + 32 * i)
                                                : zero;
          if (!have_w) take_w();
          float part[2][4];
#pragma unroll
          for (int i = 0; i < 8; ++i) part[i >> 2][i & 3] = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < PARTS; ++j)
              mma_piece(part[PARTS == 1 ? i & 1 : j], w[i >> 1][i & 1][0], w[i >> 1][i & 1][1], b[j][i]);
          // only the expert's own tokens take its products: 0 times an infinite weight is not 0
          const int c0 = q * 8 + (PAIR ? 2 * t4 & 3 : 2 * t4);
          const bool in0 = m >> c0 & 1u, in1 = m >> (c0 + 1) & 1u;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i & 1 ? in1 : in0) acc[q][i >> 2][i & 3] += part[i >> 2][i & 3];
        }
      }
      out_slot = out_slot + 1 == DEPTH ? 0 : out_slot + 1;
      --ahead;
      ks += kMfWarps;
      if (!up)
        while (ks >= dn_chunks) { ks -= dn_chunks; ++sl; }
    }
    fill(n + 1);                                           // under the join and the next unit's start

    // ---- join the warps' partial sums, in the order of the warps
    float(*red)[NG * 128] = sh.red[n & 1];
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const float* c0 = acc[q][0];
      const float* c1 = acc[q][1];
      float* mine = red[warp] + q * 128;
      *reinterpret_cast<float2*>(mine + g * 8 + 2 * t4) = make_float2(c0[0] + c1[0], c0[1] + c1[1]);
      *reinterpret_cast<float2*>(mine + (g + 8) * 8 + 2 * t4) = make_float2(c0[2] + c1[2], c0[3] + c1[3]);
    }
    if (tid == 0) sh.unit[(n + 2) & 3] = ticket;
    __syncthreads();
    auto sum_of = [&](int idx) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < kMfWarps; ++i) v += red[i][idx];
      return v;
    };
    if (up) {
      ++done_units;
      const int c = tid & 7, p = tid >> 3;                 // inner column, token of the expert
      if (p < ntok) {
        const int idx = (p >> 3) * 128 + c * 8 + (p & 7), pair = sh.slot_off[us] + p;
        const float gate = sum_of(idx), upv = sum_of(idx + 64);
        const float v = gate / (1.f + __expf(-gate)) * upv * sh.pair_w[pair];
        // a finite value may round up to infinity: cut instead, the remainder has the rest. Infinity has no remainder.
        __nv_bfloat16 h = __float2bfloat16_rn(v);
        if (__hisinf(h)) h = __float2bfloat16_rz(v);
        __nv_bfloat16* dst = a.act + (size_t)pair * a.I + (u - us * col_blocks) * 8 + c;
        dst[0] = h;
        dst[act_rows * a.I] = __float2bfloat16_rn(__hisinf(h) ? 0.f : v - __bfloat162float(h));
      }
    } else {
      const int r = tid & 15, t = tid >> 4, h = (u - n_up) * 16 + r;   // output row, token
      if (t < a.T && h < a.H) {
        const int idx = (t >> 3) * 128 + r * 8 + (t & 7);
        float v = sum_of(idx);
        if (PAIR) v += sum_of(idx + 4);
        a.out[t * a.ldo + h] = __float2bfloat16_rn(dead ? NAN : v);
      }
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
                    w.device() == x.device() && reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0,
                "moe_layer: expert weights must be packed bf16 tensors [*, 64] on x's device");
  const int64_t local = gate_up.size(0) / gu_rows;
  TORCH_CHECK(local >= 1 && gate_up.size(0) == local * gu_rows && down.size(0) == local * dn_rows,
              "moe_layer: packed expert weights have the wrong shape");
  B200_REQUIRE(first_expert >= 0 && first_expert + local <= E,
               "moe_layer: experts [" + std::to_string(first_expert) + ", " + std::to_string(first_expert + local) +
                   ") are not among the router's " + std::to_string(E));
  TORCH_CHECK(out.dim() == 2 && out.size(0) == T && out.size(1) == H && out.scalar_type() == at::kBFloat16 &&
                  out.stride(1) == 1 && (T <= 1 || out.stride(0) >= H) && out.device() == x.device(),
              "moe_layer: out must be a bf16 tensor [T, H] on x's device whose rows do not overlap");
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
  const int device = x.get_device();
  TORCH_CHECK(device < kMfMaxDevices, "moe_layer: devices 0 to 63");
  a.err = mf_error_words() + device;
  a.wait_ns = flag_wait_ns();
  auto stream = at::cuda::getCurrentCUDAStream();
  const __nv_bfloat16* rp = reinterpret_cast<const __nv_bfloat16*>(router.data_ptr());
  const dim3 rg((unsigned)E, (unsigned)((T + 3) / 4)), rb(kMfRouterThreads);
  if (T <= 1) launch_pdl(moe_router_kernel<1>, rg, rb, 0, stream, rp, a, logits, a.counters);
  else launch_pdl(moe_router_kernel<4>, rg, rb, 0, stream, rp, a, logits, a.counters);
  auto kernel = T <= 4 ? moe_few_kernel<1, true> : T <= 8 ? moe_few_kernel<1, false> : moe_few_kernel<2, false>;
  const int64_t units = std::min<int64_t>(T * k, local) * (I / 8) + (H + 15) / 16;
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const size_t smem = T <= 8 ? sizeof(MfShared<1>) : sizeof(MfShared<2>);
  B200_REQUIRE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  launch_pdl(kernel, dim3((unsigned)std::min<int64_t>(units, 2 * sms)), dim3(kMfThreads), smem, stream,
             reinterpret_cast<const __nv_bfloat16*>(gate_up.data_ptr()),
             reinterpret_cast<const __nv_bfloat16*>(down.data_ptr()), a);
}

int64_t moe_layer_error(bool reset) {
  int* words = g_mf_words;
  if (words == nullptr) return 0;                // no call so far
  volatile int* word = words + c10::cuda::current_device();
  const int v = *word;
  if (reset && v) *word = 0;
  return v;
}
