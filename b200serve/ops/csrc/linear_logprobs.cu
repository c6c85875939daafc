// Log probability of a given token and entropy of the next-token distribution for every row of
// hidden states, straight from the LM head: the logits x w^T (softcap * tanh(. / softcap) where
// the model caps them) never reach memory.
//
//   linear_logprobs: a persistent tcgen05 GEMM. The hidden states are the MMA's A operand (128
//   rows = the 128 TMEM lanes), a tile of the vocabulary its B operand (tile_n <= 256 rows = TMEM
//   columns), so a thread of the epilogue owns a row and sums up a slice's maximum and exponential
//   sums in registers, with no exchange between threads. Per (row, tile half) 16 bytes are
//   written instead of 4 * tile_n of logits.
//   linear_logprob_rows: joins the slices of every row.
//
// Roles (320 threads): warp 0 TMA producer, warp 1 MMA issuer, warps 2..9 epilogue (two per TMEM
// lane quarter, each one half of the tile's columns). The accumulator is double-buffered in TMEM, so
// the epilogue of one tile runs under the MMAs of the next.
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

constexpr int kLlBM = 128, kLlBN = 256, kLlBK = 64, kLlStages = 4, kLlThreads = 320;
constexpr int kLlA = kLlBM * kLlBK * 2, kLlW = kLlBN * kLlBK * 2, kLlStage = kLlA + kLlW;
constexpr size_t kLlSmem = 1024 + (size_t)kLlStages * kLlStage + 256;
constexpr float kLlMasked = -1e30f;      // columns past the vocabulary: e^(x - m) is 0, products stay finite
constexpr int64_t kLlRows = 8192;        // rows per pass: bounds the partial results (16 bytes per row and slice)

static __device__ int g_ll_err;          // first error code of the bounded waits, one word per device

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct LlArgs {
  int T, V, kb_total, m_tiles, v_tiles, tile_n, box_rows;
  int packed;                            // w: tile-packed [n_tile][k_block][128][64], else plain [V, H]
  float softcap;
  TokenIds tokens;
  float4* part;                          // [2 v_tiles][T] (m, s, t, the token's logit where the slice has it)
};

template <bool CAP>
__global__ void __launch_bounds__(kLlThreads, 1)
    linear_logprobs_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                           const LlArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_x = smem;
  uint8_t* s_w = smem + kLlStages * kLlA;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kLlStages * kLlStage);
  uint64_t* empty = full + kLlStages;
  uint64_t* tfull = empty + kLlStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* mma_done = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = a.m_tiles * a.v_tiles;
  int* err = &g_ll_err;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kLlStages; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 1); }
    for (int i = 0; i < 2; ++i) { tc::mbar_init(&tfull[i], 1); tc::mbar_init(&tempty[i], 8); }
    tc::mbar_init(mma_done, 1);
    *abort_flag = 0;
    tc::fence_barrier_init();
    tc::fence_proxy_async_smem();
    tc::prefetch_tmap(&tm_x);
    tc::prefetch_tmap(&tm_w);
  }
  __syncwarp();
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer ----------------
      const uint64_t pol_w = tc::policy_evict_first(), pol_x = tc::policy_evict_last();
      const uint32_t bytes = kLlA + a.tile_n * kLlBK * 2;
      int stage = 0;
      uint32_t phase = 0;
      for (int u = blockIdx.x; u < units && !*abort_flag; u += gridDim.x) {
        const int m0 = (u % a.m_tiles) * kLlBM, v0 = (u / a.m_tiles) * a.tile_n;
        for (int kb = 0; kb < a.kb_total; ++kb) {
          if (!tc::mbar_wait_bounded(&empty[stage], phase ^ 1, abort_flag, err, 11)) break;
          tc::mbar_arrive_expect_tx(&full[stage], bytes);
          tc::tma_load_2d(s_x + stage * kLlA, &tm_x, &full[stage], kb * kLlBK, m0, pol_x);
          for (int r = 0; r < a.tile_n; r += a.box_rows) {
            const int v = v0 + r;
            const int y = a.packed ? ((v >> 7) * a.kb_total + kb) * 128 + (v & 127) : v;
            tc::tma_load_2d(s_w + stage * kLlW + r * 128, &tm_w, &full[stage], a.packed ? 0 : kb * kLlBK, y, pol_w);
          }
          if (++stage == kLlStages) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------- MMA issuer ----------------
      const uint32_t idesc = tc::idesc_bf16_f32(kLlBM, a.tile_n);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      for (int u = blockIdx.x; u < units && !*abort_flag; u += gridDim.x) {
        if (!tc::mbar_wait_bounded(&tempty[acc], acc_phase ^ 1, abort_flag, err, 12)) break;
        tc::tc_fence_after();
        const uint32_t d = tmem_base + acc * kLlBN;
        for (int kb = 0; kb < a.kb_total; ++kb) {
          if (!tc::mbar_wait_bounded(&full[stage], phase, abort_flag, err, 13)) break;
          tc::tc_fence_after();
          const uint64_t da = tc::sw128_kmajor_desc(tc::smem_u32(s_x + stage * kLlA));
          const uint64_t db = tc::sw128_kmajor_desc(tc::smem_u32(s_w + stage * kLlW));
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) tc::mma_bf16(d, da + 2 * kk, db + 2 * kk, idesc, (kb | kk) ? 1u : 0u);
          tc::mma_commit(&empty[stage]);
          if (++stage == kLlStages) { stage = 0; phase ^= 1; }
        }
        tc::mma_commit(&tfull[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      // no tcgen05.mma may still be running when TMEM is released below
      tc::mma_commit(mma_done);
      volatile int never = 0;
      tc::mbar_wait_bounded(mma_done, 0, &never, err, 15);
    }
    __syncwarp();
  } else {
    // ---------------- epilogue (warps 2..9) ----------------
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const int c_lo = half ? (a.tile_n / 32) * 16 : 0;      // columns of this half, multiples of 16
    const int c_hi = half ? a.tile_n : (a.tile_n / 32) * 16;
    const float L2E = 1.4426950408889634f;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int u = blockIdx.x; u < units && !*abort_flag; u += gridDim.x) {
      const int row = (u % a.m_tiles) * kLlBM + quad * 32 + lane;
      const int v_tile = u / a.m_tiles, v0 = v_tile * a.tile_n;
      const int tok = row < a.T ? token_id(a.tokens, row, a.V) : -1;
      if (!tc::mbar_wait_bounded(&tfull[acc], acc_phase, abort_flag, err, 14)) break;
      tc::tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(quad * 32) << 16) + acc * kLlBN;
      RowStat r{kLlMasked, 0.f, 0.f};
      float xt = 0.f;
      for (int c0 = c_lo; c0 < c_hi; c0 += 16) {
        float v[16];
        tc::tmem_ld16(t_row + c0, v);
        if constexpr (CAP) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = a.softcap * tanhf(v[j] / a.softcap);
        }
        if (v0 + c0 + 16 > a.V) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (v0 + c0 + j >= a.V) v[j] = kLlMasked;
        }
        const int at = tok - (v0 + c0);
        if ((unsigned)at < 16u) {
#pragma unroll
          for (int j = 0; j < 16; ++j) xt = j == at ? v[j] : xt;
        }
        float m = r.m;
#pragma unroll
        for (int j = 0; j < 16; ++j) m = fmaxf(m, v[j]);
        const float dm = r.m - m, sc = ex2(dm * L2E);
        float s = 0.f, t = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float d = v[j] - m;
          const float e = ex2(d * L2E);
          s += e;
          t = fmaf(e, fmaxf(d, kLlMasked), t);      // a logit of -inf: 0 * -1e30
        }
        r.t = fmaf(sc, fmaf(dm, r.s, r.t), t);
        r.s = fmaf(sc, r.s, s);
        r.m = m;
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&tempty[acc]);
      // a half without a column of the vocabulary, or without columns at all, holds nothing
      const bool some = c_lo < c_hi && v0 + c_lo < a.V;
      if (row < a.T)
        a.part[(size_t)(2 * v_tile + half) * a.T + row] =
            some ? make_float4(r.s == r.s ? r.m : INFINITY, r.s, r.t, xt) : make_float4(-INFINITY, 0.f, 0.f, 0.f);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
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
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem_base, 512);
  }
}

// 256 threads per CTA on R rows (32: lane = row; 1: the CTA's threads share a row's slices)
constexpr int kLlRowThreads = 256;
template <int R>
__global__ void __launch_bounds__(kLlRowThreads) linear_logprob_rows_kernel(const LlArgs a, float* __restrict__ logprob,
                                                                            float* __restrict__ entropy) {
  constexpr int G = kLlRowThreads / R;                 // threads per row
  __shared__ RowStat st[G][R];
  pdl_wait();
  pdl_trigger();
  const int r = threadIdx.x % R, g = threadIdx.x / R;
  const int row = blockIdx.x * R + r;
  const int S = 2 * a.v_tiles;
  RowStat acc{-INFINITY, 0.f, 0.f};
  if (row < a.T) {
#pragma unroll 4
    for (int i = g; i < S; i += G) {
      const float4 p = __ldcg(a.part + (size_t)i * a.T + row);
      stat_merge(acc, RowStat{p.x, p.y, p.z});
    }
  }
  st[g][r] = acc;
  __syncthreads();
  if constexpr (R == 1) {
    if (threadIdx.x >= 32) return;
    acc = st[threadIdx.x][0];
    for (int i = threadIdx.x + 32; i < G; i += 32) stat_merge(acc, st[i][0]);
    acc = stat_warp_merge(acc);
    if (threadIdx.x != 0) return;
  } else {
    if (g != 0 || row >= a.T) return;
    for (int i = 1; i < G; ++i) stat_merge(acc, st[i][r]);
  }
  const bool ok = stat_valid(acc);
  const int tok = token_id(a.tokens, row, a.V);
  float xt = NAN;
  if (tok >= 0) {
    const int v_tile = tok / a.tile_n;
    const int half = tok - v_tile * a.tile_n >= (a.tile_n / 32) * 16;
    xt = __ldcg(&a.part[(size_t)(2 * v_tile + half) * a.T + row].w);
  }
  logprob[row] = ok ? (xt - acc.m) - logf(acc.s) : NAN;
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
  const int64_t ldx = T > 1 ? x.stride(0) : H;
  TORCH_CHECK(ldx % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0,
              "linear_logprobs: rows of x must start on 16-byte boundaries");

  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  auto stream = at::cuda::getCurrentCUDAStream();
  auto kernel = softcap > 0.0 ? linear_logprobs_kernel<true> : linear_logprobs_kernel<false>;
  B200_REQUIRE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kLlSmem));
  torch::Tensor part;
  for (int64_t t0 = 0; t0 < T; t0 += kLlRows) {
    LlArgs a{};
    a.T = (int)std::min(kLlRows, T - t0); a.V = (int)V; a.kb_total = kb; a.packed = packed;
    a.m_tiles = (a.T + kLlBM - 1) / kLlBM;
    // columns per tile: of the multiples of 16 from 128 to 256 the one whose busiest CTA has the
    // fewest columns to compute (ties: the widest, which reads x least often)
    int64_t best = INT64_MAX;
    for (int n = kLlBN; n >= 128; n -= 16) {
      const int64_t units = (int64_t)a.m_tiles * ((V + n - 1) / n);
      const int64_t cost = (units + sms - 1) / sms * n;
      if (cost < best) { best = cost; a.tile_n = n; }
    }
    a.v_tiles = (int)((V + a.tile_n - 1) / a.tile_n);
    // rows per box: a divisor of the tile that keeps a box inside one 128-row weight tile
    a.box_rows = std::min(a.tile_n & -a.tile_n, 128);
    a.softcap = (float)softcap;
    const bool is64 = tokens.scalar_type() == at::kLong;
    a.tokens = TokenIds{static_cast<const char*>(tokens.data_ptr()) + t0 * (is64 ? 8 : 4), is64};
    const int64_t need = 2 * (int64_t)a.v_tiles * a.T * 4;
    if (!part.defined() || part.numel() < need) part = torch::empty({need}, logprob.options());
    a.part = reinterpret_cast<float4*>(part.data_ptr());
    const void* xp = static_cast<const __nv_bfloat16*>(x.data_ptr()) + t0 * ldx;
    const uint64_t xd[2] = {(uint64_t)H, (uint64_t)a.T}, xs[1] = {(uint64_t)ldx * 2};
    const uint32_t xb[2] = {64, kLlBM};
    const uint64_t wd[2] = {packed ? 64ull : (uint64_t)H, (uint64_t)w.size(0)}, ws[1] = {(packed ? 64 : H) * 2ull};
    const uint32_t wb[2] = {64, (uint32_t)a.box_rows};
    const CUtensorMap tx = tma_bf16(xp, 2, xd, xs, xb), tw = tma_bf16(w.data_ptr(), 2, wd, ws, wb);
    const int64_t units = (int64_t)a.m_tiles * a.v_tiles;
    const unsigned grid = (unsigned)std::min<int64_t>(units, sms);
    launch_pdl(kernel, dim3(grid), dim3(kLlThreads), kLlSmem, stream, tx, tw, a);
    float* lp = logprob.data_ptr<float>() + t0;
    float* en = entropy.data_ptr<float>() + t0;
    if (a.T >= 64)
      launch_pdl(linear_logprob_rows_kernel<32>, dim3((unsigned)((a.T + 31) / 32)), dim3(kLlRowThreads), 0, stream, a,
                 lp, en);
    else
      launch_pdl(linear_logprob_rows_kernel<1>, dim3((unsigned)a.T), dim3(kLlRowThreads), 0, stream, a, lp, en);
  }
  return {logprob, entropy};
}

int64_t linear_logprobs_error(bool reset) {
  int v = 0;
  B200_REQUIRE_CUDA(cudaMemcpyFromSymbol(&v, g_ll_err, sizeof(int)));
  if (reset) {
    const int z = 0;
    B200_REQUIRE_CUDA(cudaMemcpyToSymbol(g_ll_err, &z, sizeof(int)));
  }
  return v;
}
