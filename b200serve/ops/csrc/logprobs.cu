// Log probabilities of given tokens from logits in memory: per row the token's log probability and
// rank, the entropy of the distribution, and the `top` most likely tokens (ties: the lowest id).
//
// One pass over the logits, in two kernels chained by programmatic dependent launch:
//   * logprob_slices: one CTA of 256 threads per (row, slice). A thread keeps its 32 logits
//     of the slice in registers, so the maximum, the sums, the rank count and the selection all
//     work on one read. With rows for every SM it is bound by instruction issue (about 25 a logit):
//     256 x 248320 fp32 with top 20 take 82 us, 3.1 TB/s.
//   * logprob_rows: one CTA per row joins the slices' statistics and merges their sorted lists.
//
// Selection. With the slice's logits in 32 groups (a lane of every warp), the `top`-th largest group
// maximum is at most the `top`-th largest logit, and for logits in no particular order few more than
// `top` reach it (31 on average for 20 of 8192). One warp finds a value just below it by descending the
// bits of the order-preserving values under votes; only threads whose maximum reaches the value look
// at their logits again and push what reaches it into a list, which is ranked by counting. The rank
// goes by a 64-bit key (value bits, then the complement of the id), so keys are unique and "ties: the
// lowest id" is the key order. Where more than the list holds reach the value (equal or sorted
// logits), the threshold is the `top`-th largest of the 256 per-thread largest keys instead: at most
// `top` threads' logits lie at or above it, for any data. The row kernel selects among the slices'
// lists the same way, from the lists' heads.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "logprobs.cuh"
#include "tma_host.h"

namespace b200 {

constexpr int kLpThreads = 256;
constexpr int kLpValues = 32;            // logits per thread

// order-preserving bits of a logit; 0 for anything that is never an alternative (-inf, NaN)
__device__ __forceinline__ uint32_t logit_bits(float x) {
  x += 0.f;                              // -0 and +0 are equal logits
  const uint32_t u = __float_as_uint(x);
  return x > -INFINITY ? u ^ ((uint32_t)((int)u >> 31) | 0x80000000u) : 0u;
}
__device__ __forceinline__ float logit_of_bits(uint32_t b) {
  return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ unsigned long long logit_key(float x, int id) {
  const uint32_t b = logit_bits(x);
  return b ? ((unsigned long long)b << 32) | (uint32_t)~id : 0ull;
}

struct LpArgs {
  const void* logits;
  long long ld;                          // elements between rows
  int V, S, top;                         // vocabulary, slices per row, alternatives
  TokenIds tokens;
  float4* part;                          // [B][S] (m, r, t, count of logits above the token's)
  unsigned long long* keys;              // [B][S][top] descending, 0 = none
};

// T = float or __nv_bfloat16. 32 logits per thread in 64 registers, four CTAs per SM: 16 of them took 114 us instead of
// 80 for 256 x 248320 fp32 with top 20 (twice the selections), 64 of them 127 instead of 97 in bf16 (half the CTAs).
template <typename T>
__global__ void __launch_bounds__(kLpThreads, 4) logprob_slices_kernel(const LpArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T), NV = kLpValues, U = NV / VEC, SLICE = kLpThreads * NV, WARPS = kLpThreads / 32;
  constexpr int CAP = kMaxTop * NV;
  __shared__ float red[WARPS][4];
  __shared__ uint32_t tmax[kLpThreads];
  __shared__ unsigned long long tkey[kLpThreads];
  __shared__ unsigned long long list[CAP];
  __shared__ float thr_s;
  __shared__ unsigned long long thr_key_s;
  __shared__ int count_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long row = blockIdx.x / a.S;
  const int slice = blockIdx.x % a.S;
  pdl_wait();
  pdl_trigger();
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  // 16-byte pieces are counted from the last aligned address at or before the row
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int base = slice * SLICE - shift + tid * VEC;  // id of this thread's first element (may be < 0)
  auto id_of = [&](int i) { return base + (i / VEC) * kLpThreads * VEC + i % VEC; };
  const int tok = token_id(a.tokens, row, a.V);
  const float xt = tok >= 0 ? (float)x[tok] : INFINITY;

  // all of the slice lies in the row (the first and the last may not)
  const bool inside = slice * SLICE >= shift && (slice + 1) * SLICE - shift <= a.V;

  float v[NV];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int id0 = id_of(u * VEC);
    if (inside || (id0 >= 0 && id0 + VEC <= a.V)) {
      const uint4 w = *reinterpret_cast<const uint4*>(x + id0);
      if constexpr (VEC == 4) {
        v[u * 4 + 0] = __uint_as_float(w.x); v[u * 4 + 1] = __uint_as_float(w.y);
        v[u * 4 + 2] = __uint_as_float(w.z); v[u * 4 + 3] = __uint_as_float(w.w);
      } else {
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[u * VEC + 2 * i] = bf16_lo(ws[i]); v[u * VEC + 2 * i + 1] = bf16_hi(ws[i]); }
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        v[u * VEC + i] = (id0 + i >= 0 && id0 + i < a.V) ? (float)x[id0 + i] : -INFINITY;
    }
  }

  // ---- maximum of the slice
  float tm = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) tm = fmaxf(tm, v[i]);
  const float wm = warp_max(tm);
  if (lane == 0) red[warp][3] = wm;
  if (a.top > 0) {
    tmax[tid] = logit_bits(tm);
    if (tid == 0) count_s = 0;
  }
  __syncthreads();
  float m = red[0][3];
#pragma unroll
  for (int i = 1; i < WARPS; ++i) m = fmaxf(m, red[i][3]);

  // ---- threshold (the other warps go on with the sums)
  if (a.top > 0 && warp == WARPS - 1) {
    uint32_t k = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) k = max(k, tmax[i * 32 + lane]);
    const uint32_t any = __reduce_or_sync(0xffffffffu, k), all = __reduce_and_sync(0xffffffffu, k);
    // the bits above the highest one in which the maxima differ are common to all of them
    int bit = 31 - __clz((any & ~all) | 1u);
    uint32_t thr = bit == 31 ? 0u : all >> (bit + 1) << (bit + 1);
    for (; bit >= 0; --bit) {
      const uint32_t c = thr | (1u << bit);
      const int n = __popc(__ballot_sync(0xffffffffu, k >= c));
      if (n >= a.top) {
        thr = c;
        if (n <= a.top + 1) break;
      }
    }
    // 0: fewer than `top` groups hold a logit above -inf; all logits are candidates
    if (lane == 0) thr_s = thr == 0u ? -3.402823466e38f : logit_of_bits(thr);
  }

  // ---- sums and the count of logits that rank before the token
  const float mm = m == -INFINITY ? 0.f : m;
  float s = 0.f, t = 0.f;
  int cnt = 0;
  bool equal = false;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const float d = v[i] - mm;
    const float e = ex2(d * 1.4426950408889634f);
    s += e;
    t = fmaf(e, fmaxf(d, -1e30f), t);                  // a masked logit: e = 0, d = -inf
    cnt += v[i] > xt;
    equal |= v[i] == xt;
  }
  if (equal) {
#pragma unroll
    for (int i = 0; i < NV; ++i)                       // padding outside the row is -inf too: only ids of the row count
      cnt += v[i] == xt && id_of(i) >= 0 && id_of(i) < tok;
  }
  s = warp_sum(s);
  t = warp_sum(t);
  if (__any_sync(0xffffffffu, tm == m)) {
    // the maximum's own terms are counted in the upper half of cnt and leave the sum: by subtraction, or, where that
    // would cost the others' bits, by another sum of the others
    if (s < 2.f && m > -INFINITY) {
      s = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (v[i] == m) cnt += 1 << 16;
        else s += ex2((v[i] - m) * 1.4426950408889634f);
      }
      s = warp_sum(s);
    } else {
      s -= 1.f;
      if (lane == 0) cnt += 1 << 16;
    }
  }
  cnt = __reduce_add_sync(0xffffffffu, cnt);
  if (lane == 0) { red[warp][0] = s; red[warp][1] = t; red[warp][2] = __int_as_float(cnt); }
  __syncthreads();
  if (tid == 0) {
    float bs = 0.f, bt = 0.f;
    int bc = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) { bs += red[i][0]; bt += red[i][1]; bc += __float_as_int(red[i][2]); }
    // a NaN marks the row through m = +inf
    a.part[row * a.S + slice] = make_float4(bs == bs ? m : INFINITY, bs + (float)((bc >> 16) - 1), bt,
                                            __int_as_float(bc & 0xffff));
  }
  if (a.top == 0) return;

  // ---- candidates (the order of the list does not matter)
  const float thr = thr_s;
  if (tm >= thr) {
    // a mask without branches first; the few logits in it are read again (registers have no index)
    uint32_t hit = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (v[i] >= thr) hit |= 1u << i;
    for (; hit; hit &= hit - 1u) {
      const int id = id_of(__ffs(hit) - 1);
      const int p = atomicAdd(&count_s, 1);
      if (p < CAP) list[p] = logit_key((float)x[id], id);
    }
  }
  __syncthreads();
  if (count_s > CAP) {
    // a thread's largest key is its maximum at the lowest id that holds it
    int at = 0;
#pragma unroll
    for (int i = NV - 1; i >= 0; --i)
      if (v[i] == tm) at = id_of(i);
    const unsigned long long mine = logit_key(tm, at);
    tkey[tid] = mine;
    __syncthreads();
    if (tid == 0) { count_s = 0; thr_key_s = 1ull; }   // 1: fewer than `top` threads hold a logit: all logits
    __syncthreads();
    int above = 0;
    for (int j = 0; j < kLpThreads; ++j) above += tkey[j] > mine;
    if (mine && above == a.top - 1) thr_key_s = mine;
    __syncthreads();
    const unsigned long long key = thr_key_s;
    if (mine >= key) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const unsigned long long k = logit_key(v[i], id_of(i));
        if (k >= key) {
          const int p = atomicAdd(&count_s, 1);
          if (p < CAP) list[p] = k;
        }
      }
    }
    __syncthreads();
  }
  const int n = min(count_s, CAP);
  unsigned long long* out = a.keys + (row * a.S + slice) * a.top;
  for (int i = tid; i < n; i += kLpThreads) {
    const unsigned long long k = list[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += list[j] > k;
    if (r < a.top) out[r] = k;
  }
  for (int i = n + tid; i < a.top; i += kLpThreads) out[i] = 0ull;
}

struct LpOut {
  float* logprob;                        // [B]
  int* rank;                             // [B]
  float* entropy;                        // [B]
  int* top_ids;                          // [B][top]
  float* top_lp;                         // [B][top]
};

// One CTA of 256 threads per row. Warp 0 joins the statistics. With S lists of `top` keys, sorted, the
// r-th largest of the d-th entries, d = max(1, ceil(top / S)) and r = ceil(top / d), has at least
// r d >= top keys at or above it: what reaches it is collected and ranked by counting.
constexpr int kLpRowThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kLpRowThreads) logprob_rows_kernel(const LpArgs a, const LpOut o) {
  extern __shared__ unsigned long long lists[];        // [S][top], then the candidates [S][top]
  __shared__ unsigned long long thr_s;
  __shared__ int count_s;
  __shared__ float max_s, log_s_s;
  const int tid = threadIdx.x, lane = tid & 31, total = a.S * a.top;
  const long long row = blockIdx.x;
  if (tid == 0) { thr_s = 0ull; count_s = 0; }
  pdl_wait();
  pdl_trigger();
  const unsigned long long* src = a.keys + row * total;
  for (int i = tid; i < total; i += kLpRowThreads) lists[i] = __ldcg(src + i);
  if (tid < 32) {
    RowStat r{-INFINITY, 0.f, 0.f};
    int cnt = 0;
    for (int i = lane; i < a.S; i += 32) {
      const float4 p = __ldcg(a.part + row * a.S + i);
      stat_merge(r, RowStat{p.x, p.y, p.z});
      cnt += __float_as_int(p.w);
    }
    r = stat_warp_merge(r);
    cnt = __reduce_add_sync(0xffffffffu, cnt);
    if (lane == 0) {
      const bool ok = stat_valid(r);
      const float log_s = ok ? stat_log(r) : NAN;
      const int tok = token_id(a.tokens, row, a.V);
      const float xt = tok >= 0 ? (float)(static_cast<const T*>(a.logits) + row * a.ld)[tok] : NAN;
      o.logprob[row] = (xt - r.m) - log_s;
      o.rank[row] = ok && tok >= 0 ? cnt : -1;
      o.entropy[row] = ok ? stat_entropy(r) : NAN;
      max_s = r.m;
      log_s_s = log_s;
    }
  }
  if (a.top == 0) return;
  __syncthreads();
  const int d = a.S >= a.top ? 1 : (a.top + a.S - 1) / a.S, r = (a.top + d - 1) / d;
  for (int i = tid; i < a.S; i += kLpRowThreads) {
    const unsigned long long h = lists[i * a.top + d - 1];
    int above = 0;
    for (int j = 0; j < a.S; ++j) above += lists[j * a.top + d - 1] > h;
    if (h && above == r - 1) thr_s = h;                // keys are unique: one thread at most
  }
  __syncthreads();
  const unsigned long long thr = thr_s ? thr_s : 1ull; // too few entries: all of them
  unsigned long long* cand = lists + total;
  for (int i = tid; i < total; i += kLpRowThreads)
    if (lists[i] >= thr) cand[atomicAdd(&count_s, 1)] = lists[i];
  __syncthreads();
  const int n = count_s;
  const float M = max_s, log_s = log_s_s;
  const bool ok = log_s == log_s;
  for (int i = tid; i < n; i += kLpRowThreads) {
    const unsigned long long k = cand[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += cand[j] > k;
    if (above < a.top) {
      o.top_ids[row * a.top + above] = ok ? (int)~(uint32_t)k : -1;
      o.top_lp[row * a.top + above] = ok ? (logit_of_bits((uint32_t)(k >> 32)) - M) - log_s : NAN;
    }
  }
  for (int i = n + tid; i < a.top; i += kLpRowThreads) {
    o.top_ids[row * a.top + i] = -1;
    o.top_lp[row * a.top + i] = ok ? -INFINITY : NAN;
  }
}

}  // namespace b200

using namespace b200;

// logits [B, V] fp32 or bf16 (unit stride along V), tokens [B] int32 or int64. Returns
// (logprob [B], rank [B], entropy [B], top_ids [B, top], top_logprobs [B, top]).
std::vector<torch::Tensor> token_logprobs(torch::Tensor logits, torch::Tensor tokens, int64_t top) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "token_logprobs: logits must be a CUDA tensor [B, V]");
  const bool bf = logits.scalar_type() == at::kBFloat16;
  TORCH_CHECK(bf || logits.scalar_type() == at::kFloat, "token_logprobs: logits must be fp32 or bf16");
  const int64_t B = logits.size(0), V = logits.size(1);
  B200_REQUIRE(V >= 1 && V <= (1 << 20), "token_logprobs: vocabulary of 1 to 1048576 tokens, got " + std::to_string(V));
  TORCH_CHECK(V == 1 || logits.stride(1) == 1, "token_logprobs: logits need unit stride along the vocabulary");
  TORCH_CHECK(tokens.dim() == 1 && tokens.size(0) == B && tokens.device() == logits.device() &&
                  tokens.is_contiguous() && (tokens.scalar_type() == at::kInt || tokens.scalar_type() == at::kLong),
              "token_logprobs: tokens must be contiguous int32 or int64 [B] on the logits' device");
  B200_REQUIRE(top >= 0 && top <= kMaxTop, "token_logprobs: top must be 0 to 32, got " + std::to_string(top));
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat), i32 = logits.options().dtype(at::kInt);
  auto logprob = torch::empty({B}, f32), entropy = torch::empty({B}, f32), top_lp = torch::empty({B, top}, f32);
  auto rank = torch::empty({B}, i32), top_ids = torch::empty({B, top}, i32);
  std::vector<torch::Tensor> res = {logprob, rank, entropy, top_ids, top_lp};
  if (B == 0) return res;
  const int64_t worst = V + (bf ? 7 : 3);               // a row may start inside a 16-byte piece
  const int64_t per = kLpThreads * kLpValues;
  LpArgs a{};
  a.logits = logits.data_ptr();
  a.ld = B > 1 ? logits.stride(0) : V;
  a.V = (int)V; a.S = (int)((worst + per - 1) / per); a.top = (int)top;
  TORCH_CHECK(B * a.S < (1ll << 31), "token_logprobs: too many rows");
  a.tokens = TokenIds{tokens.data_ptr(), tokens.scalar_type() == at::kLong};
  // partial results of this call: 16 bytes and `top` keys per slice
  auto ws = torch::empty({B * a.S * (2 + top)}, logits.options().dtype(at::kLong));
  a.part = reinterpret_cast<float4*>(ws.data_ptr());
  a.keys = reinterpret_cast<unsigned long long*>(a.part + B * a.S);
  LpOut o{logprob.data_ptr<float>(), rank.data_ptr<int>(), entropy.data_ptr<float>(), top_ids.data_ptr<int>(),
          top_lp.data_ptr<float>()};
  auto stream = at::cuda::getCurrentCUDAStream();
  const dim3 grid((unsigned)(B * a.S));
  if (bf) launch_pdl(logprob_slices_kernel<__nv_bfloat16>, grid, dim3(kLpThreads), 0, stream, a);
  else launch_pdl(logprob_slices_kernel<float>, grid, dim3(kLpThreads), 0, stream, a);
  const size_t smem = (size_t)a.S * top * 16;           // at most 129 slices of 32 keys, twice
  if (smem > 40 * 1024)
    B200_REQUIRE_CUDA(cudaFuncSetAttribute(bf ? logprob_rows_kernel<__nv_bfloat16> : logprob_rows_kernel<float>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, 72 * 1024));
  if (bf) launch_pdl(logprob_rows_kernel<__nv_bfloat16>, dim3((unsigned)B), dim3(kLpRowThreads), smem, stream, a, o);
  else launch_pdl(logprob_rows_kernel<float>, dim3((unsigned)B), dim3(kLpRowThreads), smem, stream, a, o);
  return res;
}
