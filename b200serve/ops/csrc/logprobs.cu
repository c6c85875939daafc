// Log probabilities of given tokens from logits in memory: per row the token's log probability and
// rank, the entropy of the distribution, and the `top` most likely tokens (ties: the lowest id).
//
// One pass over the logits, in two kernels chained by programmatic dependent launch:
//   * logprob_slices: one CTA of 256 threads per (row, slice). A thread keeps its 16-byte pieces
//     of the slice in registers, so the maximum, the sums, the rank count and the selection all
//     work on one read. Bound by HBM (4 or 2 bytes a logit) once there are rows for every SM.
//   * logprob_rows: one CTA per row joins the slices' statistics and merges their sorted lists.
//
// Selection. Logit and id make one 64-bit key (order-preserving bits of the value, then the
// complement of the id), so keys are unique and "ties: the lowest id" is the key order. The `top`-th
// largest of the 256 per-thread maxima is at most the `top`-th largest key of the slice; one warp
// finds a value with at least `top` and at most top + 12 maxima above it by descending the key
// bits. Only those threads push keys, at most 32 each, into a list that is ranked by counting. The
// bound on the list holds for any data (all logits equal, sorted rows), so no case needs a
// second way.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "logprobs.cuh"
#include "tma_host.h"

namespace b200 {

constexpr int kLpThreads = 256;
constexpr int kLpSlack = 12;             // accepted surplus of per-thread maxima above the threshold

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
  float4* part;                          // [B][S] (m, s, t, count of logits above the token's)
  unsigned long long* keys;              // [B][S][top] descending, 0 = none
};

// T = float or __nv_bfloat16; U 16-byte pieces per thread
template <typename T, int U>
__global__ void __launch_bounds__(kLpThreads) logprob_slices_kernel(const LpArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T), NV = U * VEC, SLICE = kLpThreads * NV;
  constexpr int CAP = (kMaxTop + kLpSlack) * NV;
  __shared__ float red[kLpThreads / 32][4];
  __shared__ unsigned long long tmax[kLpThreads];
  __shared__ unsigned long long list[CAP];
  __shared__ unsigned long long thr_s;
  __shared__ int count_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long row = blockIdx.x / a.S;
  const int slice = blockIdx.x % a.S;
  pdl_wait();
  pdl_trigger();
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  // 16-byte pieces are counted from the last aligned address at or before the row
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int base = slice * SLICE - shift;              // id of this slice's first element (may be < 0)
  const int tok = token_id(a.tokens, row, a.V);
  const float xt = tok >= 0 ? (float)x[tok] : INFINITY;

  float v[NV];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int id0 = base + (u * kLpThreads + tid) * VEC;
    if (id0 >= 0 && id0 + VEC <= a.V) {
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
  if (lane == 0) red[warp][0] = wm;
  // the thread's largest key: its maximum at the lowest id that holds it
  if (a.top > 0) {
    unsigned long long k = 0;
    if (tm > -INFINITY) {
      int at = 0;
#pragma unroll
      for (int i = NV - 1; i >= 0; --i)
        if (v[i] == tm) at = (i / VEC) * kLpThreads * VEC + i % VEC;
      k = logit_key(tm, base + tid * VEC + at);
    }
    tmax[tid] = k;
    if (tid == 0) count_s = 0;
  }
  __syncthreads();
  float m = red[0][0];
#pragma unroll
  for (int i = 1; i < kLpThreads / 32; ++i) m = fmaxf(m, red[i][0]);

  // ---- sums and the count of logits that rank before the token
  const float mm = m == -INFINITY ? 0.f : m;
  float s = 0.f, t = 0.f;
  int cnt = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int id = base + ((i / VEC) * kLpThreads + tid) * VEC + i % VEC;
    const float d = v[i] - mm;
    const float e = __expf(d);
    s += e;
    t += e * fmaxf(d, -1e30f);                         // a masked logit: e = 0, d = -inf
    cnt += v[i] > xt;
    // padding outside the row is -inf too: only ids of the row count
    if (v[i] == xt && id >= 0 && id < tok) ++cnt;
  }
  s = warp_sum(s);
  t = warp_sum(t);
  cnt = __reduce_add_sync(0xffffffffu, cnt);
  __syncthreads();                                     // red[][0] was read above
  if (lane == 0) { red[warp][0] = s; red[warp][1] = t; red[warp][2] = __int_as_float(cnt); }

  // ---- threshold: at least `top` per-thread maxima lie at or above it
  if (a.top > 0 && warp == 0) {
    unsigned long long k[kLpThreads / 32];
    uint32_t hi_or = 0, hi_and = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kLpThreads / 32; ++i) {
      k[i] = tmax[i * 32 + lane];
      hi_or |= (uint32_t)(k[i] >> 32);
      hi_and &= (uint32_t)(k[i] >> 32);
    }
    hi_or = __reduce_or_sync(0xffffffffu, hi_or);
    hi_and = __reduce_and_sync(0xffffffffu, hi_and);
    // bits above the highest differing one are common to all keys
    const uint32_t diff = hi_or & ~hi_and;
    int bit = diff ? 63 - __clz(diff) : 31;
    unsigned long long thr = bit == 63 ? 0ull : (((unsigned long long)hi_and << 32) >> (bit + 1)) << (bit + 1);
    for (; bit >= 0; --bit) {
      const unsigned long long c = thr | (1ull << bit);
      int n = 0;
#pragma unroll
      for (int i = 0; i < kLpThreads / 32; ++i) n += k[i] >= c;
      n = __reduce_add_sync(0xffffffffu, n);
      if (n >= a.top) {
        thr = c;
        if (n <= a.top + kLpSlack) break;
      }
    }
    if (lane == 0) thr_s = thr ? thr : 1ull;           // fewer than `top` threads hold a key: all keys
  }
  __syncthreads();
  if (tid == 0) {
    float bs = 0.f, bt = 0.f;
    int bc = 0;
#pragma unroll
    for (int i = 0; i < kLpThreads / 32; ++i) { bs += red[i][0]; bt += red[i][1]; bc += __float_as_int(red[i][2]); }
    // a NaN (of the data, or +inf - +inf) marks the row through m = +inf
    a.part[row * a.S + slice] = make_float4(bs == bs ? m : INFINITY, bs, bt, __int_as_float(bc));
  }
  if (a.top == 0) return;

  // ---- candidates
  const unsigned long long thr = thr_s;
  if (tmax[tid] >= thr) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const unsigned long long k = logit_key(v[i], base + ((i / VEC) * kLpThreads + tid) * VEC + i % VEC);
      if (k >= thr) {
        const int p = atomicAdd(&count_s, 1);          // the order of the list does not matter
        if (p < CAP) list[p] = k;
      }
    }
  }
  __syncthreads();
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

// One CTA of 128 threads per row. Warp 0 joins the statistics; the slices' sorted lists are
// staged in shared memory, lane l walks the heads of lists l, l + 32, ... and every round takes
// the largest head of the warp.
constexpr int kLpRowThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kLpRowThreads) logprob_rows_kernel(const LpArgs a, const LpOut o) {
  extern __shared__ unsigned long long lists[];        // [S][top], then one int per list
  int* head = reinterpret_cast<int*>(lists + (size_t)a.S * a.top);
  const int tid = threadIdx.x, lane = tid & 31;
  const long long row = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  const unsigned long long* src = a.keys + row * a.S * a.top;
  for (int i = tid; i < a.S * a.top; i += kLpRowThreads) lists[i] = __ldcg(src + i);
  if (a.top > 0)
    for (int i = tid; i < a.S; i += kLpRowThreads) head[i] = 0;
  __syncthreads();
  if (tid >= 32) return;
  RowStat r{-INFINITY, 0.f, 0.f};
  int cnt = 0;
  for (int i = lane; i < a.S; i += 32) {
    const float4 p = __ldcg(a.part + row * a.S + i);
    stat_merge(r, RowStat{p.x, p.y, p.z});
    cnt += __float_as_int(p.w);
  }
  r = stat_warp_merge(r);
  cnt = __reduce_add_sync(0xffffffffu, cnt);
  const bool ok = stat_valid(r);
  const float log_s = ok ? logf(r.s) : NAN;
  if (lane == 0) {
    const int tok = token_id(a.tokens, row, a.V);
    const float xt = tok >= 0 ? (float)(static_cast<const T*>(a.logits) + row * a.ld)[tok] : NAN;
    o.logprob[row] = (xt - r.m) - log_s;
    o.rank[row] = ok && tok >= 0 ? cnt : -1;
    o.entropy[row] = ok ? stat_entropy(r) : NAN;
  }
  for (int j = 0; j < a.top; ++j) {
    unsigned long long best = 0;
    int from = -1;
    for (int i = lane; i < a.S; i += 32) {
      const int h = head[i];
      const unsigned long long k = h < a.top ? lists[i * a.top + h] : 0ull;
      if (k > best) { best = k; from = i; }
    }
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
    if (from >= 0 && (uint32_t)(best >> 32) == hi && (uint32_t)best == lo) head[from] += 1;
    if (lane == 0) {
      const bool some = ok && hi != 0u;
      o.top_ids[row * a.top + j] = some ? (int)~lo : -1;
      o.top_lp[row * a.top + j] = some ? (logit_of_bits(hi) - r.m) - log_s : ok ? -INFINITY : NAN;
    }
  }
}

template <typename T, int U>
static void launch_slices(const LpArgs& a, int B, cudaStream_t stream) {
  launch_pdl(logprob_slices_kernel<T, U>, dim3((unsigned)(B * a.S)), dim3(kLpThreads), 0, stream, a);
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
  const int esize = bf ? 2 : 4, vec = 16 / esize;
  // 4 pieces a thread while that leaves at most two CTAs an SM (short slices: less work in a row
  // for each), else 8
  const int64_t worst = V + vec - 1;                    // a row may start inside a 16-byte piece
  const int64_t small = (int64_t)kLpThreads * 4 * vec;
  const int64_t s4 = (worst + small - 1) / small;
  const bool u4 = B * s4 <= 2 * 148 && s4 * (8 * top + 4) <= 48 * 1024;
  const int64_t per = u4 ? small : 2 * small;
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
  if (bf) {
    if (u4) launch_slices<__nv_bfloat16, 4>(a, (int)B, stream);
    else launch_slices<__nv_bfloat16, 8>(a, (int)B, stream);
  } else {
    if (u4) launch_slices<float, 4>(a, (int)B, stream);
    else launch_slices<float, 8>(a, (int)B, stream);
  }
  const size_t smem = top ? (size_t)a.S * top * 8 + (size_t)a.S * 4 : 0;
  if (bf) launch_pdl(logprob_rows_kernel<__nv_bfloat16>, dim3((unsigned)B), dim3(kLpRowThreads), smem, stream, a, o);
  else launch_pdl(logprob_rows_kernel<float>, dim3((unsigned)B), dim3(kLpRowThreads), smem, stream, a, o);
  return res;
}
