// Row statistics shared by the two log-probability kernels (logprobs.cu over logits in memory,
// linear_logprobs.cu over the product of hidden states and the LM head).
//
// A slice of a row's logits x is summed up as m = max x, s = sum e^(x-m), t = sum e^(x-m) (x-m).
// Slices join exactly: with M = max m_i and d_i = m_i - M,
//   s = sum e^d_i s_i,   t = sum e^d_i (t_i + d_i s_i),
//   log p(token) = (x_token - M) - log s,   entropy = log s - t / s.
// Kept is r = s - 1, the sum without the largest logit's own term, and log s = log1p(r): beside an almost certain
// token the others' small terms would lose their bits to the 1 (log p = -1e-4 would be off by 6e-4 of itself).
// Everything is fp32. The terms of s lie in [0, 1] and those of t in [-1/e, 0]. An exponential carries ex2's 2^-22 and
// the rounding of its argument d log2(e), 2^-23 |d| (|d| <= ln V where it matters), so log s is off by
// about (1 + ln V) 2^-22; the sums, of at most 64 terms in a row and joined in trees, add a few 2^-24.
#pragma once
#include "common.cuh"

namespace b200 {

constexpr int kMaxTop = 32;              // alternatives per row

// tokens [rows] int32 or int64; ids outside [0, V) mean "no token" and come back as -1
struct TokenIds {
  const void* ptr;
  int is64;
};

__device__ __forceinline__ int token_id(const TokenIds& t, long long row, int V) {
  const long long id = t.is64 ? static_cast<const long long*>(t.ptr)[row]
                              : (long long)static_cast<const int*>(t.ptr)[row];
  return id >= 0 && id < V ? (int)id : -1;
}

// 2^x, off by at most 2^-22 of its value
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct RowStat {
  float m, r, t;
};

// Adds slice (m, r, t) to `a`. m = -inf marks an empty slice. The differences are bounded so
// that a slice which does not count (all of it at the type's lowest value, say) adds e^d d s = 0, not 0 * -inf.
__device__ __forceinline__ void stat_merge(RowStat& a, const RowStat& b) {
  const float M = fmaxf(a.m, b.m);
  const float da = fmaxf(a.m - M, -1e30f), db = fmaxf(b.m - M, -1e30f);
  if (a.m == -INFINITY) {
    a = b;
  } else if (b.m != -INFINITY) {
    const float ea = __expf(da), eb = __expf(db);
    a.t = ea * (a.t + da * (1.f + a.r)) + eb * (b.t + db * (1.f + b.r));
    a.r = ea * a.r + eb * b.r + fminf(ea, eb);           // the larger maximum's own term stays out
    a.m = M;
  }
}

__device__ __forceinline__ RowStat stat_warp_merge(RowStat a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    RowStat b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.r = __shfl_xor_sync(0xffffffffu, a.r, o);
    b.t = __shfl_xor_sync(0xffffffffu, a.t, o);
    stat_merge(a, b);
  }
  return a;
}

// A row has a distribution unless it holds a NaN or +inf (slices with a NaN are marked by m = +inf too) or nothing
// above -inf.
__device__ __forceinline__ bool stat_valid(const RowStat& a) { return a.m > -INFINITY && a.m < INFINITY; }

__device__ __forceinline__ float stat_log(const RowStat& a) { return log1pf(a.r); }
__device__ __forceinline__ float stat_entropy(const RowStat& a) { return fmaxf(0.f, log1pf(a.r) - a.t / (1.f + a.r)); }

}  // namespace b200
