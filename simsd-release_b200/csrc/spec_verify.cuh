// Verification of drafted tokens against the target's distribution, from given
// random numbers.  For sequence b with d drafted tokens x_0 .. x_{d-1} and
// target rows 0 .. d:
//   p_i = softmax(target_i / T), q_i = softmax(draft_i / T), or one at x_i where
//   the draft gives no logits
//   x_i is kept while u_i q_i(x_i) < p_i(x_i); at the first one refused (row a)
//   the new token is argmax_v max(p_a - q_a, 0)(v) / e(v), after d kept ones
//   argmax_v p_d(v) / e(v), with e exponential noise: of independent exponential
//   variables e(v) / w(v) the smallest is v's with probability w(v) / sum w, so
//   this draws from the (residual) distribution without a running sum.
// T = 0: p and q are one at their first maximum.  NaN logits count as -inf,
// +inf as the largest finite number; a row without any finite logit has p = 0.
// Ties go to the lowest token.  A residual that is nowhere positive (p <= q
// everywhere) draws from p.
#pragma once
#include "sm100.cuh"

namespace simsd {

struct SpecVerifyArgs {
  const void* target;       // [B, K + 1, V]
  const void* draft;        // [B, K, V] or nullptr
  const long long* tokens;  // [B, K]
  const float* uniform;     // [B, K]
  const float* noise;       // [B, V]
  const float* temperature; // [B] or nullptr (1)
  const int* n_draft;       // [B] or nullptr (K)
  long long* out_tokens;    // [B, K + 1]
  long long* out_accepted;  // [B]
  float* out_logprobs;      // [B, K + 1]
  float* stat;              // [B, 2 K + 1, 3]: row maximum, sum of exp((x - max) / T), first place of the maximum
  int* err;
  long long ldt_b, ldt_r, ldd_b, ldd_r, ld_x, ld_u, ld_n;
  int B, K, V, dtype;
};

constexpr int SV_THREADS = 256;

__device__ __forceinline__ float spec_logit(const void* p, long long i, int dtype) {
  return fminf(fmaxf(load_f(p, i, dtype), -INFINITY), 3.402823466e+38f);
}
__device__ __forceinline__ int spec_count(const SpecVerifyArgs& p, int b) {
  const int d = p.n_draft ? p.n_draft[b] : p.K;
  return d < 0 ? 0 : d > p.K ? p.K : d;
}

// (maximum, sum) of two parts of a row
__device__ __forceinline__ void spec_join(float& m, float& s, float m2, float s2, float rt) {
  const float mm = fmaxf(m, m2);
  if (mm == -INFINITY) return;
  s = s * expf((m - mm) * rt) + s2 * expf((m2 - mm) * rt);
  m = mm;
}

// One CTA per row: rows 0 .. K of the target, then K of the draft.
__global__ void __launch_bounds__(SV_THREADS) spec_stat_kernel(const SpecVerifyArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ float sm[SV_THREADS], ss[SV_THREADS];
  __shared__ int si[SV_THREADS];
  const int R = p.draft ? 2 * p.K + 1 : p.K + 1;
  const int b = blockIdx.x / R, r = blockIdx.x % R;
  const int d = spec_count(p, b);
  const bool is_t = r <= p.K;
  if (is_t ? r > d : r - p.K - 1 >= d) return;
  const float T = p.temperature ? p.temperature[b] : 1.0f;
  const float rt = T > 0.0f ? 1.0f / T : 0.0f;
  const long long base = is_t ? b * p.ldt_b + r * p.ldt_r : b * p.ldd_b + (r - p.K - 1) * p.ldd_r;
  const void* x = is_t ? p.target : p.draft;
  float m = -INFINITY, s = 0.0f;
  int at = 0x7fffffff;
  for (int v = threadIdx.x; v < p.V; v += SV_THREADS) {
    const float f = spec_logit(x, base + v, p.dtype);
    if (f > m) {
      s = s * expf((m - f) * rt);
      m = f;
      at = v;
    }
    if (f != -INFINITY) s += expf((f - m) * rt);
  }
  sm[threadIdx.x] = m, ss[threadIdx.x] = s, si[threadIdx.x] = at;
  __syncthreads();
  for (int k = SV_THREADS / 2; k > 0; k >>= 1) {
    if ((int)threadIdx.x < k) {
      const float m2 = sm[threadIdx.x + k];
      const int at2 = si[threadIdx.x + k];
      if (m2 > m || (m2 == m && at2 < at)) at = at2;
      spec_join(m, s, m2, ss[threadIdx.x + k], rt);
      sm[threadIdx.x] = m, ss[threadIdx.x] = s, si[threadIdx.x] = at;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    float* o = p.stat + ((long long)b * (2 * p.K + 1) + r) * 3;
    o[0] = m, o[1] = s, o[2] = __int_as_float(m == -INFINITY ? -1 : at);
  }
}

// p(v) of a row from its statistics
__device__ __forceinline__ float spec_prob(const void* x, long long base, int v, int dtype, const float* st, float T) {
  if (st[0] == -INFINITY) return 0.0f;
  if (!(T > 0.0f)) return v == __float_as_int(st[2]) ? 1.0f : 0.0f;
  return expf((spec_logit(x, base + v, dtype) - st[0]) / T) / st[1];
}
__device__ __forceinline__ float spec_logprob(const void* x, long long base, int v, int dtype, const float* st, float T) {
  if (st[0] == -INFINITY) return -INFINITY;
  if (!(T > 0.0f)) return v == __float_as_int(st[2]) ? 0.0f : -INFINITY;
  return (spec_logit(x, base + v, dtype) - st[0]) / T - logf(st[1]);
}

// One CTA per sequence.
__global__ void __launch_bounds__(SV_THREADS) spec_draw_kernel(const SpecVerifyArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ float sv[2][SV_THREADS];
  __shared__ int si[2][SV_THREADS];
  const int b = blockIdx.x;
  const int d = spec_count(p, b);
  const float T = p.temperature ? p.temperature[b] : 1.0f;
  const float* st = p.stat + (long long)b * (2 * p.K + 1) * 3;
  int a = 0;
  bool bad = false;
  for (; a < d; ++a) {
    const long long x = p.tokens[b * p.ld_x + a];
    if (x < 0 || x >= p.V) {
      bad = true;
      break;
    }
    const float pr = spec_prob(p.target, b * p.ldt_b + a * p.ldt_r, (int)x, p.dtype, st + a * 3, T);
    const float qr = p.draft ? spec_prob(p.draft, b * p.ldd_b + a * p.ldd_r, (int)x, p.dtype, st + (p.K + 1 + a) * 3, T)
                             : 1.0f;
    if (!(p.uniform[b * p.ld_u + a] * qr < pr)) break;
  }
  if (bad && threadIdx.x == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
  const long long tb = b * p.ldt_b + a * p.ldt_r, db = b * p.ldd_b + a * p.ldd_r;
  const bool minus = a < d && !bad;
  const int hit = minus && !p.draft ? (int)p.tokens[b * p.ld_x + a] : -1;
  // the residual's best token, and p's own for a residual that is nowhere positive
  float best[2] = {-1.0f, -1.0f};
  int at[2] = {0x7fffffff, 0x7fffffff};
  for (int v = threadIdx.x; v < p.V; v += SV_THREADS) {
    const float pr = spec_prob(p.target, tb, v, p.dtype, st + a * 3, T);
    const float qr = !minus ? 0.0f : p.draft ? spec_prob(p.draft, db, v, p.dtype, st + (p.K + 1 + a) * 3, T)
                                             : v == hit ? 1.0f : 0.0f;
    const float e = p.noise[b * p.ld_n + v];
    const float w[2] = {fmaxf(pr - qr, 0.0f) / e, pr / e};
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (w[k] > best[k]) best[k] = w[k], at[k] = v;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) sv[k][threadIdx.x] = best[k], si[k][threadIdx.x] = at[k];
  __syncthreads();
  for (int s = SV_THREADS / 2; s > 0; s >>= 1) {
    if ((int)threadIdx.x < s)
      for (int k = 0; k < 2; ++k) {
        const float o = sv[k][threadIdx.x + s];
        const int oi = si[k][threadIdx.x + s];
        if (o > sv[k][threadIdx.x] || (o == sv[k][threadIdx.x] && oi < si[k][threadIdx.x]))
          sv[k][threadIdx.x] = o, si[k][threadIdx.x] = oi;
      }
    __syncthreads();
  }
  const int drawn = sv[0][0] > 0.0f ? si[0][0] : si[1][0];
  for (int i = threadIdx.x; i <= p.K; i += SV_THREADS) {
    const int x = i < a ? (int)p.tokens[b * p.ld_x + i] : drawn;
    p.out_tokens[(long long)b * (p.K + 1) + i] = i <= a ? x : -1;
    p.out_logprobs[(long long)b * (p.K + 1) + i] =
        i <= a ? spec_logprob(p.target, b * p.ldt_b + i * p.ldt_r, x, p.dtype, st + i * 3, T) : 0.0f;
  }
  if (threadIdx.x == 0) p.out_accepted[b] = a;
}

}  // namespace simsd
