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
//
// Two kernels.  spec_stat_kernel reads every row once: a warp takes 1024 logits,
// keeps them in registers between their maximum and the sum of their exponentials,
// and leaves (max, sum) as the row's partial.  spec_draw_kernel joins the partials,
// decides how many drafts are kept (every CTA of the sequence for itself: a few KB
// from L2) and races the one row that is drawn from; the sequence's last CTA to
// finish writes its outputs.  HBM bounds both; the first also runs one exponential
// per 2 bytes, about 0.7 of what the SMs' exponential units do in that time.  Rows
// are read last to first, so that the rows drawn from, mostly early ones, are the
// ones left in L2.
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
  float2* part;             // [B, 2 K + 1, parts]: maximum, sum of exp((x - max) / T) of a part of a row
  float4* cand;             // [B, chunks]: best residual race and token, best race over p and token
  int* done;                // [B]: CTAs of the sequence that have finished, zeroed by the first kernel
  int* err;
  long long ldt_b, ldt_r, ldd_b, ldd_r, ld_x, ld_u, ld_n;
  int B, K, V, parts, chunks, dtype;
};

constexpr int SV_THREADS = 256, SV_WARPS = SV_THREADS / 32;
constexpr int SV_PART = 1024;                      // logits of one partial (one warp)
constexpr int SV_CHUNK = 8192;                     // tokens that one CTA races

__device__ __forceinline__ float spec_clean(float v) { return fminf(fmaxf(v, -INFINITY), 3.402823466e+38f); }
__device__ __forceinline__ float spec_logit(const void* p, long long i, int dtype) {
  return spec_clean(load_f(p, i, dtype));
}
__device__ __forceinline__ int spec_count(const SpecVerifyArgs& p, int b) {
  const int d = p.n_draft ? p.n_draft[b] : p.K;
  return d < 0 ? 0 : d > p.K ? p.K : d;
}
__device__ __forceinline__ float spec_temperature(const SpecVerifyArgs& p, int b) {
  return p.temperature ? p.temperature[b] : 1.0f;
}
// log2(e) / T, what a difference of logits is multiplied with; 0 for greedy sequences
__device__ __forceinline__ float spec_scale(float T) { return T > 0.0f ? 1.4426950408889634f / fmaxf(T, 1e-30f) : 0.0f; }
__device__ __forceinline__ float spec_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes of logits as floats
template <int DT>
struct SpecVec {
  static constexpr int N = DT == 2 ? 4 : 8;
  __device__ static __forceinline__ void unpack(const uint4& u, float (&v)[N]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == 0) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else if constexpr (DT == 1) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      } else {
        v[i] = __uint_as_float(w[i]);
      }
    }
  }
};

// Where a row of V logits starts to be 16-byte aligned, and its whole vectors.
// Part w of the row is vectors [w, w + 1) * SV_PART / N after the `head` logits,
// which belong to part 0; those after the last whole vector to the last part.
struct SpecRow {
  int head, nvec;
};
template <int DT>
__device__ __forceinline__ SpecRow spec_row(const void* x, int V) {
  constexpr int N = SpecVec<DT>::N, ES = 16 / N;
  SpecRow r;
  r.head = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / ES));
  r.nvec = (V - r.head) / N;
  return r;
}

// Row r of the sequence: 0 .. K the target's, K + 1 .. 2 K the draft's
__device__ __forceinline__ const void* spec_row_ptr(const SpecVerifyArgs& p, int b, int r) {
  const long long es = p.dtype == 2 ? 4 : 2;
  return r <= p.K ? reinterpret_cast<const char*>(p.target) + (b * p.ldt_b + r * p.ldt_r) * es
                  : reinterpret_cast<const char*>(p.draft) + (b * p.ldd_b + (r - p.K - 1) * p.ldd_r) * es;
}

template <int DT>
__global__ void __launch_bounds__(SV_THREADS) spec_stat_kernel(const SpecVerifyArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int N = SpecVec<DT>::N, VL = SV_PART / N / 32;     // vectors per lane
  const int lane = threadIdx.x & 31;
  const int per_row = (p.parts + SV_WARPS - 1) / SV_WARPS;
  const int part = (int)(blockIdx.x % per_row) * SV_WARPS + (threadIdx.x >> 5);
  const int rest = blockIdx.x / per_row;
  const int b = rest % p.B, back = rest / p.B;
  // rows last to first: target K, then target and draft K - 1, ...
  const int r = !p.draft ? p.K - back : back & 1 ? p.K - 1 - back / 2 : back == 0 ? p.K : 2 * p.K + 1 - back / 2;
  if (blockIdx.x % per_row == 0 && threadIdx.x == 0 && r == 0) p.done[b] = 0;
  const int d = spec_count(p, b);
  if (part >= p.parts || (r <= p.K ? r > d : r - p.K - 1 >= d)) return;
  const float c = spec_scale(spec_temperature(p, b));
  const void* x = spec_row_ptr(p, b, r);
  const SpecRow row = spec_row<DT>(x, p.V);
  const uint4* xv = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(x) + row.head * (16 / N));
  uint4 raw[VL];
  // -inf in the type's own bits, where there is no vector
  constexpr uint32_t NI = DT == 0 ? 0xff80ff80u : DT == 1 ? 0xfc00fc00u : 0xff800000u;
#pragma unroll
  for (int i = 0; i < VL; ++i) {
    const int v = part * (SV_PART / N) + i * 32 + lane;
    raw[i] = v < row.nvec ? __ldg(xv + v) : make_uint4(NI, NI, NI, NI);
  }
  float extra = -INFINITY;
  const int tail = row.head + row.nvec * N;
  if (part == 0 && lane < row.head) extra = spec_logit(x, lane, DT);
  float extra2 = -INFINITY;
  if (part == p.parts - 1 && lane < p.V - tail) extra2 = spec_logit(x, tail + lane, DT);
  float m = fmaxf(extra, extra2);
#pragma unroll
  for (int i = 0; i < VL; ++i) {
    float f[N];
    SpecVec<DT>::unpack(raw[i], f);
#pragma unroll
    for (int e = 0; e < N; ++e) m = fmaxf(m, f[e]);      // ignores NaN
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
  float s = 0.0f;
  if (m == INFINITY) {                                   // +inf counts as the largest finite number
    m = spec_clean(m);
    s = spec_exp2((extra - m) * c) + spec_exp2((extra2 - m) * c);
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      float f[N];
      SpecVec<DT>::unpack(raw[i], f);
#pragma unroll
      for (int e = 0; e < N; ++e) s += spec_exp2((spec_clean(f[e]) - m) * c);
    }
  } else if (m != -INFINITY) {
    s = spec_exp2((extra - m) * c) + spec_exp2((extra2 - m) * c);
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      float f[N];
      SpecVec<DT>::unpack(raw[i], f);
#pragma unroll
      for (int e = 0; e < N; ++e) s += spec_exp2(fmaxf((f[e] - m) * c, -INFINITY));   // NaN: 0
    }
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
  if (lane == 0) p.part[((long long)b * (2 * p.K + 1) + r) * p.parts + part] = make_float2(m, s);
}

// Maximum, sum and, for greedy sequences, first place of the maximum of row r, by one warp
template <int DT>
__device__ __forceinline__ void spec_join_row(const SpecVerifyArgs& p, int b, int r, float c, float& m, float& s, int& at) {
  constexpr int N = SpecVec<DT>::N;
  const int lane = threadIdx.x & 31;
  const float2* part = p.part + ((long long)b * (2 * p.K + 1) + r) * p.parts;
  m = -INFINITY;
  for (int i = lane; i < p.parts; i += 32) m = fmaxf(m, part[i].x);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
  s = 0.0f;
  at = 0;
  if (m == -INFINITY) return;
  int first = 0x7fffffff;
  for (int i = lane; i < p.parts; i += 32) {
    const float2 x = part[i];
    s = fmaf(x.y, spec_exp2((x.x - m) * c), s);
    if (x.x == m) first = min(first, i);
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, k);
    first = min(first, __shfl_xor_sync(0xffffffffu, first, k));
  }
  if (c != 0.0f) return;
  const void* x = spec_row_ptr(p, b, r);
  const SpecRow row = spec_row<DT>(x, p.V);
  const int lo = first == 0 ? 0 : row.head + first * SV_PART;
  const int hi = first == p.parts - 1 ? p.V : min(p.V, row.head + (first + 1) * SV_PART);
  int best = 0x7fffffff;
  for (int v = lo + lane; v < hi && best == 0x7fffffff; v += 32)
    if (spec_logit(x, v, DT) == m) best = v;
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) best = min(best, __shfl_xor_sync(0xffffffffu, best, k));
  at = best;
}

// One token's race: the residual's and p's own, in ascending order of v per thread
struct SpecBest {
  float res, own;
  int ri, oi;
  __device__ __forceinline__ void see(float pr, float qr, float e, int v) {
    const float a = fmaxf(pr - qr, 0.0f) / e, o = pr / e;
    if (a > res) res = a, ri = v;
    if (o > own) own = o, oi = v;
  }
  __device__ __forceinline__ void join(float r2, int ri2, float o2, int oi2) {
    if (r2 > res || (r2 == res && ri2 < ri)) res = r2, ri = ri2;
    if (o2 > own || (o2 == own && oi2 < oi)) own = o2, oi = oi2;
  }
  __device__ __forceinline__ void join_warp() {
#pragma unroll
    for (int k = 16; k > 0; k >>= 1)
      join(__shfl_xor_sync(0xffffffffu, res, k), __shfl_xor_sync(0xffffffffu, ri, k), __shfl_xor_sync(0xffffffffu, own, k),
           __shfl_xor_sync(0xffffffffu, oi, k));
  }
};

template <int DT>
__global__ void __launch_bounds__(SV_THREADS) spec_draw_kernel(const SpecVerifyArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int N = SpecVec<DT>::N;
  extern __shared__ float sv_rows[];               // [2 K + 1][3]: maximum, 1 / sum, place of the maximum
  __shared__ SpecBest s_best[SV_WARPS];
  __shared__ int s_kept, s_last;
  __shared__ bool s_bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / p.chunks, chunk = blockIdx.x - b * p.chunks;
  const int d = spec_count(p, b);
  const float c = spec_scale(spec_temperature(p, b));
  const long long* xs = p.tokens + b * p.ld_x;
  const int R = d + 1 + (p.draft ? d : 0);
  for (int k = warp; k < R; k += SV_WARPS) {
    const int r = k <= d ? k : p.K + k - d;
    float m, s;
    int at;
    spec_join_row<DT>(p, b, r, c, m, s, at);
    if (lane == 0) sv_rows[r * 3] = m, sv_rows[r * 3 + 1] = s, sv_rows[r * 3 + 2] = __int_as_float(at);
  }
  __syncthreads();
  // the probability of token v, whose logit is x, in row r
  auto prob = [&](int r, float x, int v) {
    const float m = sv_rows[r * 3];
    if (m == -INFINITY) return 0.0f;
    if (c == 0.0f) return v == __float_as_int(sv_rows[r * 3 + 2]) ? 1.0f : 0.0f;
    return spec_exp2((spec_clean(x) - m) * c) / sv_rows[r * 3 + 1];
  };
  if (warp == 0) {
    int kept = d;
    bool bad = false;
    for (int i0 = 0; i0 < d && kept == d; i0 += 32) {
      const int i = i0 + lane;
      bool ok = true, out = false;
      if (i < d) {
        const long long x = xs[i];
        out = x < 0 || x >= p.V;
        if (out) {
          ok = false;
        } else {
          const float pr = prob(i, load_f(spec_row_ptr(p, b, i), x, DT), (int)x);
          const float qr = p.draft ? prob(p.K + 1 + i, load_f(spec_row_ptr(p, b, p.K + 1 + i), x, DT), (int)x) : 1.0f;
          ok = p.uniform[b * p.ld_u + i] * qr < pr;
        }
      }
      const uint32_t no = __ballot_sync(0xffffffffu, !ok), ob = __ballot_sync(0xffffffffu, out);
      if (no) {
        kept = i0 + __ffs(no) - 1;
        bad = (ob >> (__ffs(no) - 1)) & 1;
      }
    }
    if (lane == 0) {
      s_kept = kept;
      s_bad = bad;
      if (bad && chunk == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
    }
  }
  __syncthreads();
  const int a = s_kept;
  const bool minus = a < d && !s_bad;
  SpecBest best = {-1.0f, -1.0f, 0x7fffffff, 0x7fffffff};
  if (c != 0.0f) {
    const void* tr = spec_row_ptr(p, b, a);
    const void* dr = minus && p.draft ? spec_row_ptr(p, b, p.K + 1 + a) : nullptr;
    const int hit = minus && !p.draft ? (int)xs[a] : -1;
    const float* e = p.noise + b * p.ld_n;
    const float mt = sv_rows[a * 3], it = mt == -INFINITY ? 0.0f : 1.0f / sv_rows[a * 3 + 1];
    const float md = dr ? sv_rows[(p.K + 1 + a) * 3] : -INFINITY, id = md == -INFINITY ? 0.0f : 1.0f / sv_rows[(p.K + 1 + a) * 3 + 1];
    const float mtu = mt == -INFINITY ? 0.0f : mt, mdu = md == -INFINITY ? 0.0f : md;
    auto see = [&](float x, float y, float noise, int v) {
      const float pr = spec_exp2((spec_clean(x) - mtu) * c) * it;
      const float qr = dr ? spec_exp2((spec_clean(y) - mdu) * c) * id : v == hit ? 1.0f : 0.0f;
      best.see(pr, qr, noise, v);
    };
    const int lo = chunk * SV_CHUNK, hi = min(p.V, lo + SV_CHUNK);
    auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    if (aligned(tr) && aligned(e) && (!dr || aligned(dr))) {
      const int vec_hi = hi - (hi - lo) % N;
      for (int v0 = lo + tid * N; v0 < vec_hi; v0 += SV_THREADS * N) {
        float x[N], y[N];
        SpecVec<DT>::unpack(*reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(tr) + (long long)v0 * (16 / N)), x);
        const uint4 yr = dr ? *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(dr) + (long long)v0 * (16 / N))
                            : make_uint4(0, 0, 0, 0);
        SpecVec<DT>::unpack(yr, y);
        float4 n4[N / 4];
#pragma unroll
        for (int k = 0; k < N / 4; ++k) n4[k] = *reinterpret_cast<const float4*>(e + v0 + 4 * k);
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
          see(x[4 * k], y[4 * k], n4[k].x, v0 + 4 * k);
          see(x[4 * k + 1], y[4 * k + 1], n4[k].y, v0 + 4 * k + 1);
          see(x[4 * k + 2], y[4 * k + 2], n4[k].z, v0 + 4 * k + 2);
          see(x[4 * k + 3], y[4 * k + 3], n4[k].w, v0 + 4 * k + 3);
        }
      }
      for (int v = vec_hi + tid; v < hi; v += SV_THREADS) see(load_f(tr, v, DT), dr ? load_f(dr, v, DT) : 0.0f, e[v], v);
    } else {
      for (int v = lo + tid; v < hi; v += SV_THREADS) see(load_f(tr, v, DT), dr ? load_f(dr, v, DT) : 0.0f, e[v], v);
    }
    best.join_warp();
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
  }
  if (tid == 0) {
    if (c != 0.0f) {
      for (int w = 1; w < SV_WARPS; ++w) best.join(s_best[w].res, s_best[w].ri, s_best[w].own, s_best[w].oi);
      p.cand[(long long)b * p.chunks + chunk] = make_float4(best.res, __int_as_float(best.ri), best.own, __int_as_float(best.oi));
    }
    __threadfence();
    s_last = atomicAdd(p.done + b, 1) == p.chunks - 1;
  }
  __syncthreads();
  if (!s_last || warp != 0) return;
  // the sequence's last CTA: the best of all chunks, and the outputs
  __threadfence();
  int drawn = __float_as_int(sv_rows[a * 3 + 2]);
  if (c != 0.0f) {
    best = {-1.0f, -1.0f, 0x7fffffff, 0x7fffffff};
    for (int k = lane; k < p.chunks; k += 32) {
      const float4 x = __ldcg(p.cand + (long long)b * p.chunks + k);
      best.join(x.x, __float_as_int(x.y), x.z, __float_as_int(x.w));
    }
    best.join_warp();
    drawn = best.res > 0.0f ? best.ri : best.oi;
  }
  for (int i = lane; i <= p.K; i += 32) {
    const int v = i < a ? (int)xs[i] : drawn;
    float lp = 0.0f;
    if (i <= a) {
      const float m = sv_rows[i * 3];
      if (m == -INFINITY)
        lp = -INFINITY;
      else if (c == 0.0f)
        lp = v == __float_as_int(sv_rows[i * 3 + 2]) ? 0.0f : -INFINITY;
      else
        lp = (spec_logit(spec_row_ptr(p, b, i), v, DT) - m) / fmaxf(spec_temperature(p, b), 1e-30f) - logf(sv_rows[i * 3 + 1]);
    }
    p.out_tokens[(long long)b * (p.K + 1) + i] = i <= a ? v : -1;
    p.out_logprobs[(long long)b * (p.K + 1) + i] = lp;
  }
  if (lane == 0) p.out_accepted[b] = a;
}

}  // namespace simsd
