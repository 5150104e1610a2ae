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
// T = 0: p and q are one at their first maximum; T = inf: alike at every logit over -inf.  NaN logits count as -inf,
// +inf as the largest finite number; a row without any finite logit has p = 0.
// Ties go to the lowest token.  A residual that is nowhere positive (p <= q
// everywhere, to 2^-21 of p) draws from p.
//
// Two kernels.  spec_stat_kernel reads every row once: a warp takes `blocks` times
// 1024 logits, keeps each block in registers between its maximum and the sum of its
// exponentials, the next one on its way, and leaves (max, sum) as the row's part.
// spec_draw_kernel joins the parts, decides how many drafts are kept (every CTA of the
// sequence for itself: a few KB from L2) and races the one row that is drawn from; the sequence's last CTA to
// finish writes its outputs.  HBM bounds both; the first also runs one exponential
// per 2 bytes, about 0.7 of what the SMs' exponential units do in that time, so the
// rest of its arithmetic is packed: the maximum in the 16-bit type itself, the
// differences and sums two at a time.  Rows
// are read last to first, so that the rows drawn from, mostly early ones, are the
// ones left in L2.  64 x 7 drafts of 151936 tokens, bf16: 74 us on the device in a graph of
// calls, 4.5 TB/s (82 us one after the other on a stream); 1 x 4 of 32000 8.4 us, the
// latency of two kernels.
#pragma once
#include <type_traits>

#include "sm100.cuh"

namespace simsd {

// What a part of a row comes to.  A likely token leaves a sum of 1 and a little,
// whose logarithm is that little: the sums of lanes and parts are joined in 64 bits
// (a lane's own, in eight 32-bit runs, are taken apart where the 1 outweighs the rest), so
// that log p keeps its relative precision: the exponentials' arguments, 2^-23 of the
// difference to the maximum, and 2^-16 at most of the runs.
struct SpecPart {
  double s;                 // sum of exp((x - m) / T)
  float m;                  // maximum
  int at;                   // greedy sequences: where the maximum is first
};

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
  SpecPart* part;           // [B, 2 K + 1, parts]
  float2* cand;             // [B, chunks]: best race and its token
  int* done;                // [B]: CTAs of the sequence that have finished, zeroed by the first kernel
  int* err;
  long long ldt_b, ldt_r, ldd_b, ldd_r, ld_x, ld_u, ld_n;
  int B, K, V, blocks, parts, chunk, chunks, dtype;
};

constexpr int SV_THREADS = 256, SV_WARPS = SV_THREADS / 32;
constexpr int SV_BLOCK = 1024;                     // logits that a warp holds at a time
constexpr int SV_CHUNK = 2048;                     // tokens that a CTA races at a time
// p - q counts where it is more than p's rounding.  The same logits in two rows, split into
// parts at the same places (rows alike modulo 16 bytes), have the same sum, and p and q
// differ by a rounding of its reciprocal and of the product each, at most 2^-22 of p.
// Rows that start elsewhere split the sum otherwise and may be further apart: the margin
// does not cover them.  Without it two equal rows leave noise for a residual, which is
// drawn from.
constexpr float SV_OVER = 1.0f - 0x1p-21f;

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
// log2(e) / T, what a difference of logits is multiplied with; 0 for greedy sequences only
// (an infinite T takes the smallest positive number: differences of finite logits come to
// nothing, -inf stays)
__device__ __forceinline__ float spec_scale(float T) {
  return T > 0.0f ? fmaxf(1.4426950408889634f / fmaxf(T, 1e-30f), 1.4e-45f) : 0.0f;
}
__device__ __forceinline__ float spec_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int DT>
__device__ __forceinline__ float spec_half(uint32_t w, int hi) {
  if constexpr (DT == 0) return __uint_as_float(hi ? w & 0xffff0000u : w << 16);
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  return hi ? __high2float(h) : __low2float(h);
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

// Largest of a lane's vectors, NaN ignored: 16-bit types two at a time
template <int DT, int VL>
__device__ __forceinline__ float spec_max(const uint4 (&raw)[VL]) {
  if constexpr (DT == 2) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < VL; ++i)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(raw[i].x), __uint_as_float(raw[i].y)),
                         fmaxf(__uint_as_float(raw[i].z), __uint_as_float(raw[i].w))));
    return m;
  } else {
    uint32_t m = DT == 0 ? 0xff80ff80u : 0xfc00fc00u;
    auto see = [&](uint32_t x) {
      if constexpr (DT == 0)
        asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(x));
      else
        asm("max.f16x2 %0, %0, %1;" : "+r"(m) : "r"(x));
    };
#pragma unroll
    for (int i = 0; i < VL; ++i) see(raw[i].x), see(raw[i].y), see(raw[i].z), see(raw[i].w);
    return fmaxf(spec_half<DT>(m, 0), spec_half<DT>(m, 1));
  }
}

// Sum of exp2((x - m) c) over a lane's vectors, two values an instruction but for
// the exponential; `near` is the same in 32 bits
template <int DT, int VL>
__device__ __forceinline__ double spec_sum(const uint4 (&raw)[VL], float m, float c, float& near) {
  uint64_t nm, cc, sum[4] = {0, 0, 0, 0};
  asm("mov.b64 %0, {%1, %1};" : "=l"(nm) : "f"(-m));
  asm("mov.b64 %0, {%1, %1};" : "=l"(cc) : "f"(c));
  auto see = [&](float a, float b, uint64_t& to) {
    uint64_t x;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(nm));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(cc));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
    a = spec_exp2(a), b = spec_exp2(b);
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(to) : "l"(x));
  };
#pragma unroll
  for (int i = 0; i < VL; ++i) {
    float f[SpecVec<DT>::N];
    SpecVec<DT>::unpack(raw[i], f);
#pragma unroll
    for (int e = 0; e < SpecVec<DT>::N; e += 2) see(f[e], f[e + 1], sum[(i * SpecVec<DT>::N + e) / 2 % 4]);
  }
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum[0]) : "l"(sum[1]));
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum[2]) : "l"(sum[3]));
  float a, b, c2, d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(sum[0]));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(c2), "=f"(d) : "l"(sum[2]));
  near = (a + b) + (c2 + d);
  return ((double)a + b) + ((double)c2 + d);
}

// Where a row of V logits starts to be 16-byte aligned, and its whole vectors.
// Part w of the row is vectors [w, w + 1) * blocks * SV_BLOCK / N after the `head`
// logits, which belong to part 0; those after the last whole vector to the last part.
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

// Grid: x parts of a row, y sequences, z rows
template <int DT>
__global__ void __launch_bounds__(SV_THREADS, DT == 2 ? 3 : 4) spec_stat_kernel(const SpecVerifyArgs p) {
  griddep_wait();
  griddep_launch_dependents();             // after it: the second kernel reads inputs before its own wait
  constexpr int N = SpecVec<DT>::N, VL = SV_BLOCK / N / 32;    // vectors per lane
  static_assert(VL * N == 32);
  const int lane = threadIdx.x & 31, b = blockIdx.y, back = blockIdx.z;
  const int part = blockIdx.x * SV_WARPS + (threadIdx.x >> 5);
  // rows last to first: target K, then target and draft K - 1, ...
  const int r = !p.draft ? p.K - back : back & 1 ? p.K - 1 - back / 2 : back == 0 ? p.K : 2 * p.K + 1 - back / 2;
  if (blockIdx.x == 0 && threadIdx.x == 0 && r == 0) p.done[b] = 0;
  const int d = spec_count(p, b);
  if (part >= p.parts || (r <= p.K ? r > d : r - p.K - 1 >= d)) return;
  const float c = spec_scale(spec_temperature(p, b));
  const void* x = spec_row_ptr(p, b, r);
  const SpecRow row = spec_row<DT>(x, p.V);
  const uint4* xv = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(x) + row.head * (16 / N)) + lane;
  // -inf in the type's own bits, where there is no vector
  constexpr uint32_t NI = DT == 0 ? 0xff80ff80u : DT == 1 ? 0xfc00fc00u : 0xff800000u;
  uint4 raw[VL], next[VL];
  int v = part * p.blocks * (SV_BLOCK / N);                    // the block's first vector
  auto fetch = [&](int v0) {
    const uint4* src = xv + v0;
    if (v0 + SV_BLOCK / N <= row.nvec) {
#pragma unroll
      for (int i = 0; i < VL; ++i) next[i] = __ldg(src + i * 32);
    } else {
#pragma unroll
      for (int i = 0; i < VL; ++i) next[i] = v0 + i * 32 + lane < row.nvec ? __ldg(src + i * 32) : make_uint4(NI, NI, NI, NI);
    }
  };
  fetch(v);
  float extra = -INFINITY, extra2 = -INFINITY;           // before and after the row's whole vectors
  const int tail = row.head + row.nvec * N;
  if (part == 0 && lane < row.head) extra = spec_logit(x, lane, DT);
  if (part == p.parts - 1 && lane < p.V - tail) extra2 = spec_logit(x, tail + lane, DT);
  auto warp_max = [](float m) {
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
    return m;
  };
  float m = spec_clean(warp_max(fmaxf(extra, extra2)));
  double s = 0.0;                                        // this lane's
  int at = 0x7fffffff;                                   // greedy: the first place of m that this lane saw
  if (m != -INFINITY) {
    s = (double)spec_exp2((extra - m) * c) + spec_exp2((extra2 - m) * c);
    if (extra2 == m) at = tail + lane;
    if (extra == m) at = lane;
  }
  for (int n = 0; n < p.blocks && v < row.nvec; ++n, v += SV_BLOCK / N) {
#pragma unroll
    for (int i = 0; i < VL; ++i) raw[i] = next[i];
    if (n + 1 < p.blocks) fetch(v + SV_BLOCK / N);
    const float m2 = warp_max(spec_max<DT, VL>(raw)), mn = fmaxf(m, spec_clean(m2));
    if (mn == -INFINITY) continue;
    if (mn > m) s *= spec_exp2((m - mn) * c), at = 0x7fffffff;
    m = mn;
    if (c == 0.0f) {
#pragma unroll
      for (int i = VL - 1; i >= 0; --i) {
        const int vi = v + i * 32 + lane;
        float f[N];
        SpecVec<DT>::unpack(raw[i], f);
#pragma unroll
        for (int e = N - 1; e >= 0; --e)
          if (spec_clean(f[e]) == m) at = min(at, row.head + vi * N + e);
      }
      continue;
    }
    float near;
    double add = spec_sum<DT, VL>(raw, m, c, near);
    if (!(add < INFINITY)) {                             // NaN or +inf among the lane's logits
      add = 0.0;
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        float f[N];
        SpecVec<DT>::unpack(raw[i], f);
#pragma unroll
        for (int e = 0; e < N; ++e) add += spec_exp2((spec_clean(f[e]) - m) * c);
      }
    }
    if (m2 == m) {
      // A likely token: in the run of the maximum's 1 the others, of little weight beside it,
      // lose their last bits (four roundings of 2^-24), which log p is made of.  Where they
      // come to less than 2^-6, the lanes share that lane's logits out, one each (read
      // again: kept in registers they cost 17 us at 64 x 7; up to 2^-3 2 us more).
      for (uint32_t likely = __ballot_sync(0xffffffffu, near >= 1.0f && near < 1.015625f); likely; likely &= likely - 1) {
        const int other = __ffs(likely) - 1, vi = v + lane / N * 32 + other;
        if (lane == other) add = 0.0;
        const float one = vi < row.nvec ? spec_logit(x, row.head + (long long)vi * N + lane % N, DT) : -INFINITY;
        s += spec_exp2((one - m) * c);
      }
    }
    s += add;
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, k);
    at = min(at, __shfl_xor_sync(0xffffffffu, at, k));
  }
  if (lane == 0)
    p.part[((long long)b * (2 * p.K + 1) + r) * p.parts + part] = {s, m, at};
}

// Row r from its parts, by one warp (every lane has the result)
__device__ __forceinline__ SpecPart spec_join_row(const SpecVerifyArgs& p, int b, int r, float c) {
  constexpr int HOLD = 3;                          // parts that a lane holds
  const int lane = threadIdx.x & 31;
  const SpecPart* part = p.part + ((long long)b * (2 * p.K + 1) + r) * p.parts;
  auto get = [&](int i) {
    const int4 x = __ldcg(reinterpret_cast<const int4*>(part + i));
    return SpecPart{__hiloint2double(x.y, x.x), __int_as_float(x.z), x.w};
  };
  SpecPart x[HOLD];
#pragma unroll
  for (int k = 0; k < HOLD; ++k) x[k] = lane + k * 32 < p.parts ? get(lane + k * 32) : SpecPart{0.0, -INFINITY, 0x7fffffff};
  SpecPart y = {0.0, -INFINITY, 0x7fffffff};
#pragma unroll
  for (int k = 0; k < HOLD; ++k) y.m = fmaxf(y.m, x[k].m);
  for (int i = lane + HOLD * 32; i < p.parts; i += 32) y.m = fmaxf(y.m, get(i).m);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) y.m = fmaxf(y.m, __shfl_xor_sync(0xffffffffu, y.m, k));
  if (y.m == -INFINITY) return y;
  auto see = [&](const SpecPart& z) {
    y.s += z.s * spec_exp2((z.m - y.m) * c);
    if (z.m == y.m) y.at = min(y.at, z.at);
  };
#pragma unroll
  for (int k = 0; k < HOLD; ++k) see(x[k]);
  for (int i = lane + HOLD * 32; i < p.parts; i += 32) see(get(i));
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) {
    y.s += __shfl_xor_sync(0xffffffffu, y.s, k);
    y.at = min(y.at, __shfl_xor_sync(0xffffffffu, y.at, k));
  }
  return y;
}

// The best race so far, in ascending order of tokens per thread
struct SpecBest {
  float v;
  int at;
  __device__ __forceinline__ void see(float x, int i) {
    if (x > v) v = x, at = i;
  }
  __device__ __forceinline__ void join(float x, int i) {
    if (x > v || (x == v && i < at)) v = x, at = i;
  }
  __device__ __forceinline__ void join_warp() {
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) join(__shfl_xor_sync(0xffffffffu, v, k), __shfl_xor_sync(0xffffffffu, at, k));
  }
};

__device__ __forceinline__ float spec_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's probabilities: exp2((x - m) c) inv, 0 for an empty row (inv = 0)
struct SpecLaw {
  float m, inv;
};

// p / e, or max(p - q, 0) / e, of a lane's run of N tokens.  The differences are taken two
// at a time; the exponential is clamped to [0, 1], which makes NaN 0 and the +inf of a
// row whose maximum is the largest finite number 1, as the cleaned logit would.
template <int N, bool MINUS>
__device__ __forceinline__ void spec_race(const float (&x)[N], const float (&y)[N], const float (&e)[N], SpecLaw pt,
                                          SpecLaw pd, float c, float (&out)[N]) {
  uint64_t cc, nt, nd;
  asm("mov.b64 %0, {%1, %1};" : "=l"(cc) : "f"(c));
  asm("mov.b64 %0, {%1, %1};" : "=l"(nt) : "f"(-pt.m));
  asm("mov.b64 %0, {%1, %1};" : "=l"(nd) : "f"(-pd.m));
  auto weight = [&](float a, float b, uint64_t nm, float& wa, float& wb) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(d) : "l"(nm));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(d) : "l"(cc));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d));
    wa = __saturatef(spec_exp2(a)), wb = __saturatef(spec_exp2(b));
  };
#pragma unroll
  for (int k = 0; k < N; k += 2) {
    float p[2], q[2];
    weight(x[k], x[k + 1], nt, p[0], p[1]);
    if constexpr (MINUS) weight(y[k], y[k + 1], nd, q[0], q[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float w = p[h] * pt.inv;
      if constexpr (MINUS) w = fmaxf(w - q[h] * pd.inv, 0.0f);
      out[k + h] = w * spec_rcp(e[k + h]);
    }
  }
}

template <int DT>
__global__ void __launch_bounds__(SV_THREADS, 4) spec_draw_kernel(const SpecVerifyArgs p) {
  griddep_launch_dependents();
  constexpr int N = SpecVec<DT>::N;
  extern __shared__ SpecPart sv_rows[];            // [2 K + 1]
  __shared__ SpecBest s_best[SV_WARPS];
  __shared__ int s_kept, s_last;
  __shared__ bool s_bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / p.chunks, chunk = blockIdx.x - b * p.chunks;
  const int d = spec_count(p, b);
  const float T = spec_temperature(p, b), c = spec_scale(T);
  const long long* xs = p.tokens + b * p.ld_x;
  // the first warp fetches what decides about the first 32 drafts while the others join the rows' parts
  long long x0 = -1;
  float u0 = 0.0f, t0 = 0.0f, d0 = 0.0f;
  auto fetch = [&](int i) {
    x0 = i < d ? xs[i] : 0;
    if (i < d && x0 >= 0 && x0 < p.V) {
      t0 = load_f(spec_row_ptr(p, b, i), x0, DT);
      if (p.draft) d0 = load_f(spec_row_ptr(p, b, p.K + 1 + i), x0, DT);
      u0 = p.uniform[b * p.ld_u + i];
    }
  };
  if (warp == 0) fetch(lane);
  // all that was read so far is input: the first kernel lets this one start after its own wait
  const int lo = chunk * p.chunk, hi = min(p.V, lo + p.chunk);
  griddep_wait();
  const int R = d + 1 + (p.draft ? d : 0);
  for (int k = SV_WARPS - 1 - warp; k < R; k += SV_WARPS) {
    const int r = k <= d ? k : p.K + k - d;
    const SpecPart y = spec_join_row(p, b, r, c);
    if (lane == 0) sv_rows[r] = y;
  }
  __syncthreads();
  // the probability of token v, whose logit is x, in row r
  auto prob = [&](int r, float x, int v) {
    const SpecPart& y = sv_rows[r];
    if (y.m == -INFINITY) return 0.0f;
    if (c == 0.0f) return v == y.at ? 1.0f : 0.0f;
    return spec_exp2((spec_clean(x) - y.m) * c) / (float)y.s;
  };
  if (warp == 0) {
    int kept = d;
    bool bad = false;
    for (int i0 = 0; i0 < d && kept == d; i0 += 32) {
      const int i = i0 + lane;
      if (i0 > 0) fetch(i);
      const bool out = i < d && (x0 < 0 || x0 >= p.V);
      bool ok = !out;
      if (i < d && ok)
        ok = u0 * (p.draft ? prob(p.K + 1 + i, d0, (int)x0) : 1.0f) < prob(i, t0, (int)x0);
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
  // the row that is drawn from, less (minus) the draft's
  const void* tr = spec_row_ptr(p, b, a);
  const void* dr = minus && p.draft ? spec_row_ptr(p, b, p.K + 1 + a) : nullptr;
  const int hit = minus && !p.draft ? (int)xs[a] : -1;
  const float* e = p.noise + b * p.ld_n;
  auto law = [&](int r) {
    const SpecPart& y = sv_rows[r];
    return y.m == -INFINITY ? SpecLaw{0.0f, 0.0f} : SpecLaw{y.m, 1.0f / (float)y.s};
  };
  SpecLaw pt = law(a);
  const SpecLaw pd = dr ? law(p.K + 1 + a) : SpecLaw{0.0f, 0.0f};
  if (dr) pt.inv *= SV_OVER;
  SpecBest best = {-1.0f, 0x7fffffff};
  const bool vectors = ((reinterpret_cast<uintptr_t>(tr) | reinterpret_cast<uintptr_t>(e) | reinterpret_cast<uintptr_t>(dr)) & 15) == 0;
  // tokens lo .. hi - 1, a thread's in ascending order
  auto run = [&](int lo, int hi, int skip, auto minus_q) {
    constexpr bool MINUS = decltype(minus_q)::value;
    int vec_hi = lo;
    if (vectors) {
      vec_hi = hi - (hi - lo) % N;
#pragma unroll 1
      for (int v0 = lo + tid * N; v0 < vec_hi; v0 += SV_THREADS * N) {
        float x[N], y[N], z[N], w[N];
        const uint4 xr = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(tr) + (long long)v0 * (16 / N)));
        uint4 yr;
        if constexpr (MINUS) yr = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(dr) + (long long)v0 * (16 / N)));
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
          const float4 f = __ldg(reinterpret_cast<const float4*>(e + v0) + k);
          z[4 * k] = f.x, z[4 * k + 1] = f.y, z[4 * k + 2] = f.z, z[4 * k + 3] = f.w;
        }
        SpecVec<DT>::unpack(xr, x);
        if constexpr (MINUS) SpecVec<DT>::unpack(yr, y);
        spec_race<N, MINUS>(x, y, z, pt, pd, c, w);
        if (!MINUS && (unsigned)(skip - v0) < (unsigned)N) {
#pragma unroll
          for (int k = 0; k < N; ++k)
            if (v0 + k == skip) w[k] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < N; ++k) best.see(w[k], v0 + k);
      }
    }
#pragma unroll 4
    for (int v = vec_hi + tid; v < hi; v += 2 * SV_THREADS) {
      const int v2 = v + SV_THREADS < hi ? v + SV_THREADS : v;
      const float x[2] = {load_f(tr, v, DT), load_f(tr, v2, DT)}, z[2] = {e[v], e[v2]};
      float y[2], w[2];
      if constexpr (MINUS) y[0] = load_f(dr, v, DT), y[1] = load_f(dr, v2, DT);
      spec_race<2, MINUS>(x, y, z, pt, pd, c, w);
      best.see(v == skip ? 0.0f : w[0], v);
      best.see(v2 == skip ? 0.0f : w[1], v2);
    }
  };
  // p, p without the refused token (q one there: max(p - q, 0) is 0), or p - q
  auto race = [&](int lo, int hi, bool less) {
    if (less && dr)
      run(lo, hi, -1, std::true_type());
    else
      run(lo, hi, less ? hit : -1, std::false_type());
  };
  if (c != 0.0f) {
    race(lo, hi, minus);
    best.join_warp();
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
  }
  if (tid == 0) {
    if (c != 0.0f) {
      for (int w = 1; w < SV_WARPS; ++w) best.join(s_best[w].v, s_best[w].at);
      p.cand[(long long)b * p.chunks + chunk] = make_float2(best.v, __int_as_float(best.at));
    }
    __threadfence();
    s_last = atomicAdd(p.done + b, 1) == p.chunks - 1;
    __threadfence();
  }
  __syncthreads();
  if (!s_last) return;
  // the sequence's last CTA: the best of all chunks, and the outputs
  int drawn = sv_rows[a].at;
  if (sv_rows[a].m == -INFINITY) {
    drawn = 0;
  } else if (c != 0.0f) {
    best = {-1.0f, 0x7fffffff};
    for (int k = lane; k < p.chunks; k += 32) {
      const float2 x = __ldcg(p.cand + (long long)b * p.chunks + k);
      best.join(x.x, __float_as_int(x.y));
    }
    best.join_warp();
    if (minus && !(best.v > 0.0f)) {
      // p nowhere over q: drawn from p (every thread has the same `best` here)
      best = {-1.0f, 0x7fffffff};
      race(0, p.V, false);
      best.join_warp();
      __syncthreads();
      if (lane == 0) s_best[warp] = best;
      __syncthreads();
      for (int w = 0; w < SV_WARPS; ++w) best.join(s_best[w].v, s_best[w].at);
    }
    drawn = best.at;
    // no token won (noise that is NaN throughout, say): nothing is read for such an index
    if ((unsigned)drawn >= (unsigned)p.V) {
      drawn = 0;
      if (tid == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
    }
  }
  if (warp != 0) return;
  for (int i = lane; i <= p.K; i += 32) {
    const int v = i < a ? (int)xs[i] : drawn;
    float lp = 0.0f;
    if (i <= a) {
      const SpecPart& y = sv_rows[i];
      if (y.m == -INFINITY)
        lp = -INFINITY;
      else if (c == 0.0f)
        lp = v == y.at ? 0.0f : -INFINITY;
      else
        lp = (spec_logit(spec_row_ptr(p, b, i), v, DT) - y.m) / fmaxf(T, 1e-30f) - log1pf((float)(y.s - 1.0));
    }
    p.out_tokens[(long long)b * (p.K + 1) + i] = i <= a ? v : -1;
    p.out_logprobs[(long long)b * (p.K + 1) + i] = lp;
  }
  if (lane == 0) p.out_accepted[b] = a;
}

}  // namespace simsd
