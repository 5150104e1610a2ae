// Rules on logits before a token is drawn: penalties for repeated tokens, biases and
// grammar masks, for every drafted row of a sequence.  Row i of sequence b, token v, with
//   c = counts[b, v] + the number of j < i with drafts[b, j] = v:
//   x = logits[b, i, v]
//   x = x > 0 ? x / repetition[b] : x repetition[b]     where c > 0 or seen[b] has v
//   x = x - frequency[b] c - presence[b]                where c > 0
//   x = x + the biases of v in sequence b's list, summed in the list's order
//   x = -inf                                            where allowed[b, i] lacks v
// in fp32, rounded once to the logits' type.
//
// HBM bounds it: every logit read and written once.  A CTA takes 2048 tokens of one
// sequence through all its rows, so that counts, the prompt's bits and the biases are
// read once a sequence and stay in registers; after row i the thread that owns drafted
// token i counts it.  The next row is on its way while one is worked on, and tokens
// without a rule (nearly all) cost a conversion there and back.
#pragma once
#include "spec_verify.cuh"

namespace simsd {

struct LogitRulesArgs {
  const void* logits;       // [B, R, V]
  void* out;                // [B, R, V]
  const int* counts;        // [B, V] or nullptr (none yet)
  const long long* drafts;  // [B, R - 1] or nullptr
  const uint32_t* seen;     // [B, words] or nullptr
  const float* repetition;  // [B] or nullptr (1)
  const float* presence;    // [B] or nullptr (0)
  const float* frequency;   // [B] or nullptr (0)
  const int* bias_ids;      // [B, n_bias]
  const float* bias;        // [B, n_bias]
  const uint32_t* allowed;  // [B, R, words] or nullptr
  int* err;
  long long ld_b, ld_r, ldo_b, ldo_r, ld_c, ld_d, ld_s, ld_i, ld_v, lda_b, lda_r;
  int B, R, V, n_bias;
  bool penal;               // one of the penalties is there
};

constexpr int LR_THREADS = 256, LR_EACH = 8, LR_TOKENS = LR_THREADS * LR_EACH;

// VEC: a thread owns 8 tokens in a row (16-byte loads and stores), else 8 tokens 32
// apart, a warp's next to each other (rows that start anywhere).
template <int DT, bool VEC>
__global__ void __launch_bounds__(LR_THREADS) logit_rules_kernel(const LogitRulesArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int VECS = DT == 2 ? 2 : 1;           // 16-byte loads of 8 logits
  __shared__ int s_id[LR_THREADS], s_n[LR_THREADS / 32];
  __shared__ float s_val[LR_THREADS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.y;
  const int v0 = blockIdx.x * LR_TOKENS;
  const int first = VEC ? v0 + tid * LR_EACH : v0 + warp * 32 * LR_EACH + lane;   // the thread's tokens: first + k step
  constexpr int step = VEC ? 1 : 32;
  // the thread's place for a token of the CTA (0 .. LR_TOKENS - 1), or -1
  auto mine = [&](int at) {
    if (VEC) return at / LR_EACH == tid ? at % LR_EACH : -1;
    return at / (32 * LR_EACH) == warp && at % 32 == lane ? at / 32 % LR_EACH : -1;
  };
  // 8 bits of a word list, the thread's tokens'
  auto bits = [&](const uint32_t* w) {
    const int words = (p.V + 31) / 32;
    if (VEC) return first < p.V ? w[first / 32] >> first % 32 & 0xffu : 0u;
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < LR_EACH; ++k) {
      const int at = first / 32 + k;
      m |= (at < words ? w[at] >> lane & 1u : 0u) << k;
    }
    return m;
  };

  uint4 raw[2][VECS];                             // VEC: this row and the next
  float val[2][VEC ? 1 : LR_EACH];                // else
  uint32_t ok[2] = {0xffu, 0xffu};
  long long draft[2] = {-1, -1};
  auto fetch = [&](int i, int at) {
    if (i >= p.R) return;
    const long long off = b * p.ld_b + i * p.ld_r + first;
    if constexpr (VEC) {
      if (first < p.V) {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const char*>(p.logits) + off * (DT == 2 ? 4 : 2));
#pragma unroll
        for (int x = 0; x < VECS; ++x) raw[at][x] = src[x];
      }
    } else {
#pragma unroll
      for (int k = 0; k < LR_EACH; ++k)
        if (first + k * step < p.V) val[at][k] = load_f(p.logits, off + k * step, DT);
    }
    if (p.allowed) ok[at] = bits(p.allowed + b * p.lda_b + i * p.lda_r);
    draft[at] = p.drafts && i + 1 < p.R ? p.drafts[b * p.ld_d + i] : -1;
  };
  fetch(0, 0);

  int c[LR_EACH];
  uint32_t met = 0, again = 0;                    // tokens counted, and those or in the prompt
#pragma unroll
  for (int k = 0; k < LR_EACH; ++k) c[k] = 0;
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  if (p.penal) {
    if (p.counts) {
      const int* src = p.counts + b * p.ld_c + first;
      if (VEC) {
        if (first < p.V) {
          const int4 a = reinterpret_cast<const int4*>(src)[0], d = reinterpret_cast<const int4*>(src)[1];
          c[0] = a.x, c[1] = a.y, c[2] = a.z, c[3] = a.w, c[4] = d.x, c[5] = d.y, c[6] = d.z, c[7] = d.w;
        }
      } else {
#pragma unroll
        for (int k = 0; k < LR_EACH; ++k)
          if (first + k * step < p.V) c[k] = src[k * step];
      }
    }
    if (p.seen) again = bits(p.seen + b * p.ld_s);
#pragma unroll
    for (int k = 0; k < LR_EACH; ++k) met |= (uint32_t)(c[k] > 0) << k;
    again |= met;
    if (p.repetition) rep = p.repetition[b];
    if (p.presence) pres = p.presence[b];
    if (p.frequency) freq = p.frequency[b];
  }
  float bias[LR_EACH];
  bool biased = false;
#pragma unroll
  for (int k = 0; k < LR_EACH; ++k) bias[k] = 0.0f;
  for (int base = 0; base < p.n_bias; base += LR_THREADS) {
    // the list's entries that fall on the CTA's tokens, in its order
    const int n = base + tid;
    const int id = n < p.n_bias ? p.bias_ids[b * p.ld_i + n] : -1;
    if (id >= p.V && blockIdx.x == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
    const bool in = id >= v0 && id < v0 + LR_TOKENS && id < p.V;
    const uint32_t who = __ballot_sync(0xffffffffu, in);
    if (lane == 0) s_n[warp] = __popc(who);
    __syncthreads();
    int at = __popc(who & ((1u << lane) - 1)), all = 0;
#pragma unroll
    for (int w = 0; w < LR_THREADS / 32; ++w) {
      if (w < warp) at += s_n[w];
      all += s_n[w];
    }
    if (in) s_id[at] = id - v0, s_val[at] = p.bias[b * p.ld_v + n];
    __syncthreads();
    for (int e = 0; e < all; ++e) {
      const int k = mine(s_id[e]);
      if (k < 0) continue;
      biased = true;
#pragma unroll
      for (int x = 0; x < LR_EACH; ++x) bias[x] += x == k ? s_val[e] : 0.0f;
    }
    __syncthreads();
  }

  auto row = [&](int i, int at) {
    fetch(i + 1, at ^ 1);
    float x[LR_EACH];
    if constexpr (VEC) {
#pragma unroll
      for (int h = 0; h < VECS; ++h) {
        float y[SpecVec<DT>::N];
        SpecVec<DT>::unpack(raw[at][h], y);
#pragma unroll
        for (int k = 0; k < SpecVec<DT>::N; ++k) x[h * SpecVec<DT>::N + k] = y[k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < LR_EACH; ++k) x[k] = val[at][k];
    }
    if (again != 0) {
#pragma unroll
      for (int k = 0; k < LR_EACH; ++k) {
        if (again >> k & 1) x[k] = x[k] > 0.0f ? x[k] / rep : x[k] * rep;
        if (met >> k & 1) x[k] = fmaf(-freq, (float)c[k], x[k]) - pres;
      }
    }
    if (biased) {
#pragma unroll
      for (int k = 0; k < LR_EACH; ++k) x[k] += bias[k];
    }
#pragma unroll
    for (int k = 0; k < LR_EACH; ++k)
      if (!(ok[at] >> k & 1)) x[k] = -INFINITY;
    const long long off = b * p.ldo_b + i * p.ldo_r + first;
    if constexpr (VEC) {
      if (first < p.V) {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<char*>(p.out) + off * (DT == 2 ? 4 : 2));
        if constexpr (DT == 2) {
          dst[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
          dst[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
        } else {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = (uint32_t)f32_to_16bit(x[2 * k], DT) | (uint32_t)f32_to_16bit(x[2 * k + 1], DT) << 16;
          dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < LR_EACH; ++k)
        if (first + k * step < p.V) store_f(p.out, off + k * step, x[k], DT);
    }
    const long long d = draft[at];
    if (p.penal && d >= v0 && d < min(v0 + LR_TOKENS, p.V)) {     // the rows after this one count it
      const int k = mine((int)(d - v0));
      if (k >= 0) {
        met |= 1u << k, again |= 1u << k;
#pragma unroll
        for (int y = 0; y < LR_EACH; ++y) c[y] += y == k;
      }
    }
  };
  for (int i = 0; i < p.R; i += 2) {
    row(i, 0);
    if (i + 1 < p.R) row(i + 1, 1);
  }
}

// counts[b, v] += how often v is among tokens[b, :]; negative ones are none.
__global__ void __launch_bounds__(256) count_tokens_kernel(int* counts, long long ld_c, const long long* tokens, long long ld_t,
                                                           int B, int N, int V, int* err) {
  griddep_launch_dependents();
  griddep_wait();
  const long long all = (long long)B * N;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
    const long long b = i / N, v = tokens[b * ld_t + i % N];
    if (v < 0) continue;
    if (v < V)
      atomicAdd(counts + b * ld_c + v, 1);
    else if (err)
      atomicOr(err, SIMSD_DEV_ERR_BAD_INDEX);
  }
}

}  // namespace simsd
