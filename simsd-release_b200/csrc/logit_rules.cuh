// Rules on logits before a token is drawn: penalties for repeated tokens, biases and
// grammar masks, for every drafted row of a sequence.  Row i of sequence b, token v, with
//   c = counts[b, v] + the number of j < i with drafts[b, j] = v:
//   x = logits[b, i, v]
//   x = x > 0 ? x / repetition[b] : x repetition[b]     where c > 0 or seen[b] has v
//   x = x - frequency[b] c - presence[b]                where c > 0
//   x = x + the biases of v in sequence b's list, summed in the list's order
//   x = -inf                                            where allowed[b, i] lacks v
// in fp32 (x times a factor plus one number, the division as a product with the reciprocal),
// rounded once to the logits' type.
//
// HBM bounds it: every logit read and written once.  A CTA takes 2048 tokens of one
// sequence through all its rows, so that counts, the prompt's bits and the biases are
// read once a sequence; what stays of them in registers is a number to add and a bit for each token.
// After row i the thread that owns drafted token i counts it.  Several rows are on their way at a time.
// Its threads look through the bias list, an entry each, for those on the CTA's tokens.
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

constexpr int LR_THREADS = 256, LR_EACH = 8, LR_TOKENS = LR_THREADS * LR_EACH, LR_LIST = 1024;

// VEC: a thread owns 8 tokens in a row (16-byte loads and stores), else 8 tokens 32
// apart, a warp's next to each other (rows that start anywhere).
template <int DT, bool VEC>
__global__ void __launch_bounds__(LR_THREADS, 4) logit_rules_kernel(const LogitRulesArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int VECS = DT == 2 ? 2 : 1;           // 16-byte loads of 8 logits
  constexpr int ROWS = VEC && DT != 2 ? 4 : 2;    // rows in registers
  constexpr int SIZE = DT == 2 ? 4 : 2;
  __shared__ int s_draft[LR_THREADS], s_hit[LR_LIST], s_order[LR_LIST], s_hits;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.y;
  const int v0 = blockIdx.x * LR_TOKENS, w0 = v0 + warp * 32 * LR_EACH;
  const int first = VEC ? w0 + lane * LR_EACH : w0 + lane;   // the thread's tokens: first + k step
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

  // rows that are on their way; the next one's places
  uint4 raw[VEC ? ROWS : 1][VECS];
  float val[VEC ? 1 : ROWS][LR_EACH];
  uint32_t ok[ROWS];
  const char* src = static_cast<const char*>(p.logits) + (b * p.ld_b + first) * SIZE;
  const uint32_t* mask = p.allowed ? p.allowed + b * p.lda_b : nullptr;
  int fetched = 0;
  auto fetch = [&](int at) {
    ok[at] = 0xffu;
    if (fetched >= p.R) return;
    if constexpr (VEC) {
      if (first < p.V) {
#pragma unroll
        for (int x = 0; x < VECS; ++x) raw[at][x] = reinterpret_cast<const uint4*>(src)[x];
      }
    } else {
#pragma unroll
      for (int k = 0; k < LR_EACH; ++k)
        if (first + k * step < p.V) val[at][k] = load_f(src, k * step, DT);
    }
    if (mask) ok[at] = bits(mask), mask += p.lda_r;
    src += p.ld_r * SIZE;
    ++fetched;
  };
#pragma unroll
  for (int x = 0; x < ROWS; ++x) fetch(x);

  // what the sequence has, all of it sent for before any is waited for
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  uint32_t again = 0;                             // tokens that the repetition penalty holds for
  const int* counts = p.counts ? p.counts + b * p.ld_c + first : nullptr;
  int c[LR_EACH];
#pragma unroll
  for (int k = 0; k < LR_EACH; ++k) c[k] = 0;
  if (p.penal) {
    if (counts) {
      if (VEC) {
        if (first < p.V) {
          const int4 a = reinterpret_cast<const int4*>(counts)[0], d = reinterpret_cast<const int4*>(counts)[1];
          c[0] = a.x, c[1] = a.y, c[2] = a.z, c[3] = a.w, c[4] = d.x, c[5] = d.y, c[6] = d.z, c[7] = d.w;
        }
      } else {
#pragma unroll
        for (int k = 0; k < LR_EACH; ++k)
          if (first + k * step < p.V) c[k] = counts[k * step];
      }
    }
    if (p.seen) again = bits(p.seen + b * p.ld_s);
    if (p.repetition) rep = p.repetition[b];
    if (p.presence) pres = p.presence[b];
    if (p.frequency) freq = p.frequency[b];
  }
  auto stage_drafts = [&](int i) {                // rows i on: their drafted tokens that are the CTA's
    const long long v = p.drafts && i + tid + 1 < p.R ? p.drafts[b * p.ld_d + i + tid] : -1;
    s_draft[tid] = v >= v0 && v < min(v0 + LR_TOKENS, p.V) ? (int)(v - v0) : -1;
  };
  if (p.penal) stage_drafts(0);

  // per token: what is added
  float add[LR_EACH];
#pragma unroll
  for (int k = 0; k < LR_EACH; ++k) add[k] = 0.0f;
  const int* ids = p.bias_ids + b * p.ld_i;
  const float* values = p.bias + b * p.ld_v;
  for (int base = 0; base < p.n_bias; base += LR_LIST) {
    // the list's entries that are the CTA's, as (place in the list, token), in the list's order: found in any, then ranked
    const int n = min(LR_LIST, p.n_bias - base);
    if (tid == 0) s_hits = 0;
    __syncthreads();
    for (int x = tid; x < n; x += LR_THREADS) {
      const int id = ids[base + x];
      if (id >= p.V && blockIdx.x == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
      if ((uint32_t)(id - v0) < (uint32_t)LR_TOKENS && id < p.V) s_hit[atomicAdd(&s_hits, 1)] = x * LR_TOKENS + id - v0;
    }
    __syncthreads();
    const int hits = s_hits;
    for (int x = tid; x < hits; x += LR_THREADS) {
      int rank = 0;
      for (int y = 0; y < hits; ++y) rank += s_hit[y] < s_hit[x];
      s_order[rank] = s_hit[x];
    }
    __syncthreads();
    for (int x = 0; x < hits; ++x) {
      const int hit = s_order[x], k = mine(hit % LR_TOKENS);
      if (k < 0) continue;
      const float v = values[base + hit / LR_TOKENS];
#pragma unroll
      for (int y = 0; y < LR_EACH; ++y) add[y] += y == k ? v : 0.0f;
    }
  }
  const float inv = 1.0f / rep;
#pragma unroll
  for (int k = 0; k < LR_EACH; ++k)
    if (c[k] > 0) add[k] -= fmaf(freq, (float)c[k], pres), again |= 1u << k;

  char* dst = static_cast<char*>(p.out) + (b * p.ldo_b + first) * SIZE;
  auto row = [&](int i, int at) {
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
#pragma unroll
    for (int k = 0; k < LR_EACH; ++k) x[k] = fmaf(x[k], again >> k & 1 ? x[k] > 0.0f ? inv : rep : 1.0f, add[k]);
    if ((!VEC || DT == 2) && ok[at] != 0xffu) {
#pragma unroll
      for (int k = 0; k < LR_EACH; ++k)
        if (!(ok[at] >> k & 1)) x[k] = -INFINITY;
    }
    if constexpr (VEC) {
      if (first < p.V) {
        uint4* to = reinterpret_cast<uint4*>(dst);
        if constexpr (DT == 2) {
          to[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
          to[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
        } else {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (DT == 0)
              asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(x[2 * k + 1]), "f"(x[2 * k]));
            else
              asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(x[2 * k + 1]), "f"(x[2 * k]));
          }
          if (ok[at] != 0xffu) {
            // four bits to the top bits of four bytes, and those over the two halves of two words
            constexpr uint32_t LOW = DT == 0 ? 0xff80ff80u : 0xfc00fc00u;      // two -inf
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t t = (ok[at] >> 4 * h & 15u) * 0x10204080u;
              uint32_t m0, m1;
              asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(m0) : "r"(t));          // a byte's top bit, eight times
              asm("prmt.b32 %0, %1, 0, 0xbbaa;" : "=r"(m1) : "r"(t));
              w[2 * h] = (w[2 * h] & m0) | (LOW & ~m0), w[2 * h + 1] = (w[2 * h + 1] & m1) | (LOW & ~m1);
            }
          }
          to[0] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < LR_EACH; ++k)
        if (first + k * step < p.V) store_f(dst, k * step, x[k], DT);
    }
    dst += p.ldo_r * SIZE;
    const int d = p.penal ? s_draft[i % LR_THREADS] : -1;
    if (d >= 0 && d / (32 * LR_EACH) == warp) {   // the rows after this one count it
      float sum = 0.0f;                           // its biases once more
#pragma unroll 4
      for (int y = 0; y < p.n_bias; y += 32) {
        const int id = y + lane < p.n_bias ? ids[y + lane] : -1;
        for (uint32_t who = __ballot_sync(0xffffffffu, id == v0 + d); who != 0; who &= who - 1) sum += values[y + __ffs(who) - 1];
      }
      const int k = mine(d);
      if (k >= 0) {
        int c = counts ? counts[k * step] : 0;
        for (int y = 0; y <= i; ++y) c += p.drafts[b * p.ld_d + y] == v0 + d;
        const float now = c > 0 ? sum - fmaf(freq, (float)c, pres) : sum;
        if (c > 0) again |= 1u << k;
#pragma unroll
        for (int y = 0; y < LR_EACH; ++y) add[y] = y == k ? now : add[y];
      }
    }
  };
  for (int i = 0; i < p.R; i += ROWS) {
    if (p.penal && i % LR_THREADS == 0) {
      if (i > 0) {
        __syncthreads();
        stage_drafts(i);
      }
      __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < ROWS; ++x) {
      if (i + x < p.R) row(i + x, x);
      fetch(x);
    }
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
