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
// HBM bounds it: every logit read and written once.  A warp takes 256 tokens of one sequence
// through all its rows, so that counts, the prompt's bits and the biases are read once a sequence; what
// stays of them in registers is two factors and a number to add for each token.  Several rows are on
// their way at a time.  After row i the lane that owns drafted token i counts it.  Each warp looks through
// the bias list itself, an entry a lane, and needs no barrier.
//
// Measured (B200, device time in a graph of calls; bf16, 151936 tokens, counts, prompt bits, 300 biases and a mask a
// row): 64 x 8 rows 83.6 us, 4.3 TB/s (66 % of the bytes' time at the copy rate), without biases 73.5, with no
// rule at all 52 (91 %); 64 x 1 row 35.  A CTA for 2048 tokens with the biases and drafts in shared memory took
// 117, 101, 61 and 45: some 100 instructions a warp's row instead of 150, and no waits for the CTA.  What is left is the
// setup, 570 instructions a warp and its loads' latency, at 60 % of the issue slots.  A list of n biases is read by each
// of the V / 256 warps of a sequence: 3000 take 194 us, 10000 518, most of it the lists.  fp32, 32 x 4 rows 41 us (66 %).
// Rows whose 8 tokens do not lie on 16 bytes take 2.8 times their bytes' time (64 x 4 x 151937: 86 us; fp32, 32 x 4 x
// 50021: 22, 2.5 times), loads and stores of single numbers.
#pragma once
#include "paged.cuh"
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

constexpr int LR_THREADS = 128, LR_EACH = 8, LR_TOKENS = 32 * LR_EACH;   // tokens of a warp
constexpr int LR_CTAS = 8;                        // CTAs that an SM holds; 9, with spills: 90 us at 64 x 8, not 84

// VEC: a lane owns 8 tokens in a row (16-byte loads and stores), else 8 tokens 32 apart, a warp's next to
// each other (rows that start anywhere).  PENAL: one of the penalties is there.
template <int DT, bool VEC, bool PENAL>
__global__ void __launch_bounds__(LR_THREADS, LR_CTAS) logit_rules_kernel(const LogitRulesArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int VECS = DT == 2 ? 2 : 1;           // 16-byte loads of 8 logits
  // rows in registers: with penalties 4 take 98 us at 64 x 8 at best where 2 took 89.5; without, 52 and 54
  constexpr int ROWS = VEC && DT != 2 && !PENAL ? 4 : 2;
  constexpr int SIZE = DT == 2 ? 4 : 2;
  constexpr int step = VEC ? 1 : 32;
  const int lane = threadIdx.x & 31, b = blockIdx.y;
  const int w0 = (blockIdx.x * (LR_THREADS / 32) + (threadIdx.x >> 5)) * LR_TOKENS;
  if (w0 >= p.V) return;
  const int first = VEC ? w0 + lane * LR_EACH : w0 + lane;   // the lane's tokens: first + k step
  const bool in = first < p.V;
  // who owns token w0 + at, and as which of its own
  auto owner = [](int at) { return VEC ? at / LR_EACH : at % 32; };
  auto place = [](int at) { return VEC ? at % LR_EACH : at / 32; };
  // 8 bits of a word list, the lane's tokens'
  auto bits = [&](const uint32_t* w) {
    if (VEC) return w[first / 32] >> first % 32 & 0xffu;
    const int words = (p.V + 31) / 32;
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < LR_EACH; ++k) {
      const int at = w0 / 32 + k;
      m |= (at < words ? w[at] >> lane & 1u : 0u) << k;
    }
    return m;
  };

  // rows that are on their way
  uint4 raw[VEC ? ROWS : 1][VECS];
  float val[VEC ? 1 : ROWS][LR_EACH];
  uint32_t ok[ROWS];
  const char* src = static_cast<const char*>(p.logits) + (b * p.ld_b + first) * SIZE;
  const uint32_t* mask = p.allowed ? p.allowed + b * p.lda_b : nullptr;
  auto fetch = [&](int at, int row) {
    ok[at] = 0xffu;
    if (in && row < p.R) {
      if constexpr (VEC) {
#pragma unroll
        for (int x = 0; x < VECS; ++x) raw[at][x] = reinterpret_cast<const uint4*>(src)[x];
      } else {
#pragma unroll
        for (int k = 0; k < LR_EACH; ++k)
          if (first + k * step < p.V) val[at][k] = load_f(src, k * step, DT);
      }
      if (mask) ok[at] = bits(mask);
    }
    src += p.ld_r * SIZE;
    if (mask) mask += p.lda_r;
  };
#pragma unroll
  for (int x = 0; x < ROWS; ++x) fetch(x, x);

  // what the sequence has, all of it sent for before any is waited for
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  uint32_t again = 0;                             // tokens that the repetition penalty holds for
  const int* counts = PENAL && p.counts ? p.counts + b * p.ld_c + first : nullptr;
  const long long* drafts = PENAL && p.drafts ? p.drafts + b * p.ld_d : nullptr;
  int c[LR_EACH];
#pragma unroll
  for (int k = 0; k < LR_EACH; ++k) c[k] = 0;
  int d = -1;                                     // drafted token of row 32 i + lane, where it is the warp's
  uint32_t drafted = 0;                           // the rows that have one
  auto draft_of = [&](int row) { return drafts && row + lane + 1 < p.R ? drafts[row + lane] : -1; };
  auto stage_drafts = [&](long long v) {
    d = v >= w0 && v < min((long long)w0 + LR_TOKENS, (long long)p.V) ? (int)(v - w0) : -1;
    drafted = __ballot_sync(0xffffffffu, d >= 0);
  };
  long long draft = -1;
  if constexpr (PENAL) {
    draft = draft_of(0);
    if (counts && in) {
      if (VEC) {
        const int4 x = reinterpret_cast<const int4*>(counts)[0], y = reinterpret_cast<const int4*>(counts)[1];
        c[0] = x.x, c[1] = x.y, c[2] = x.z, c[3] = x.w, c[4] = y.x, c[5] = y.y, c[6] = y.z, c[7] = y.w;
      } else {
#pragma unroll
        for (int k = 0; k < LR_EACH; ++k)
          if (first + k * step < p.V) c[k] = counts[k * step];
      }
    }
    if (p.seen && in) again = bits(p.seen + b * p.ld_s);
    if (p.repetition) rep = p.repetition[b];
    if (p.presence) pres = p.presence[b];
    if (p.frequency) freq = p.frequency[b];
  }

  // per token: what is added
  float add[LR_EACH];
#pragma unroll
  for (int k = 0; k < LR_EACH; ++k) add[k] = 0.0f;
  const int* ids = p.bias_ids + b * p.ld_i;
  const float* values = p.bias + b * p.ld_v;
  // entries of a lane at a time; hardly ever is one of them the warp's
  constexpr int LIST = 4;
  const uint32_t mine = min(LR_TOKENS, p.V - w0);
  for (int base = 0; base < p.n_bias; base += 32 * LIST) {
    int id[LIST];
    bool any = false;
#pragma unroll
    for (int q = 0; q < LIST; ++q) {
      id[q] = base + q * 32 + lane < p.n_bias ? ids[base + q * 32 + lane] : -1;
      any |= (uint32_t)id[q] - (uint32_t)w0 < mine;
    }
    if (w0 == 0 && p.err) {
#pragma unroll
      for (int q = 0; q < LIST; ++q)
        if (id[q] >= p.V) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
    }
    if (!__any_sync(0xffffffffu, any)) continue;
#pragma unroll
    for (int q = 0; q < LIST; ++q) {
      // in the list's order
      uint32_t who = __ballot_sync(0xffffffffu, (uint32_t)id[q] - (uint32_t)w0 < mine);
      for (; who != 0; who &= who - 1) {
        const int from = __ffs(who) - 1, at = __shfl_sync(0xffffffffu, id[q], from) - w0;
        const float v = owner(at) == lane ? values[base + q * 32 + from] : 0.0f;
#pragma unroll
        for (int k = 0; k < LR_EACH; ++k) add[k] += place(at) == k ? v : 0.0f;
      }
    }
  }
  const float inv = 1.0f / rep;
  float up[LR_EACH], down[LR_EACH];               // factors of a logit over 0 and of another one
  if constexpr (PENAL) {
    stage_drafts(draft);
    if (c[0] | c[1] | c[2] | c[3] | c[4] | c[5] | c[6] | c[7]) {
#pragma unroll
      for (int k = 0; k < LR_EACH; ++k)
        if (c[k] > 0) add[k] -= fmaf(freq, (float)c[k], pres), again |= 1u << k;
    }
#pragma unroll
    for (int k = 0; k < LR_EACH; ++k) up[k] = again >> k & 1 ? inv : 1.0f, down[k] = again >> k & 1 ? rep : 1.0f;
  }

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
    for (int k = 0; k < LR_EACH; k += 2) {
      uint64_t z = f2_pack(x[k], x[k + 1]);
      const uint64_t y = f2_pack(add[k], add[k + 1]);
      if (PENAL)
        z = f2_fma(z, f2_pack(x[k] > 0.0f ? up[k] : down[k], x[k + 1] > 0.0f ? up[k + 1] : down[k + 1]), y);
      else
        z = f2_add(z, y);
      const float2 w = f2_unpack(z);
      x[k] = w.x, x[k + 1] = w.y;
    }
    if ((!VEC || DT == 2) && ok[at] != 0xffu) {
#pragma unroll
      for (int k = 0; k < LR_EACH; ++k)
        if (!(ok[at] >> k & 1)) x[k] = -INFINITY;
    }
    if constexpr (VEC) {
      uint4* to = reinterpret_cast<uint4*>(dst);
      if constexpr (DT == 2) {
        if (in) {
          to[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
          to[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
        }
      } else {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (DT == 0)
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(x[2 * k + 1]), "f"(x[2 * k]));
          else
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(x[2 * k + 1]), "f"(x[2 * k]));
        }
        if (p.allowed) {
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
        if (in) to[0] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < LR_EACH; ++k)
        if (first + k * step < p.V) store_f(dst, k * step, x[k], DT);
    }
    dst += p.ldo_r * SIZE;
    if (PENAL && drafted >> (i & 31) & 1) {       // the rows after this one count it
      const int at = __shfl_sync(0xffffffffu, d, i & 31), token = w0 + at;
      float sum = 0.0f;                           // its biases once more
      for (int y = 0; y < p.n_bias; y += 32) {
        const int id = y + lane < p.n_bias ? ids[y + lane] : -1;
        for (uint32_t who = __ballot_sync(0xffffffffu, id == token); who != 0; who &= who - 1) sum += values[y + __ffs(who) - 1];
      }
      int n = 0;
      for (int y = lane; y <= i; y += 32) n += drafts[y] == token;
      n = __reduce_add_sync(0xffffffffu, n);
      if (owner(at) == lane) {
        const int k = place(at), all = n + (counts ? counts[k * step] : 0);
        const float now = all > 0 ? sum - fmaf(freq, (float)all, pres) : sum;
#pragma unroll
        for (int y = 0; y < LR_EACH; ++y)
          if (y == k) {
            add[y] = now;
            if (all > 0) up[y] = inv, down[y] = rep;
          }
      }
    }
  };
  for (int i = 0; i < p.R; i += ROWS) {
    if (PENAL && i % 32 == 0 && i > 0) stage_drafts(draft_of(i));
#pragma unroll
    for (int x = 0; x < ROWS; ++x) {
      if (i + x < p.R) row(i + x, x);
      fetch(x, i + x + ROWS);
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
