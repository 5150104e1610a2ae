// Attention of a few query tokens per sequence over a paged key-value cache.
//   o[b, t, h, :] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max),
// over the visible keys j < n = min(seq_lens[b], max_pages page_size) of KV head
// g = h / G (G = Hq / Hk).  The newest L keys belong to the L query tokens: with jt
// = j - (n - L), a key with jt < 0 is visible to all of them, the others where
// jt <= t, or where tail_mask[b, t, jt] is set.  No visible key: o = 0, lse = -inf.
//
// This file: up to 16 rows (G L) per KV head; more in paged_attn_tc.cuh.
//
// What bounds it: every key and value is read once for the G L rows that share it
// (4 G L operations per 2-byte element), so up to some 64 rows HBM bounds it and
// the work is to keep loads in flight on every SM and to cut any mix of lengths
// evenly.
//
// Split.  A unit is TK keys of one (sequence, KV head, row tile); the units of the
// whole call, in that order, are cut into equal contiguous ranges, one per CTA of
// what the SMs hold at once, from the lengths on the device (no host knowledge of them, so a
// graph replays as sequences grow).  A range may hold many short sequences or a
// slice of a long one; a sequence cut between CTAs leaves each part's (O, max,
// sum) in the workspace, and the last of its CTAs to finish (a counter per first
// CTA, zero again afterwards) joins the parts, always in key order.
//
// In a CTA each of four warps takes 16 keys of every unit through a ring of its own
// (cp.async, no barrier between warps until the sequence ends), loading ahead across
// sequence ends; the next sequence's queries are fetched a sequence ahead.
// Products with the roles swapped, so that few rows waste little: S^T = K Q^T
// (m16n8k16: 16 keys x 8 rows), P^T turned into the second product's operand with
// movmatrix, O^T = V^T P^T (16 dims x 8 rows).  Softmax in fp32 with exp2 of
// log2-scaled scores; the running maximum moves (and O is rescaled) only when a
// score exceeds it.  P is rounded to the 16-bit type for the second product: the
// weights are <= 1 and their sum, kept in fp32, is of the unrounded ones, so the
// rounding errs by at most half a step per weight (bf16: error 1.8e-3 of the output in the
// 2-norm against 1.7e-3 for its own rounding alone).  A second product of what the rounding
// leaves would double the tensor work for that.
//
// Masked keys: keys past n are zero-filled in shared memory, whatever stale memory
// holds.  A tail key that some rows of the unit see and others do not takes part
// with weight 0 in the second product; where its value is not finite (0 x inf), the
// unit's product runs row by row with the hidden keys zeroed instead.  An infinite value
// that a row sees gives an infinite output, but NaN in fp16 where its weight is under 2^-25
// and rounds to 0.
//
// Measured (B200, 8 KV heads x 128, 4 query heads each, bf16; device time in a graph of
// calls, in brackets calls one after the other on a stream): 2 x 120-128k tokens 173 us
// (177), 6.2 TB/s, 94 % of the measured copy rate; 32 x 0.3-4k 38 us (40), 4.7 TB/s, 72 %;
// 1 x 100 7.9 us (10.2, the host's time for a call).
// With a window only the units that some row sees are cut up: 16 x 8-32k tokens in a window of 4096 and 4
// first keys 52 us, 5.2 TB/s, 79 %.
#pragma once
#include "paged.cuh"

namespace simsd {

struct PagedAttnArgs {
  const void* q;            // [B, L, Hq, D]
  const void* k_cache;
  const void* v_cache;
  const int* page_table;    // [B, ld_table]
  const int* seq_lens;      // [B]
  const uint8_t* tail;      // [B, L, L] bytes or nullptr
  void* o;                  // [B, L, Hq, D]
  float* lse;               // [B, L, Hq] or nullptr
  int* err;
  int* arrived;             // [grid]: parts written of the cut sequence that starts in that CTA; zero between calls
  float4* part_o;           // [2 grid][D / 16][NR / 8][32] fragments
  float2* part_ml;          // [2 grid][NR] (max in log2 units, sum)
  long long ld_page, ld_head, ld_tok, ld_table, ldm_b, ldm_t;
  int B, L, Hq, Hk, G, num_pages, page_size, max_pages, rows, row_tiles;
  PagedDiv page_div, g_div; // by page_size, by G
  int window, sinks;        // a query at position x sees j > x - window and j < sinks; read where WIN
  uint32_t q_sign;          // 0x80008000 flips the queries' signs (a negative scale)
  float scale_log2;         // |scale| log2(e), positive
};

// A CTA is 4 warps of 16 keys (a unit is one step of all of them) x NT 8-row tiles.
constexpr int PAT_WARPS = 4, PAT_THREADS = PAT_WARPS * 32, PAT_TK = 16 * PAT_WARPS;
constexpr int PAT_CTAS_PER_SM = 2;
// CTAs of the forms with tcgen05 at most: a sequence may be cut between all of them, and who joins its parts holds a
// maximum and a sum of every part's rows in shared memory (their shapes assert it; a B200 has 148 SMs).
constexpr int PTC_MAX_PARTS = 156;

template <int D, int NT>
struct PatShape {
  static constexpr int NR = NT * 8;
  static constexpr int STAGES = 3;
  static constexpr int MAT = 16 * D * 2;                       // 16 keys (or values)
  static constexpr int RING = PAT_WARPS * STAGES * 2 * MAT;
  static constexpr int OBUF = PAT_WARPS * (D / 16) * 32 * 16;  // one 8-row tile of every warp's O
  static constexpr int ML = 2 * PAT_WARPS * NR * 4;
  static constexpr int BYTES = RING + OBUF + ML;
};

// the warps that hold O; another one of the CTA may be loading
__device__ __forceinline__ void pat_sync() { named_bar_sync(1, PAT_THREADS); }
__device__ __forceinline__ void pat_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pat_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t pat_transpose(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <bool BF>
__device__ __forceinline__ void pat_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF>
__device__ __forceinline__ uint32_t pat_pack(float lo, float hi) {
  uint32_t r;
  if (BF)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float pat_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 16 bytes into shared memory, zeros where !ok (nothing is read then)
__device__ __forceinline__ void pat_cp16(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void pat_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pat_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ int paged_len(const PagedAttnArgs& p, int b) {
  const int n = p.seq_lens[b];
  const long long cap = (long long)p.max_pages * p.page_size;
  return n < 0 ? 0 : n > cap ? (int)cap : n;
}
// units of one (head, row tile) of a sequence; an empty one has a unit, which writes its rows
template <int TK>
__device__ __forceinline__ int paged_units(int n) {
  return n <= TK ? 1 : (n + TK - 1) / TK;
}

// The end of a sequence's row tile (joining the warps, writing, the next queries) takes
// a CTA as long as one or two units do, and is weighed as that many in the cut: with
// 64-key units 64 sequences of 0.1 - 2k tokens take 50 us at 0, 44 at 1, 40 at 2 and 32
// of 0.3 - 4k 41, 38, 38; with the 128-key units of paged_attn_tc.cuh 16 x 8 rows take
// 41, 39.5, 41.
template <int TK>
struct PagedEnd {
  static constexpr int UNITS = TK == 64 ? 2 : 1;
};
constexpr int PAGED_END_MAX = 2;

// Through a window, the first key after the sinks that some row of a sequence of n sees
__device__ __forceinline__ int paged_first(const PagedAttnArgs& p, int n) {
  return (int)max(0LL, (long long)n - p.L + 1 - p.window);
}
// units of TK keys between those of the sinks and that key's: no row sees any of their keys
template <int TK>
__device__ __forceinline__ int paged_skip(const PagedAttnArgs& p, int n) {
  return max(0, paged_first(p, n) / TK - (p.sinks / TK + (p.sinks % TK != 0)));
}

// whether a window hides one of `keys` keys from key0 on from a row of the last token, at n - 1
__device__ __forceinline__ bool paged_out(const PagedAttnArgs& p, int n, int key0, int keys) {
  return key0 < n - p.window && key0 + keys > p.sinks;
}

// Position in the unit order: sequence b (length n, nu units per KV head and row
// tile), KV head g, row tile rt, unit of it; w counts units and ends before it.
// WIN: through a window, whose units are the sequence's but the `skip` ones in its middle.
template <int TK, bool WIN = false, int ENDS = PagedEnd<TK>::UNITS>
struct PagedPos {
  static constexpr int END = ENDS;
  int b, g, rt, unit, n, nu, w, skip;
  __device__ __forceinline__ void next(const PagedAttnArgs& p) {
    ++w;
    if (++unit < nu) return;
    w += END;
    unit = 0;
    if (!next_rows(p, b, g, rt) || b >= p.B) return;
    measure(p);
  }
  __device__ __forceinline__ void measure(const PagedAttnArgs& p) {
    n = paged_len(p, b);
    skip = WIN ? paged_skip<TK>(p, n) : 0;
    nu = paged_units<TK>(n) - skip;
  }
  // the unit's first key
  __device__ __forceinline__ int key(const PagedAttnArgs& p) const {
    return (WIN && unit >= p.sinks / TK + (p.sinks % TK != 0) ? unit + skip : unit) * TK;
  }
  // the row tile, head or sequence after (b, g, rt); true for another sequence
  __device__ static __forceinline__ bool next_rows(const PagedAttnArgs& p, int& b, int& g, int& rt) {
    if (++rt < p.row_tiles) return false;
    rt = 0;
    if (++g < p.Hk) return false;
    g = 0;
    ++b;
    return true;
  }
};

// The equal cut of `total` units and ends over `ctas` CTAs, the first `extra` of which have one more
struct PagedCut {
  int ctas, base, extra;
  __device__ __forceinline__ int first(int c) const { return c * base + min(c, extra); }
  __device__ __forceinline__ int cta_of(int u) const {
    const int lead = extra * (base + 1);
    return u < lead ? u / (base + 1) : extra + (u - lead) / base;
  }
};

// Whether query row r (token t = r / G) sees key j, j < n or not; rows past the last
// one count as the last token's.  No branch around the mask's byte, so that several are fetched at once.
template <bool WIN = false>
__device__ __forceinline__ bool paged_visible(const PagedAttnArgs& p, int b, int n, int j, int r) {
  const int t = min(p.g_div(r), p.L - 1), jt = j - (n - p.L);
  bool see = jt <= t;
  if (p.tail) see = jt < 0 || p.tail[b * p.ldm_b + t * p.ldm_t + max(0, min(jt, p.L - 1))] != 0;
  if (WIN) see = see && (j < p.sinks || jt > t - p.window);
  return see && j < n;
}

// Where row r of KV head g lies in o and lse, in heads
__device__ __forceinline__ long long paged_row(const PagedAttnArgs& p, int b, int g, int r) {
  const int t = p.g_div(r);
  return ((long long)b * p.L + t) * p.Hq + g * p.G + (r - t * p.G);
}
// 16 dims (from mt * 16) of 8 rows (from r8) out of a fragment of O^T (v: dims d, d
// + 8 of two rows): packed and transposed, so that a lane holds two dims of row
// lane / 4 and stores 4 bytes twice.  `row`: the lane's row's place, or -1.
template <bool BF, int D>
__device__ __forceinline__ void paged_store(const PagedAttnArgs& p, long long row, int mt, int lane, float4 v) {
  const uint32_t lo = pat_transpose(pat_pack<BF>(v.x, v.y)), hi = pat_transpose(pat_pack<BF>(v.z, v.w));
  if (row < 0) return;
  uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(p.o) + row * D + mt * 16) + (lane & 3);
  dst[0] = lo;
  dst[4] = hi;
}
__device__ __forceinline__ void paged_store_lse(const PagedAttnArgs& p, int b, int g, int r, float m, float l) {
  if (p.lse == nullptr || r >= p.rows) return;
  p.lse[paged_row(p, b, g, r)] = l == 0.0f ? -INFINITY : fmaf(0.69314718055994531f, m, logf(l));
}

// This CTA's place in the cut of the call's units and ends, and the position of its
// first unit.  False: this CTA has none.
template <int THREADS, int TK, bool WIN = false, int ENDS>
__device__ __forceinline__ bool paged_range(const PagedAttnArgs& p, PagedCut& cut, PagedPos<TK, WIN, ENDS>& pos) {
  constexpr int WARPS = THREADS / 32;
  __shared__ int s_sum[WARPS], s_more[WARPS];
  __shared__ int s_b, s_first;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = p.Hk * p.row_tiles;
  const bool flag = blockIdx.x == 0 && p.err != nullptr;
  auto units = [&](int b) {
    if (b >= p.B) return 0;
    if (flag && p.seq_lens[b] > (long long)p.max_pages * p.page_size) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
    const int n = paged_len(p, b), skip = WIN ? paged_skip<TK>(p, n) : 0;
    return (paged_units<TK>(n) - skip + ENDS) * per;
  };
  // sequences tid, tid + THREADS, ...: the first of them scanned, the others summed
  int u = units(tid), incl = u, more = 0;
  for (int b = tid + THREADS; b < p.B; b += THREADS) more += units(b);
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, m);
    if (lane >= m) incl += v;
    more += __shfl_xor_sync(0xffffffffu, more, m);
  }
  if (lane == 31) s_sum[warp] = incl, s_more[warp] = more;
  __syncthreads();
  int off = 0, head = 0, total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) off += s_sum[w];
    head += s_sum[w];
    total += s_sum[w] + s_more[w];
  }
  cut.ctas = min((int)gridDim.x, total);
  const int c = blockIdx.x;
  if (c >= cut.ctas) return false;
  cut.base = total / cut.ctas;
  cut.extra = total - cut.base * cut.ctas;
  const int w0 = cut.first(c);
  if (off + incl - u <= w0 && w0 < off + incl) s_b = tid, s_first = off + incl - u;
  for (int base = THREADS, before = head; before <= w0; base += THREADS) {   // past the first sequences
    u = incl = units(base + tid);
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, m);
      if (lane >= m) incl += v;
    }
    __syncthreads();
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    off = before;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) off += s_sum[w];
      before += s_sum[w];
    }
    if (off + incl - u <= w0 && w0 < off + incl) s_b = base + tid, s_first = off + incl - u;
  }
  __syncthreads();
  pos.b = s_b;
  pos.measure(p);
  const int rem = w0 - s_first, hr = rem / (pos.nu + ENDS);
  pos.unit = rem - hr * (pos.nu + ENDS);
  pos.w = w0;
  pos.g = hr / p.row_tiles;
  pos.rt = hr - pos.g * p.row_tiles;
  if (pos.unit >= pos.nu) {          // an end: the unit after it
    const int w = w0 + pos.nu + ENDS - pos.unit;
    pos.unit = pos.nu - 1;
    pos.next(p);
    pos.w = w;
  }
  return pos.w < cut.first(c + 1);
}

// A cut sequence (one KV head and row tile, rows from r0): its first CTA and how many it lies in
struct PagedPart {
  int b, g, r0, c0, parts;
};

// Counts a part that its CTA has written (and a barrier has followed) in; by one thread.  True for the last.
__device__ __forceinline__ bool paged_arrive(const PagedAttnArgs& p, const PagedPart& x) {
  __threadfence();
  const bool last = atomicAdd(p.arrived + x.c0, 1) == x.parts - 1;
  if (last) p.arrived[x.c0] = 0;
  __threadfence();
  return last;
}

// Joins the parts of a cut sequence (one KV head and row tile of it) that starts
// in CTA c0: part i's max, sum and O lie in slot 1 of CTA c0 for i = 0, in slot 0
// of CTA c0 + i for the others.  `buf`: `room` bytes of shared memory, at least
// a part's O and its weights and 2 KB.  The parts of O come in by cp.async, as many at a time as there is room
// for (28 parts one after the other, four on their way, took 7 us at the end of a kernel).
template <int D, int NT, bool BF>
__device__ __noinline__ void paged_join(const PagedAttnArgs& p, int b, int g, int r0, int c0, int parts, uint8_t* buf, int room) {
  constexpr int NR = NT * 8, THREADS = PAT_THREADS, PART = D * NR * 4;
  constexpr int ALL = PART / 16, PER = ALL / THREADS;                    // fragments, and of a thread
  constexpr int GR = THREADS / NR;                                       // threads of a row
  const int tid = threadIdx.x, lane = tid & 31, r = tid % NR, grp = tid / NR;
  auto slot = [&](int i) { return (long long)(i == 0 ? 2 * c0 + 1 : 2 * (c0 + i)); };
  float* red = reinterpret_cast<float*>(buf);                            // [2][GR][NR]
  float* weight = red + 2 * GR * NR;                                     // [parts of a batch][NR]
  const int batch = min(parts, (room - 2 * GR * NR * 4) / (PART + NR * 4));
  const uint32_t stage = smem_u32(weight + batch * NR);
  auto fetch = [&](int i0) {
    const int n = min(batch, parts - i0);
    for (int i = 0; i < n; ++i) {
      const float4* o = p.part_o + slot(i0 + i) * ALL;
#pragma unroll
      for (int k = 0; k < PER; ++k)
        paged_cp16(stage + i * PART + (tid + k * THREADS) * 16, o + tid + k * THREADS);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(0);
  float mm = -INFINITY, ll = 0.0f;
  auto see = [&](float2 x) {
    const float mn = fmaxf(mm, x.x), mu = mn == -INFINITY ? 0.0f : mn;
    ll = fmaf(ll, pat_exp2(mm - mu), x.y * pat_exp2(x.x - mu));
    mm = mn;
  };
#pragma unroll 4
  for (int i = grp; i < parts; i += GR) see(__ldcg(p.part_ml + slot(i) * NR + r));
  red[grp * NR + r] = mm, red[(GR + grp) * NR + r] = ll;
  pat_sync();
  mm = -INFINITY, ll = 0.0f;
#pragma unroll
  for (int k = 0; k < GR; ++k) see(make_float2(red[k * NR + r], red[(GR + k) * NR + r]));
  if (grp == 0) paged_store_lse(p, b, g, r0 + r, mm, ll);
  const float mu = mm == -INFINITY ? 0.0f : mm, inv = ll == 0.0f ? 0.0f : 1.0f / ll;
  float4 a[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) a[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i0 = 0; i0 < parts; i0 += batch) {
    const int n = min(batch, parts - i0);
    for (int i = grp; i < n; i += GR) weight[i * NR + r] = pat_exp2(__ldcg(p.part_ml + slot(i0 + i) * NR + r).x - mu) * inv;
    pat_wait<0>();
    pat_sync();
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int x = tid + k * THREADS;
        const int rr = x / 32 % NT * 8 + 2 * (lane & 3);
        const float f0 = weight[i * NR + rr], f1 = weight[i * NR + rr + 1];
        float4 v;
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(stage + i * PART + x * 16) : "memory");
        a[k].x = fmaf(v.x, f0, a[k].x), a[k].y = fmaf(v.y, f1, a[k].y);
        a[k].z = fmaf(v.z, f0, a[k].z), a[k].w = fmaf(v.w, f1, a[k].w);
      }
    }
    pat_sync();
    if (i0 + batch < parts) fetch(i0 + batch);
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int x = tid + k * THREADS, rr = r0 + x / 32 % NT * 8 + (lane >> 2);
    paged_store<BF, D>(p, rr < p.rows ? paged_row(p, b, g, rr) : -1, x / (NT * 32), lane, a[k]);
  }
}

// The end of a sequence's row tile, or of the CTA's range inside it (whole: neither end was
// cut): the warps are joined, a whole sequence is written, a part goes to the workspace.
// o, m (in log2 units), l: a warp's fragments; l is not summed over the lanes yet.  obuf: room
// for one 8-row tile of O of every warp.
template <int D, int NT, bool BF, typename Pos>
__device__ __forceinline__ void paged_finish(const PagedAttnArgs& p, const Pos& at, bool whole, int part, float (&o)[D / 16][NT][4],
                                             const float (&m)[NT][2], const float (&l)[NT][2], float4* obuf, float* sm_m,
                                             float* sm_l, const PagedCut& range, PagedPart* cuts, bool* joins) {
  constexpr int MT = D / 16, NR = NT * 8;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = 2 * blockIdx.x + part, r0 = at.rt * NR;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[nt][e];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (lane < 4) {
        sm_m[warp * NR + nt * 8 + 2 * lane + e] = m[nt][e];
        sm_l[warp * NR + nt * 8 + 2 * lane + e] = x;
      }
    }
  pat_sync();
  float inv[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = nt * 8 + 2 * (lane & 3) + e;
      float mm = -INFINITY, ll = 0.0f;
#pragma unroll
      for (int w = 0; w < PAT_WARPS; ++w) mm = fmaxf(mm, sm_m[w * NR + r]);
      const float mu = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
      for (int w = 0; w < PAT_WARPS; ++w) ll = fmaf(sm_l[w * NR + r], pat_exp2(sm_m[w * NR + r] - mu), ll);
      const float f = pat_exp2(m[nt][e] - mu);
      inv[nt][e] = !whole ? 1.0f : ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[mt][nt][e] *= f, o[mt][nt][e + 2] *= f;
      if (warp == 0 && lane < 4) {
        if (whole)
          paged_store_lse(p, at.b, at.g, r0 + r, mm, ll);
        else
          p.part_ml[slot * NR + r] = make_float2(mm, ll);
      }
    }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = r0 + nt * 8 + (lane >> 2);
    const long long row = r < p.rows ? paged_row(p, at.b, at.g, r) : -1;
    if (nt > 0) pat_sync();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      obuf[(warp * MT + mt) * 32 + lane] = make_float4(o[mt][nt][0], o[mt][nt][1], o[mt][nt][2], o[mt][nt][3]);
    pat_sync();
#pragma unroll
    for (int k = 0; k < MT / PAT_WARPS; ++k) {
      const int mt = warp + k * PAT_WARPS;
      const float4* from = obuf + mt * 32 + lane;
      float4 a = from[0];
#pragma unroll
      for (int w = 1; w < PAT_WARPS; ++w) {
        const float4 x = from[w * MT * 32];
        a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
      }
      a.x *= inv[nt][0], a.y *= inv[nt][1], a.z *= inv[nt][0], a.w *= inv[nt][1];
      if (whole)
        paged_store<BF, D>(p, row, mt, lane, a);
      else
        p.part_o[(((long long)slot * MT + mt) * NT + nt) * 32 + lane] = a;
    }
  }
  pat_sync();
  if (!whole && tid == 0) {
    const int head = at.w - at.unit, c0 = range.cta_of(head);   // the sequence's first unit and CTA
    cuts[part] = {at.b, at.g, r0, c0, range.cta_of(head + at.nu - 1) - c0 + 1};
    // the first part at once, so that it is not this CTA that everyone else waits for in the end
    if (part == 0) joins[0] = paged_arrive(p, cuts[0]);
  }
}
// Cut sequences (at most the range's first and last): the last of their CTAs to get here joins the parts.
template <int D, int NT, bool BF>
__device__ __forceinline__ void paged_leave(const PagedAttnArgs& p, const PagedPart* cuts, bool* joins, uint8_t* buf, int room) {
  if (threadIdx.x == 0 && cuts[1].parts > 0) joins[1] = paged_arrive(p, cuts[1]);
  pat_sync();
  for (int k = 0; k < 2; ++k) {
    const PagedPart x = cuts[k];
    if (joins[k]) paged_join<D, NT, BF>(p, x.b, x.g, x.r0, x.c0, x.parts, buf, room);
    pat_sync();
  }
}
// Page of `keys` keys (of one page, from `key` on) through a window; PAGED_UNSEEN where no row
// sees any of them: their pages may have been given back.
constexpr int PAGED_UNSEEN = -0x7fffffff;
template <typename Pos>
__device__ __forceinline__ int paged_page(const PagedAttnArgs& p, const Pos& x, int key, int keys) {
  if (key >= x.n) return -1;
  if (key >= p.sinks && key + keys <= paged_first(p, x.n)) return PAGED_UNSEEN;
  return p.page_table[x.b * p.ld_table + p.page_div(key)];
}

template <int D, int NT, bool BF, bool WIN>
__global__ void __launch_bounds__(PAT_THREADS, PAT_CTAS_PER_SM) paged_attention_kernel(const __grid_constant__ PagedAttnArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  using S = PatShape<D, NT>;
  constexpr int NR = S::NR;
  constexpr int MT = D / 16, CH = D / 8;                  // 16-dim tiles, 16-byte chunks of a key
  constexpr int KPI = 32 / CH;                            // keys per cp.async of the warp
  constexpr int QW = MT * NT * 2;                         // words of the queries in a thread
  extern __shared__ __align__(256) uint8_t pat_smem[];
  __shared__ PagedPart s_cut[2];
  __shared__ bool s_join[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ring = smem_u32(pat_smem) + warp * S::STAGES * 2 * S::MAT;
  float4* obuf = reinterpret_cast<float4*>(pat_smem + S::RING);
  float* sm_m = reinterpret_cast<float*>(pat_smem + S::RING + S::OBUF);
  float* sm_l = sm_m + PAT_WARPS * NR;

  __shared__ PagedCut s_range;
  PagedPos<PAT_TK, WIN> ld;
  int end;
  {
    PagedCut cut;
    if (!paged_range<PAT_THREADS, PAT_TK, WIN>(p, cut, ld)) return;
    end = cut.first(blockIdx.x + 1);
    if (tid == 0) s_range = cut;
  }
  if (tid < 2) s_cut[tid].parts = 0, s_join[tid] = false;
  PagedPos<PAT_TK, WIN> at = ld;

  // ---- loads: the warp's 16 keys of position `ld` into its next ring slot.
  // Pages of a multiple of 16 tokens hold all sixteen in one page, a fixed distance
  // apart; otherwise every key's place is looked up (by lane key % 16, handed round).
  // The page numbers are fetched a step ahead.
  const bool page16 = p.page_size % 16 == 0;
  const int kc = lane % CH, khi = lane / CH;
  const uint32_t swz = (uint32_t)(khi * (D * 2) + ((kc ^ khi) << 4));
  auto fetch_page = [&](const PagedPos<PAT_TK, WIN>& x) {
    const int key = x.key(p) + warp * 16 + (page16 ? 0 : lane & 15);
    return WIN ? paged_page(p, x, key, page16 ? 16 : 1) : key < x.n ? p.page_table[x.b * p.ld_table + p.page_div(key)] : -1;
  };
  int page = fetch_page(ld);
  uint32_t load_slot = ring;
  auto load = [&]() {
    if (ld.w < end) {
      const uint32_t dst = load_slot + swz;
      const int key0 = ld.key(p) + warp * 16;
      if (key0 < ld.n) {
        const bool fine = page >= 0 && page < p.num_pages;
        const int from = WIN ? paged_first(p, ld.n) : 0;      // keys from the sinks' end on that no row sees
        if (page16) {
          if (!fine && p.err && !(WIN && page == PAGED_UNSEEN)) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
          const int in = key0 - p.page_div(key0) * p.page_size;
          const long long off = fine ? page * p.ld_page + ld.g * p.ld_head + (in + khi) * p.ld_tok + kc * 8 : 0;
          const char* k = reinterpret_cast<const char*>(p.k_cache) + off * 2;
          const char* v = reinterpret_cast<const char*>(p.v_cache) + off * 2;
          const long long step = fine ? KPI * p.ld_tok * 2 : 0;
          const int left = fine ? ld.n - key0 - khi : 0;      // > i KPI where the key exists
#pragma unroll
          for (int i = 0; i < 16 / KPI; ++i) {
            const uint32_t s = (dst ^ ((i * KPI & 7) << 4)) + i * KPI * (D * 2);
            const int key = key0 + khi + i * KPI;
            const bool ok = left > i * KPI && !(WIN && key >= p.sinks && key < from);
            pat_cp16(s, ok ? k : reinterpret_cast<const char*>(p.k_cache), ok);
            pat_cp16(s + S::MAT, ok ? v : reinterpret_cast<const char*>(p.v_cache), ok);
            k += step;
            v += step;
          }
        } else {
          const int key = key0 + (lane & 15);
          long long off = -1;
          if (key < ld.n) {
            if (fine)
              off = page * p.ld_page + ld.g * p.ld_head +
                    (key - p.page_div(key) * p.page_size) * p.ld_tok;
            else if (p.err && !(WIN && page == PAGED_UNSEEN))
              atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
          }
#pragma unroll
          for (int i = 0; i < 16 / KPI; ++i) {
            const long long o = __shfl_sync(0xffffffffu, off, i * KPI + khi);
            const uint32_t s = (dst ^ ((i * KPI & 7) << 4)) + i * KPI * (D * 2);
            const long long e = o < 0 ? 0 : o + kc * 8;
            pat_cp16(s, reinterpret_cast<const uint16_t*>(p.k_cache) + e, o >= 0);
            pat_cp16(s + S::MAT, reinterpret_cast<const uint16_t*>(p.v_cache) + e, o >= 0);
          }
        }
      }
      load_slot += 2 * S::MAT;
      if (load_slot == ring + S::STAGES * 2 * S::MAT) load_slot = ring;
      ld.next(p);
      if (ld.w < end) page = fetch_page(ld);
    }
    pat_commit();
  };

  // ---- queries of a row tile, as the first product's fragments
  uint32_t qnext[QW];
  auto fetch_queries = [&](int b, int g, int rt) {
    const uint16_t* qb = reinterpret_cast<const uint16_t*>(p.q);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = rt * NR + nt * 8 + (lane >> 2);
      const bool in = r < p.rows && b < p.B;
      const uint16_t* src = qb + (in ? paged_row(p, b, g, r) * D : 0) + 2 * (lane & 3);
#pragma unroll
      for (int k = 0; k < MT * 2; ++k)
        qnext[k * NT + nt] = in ? __ldg(reinterpret_cast<const uint32_t*>(src + k * 8)) ^ p.q_sign : 0u;
    }
  };
  fetch_queries(at.b, at.g, at.rt);
#pragma unroll
  for (int s = 0; s < S::STAGES - 1; ++s) load();

  // What a lane reads of a swizzled tile (rows of D * 2 bytes on multiples of that):
  // chunk c of row r at r * D * 2 + ((c ^ r % 8) << 4), so that stepping by two chunks
  // is an exclusive or with multiples of 32.
  const uint32_t k_lane = (lane & 15) * (D * 2) + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_lane = ((lane & 7) + (lane >> 4) * 8) * (D * 2) + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);

  float o[MT][NT][4], m[NT][2], l[NT][2];
  uint32_t bq[QW];
  int first_unit = at.unit;
  uint32_t slot_at = ring;
  for (bool start = true; at.w < end; start = false) {
    if (start || at.unit == 0) {
      // a new sequence, head or row tile: its queries, and empty sums
      first_unit = at.unit;
#pragma unroll
      for (int k = 0; k < QW; ++k) bq[k] = qnext[k];
      if (at.w + at.nu - at.unit + at.END < end) {
        int b = at.b, g = at.g, rt = at.rt;
        PagedPos<PAT_TK, WIN>::next_rows(p, b, g, rt);
        fetch_queries(b, g, rt);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[mt][nt][e] = 0.0f;
      }
    }
    load();
    pat_wait<S::STAGES - 1>();
    __syncwarp();
    const uint32_t ks_base = slot_at, vs_base = ks_base + S::MAT;
    slot_at += 2 * S::MAT;
    if (slot_at == ring + S::STAGES * 2 * S::MAT) slot_at = ring;
    const int key0 = at.key(p) + warp * 16;
    if (key0 < at.n) {
      // S^T = K Q^T
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < MT; ++ks) {
        uint32_t a[4];
        pat_ldsm((ks_base + k_lane) ^ (ks << 5), a);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) pat_mma<BF>(s[nt], a, bq[2 * ks * NT + nt], bq[(2 * ks + 1) * NT + nt]);
      }
      const int r0 = at.rt * NR;
      // some key of the sixteen may be hidden from some row
      const bool edge = key0 + 16 > at.n - p.L || (WIN && paged_out(p, at.n, key0, 16));
      if (edge) {
        uint32_t see = 0;
#pragma unroll
        for (int x = 0; x < NT * 4; ++x)
          see |= (uint32_t)paged_visible<WIN>(p, at.b, at.n, key0 + (lane >> 2) + (x & 2) * 4,
                                         r0 + (x >> 2) * 8 + 2 * (lane & 3) + (x & 1)) << x;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(see >> (nt * 4 + e) & 1)) s[nt][e] = -INFINITY;
      }
      // m: the running maximum of the unscaled scores (the scale is positive)
      bool up = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) up |= fmaxf(s[nt][e], s[nt][e + 2]) > m[nt][e];
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(s[nt][e], s[nt][e + 2]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            x = fmaxf(x, m[nt][e]);
            const float f = x == -INFINITY ? 1.0f : pat_exp2(m[nt][e] * p.scale_log2 - x * p.scale_log2);
            m[nt][e] = x;
            l[nt][e] *= f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) o[mt][nt][e] *= f, o[mt][nt][e + 2] *= f;
          }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float ms = m[nt][e] == -INFINITY ? 0.0f : m[nt][e] * p.scale_log2;
          s[nt][e] = pat_exp2(fmaf(s[nt][e], p.scale_log2, -ms));
          s[nt][e + 2] = pat_exp2(fmaf(s[nt][e + 2], p.scale_log2, -ms));
          l[nt][e] += s[nt][e] + s[nt][e + 2];
        }
        pb[nt][0] = pat_transpose(pat_pack<BF>(s[nt][0], s[nt][1]));
        pb[nt][1] = pat_transpose(pat_pack<BF>(s[nt][2], s[nt][3]));
      }
      // O^T += V^T P^T
      bool odd = false;
      if (edge && (p.L > 1 || p.tail)) {   // a value that is not finite, of a key that some row does not see?
        for (int x = lane; x < 16 * CH; x += 32) {
          uint32_t w[4];
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(vs_base + x * 16) : "memory");
          constexpr uint32_t EXP = BF ? 0x7f80u : 0x7c00u;
#pragma unroll
          for (int k = 0; k < 4; ++k) odd |= (w[k] & EXP) == EXP || ((w[k] >> 16) & EXP) == EXP;
        }
        odd = __any_sync(0xffffffffu, odd);
      }
      if (!odd) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t a[4];
          pat_ldsm_t((vs_base + v_lane) ^ (mt << 5), a);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) pat_mma<BF>(o[mt][nt], a, pb[nt][0], pb[nt][1]);
        }
      } else {
        // row by row, the keys hidden from it zeroed
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          for (int r = 0; r < 8; ++r) {
            uint32_t keep[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = key0 + 2 * (lane & 3) + e * 8, row = r0 + nt * 8 + r;
              keep[e] = (paged_visible<WIN>(p, at.b, at.n, j, row) ? 0xffffu : 0u) |
                        (paged_visible<WIN>(p, at.b, at.n, j + 1, row) ? 0xffff0000u : 0u);
            }
            const bool mine = (r >> 1) == (lane & 3);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              uint32_t a[4];
              pat_ldsm_t((vs_base + v_lane) ^ (mt << 5), a);
              a[0] &= keep[0], a[1] &= keep[0], a[2] &= keep[1], a[3] &= keep[1];
              float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              pat_mma<BF>(d, a, pb[nt][0], pb[nt][1]);
              if (mine && (r & 1)) o[mt][nt][1] += d[1], o[mt][nt][3] += d[3];
              if (mine && !(r & 1)) o[mt][nt][0] += d[0], o[mt][nt][2] += d[2];
            }
          }
      }
    }
    __syncwarp();
    const bool ends = at.unit + 1 == at.nu;
    if (ends || at.w + 1 >= end) {
      // join the warps; a whole sequence is written, a part goes to the workspace
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) m[nt][e] *= p.scale_log2;
      paged_finish<D, NT, BF>(p, at, ends && first_unit == 0, first_unit == 0 ? 1 : 0, o, m, l, obuf, sm_m, sm_l,
                                         s_range, s_cut, s_join);
    }
    at.next(p);
  }
  pat_wait<0>();
  paged_leave<D, NT, BF>(p, s_cut, s_join, pat_smem, S::RING + S::OBUF);
}

}  // namespace simsd
