// Attention of a few query tokens per sequence over a paged key-value cache.
//   o[b, t, h, :] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max),
// over the visible keys j < n = min(seq_lens[b], max_pages page_size) of KV head
// g = h / G (G = Hq / Hk).  The newest L keys belong to the L query tokens: with jt
// = j - (n - L), a key with jt < 0 is visible to all of them, the others where
// jt <= t, or where tail_mask[b, t, jt] is set.  No visible key: o = 0, lse = -inf.
//
// What bounds it: every key and value is read once for the G L rows that share it
// (4 G L operations per 2-byte element), so up to some 64 rows HBM bounds it and
// the work is to keep loads in flight on every SM and to cut any mix of lengths
// evenly.
//
// Split.  A unit is 64 keys of one (sequence, KV head, row tile); the units of the
// whole call, in that order, are cut into equal contiguous ranges, one per CTA, two
// CTAs per SM, from the lengths on the device (no host knowledge of them, so a
// graph replays as sequences grow).  A range may hold many short sequences or a
// slice of a long one; a sequence cut between CTAs leaves each part's (O, max,
// sum) in the workspace, and paged_combine_kernel joins the parts in key order.
//
// In a CTA each of the 4 warps takes 16 keys of every unit through a ring of its
// own (cp.async, no barrier between warps until the sequence ends), loading ahead
// across sequence ends.  Products with the roles swapped, so that few rows waste
// little: S^T = K Q^T (m16n8k16: 16 keys x 8 rows), P^T turned into the second
// product's operand with movmatrix, O^T = V^T P^T (16 dims x 8 rows).  Softmax in
// fp32 with exp2 of log2-scaled scores; the running maximum moves (and O is
// rescaled) only when a score exceeds it.  P is rounded to the 16-bit type for the
// second product: the weights are <= 1 and their sum, kept in fp32, is of the
// unrounded ones, so the rounding errs by at most half a step per weight.
//
// Masked keys: keys past n are zero-filled in shared memory, whatever stale memory
// holds.  A tail key that some rows of the unit see and others do not takes part
// with weight 0 in the second product; where its value is not finite (0 x inf), the
// unit's product runs row by row with the hidden keys zeroed instead.
#pragma once
#include "sm100.cuh"

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
  float4* part_o;           // [2 grid][D / 16][NT][32] fragments
  float* part_ml;           // [2 grid][NR][2] (max in log2 units, sum)
  int4* desc;               // [grid]: the cut sequence that starts in this CTA (b, head and row tile, last CTA or -1)
  long long ld_page, ld_head, ld_tok, ld_table, ldm_b, ldm_t;
  int B, L, Hq, Hk, G, num_pages, page_size, max_pages, rows, row_tiles;
  float scale_log2;         // scale * log2(e)
};

constexpr int PAT_WARPS = 4, PAT_THREADS = PAT_WARPS * 32, PAT_TK = 16 * PAT_WARPS;
constexpr int PAT_CTAS_PER_SM = 2;
constexpr int PAC_THREADS = 256;

template <int D, int NT>
struct PatSmem {
  static constexpr int STAGES = NT <= 2 ? 3 : 2;
  static constexpr int MAT = 16 * D * 2;                       // 16 keys (or values)
  static constexpr int RING = PAT_WARPS * STAGES * 2 * MAT;
  static constexpr int OBUF = PAT_WARPS * (D / 16) * 32 * 16;  // one 8-row tile of every warp's O
  static constexpr int Q = NT > 2 ? NT * 8 * D * 2 : 0;
  static constexpr int ML = 2 * PAT_WARPS * NT * 8 * 4;
  static constexpr int BYTES = RING + OBUF + Q + ML + 64;
};

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
  return (uint32_t)f32_to_16bit(lo, BF ? 0 : 1) | ((uint32_t)f32_to_16bit(hi, BF ? 0 : 1) << 16);
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
__device__ __forceinline__ int paged_units(int n) { return n <= PAT_TK ? 1 : (n + PAT_TK - 1) / PAT_TK; }

// Position in the unit order: sequence b (length n, nu units per head and row
// tile), hr = KV head * row_tiles + row tile, unit of it.
struct PagedPos {
  int b, hr, unit, n, nu;
  __device__ __forceinline__ void next(const PagedAttnArgs& p) {
    if (++unit < nu) return;
    unit = 0;
    if (++hr < p.Hk * p.row_tiles) return;
    hr = 0;
    if (++b >= p.B) return;
    n = paged_len(p, b);
    nu = paged_units(n);
  }
};

// Whether row r of the sequence's rows (t = r / G) sees key j < n
__device__ __forceinline__ bool paged_visible(const PagedAttnArgs& p, int b, int n, int j, int r) {
  if (j >= n) return false;
  const int jt = j - (n - p.L);
  if (jt < 0 || r >= p.rows) return true;
  const int t = r / p.G;
  return p.tail ? p.tail[b * p.ldm_b + t * p.ldm_t + jt] != 0 : jt <= t;
}

// The rows of one 8-row tile from a fragment of O^T (dims d, d + 8 of rows r, r + 1)
template <bool BF, int D>
__device__ __forceinline__ void paged_store(const PagedAttnArgs& p, int b, int hr, int nt8, int mt, int lane, float4 v) {
  const int g = hr / p.row_tiles;
  const int r = nt8 + 2 * (lane & 3), d = mt * 16 + (lane >> 2);
  uint16_t* o = reinterpret_cast<uint16_t*>(p.o);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (r + e >= p.rows) continue;
    const int t = (r + e) / p.G, h = g * p.G + (r + e) - t * p.G;
    uint16_t* dst = o + (((long long)b * p.L + t) * p.Hq + h) * D + d;
    dst[0] = f32_to_16bit(e ? v.y : v.x, BF ? 0 : 1);
    dst[8] = f32_to_16bit(e ? v.w : v.z, BF ? 0 : 1);
  }
}
__device__ __forceinline__ void paged_store_lse(const PagedAttnArgs& p, int b, int hr, int r, float m, float l) {
  if (p.lse == nullptr || r >= p.rows) return;
  const int t = r / p.G, h = hr / p.row_tiles * p.G + r - t * p.G;
  p.lse[((long long)b * p.L + t) * p.Hq + h] = l == 0.0f ? -INFINITY : fmaf(0.69314718055994531f, m, logf(l));
}

// The CTA's range [w0, w1) of the call's units and the position of w0, for the
// `ctas` CTAs that take part.  False: this CTA has none.
__device__ __forceinline__ bool paged_range(const PagedAttnArgs& p, long long& total, long long& w0, long long& w1,
                                            int& ctas, PagedPos& pos) {
  __shared__ long long s_sum[PAT_WARPS];
  __shared__ long long s_total;
  __shared__ long long s_first;
  __shared__ int s_b;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = p.Hk * p.row_tiles;
  long long sum = 0;
  for (int b = tid; b < p.B; b += PAT_THREADS) {
    sum += (long long)paged_units(paged_len(p, b)) * per;
    if (blockIdx.x == 0 && p.err && p.seq_lens[b] > (long long)p.max_pages * p.page_size)
      atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < PAT_WARPS; ++w) total += s_sum[w];
  ctas = (int)min((long long)gridDim.x, total);
  const int c = blockIdx.x;
  if (c >= ctas) return false;
  w0 = total * c / ctas;
  w1 = total * (c + 1) / ctas;
  // the sequence that holds w0
  long long before = 0;
  for (int base = 0; base < p.B; base += PAT_THREADS) {
    const int b = base + tid;
    long long u = b < p.B ? (long long)paged_units(paged_len(p, b)) * per : 0;
    long long incl = u;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, m);
      if (lane >= m) incl += v;
    }
    __syncthreads();
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    long long off = before;
    for (int w = 0; w < warp; ++w) off += s_sum[w];
    if (off + incl - u <= w0 && w0 < off + incl) s_b = b, s_first = off + incl - u;
    if (tid == PAT_THREADS - 1) s_total = off + incl;
    __syncthreads();
    before = s_total;
    if (before > w0) break;
  }
  pos.b = s_b;
  pos.n = paged_len(p, pos.b);
  pos.nu = paged_units(pos.n);
  const long long rem = w0 - s_first;
  pos.hr = (int)(rem / pos.nu);
  pos.unit = (int)(rem - (long long)pos.hr * pos.nu);
  return true;
}

template <int D, int NT, bool BF>
__global__ void __launch_bounds__(PAT_THREADS, PAT_CTAS_PER_SM) paged_attention_kernel(const PagedAttnArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  using S = PatSmem<D, NT>;
  constexpr int MT = D / 16, NR = NT * 8, CH = D / 8;     // 16-byte chunks of a key
  constexpr int KPI = 32 / CH;                            // keys per cp.async of the warp
  constexpr bool QREG = NT <= 2;
  extern __shared__ __align__(128) uint8_t pat_smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ring = smem_u32(pat_smem) + warp * S::STAGES * 2 * S::MAT;
  float4* obuf = reinterpret_cast<float4*>(pat_smem + S::RING);
  uint8_t* qs = pat_smem + S::RING + S::OBUF;
  float* sm_m = reinterpret_cast<float*>(pat_smem + S::RING + S::OBUF + S::Q);
  float* sm_l = sm_m + PAT_WARPS * NR;

  long long total, w0, w1;
  int ctas;
  PagedPos ld;
  if (!paged_range(p, total, w0, w1, ctas, ld)) {
    if (tid == 0) p.desc[blockIdx.x] = make_int4(0, 0, -1, 0);
    return;
  }
  if (tid == 0) p.desc[blockIdx.x] = make_int4(0, 0, -1, 0);
  PagedPos at = ld;
  const int steps = (int)(w1 - w0);

  // the page of the key that this lane (< 16) places next, fetched a step ahead
  auto fetch_page = [&](const PagedPos& x) {
    const int key = x.unit * PAT_TK + warp * 16 + (lane & 15);
    return key < x.n ? p.page_table[x.b * p.ld_table + key / p.page_size] : -1;
  };
  int page = fetch_page(ld);
  int loaded = 0;
  auto load = [&]() {
    if (loaded < steps) {
      const uint32_t dst = ring + (loaded % S::STAGES) * 2 * S::MAT;
      const int key = ld.unit * PAT_TK + warp * 16 + (lane & 15);
      long long off = -1;
      if (key < ld.n) {
        if (page >= 0 && page < p.num_pages)
          off = page * p.ld_page + (ld.hr / p.row_tiles) * p.ld_head + (key % p.page_size) * p.ld_tok;
        else if (p.err)
          atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
      }
      const int c = lane % CH;
#pragma unroll
      for (int i = 0; i < 16 / KPI; ++i) {
        const int r = i * KPI + lane / CH;
        const long long o = __shfl_sync(0xffffffffu, off, r);
        const uint32_t s = dst + r * (D * 2) + ((c ^ (r & 7)) << 4);
        const long long e = o < 0 ? 0 : o + c * 8;
        pat_cp16(s, reinterpret_cast<const uint16_t*>(p.k_cache) + e, o >= 0);
        pat_cp16(s + S::MAT, reinterpret_cast<const uint16_t*>(p.v_cache) + e, o >= 0);
      }
      ++loaded;
      if (loaded < steps) {
        ld.next(p);
        page = fetch_page(ld);
      }
    }
    pat_commit();
  };
#pragma unroll
  for (int s = 0; s < S::STAGES - 1; ++s) load();

  float o[MT][NT][4], m[NT][2], l[NT][2];
  uint32_t bq[QREG ? MT : 1][QREG ? NT : 1][2];
  int first_unit = at.unit;
  for (int i = 0; i < steps; ++i) {
    if (i == 0 || at.unit == 0) {
      // a new sequence, head or row tile: its queries, and empty sums
      first_unit = at.unit;
      const int g = at.hr / p.row_tiles, r0 = (at.hr - g * p.row_tiles) * NR;
      const uint16_t* qb = reinterpret_cast<const uint16_t*>(p.q);
      if constexpr (QREG) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int r = r0 + nt * 8 + (lane >> 2);
          const int t = r / p.G, h = g * p.G + r - t * p.G;
          const uint16_t* src = qb + (((long long)at.b * p.L + t) * p.Hq + h) * D + 2 * (lane & 3);
#pragma unroll
          for (int ks = 0; ks < MT; ++ks)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              bq[ks][nt][e] = r < p.rows ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + e * 8) : 0u;
        }
      } else {
        for (int x = tid; x < NR * CH; x += PAT_THREADS) {
          const int rr = x / CH, c = x % CH, r = r0 + rr;
          const int t = r / p.G, h = g * p.G + r - t * p.G;
          const uint4 v = r < p.rows ? *reinterpret_cast<const uint4*>(
                                           qb + (((long long)at.b * p.L + t) * p.Hq + h) * D + c * 8)
                                     : make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(qs + rr * (D * 2) + ((c ^ (rr & 7)) << 4)) = v;
        }
        __syncthreads();
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
    const uint32_t ks_base = ring + (i % S::STAGES) * 2 * S::MAT, vs_base = ks_base + S::MAT;
    const int key0 = at.unit * PAT_TK + warp * 16;
    if (key0 < at.n) {
      // S^T = K Q^T
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
      const int kr = lane & 15;
#pragma unroll
      for (int ks = 0; ks < MT; ++ks) {
        uint32_t a[4];
        pat_ldsm(ks_base + kr * (D * 2) + (((ks * 2 + (lane >> 4)) ^ (kr & 7)) << 4), a);
        if constexpr (QREG) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) pat_mma<BF>(s[nt], a, bq[ks][nt][0], bq[ks][nt][1]);
        } else {
#pragma unroll
          for (int nt = 0; nt < NT; nt += 2) {
            // rows nt * 8 .. + 15, both 8-element halves of this k step
            const int rr = nt * 8 + (lane >> 4) * 8 + (lane & 7);
            uint32_t b[4];
            pat_ldsm(smem_u32(qs) + rr * (D * 2) + (((ks * 2 + ((lane >> 3) & 1)) ^ (rr & 7)) << 4), b);
            pat_mma<BF>(s[nt], a, b[0], b[1]);
            pat_mma<BF>(s[nt + 1], a, b[2], b[3]);
          }
        }
      }
      const int g = at.hr / p.row_tiles, r0 = (at.hr - g * p.row_tiles) * NR;
      const bool edge = key0 + 16 > at.n - p.L;          // some key of the sixteen may be hidden from some row
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt][e] *= p.scale_log2;
          if (edge && !paged_visible(p, at.b, at.n, key0 + (lane >> 2) + (e >> 1) * 8,
                                     r0 + nt * 8 + 2 * (lane & 3) + (e & 1)))
            s[nt][e] = -INFINITY;
        }
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
            const float f = x == -INFINITY ? 1.0f : exp2f(m[nt][e] - x);
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
        for (int e = 0; e < 4; ++e) {
          const float mm = m[nt][e & 1];
          s[nt][e] = exp2f(s[nt][e] - (mm == -INFINITY ? 0.0f : mm));
        }
        l[nt][0] += s[nt][0] + s[nt][2];
        l[nt][1] += s[nt][1] + s[nt][3];
        pb[nt][0] = pat_transpose(pat_pack<BF>(s[nt][0], s[nt][1]));
        pb[nt][1] = pat_transpose(pat_pack<BF>(s[nt][2], s[nt][3]));
      }
      // O^T += V^T P^T
      const int vr = (lane & 7) + (lane >> 4) * 8, vc = (lane >> 3) & 1;
      bool odd = false;
      if (edge) {   // a value that is not finite, of a key that some row may not see?
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
          pat_ldsm_t(vs_base + vr * (D * 2) + (((mt * 2 + vc) ^ (vr & 7)) << 4), a);
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
              keep[e] = (paged_visible(p, at.b, at.n, j, row) ? 0xffffu : 0u) |
                        (paged_visible(p, at.b, at.n, j + 1, row) ? 0xffff0000u : 0u);
            }
            const bool mine = (r >> 1) == (lane & 3);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              uint32_t a[4];
              pat_ldsm_t(vs_base + vr * (D * 2) + (((mt * 2 + vc) ^ (vr & 7)) << 4), a);
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
    if (ends || i + 1 == steps) {
      // join the four warps; a whole sequence is written, a part goes to the workspace
      const bool whole = ends && first_unit == 0;
      const int slot = 2 * blockIdx.x + (first_unit == 0 ? 1 : 0);
      if (first_unit == 0 && !ends && tid == 0) {
        const long long last = w0 + i - at.unit + at.nu;    // one past the sequence's last unit
        p.desc[blockIdx.x] = make_int4(at.b, at.hr, (int)((last * ctas - 1) / total), 0);
      }
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
      __syncthreads();
      const int r0 = at.hr % p.row_tiles * NR;
      for (int r = tid; r < NR; r += PAT_THREADS) {
        float mm = -INFINITY, ll = 0.0f;
        for (int w = 0; w < PAT_WARPS; ++w) mm = fmaxf(mm, sm_m[w * NR + r]);
        for (int w = 0; w < PAT_WARPS; ++w) ll += sm_l[w * NR + r] * exp2f(sm_m[w * NR + r] - (mm == -INFINITY ? 0.0f : mm));
        if (whole) {
          paged_store_lse(p, at.b, at.hr, r0 + r, mm, ll);
        } else {
          p.part_ml[((long long)slot * NR + r) * 2] = mm;
          p.part_ml[((long long)slot * NR + r) * 2 + 1] = ll;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2], inv[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + 2 * (lane & 3) + e;
          float mm = -INFINITY, ll = 0.0f;
          for (int w = 0; w < PAT_WARPS; ++w) mm = fmaxf(mm, sm_m[w * NR + r]);
          if (mm == -INFINITY) mm = 0.0f;
          for (int w = 0; w < PAT_WARPS; ++w) ll += sm_l[w * NR + r] * exp2f(sm_m[w * NR + r] - mm);
          f[e] = exp2f(m[nt][e] - mm);
          inv[e] = !whole ? 1.0f : ll == 0.0f ? 0.0f : 1.0f / ll;
        }
        if (nt > 0) __syncthreads();
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          obuf[(warp * MT + mt) * 32 + lane] =
              make_float4(o[mt][nt][0] * f[0], o[mt][nt][1] * f[1], o[mt][nt][2] * f[0], o[mt][nt][3] * f[1]);
        __syncthreads();
#pragma unroll
        for (int mt = warp; mt < MT; mt += PAT_WARPS) {
          float4 a = obuf[mt * 32 + lane];
#pragma unroll
          for (int w = 1; w < PAT_WARPS; ++w) {
            const float4 x = obuf[(w * MT + mt) * 32 + lane];
            a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
          }
          a.x *= inv[0], a.y *= inv[1], a.z *= inv[0], a.w *= inv[1];
          if (whole)
            paged_store<BF, D>(p, at.b, at.hr, r0 + nt * 8, mt, lane, a);
          else
            p.part_o[(((long long)slot * MT + mt) * NT + nt) * 32 + lane] = a;
        }
      }
      __syncthreads();
    }
    at.next(p);
  }
}

// One CTA per CTA of paged_attention_kernel: joins the parts of the sequence (one
// KV head and row tile of it) that starts there and goes on in later CTAs.
template <int D, int NT, bool BF>
__global__ void __launch_bounds__(PAC_THREADS) paged_combine_kernel(const PagedAttnArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int MT = D / 16, NR = NT * 8;
  extern __shared__ float pac_w[];                 // [parts][NR]
  const int c = blockIdx.x;
  const int4 d = p.desc[c];
  if (d.z < 0) return;
  const int parts = d.z - c + 1, tid = threadIdx.x, lane = tid & 31;
  const int r0 = d.y % p.row_tiles * NR;
  auto slot = [&](int i) { return (long long)(i == 0 ? 2 * c + 1 : 2 * (c + i)); };
  for (int r = tid >> 5; r < NR; r += PAC_THREADS / 32) {
    float mm = -INFINITY, ll = 0.0f;
    for (int i = lane; i < parts; i += 32) mm = fmaxf(mm, p.part_ml[(slot(i) * NR + r) * 2]);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, k));
    const float mu = mm == -INFINITY ? 0.0f : mm;
    for (int i = lane; i < parts; i += 32) {
      const float2 x = *reinterpret_cast<const float2*>(p.part_ml + (slot(i) * NR + r) * 2);
      const float f = exp2f(x.x - mu);
      pac_w[i * NR + r] = f;
      ll += x.y * f;
    }
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, k);
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
    __syncwarp();
    for (int i = lane; i < parts; i += 32) pac_w[i * NR + r] *= inv;
    if (lane == 0) paged_store_lse(p, d.x, d.y, r0 + r, mm, ll);
  }
  __syncthreads();
  for (int x = tid; x < MT * NT * 32; x += PAC_THREADS) {
    const int mt = x / (NT * 32), nt = x / 32 % NT;
    const int r = nt * 8 + 2 * (lane & 3);
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int i = 0; i < parts; ++i) {
      const float4 v = p.part_o[slot(i) * (MT * NT * 32) + x];
      const float f0 = pac_w[i * NR + r], f1 = pac_w[i * NR + r + 1];
      a.x = fmaf(v.x, f0, a.x), a.y = fmaf(v.y, f1, a.y), a.z = fmaf(v.z, f0, a.z), a.w = fmaf(v.w, f1, a.w);
    }
    paged_store<BF, D>(p, d.x, d.y, r0 + nt * 8, mt, lane, a);
  }
}

}  // namespace simsd
