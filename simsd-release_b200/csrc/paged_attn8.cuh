// Attention of a few query tokens per sequence over a paged cache held in 8 bits (e4m3,
// a scale for each block of tokens and head; paged8.cuh):
//   k_j = ks_j K_j, v_j = vs_j V_j, K, V the stored numbers
//   o = sum_j p_j vs_j V_j / sum_j p_j,  p_j = exp2(x_j - m),  x_j = scale log2(e) ks_j (q . K_j)
// with the operator's masks, cut, parts and workspace of paged_attn.cuh, of which this is
// the 8-bit form.
//
// Arithmetic.  K and V go to fp16 in registers, exactly.  The queries are put in fp16 with
// a power of two for each row, its largest element in [2^14, 2^15): bf16 ones exactly,
// down to 2^-38 of it, half the smallest fp16 number.  The block's value scale goes into the
// weight, w_j = p_j vs_j, rounded to fp16 for the second product (2^-12 of it).  m is
// chosen so that the largest w is some 2^8 when it moves, and moves again when one would
// pass 2^15: hardly ever, and a weight keeps its 11 bits down to 2^-22 of the largest.
// It follows x_j + lv_j, lv_j = log2 vs_j (-64 at least; only the choice of m goes by it), so
// scales of very different sizes meet in one sequence; p_j and its sum stay in fp32.
//
// A unit is 128 keys, of which four warps take 32 each; a fifth loads ahead into a ring of
// units: TMA where pages are a multiple of 8 tokens, a lane per run of tokens that lies in one
// page, else cp.async into the same swizzled layout; the scales by cp.async.  What the
// loads take of instructions is so spent once a unit: 16384 warps' units of 32 keys took 893
// instructions each with loads of their own by cp.async and 737 with TMA, and the SMs issue
// half the time at best.
//
// Measured (B200, 8 KV heads x 128, 4 query heads each, bf16, device time in a graph of calls): 2 x
// 120-128k tokens 90 us, 6.0 TB/s, 90 % of the bytes' time at the copy rate (101 with each warp loading for itself by
// cp.async); 32 x 0.3-4k 26 us, 53 %, of which the first units' lengths, pages and data take 5; 1 x
// 100 7.8.  16 x 8-16k tokens with pages of one token,
// by cp.async, take 112 us (floor 56).  16 x 8-32k in a window of 4096 and 4 first keys 35 us (floor 20.5).
// Up to 16 rows a KV head, 9 to 16 in two tiles that each read the keys (paged_plan8 has the figures); more in
// paged_attn8_tc.cuh.
//
// In an operand of the first product a lane's four bytes are four
// neighbouring dims of a key (the queries' dims are ordered alike).  For the second,
// ldmatrix.trans.b8 hands a lane four keys of a dim, of which two and two are neighbours in
// the product: rows 8 - 15 of S^T are therefore keys 12 - 15 and 8 - 11 (p8_key), and V's rows are
// addressed in the order that goes with that (p8_row), which keeps both reads free of bank
// conflicts.  A conversion is one instruction for two numbers, and no byte is moved besides.
//
// A hidden key counts as nothing, whatever its memory or scale holds: its weight is set to
// zero, keys that no row sees are not read, and where a value of a key that some row does
// not see is NaN, the product runs row by row without the keys hidden from it.
#pragma once
#include "paged8.cuh"
#include "paged_attn.cuh"

namespace simsd {

struct PagedAttn8Args {
  CUtensorMap k, v;         // [pages, Hk, page size, D], box {D, run tokens, 1, 1}; where run > 0
  PagedAttnArgs a;          // caches: e4m3, strides in bytes
  const float* k_scale;     // [pages, Hk, page_size / block]
  const float* v_scale;
  long long lds_page, lds_head, lds_block;
  PagedDiv block_div;       // by block
  int run;                  // tokens of a TMA load: the largest power of two <= 32 in the page size, or 0
};

// Positions in units of 128 keys; a sequence's end weighs as three of them in the cut: at 1, 2, 3, 4 and 6
// 32 x 0.3 - 4k tokens take 28.5, 27, 26.3, 27.4 and 29 us; 19 windowed rows of 5 take 28.3 at 2 and 29 at 3.
constexpr int P8_END = 3;
template <bool WIN>
using P8Pos = PagedPos<128, WIN, P8_END>;

template <int D>
struct Pat8Shape {
  static constexpr int NR = 8;
  static constexpr int TK = 32 * PAT_WARPS;                    // keys of a unit
  static constexpr int THREADS = PAT_THREADS + 32;             // with the loading warp
  static constexpr int CTAS = 3, STAGES = 2;                   // CTAs that an SM holds, units in a ring
  static constexpr int MAT = TK * D;                           // a unit's keys (or values)
  static constexpr int STAGE = 2 * MAT;
  static constexpr int SCALES = 2 * TK * 4;                    // a unit's scales of keys, then of values
  static constexpr int RING = STAGES * STAGE;
  static constexpr int ML = 2 * PAT_WARPS * NR * 4;
  static constexpr int BYTES = 1024 + RING + STAGES * SCALES + ML + 2 * STAGES * 8;
  static_assert(MAT >= PatShape<D, 1>::OBUF);                  // a stage has room for every warp's O
};

// 4 bytes into shared memory, zeros where !ok
__device__ __forceinline__ void pat8_cp4(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
// e with the row's largest |q| / 2^e in [2^14, 2^15)
__device__ __forceinline__ int p8_query_exponent(float top) {
  return max(-100, min(127, (__float_as_int(top) >> 23) - 127)) - 14;
}
__device__ __forceinline__ float p8_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pat8_lds(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
// 16-byte chunk c of row r of a tile with rows of D bytes: the chunks that eight
// neighbouring rows have at one place lie in different banks
template <int D>
__device__ __forceinline__ uint32_t pat8_off(int r, int c) {
  return D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ (r >> 1 & 3)) << 4);
}

// The key in row r of a 16-key tile of S^T, and the key whose values are row r of the
// matrix that is read transposed (four neighbours r: rows 2 c, 2 c + 1, 8 + 2 c, 9 + 2 c of P^T).
__device__ __forceinline__ int p8_key(int r) { return r < 8 ? r : r ^ 4; }
__device__ __forceinline__ int p8_row(int r) { return p8_key((r >> 1 & 1) * 8 + (r >> 2) * 2 + (r & 1)); }
// 16 dims x 32 keys from two 16-key tiles: words 2 kt, 2 kt + 1 are dims i8, i8 + 8, four keys each
__device__ __forceinline__ void p8_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void p8_tma(uint32_t dst, const void* map, uint32_t bar, int tok, int head, int page, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(0), "r"(tok), "r"(head), "r"(page), "l"(policy)
      : "memory");
}

// Counts the thread's cp.async so far in at `bar` once they have landed.
__device__ __forceinline__ void p8_cp_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// The loading warp: units from `ld` up to `end` into the ring.  The page numbers are fetched a
// unit ahead.  TMA: a lane per run; one without a key that is read loads zeros, from past the
// last page.  Else the lane's keys are lane, 32 + lane, ...: their places are handed round.
template <int D, bool WIN, bool TMA>
__device__ __forceinline__ void p8_load(const PagedAttn8Args& args, P8Pos<WIN> ld, int end, uint32_t ring, uint32_t scales,
                                        uint32_t full, uint32_t empty, volatile int* abort_flag) {
  using S = Pat8Shape<D>;
  constexpr int TK = S::TK;
  using Pos = P8Pos<WIN>;
  constexpr int CH = D / 16, KPI = 32 / CH, EACH = TK / 32;      // chunks of a key, keys of a copy, keys of a lane
  const PagedAttnArgs& p = args.a;
  const int lane = threadIdx.x & 31, kc = lane % CH, khi = lane / CH;
  const int run = TMA ? args.run : 1, runs = TK / run;               // TMA: up to 32 runs
  constexpr int PAGES = TMA ? 1 : EACH;
  const uint64_t policy = policy_evict_first();
  if (TMA && lane == 0) prefetch_tmap(&args.k), prefetch_tmap(&args.v);
  int page[PAGES];
  auto fetch_pages = [&](const Pos& x) {
#pragma unroll
    for (int i = 0; i < PAGES; ++i) {
      const int key = x.key(p) + (TMA ? lane * run : i * 32 + lane);
      page[i] = -1;
      if (!TMA || lane < runs)
        page[i] = WIN ? paged_page(p, x, key, run) : key < x.n ? p.page_table[x.b * p.ld_table + p.page_div(key)] : -1;
    }
  };
  fetch_pages(ld);
  int slot = 0;
  uint32_t phase = 0, filled = 0, parity = 0;                        // slots that have been loaded, and their phases
  bool ok = true;
  while (ld.w < end) {
    const int key0 = ld.key(p), n = ld.n, g = ld.g;
    int from[PAGES];
#pragma unroll
    for (int i = 0; i < PAGES; ++i) {
      const bool fine = page[i] >= 0 && page[i] < p.num_pages;
      const int key = key0 + (TMA ? lane * run : i * 32 + lane);
      if (!fine && key < n && (!TMA || lane < runs) && p.err && !(WIN && page[i] == PAGED_UNSEEN))
        atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
      from[i] = fine ? page[i] : -1;
    }
    ld.next(p);
    if (ld.w < end) fetch_pages(ld);
    ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * slot, phase ^ 1, abort_flag, p.err));
    if (!ok) break;
    const uint32_t bar = full + 8 * slot, dst = ring + slot * S::STAGE, sdst = scales + slot * S::SCALES;
    if constexpr (TMA) {
      if (lane == 0) mbar_arrive_expect_tx(bar, S::STAGE);
      __syncwarp();
      if (lane < runs) {
        const int first = key0 + lane * run, tok = first - p.page_div(first) * p.page_size, x = from[0] < 0 ? p.num_pages : from[0];
        p8_tma(dst + lane * run * D, &args.k, bar, tok, g, x, policy);
        p8_tma(dst + S::MAT + lane * run * D, &args.v, bar, tok, g, x, policy);
      }
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int at = i * 32 + lane, key = key0 + at, tok = key - p.page_div(key) * p.page_size;
      const int mine = TMA ? __shfl_sync(0xffffffffu, from[0], at / run) : from[TMA ? 0 : i];
      const bool real = mine >= 0 && key < n;
      const long long soff = real ? mine * args.lds_page + g * args.lds_head + args.block_div(tok) * args.lds_block : 0;
      pat8_cp4(sdst + at * 4, args.k_scale + soff, real);
      pat8_cp4(sdst + TK * 4 + at * 4, args.v_scale + soff, real);
      if constexpr (!TMA) {
        const long long off = real ? mine * p.ld_page + g * p.ld_head + tok * p.ld_tok : -1;
#pragma unroll
        for (int x = 0; x < 32 / KPI; ++x) {
          const long long o = __shfl_sync(0xffffffffu, off, x * KPI + khi);
          const long long e = o < 0 ? 0 : o + kc * 16;
          const uint32_t s = dst + pat8_off<D>(i * 32 + x * KPI + khi, kc);
          pat_cp16(s, reinterpret_cast<const uint8_t*>(p.k_cache) + e, o >= 0);
          pat_cp16(s + S::MAT, reinterpret_cast<const uint8_t*>(p.v_cache) + e, o >= 0);
        }
      }
    }
    if (!TMA && lane == 0) mbar_arrive(bar);
    p8_cp_arrive(bar);
    filled |= 1u << slot;
    parity = (parity & ~(1u << slot)) | phase << slot;
    if (++slot == S::STAGES) slot = 0, phase ^= 1;
  }
  // giving up: no copy may land after the CTA has left
  if (!ok) {
    pat_commit();
    pat_wait<0>();
    for (int s = 0; s < S::STAGES; ++s)
      if (filled >> s & 1) mbar_wait_drain(full + 8 * s, parity >> s & 1, 100000000ull);
  }
}

template <int D, bool BF, bool WIN, bool TMA>
__global__ void __launch_bounds__(Pat8Shape<D>::THREADS, Pat8Shape<D>::CTAS) paged_attention8_kernel(const __grid_constant__ PagedAttn8Args args) {
  griddep_launch_dependents();
  griddep_wait();
  const PagedAttnArgs& p = args.a;
  using S = Pat8Shape<D>;
  constexpr int NR = S::NR;
  constexpr int MT = D / 16, CH = D / 16;                 // 16-dim tiles, 16-byte chunks of a key
  using Pos = P8Pos<WIN>;
  extern __shared__ uint8_t pat8_raw[];
  __shared__ PagedPart s_cut[2];
  __shared__ bool s_join[2];
  __shared__ PagedCut s_range;
  __shared__ int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c4 = lane & 3, i8 = lane >> 2;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pat8_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t ring = smem_u32(smem), scales = ring + S::RING;
  float* sm_m = reinterpret_cast<float*>(smem + S::RING + S::STAGES * S::SCALES);
  float* sm_l = sm_m + PAT_WARPS * NR;
  const uint32_t full = scales + S::STAGES * S::SCALES + S::ML, empty = full + 8 * S::STAGES;
  if (tid == 0) {
    s_abort = 0;
#pragma unroll
    for (int s = 0; s < S::STAGES; ++s) mbar_init(full + 8 * s, 33), mbar_init(empty + 8 * s, PAT_WARPS);
    fence_mbar_init();
  }
  Pos at;
  int end;
  {
    PagedCut cut;
    if (!paged_range<S::THREADS, S::TK, WIN>(p, cut, at)) return;
    end = cut.first(blockIdx.x + 1);
    if (tid == 0) s_range = cut;
  }
  if (tid < 2) s_cut[tid].parts = 0, s_join[tid] = false;   // warp 0 alone reads and writes them before the next barrier
  if (warp == PAT_WARPS) {
    p8_load<D, WIN, TMA>(args, at, end, ring, scales, full, empty, &s_abort);
    return;
  }
  bool dead = false;                   // a wait has given up: nothing more is waited for

  // ---- queries of a row tile: the lane's row i8 of each 8, four dims of every 16.  They stay out
  // of registers until their sequence comes; its lines are sent for a sequence ahead.
  auto expect_queries = [&](int b, int g, int rt) {
    for (int x = tid; x < NR * D / 64; x += PAT_THREADS) {
      const int r = rt * NR + x / (D / 64);
      if (r < p.rows && b < p.B)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const uint16_t*>(p.q) + paged_row(p, b, g, r) * D + x % (D / 64) * 64));
    }
  };
  uint32_t bq[2 * MT];                 // as fp16, divided by the row's power of two
  uint64_t qs;                         // scale log2(e) times those of rows 2 c4, 2 c4 + 1
  auto take_queries = [&](int b, int g, int rt) {
    const int r = rt * NR + i8;
    const bool in = r < p.rows;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) + (in ? paged_row(p, b, g, r) * D : 0) + 4 * c4;
    uint2 q[MT];
#pragma unroll
    for (int k = 0; k < MT; ++k) q[k] = in ? __ldg(reinterpret_cast<const uint2*>(src + k * 16)) : make_uint2(0, 0);
    float unit = 1.0f;
    if constexpr (BF) {
      float top = 0.0f;
#pragma unroll
      for (int k = 0; k < MT; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t w = e ? q[k].y : q[k].x;
          top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u))));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int ex = p8_query_exponent(top);
      const float up = p8_power(-ex);
      unit = p8_power(ex);
#pragma unroll
      for (int k = 0; k < MT; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t w = e ? q[k].y : q[k].x;
          bq[2 * k + e] = pat_pack<false>(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
        }
    } else {
#pragma unroll
      for (int k = 0; k < MT; ++k) bq[2 * k] = q[k].x, bq[2 * k + 1] = q[k].y;
    }
    qs = f2_pack(__shfl_sync(0xffffffffu, unit, 8 * c4) * p.scale_log2, __shfl_sync(0xffffffffu, unit, 8 * c4 + 4) * p.scale_log2);
  };

  // What a lane reads of a tile: of the keys, the row of S^T lane % 16 in chunk lane / 16 of
  // two; of the values, row lane % 16 of tile lane / 16.  Chunks are stepped by exclusive or.
  const uint32_t k_lane = warp * 32 * D + pat8_off<D>(p8_key(lane & 15), lane >> 4);
  const uint32_t v_lane = warp * 32 * D + pat8_off<D>((lane & 16) + p8_row(lane & 15), 0);

  float o[MT][1][4], m[1][2], l[1][2];
  int first_unit = at.unit;
  int slot = 0;
  uint32_t phase = 0;
  for (bool start = true; at.w < end; start = false) {
    if (start || at.unit == 0) {
      // a new sequence, head or row tile: its queries, and empty sums
      first_unit = at.unit;
      take_queries(at.b, at.g, at.rt);
      if (at.w + at.nu - at.unit + at.END < end) {
        int b = at.b, g = at.g, rt = at.rt;
        Pos::next_rows(p, b, g, rt);
        expect_queries(b, g, rt);
      }
      m[0][0] = m[0][1] = -INFINITY;
      l[0][0] = l[0][1] = 0.0f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[mt][0][0] = o[mt][0][1] = o[mt][0][2] = o[mt][0][3] = 0.0f;
    }
    if (!dead && !mbar_wait(full + 8 * slot, phase, &s_abort, p.err)) dead = true;
    __syncwarp();
    const uint32_t ks_base = ring + slot * S::STAGE, vs_base = ks_base + S::MAT, sc_base = scales + slot * S::SCALES + warp * 128;
    const int key0 = at.key(p) + warp * 32;
    if (key0 < at.n) {
      // S^T = K Q^T, rows i8 and i8 + 8 of two tiles of 16 keys
      float s[2][4] = {};
#pragma unroll
      for (int k2 = 0; k2 < MT / 2; ++k2) {
        uint32_t r[2][4];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) pat_ldsm((ks_base + kt * 16 * D + k_lane) ^ (k2 << 5), r[kt]);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) {
            const uint32_t a[4] = {p8_half2(r[kt][2 * x] & 0xffffu), p8_half2(r[kt][2 * x + 1] & 0xffffu),
                                   p8_half2(r[kt][2 * x] >> 16), p8_half2(r[kt][2 * x + 1] >> 16)};
            pat_mma<false>(s[kt], a, bq[2 * (2 * k2 + x)], bq[2 * (2 * k2 + x) + 1]);
          }
      }
      float vs[2][2], lv[2][2];                            // of row i8 + 8 e of a tile
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t from = sc_base + (kt * 16 + p8_key(e * 8 + i8)) * 4;
          const float ks = pat8_lds(from);
          vs[kt][e] = pat8_lds(from + S::TK * 4);
          lv[kt][e] = fmaxf(p8_log2(vs[kt][e]), -64.0f);
          const float2 z = f2_unpack(f2_mul(f2_pack(s[kt][2 * e], s[kt][2 * e + 1]), f2_mul(f2_pack(ks, ks), qs)));
          s[kt][2 * e] = z.x, s[kt][2 * e + 1] = z.y;
        }
      const int r0 = at.rt * NR;
      // some key of the 32 may be hidden from some row
      const bool edge = key0 + 32 > at.n - p.L || (WIN && paged_out(p, at.n, key0, 32));
      uint32_t see = 0xffu;
      if (edge) {
        see = 0;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          see |= (uint32_t)paged_visible<WIN>(p, at.b, at.n, key0 + (x >> 2) * 16 + p8_key(i8 + (x & 2) * 4),
                                              r0 + 2 * c4 + (x & 1)) << x;
          if (!(see >> x & 1)) s[x >> 2][x & 3] = -INFINITY;
        }
      }
      // m moves where a weight would pass 2^15
      float top[2];
#pragma unroll
      for (int e = 0; e < 2; ++e)
        top[e] = fmaxf(fmaxf(s[0][e] + lv[0][0], s[0][e + 2] + lv[0][1]), fmaxf(s[1][e] + lv[1][0], s[1][e + 2] + lv[1][1]));
      if (__any_sync(0xffffffffu, top[0] > m[0][0] + 15.0f || top[1] > m[0][1] + 15.0f)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = top[e];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          x = fmaxf(x - 8.0f, m[0][e]);
          const float f = x == -INFINITY ? 1.0f : pat_exp2(m[0][e] - x);
          m[0][e] = x;
          l[0][e] *= f;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) o[mt][0][e] *= f, o[mt][0][e + 2] *= f;
        }
      }
      uint32_t pb[2][2];
      const uint64_t ms = f2_pack(m[0][0] == -INFINITY ? 0.0f : -m[0][0], m[0][1] == -INFINITY ? 0.0f : -m[0][1]);
      uint64_t sum = f2_pack(l[0][0], l[0][1]);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 z = f2_unpack(f2_add(f2_pack(s[kt][2 * e], s[kt][2 * e + 1]), ms));
          const uint64_t q = f2_pack(pat_exp2(z.x), pat_exp2(z.y));
          sum = f2_add(sum, q);
          const float2 y = f2_unpack(f2_mul(q, f2_pack(vs[kt][e], vs[kt][e])));
          w[2 * e] = y.x, w[2 * e + 1] = y.y;
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = see >> (kt * 4 + e) & 1 ? w[e] : 0.0f;
        }
        pb[kt][0] = pat_transpose(pat_pack<false>(w[0], w[1]));
        pb[kt][1] = pat_transpose(pat_pack<false>(w[2], w[3]));
      }
      const float2 sums = f2_unpack(sum);
      l[0][0] = sums.x, l[0][1] = sums.y;
      // NaN in a value, of a key that some row does not see?  (A run is read whole, what its page
      // holds behind the sequence with it.)
      bool odd = false;
      if (edge && (TMA || p.L > 1 || p.tail)) {
        for (int x = lane; x < 32 * CH; x += 32) {
          uint32_t w[4];
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(vs_base + warp * 32 * D + x * 16) : "memory");
#pragma unroll
          for (int k = 0; k < 4; ++k) odd |= (((w[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
        }
        odd = __any_sync(0xffffffffu, odd);
      }
      // O^T += V^T P^T
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t r[4], a[2][4];
        p8_ldsm_t((vs_base + v_lane) ^ (mt << 4), r);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          a[kt][0] = p8_half2(r[2 * kt] & 0xffffu), a[kt][1] = p8_half2(r[2 * kt + 1] & 0xffffu);
          a[kt][2] = p8_half2(r[2 * kt] >> 16), a[kt][3] = p8_half2(r[2 * kt + 1] >> 16);
        }
        if (!odd) {
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) pat_mma<false>(o[mt][0], a[kt], pb[kt][0], pb[kt][1]);
        } else {
          // row by row, the keys hidden from it zeroed
          for (int y = 0; y < 8; ++y) {
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
              uint32_t z[4];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int j = key0 + kt * 16 + p8_key(2 * c4 + e * 8);
                const uint32_t keep = (paged_visible<WIN>(p, at.b, at.n, j, r0 + y) ? 0xffffu : 0u) |
                                      (paged_visible<WIN>(p, at.b, at.n, j + 1, r0 + y) ? 0xffff0000u : 0u);
                z[2 * e] = a[kt][2 * e] & keep, z[2 * e + 1] = a[kt][2 * e + 1] & keep;
              }
              pat_mma<false>(d, z, pb[kt][0], pb[kt][1]);
            }
            const bool mine = (y >> 1) == c4;
            if (mine && (y & 1)) o[mt][0][1] += d[1], o[mt][0][3] += d[3];
            if (mine && !(y & 1)) o[mt][0][0] += d[0], o[mt][0][2] += d[2];
          }
        }
      }
    }
    const bool ends = at.unit + 1 == at.nu;
    if (ends || at.w + 1 >= end) {
      pat_sync();                      // the unit's keys have been read: O goes there
      paged_finish<D, 1, BF>(p, at, ends && first_unit == 0, first_unit == 0 ? 1 : 0, o, m, l,
                             reinterpret_cast<float4*>(smem + slot * S::STAGE), sm_m, sm_l, s_range, s_cut, s_join);
      fence_proxy_async_smem();        // before the slot is loaded again
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + 8 * slot);
    if (++slot == S::STAGES) slot = 0, phase ^= 1;
    at.next(p);
  }
  paged_leave<D, 1, BF>(p, s_cut, s_join, smem, S::RING);
}

}  // namespace simsd
