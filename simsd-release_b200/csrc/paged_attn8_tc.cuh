// Attention over the 8-bit paged cache for more than 16 rows per KV head, on the 5th-generation
// tensor cores: the operator and arithmetic of paged_attn8.cuh with the products of
// paged_attn_tc.cuh (a unit of 128 keys; the R queries stand 128 / R times in a product of 128
// rows, copy f of a row keeping the unit's keys f R .. f R + R - 1).
//
// tcgen05 takes fp16 queries and weights with fp16 keys and values, so K and V are brought to fp16
// on the way, exactly: two warps load 8-bit tiles of keys and of values into a ring (as
// paged_attn8.cuh does), four write them into a ring of fp16 tiles in the layout of the products (a
// conversion is one instruction for two numbers), four do the softmax, one issues the products.
// Reading and writing rows r and r ^ 5 together, eight lanes meet no bank conflict on either side.
// A last warp brings the units' scales, with log2 of those of the values, which the choice of the
// maximum goes by, so that the softmax takes none.
//
// What bounds it is not HBM but the chain of a unit: S (some 1000 cycles with its waits), the
// softmax of 32 keys a thread (1100 - 1300), the weights' way back into TMEM and O, 2.1 us a unit at 2 x 64k
// tokens x 8 rows x 4 heads (8192 units on 148 CTAs).  paged_attn_tc.cuh, the same chain without a conversion before it, takes
// 1.7 there, on twice the bytes; what the 0.4 consist of has not been taken apart (the fp16 ring holds two
// units, its ring three).  The 16-bit cache is therefore the faster one for more than 16 rows without a window.
// Other loads change little: one warp for all of them 126 us at 2 x 64k x 8 rows, the
// converting warps for themselves by cp.async 134, this 133 (in one run then).
// Measured (B200, 8 KV heads x 128, 4 query heads each, pages of 16, bf16; device time in a graph of
// calls, in brackets over the 16-bit cache): 16 x 1-3k tokens x 8 rows 49 us (37), x 16 rows 64 (51); with mma.sync in tiles of
// 16 rows 53 and 89 (its sequences' ends weighed as one unit, as here then: 54 and 75).  2 x 64k tokens x 8 rows 115 us (95); 19 x
// 0-9k in a window of 1000, 5 rows x 7 heads, 29; 16 x 8-32k in a window of 4096 x 8 and 32 rows 81 (101) and 249 (360).
//
// Hidden keys as there: a key that no row sees becomes zeros in the fp16 tile, as does one that
// some rows do not see where its values hold NaN; the rows that see that one add it by
// themselves.  All waits are bounded.
#pragma once
#include "paged_attn8.cuh"
#include "paged_attn_tc.cuh"

namespace simsd {

constexpr int P8T_THREADS = 384;

template <int D, int R>
struct P8tShape {
  static constexpr int F = 128 / R;
  static constexpr int RAW = 128 * D, TILE = 2 * RAW;          // 128 keys or values: in 8 bits, in fp16
  static constexpr int NR = D == 128 ? 4 : 8, NS = 4, NU = 8;  // tiles of both rings (8-bit ones of keys and values in turn), units of scales
  static constexpr int SC = 3 * 512;                           // a unit's scales: of keys, of values, log2 of these
  static constexpr int X = 16384;                              // 32 dims of every lane's O, where copies are joined
  static constexpr int BYTES = 1024 + NS * TILE + NR * RAW + X + 1024 + NU * SC + 512;
  static_assert(PTC_MAX_PARTS * R * 8 <= BYTES - 1024 - 512);  // ptc_join, in front of the barriers
  using Tmem = PtcShape<D, R>;
};

// The warp that loads keys (kv 0) or values (1), units from `ld` up to `end`.  TMA: a lane per run of
// tokens of one page; one without a key that is read loads zeros, from past the last page.  Else
// the lane's keys are lane, 32 + lane, ...: their places are handed round.  The page numbers are
// fetched a unit ahead.
template <int D, bool TMA, typename S>
__device__ __forceinline__ void p8t_load(const PagedAttn8Args& args, P8Pos<true> ld, int end, int kv, uint32_t raw,
                                         uint32_t full, uint32_t empty, volatile int* abort_flag) {
  constexpr int CH = D / 16, KPI = 32 / CH, EACH = PTC_TK / 32, PAGES = TMA ? 1 : EACH;
  const PagedAttnArgs& p = args.a;
  const int lane = threadIdx.x & 31, kc = lane % CH, khi = lane / CH;
  const int run = TMA ? args.run : 1, runs = PTC_TK / run;           // TMA: up to 16 runs
  const uint64_t policy = policy_evict_first();
  const CUtensorMap* map = kv ? &args.v : &args.k;
  const uint8_t* base = reinterpret_cast<const uint8_t*>(kv ? p.v_cache : p.k_cache);
  if (TMA && lane == 0) prefetch_tmap(map);
  int page[PAGES];
  auto fetch_pages = [&](const P8Pos<true>& x) {
#pragma unroll
    for (int i = 0; i < PAGES; ++i)
      page[i] = !TMA || lane < runs ? paged_page(p, x, x.key(p) + (TMA ? lane * run : i * 32 + lane), run) : -1;
  };
  fetch_pages(ld);
  int slot = kv;
  uint32_t phase = 0, filled = 0, parity = 0;
  bool ok = true;
  while (ld.w < end) {
    const int key0 = ld.key(p), n = ld.n, g = ld.g;
    int from[PAGES];
#pragma unroll
    for (int i = 0; i < PAGES; ++i) from[i] = page[i] >= 0 && page[i] < p.num_pages ? page[i] : TMA ? p.num_pages : -1;
    ld.next(p);
    if (ld.w < end) fetch_pages(ld);
    const int first = key0 + lane * run, tok = first - p.page_div(first) * p.page_size;
    ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * slot, phase ^ 1, abort_flag, p.err));
    if (!ok) break;
    const uint32_t bar = full + 8 * slot, dst = raw + slot * S::RAW;
    if constexpr (TMA) {
      if (lane == 0) mbar_arrive_expect_tx(bar, S::RAW);
      __syncwarp();
      if (lane < runs) p8_tma(dst + lane * run * D, map, bar, tok, g, from[0], policy);
    } else {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int key = key0 + i * 32 + lane;
        const long long off = from[i] >= 0 && key < n ? from[i] * p.ld_page + g * p.ld_head +
                                                            (key - p.page_div(key) * p.page_size) * p.ld_tok : -1;
#pragma unroll
        for (int x = 0; x < 32 / KPI; ++x) {
          const long long o = __shfl_sync(0xffffffffu, off, x * KPI + khi);
          pat_cp16(dst + pat8_off<D>(i * 32 + x * KPI + khi, kc), base + (o < 0 ? 0 : o + kc * 16), o >= 0);
        }
      }
      p8_cp_arrive(bar);
    }
    filled |= 1u << slot;
    parity = (parity & ~(1u << slot)) | phase << slot;
    if ((slot += 2) >= S::NR) slot = kv, phase ^= 1;
  }
  // giving up: no copy may land after the CTA has left
  if (!ok) {
    pat_commit();
    pat_wait<0>();
    if (TMA)
      for (int s = 0; s < S::NR; ++s)
        if (filled >> s & 1) mbar_wait_drain(full + 8 * s, parity >> s & 1, 100000000ull);
  }
  __syncwarp();
}

// The warp that brings the scales: lane, 32 + lane, ... of every unit, loaded a unit ahead of
// their use, their pages two.
template <typename S>
__device__ __forceinline__ void p8t_scales(const PagedAttn8Args& args, P8Pos<true> ld, int end, float* sc, uint32_t full,
                                           uint32_t empty, volatile int* abort_flag) {
  constexpr int EACH = PTC_TK / 32;
  const PagedAttnArgs& p = args.a;
  const int lane = threadIdx.x & 31;
  int page[EACH];
  float ks[EACH], vs[EACH];
  auto fetch_pages = [&]() {
#pragma unroll
    for (int i = 0; i < EACH; ++i) page[i] = ld.w < end ? paged_page(p, ld, ld.key(p) + i * 32 + lane, 1) : PAGED_UNSEEN;
  };
  auto fetch = [&]() {                             // of unit `ld`, which moves on
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int key = ld.key(p) + i * 32 + lane, tok = key - p.page_div(key) * p.page_size;
      const bool fine = page[i] >= 0 && page[i] < p.num_pages;
      if (!fine && page[i] != PAGED_UNSEEN && key < ld.n && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
      const long long at = page[i] * args.lds_page + ld.g * args.lds_head + args.block_div(tok) * args.lds_block;
      ks[i] = fine ? __ldg(args.k_scale + at) : 0.0f;
      vs[i] = fine ? __ldg(args.v_scale + at) : 0.0f;
    }
    if (ld.w < end) ld.next(p);
    fetch_pages();
  };
  fetch_pages();
  fetch();
  int unit = 0;
  uint32_t phase = 0;
  for (int w = 0, left = 1; left; ++w) {
    left = ld.w < end;                             // after the unit in hand
    float k[EACH], v[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) k[i] = ks[i], v[i] = vs[i];
    if (left) fetch();
    if (!__all_sync(0xffffffffu, mbar_wait(empty + 8 * unit, phase ^ 1, abort_flag, p.err))) break;
    float* to = sc + unit * 384 + lane;
#pragma unroll
    for (int i = 0; i < EACH; ++i) to[i * 32] = k[i], to[128 + i * 32] = v[i], to[256 + i * 32] = fmaxf(p8_log2(v[i]), -64.0f);
    mbar_arrive(full + 8 * unit);
    if (++unit == S::NU) unit = 0, phase ^= 1;
  }
}

template <int D, int R, bool BF>
__global__ void __launch_bounds__(P8T_THREADS, 1) paged_attention8_tc_kernel(const __grid_constant__ PagedAttn8Args args) {
  const PagedAttnArgs& p = args.a;
  using S = P8tShape<D, R>;
  using T = typename S::Tmem;
  constexpr int F = S::F, NS = S::NS, CH = D / 8;
  extern __shared__ uint8_t ptc_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ptc_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* raw = tiles + NS * S::TILE;
  uint8_t* own_x = raw + S::NR * S::RAW;
  float* xm = reinterpret_cast<float*>(own_x + S::X);    // [128] maximum, then [128] sum of a lane
  float* xl = xm + 128;
  float* sc = xl + 128;                                  // [NU][3][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sc + S::NU * 384);
  uint64_t *raw_full = bars, *raw_empty = bars + 8, *full = bars + 16, *empty = bars + 20, *sc_full = bars + 24, *sc_empty = bars + 32,
           *q_full = bars + 40, *s_full = bars + 41, *p_full = bars + 43, *pv_done = bars + 44, *drained = bars + 45;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 46);
  volatile int* abort_flag = reinterpret_cast<int*>(bars + 46) + 1;
  uint32_t* bad = reinterpret_cast<uint32_t*>(bars + 47);  // [4] keys of the unit with values that are not finite
  __shared__ PagedPart s_cut[2];
  __shared__ PagedCut s_range;
  __shared__ bool s_join[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) mbar_init(smem_u32(full + s), 128), mbar_init(smem_u32(empty + s), 1);
    for (int s = 0; s < S::NR; ++s) mbar_init(smem_u32(raw_full + s), args.run ? 1 : 32), mbar_init(smem_u32(raw_empty + s), 4);
    for (int s = 0; s < S::NU; ++s) mbar_init(smem_u32(sc_full + s), 32), mbar_init(smem_u32(sc_empty + s), 4);
    mbar_init(smem_u32(q_full), PTC_SOFTMAX);
    mbar_init(smem_u32(s_full), 1);
    mbar_init(smem_u32(s_full + 1), 1);
    mbar_init(smem_u32(p_full), PTC_SOFTMAX);
    mbar_init(smem_u32(pv_done), 1);
    mbar_init(smem_u32(drained), 1);
    *abort_flag = 0;
    s_cut[0].parts = s_cut[1].parts = 0;
    s_join[0] = s_join[1] = false;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  griddep_launch_dependents();
  griddep_wait();
  P8Pos<true> at;
  PagedCut cut;
  tc_fence_before();
  __syncthreads();
  const bool mine = paged_range<P8T_THREADS, PTC_TK, true>(p, cut, at);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t o_col = tmem + T::O;
  if (mine) {
    const int end = cut.first(blockIdx.x + 1);
    if (tid == 0) s_range = cut;
    if (warp == 9 || warp == 10) {
      // ================= loads
      if (args.run)
        p8t_load<D, true, S>(args, at, end, warp - 9, smem_u32(raw), smem_u32(raw_full), smem_u32(raw_empty), abort_flag);
      else
        p8t_load<D, false, S>(args, at, end, warp - 9, smem_u32(raw), smem_u32(raw_full), smem_u32(raw_empty), abort_flag);
    } else if (warp == 11) {
      p8t_scales<S>(args, at, end, sc, smem_u32(sc_full), smem_u32(sc_empty), abort_flag);
    } else if (warp >= 4 && warp < 8) {
      // ================= tiles to fp16: 32 rows a warp, 8 rows x 64 bytes at a time
      constexpr int H = D / 64;
      const int row0 = (warp - 4) * 32 + ((lane >> 3) ^ (lane & 4 ? 5 : 0)), c8 = lane & 3;
      int rs = 0, fs = 0;
      uint32_t rph = 0, fph = 0;
      auto wait = [&](uint64_t* bar, uint32_t par) {
        return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), par, abort_flag, p.err)) != 0;
      };
      bool ok = true;
      while (ok && at.w < end) {
        at.next(p);
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          if (!(ok = wait(raw_full + rs + kv, rph))) break;
          uint4 u[4][H];
          const uint32_t src = smem_u32(raw) + (rs + kv) * S::RAW;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < H; ++h)
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(u[i][h].x), "=r"(u[i][h].y), "=r"(u[i][h].z), "=r"(u[i][h].w)
                           : "r"(src + pat8_off<D>(row0 + 8 * i, c8 + 4 * h)) : "memory");
          if (!(ok = wait(empty + fs + kv, fph ^ 1))) break;
          uint8_t* dst = tiles + (fs + kv) * S::TILE;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < H; ++h) {
              const uint32_t w[4] = {u[i][h].x, u[i][h].y, u[i][h].z, u[i][h].w};
              uint32_t y[8];
#pragma unroll
              for (int k = 0; k < 4; ++k) y[2 * k] = p8_half2(w[k] & 0xffffu), y[2 * k + 1] = p8_half2(w[k] >> 16);
              const int row = row0 + 8 * i, c = 2 * (c8 + 4 * h);
              *reinterpret_cast<uint4*>(dst + ptc_off(row, c)) = make_uint4(y[0], y[1], y[2], y[3]);
              *reinterpret_cast<uint4*>(dst + ptc_off(row, c + 1)) = make_uint4(y[4], y[5], y[6], y[7]);
            }
          fence_proxy_async_smem();
          mbar_arrive(smem_u32(full + fs + kv));
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(raw_empty + rs + kv));
        }
        if ((rs += 2) == S::NR) rs = 0, rph ^= 1;
        if ((fs += 2) == NS) fs = 0, fph ^= 1;
      }
    } else if (warp == 8) {
      // ================= products
      const uint32_t idesc_s = make_idesc_f16(false, 128, 128);
      const uint32_t idesc_o = make_idesc_f16(false, 128, D) | (1u << 16);   // V is MN-major
      uint32_t ks = 0, kph = 0, vs = 1, vph = 0, items = 0;
      bool ok = true, first = true, prev_first = true, any = false;
      // operand descriptors of the ring's first tile; addresses in them count 16 bytes
      const uint64_t desc_k = make_sw128_desc(smem_u32(tiles)), desc_v = ptc_desc_mn(smem_u32(tiles));
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, abort_flag, p.err)) != 0;
      };
      auto product_s = [&](int n) {
        if (first && !wait(q_full, items++ & 1)) return false;
        if (!wait(full + ks, kph)) return false;
        tc_fence_after();
        const uint64_t kt = desc_k + ks * (S::TILE >> 4);
        if (ptc_elect()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            ptc_mma(tmem + (n & 1) * 128, tmem + T::Q + kk * 8, kt + (kk >> 2) * 1024 + 2 * (kk & 3), idesc_s, kk > 0);
          tc_commit(smem_u32(s_full + (n & 1)));
          tc_commit(smem_u32(empty + ks));
        }
        __syncwarp();
        any = true;
        ks += 2;
        if (ks >= NS) ks -= NS, kph ^= 1;
        return true;
      };
      auto product_o = [&](int n, bool start) {
        if (!wait(p_full, n & 1) || !wait(full + vs, vph)) return false;
        tc_fence_after();
        const uint64_t vt = desc_v + vs * (S::TILE >> 4);
        if (ptc_elect()) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            ptc_mma(o_col, tmem + T::P + kk * 8, vt + kk * 128, idesc_o, kk > 0 || !start);
          tc_commit(smem_u32(empty + vs));
          tc_commit(smem_u32(pv_done));
        }
        __syncwarp();
        vs += 2;
        if (vs >= NS) vs -= NS, vph ^= 1;
        return true;
      };
      // S of a unit goes before O of the one before it, except where a new sequence's
      // queries are still on their way
      int n = 0;
      for (; ok && at.w < end; ++n) {
        first = n == 0 || at.unit == 0;
        if (first && n > 0) ok = product_o(n - 1, prev_first);
        ok = ok && product_s(n);
        if (!first && ok) ok = product_o(n - 1, prev_first);
        prev_first = first;
        at.next(p);
      }
      if (ok) ok = product_o(n - 1, prev_first);
      if (any) {   // nothing in flight when the CTA gives its TMEM back
        if (ptc_elect()) tc_commit(smem_u32(drained));
        __syncwarp();
        mbar_wait_drain(smem_u32(drained), 0, 100000000ull);
      }
      __syncwarp();
    } else if (warp < 4) {
      // ================= softmax and epilogue: a thread per TMEM lane, copy f of row `row`
      const int row = tid % R, f = tid / R;
      const uint32_t t_lane = (uint32_t)(warp * 32) << 16;
      {
        float zero[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) zero[e] = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) ptc_st16(tmem + T::P + t_lane + c * 16, zero);
      }
      float q_next = 1.0f;                 // scale log2(e) times the power of two that the next queries are divided by
      // the queries of a sequence, head and row tile into TMEM as fp16, the copies alike
      auto put_queries = [&](int b, int g, int rt) {
        const int r = rt * R + row;
        const bool in = r < p.rows && b < p.B;
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) +
                                                          (in ? paged_row(p, b, g, r) * D : 0));
        float up = 1.0f;
        q_next = p.scale_log2;
        if constexpr (BF) {
          float top = 0.0f;
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            const uint4 y = in ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xffff0000u))));
          }
          const int ex = p8_query_exponent(top);
          up = p8_power(-ex);
          q_next *= p8_power(ex);
        }
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float x[16];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint4 y = in ? __ldg(src + 4 * c + e) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              x[4 * e + k] = __uint_as_float(BF ? pat_pack<false>(__uint_as_float(w[k] << 16) * up, __uint_as_float(w[k] & 0xffff0000u) * up) : w[k]);
          }
          ptc_st16(tmem + T::Q + t_lane + c * 16, x);
        }
        ptc_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(q_full));
      };
      put_queries(at.b, at.g, at.rt);
      float m = -INFINITY, l = 0.0f, qs = 0.0f;
      int first_unit = at.unit, unit = 0;
      uint32_t uph = 0, vs = 1, vph = 0;
      bool ok = true;
      auto wait_all = [&](uint64_t* bar, uint32_t parity) {
        return named_bar_and(1, PTC_SOFTMAX, mbar_wait(smem_u32(bar), parity, abort_flag, p.err));
      };
      for (int n = 0; ok && at.w < end; ++n) {
        if (n == 0 || at.unit == 0) {
          first_unit = at.unit;
          m = -INFINITY, l = 0.0f, qs = q_next;
        }
        if (!(ok = named_bar_and(1, PTC_SOFTMAX, mbar_wait(smem_u32(s_full + (n & 1)), (n >> 1) & 1, abort_flag, p.err) &&
                                                     mbar_wait(smem_u32(sc_full + unit), uph, abort_flag, p.err))))
          break;
        tc_fence_after();
        float v[R];
#pragma unroll
        for (int c = 0; c < R / 16; ++c)
          tmem_ld16(tmem + t_lane + (n & 1) * 128 + f * R + c * 16, *reinterpret_cast<float(*)[16]>(v + c * 16));
        const float4* scale_k = reinterpret_cast<const float4*>(sc + unit * 384 + f * R);
        const float4* scale_v = scale_k + 32;
        const float4* log_v = scale_k + 64;
        tmem_wait_ld();
        const uint64_t qs2 = f2_pack(qs, qs);
#pragma unroll
        for (int c = 0; c < R; c += 4) {
          const float4 k4 = scale_k[c / 4];
          const float2 a = f2_unpack(f2_mul(f2_pack(v[c], v[c + 1]), f2_mul(f2_pack(k4.x, k4.y), qs2)));
          const float2 b = f2_unpack(f2_mul(f2_pack(v[c + 2], v[c + 3]), f2_mul(f2_pack(k4.z, k4.w), qs2)));
          v[c] = a.x, v[c + 1] = a.y, v[c + 2] = b.x, v[c + 3] = b.y;
        }
        const int k0 = at.key(p), key0 = k0 + f * R, base = at.n - p.L;
        const bool edge = k0 + PTC_TK > base || paged_out(p, at.n, k0, PTC_TK);
        uint32_t see[R / 32];
        bool strange = false;
        if (edge) {
          // the lane's keys that its row sees: below `lim`, or in the mask; not from `sinks` to `gone`
          const int t = min(p.g_div(at.rt * R + row), p.L - 1);
          const int lim = (p.tail ? min(at.n, base) : min(at.n, base + t + 1)) - key0;
          const int from = min(p.sinks, at.n) - key0, gone = max(base + t - p.window + 1, 0) - key0;
          const uint8_t* tm = p.tail ? p.tail + at.b * p.ldm_b + t * p.ldm_t : nullptr;
          auto below = [](int k) { return k <= 0 ? 0u : k >= 32 ? 0xffffffffu : (1u << k) - 1u; };
#pragma unroll
          for (int w = 0; w < R / 32; ++w) {
            see[w] = below(lim - 32 * w);
            if (tm) {
              const int lo = max(0, base - (key0 + 32 * w)), hi = min(32, at.n - (key0 + 32 * w));
#pragma unroll 8
              for (int c = lo; c < hi; ++c) see[w] |= (uint32_t)(tm[key0 + 32 * w + c - base] != 0) << c;
            }
            see[w] &= ~(below(gone - 32 * w) & ~below(from - 32 * w));
          }
#pragma unroll
          for (int c = 0; c < R; ++c)
            if (!(see[c / 32] >> (c % 32) & 1)) v[c] = -INFINITY;
          // Values of keys that no row sees are whatever their page holds (a run is read whole):
          // zero.  Of keys that some row may not see, values that are not finite leave the product.
          if (!(ok = wait_all(full + vs, vph))) break;
          uint8_t* vt = tiles + vs * S::TILE;
          const int key = k0 + tid;
          const bool never = key >= at.n || (key >= p.sinks && key < paged_first(p, at.n));
          bool odd = false;
          if (!never && (key >= base || (key >= p.sinks && key < at.n - p.window))) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
              const uint4 u = *reinterpret_cast<const uint4*>(vt + ptc_off(tid, c));
              const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) odd |= (w[k] & 0x7c00u) == 0x7c00u || ((w[k] >> 16) & 0x7c00u) == 0x7c00u;
            }
          }
          if (odd || never) {
#pragma unroll
            for (int c = 0; c < CH; ++c) *reinterpret_cast<uint4*>(vt + ptc_off(tid, c)) = make_uint4(0, 0, 0, 0);
          }
          const uint32_t b = __ballot_sync(0xffffffffu, odd);
          if (lane == 0) bad[warp] = b;
          named_bar_sync(1, PTC_SOFTMAX);
          strange = (bad[0] | bad[1] | bad[2] | bad[3]) != 0;
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < R; c += 4) {
          const float4 g4 = log_v[c / 4];
          m4[0] = fmaxf(m4[0], v[c] + g4.x), m4[1] = fmaxf(m4[1], v[c + 1] + g4.y);
          m4[2] = fmaxf(m4[2], v[c + 2] + g4.z), m4[3] = fmaxf(m4[3], v[c + 3] + g4.w);
        }
        const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        const bool up = mx > m + 15.0f;          // a weight would pass 2^15: the largest becomes 2^8
        float w_old = 1.0f;                      // what the sums so far are scaled by
        if (up) {
          w_old = m == -INFINITY ? 0.0f : pat_exp2(m - (mx - 8.0f));
          m = mx - 8.0f;
        }
        const float ms = m == -INFINITY ? 0.0f : -m;
        const uint64_t ms2 = f2_pack(ms, ms);
        uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
        for (int c = 0; c < R; c += 4) {
          const float4 v4 = scale_v[c / 4];
          const float2 a = f2_unpack(f2_add(f2_pack(v[c], v[c + 1]), ms2)), b = f2_unpack(f2_add(f2_pack(v[c + 2], v[c + 3]), ms2));
          const uint64_t x = f2_pack(pat_exp2(a.x), pat_exp2(a.y)), y = f2_pack(pat_exp2(b.x), pat_exp2(b.y));
          sum0 = f2_add(sum0, x), sum1 = f2_add(sum1, y);
          const float2 wx = f2_unpack(f2_mul(x, f2_pack(v4.x, v4.y))), wy = f2_unpack(f2_mul(y, f2_pack(v4.z, v4.w)));
          v[c] = wx.x, v[c + 1] = wx.y, v[c + 2] = wy.x, v[c + 3] = wy.y;
        }
        if (edge) {
#pragma unroll
          for (int c = 0; c < R; ++c)
            if (!(see[c / 32] >> (c % 32) & 1)) v[c] = 0.0f;       // whatever the scale of a hidden key is
        }
        const float2 s0 = f2_unpack(sum0), s1 = f2_unpack(sum1);
        l = fmaf(l, w_old, (s0.x + s0.y) + (s1.x + s1.y));
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(sc_empty + unit));
        if (++unit == S::NU) unit = 0, uph ^= 1;
        // O of the units before has been summed, P may be written
        if (n > 0) {
          if (!(ok = wait_all(pv_done, (n - 1) & 1))) break;
          tc_fence_after();
        }
        if (n > 0 && at.unit > first_unit && __any_sync(0xffffffffu, up)) {
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            float x[16];
            tmem_ld16(o_col + t_lane + c * 16, x);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] *= w_old;
            ptc_st16(o_col + t_lane + c * 16, x);
          }
          ptc_wait_st();
        }
#pragma unroll
        for (int c = 0; c < R / 32; ++c) {
          float x[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = __uint_as_float(pat_pack<false>(v[32 * c + 2 * e], v[32 * c + 2 * e + 1]));
          ptc_st16(tmem + T::P + t_lane + f * (R / 2) + c * 16, x);
        }
        ptc_wait_st();
        tc_fence_before();
        if (edge) fence_proxy_async_smem();      // values that were zeroed
        mbar_arrive(smem_u32(p_full));
        vs += 2;
        if (vs >= NS) vs -= NS, vph ^= 1;
        const bool ends = at.unit + 1 == at.nu, leaves = ends || at.w + 1 >= end;
        if (ends && at.w + 1 + at.END < end) {
          int b = at.b, g = at.g, rt = at.rt;
          P8Pos<true>::next_rows(p, b, g, rt);
          put_queries(b, g, rt);
        }
        if (strange || leaves) {
          if (!(ok = wait_all(pv_done, n & 1))) break;
          tc_fence_after();
        }
        if (strange) {
          // the values that were taken out, for the rows that see them
#pragma unroll 1
          for (int k = 0; k < 128; ++k) {
            if (!(bad[k / 32] >> (k % 32) & 1)) continue;
            const int j = k0 + k, c = k - f * R;
            float w = 0.0f;
            bool on = false;
#pragma unroll
            for (int e = 0; e < R; ++e)
              if (e == c) w = v[e], on = see[e / 32] >> (e % 32) & 1;
            const int page = p.page_table[at.b * p.ld_table + p.page_div(j)];
            if (page < 0 || page >= p.num_pages) continue;
            const uint8_t* from = reinterpret_cast<const uint8_t*>(p.v_cache) + page * p.ld_page + at.g * p.ld_head +
                                  (j - p.page_div(j) * p.page_size) * p.ld_tok;
#pragma unroll 1
            for (int d = 0; d < D / 16; ++d) {
              float x[16];
              tmem_ld16(o_col + t_lane + d * 16, x);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const uint32_t two = p8_half2(from[d * 16 + e]);
                if (on) x[e] = fmaf(w, __half2float(__ushort_as_half((unsigned short)(two & 0xffffu))), x[e]);
              }
              ptc_st16(o_col + t_lane + d * 16, x);
            }
            ptc_wait_st();
          }
          named_bar_sync(1, PTC_SOFTMAX);          // `bad` read
          tc_fence_before();
        }
        if (leaves) {
          // a whole sequence is written, a part goes to the workspace
          const bool whole = ends && first_unit == 0;
          const int part = first_unit == 0 ? 1 : 0, r0 = at.rt * R;
          const long long slot = 2LL * blockIdx.x + part;
          float mm = m, ll = l, w = 1.0f;
          if constexpr (F > 1) {
            xm[tid] = m, xl[tid] = l;
            named_bar_sync(1, PTC_SOFTMAX);
            mm = -INFINITY, ll = 0.0f;
#pragma unroll
            for (int k = 0; k < F; ++k) mm = fmaxf(mm, xm[k * R + row]);
            const float mu = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
            for (int k = 0; k < F; ++k) ll = fmaf(xl[k * R + row], pat_exp2(xm[k * R + row] - mu), ll);
            w = pat_exp2(m - mu);
          }
          if (whole) w *= ll == 0.0f ? 0.0f : 1.0f / ll;
          if (f == 0) {
            if (whole)
              paged_store_lse(p, at.b, at.g, r0 + row, mm, ll);
            else
              p.part_ml[slot * R + row] = make_float2(mm, ll);
          }
          if (whole && ll == 0.0f) w = 0.0f;
          float* po = reinterpret_cast<float*>(p.part_o) + slot * R * D;
          auto put = [&](int r, int q4, float4 a) {          // four dims of a row
            if (!whole) {
              *(reinterpret_cast<float4*>(po + r * D) + q4) = a;
            } else if (r0 + r < p.rows) {
              *(reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.o) + paged_row(p, at.b, at.g, r0 + r) * D) + q4) =
                  make_uint2(pat_pack<BF>(a.x, a.y), pat_pack<BF>(a.z, a.w));
            }
          };
#pragma unroll 1
          for (int h = 0; h < D / 32; ++h) {
            float x[2][16];
#pragma unroll
            for (int c = 0; c < 2; ++c) tmem_ld16(o_col + t_lane + h * 32 + c * 16, x[c]);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int q4 = c * 4 + e;
                const float4 a = make_float4(x[c][4 * e] * w, x[c][4 * e + 1] * w, x[c][4 * e + 2] * w, x[c][4 * e + 3] * w);
                if constexpr (F == 1)
                  put(row, h * 8 + q4, a);
                else
                  *reinterpret_cast<float4*>(own_x + ptc_off(tid, q4)) = a;
              }
            }
            if constexpr (F > 1) {
              named_bar_sync(1, PTC_SOFTMAX);
#pragma unroll
              for (int k = 0; k < R * 8 / PTC_SOFTMAX; ++k) {
                const int x = tid + k * PTC_SOFTMAX, r = x / 8, q4 = x % 8;
                float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int i = 0; i < F; ++i) {
                  const float4 y = *reinterpret_cast<const float4*>(own_x + ptc_off(i * R + r, q4));
                  a.x += y.x, a.y += y.y, a.z += y.z, a.w += y.w;
                }
                put(r, h * 8 + q4, a);
              }
              named_bar_sync(1, PTC_SOFTMAX);
            }
          }
          tc_fence_before();
          if (!whole) {
            if (part == 0) named_bar_sync(1, PTC_SOFTMAX);
            if (tid == 0) {
              const PagedCut range = s_range;
              const int head = at.w - at.unit, c0 = range.cta_of(head);
              s_cut[part] = {at.b, at.g, r0, c0, range.cta_of(head + at.nu - 1) - c0 + 1};
              // the first part at once, so that it is not this CTA that everyone else waits for in the end
              if (part == 0) s_join[0] = paged_arrive(p, s_cut[0]);
            }
          }
        }
        at.next(p);
      }
      if (!ok && tid == 0) s_join[0] = false, s_cut[1].parts = 0;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  // cut sequences (at most the range's first and last): the last of their CTAs to get here joins the parts
  if (tid == 0 && s_cut[1].parts > 0) s_join[1] = paged_arrive(p, s_cut[1]);
  __syncthreads();
  for (int k = 0; k < 2; ++k)
    if (s_join[k]) ptc_join<D, R, BF, P8T_THREADS>(p, s_cut[k], reinterpret_cast<float2*>(tiles));
}

}  // namespace simsd
