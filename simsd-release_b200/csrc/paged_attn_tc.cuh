// Paged attention for more than 16 rows per KV head (several drafted tokens times
// the head group), on the 5th-generation tensor cores.  Same operator, cut and
// workspace scheme as paged_attn.cuh, whose mma.sync products at 32 rows already
// cost more than reading the keys and values: 16 x 8 drafted rows x 4 heads took 51 to
// 57 us there, against 21 of HBM.
//
// A unit is 128 keys of one (sequence, KV head, row tile of R = 32, 64 or 128 rows).
// The products are 128 rows tall whatever R is; the R queries stand in them F = 128 /
// R times, and copy f of a row keeps only the keys [f R, f R + R) of every unit:
//   S = Q K^T       [128 x 128 keys], TMEM; a thread per TMEM lane reads its R keys
//   softmax         per lane (a row's copy is a softmax of its own, joined at the end):
//                   no exchange between threads, R exponentials each
//   P               16-bit, in TMEM, zero outside a copy's own keys
//   O += P V        [128 x D], TMEM, accumulated over the units of the sequence
// so a unit's softmax is spread over all 128 lanes at 32 rows too.  Q and P are read
// from TMEM, which leaves 64 KB of shared memory to the ring (47 -> 44 us).  The running
// maximum moves only when a score passes it by more than 2^8 (P <= 256 keeps its
// relative precision in 16 bits), so O is hardly ever rescaled in TMEM.  P is rounded to
// the 16-bit type as there, the largest weight too: error 2.2e-3 of the output in the
// 2-norm against 1.7e-3 for its own rounding alone.
//
// Warps 0-3 softmax and epilogue, 4-7 loads into a ring of NS operand tiles K, V, K,
// V, ..., 8 issues the products: S of unit n + 1 before O of unit n, so that they
// overlap its softmax.  One CTA per SM.  Pages of a multiple of 8 tokens are loaded
// with TMA, a lane per run of `block` tokens that lies in one page, spread over warps
// 4-7 (by one warp alone 16 x 8 rows take 54 us with pages of 8, 39.5 with 16; by four
// 37 each); other pages with cp.async into the same swizzled layout (41 us, pages of 1,
// 4 and 12).  At 2 x 64k x 8 rows TMA takes 91-92 us and cp.async 95 with pages of 8 to
// 128; with 64 dims and pages of 8 TMA is behind, 120 against 117 at 4 x 64k.
//
// A value that is not finite, of a key that some rows do not see, is taken out of the
// product and added to the rows that see it by themselves.  One that all rows see stays,
// and makes NaN of the sums of the copies that do not keep its key (P = 0 there): where the
// copies of a row join to no finite number, what the row's keys hold says which it is.
// All waits are bounded.
//
// Measured (B200, 8 KV heads x 128, 4 query heads each, bf16; device time in a graph of
// calls): 16 x 1-3k tokens x 8 rows 37 us (39 one after the other on a stream), 3.8 TB/s;
// 2 x 64k x 8 rows 91-93 us, 5.5 TB/s, 85 % of the measured copy rate.  64 and 128 rows,
// with R keys a softmax thread: 16 x 1-3k 51 and 76 us.  Looking for values that are not
// finite in every unit instead of in the joined sums took 40 and 54 us at 32 and 64 rows.
#pragma once
#include "paged_attn.cuh"

namespace simsd {

constexpr int PTC_THREADS = 288, PTC_SOFTMAX = 128, PTC_TK = 128;

template <int D, int R>
struct PtcShape {
  static constexpr int F = 128 / R;
  static constexpr int TILE = 128 * D * 2;              // 128 keys or values
  static constexpr int NS = D == 128 ? 6 : 8;
  static constexpr int X = 32768;                       // 64 dims of every lane's O, where copies are joined
  static constexpr int BYTES = 1024 + NS * TILE + X + 1024 + 512;
  // TMEM columns: S of even and odd units, O, then Q and P, two 16-bit values a column
  static constexpr int O = 256, Q = O + D, P = Q + D / 2;
  static_assert(P + 64 <= 512);
};

// D (+)= A B^T with A in TMEM (a lane per row, two 16-bit values a column)
__device__ __forceinline__ void ptc_mma(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void ptc_st16(uint32_t taddr, const float (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
      "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
      "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
      "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])), "r"(__float_as_uint(v[15]))
      : "memory");
}
__device__ __forceinline__ void ptc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One lane of a converged warp.  The product warp runs its loop with all lanes, so
// that what the instructions take stays in uniform registers.
__device__ __forceinline__ bool ptc_elect() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// MN-major operand in the 128-byte swizzle: V as it lies, 16 keys a step
__device__ __forceinline__ uint64_t ptc_desc_mn(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFF);
  d |= (uint64_t)(16384 >> 4) << 16;      // to the next 64 dims
  d |= (uint64_t)(1024 >> 4) << 32;       // to the next 8 keys
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// 16-byte chunk c of row r of an operand tile (blocks of 64 elements x 128 rows)
__device__ __forceinline__ uint32_t ptc_off(int r, int c) {
  return (uint32_t)((c >> 3) * 16384 + r * 128 + (((c ^ r) & 7) << 4));
}

struct PtcArgs {
  PagedAttnArgs a;
  CUtensorMap k, v;        // [pages, Hk, page size, D], box {64 dims, block tokens, 1, 1}; where block > 0
  int block;               // tokens of a TMA load: the largest power of two <= 128 in the page size, or 0
};

__device__ __forceinline__ void ptc_tma(uint32_t dst, const void* map, uint32_t bar, int x, int tok, int head, int page,
                                        uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(tok), "r"(head), "r"(page), "l"(policy)
      : "memory");
}

// Joins the parts of a cut sequence (rows r0 .. r0 + R - 1 of KV head g), as
// paged_join; parts hold R rows of D.  `buf`: parts * R float2 of shared memory.
template <int D, int R, bool BF>
__device__ void ptc_join(const PagedAttnArgs& p, const PagedPart& x, float2* buf) {
  const int tid = threadIdx.x;
  auto slot = [&](int i) { return (long long)(i == 0 ? 2 * x.c0 + 1 : 2 * (x.c0 + i)); };
  for (int k = tid; k < x.parts * R; k += PTC_THREADS) buf[k] = __ldcg(p.part_ml + slot(k / R) * R + k % R);
  __syncthreads();
  // (maximum, 1 / sum) of a row from its parts, in order
  auto law = [&](int r, bool lse) {
    float mm = -INFINITY, ll = 0.0f;
    for (int i = 0; i < x.parts; ++i) mm = fmaxf(mm, buf[i * R + r].x);
    const float mu = mm == -INFINITY ? 0.0f : mm;
    for (int i = 0; i < x.parts; ++i) ll = fmaf(buf[i * R + r].y, pat_exp2(buf[i * R + r].x - mu), ll);
    if (lse) paged_store_lse(p, x.b, x.g, x.r0 + r, mm, ll);
    return make_float2(mu, ll == 0.0f ? 0.0f : 1.0f / ll);
  };
  const float* po = reinterpret_cast<const float*>(p.part_o);
  // four dims of IT rows a thread at a time, so that several parts of each are on their way
  constexpr int IT = 4, ALL = R * (D / 4), C4 = D / 4;
  for (int k0 = 0; k0 < ALL; k0 += IT * PTC_THREADS) {
    float4 a[IT];
    float2 lw[IT];
    int r[IT], c[IT];
#pragma unroll
    for (int u = 0; u < IT; ++u) {
      const int k = k0 + u * PTC_THREADS + tid;
      r[u] = min(k / C4, R - 1), c[u] = k % C4;
      a[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      lw[u] = law(r[u], k < ALL && c[u] == 0);
    }
#pragma unroll 2
    for (int i = 0; i < x.parts; ++i) {
      const float* from = po + slot(i) * R * D;
      float4 v[IT];
#pragma unroll
      for (int u = 0; u < IT; ++u) v[u] = __ldcg(reinterpret_cast<const float4*>(from + r[u] * D) + c[u]);
#pragma unroll
      for (int u = 0; u < IT; ++u) {
        const float w = pat_exp2(buf[i * R + r[u]].x - lw[u].x) * lw[u].y;
        a[u].x = fmaf(v[u].x, w, a[u].x), a[u].y = fmaf(v[u].y, w, a[u].y);
        a[u].z = fmaf(v[u].z, w, a[u].z), a[u].w = fmaf(v[u].w, w, a[u].w);
      }
    }
#pragma unroll
    for (int u = 0; u < IT; ++u)
      if (k0 + u * PTC_THREADS + tid < ALL && x.r0 + r[u] < p.rows)
        *(reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.o) + paged_row(p, x.b, x.g, x.r0 + r[u]) * D) + c[u]) =
            make_uint2(pat_pack<BF>(a[u].x, a[u].y), pat_pack<BF>(a[u].z, a[u].w));
  }
  __syncthreads();
}

// Sum of the values that are not finite, of four dims (from d) of keys lo .. hi - 1, of those
// that row `row` sees or (row < 0) of all: what the dims come to where their sum is not
// finite, since weights are positive (+inf or -inf, NaN where both occur or NaN does; 0:
// there are none).  Off the product's path: eight keys at a time.
template <int D, bool BF>
__device__ __noinline__ float4 ptc_odd_values(const PagedAttnArgs& p, int b, int g, int n, int row, int lo, int hi, int d) {
  constexpr int AT = 8;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j0 = lo; j0 < hi; j0 += AT) {
    int page[AT];
#pragma unroll
    for (int k = 0; k < AT; ++k) page[k] = j0 + k < hi ? p.page_table[b * p.ld_table + p.page_div(j0 + k)] : -1;
    uint2 u[AT];
#pragma unroll
    for (int k = 0; k < AT; ++k) {
      const int j = j0 + k;
      const long long off = page[k] * p.ld_page + g * p.ld_head + (j - p.page_div(j) * p.page_size) * p.ld_tok + d;
      const bool ok = page[k] >= 0 && page[k] < p.num_pages;
      u[k] = ok ? __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p.v_cache) + off)) : make_uint2(0, 0);
    }
#pragma unroll
    for (int k = 0; k < AT; ++k) {
      const uint32_t w[2] = {u[k].x, u[k].y};
      const bool see = row < 0 || paged_visible(p, b, n, j0 + k, row);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t h = w[e / 2] >> (16 * (e & 1)) & 0xffffu;
        const float x = BF ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
        if (see && !isfinite(x)) sum[e] += x;
      }
    }
  }
  return make_float4(sum[0], sum[1], sum[2], sum[3]);
}

template <int D, int R, bool BF>
__global__ void __launch_bounds__(PTC_THREADS, 1) paged_attention_tc_kernel(const __grid_constant__ PtcArgs args) {
  const PagedAttnArgs& p = args.a;
  using S = PtcShape<D, R>;
  constexpr int F = S::F, NS = S::NS, CH = D / 8, KPI = 32 / CH;
  extern __shared__ uint8_t ptc_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ptc_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* own_x = ring + NS * S::TILE;
  float* xm = reinterpret_cast<float*>(own_x + S::X);    // [128] maximum, then [128] sum of a lane
  float* xl = xm + 128;
  uint64_t* bars = reinterpret_cast<uint64_t*>(xl + 128);
  uint64_t *full = bars, *empty = bars + 8, *q_full = bars + 16, *s_full = bars + 18,
           *p_full = bars + 20, *pv_done = bars + 21, *drained = bars + 22;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 23);
  volatile int* abort_flag = reinterpret_cast<int*>(bars + 23) + 1;
  uint32_t* bad = reinterpret_cast<uint32_t*>(bars + 24);  // [4] keys of the unit with values that are not finite
  __shared__ PagedPart s_cut[2];
  __shared__ PagedCut s_range;
  __shared__ bool s_join[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int runs = args.block ? PTC_TK / args.block : 0, loaders = min(4, runs);   // powers of two

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) mbar_init(smem_u32(full + s), args.block ? loaders : 128), mbar_init(smem_u32(empty + s), 1);
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
  PagedPos<PTC_TK> at;
  PagedCut cut;
  tc_fence_before();
  __syncthreads();
  const bool mine = paged_range<PTC_THREADS, PTC_TK>(p, cut, at);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t o_col = tmem + S::O;
  if (mine) {
    const int end = cut.first(blockIdx.x + 1);
    if (tid == 0) s_range = cut;
    if (args.block && warp >= 4 && warp < 4 + loaders) {
      // ================= loads of keys and values by TMA: a lane per `block` tokens of the
      // unit, its runs spread over up to four warps (a warp issues its lanes' boxes one
      // after the other)
      uint32_t slot = 0, phase = 0;
      const int own = runs / loaders, first_key = ((warp - 4) * own + lane) * args.block;
      const uint64_t policy = policy_evict_first();
      if (lane == 0) prefetch_tmap(&args.k), prefetch_tmap(&args.v);
      // the page of the lane's run; one past the last (which loads zeros) where it holds no key
      auto run_page = [&](const PagedPos<PTC_TK>& x) {
        const int key = x.unit * PTC_TK + first_key;
        return lane < own && key < x.n ? p.page_table[x.b * p.ld_table + p.page_div(key)] : p.num_pages;
      };
      int page = run_page(at);
      uint32_t filled = 0, parity = 0;           // tiles with a load in flight, and its phase
      bool ok = true;
      while (ok && at.w < end) {
        if (page < 0 || page > p.num_pages || (page == p.num_pages && lane < own && at.unit * PTC_TK + first_key < at.n)) {
          if (p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
          page = p.num_pages;
        }
        const int now = page, head = at.g, key = at.unit * PTC_TK + first_key, tok = key - p.page_div(key) * p.page_size;
        at.next(p);
        if (at.w < end) page = run_page(at);
        for (int kv = 0; kv < 2; ++kv) {
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(empty + slot), phase ^ 1, abort_flag, p.err));
          if (!ok) break;
          const uint32_t bar = smem_u32(full + slot), dst = smem_u32(ring) + slot * S::TILE + first_key * 128;
          if (lane == 0) mbar_arrive_expect_tx(bar, S::TILE / loaders);
          __syncwarp();
          if (lane < own) {
            const void* map = kv ? &args.v : &args.k;
#pragma unroll
            for (int x = 0; x < D / 64; ++x) ptc_tma(dst + x * 16384, map, bar, x * 64, tok, head, now, policy);
          }
          filled |= 1u << slot;
          parity = (parity & ~(1u << slot)) | (phase << slot);
          if (++slot == NS) slot = 0, phase ^= 1;
        }
      }
      // giving up: no copy may land after the CTA has left (where another warp gave up
      // first, the tile's phase stays open and the wait's limit outlasts the copies)
      if (!ok && lane == 0)
        for (int s = 0; s < NS; ++s)
          if (filled >> s & 1) mbar_wait_drain(smem_u32(full + s), parity >> s & 1, 100000000ull);
      __syncwarp();
    } else if (args.block && warp >= 4 && warp < 8) {
      // no run left for this warp
    } else if (warp >= 4 && warp < 8) {
      // ================= loads by cp.async
      const int lt = tid - 128, lw = warp - 4, kc = lane % CH, khi = lane / CH;
      uint32_t slot = 0, phase = 0;
      // groups of copies that have been issued and not handed over, oldest first
      uint32_t w0 = 0, w1 = 0, w2 = 0;
      int waiting = 0;
      auto flush = [&]() {
        pat_wait<0>();
        fence_proxy_async_smem();
        if (waiting > 0) mbar_arrive(w0);
        if (waiting > 1) mbar_arrive(w1);
        if (waiting > 2) mbar_arrive(w2);
        waiting = 0;
      };
      auto issued = [&](uint32_t bar) {
        pat_commit();
        if (waiting == 3) {
          pat_wait<3>();
          fence_proxy_async_smem();
          mbar_arrive(w0);
          w0 = w1, w1 = w2, w2 = bar;
        } else {
          if (waiting == 0) w0 = bar;
          if (waiting == 1) w1 = bar;
          if (waiting == 2) w2 = bar;
          ++waiting;
        }
      };
      // nothing waits for a free tile while it holds back one that has been filled
      auto wait_for = [&](uint32_t bar, uint32_t parity) {
        bool ok = mbar_try_wait(bar, parity);
        if (!__all_sync(0xffffffffu, ok)) {
          flush();
          ok = mbar_wait(bar, parity, abort_flag, p.err);
        }
        return __all_sync(0xffffffffu, ok) != 0;
      };
      auto key_page = [&](const PagedPos<PTC_TK>& x) {
        const int key = x.unit * PTC_TK + lt;
        return key < x.n ? p.page_table[x.b * p.ld_table + p.page_div(key)] : -1;
      };
      int page = key_page(at);
      // Pages of a multiple of 16 tokens: the warp's keys 0 - 15 and 16 - 31 each lie a
      // fixed distance apart; otherwise each key's place is handed round.
      const bool page16 = p.page_size % 16 == 0;
      const uint32_t lane_dst = ptc_off(lw * 32 + khi, kc);
      while (at.w < end) {
        const int key = at.unit * PTC_TK + lt;
        long long off = -1;
        if (key < at.n) {
          if (page >= 0 && page < p.num_pages)
            off = page * p.ld_page + at.g * p.ld_head + (key - p.page_div(key) * p.page_size) * p.ld_tok;
          else if (p.err)
            atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
        }
        const PagedPos<PTC_TK> cur = at;
        at.next(p);
        if (at.w < end) page = key_page(at);
        long long half[2];                       // keys khi and 16 + khi of the warp, chunk kc
        int live[2];                             // keys of that half that exist, from khi on
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const long long o = __shfl_sync(0xffffffffu, off, 16 * h);
          half[h] = o < 0 ? 0 : o + khi * p.ld_tok + kc * 8;
          live[h] = o < 0 ? 0 : cur.n - (cur.unit * PTC_TK + lw * 32 + 16 * h) - khi;
        }
        auto copy = [&](const void* src) {
          const uint32_t dst = smem_u32(ring) + slot * S::TILE + lane_dst;
          const uint16_t* from = reinterpret_cast<const uint16_t*>(src);
          if (page16) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint16_t* k = from + half[h];
#pragma unroll
              for (int i = 0; i < 16 / KPI; ++i) {
                const bool ok = live[h] > i * KPI;
                pat_cp16((dst ^ ((i * KPI & 7) << 4)) + (16 * h + i * KPI) * 128, ok ? k : from, ok);
                k += KPI * p.ld_tok;
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32 / KPI; ++i) {
              const long long o = __shfl_sync(0xffffffffu, off, i * KPI + khi);
              pat_cp16((dst ^ ((i * KPI & 7) << 4)) + i * KPI * 128, from + (o < 0 ? 0 : o + kc * 8), o >= 0);
            }
          }
          issued(smem_u32(full + slot));
          if (++slot == NS) slot = 0, phase ^= 1;
        };
        if (!wait_for(smem_u32(empty + slot), phase ^ 1)) break;
        copy(p.k_cache);
        if (!wait_for(smem_u32(empty + slot), phase ^ 1)) break;
        copy(p.v_cache);
      }
      flush();
    } else if (warp == 8) {
      // ================= products
      {
        const uint32_t idesc_s = make_idesc_f16(BF, 128, 128);
        const uint32_t idesc_o = make_idesc_f16(BF, 128, D) | (1u << 16);   // V is MN-major
        uint32_t ks = 0, kph = 0, vs = 1, vph = 0, items = 0;
        bool ok = true, first = true, prev_first = true, any = false;
        // operand descriptors of the ring's first tile; addresses in them count 16 bytes
        const uint64_t desc_k = make_sw128_desc(smem_u32(ring)), desc_v = ptc_desc_mn(smem_u32(ring));
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
              ptc_mma(tmem + (n & 1) * 128, tmem + S::Q + kk * 8, kt + (kk >> 2) * 1024 + 2 * (kk & 3), idesc_s, kk > 0);
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
              ptc_mma(o_col, tmem + S::P + kk * 8, vt + kk * 128, idesc_o, kk > 0 || !start);
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
        for (int c = 0; c < 4; ++c) ptc_st16(tmem + S::P + t_lane + c * 16, zero);
      }
      // the queries of a sequence, head and row tile into TMEM, the copies alike
      auto put_queries = [&](int b, int g, int rt) {
        const int r = rt * R + row;
        const bool in = r < p.rows && b < p.B;
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) +
                                                          (in ? paged_row(p, b, g, r) * D : 0));
        uint4 u[D / 8];
#pragma unroll
        for (int c = 0; c < D / 8; ++c) u[c] = in ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float x[16];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint4 y = u[4 * c + e];
            x[4 * e] = __uint_as_float(y.x), x[4 * e + 1] = __uint_as_float(y.y);
            x[4 * e + 2] = __uint_as_float(y.z), x[4 * e + 3] = __uint_as_float(y.w);
          }
          ptc_st16(tmem + S::Q + t_lane + c * 16, x);
        }
        ptc_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(q_full));
      };
      put_queries(at.b, at.g, at.rt);
      float m = -INFINITY, l = 0.0f;       // the maximum in use, unscaled; the sum
      int first_unit = at.unit;
      uint32_t vs = 1, vph = 0;
      bool ok = true;
      auto wait_all = [&](uint64_t* bar, uint32_t parity) {
        return named_bar_and(1, PTC_SOFTMAX, mbar_wait(smem_u32(bar), parity, abort_flag, p.err));
      };
      for (int n = 0; ok && at.w < end; ++n) {
        if (n == 0 || at.unit == 0) {
          first_unit = at.unit;
          m = -INFINITY, l = 0.0f;
        }
        if (!(ok = wait_all(s_full + (n & 1), (n >> 1) & 1))) break;
        tc_fence_after();
        float v[R];
#pragma unroll
        for (int c = 0; c < R / 16; ++c)
          tmem_ld16(tmem + t_lane + (n & 1) * 128 + f * R + c * 16, *reinterpret_cast<float(*)[16]>(v + c * 16));
        tmem_wait_ld();
        if (p.q_sign) {
#pragma unroll
          for (int c = 0; c < R; ++c) v[c] = -v[c];
        }
        const int k0 = at.unit * PTC_TK, key0 = k0 + f * R, base = at.n - p.L;
        const bool edge = k0 + PTC_TK > base;
        uint32_t see[R / 32];
        bool strange = false;
        if (edge) {
          // the lane's keys that its row sees
          const int t = min(p.g_div(at.rt * R + row), p.L - 1);
          const int lim = (p.tail ? min(at.n, base) : min(at.n, base + t + 1)) - key0;
          const uint8_t* tm = p.tail ? p.tail + at.b * p.ldm_b + t * p.ldm_t : nullptr;
#pragma unroll
          for (int w = 0; w < R / 32; ++w) {
            const int k = lim - 32 * w;
            see[w] = k <= 0 ? 0u : k >= 32 ? 0xffffffffu : (1u << k) - 1u;
            if (tm) {
              const int lo = max(0, base - (key0 + 32 * w)), hi = min(32, at.n - (key0 + 32 * w));
#pragma unroll 8
              for (int c = lo; c < hi; ++c) see[w] |= (uint32_t)(tm[key0 + 32 * w + c - base] != 0) << c;
            }
          }
#pragma unroll
          for (int c = 0; c < R; ++c)
            if (!(see[c / 32] >> (c % 32) & 1)) v[c] = -INFINITY;
          // Values past the sequence's end are whatever the page holds: zero.  Of keys that
          // some row may not see, values that are not finite leave the product.
          if (!(ok = wait_all(full + vs, vph))) break;
          uint8_t* vt = ring + vs * S::TILE;
          bool odd = false;
          if (k0 + tid >= base && k0 + tid < at.n) {
            constexpr uint32_t EXP = BF ? 0x7f80u : 0x7c00u;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
              const uint4 u = *reinterpret_cast<const uint4*>(vt + ptc_off(tid, c));
              const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) odd |= (w[k] & EXP) == EXP || ((w[k] >> 16) & EXP) == EXP;
            }
          }
          if (odd || k0 + tid >= at.n) {
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
        for (int c = 0; c < R; ++c) m4[c & 3] = fmaxf(m4[c & 3], v[c]);
        const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        const bool up = m == -INFINITY ? mx > m : (mx - m) * p.scale_log2 > 8.0f;
        float w_old = 1.0f;                      // what the sums so far are scaled by
        if (up) {
          w_old = m == -INFINITY ? 0.0f : pat_exp2((m - mx) * p.scale_log2);
          m = mx;
        }
        const float ms = m == -INFINITY ? 0.0f : m * p.scale_log2;
        float l4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < R; ++c) {
          v[c] = pat_exp2(fmaf(v[c], p.scale_log2, -ms));
          l4[c & 3] += v[c];
        }
        l = fmaf(l, w_old, (l4[0] + l4[1]) + (l4[2] + l4[3]));
        // O of the units before has been summed, P may be written
        if (n > 0 && !(ok = wait_all(pv_done, (n - 1) & 1))) break;
        if (n > 0 && at.unit > first_unit && __any_sync(0xffffffffu, up)) {
          tc_fence_after();
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
          for (int e = 0; e < 16; ++e) x[e] = __uint_as_float(pat_pack<BF>(v[32 * c + 2 * e], v[32 * c + 2 * e + 1]));
          ptc_st16(tmem + S::P + t_lane + f * (R / 2) + c * 16, x);
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
          PagedPos<PTC_TK>::next_rows(p, b, g, rt);
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
            const long long off = page * p.ld_page + at.g * p.ld_head + (j - p.page_div(j) * p.page_size) * p.ld_tok;
#pragma unroll 1
            for (int d = 0; d < D / 16; ++d) {
              float x[16];
              tmem_ld16(o_col + t_lane + d * 16, x);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (on) x[e] = fmaf(w, load_f(p.v_cache, off + d * 16 + e, BF ? 0 : 1), x[e]);
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
          m *= p.scale_log2;
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
          for (int h = 0; h < D / 64; ++h) {
            float x[4][16];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld16(o_col + t_lane + h * 64 + c * 16, x[c]);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 4; ++c) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int q4 = c * 4 + e;
                const float4 a = make_float4(x[c][4 * e] * w, x[c][4 * e + 1] * w, x[c][4 * e + 2] * w, x[c][4 * e + 3] * w);
                if constexpr (F == 1)
                  put(row, h * 16 + q4, a);
                else
                  *reinterpret_cast<float4*>(own_x + ptc_off(tid, q4)) = a;
              }
            }
            if constexpr (F > 1) {
              named_bar_sync(1, PTC_SOFTMAX);
              auto joined = [&](int r, int q4) {
                float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int i = 0; i < F; ++i) {
                  const float4 y = *reinterpret_cast<const float4*>(own_x + ptc_off(i * R + r, q4));
                  a.x += y.x, a.y += y.y, a.z += y.z, a.w += y.w;
                }
                return a;
              };
              float4 nul = make_float4(0.0f, 0.0f, 0.0f, 0.0f);   // NaN where a sum is not finite
#pragma unroll
              for (int k = 0; k < R * 16 / PTC_SOFTMAX; ++k) {
                const int x = tid + k * PTC_SOFTMAX, r = x / 16, q4 = x % 16;
                const float4 a = joined(r, q4);
                nul.x = fmaf(a.x, 0.0f, nul.x), nul.y = fmaf(a.y, 0.0f, nul.y);
                nul.z = fmaf(a.z, 0.0f, nul.z), nul.w = fmaf(a.w, 0.0f, nul.w);
                put(r, h * 16 + q4, a);
              }
              if (isnan((nul.x + nul.y) + (nul.z + nul.w))) {
                // the thread's sums are all of the same four dims: keys before the tail count
                // for every row
                const int d = h * 64 + tid % 16 * 4, lo = first_unit * PTC_TK, hi = min(at.n, (at.unit + 1) * PTC_TK);
                const float4 old = ptc_odd_values<D, BF>(p, at.b, at.g, at.n, -1, lo, min(hi, base), d);
#pragma unroll 1
                for (int r = tid / 16; r < R; r += PTC_SOFTMAX / 16) {
                  bool scored = r0 + r < p.rows;           // NaN scores leave NaN
                  for (int i = 0; i < F; ++i) scored &= !isnan(xl[i * R + r]);
                  if (!scored) continue;
                  const float4 odd = ptc_odd_values<D, BF>(p, at.b, at.g, at.n, r0 + r, max(lo, base), hi, d);
                  const float x[4] = {old.x + odd.x, old.y + odd.y, old.z + odd.z, old.w + odd.w};
                  float4 a = joined(r, tid % 16);
                  a.x = isfinite(a.x) || x[0] == 0.0f ? a.x : x[0], a.y = isfinite(a.y) || x[1] == 0.0f ? a.y : x[1];
                  a.z = isfinite(a.z) || x[2] == 0.0f ? a.z : x[2], a.w = isfinite(a.w) || x[3] == 0.0f ? a.w : x[3];
                  put(r, h * 16 + tid % 16, a);
                }
              }
              __syncwarp();
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
    if (s_join[k]) ptc_join<D, R, BF>(p, s_cut[k], reinterpret_cast<float2*>(ring));
}

}  // namespace simsd
