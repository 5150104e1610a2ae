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
// It follows x_j + lv_j, 2^lv_j the power of two above vs_j (lv_j cut to -64 .. 64), so
// scales of very different sizes meet in one sequence; p_j and its sum stay in fp32.
//
// A warp takes 32 keys of a unit of 128.  In an operand of the first product a lane's four
// bytes are four neighbouring dims of a key (the queries' dims are ordered alike); in the
// second, ldmatrix.trans hands a lane two neighbouring dims of two keys, and even and odd
// dims become the upper and lower rows of the product.
//
// A hidden key counts as nothing, whatever its memory or scale holds: its weight is set to
// zero, keys that no row sees are not read, and where a value of a key that some row does
// not see is NaN, the product runs row by row without the keys hidden from it.
#pragma once
#include "paged8.cuh"
#include "paged_attn.cuh"

namespace simsd {

struct PagedAttn8Args {
  PagedAttnArgs a;          // caches: e4m3, strides in bytes
  const float* k_scale;     // [pages, Hk, page_size / block]
  const float* v_scale;
  long long lds_page, lds_head, lds_block;
  PagedDiv block_div;       // by block
};

constexpr int PA8_TK = 32 * PAT_WARPS;

template <int D, int NT>
struct Pat8Shape {
  static constexpr int NR = NT * 8;
  static constexpr int STAGES = 3;
  static constexpr int MAT = 32 * D;                           // 32 keys (or values)
  static constexpr int STAGE = 2 * MAT + 2 * 32 * 4;           // with their scales
  static constexpr int RING = PAT_WARPS * STAGES * STAGE;
  static constexpr int OBUF = PatShape<D, NT>::OBUF;
  static constexpr int ML = 2 * PAT_WARPS * NR * 4;
  static constexpr int BYTES = RING + OBUF + ML;
};

// 4 bytes into shared memory, zeros where !ok
__device__ __forceinline__ void pat8_cp4(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
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

template <int D, int NT, bool BF, bool WIN>
__global__ void __launch_bounds__(PAT_THREADS, PAT_CTAS_PER_SM) paged_attention8_kernel(const __grid_constant__ PagedAttn8Args args) {
  griddep_launch_dependents();
  griddep_wait();
  const PagedAttnArgs& p = args.a;
  using S = Pat8Shape<D, NT>;
  constexpr int NR = S::NR;
  constexpr int MT = D / 16, CH = D / 16;                 // 16-dim tiles, 16-byte chunks of a key
  constexpr int KPI = 32 / CH;                            // keys per cp.async of the warp
  constexpr int QW = MT * NT * 2;                         // words of the queries in a thread
  using Pos = PagedPos<PA8_TK, WIN>;
  extern __shared__ __align__(256) uint8_t pat_smem[];
  __shared__ PagedPart s_cut[2];
  __shared__ bool s_join[2];
  __shared__ PagedCut s_range;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c4 = lane & 3, i8 = lane >> 2;
  const uint32_t ring = smem_u32(pat_smem) + warp * S::STAGES * S::STAGE;
  float4* obuf = reinterpret_cast<float4*>(pat_smem + S::RING);
  float* sm_m = reinterpret_cast<float*>(pat_smem + S::RING + S::OBUF);
  float* sm_l = sm_m + PAT_WARPS * NR;

  Pos ld;
  int end;
  {
    PagedCut cut;
    if (!paged_range<PAT_THREADS, PA8_TK, WIN>(p, cut, ld)) return;
    end = cut.first(blockIdx.x + 1);
    if (tid == 0) s_range = cut;
  }
  if (tid < 2) s_cut[tid].parts = 0, s_join[tid] = false;
  Pos at = ld;

  // ---- loads: the warp's 32 keys of position `ld` into its next ring slot.  Each lane
  // looks up a key's place; pages of a multiple of 16 tokens hold keys 0 - 15 and 16 - 31 a
  // fixed distance apart each, otherwise every key's place is handed round.  The page
  // numbers are fetched a step ahead.
  const bool page16 = p.page_size % 16 == 0;
  const int kc = lane % CH, khi = lane / CH;
  auto fetch_page = [&](const Pos& x) {
    const int key = x.key(p) + warp * 32 + lane;
    return WIN ? paged_page(p, x, key, 1) : key < x.n ? p.page_table[x.b * p.ld_table + p.page_div(key)] : -1;
  };
  int page = fetch_page(ld);
  uint32_t load_slot = ring;
  const uint8_t* kb = reinterpret_cast<const uint8_t*>(p.k_cache);
  const uint8_t* vb = reinterpret_cast<const uint8_t*>(p.v_cache);
  auto load = [&]() {
    if (ld.w < end) {
      const int key0 = ld.key(p) + warp * 32, key = key0 + lane;
      if (key0 < ld.n) {
        long long off = -1, soff = 0;
        if (key < ld.n) {
          if (page >= 0 && page < p.num_pages) {
            const int tok = key - p.page_div(key) * p.page_size;
            off = page * p.ld_page + ld.g * p.ld_head + tok * p.ld_tok;
            soff = page * args.lds_page + ld.g * args.lds_head + args.block_div(tok) * args.lds_block;
          } else if (p.err && !(WIN && page == PAGED_UNSEEN)) {
            atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
          }
        }
        const uint32_t sdst = load_slot + 2 * S::MAT + lane * 4;
        pat8_cp4(sdst, args.k_scale + soff, off >= 0);
        pat8_cp4(sdst + 128, args.v_scale + soff, off >= 0);
        if (page16) {
          // a half's keys that are read: all that lie in its page; those before or after them have no place
          const uint32_t have = __ballot_sync(0xffffffffu, off >= 0);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t mine = have >> 16 * h & 0xffffu;
            const int one = mine ? __ffs(mine) - 1 : 0;         // a key with a place, and the half's first from there
            const long long o = __shfl_sync(0xffffffffu, off, 16 * h + one) - one * p.ld_tok + khi * p.ld_tok + kc * 16;
#pragma unroll
            for (int i = 0; i < 16 / KPI; ++i) {
              const bool ok = mine >> (i * KPI + khi) & 1;
              const long long e = ok ? o + i * KPI * p.ld_tok : 0;
              const uint32_t s = load_slot + pat8_off<D>(16 * h + i * KPI + khi, kc);
              pat_cp16(s, kb + e, ok);
              pat_cp16(s + S::MAT, vb + e, ok);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32 / KPI; ++i) {
            const long long o = __shfl_sync(0xffffffffu, off, i * KPI + khi);
            const long long e = o < 0 ? 0 : o + kc * 16;
            const uint32_t s = load_slot + pat8_off<D>(i * KPI + khi, kc);
            pat_cp16(s, kb + e, o >= 0);
            pat_cp16(s + S::MAT, vb + e, o >= 0);
          }
        }
      }
      load_slot += S::STAGE;
      if (load_slot == ring + S::STAGES * S::STAGE) load_slot = ring;
      ld.next(p);
      if (ld.w < end) page = fetch_page(ld);
    }
    pat_commit();
  };

  // ---- queries of a row tile: the lane's row i8 of each 8, four dims of every 16
  uint2 qnext[NT][MT];
  auto fetch_queries = [&](int b, int g, int rt) {
    const uint16_t* qb = reinterpret_cast<const uint16_t*>(p.q);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = rt * NR + nt * 8 + i8;
      const bool in = r < p.rows && b < p.B;
      const uint16_t* src = qb + (in ? paged_row(p, b, g, r) * D : 0) + 4 * c4;
#pragma unroll
      for (int k = 0; k < MT; ++k)
        qnext[nt][k] = in ? __ldg(reinterpret_cast<const uint2*>(src + k * 16)) : make_uint2(0, 0);
    }
  };
  uint32_t bq[QW];
  float qs[NT][2];                     // scale log2(e) times the power of two that rows 2 c4, 2 c4 + 1 were divided by
  auto take_queries = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float unit = 1.0f;
      if constexpr (BF) {
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < MT; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t w = e ? qnext[nt][k].y : qnext[nt][k].x;
            top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u))));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int ex = max(-100, min(127, (__float_as_int(top) >> 23) - 127)) - 14;
        const float up = p8_power(-ex);
        unit = p8_power(ex);
#pragma unroll
        for (int k = 0; k < MT; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t w = e ? qnext[nt][k].y : qnext[nt][k].x;
            bq[(2 * k + e) * NT + nt] =
                pat_pack<false>(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
          }
      } else {
#pragma unroll
        for (int k = 0; k < MT; ++k) bq[2 * k * NT + nt] = qnext[nt][k].x, bq[(2 * k + 1) * NT + nt] = qnext[nt][k].y;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) qs[nt][e] = __shfl_sync(0xffffffffu, unit, (2 * c4 + e) * 4) * p.scale_log2;
    }
  };
  fetch_queries(at.b, at.g, at.rt);
#pragma unroll
  for (int s = 0; s < S::STAGES - 1; ++s) load();

  // What a lane reads of a tile: rows lane % 16 and chunk lane / 16 of two for the keys; key
  // lane % 32 for the values.  Chunks are stepped by exclusive or.
  const uint32_t k_lane = pat8_off<D>(lane & 15, lane >> 4);
  const uint32_t v_lane = pat8_off<D>(lane, 0);

  float o[MT][NT][4], m[NT][2], l[NT][2];
  int first_unit = at.unit;
  uint32_t slot_at = ring;
  for (bool start = true; at.w < end; start = false) {
    if (start || at.unit == 0) {
      // a new sequence, head or row tile: its queries, and empty sums
      first_unit = at.unit;
      take_queries();
      if (at.w + at.nu - at.unit + at.END < end) {
        int b = at.b, g = at.g, rt = at.rt;
        Pos::next_rows(p, b, g, rt);
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
    const uint32_t ks_base = slot_at, vs_base = ks_base + S::MAT, sc_base = ks_base + 2 * S::MAT;
    slot_at += S::STAGE;
    if (slot_at == ring + S::STAGES * S::STAGE) slot_at = ring;
    const int key0 = at.key(p) + warp * 32;
    if (key0 < at.n) {
      // S^T = K Q^T, keys 16 kt + i8 and + 8
      float s[2][NT][4];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[kt][nt][0] = s[kt][nt][1] = s[kt][nt][2] = s[kt][nt][3] = 0.0f;
#pragma unroll
        for (int k2 = 0; k2 < MT / 2; ++k2) {
          uint32_t r[4];
          pat_ldsm((ks_base + kt * 16 * D + k_lane) ^ (k2 << 5), r);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t a[4] = {p8_half2(r[2 * x] & 0xffffu), p8_half2(r[2 * x + 1] & 0xffffu), p8_half2(r[2 * x] >> 16),
                                   p8_half2(r[2 * x + 1] >> 16)};
            const int k = 2 * k2 + x;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) pat_mma<false>(s[kt][nt], a, bq[2 * k * NT + nt], bq[(2 * k + 1) * NT + nt]);
          }
        }
      }
      const int r0 = at.rt * NR;
      // some key of the 32 may be hidden from some row
      const bool edge = key0 + 32 > at.n - p.L || (WIN && paged_out(p, at.n, key0, 32));
      float vs[2][2], lv[2][2];                            // of keys 16 kt + i8 + 8 e
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t from = sc_base + (kt * 16 + e * 8 + i8) * 4;
          const float ks = pat8_lds(from);
          vs[kt][e] = pat8_lds(from + 128);
          lv[kt][e] = (float)max(-64, min(64, (__float_as_int(vs[kt][e]) >> 23) - 126));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) s[kt][nt][2 * e] *= ks * qs[nt][0], s[kt][nt][2 * e + 1] *= ks * qs[nt][1];
        }
      uint32_t see = 0xffffffffu;
      if (edge) {
        see = 0;
#pragma unroll
        for (int x = 0; x < NT * 8; ++x)
          see |= (uint32_t)paged_visible<WIN>(p, at.b, at.n, key0 + (x >> 2 & 1) * 16 + i8 + (x & 2) * 4,
                                              r0 + (x >> 3) * 8 + 2 * c4 + (x & 1)) << x;
#pragma unroll
        for (int x = 0; x < NT * 8; ++x)
          if (!(see >> x & 1)) s[x >> 2 & 1][x >> 3][x & 3] = -INFINITY;
      }
      // m moves where a weight would pass 2^15
      bool up = false;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[nt][e] = fmaxf(fmaxf(s[0][nt][e] + lv[0][0], s[0][nt][e + 2] + lv[0][1]),
                             fmaxf(s[1][nt][e] + lv[1][0], s[1][nt][e + 2] + lv[1][1]));
          up |= top[nt][e] > m[nt][e] + 15.0f;
        }
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = top[nt][e];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            x = fmaxf(x - 8.0f, m[nt][e]);
            const float f = x == -INFINITY ? 1.0f : pat_exp2(m[nt][e] - x);
            m[nt][e] = x;
            l[nt][e] *= f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) o[mt][nt][e] *= f, o[mt][nt][e + 2] *= f;
          }
      }
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float ms[2] = {m[nt][0] == -INFINITY ? 0.0f : m[nt][0], m[nt][1] == -INFINITY ? 0.0f : m[nt][1]};
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float q = pat_exp2(s[kt][nt][e] - ms[e & 1]);
            l[nt][e & 1] += q;
            w[e] = q * vs[kt][e >> 1];
          }
          if (edge) {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = see >> (nt * 8 + kt * 4 + e) & 1 ? w[e] : 0.0f;
          }
          pb[kt][nt][0] = pat_transpose(pat_pack<false>(w[0], w[1]));
          pb[kt][nt][1] = pat_transpose(pat_pack<false>(w[2], w[3]));
        }
      }
      // O^T += V^T P^T
      bool odd = false;
      if (edge && (p.L > 1 || p.tail)) {   // NaN in a value, of a key that some row does not see?
        for (int x = lane; x < 32 * CH; x += 32) {
          uint32_t w[4];
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(vs_base + x * 16) : "memory");
#pragma unroll
          for (int k = 0; k < 4; ++k) odd |= (((w[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
        }
        odd = __any_sync(0xffffffffu, odd);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t r[4], a[2][4];
        pat_ldsm_t((vs_base + v_lane) ^ (mt << 4), r);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t two = __byte_perm(r[2 * kt + e], 0, 0x3120);      // even dims of both keys, then odd ones
            a[kt][2 * e] = p8_half2(two & 0xffffu), a[kt][2 * e + 1] = p8_half2(two >> 16);
          }
        if (!odd) {
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) pat_mma<false>(o[mt][nt], a[kt], pb[kt][nt][0], pb[kt][nt][1]);
        } else {
          // row by row, the keys hidden from it zeroed
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            for (int y = 0; y < 8; ++y) {
              float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int kt = 0; kt < 2; ++kt) {
                uint32_t z[4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int j = key0 + kt * 16 + 2 * c4 + e * 8, row = r0 + nt * 8 + y;
                  const uint32_t keep = (paged_visible<WIN>(p, at.b, at.n, j, row) ? 0xffffu : 0u) |
                                        (paged_visible<WIN>(p, at.b, at.n, j + 1, row) ? 0xffff0000u : 0u);
                  z[2 * e] = a[kt][2 * e] & keep, z[2 * e + 1] = a[kt][2 * e + 1] & keep;
                }
                pat_mma<false>(d, z, pb[kt][nt][0], pb[kt][nt][1]);
              }
              const bool mine = (y >> 1) == c4;
              if (mine && (y & 1)) o[mt][nt][1] += d[1], o[mt][nt][3] += d[3];
              if (mine && !(y & 1)) o[mt][nt][0] += d[0], o[mt][nt][2] += d[2];
            }
        }
      }
    }
    __syncwarp();
    const bool ends = at.unit + 1 == at.nu;
    if (ends || at.w + 1 >= end)
      paged_finish<D, NT, BF, true>(p, at, ends && first_unit == 0, first_unit == 0 ? 1 : 0, o, m, l, obuf, sm_m, sm_l, s_range,
                                    s_cut, s_join);
    at.next(p);
  }
  paged_leave<D, NT, BF, true>(p, s_cut, s_join, obuf);
}

}  // namespace simsd
