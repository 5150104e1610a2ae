// The append of a paged key-value cache held in 8 bits (the attention that reads it
// is in paged_attn8.cuh).
//
// Keys and values are e4m3 with a scale for each block of `block` tokens and head: the
// number that is stored for x is rn(x (1 / s)), and stands for s times that.  The product and the
// reciprocal are fp32: exact for the powers of two that appends make, 2^-23 off at most for an older
// block's other scale, against e4m3's 2^-4.  Sequence b's
// new tokens are its newest, at positions n - c .. n - 1 (n = seq_lens[b], c = count[b]),
// in the last c of its L rows.  Per block and head that they touch, with a the largest
// finite |x| among the block's new tokens (x: the normed and rotated key, the value; fp32):
//   want = 2^e, the smallest with a <= 448 2^e, e from -64 to 64
//   s    = want where the block's first token is new, else max(the block's scale, want)
// and where s has grown, the block's older tokens are stored anew, rn(stored (s_old / s)).
// A power of two costs e4m3 no precision but near its smallest numbers, and makes that
// step exact there too.  Values that are not finite are stored as NaN and do not take
// part in a; finite ones past 448 2^64 are stored as 448.
//
// Every (sequence, block, head) is one warp's: no two warps meet in a block, and the
// scale needs no atomics.
//
// What bounds it is the issue of some half the slots, and the loads that wait for the lengths and
// tables: each element is widened, normed, rotated, compared, scaled and narrowed.  Measured (B200, 32 + 2 x
// 8 heads x 128, bf16, device time in a graph of calls): 4 x 2048 tokens in blocks of 16 41 us, 63 % of
// the bytes' time at the copy rate (51 with a block's rows in registers, of which some spilled, instead of in
// shared memory); blocks of 64 tokens 43, of 8 and of 1 51 and 52, 16 tokens a task.  4 tokens 4.1.  64 dims, blocks of 16 28 (floor 14.4).
#pragma once
#include "paged.cuh"
#include "paged8_rows.cuh"

namespace simsd {

struct PagedAppend8Args {
  const void* qkv;          // [B, L, (Hq + 2 Hk) D], strides ldq_b, ldq_t
  const void* qw;           // [D] or nullptr
  const void* kw;
  const float* cos;         // [n_pos, R / 2]
  const float* sin;
  const int* page_table;    // [B, max_pages]
  const int* seq_lens;      // [B]
  const int* count;         // [B] or nullptr (L each)
  void* q_out;              // [B, L, Hq, D]
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scale;           // [pages, Hk, page_size / block]
  float* v_scale;
  int* err;
  long long ldq_b, ldq_t, n_pos, ld_table, ld_page, ld_head, ld_tok, lds_page, lds_head, lds_block;
  int kv_tasks, tasks;      // warps' tasks: blocks of a key or value head, then rows of some query heads
  int B, L, Hq, Hk, R, page_size, block, num_pages, max_pages, blocks;   // blocks that a sequence's rows can touch
  int q_heads, q_groups, q_chunks;   // query heads of a task, groups of them, groups of rows
  int span;                 // tokens of a task of keys or values: a block, or 16 where blocks are smaller and divide that
  float eps;
};

constexpr int PA8_WARPS = 4, PA8_THREADS = PA8_WARPS * 32;
constexpr int PA8_ROWS = 16;          // rows that a warp holds

// 2^e as a float, e from -126 to 127
__device__ __forceinline__ float p8_power(int e) { return __int_as_float((e + 127) << 23); }
// the smallest e in -64 .. 64 with a <= 448 2^e (a finite, >= 0)
__device__ __forceinline__ int p8_exponent(float a) {
  const int u = __float_as_int(a);
  const int e = (u >> 23) - 127 - 8 + ((u & 0x7fffff) > 0x600000);
  return max(-64, min(64, e));
}
// two numbers as e4m3, the first in the low byte; 448 where larger
__device__ __forceinline__ uint32_t p8_pack2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t p8_half2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}

// A lane's 8 elements x and 8 more y of a row: the norm, over all lanes of the row, and the rotation
// of pairs (x, y)
template <int D, bool BF>
__device__ __forceinline__ void p8_norm(uint64_t (&x)[4], uint64_t (&y)[4], uint32_t row_mask, float eps, const uint64_t (&wx)[4],
                                        const uint64_t (&wy)[4]) {
  uint64_t sx = 0, sy = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) sx = f2_fma(x[e], x[e], sx), sy = f2_fma(y[e], y[e], sy);
  const float2 s0 = f2_unpack(sx), s1 = f2_unpack(sy);
  float ss = (s0.x + s0.y) + (s1.x + s1.y);
#pragma unroll
  for (int m = D / 32; m > 0; m >>= 1) ss += __shfl_xor_sync(row_mask, ss, m);
  const float inv = rsqrtf(fmaf(ss, 1.0f / D, eps));
  const uint64_t inv2 = f2_pack(inv, inv);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = f2_mul(f2_mul(x[e], inv2), wx[e]), y[e] = f2_mul(f2_mul(y[e], inv2), wy[e]);
}
__device__ __forceinline__ void p8_rotate(uint64_t (&x)[4], uint64_t (&y)[4], const uint64_t (&cs)[4], const uint64_t (&sn)[4],
                                          const uint64_t (&ns)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint64_t x0 = x[e];
    x[e] = f2_fma(y[e], ns[e], f2_mul(x0, cs[e]));
    y[e] = f2_fma(x0, sn[e], f2_mul(y[e], cs[e]));
  }
}
struct P8Turn {               // a lane's cos, sin and -sin
  uint64_t c[4], s[4], n[4];
  __device__ __forceinline__ void load(const float* cos, const float* sin, long long at) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(cos + at) + q), b = __ldg(reinterpret_cast<const float4*>(sin + at) + q);
      c[2 * q] = f2_pack(a.x, a.y), c[2 * q + 1] = f2_pack(a.z, a.w);
      s[2 * q] = f2_pack(b.x, b.y), s[2 * q + 1] = f2_pack(b.z, b.w);
      n[2 * q] = f2_pack(-b.x, -b.y), n[2 * q + 1] = f2_pack(-b.z, -b.w);
    }
  }
};

// D / 16 lanes share a row of a head, each with elements 8 j .. 8 j + 7 and their pairs R / 2 further
// (or 16 next to each other of the unrotated rest), so that the rotation needs no exchange.
//
// A task of keys or values is one (sequence, block, head): 16 rows in shared memory (longer blocks
// twice over: for the largest magnitude, then to be stored); blocks of 1, 2, 4 or 8 tokens go 16
// tokens a task.  A task of queries is four (D
// 128) or eight rows of some neighbouring heads: the rotary row and the weight stay in registers over these.
template <int D, bool BF>
__global__ void __launch_bounds__(PA8_THREADS, 4) paged_append8_kernel(const PagedAppend8Args p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int LANES = D / 16, ROWS = 32 / LANES, TURNS = PA8_ROWS / ROWS;   // threads of a row, rows of a warp at a time
  const int lane = threadIdx.x & 31, j = lane % LANES, sub = lane / LANES;
  const uint32_t row_mask = ((1u << LANES) - 1u) << (lane & ~(LANES - 1));
  const bool pair = 16 * j < p.R;                // this thread's elements are rotated
  const int e0 = pair ? 8 * j : 16 * j, e1 = pair ? p.R / 2 + 8 * j : 16 * j + 8;
  const uint16_t* qkv = reinterpret_cast<const uint16_t*>(p.qkv);
  __shared__ float4 rows[PA8_WARPS][TURNS * 4 * 32];   // a warp's rows in fp32, every lane's its own
  __shared__ float row_tops[PA8_WARPS][PA8_ROWS];
  float4* own = rows[threadIdx.x >> 5] + lane;
  float* tops = row_tops[threadIdx.x >> 5];

  for (uint32_t task = blockIdx.x * PA8_WARPS + (threadIdx.x >> 5); task < (uint32_t)p.tasks; task += gridDim.x * PA8_WARPS) {
    // ---- which rows of which heads: keys first, then values, then queries
    const bool kv = task < (uint32_t)p.kv_tasks;
    const uint32_t at = kv ? task : task - p.kv_tasks, heads = kv ? 2 * p.Hk : p.q_groups, per = kv ? p.blocks : p.q_chunks;
    const int h = (int)(at % heads), k = (int)(at / heads % per), b = (int)(at / heads / per);
    const bool key = kv && h < p.Hk;
    const int n = max(0, p.seq_lens[b]);
    const int c = min(n, p.count ? max(0, min(p.count[b], p.L)) : p.L);
    // positions past the tables are no places: flagged, not written
    const long long cap = min((long long)p.max_pages * p.page_size, p.n_pos);
    const int top = (int)min((long long)n, cap), old = n - c;
    const int shift = n - p.L;                   // position of row 0
    const uint16_t* weight = reinterpret_cast<const uint16_t*>(key ? p.kw : p.qw);
    uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0;
    if (weight != nullptr && (key || !kv))
      w0 = __ldg(reinterpret_cast<const uint4*>(weight + e0)), w1 = __ldg(reinterpret_cast<const uint4*>(weight + e1));
    if (!kv) {
      uint64_t wx[4], wy[4];
      paged_unpack8<BF>(w0, wx);
      paged_unpack8<BF>(w1, wy);
      const int t = k * ROWS + sub;
      if (n > top && c > 0 && k == 0 && h == 0 && lane == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
      const bool in = t < p.L, real = in && t + shift >= old && t + shift < top;
      P8Turn turn;
      if (pair && real) turn.load(p.cos, p.sin, (long long)(t + shift) * (p.R / 2) + 8 * j);
      const int h0 = h * p.q_heads, h1 = min(p.Hq, h0 + p.q_heads);
      const uint16_t* src = qkv + b * p.ldq_b + (real ? t : 0) * p.ldq_t + h0 * D;
      uint16_t* dst = reinterpret_cast<uint16_t*>(p.q_out) + (((long long)b * p.L + (in ? t : 0)) * p.Hq + h0) * D;
      // AHEAD heads' loads are on their way
      constexpr int AHEAD = 4;
      uint4 u[AHEAD][2];
      auto fetch = [&](int i, int head) {
        u[i][0] = u[i][1] = make_uint4(0, 0, 0, 0);
        if (real && head < h1) {
          u[i][0] = __ldg(reinterpret_cast<const uint4*>(src + e0)), u[i][1] = __ldg(reinterpret_cast<const uint4*>(src + e1));
        }
        src += D;
      };
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) fetch(i, h0 + i);
      for (int head = h0; head < h1; head += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          if (head + i >= h1) break;
          uint64_t x[4], y[4];
          paged_unpack8<BF>(u[i][0], x);
          paged_unpack8<BF>(u[i][1], y);
          fetch(i, head + i + AHEAD);
          if (weight != nullptr) p8_norm<D, BF>(x, y, row_mask, p.eps, wx, wy);
          if (pair) p8_rotate(x, y, turn.c, turn.s, turn.n);
          if (in) {
            const uint4 nul = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(dst + e0) = real ? paged_pack8<BF>(x) : nul;
            *reinterpret_cast<uint4*>(dst + e1) = real ? paged_pack8<BF>(y) : nul;
          }
          dst += D;
        }
      }
      continue;
    }
    // ---- keys or values: the block's rows t, lo <= t < hi, its page and scale
    const PagedRows8 own_rows = paged_rows8(n, c, top, p.L, p.span, k);
    const int block_at = own_rows.at, lo = own_rows.lo, hi = own_rows.hi;
    if (lo >= hi) continue;
    const uint16_t* src = qkv + b * p.ldq_b + (long long)(p.Hq + h) * D;
    // rows base .. base + 15 into the lane's places of shared memory; the largest magnitudes of its part of
    // each, infinities among them or not (NaN never)
    float peak[TURNS];
    auto fill = [&](int base, bool all) {
      uint4 u[TURNS][2];
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int t = base + i * ROWS + sub;
        u[i][0] = u[i][1] = make_uint4(0, 0, 0, 0);
        if (t >= lo && t < hi) {
          u[i][0] = __ldg(reinterpret_cast<const uint4*>(src + t * p.ldq_t + e0));
          u[i][1] = __ldg(reinterpret_cast<const uint4*>(src + t * p.ldq_t + e1));
        }
      }
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        float a = 0.0f;
        uint64_t x[4], y[4];
        paged_unpack8<BF>(u[i][0], x);
        paged_unpack8<BF>(u[i][1], y);
        if (key) {
          if (weight != nullptr) {
            uint64_t wx[4], wy[4];
            paged_unpack8<BF>(w0, wx);
            paged_unpack8<BF>(w1, wy);
            p8_norm<D, BF>(x, y, row_mask, p.eps, wx, wy);
          }
          const int t = base + i * ROWS + sub;
          if (pair && t >= lo && t < hi) {
            P8Turn turn;
            turn.load(p.cos, p.sin, (long long)(t + shift) * (p.R / 2) + 8 * j);
            p8_rotate(x, y, turn.c, turn.s, turn.n);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float2 x0 = f2_unpack(x[e]), x1 = f2_unpack(x[e + 1]), y0 = f2_unpack(y[e]), y1 = f2_unpack(y[e + 1]);
          own[(i * 4 + e / 2) * 32] = make_float4(x0.x, x0.y, x1.x, x1.y);
          own[(i * 4 + 2 + e / 2) * 32] = make_float4(y0.x, y0.y, y1.x, y1.y);
          if (all) {
            a = fmaxf(fmaxf(a, fabsf(x0.x)), fabsf(x0.y)), a = fmaxf(fmaxf(a, fabsf(x1.x)), fabsf(x1.y));
            a = fmaxf(fmaxf(a, fabsf(y0.x)), fabsf(y0.y)), a = fmaxf(fmaxf(a, fabsf(y1.x)), fabsf(y1.y));
          } else {
            const float w[8] = {x0.x, x0.y, x1.x, x1.y, y0.x, y0.y, y1.x, y1.y};
#pragma unroll
            for (int z = 0; z < 8; ++z) a = fmaxf(a, fabsf(w[z]) < INFINITY ? fabsf(w[z]) : 0.0f);
          }
        }
        peak[i] = a;
      }
    };
    // a row's stored numbers from its fp32 ones
    auto put = [&](int i, uint8_t* dst, float inv, bool infinite) {
      const uint64_t inv2 = f2_pack(inv, inv);
      uint32_t w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 z = own[(i * 4 + q) * 32];
        float2 u = f2_unpack(f2_mul(f2_pack(z.x, z.y), inv2)), v = f2_unpack(f2_mul(f2_pack(z.z, z.w), inv2));
        if (infinite) u.x -= u.x - u.x, u.y -= u.y - u.y, v.x -= v.x - v.x, v.y -= v.y - v.y;   // infinities become NaN
        w[q] = p8_pack2(u.x, u.y) | p8_pack2(v.x, v.y) << 16;
      }
      *reinterpret_cast<uint2*>(dst + e0) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(dst + e1) = make_uint2(w[2], w[3]);
    };
    // a stored row, rounded anew
    auto again = [&](uint8_t* row, float ratio) {
      uint4* at16 = reinterpret_cast<uint4*>(row + 16 * j);
      const uint4 u = *at16;
      uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t h0 = p8_half2(w[q] & 0xffffu), h1 = p8_half2(w[q] >> 16);
        const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
        const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
        w[q] = p8_pack2(f0.x * ratio, f0.y * ratio) | p8_pack2(f1.x * ratio, f1.y * ratio) << 16;
      }
      *at16 = make_uint4(w[0], w[1], w[2], w[3]);
    };
    const int g = key ? h : h - p.Hk;
    uint8_t* caches = (key ? p.k_cache : p.v_cache) + g * p.ld_head;
    float* scales = (key ? p.k_scale : p.v_scale) + g * p.lds_head;
    if (p.span != p.block) {
      // ---- blocks of less than 16 tokens: those of 16 neighbouring tokens together
      const int base = block_at - shift;             // row of the first of them; rows lo .. hi - 1 are new
      fill(base, false);
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        float a = peak[i];
#pragma unroll
        for (int m = LANES / 2; m > 0; m >>= 1) a = fmaxf(a, __shfl_xor_sync(row_mask, a, m));
        if (j == 0) tops[i * ROWS + sub] = a;        // 0 for a row that is none
      }
      __syncwarp();
      float s[TURNS], had[TURNS];
      long long at_page[TURNS];                      // the row's page, or -1
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int r = i * ROWS + sub, t = base + r, pos = t + shift, first = r / p.block * p.block;
        at_page[i] = -1, s[i] = had[i] = 0.0f;
        if (t < lo || t >= hi) continue;
        const int page = p.page_table[b * p.ld_table + pos / p.page_size];
        if (page < 0 || page >= p.num_pages) {
          if (h == 0 && j == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
          continue;
        }
        at_page[i] = page;
        float a = 0.0f;
        for (int q = 0; q < p.block; ++q) a = fmaxf(a, tops[first + q]);
        if (block_at + first < old) had[i] = scales[page * p.lds_page + pos % p.page_size / p.block * p.lds_block];
        s[i] = fmaxf(had[i], p8_power(p8_exponent(a)));
      }
      __syncwarp();                                  // the scales have been read
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int r = i * ROWS + sub, t = base + r, pos = t + shift, first = r / p.block * p.block, in = pos % p.page_size;
        if (at_page[i] < 0) continue;
        uint8_t* row = caches + at_page[i] * p.ld_page + in * p.ld_tok;
        put(i, row, 1.0f / s[i], true);
        if (t != max(lo, base + first)) continue;
        // the block's first new row: its scale, and where that has grown the older tokens
        if (j == 0) scales[at_page[i] * p.lds_page + in / p.block * p.lds_block] = s[i];
        if (block_at + first < old && s[i] != had[i])
          for (int x = block_at + first; x < old; ++x) again(row - (pos - x) * p.ld_tok, had[i] / s[i]);
      }
      __syncwarp();                                  // `tops` has been read
      continue;
    }
    const int page = p.page_table[b * p.ld_table + block_at / p.page_size];
    if (page < 0 || page >= p.num_pages) {
      if (h == 0 && lane == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
      continue;
    }
    const int in = block_at % p.page_size;
    uint8_t* cache = caches + page * p.ld_page + in * p.ld_tok;
    float* scale = scales + page * p.lds_page + in / p.block * p.lds_block;
    const bool fresh = block_at >= old;
    const float had = fresh ? 0.0f : *scale;
    // the largest magnitude; where an infinity is it, once more without those
    const int last = lo + (hi - lo - 1) / PA8_ROWS * PA8_ROWS;
    auto largest = [&](bool all) {
      float a = 0.0f;
      for (int base = lo; base <= last; base += PA8_ROWS) {
        fill(base, all);
#pragma unroll
        for (int i = 0; i < TURNS; ++i) a = fmaxf(a, peak[i]);
      }
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, m));
      return a;
    };
    float a = largest(true);
    const bool infinite = a == INFINITY;
    if (infinite) a = largest(false);
    const float s = fmaxf(had, p8_power(p8_exponent(a))), inv = 1.0f / s;
    __syncwarp();                                    // every lane has read the scale
    if (lane == 0) *scale = s;
    // the new tokens; the last rows are still at hand
    for (int base = last; base >= lo; base -= PA8_ROWS) {
      if (base != last) fill(base, true);
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int t = base + i * ROWS + sub;
        if (t < hi) put(i, cache + (t + shift - block_at) * p.ld_tok, inv, infinite);
      }
    }
    // the block's older tokens, where the scale has grown
    if (!fresh && s != had)
      for (int t = sub; t < old - block_at; t += ROWS) again(cache + t * p.ld_tok, had * inv);
  }
}

}  // namespace simsd
