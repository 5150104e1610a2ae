// The append of a paged key-value cache held in 8 bits (the attention that reads it
// is in paged_attn8.cuh).
//
// Keys and values are e4m3 with a scale for each block of `block` tokens and head: the
// number that is stored for x is rn(x / s), and stands for s times that.  Sequence b's
// new tokens are its newest, at positions n - c .. n - 1 (n = seq_lens[b], c = count[b]),
// in the last c of its L rows.  Per block and head that they touch, with a the largest
// finite |x| among the block's new tokens (x: the normed and rotated key, the value; fp32):
//   want = 2^e, the smallest with a <= 448 2^e, e from -64 to 64
//   s    = want where the block's first token is new, else max(the block's scale, want)
// and where s has grown, the block's older tokens are stored anew, rn(stored s_old / s).
// A power of two costs e4m3 no precision but near its smallest numbers, and makes that
// step exact there too.  Values that are not finite are stored as NaN and do not take
// part in a; finite ones past 448 2^64 are stored as 448.
//
// Every (sequence, block, head) is one warp's: no two warps meet in a block, and the
// scale needs no atomics.
#pragma once
#include "paged.cuh"

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
  int kv_tasks, tasks;      // warps' tasks: blocks of keys and values, then rows of queries
  int B, L, Hq, Hk, R, page_size, block, num_pages, max_pages, blocks, chunks;   // blocks of a sequence, row chunks
  float eps;
};

constexpr int PA8_WARPS = 4, PA8_THREADS = PA8_WARPS * 32;
constexpr int PA8_ROWS = 16;          // rows that a warp holds in registers

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

template <int D, bool BF>
__global__ void __launch_bounds__(PA8_THREADS) paged_append8_kernel(const PagedAppend8Args p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int LANES = D / 16, ROWS = 32 / LANES, TURNS = PA8_ROWS / ROWS;   // threads of a row, rows of a warp at a time
  const int lane = threadIdx.x & 31, j = lane % LANES, sub = lane / LANES;
  const uint32_t row_mask = ((1u << LANES) - 1u) << (lane & ~(LANES - 1));
  const bool pair = 16 * j < p.R;                // this thread's elements are rotated
  const int e0 = pair ? 8 * j : 16 * j, e1 = pair ? p.R / 2 + 8 * j : 16 * j + 8;
  const uint16_t* qkv = reinterpret_cast<const uint16_t*>(p.qkv);

  for (uint32_t task = blockIdx.x * PA8_WARPS + (threadIdx.x >> 5); task < (uint32_t)p.tasks; task += gridDim.x * PA8_WARPS) {
    // ---- which rows of which head: keys first, then values, then queries
    const bool kv = task < (uint32_t)p.kv_tasks;
    const uint32_t at = kv ? task : task - p.kv_tasks, heads = kv ? 2 * p.Hk : p.Hq, per = kv ? p.blocks : p.chunks;
    const int h = (int)(at % heads), k = (int)(at / heads % per), b = (int)(at / heads / per);
    const int head = kv ? p.Hq + h : h;
    const bool key = kv && h < p.Hk, turned = !kv || key;
    const int n = max(0, p.seq_lens[b]);
    const int c = min(n, p.count ? max(0, min(p.count[b], p.L)) : p.L);
    // positions past the tables are no places: flagged, not written
    const long long cap = min((long long)p.max_pages * p.page_size, p.n_pos);
    const int top = (int)min((long long)n, cap), old = n - c;
    if (n > top && c > 0 && k == 0 && h == 0 && lane == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
    const int shift = n - p.L;                   // position of row 0
    int lo, hi, block_at = 0;                    // rows t, lo <= t < hi
    if (kv) {
      block_at = (old / p.block + k) * p.block;
      if (block_at >= top || c == 0) continue;
      lo = max(old, block_at) - shift, hi = min(top, block_at + p.block) - shift;
      if (lo >= hi) continue;
    } else {
      lo = k * PA8_ROWS, hi = min(p.L, lo + PA8_ROWS);
    }
    const uint16_t* src = qkv + b * p.ldq_b + (long long)head * D;
    const uint16_t* weight = reinterpret_cast<const uint16_t*>(key ? p.kw : p.qw);
    // rows base .. base + 15 of the head: normed, rotated
    float x[TURNS][16];
    auto fill = [&](int base) {
      uint4 u[TURNS][2];
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int t = base + i * ROWS + sub;
        const bool real = t < hi && t + shift >= old && t + shift < top;
        u[i][0] = u[i][1] = make_uint4(0, 0, 0, 0);
        if (real) {
          u[i][0] = __ldg(reinterpret_cast<const uint4*>(src + t * p.ldq_t + e0));
          u[i][1] = __ldg(reinterpret_cast<const uint4*>(src + t * p.ldq_t + e1));
        }
      }
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        uint64_t v[4], y[4];
        paged_unpack8<BF>(u[i][0], v);
        paged_unpack8<BF>(u[i][1], y);
        if (turned) {
          if (weight != nullptr) {
            uint64_t sx = 0, sy = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) sx = f2_fma(v[e], v[e], sx), sy = f2_fma(y[e], y[e], sy);
            const float2 s0 = f2_unpack(sx), s1 = f2_unpack(sy);
            float ss = (s0.x + s0.y) + (s1.x + s1.y);
#pragma unroll
            for (int m = LANES / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(row_mask, ss, m);
            const float inv = rsqrtf(fmaf(ss, 1.0f / D, p.eps));
            const uint64_t inv2 = f2_pack(inv, inv);
            uint64_t wx[4], wy[4];
            paged_unpack8<BF>(__ldg(reinterpret_cast<const uint4*>(weight + e0)), wx);
            paged_unpack8<BF>(__ldg(reinterpret_cast<const uint4*>(weight + e1)), wy);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = f2_mul(f2_mul(v[e], inv2), wx[e]), y[e] = f2_mul(f2_mul(y[e], inv2), wy[e]);
          }
          const int t = base + i * ROWS + sub;
          if (pair && t < hi && t + shift >= old && t + shift < top) {
            const long long row = (long long)(t + shift) * (p.R / 2) + 8 * j;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const float4 cs = __ldg(reinterpret_cast<const float4*>(p.cos + row) + q);
              const float4 sn = __ldg(reinterpret_cast<const float4*>(p.sin + row) + q);
              const uint64_t c2[2] = {f2_pack(cs.x, cs.y), f2_pack(cs.z, cs.w)};
              const uint64_t s2[2] = {f2_pack(sn.x, sn.y), f2_pack(sn.z, sn.w)};
              const uint64_t n2[2] = {f2_pack(-sn.x, -sn.y), f2_pack(-sn.z, -sn.w)};
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint64_t v0 = v[2 * q + e];
                v[2 * q + e] = f2_fma(y[2 * q + e], n2[e], f2_mul(v0, c2[e]));
                y[2 * q + e] = f2_fma(v0, s2[e], f2_mul(y[2 * q + e], c2[e]));
              }
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 a = f2_unpack(v[e]), d = f2_unpack(y[e]);
          x[i][2 * e] = a.x, x[i][2 * e + 1] = a.y, x[i][8 + 2 * e] = d.x, x[i][8 + 2 * e + 1] = d.y;
        }
      }
    };
    if (!kv) {
      fill(lo);
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int t = lo + i * ROWS + sub;
        if (t >= hi) continue;
        const bool real = t + shift >= old && t + shift < top;
        uint16_t* dst = reinterpret_cast<uint16_t*>(p.q_out) + (((long long)b * p.L + t) * p.Hq + h) * D;
        uint64_t v[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = f2_pack(x[i][2 * e], x[i][2 * e + 1]), y[e] = f2_pack(x[i][8 + 2 * e], x[i][8 + 2 * e + 1]);
        const uint4 nul = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + e0) = real ? paged_pack8<BF>(v) : nul;
        *reinterpret_cast<uint4*>(dst + e1) = real ? paged_pack8<BF>(y) : nul;
      }
      continue;
    }
    // ---- keys or values: the block's page and scale
    const int page = p.page_table[b * p.ld_table + block_at / p.page_size];
    if (page < 0 || page >= p.num_pages) {
      if (h == 0 && lane == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
      continue;
    }
    const int g = key ? h : h - p.Hk, in = block_at % p.page_size;
    uint8_t* cache = (key ? p.k_cache : p.v_cache) + page * p.ld_page + g * p.ld_head + in * p.ld_tok;
    float* scale = (key ? p.k_scale : p.v_scale) + page * p.lds_page + g * p.lds_head + in / p.block * p.lds_block;
    const bool fresh = block_at >= old;
    const float had = fresh ? 0.0f : *scale;
    float a = 0.0f;
    const int last = lo + (hi - lo - 1) / PA8_ROWS * PA8_ROWS;
    for (int base = lo; base <= last; base += PA8_ROWS) {
      fill(base);
#pragma unroll
      for (int i = 0; i < TURNS; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float y = fabsf(x[i][e]);
          a = fmaxf(a, y < INFINITY ? y : 0.0f);
        }
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, m));
    const float s = fmaxf(had, p8_power(p8_exponent(a))), inv = 1.0f / s;
    if (lane == 0) *scale = s;
    // the new tokens; the last rows are still in registers
    for (int base = last; base >= lo; base -= PA8_ROWS) {
      if (base != last) fill(base);
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int t = base + i * ROWS + sub;
        if (t >= hi) continue;
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float z = x[i][4 * q + e];
            y[e] = fabsf(z) < INFINITY ? z * inv : __int_as_float(0x7fffffff);
          }
          w[q] = p8_pack2(y[0], y[1]) | p8_pack2(y[2], y[3]) << 16;
        }
        uint8_t* dst = cache + (t + shift - block_at) * p.ld_tok;
        *reinterpret_cast<uint2*>(dst + e0) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(dst + e1) = make_uint2(w[2], w[3]);
      }
    }
    // the block's older tokens, where the scale has grown
    if (!fresh && s != had) {
      const float ratio = had * inv;
      for (int t = sub; t < old - block_at; t += ROWS) {
        uint4* at16 = reinterpret_cast<uint4*>(cache + t * p.ld_tok + 16 * j);
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
      }
    }
  }
}

}  // namespace simsd
