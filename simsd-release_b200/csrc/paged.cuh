// The append of a paged key-value cache (the attention that reads it is in
// paged_attn.cuh).
//
// The cache is [pages, Hk, page size, D] with any page, head and token strides
// (unit D stride), so a head-major and a token-major cache are the same code.
// Slot s is token s % page_size of page s / page_size; sequence b's key j is
// token j % page_size of page page_table[b, j / page_size].  Every offset into
// the cache is 64-bit.
#pragma once
#include "sm100.cuh"

namespace simsd {

// x / d for 0 <= x < 2^31: x * magic >> shift, magic the reciprocal rounded up
struct PagedDiv {
  uint32_t magic;
  int shift;
  __device__ __forceinline__ int operator()(int x) const { return (int)((uint64_t)(uint32_t)x * magic >> shift); }
};

// ---------------------------------------------------------------- append
// Per token t with slot s >= 0 (s < 0: nothing written to the cache, q row zero):
//   n(x)  = w x / sqrt(mean(x^2) + eps)   (q and k heads; w == nullptr: n(x) = x)
//   r(x)  = (x_i c_i - x_{i+R/2} s_i, x_{i+R/2} c_i + x_i s_i) for i < R/2, the
//           rest unchanged; c, s: the rows of the position's table entry
//   q_out[t, h] = r(n(q)), K[s] = r(n(k)), V[s] = v
// in fp32 with one rounding at the end.
struct PagedAppendArgs {
  const void* qkv;        // [T, (Hq + 2 Hk) D], row stride ldqkv
  const void* qw;         // [D] or nullptr
  const void* kw;
  const float* cos;       // [n_pos, R / 2]
  const float* sin;
  const long long* positions;
  const long long* slots;
  void* q_out;            // [T, Hq, D]
  void* k_cache;
  void* v_cache;
  int* err;
  long long ldqkv, n_pos, n_slots, ld_page, ld_head, ld_tok;
  int Hq, Hk, R, page_size;
  PagedDiv page_div;        // by page_size
  float eps;
};

constexpr int PA_THREADS = 256, PA_UNROLL = 4;

template <bool BF>
__device__ __forceinline__ void paged_unpack4(uint2 u, float (&v)[4]) {
  const uint32_t w[2] = {u.x, u.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (BF) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}
template <bool BF>
__device__ __forceinline__ uint2 paged_pack4(const float (&f)[4]) {
  uint2 r;
  if constexpr (BF) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r.x) : "f"(f[1]), "f"(f[0]));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r.y) : "f"(f[3]), "f"(f[2]));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r.x) : "f"(f[1]), "f"(f[0]));
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r.y) : "f"(f[3]), "f"(f[2]));
  }
  return r;
}

// One CTA per token.  D / 8 neighbouring threads share a head; PA_THREADS is a
// multiple of that, so a thread keeps its place in the head over its heads and its
// rotary row and weights stay in registers.  The first R / 8 of them hold elements
// 4 j .. 4 j + 3 and their pairs R / 2 further, so the rotation needs no exchange
// (8-byte loads and stores; a warp's are still whole 128-byte lines); the others
// hold the 8 next elements of the unrotated rest.  HBM bounds it: the row's loads
// (PA_UNROLL heads a thread at a time) are issued before the slot, the position and
// the rotary row are known, so that one round of latency covers them all.
template <int D, bool BF>
__global__ void __launch_bounds__(PA_THREADS, 4) paged_append_kernel(const PagedAppendArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int LANES = D / 8, HEADS = PA_THREADS / LANES;    // threads of a head, heads at a time
  const int t = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  const int j = tid % LANES, h_at = tid / LANES;
  const int H = p.Hq + 2 * p.Hk;
  const bool pair = 8 * j < p.R;                 // this thread's elements are rotated
  const int e0 = pair ? 4 * j : 8 * j, e1 = pair ? p.R / 2 + 4 * j : 8 * j + 4;
  const uint16_t* row = reinterpret_cast<const uint16_t*>(p.qkv) + t * p.ldqkv;
  uint2 lo[PA_UNROLL], hi[PA_UNROLL];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int u = 0; u < PA_UNROLL; ++u) {
      const int h = h0 + u * HEADS + h_at;
      lo[u] = hi[u] = make_uint2(0, 0);
      if (h < H) {
        lo[u] = __ldg(reinterpret_cast<const uint2*>(row + h * D + e0));
        hi[u] = __ldg(reinterpret_cast<const uint2*>(row + h * D + e1));
      }
    }
  };
  fetch(0);
  const long long slot = p.slots[t];
  const long long pos = p.positions[t];
  const bool bad = slot >= p.n_slots || (slot >= 0 && (pos < 0 || pos >= p.n_pos));
  if (bad && tid == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
  const bool live = slot >= 0 && !bad;
  float4 c = make_float4(1.0f, 1.0f, 1.0f, 1.0f), s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (pair && live) {
    const long long at = pos * (p.R / 2) + 4 * j;
    c = __ldg(reinterpret_cast<const float4*>(p.cos + at));
    s = __ldg(reinterpret_cast<const float4*>(p.sin + at));
  }
  long long base = 0;
  if (live) {
    const long long page = p.n_slots <= 0x7fffffffLL ? p.page_div((int)slot) : slot / p.page_size;
    base = page * p.ld_page + (slot - page * p.page_size) * p.ld_tok;
  }
  uint16_t* q = reinterpret_cast<uint16_t*>(p.q_out) + (long long)t * p.Hq * D;
  for (int h0 = 0; h0 < H; h0 += HEADS * PA_UNROLL) {
    if (h0 > 0) fetch(h0);
#pragma unroll
    for (int u = 0; u < PA_UNROLL; ++u) {
      const int h = h0 + u * HEADS + h_at;
      if (h0 + u * HEADS >= H) break;              // the whole CTA
      const int kv = h - p.Hq;
      uint2 a = lo[u], b = hi[u];
      if (kv < p.Hk) {                             // q and k; all of a head's threads take the same side
        float x[4], y[4];
        paged_unpack4<BF>(a, x);
        paged_unpack4<BF>(b, y);
        const uint16_t* w = reinterpret_cast<const uint16_t*>(kv < 0 ? p.qw : p.kw);
        if (w != nullptr) {
          float ss = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; ++e) ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
          const uint32_t mask = ((1u << LANES) - 1u) << (lane & ~(LANES - 1));
#pragma unroll
          for (int m = LANES / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(mask, ss, m);
          const float inv = rsqrtf(fmaf(ss, 1.0f / D, p.eps));
          float wx[4], wy[4];
          paged_unpack4<BF>(__ldg(reinterpret_cast<const uint2*>(w + e0)), wx);
          paged_unpack4<BF>(__ldg(reinterpret_cast<const uint2*>(w + e1)), wy);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = x[e] * inv * wx[e], y[e] = y[e] * inv * wy[e];
        }
        const float cc[4] = {c.x, c.y, c.z, c.w}, sc[4] = {s.x, s.y, s.z, s.w};
        float ox[4], oy[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ox[e] = pair ? fmaf(-y[e], sc[e], x[e] * cc[e]) : x[e];
          oy[e] = pair ? fmaf(x[e], sc[e], y[e] * cc[e]) : y[e];
        }
        a = paged_pack4<BF>(ox);
        b = paged_pack4<BF>(oy);
      }
      uint16_t* dst;
      if (kv < 0) {
        dst = q + h * D;
        if (!live) a = b = make_uint2(0, 0);
      } else {
        if (!live || h >= H) continue;
        dst = kv < p.Hk ? reinterpret_cast<uint16_t*>(p.k_cache) + base + kv * p.ld_head
                        : reinterpret_cast<uint16_t*>(p.v_cache) + base + (kv - p.Hk) * p.ld_head;
      }
      *reinterpret_cast<uint2*>(dst + e0) = a;
      *reinterpret_cast<uint2*>(dst + e1) = b;
    }
  }
}

}  // namespace simsd
