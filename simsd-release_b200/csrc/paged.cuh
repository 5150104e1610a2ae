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
  int Hq, Hk, R, page_size, dtype;
  float eps;
};

constexpr int PA_THREADS = 256, PA_UNROLL = 4;

__device__ __forceinline__ void paged_unpack8(uint4 u, int dtype, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f;
    if (dtype == 0) {
      f.x = __uint_as_float(w[i] << 16);
      f.y = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    }
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 paged_pack8(const float (&f)[8], int dtype) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = (uint32_t)f32_to_16bit(f[2 * i], dtype) | ((uint32_t)f32_to_16bit(f[2 * i + 1], dtype) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One CTA per token.  A head's D elements are D / 8 neighbouring threads of 8
// elements (16-byte loads and stores); PA_THREADS is a multiple of D / 8, so a
// thread keeps its place in the head over its heads and its rotary row stays in
// registers.  The pair of element i lies R / 16 threads away.  HBM bounds it: the
// row's loads (PA_UNROLL vectors a thread at a time) are issued before the slot,
// the position and the rotary row are known, so that one round of latency covers
// them all.
template <int D>
__global__ void __launch_bounds__(PA_THREADS) paged_append_kernel(const PagedAppendArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int LANES = D / 8, HEADS = PA_THREADS / LANES;    // threads of a head, heads at a time
  const long long t = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  const int i8 = tid % LANES, h_at = tid / LANES;
  const int H = p.Hq + 2 * p.Hk;
  const uint16_t* row = reinterpret_cast<const uint16_t*>(p.qkv) + t * p.ldqkv + i8 * 8;
  uint4 raw[PA_UNROLL];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int u = 0; u < PA_UNROLL; ++u) {
      const int h = h0 + u * HEADS + h_at;
      raw[u] = h < H ? __ldg(reinterpret_cast<const uint4*>(row + (long long)h * D)) : make_uint4(0, 0, 0, 0);
    }
  };
  fetch(0);
  const long long slot = p.slots[t];
  const long long pos = p.positions[t];
  auto weight = [&](const void* w) {
    return w ? __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(w) + i8 * 8)) : make_uint4(0, 0, 0, 0);
  };
  const uint4 qw = weight(p.qw), kw = weight(p.kw);
  const bool bad = slot >= p.n_slots || (slot >= 0 && (pos < 0 || pos >= p.n_pos));
  if (bad && tid == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
  const bool live = slot >= 0 && !bad;
  const int rl = p.R / 16;                       // threads of half a rotation
  const bool rot = live && i8 < 2 * rl;
  const bool low = i8 < rl;
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = 1.0f, s[e] = 0.0f;
  if (rot) {
    const long long at = pos * (p.R / 2) + (low ? i8 : i8 - rl) * 8;
    const float4 c0 = *reinterpret_cast<const float4*>(p.cos + at), c1 = *reinterpret_cast<const float4*>(p.cos + at + 4);
    const float4 s0 = *reinterpret_cast<const float4*>(p.sin + at), s1 = *reinterpret_cast<const float4*>(p.sin + at + 4);
    c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
    s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w, s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
    if (low) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = -s[e];
    }
  }
  const int partner = !rot ? lane : low ? lane + rl : lane - rl;
  const long long page = live ? slot / p.page_size : 0;
  const long long base = live ? page * p.ld_page + (slot - page * p.page_size) * p.ld_tok + i8 * 8 : 0;
  uint16_t* q = reinterpret_cast<uint16_t*>(p.q_out) + t * p.Hq * D + i8 * 8;
  for (int h0 = 0; h0 < H; h0 += HEADS * PA_UNROLL) {
    if (h0 > 0) fetch(h0);
#pragma unroll
    for (int u = 0; u < PA_UNROLL; ++u) {
      const int h = h0 + u * HEADS + h_at;
      if (h0 + u * HEADS >= H) break;              // the whole CTA
      float x[8];
      paged_unpack8(raw[u], p.dtype, x);
      const bool is_q = h < p.Hq;
      if (is_q ? p.qw != nullptr : p.kw != nullptr) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
        // the head's threads all take this branch; their lanes are the mask
        const uint32_t mask = (LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u)) << (lane & ~(LANES - 1));
#pragma unroll
        for (int m = LANES / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(mask, ss, m);
        const float inv = rsqrtf(ss * (1.0f / D) + p.eps);
        float wf[8];
        paged_unpack8(is_q ? qw : kw, p.dtype, wf);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * wf[e];
      }
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = __shfl_sync(0xffffffffu, x[e], partner);
        o[e] = rot ? fmaf(other, s[e], x[e] * c[e]) : x[e];
      }
      if (is_q) {
        *reinterpret_cast<uint4*>(q + (long long)h * D) = live ? paged_pack8(o, p.dtype) : make_uint4(0, 0, 0, 0);
      } else if (live && h < H) {
        const bool is_k = h < p.Hq + p.Hk;
        uint16_t* dst = reinterpret_cast<uint16_t*>(is_k ? p.k_cache : p.v_cache) + base +
                        (long long)(h - p.Hq - (is_k ? 0 : p.Hk)) * p.ld_head;
        *reinterpret_cast<uint4*>(dst) = is_k ? paged_pack8(o, p.dtype) : raw[u];
      }
    }
  }
}

}  // namespace simsd
