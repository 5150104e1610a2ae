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
  int T, Hq, Hk, R, page_size;
  PagedDiv page_div;        // by page_size
  float eps;
};

constexpr int PA_THREADS = 128, PA_STAGES = 3, PA_CTAS_PER_SM = 4;

// Two fp32 values in a 64-bit register, worked on by one instruction
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 f2_unpack(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 8 16-bit elements as four pairs of fp32, and back
template <bool BF>
__device__ __forceinline__ void paged_unpack8(uint4 u, uint64_t (&v)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF) {
      v[i] = f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[i] = f2_pack(f.x, f.y);
    }
  }
}
template <bool BF>
__device__ __forceinline__ uint4 paged_pack8(const uint64_t (&v)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = f2_unpack(v[i]);
    if constexpr (BF)
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(f.y), "f"(f.x));
    else
      asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(f.y), "f"(f.x));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void paged_cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// A CTA takes tokens blockIdx.x, + gridDim.x, ...  D / 16 neighbouring threads share
// a head; PA_THREADS is a multiple of that, so a thread keeps its place in the head
// over its heads and its rotary row stays in registers.  The first R / 16 of them
// hold elements 8 j .. 8 j + 7 and their pairs R / 2 further, so the rotation needs
// no exchange; the others hold the 16 next elements of the unrotated rest.
//
// HBM bounds it, with the issue of instructions close behind (hence 16 elements a
// thread and two a multiplication).  Loads run ahead: each thread copies its own
// elements of the next PA_STAGES - 1 tokens into its own places of a ring (cp.async;
// no barrier, since no thread reads another's), and the rotary row is fetched one
// token ahead, the slot and position two.  8192 tokens of 48 heads x 128: 40 us on the
// device in a graph of calls, 5.1 TB/s, 78 % of the measured copy rate (42 us one after the
// other on a stream; loads of one token at a time 50; 8 elements a thread with the pairs
// exchanged by shuffles 70).
template <int D, bool BF>
__global__ void __launch_bounds__(PA_THREADS, PA_CTAS_PER_SM) paged_append_kernel(const PagedAppendArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int LANES = D / 16, HEADS = PA_THREADS / LANES;   // threads of a head, heads at a time
  constexpr int PLANE = PA_THREADS * 16;                      // bytes of one half of HEADS heads
  extern __shared__ __align__(16) uint8_t pa_ring[];          // [PA_STAGES][turns][2][PA_THREADS] x 16 bytes
  const int tid = threadIdx.x, lane = tid & 31;
  const int j = tid % LANES, h_at = tid / LANES;
  const int H = p.Hq + 2 * p.Hk, turns = (H + HEADS - 1) / HEADS;
  const bool pair = 16 * j < p.R;                // this thread's elements are rotated
  const int e0 = pair ? 8 * j : 16 * j, e1 = pair ? p.R / 2 + 8 * j : 16 * j + 8;
  const int stage_bytes = turns * 2 * PLANE;
  const uint32_t place = smem_u32(pa_ring) + tid * 16;

  int ahead = blockIdx.x;                        // the token whose loads come next, and its stage
  uint32_t ahead_at = place;
  auto fetch = [&]() {
    if (ahead < p.T) {
      const uint16_t* src = reinterpret_cast<const uint16_t*>(p.qkv) + ahead * p.ldqkv + h_at * D;
      uint32_t dst = ahead_at;
      for (int h = h_at; h < H; h += HEADS) {
        paged_cp16(dst, src + e0);
        paged_cp16(dst + PLANE, src + e1);
        src += HEADS * D;
        dst += 2 * PLANE;
      }
      ahead += gridDim.x;
      ahead_at += stage_bytes;
      if (ahead_at == place + PA_STAGES * stage_bytes) ahead_at = place;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < PA_STAGES - 1; ++s) fetch();

  struct Place {
    long long slot, pos;
  };
  auto where = [&](int x) { return x < p.T ? Place{p.slots[x], p.positions[x]} : Place{-1, 0}; };
  auto good = [&](const Place& x) { return x.slot >= 0 && x.slot < p.n_slots && x.pos >= 0 && x.pos < p.n_pos; };
  float4 row[4];                                 // the next token's cos and sin
  auto table = [&](const Place& x) {
    if (pair && good(x)) {
      const long long at = x.pos * (p.R / 2) + 8 * j;
      row[0] = __ldg(reinterpret_cast<const float4*>(p.cos + at)), row[1] = __ldg(reinterpret_cast<const float4*>(p.cos + at) + 1);
      row[2] = __ldg(reinterpret_cast<const float4*>(p.sin + at)), row[3] = __ldg(reinterpret_cast<const float4*>(p.sin + at) + 1);
    }
  };
  Place now = where(blockIdx.x), next = where(blockIdx.x + gridDim.x);
  table(now);
  const uint32_t mask = ((1u << LANES) - 1u) << (lane & ~(LANES - 1));
  uint32_t at = 0;                               // this token's stage
  for (int t = blockIdx.x; t < p.T; t += gridDim.x) {
    uint64_t c[4], s[4], ns[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      c[2 * e] = f2_pack(row[e].x, row[e].y), c[2 * e + 1] = f2_pack(row[e].z, row[e].w);
      s[2 * e] = f2_pack(row[2 + e].x, row[2 + e].y), s[2 * e + 1] = f2_pack(row[2 + e].z, row[2 + e].w);
      ns[2 * e] = f2_pack(-row[2 + e].x, -row[2 + e].y), ns[2 * e + 1] = f2_pack(-row[2 + e].z, -row[2 + e].w);
    }
    const bool live = good(now);
    if (!live && now.slot >= 0 && tid == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
    long long base = 0;
    if (live) {
      const long long page = p.n_slots <= 0x7fffffffLL ? p.page_div((int)now.slot) : now.slot / p.page_size;
      base = page * p.ld_page + (now.slot - page * p.page_size) * p.ld_tok;
    }
    now = next;
    table(now);
    next = where(t + 2 * gridDim.x);
    fetch();
    asm volatile("cp.async.wait_group %0;" ::"n"(PA_STAGES - 1) : "memory");
    uint16_t* q = reinterpret_cast<uint16_t*>(p.q_out) + (long long)t * p.Hq * D;
    const uint8_t* from = pa_ring + at + tid * 16;
    for (int h = h_at; h < H; h += HEADS, from += 2 * PLANE) {
      const int kv = h - p.Hq;
      uint4 a = *reinterpret_cast<const uint4*>(from), b = *reinterpret_cast<const uint4*>(from + PLANE);
      if (kv < p.Hk) {                             // q and k; all of a head's threads take the same side
        uint64_t x[4], y[4];
        paged_unpack8<BF>(a, x);
        paged_unpack8<BF>(b, y);
        const uint16_t* w = reinterpret_cast<const uint16_t*>(kv < 0 ? p.qw : p.kw);
        if (w != nullptr) {
          uint64_t sx = 0, sy = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) sx = f2_fma(x[e], x[e], sx), sy = f2_fma(y[e], y[e], sy);
          const float2 s0 = f2_unpack(sx), s1 = f2_unpack(sy);
          float ss = (s0.x + s0.y) + (s1.x + s1.y);
#pragma unroll
          for (int m = LANES / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(mask, ss, m);
          const float inv = rsqrtf(fmaf(ss, 1.0f / D, p.eps));
          const uint64_t inv2 = f2_pack(inv, inv);
          uint64_t wx[4], wy[4];
          paged_unpack8<BF>(__ldg(reinterpret_cast<const uint4*>(w + e0)), wx);
          paged_unpack8<BF>(__ldg(reinterpret_cast<const uint4*>(w + e1)), wy);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = f2_mul(f2_mul(x[e], inv2), wx[e]), y[e] = f2_mul(f2_mul(y[e], inv2), wy[e]);
        }
        if (pair) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint64_t x0 = x[e];
            x[e] = f2_fma(y[e], ns[e], f2_mul(x0, c[e]));
            y[e] = f2_fma(x0, s[e], f2_mul(y[e], c[e]));
          }
        }
        a = paged_pack8<BF>(x);
        b = paged_pack8<BF>(y);
      }
      uint16_t* dst;
      if (kv < 0) {
        dst = q + h * D;
        if (!live) a = b = make_uint4(0, 0, 0, 0);
      } else {
        if (!live) continue;
        dst = kv < p.Hk ? reinterpret_cast<uint16_t*>(p.k_cache) + base + kv * p.ld_head
                        : reinterpret_cast<uint16_t*>(p.v_cache) + base + (kv - p.Hk) * p.ld_head;
      }
      *reinterpret_cast<uint4*>(dst + e0) = a;
      *reinterpret_cast<uint4*>(dst + e1) = b;
    }
    at += stage_bytes;
    if (at == (uint32_t)(PA_STAGES * stage_bytes)) at = 0;
  }
}

}  // namespace simsd
