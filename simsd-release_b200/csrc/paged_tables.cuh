// Page tables and slot maps of a paged cache, built on the device from the
// sequences' lengths.  Free pages are a stack: `free_pages` [P], the lowest
// free_count of them free, taken from the top.
//
// Reserve.  Sequence b has n = lens[b] tokens in h = max(held[b], ceil(n / ps)) pages
// (held[b] where the row has not so many) and is to get c = count[b] (0 .. L) more: t = max(0, ceil((n + c) / ps) - h) pages.
//   T_b = t_0 + .. + t_b;   b is served where t = 0 or T_b <= free_count
// (from the first one that the stack does not reach on, only those that need no page).
// Its i-th new page is free_pages[free_count - 1 - (T_b - t) - i].  Row b of slots and
// positions [B, L] holds the c tokens at its end: positions n .. n + c - 1 and their
// slots; before them, and in a row that is not served, -1 and 0.  No atomics decide
// anything: the same lengths give the same pages.
//
// Release.  Sequence b keeps the pages of keep[b] tokens; its others, r_b =
// held[b] - ceil(keep[b] / ps), go onto the stack, sequence by sequence, each
// sequence's in order.
//
// What bounds them: 16 bytes written a place and the trip to memory and back, three
// times over (lengths, page, store); at a few hundred places it is latency alone.  So
// one launch each: every CTA scans all sequences (a block of 256 at a time) and writes
// its share of the places, and the last one to finish moves the state on that the
// others were reading (held, free_count).
//
// Measured (B200, device time in a graph of calls): reserve and release together 8 - 9.5 us for 32
// sequences x 4 tokens, 12 for 64 prompts of up to 2048 tokens; 13 issued from Python, which is
// the time of the two calls on the host.
#pragma once
#include "paged.cuh"

namespace simsd {

constexpr int PT_THREADS = 256;

struct PagedReserveArgs {
  int* table;               // [B, max_pages], row stride ld_table
  const int* lens;          // [B]
  const int* count;         // [B] or nullptr (L each)
  int* held;                // [B]
  int* free_pages;          // [P]
  int* free_count;          // [1]
  long long* slots;         // [B, L]
  long long* positions;     // [B, L]
  int* total;               // [B]: lens + count, where served
  int* err;
  int* arrived;             // CTAs that are done; zero between calls
  long long ld_table;
  int B, L, max_pages, P, page_size;
  PagedDiv page_div, l_div; // by page_size, by L
};

struct PagedReleaseArgs {
  const int* table;
  int* held;
  int* free_pages;
  int* free_count;
  const int* keep;          // [B] tokens
  int* err;
  int* arrived;
  long long ld_table;
  int B, max_pages, P, page_size;
};

// Inclusive sum of v over the CTA's threads, and the sum of all of them.
__device__ __forceinline__ long long pt_scan(long long v, long long& all) {
  __shared__ long long sums[PT_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, v, m);
    if (lane >= m) v += x;
  }
  __syncthreads();                     // sums of the scan before have been read
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  all = 0;
  long long before = 0;
#pragma unroll
  for (int w = 0; w < PT_THREADS / 32; ++w) {
    if (w < warp) before += sums[w];
    all += sums[w];
  }
  return before + v;
}

// Counts the CTA in, once all its threads are done; true in all of them for the last one.
__device__ __forceinline__ bool pt_last(int* arrived) {
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    last = true;
    if (gridDim.x > 1) {
      __threadfence();
      last = atomicAdd(arrived, 1) == (int)gridDim.x - 1;
      if (last) *arrived = 0;
      __threadfence();
    }
  }
  __syncthreads();
  return last;
}

__device__ __forceinline__ int pt_free(const int* free_count, int P) { return max(0, min(*free_count, P)); }

__global__ void __launch_bounds__(PT_THREADS) paged_reserve_kernel(const PagedReserveArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ int s_len[PT_THREADS], s_new[PT_THREADS], s_have[PT_THREADS];
  __shared__ long long s_at[PT_THREADS];       // what the stack has given to the sequences before
  const int tid = threadIdx.x, free = pt_free(p.free_count, p.P);
  struct Wish {
    int len, fresh, have, take;
    bool served;
  };
  long long before = 0;                        // pages that the sequences of earlier blocks asked for
  auto wish = [&](int b, long long& at) {
    Wish w = {0, 0, 0, 0, true};
    bool short_of = false, bad = false;
    if (b < p.B) {
      const int n = p.lens[b], c = p.count ? p.count[b] : p.L;
      w.len = max(n, 0);
      w.fresh = max(0, min(c, p.L));
      const int mine = (w.len + (long long)p.page_size - 1) / p.page_size;
      const int held = max(0, min(p.held[b], p.max_pages));
      w.have = mine > p.max_pages ? held : max(held, mine);       // tokens past the row: no pages that it has
      const long long need = ((long long)w.len + w.fresh + p.page_size - 1) / p.page_size;
      bad = n < 0;
      short_of = need > p.max_pages;
      w.take = bad || short_of ? 0 : (int)max(0LL, need - w.have);
    }
    long long all;
    const long long upto = before + pt_scan(w.take, all);
    before += all;
    at = upto - w.take;
    if (w.take > 0 && upto > free) short_of = true;
    if (bad || short_of) w.served = false, w.fresh = w.take = 0;
    if (blockIdx.x == 0 && p.err) {
      if (bad) atomicOr(p.err, SIMSD_DEV_ERR_BAD_INDEX);
      if (short_of) atomicOr(p.err, SIMSD_DEV_ERR_CAPACITY);
    }
    return w;
  };
  long long taken = 0;                         // pages handed out, of this thread's sequences
  Wish w;
  for (int base = 0; base < p.B; base += PT_THREADS) {
    long long at;
    w = wish(base + tid, at);
    taken += w.take;
    s_len[tid] = w.len, s_new[tid] = w.fresh, s_have[tid] = w.have, s_at[tid] = at;
    if (blockIdx.x == 0 && base + tid < p.B) p.total[base + tid] = w.len + w.fresh;
    __syncthreads();
    const int places = min(PT_THREADS, p.B - base) * p.L;
    for (int i = blockIdx.x * PT_THREADS + tid; i < places; i += gridDim.x * PT_THREADS) {
      const int k = p.l_div(i), t = i - k * p.L, c = s_new[k];
      long long slot = -1, pos = 0;
      if (t >= p.L - c) {
        const int x = s_len[k] + c - p.L + t, page_at = p.page_div(x), have = s_have[k], in = x - page_at * p.page_size;
        int* entry = p.table + (base + k) * p.ld_table + page_at;
        int page;
        if (page_at < have) {
          page = *entry;
        } else {
          page = p.free_pages[free - 1 - s_at[k] - (page_at - have)];
          if (in == 0) *entry = page;          // a new page's first place
        }
        pos = x;
        slot = page < 0 ? -1 : (long long)page * p.page_size + in;
      }
      p.slots[(long long)base * p.L + i] = slot;
      p.positions[(long long)base * p.L + i] = pos;
    }
    __syncthreads();
  }
  if (!pt_last(p.arrived)) return;
  // nobody reads the state any more
  if (p.B <= PT_THREADS) {
    if (tid < p.B) p.held[tid] = w.have + w.take;
  } else {
    before = 0;
    for (int base = 0; base < p.B; base += PT_THREADS) {
      long long at;
      w = wish(base + tid, at);
      if (base + tid < p.B) p.held[base + tid] = w.have + w.take;
    }
  }
  long long all;
  pt_scan(taken, all);
  if (tid == 0) *p.free_count = free - (int)all;
}

__global__ void __launch_bounds__(PT_THREADS) paged_release_kernel(const PagedReleaseArgs p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int WARPS = PT_THREADS / 32;
  __shared__ int s_keep[PT_THREADS], s_back[PT_THREADS];
  __shared__ long long s_at[PT_THREADS];
  const int tid = threadIdx.x, lane = tid & 31, free = pt_free(p.free_count, p.P);
  long long before = 0;
  int held, keep;
  auto wish = [&](int b, long long& at) {      // pages that go back; none where the stack has no room for them
    held = keep = 0;
    if (b < p.B) {
      held = max(0, min(p.held[b], p.max_pages));
      keep = (int)min((long long)held, ((long long)max(p.keep[b], 0) + p.page_size - 1) / p.page_size);
    }
    const int back = held - keep;
    long long all;
    const long long upto = before + pt_scan(back, all);
    before += all;
    at = upto - back;
    if (back > 0 && free + upto > p.P) {
      if (blockIdx.x == 0 && p.err) atomicOr(p.err, SIMSD_DEV_ERR_CAPACITY);
      return 0;
    }
    return back;
  };
  long long given = 0;
  int back = 0;
  for (int base = 0; base < p.B; base += PT_THREADS) {
    long long at;
    back = wish(base + tid, at);
    given += back;
    s_keep[tid] = keep, s_back[tid] = back, s_at[tid] = at;
    __syncthreads();
    // a warp per sequence
    const int rows = min(PT_THREADS, p.B - base);
    for (int k = blockIdx.x * WARPS + (tid >> 5); k < rows; k += gridDim.x * WARPS)
      for (int i = lane; i < s_back[k]; i += 32)
        p.free_pages[free + s_at[k] + i] = p.table[(base + k) * p.ld_table + s_keep[k] + i];
    __syncthreads();
  }
  if (!pt_last(p.arrived)) return;
  if (p.B <= PT_THREADS) {
    if (tid < p.B) p.held[tid] = held - back;
  } else {
    before = 0;
    for (int base = 0; base < p.B; base += PT_THREADS) {
      long long at;
      back = wish(base + tid, at);
      if (base + tid < p.B) p.held[base + tid] = held - back;
    }
  }
  long long all;
  pt_scan(given, all);
  if (tid == 0) *p.free_count = free + (int)all;
}

}  // namespace simsd
