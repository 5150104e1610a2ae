// What the translation units of the batched serving operators share on the host.
#pragma once
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <utility>

#include "paged_attn.cuh"
#include "simsd_b200.h"

namespace simsd {

constexpr int kMaxDev = 64;
constexpr int kMaxSmem = 227 * 1024;

inline size_t align256(size_t v) { return (v + 255) & ~size_t(255); }
inline long long cdiv(long long a, long long b) { return (a + b - 1) / b; }
inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline int sm_count() {
  const int n = simsd_device_sm_count();
  return n > 0 ? n : 148;
}

// Launch on `s`; as a programmatic dependent of the kernel before it on the
// stream when `dependent` (the second kernel of one call) or SIMSD_LAUNCH_PDL is
// set.  Every kernel here starts with griddepcontrol.wait.
template <typename... KArgs, typename... Args>
int launch_on(void (*kern)(KArgs...), dim3 grid, int block, size_t smem, void* s, bool dependent, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)s;
  cudaLaunchAttribute attr[1];
  if (dependent || (simsd_get_launch_flags() & SIMSD_LAUNCH_PDL)) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  if (cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...) != cudaSuccess) return SIMSD_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? SIMSD_OK : SIMSD_ERR_LAUNCH;
}

inline PagedDiv paged_div(int d) {
  int sh = 0;
  while ((1LL << sh) < d) ++sh;
  return {(uint32_t)(((1ULL << (31 + sh)) + d - 1) / d), 31 + sh};
}

// Raise a kernel's shared-memory limit once per device.
template <typename F>
int allow_smem(F* kern, int bytes, bool* done) {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return SIMSD_ERR_DEVICE;
  static std::mutex mu;
  std::lock_guard<std::mutex> lk(mu);
  if (done[dev]) return SIMSD_OK;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return SIMSD_ERR_LAUNCH;
  done[dev] = true;
  return SIMSD_OK;
}

// Whether no two elements of a tensor that is written meet: rows of `row` elements along
// dimensions of (stride, size), each one reaching past all of the smaller strides together.
inline bool rows_apart(int64_t row, std::initializer_list<std::pair<int64_t, int64_t>> dims) {
  std::pair<int64_t, int64_t> d[4];
  int n = 0;
  for (const auto& x : dims)
    if (x.second > 1) d[n++] = x;
  std::sort(d, d + n);
  for (int i = 0; i < n; ++i) {
    if (d[i].first < row) return false;
    row += (d[i].second - 1) * d[i].first;
  }
  return true;
}

// How paged attention runs the G L rows of a KV head: `nr` rows a CTA, the grid, and the
// workspace: the arrival counters, then two parts per CTA (the end of a sequence
// it started inside, the start of one it leaves unfinished).
struct PagedPlan {
  int nr, grid;
  size_t ml_at, bytes;
};
inline PagedPlan paged_plan_of(int nr, int ctas_per_sm, int D) {
  PagedPlan p;
  p.nr = nr;
  p.grid = std::min(ctas_per_sm * sm_count(), nr > 16 ? PTC_MAX_PARTS : SIMSD_PAGED_COUNTER_BYTES / (int)sizeof(int));
  p.ml_at = SIMSD_PAGED_COUNTER_BYTES + align256((size_t)2 * p.grid * D * p.nr * sizeof(float));
  p.bytes = p.ml_at + align256((size_t)2 * p.grid * p.nr * sizeof(float2));
  return p;
}
// with mma.sync: tiles of 8 or 16 rows
inline PagedPlan paged_plan_tiles(long long rows, int D) { return paged_plan_of(rows <= 8 ? 8 : 16, PAT_CTAS_PER_SM, D); }
// over the 8-bit cache: up to 16 rows with mma.sync in tiles of 8, three CTAs an SM, else tcgen05, whose time hardly goes
// by the rows.  Two tiles and tcgen05 at 9 to 16 rows (us; 128 dims, 8 KV heads): 16 x 1-3k tokens 31 and 46, 32 x
// 0.3-4k 40 and 60, 2 x 64k 79 and 112, 19 x 0-9k in a window of 1000 24 and 31, pages of one token 52 and 59, 1 x 100
// 8.3 and 11.5.  Three at 17 to 24: 41 and 47, 59 and 61, 125 and 113, 34 and 32, 70 and 60, 8.3 and 12.  Four at 32: 51
// and 48, 68 and 63, 141 and 115, 36 and 34, 85 and 61, 8.4 and 13.
inline PagedPlan paged_plan8(long long rows, int D) {
  if (rows <= 16) return paged_plan_of(8, 3, D);
  return paged_plan_of(rows <= 32 ? 32 : rows <= 64 ? 64 : 128, 1, D);
}

// The longest sequence, and the largest window, where there is one (or the form always has one):
// a position less a window, or plus some tokens, stays in 32 bits.
constexpr int PAGED_WINDOW_MAX = 0x40000000;

// A request of paged attention, the sizes that every form of it refuses, and its arguments
// but for what goes by the form: the caches' strides and the plan's part.
inline int paged_attn_request(PagedAttnArgs& a, const void* q, const void* k_cache, const void* v_cache, int num_pages,
                              int page_size, const int32_t* page_table, int64_t ld_table, int max_pages, const int32_t* seq_lens,
                              const uint8_t* tail_mask, int64_t ldm_b, int64_t ldm_t, int B, int L, int Hq, int Hk, int head_dim,
                              float scale, int window, int sinks, void* o, float* lse, int dtype, int* err_word) {
  if (B < 0 || L < 0 || Hq < 1 || Hk < 1 || Hq % Hk || num_pages < 1 || page_size < 1 || max_pages < 0 || window < 0 || sinks < 0)
    return SIMSD_ERR_SHAPE;
  if (dtype != SIMSD_BF16 && dtype != SIMSD_F16) return SIMSD_ERR_DTYPE;
  if (head_dim != 64 && head_dim != 128) return SIMSD_ERR_UNSUPPORTED;
  if (B == 0 || L == 0) return SIMSD_OK;
  const int64_t places = (int64_t)max_pages * page_size;
  if (places > (window > 0 ? PAGED_WINDOW_MAX : 0x7fff0000LL)) return SIMSD_ERR_UNSUPPORTED;
  if (!q || !k_cache || !v_cache || (max_pages > 0 && !page_table) || !seq_lens || !o || ld_table < 0)
    return SIMSD_ERR_SHAPE;
  if (!al16(q) || !al16(o)) return SIMSD_ERR_ALIGN;
  a.q = q;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.page_table = page_table;
  a.seq_lens = seq_lens;
  a.tail = tail_mask;
  a.o = o;
  a.lse = lse;
  a.err = err_word;
  a.ld_table = ld_table;
  a.ldm_b = ldm_b;
  a.ldm_t = ldm_t;
  a.B = B;
  a.L = L;
  a.Hq = Hq;
  a.Hk = Hk;
  a.G = Hq / Hk;
  a.num_pages = num_pages;
  a.page_size = page_size;
  a.max_pages = max_pages;
  a.page_div = paged_div(page_size);
  a.g_div = paged_div(a.G);
  // A window as long as the table hides nothing (j >= 0 > x - window for every position x), and is none: more than 16
  // rows then take the form with tcgen05.  16 x 8-32k tokens, 4 query heads on each of 8, 32 and 128 rows: 404 and
  // 1793 us in the windowed form's tiles of 16, 214 and 380 with tcgen05.
  a.window = window < places ? window : 0;
  a.sinks = std::min(sinks, PAGED_WINDOW_MAX);
  a.q_sign = scale < 0.0f ? 0x80008000u : 0u;
  a.scale_log2 = std::max(std::fabs(scale) * 1.4426950408889634f, 1e-30f);
  a.rows = a.G * L;
  return SIMSD_OK;
}
// A TMA map of a cache for loads of `dims` dims of `block` tokens of one page and head; false
// where the driver will not describe it (a stride of 0, say).
inline bool paged_cache_map(CUtensorMap* m, const void* base, const PagedAttnArgs& a, CUtensorMapDataType type, int size, int D,
                            int dims, int block, CUtensorMapSwizzle swizzle) {
  static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      fn = nullptr;
    }
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  }();
  if (encode == nullptr) return false;
  const cuuint64_t extent[4] = {(cuuint64_t)D, (cuuint64_t)a.page_size, (cuuint64_t)a.Hk, (cuuint64_t)a.num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)a.ld_tok * size, (cuuint64_t)a.ld_head * size, (cuuint64_t)a.ld_page * size};
  const cuuint32_t box[4] = {(cuuint32_t)dims, (cuuint32_t)block, 1, 1}, step[4] = {1, 1, 1, 1};
  if (a.ld_tok <= 0 || a.ld_head <= 0 || a.ld_page <= 0) return false;
  return encode(m, type, 4, const_cast<void*>(base), extent, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// `end`: what a sequence's end weighs in the cut
inline int paged_attn_plan(PagedAttnArgs& a, const PagedPlan& pl, void* workspace, size_t workspace_bytes, int end = PAGED_END_MAX) {
  if (workspace == nullptr || workspace_bytes < pl.bytes) return SIMSD_ERR_WORKSPACE;
  a.row_tiles = (a.rows + pl.nr - 1) / pl.nr;
  if ((long long)a.B * a.Hk * a.row_tiles * ((int64_t)a.max_pages * a.page_size / PAT_TK + 1 + end) > 0x7fffffffLL)
    return SIMSD_ERR_UNSUPPORTED;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  a.arrived = reinterpret_cast<int*>(ws);
  a.part_o = reinterpret_cast<float4*>(ws + SIMSD_PAGED_COUNTER_BYTES);
  a.part_ml = reinterpret_cast<float2*>(ws + pl.ml_at);
  return SIMSD_OK;
}

}  // namespace simsd
