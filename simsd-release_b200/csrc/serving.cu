// extern "C" entry points of the batched serving operators (declared in
// include/simsd_b200.h): the paged key-value cache and draft verification.
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstring>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <utility>

#include "paged.cuh"
#include "paged_attn.cuh"
#include "paged_attn_tc.cuh"
#include "simsd_b200.h"
#include "spec_verify.cuh"

using namespace simsd;

namespace {

constexpr int kMaxDev = 64;
constexpr int kMaxSmem = 227 * 1024;
std::mutex g_attr_mu;

inline size_t align256(size_t v) { return (v + 255) & ~size_t(255); }
inline long long cdiv(long long a, long long b) { return (a + b - 1) / b; }
inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

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

// 16-byte rows of a paged cache
int cache_check(const void* k, const void* v, int64_t ld_page, int64_t ld_head, int64_t ld_tok) {
  if (!al16(k) || !al16(v) || (ld_page & 7) || (ld_head & 7) || (ld_tok & 7)) return SIMSD_ERR_ALIGN;
  return SIMSD_OK;
}

// What paged attention does with G L rows per KV head: the rows of a CTA (up to 16
// with mma.sync, 32, 64 or 128 with tcgen05; more go in tiles of 128), the grid, and
// the workspace: the arrival counters, then two parts per CTA (the end of a sequence
// it started inside, the start of one it leaves unfinished).
struct PagedPlan {
  int nr, grid;
  size_t ml_at, bytes;
};
PagedPlan paged_plan(int L, int G, int D) {
  PagedPlan p;
  const long long rows = (long long)L * G;
  p.nr = rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
  const int sms = simsd_device_sm_count();
  p.grid = std::min((p.nr <= 16 ? PAT_CTAS_PER_SM : 1) * (sms > 0 ? sms : 148), SIMSD_PAGED_COUNTER_BYTES / (int)sizeof(int));
  p.ml_at = SIMSD_PAGED_COUNTER_BYTES + align256((size_t)2 * p.grid * D * p.nr * sizeof(float));
  p.bytes = p.ml_at + align256((size_t)2 * p.grid * p.nr * sizeof(float2));
  return p;
}

PagedDiv paged_div(int d) {
  int sh = 0;
  while ((1LL << sh) < d) ++sh;
  return {(uint32_t)(((1ULL << (31 + sh)) + d - 1) / d), 31 + sh};
}

// Raise a kernel's shared-memory limit once per device.
template <typename F>
int allow_smem(F* kern, int bytes, bool* done) {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return SIMSD_ERR_DEVICE;
  std::lock_guard<std::mutex> lk(g_attr_mu);
  if (done[dev]) return SIMSD_OK;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return SIMSD_ERR_LAUNCH;
  done[dev] = true;
  return SIMSD_OK;
}

// How verification splits its rows.  A warp takes 4 blocks of 1024 logits where that
// still leaves 32 warps per SM, else one (few rows: latency).  The race runs in about
// four CTAs per SM, each a multiple of SV_CHUNK tokens of one sequence: every CTA of a
// sequence joins its rows' parts anew.
struct SpecPlan {
  int blocks, parts, chunk, chunks;
  size_t cand_at, done_at, bytes;
};
SpecPlan spec_plan(int B, int K, int V) {
  SpecPlan p;
  const int sms = simsd_device_sm_count() > 0 ? simsd_device_sm_count() : 148;
  const long long all = (long long)B * (2 * K + 1) * V;
  p.blocks = all >= (long long)sms * 32 * 4 * SV_BLOCK ? 4 : 1;
  p.parts = (int)cdiv(V, p.blocks * SV_BLOCK);
  p.chunk = (int)std::min<long long>(cdiv(cdiv((long long)B * V, 4 * sms), SV_CHUNK), cdiv(V, SV_CHUNK)) * SV_CHUNK;
  p.chunks = (int)cdiv(V, p.chunk);
  p.cand_at = align256((size_t)B * (2 * K + 1) * p.parts * sizeof(SpecPart));
  p.done_at = p.cand_at + align256((size_t)B * p.chunks * sizeof(float2));
  p.bytes = p.done_at + align256((size_t)B * sizeof(int));
  return p;
}

template <int DT>
int verify_drafts(const SpecVerifyArgs& a, void* stream) {
  const dim3 grid((unsigned)cdiv(a.parts, SV_WARPS), (unsigned)a.B, (unsigned)(a.draft ? 2 * a.K + 1 : a.K + 1));
  int rc = launch_on(spec_stat_kernel<DT>, grid, SV_THREADS, 0, stream, false, a);
  if (rc != SIMSD_OK) return rc;
  return launch_on(spec_draw_kernel<DT>, dim3((unsigned)(a.B * a.chunks)), SV_THREADS, (size_t)(2 * a.K + 1) * sizeof(SpecPart),
                   stream, true, a);
}

template <int D, bool BF>
int append(const PagedAppendArgs& a, void* stream) {
  static bool done[kMaxDev];
  const long long turns = cdiv(a.Hq + 2 * a.Hk, PA_THREADS / (D / 16)), smem = PA_STAGES * turns * 2 * PA_THREADS * 16;
  if (smem > 48 * 1024) {
    const int rc = allow_smem(paged_append_kernel<D, BF>, kMaxSmem, done);
    if (rc != SIMSD_OK) return rc;
  }
  const int sms = simsd_device_sm_count();
  const int grid = std::min(a.T, PA_CTAS_PER_SM * (sms > 0 ? sms : 148));
  return launch_on(paged_append_kernel<D, BF>, dim3((unsigned)grid), PA_THREADS, (size_t)smem, stream, false, a);
}

template <int D, int NT, bool BF>
int attend(const PagedAttnArgs& a, const PagedPlan& pl, void* stream) {
  static bool done[kMaxDev];
  constexpr int smem = PatShape<D, NT>::BYTES;
  const int rc = allow_smem(paged_attention_kernel<D, NT, BF>, smem, done);
  if (rc != SIMSD_OK) return rc;
  return launch_on(paged_attention_kernel<D, NT, BF>, dim3((unsigned)pl.grid), PAT_THREADS, smem, stream, false, a);
}
// A TMA map of a cache for loads of `block` tokens of one page and head; false where
// the driver will not describe it (a stride of 0, say).
bool cache_map(CUtensorMap* m, const void* base, const PagedAttnArgs& a, int D, int block, bool bf) {
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
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)a.page_size, (cuuint64_t)a.Hk, (cuuint64_t)a.num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)a.ld_tok * 2, (cuuint64_t)a.ld_head * 2, (cuuint64_t)a.ld_page * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)block, 1, 1}, step[4] = {1, 1, 1, 1};
  if (a.ld_tok <= 0 || a.ld_head <= 0 || a.ld_page <= 0) return false;
  return encode(m, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims,
                strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int R, bool BF>
int attend_tc(const PagedAttnArgs& a, const PagedPlan& pl, void* stream) {
  static bool done[kMaxDev];
  constexpr int smem = PtcShape<D, R>::BYTES;
  const int rc = allow_smem(paged_attention_tc_kernel<D, R, BF>, smem, done);
  if (rc != SIMSD_OK) return rc;
  PtcArgs t;
  std::memset(&t, 0, sizeof(t));
  t.a = a;
  t.block = std::min(a.page_size & -a.page_size, PTC_TK);
  if (t.block < 8 || !cache_map(&t.k, a.k_cache, a, D, t.block, BF) || !cache_map(&t.v, a.v_cache, a, D, t.block, BF))
    t.block = 0;
  return launch_on(paged_attention_tc_kernel<D, R, BF>, dim3((unsigned)pl.grid), PTC_THREADS, smem, stream, false, t);
}
template <int D, bool BF>
int attend_rows(const PagedAttnArgs& a, const PagedPlan& pl, void* stream) {
  switch (pl.nr) {
    case 8: return attend<D, 1, BF>(a, pl, stream);
    case 16: return attend<D, 2, BF>(a, pl, stream);
    case 32: return attend_tc<D, 32, BF>(a, pl, stream);
    case 64: return attend_tc<D, 64, BF>(a, pl, stream);
    default: return attend_tc<D, 128, BF>(a, pl, stream);
  }
}

}  // namespace

extern "C" {

int simsd_paged_append(const void* qkv, int64_t ldqkv, int T, int Hq, int Hk, int head_dim, int rotary_dim,
                       const void* q_weight, const void* k_weight, float eps, const float* cos, const float* sin,
                       int64_t n_positions, const int64_t* positions, const int64_t* slots, void* q_out, void* k_cache,
                       void* v_cache, int num_pages, int page_size, int64_t ld_page, int64_t ld_head, int64_t ld_tok,
                       int dtype, int* err_word, void* stream) {
  if (T < 0 || Hq < 1 || Hk < 1 || num_pages < 1 || page_size < 1 || n_positions < 1) return SIMSD_ERR_SHAPE;
  if (dtype != SIMSD_BF16 && dtype != SIMSD_F16) return SIMSD_ERR_DTYPE;
  if (head_dim != 64 && head_dim != 128) return SIMSD_ERR_UNSUPPORTED;
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16) return SIMSD_ERR_UNSUPPORTED;
  if ((int64_t)(Hq + 2LL * Hk) * head_dim > 36864) return SIMSD_ERR_UNSUPPORTED;   // its ring in shared memory
  if (T == 0) return SIMSD_OK;
  if (!qkv || (rotary_dim > 0 && (!cos || !sin)) || !positions || !slots || !q_out || !k_cache || !v_cache) return SIMSD_ERR_SHAPE;
  if (ldqkv < (int64_t)(Hq + 2 * Hk) * head_dim) return SIMSD_ERR_SHAPE;
  if (!al16(qkv) || (ldqkv & 7) || !al16(q_out) || !al16(cos) || !al16(sin) || !al16(q_weight) || !al16(k_weight))
    return SIMSD_ERR_ALIGN;
  int rc = cache_check(k_cache, v_cache, ld_page, ld_head, ld_tok);
  if (rc != SIMSD_OK) return rc;
  PagedAppendArgs a;
  a.qkv = qkv;
  a.qw = q_weight;
  a.kw = k_weight;
  a.cos = cos;
  a.sin = sin;
  a.positions = reinterpret_cast<const long long*>(positions);
  a.slots = reinterpret_cast<const long long*>(slots);
  a.q_out = q_out;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.err = err_word;
  a.ldqkv = ldqkv;
  a.n_pos = n_positions;
  a.n_slots = (long long)num_pages * page_size;
  a.ld_page = ld_page;
  a.ld_head = ld_head;
  a.ld_tok = ld_tok;
  a.Hq = Hq;
  a.Hk = Hk;
  a.R = rotary_dim;
  a.page_size = page_size;
  a.page_div = paged_div(page_size);
  a.eps = eps;
  a.T = T;
  if (dtype == SIMSD_BF16) return head_dim == 64 ? append<64, true>(a, stream) : append<128, true>(a, stream);
  return head_dim == 64 ? append<64, false>(a, stream) : append<128, false>(a, stream);
}

size_t simsd_paged_attention_workspace_size(int L, int Hq, int Hk, int head_dim) {
  if (L < 1 || Hq < 1 || Hk < 1 || Hq % Hk || head_dim < 1) return 256;
  return paged_plan(L, Hq / Hk, head_dim).bytes;
}

int simsd_paged_attention(const void* q, const void* k_cache, const void* v_cache, int num_pages, int page_size,
                          int64_t ld_page, int64_t ld_head, int64_t ld_tok, const int32_t* page_table, int64_t ld_table,
                          int max_pages, const int32_t* seq_lens, const uint8_t* tail_mask, int64_t ldm_b, int64_t ldm_t,
                          int B, int L, int Hq, int Hk, int head_dim, float scale, void* o, float* lse, int dtype,
                          void* workspace, size_t workspace_bytes, int* err_word, void* stream) {
  if (B < 0 || L < 0 || Hq < 1 || Hk < 1 || Hq % Hk || num_pages < 1 || page_size < 1 || max_pages < 0)
    return SIMSD_ERR_SHAPE;
  if (dtype != SIMSD_BF16 && dtype != SIMSD_F16) return SIMSD_ERR_DTYPE;
  if (head_dim != 64 && head_dim != 128) return SIMSD_ERR_UNSUPPORTED;
  if (B == 0 || L == 0) return SIMSD_OK;
  if ((int64_t)max_pages * page_size > 0x7fff0000LL) return SIMSD_ERR_UNSUPPORTED;
  if (!q || !k_cache || !v_cache || (max_pages > 0 && !page_table) || !seq_lens || !o || ld_table < 0)
    return SIMSD_ERR_SHAPE;
  if (!al16(q) || !al16(o)) return SIMSD_ERR_ALIGN;
  int rc = cache_check(k_cache, v_cache, ld_page, ld_head, ld_tok);
  if (rc != SIMSD_OK) return rc;
  if (workspace == nullptr || workspace_bytes < simsd_paged_attention_workspace_size(L, Hq, Hk, head_dim))
    return SIMSD_ERR_WORKSPACE;
  PagedAttnArgs a;
  a.q = q;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.page_table = page_table;
  a.seq_lens = seq_lens;
  a.tail = tail_mask;
  a.o = o;
  a.lse = lse;
  a.err = err_word;
  a.ld_page = ld_page;
  a.ld_head = ld_head;
  a.ld_tok = ld_tok;
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
  a.q_sign = scale < 0.0f ? 0x80008000u : 0u;
  a.scale_log2 = std::max(std::fabs(scale) * 1.4426950408889634f, 1e-30f);
  const PagedPlan pl = paged_plan(L, a.G, head_dim);
  a.rows = a.G * L;
  a.row_tiles = (a.rows + pl.nr - 1) / pl.nr;
  if ((long long)B * Hk * a.row_tiles * ((int64_t)max_pages * page_size / PAT_TK + 1 + PAGED_END_MAX) > 0x7fffffffLL)
    return SIMSD_ERR_UNSUPPORTED;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  a.arrived = reinterpret_cast<int*>(ws);
  a.part_o = reinterpret_cast<float4*>(ws + SIMSD_PAGED_COUNTER_BYTES);
  a.part_ml = reinterpret_cast<float2*>(ws + pl.ml_at);
  if (dtype == SIMSD_BF16)
    return head_dim == 64 ? attend_rows<64, true>(a, pl, stream) : attend_rows<128, true>(a, pl, stream);
  return head_dim == 64 ? attend_rows<64, false>(a, pl, stream) : attend_rows<128, false>(a, pl, stream);
}

size_t simsd_speculative_verify_workspace_size(int B, int K, int V) {
  if (B < 1 || K < 0 || V < 1) return 256;
  return spec_plan(B, K, V).bytes;
}

int simsd_speculative_verify(const void* target_logits, int64_t ldt_b, int64_t ldt_r, const void* draft_logits,
                             int64_t ldd_b, int64_t ldd_r, const int64_t* draft_tokens, int64_t ld_x,
                             const float* uniform, int64_t ld_u, const float* noise, int64_t ld_n,
                             const float* temperature, const int32_t* n_draft, int B, int K, int V, int dtype,
                             int64_t* tokens, int64_t* accepted, float* logprobs, void* workspace,
                             size_t workspace_bytes, int* err_word, void* stream) {
  if (B < 0 || K < 0 || V < 1) return SIMSD_ERR_SHAPE;
  if (B > 65535 || K > 1024 || V > 0x7fff0000) return SIMSD_ERR_UNSUPPORTED;
  if (dtype != SIMSD_BF16 && dtype != SIMSD_F16 && dtype != SIMSD_F32) return SIMSD_ERR_DTYPE;
  if (B == 0) return SIMSD_OK;
  if (!target_logits || !noise || !tokens || !accepted || !logprobs) return SIMSD_ERR_SHAPE;
  if (K > 0 && (!draft_tokens || !uniform)) return SIMSD_ERR_SHAPE;
  if (workspace == nullptr || workspace_bytes < simsd_speculative_verify_workspace_size(B, K, V))
    return SIMSD_ERR_WORKSPACE;
  SpecVerifyArgs a;
  a.target = target_logits;
  a.draft = draft_logits;
  a.tokens = reinterpret_cast<const long long*>(draft_tokens);
  a.uniform = uniform;
  a.noise = noise;
  a.temperature = temperature;
  a.n_draft = n_draft;
  a.out_tokens = reinterpret_cast<long long*>(tokens);
  a.out_accepted = reinterpret_cast<long long*>(accepted);
  a.out_logprobs = logprobs;
  const SpecPlan pl = spec_plan(B, K, V);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  if ((long long)B * pl.chunks > 0x7fffffffLL) return SIMSD_ERR_UNSUPPORTED;
  a.part = reinterpret_cast<SpecPart*>(ws);
  a.cand = reinterpret_cast<float2*>(ws + pl.cand_at);
  a.done = reinterpret_cast<int*>(ws + pl.done_at);
  a.blocks = pl.blocks;
  a.parts = pl.parts;
  a.chunk = pl.chunk;
  a.chunks = pl.chunks;
  a.err = err_word;
  a.ldt_b = ldt_b;
  a.ldt_r = ldt_r;
  a.ldd_b = ldd_b;
  a.ldd_r = ldd_r;
  a.ld_x = ld_x;
  a.ld_u = ld_u;
  a.ld_n = ld_n;
  a.B = B;
  a.K = K;
  a.V = V;
  a.dtype = dtype;
  if (dtype == SIMSD_BF16) return verify_drafts<0>(a, stream);
  if (dtype == SIMSD_F16) return verify_drafts<1>(a, stream);
  return verify_drafts<2>(a, stream);
}

}  // extern "C"
