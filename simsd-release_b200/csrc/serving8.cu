// extern "C" entry points of the paged key-value cache held in 8 bits (declared in
// include/simsd_b200.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>

#include "paged8.cuh"
#include "paged_attn8_run.cuh"
#include "serving_host.cuh"
#include "simsd_b200.h"

using namespace simsd;

namespace {

// 16-byte rows, and blocks that pages are made of
int cache8_check(const void* k, const void* v, int64_t ld_page, int64_t ld_head, int64_t ld_tok, int page_size, int block) {
  if (block < 1 || page_size % block) return SIMSD_ERR_SHAPE;
  if (!al16(k) || !al16(v) || (ld_page & 15) || (ld_head & 15) || (ld_tok & 15)) return SIMSD_ERR_ALIGN;
  return SIMSD_OK;
}

template <int D, bool BF>
int append8(const PagedAppend8Args& a, void* stream) {
  const int grid = (int)std::min<long long>(cdiv(a.tasks, PA8_WARPS), 32LL * sm_count());
  return launch_on(paged_append8_kernel<D, BF>, dim3((unsigned)grid), PA8_THREADS, 0, stream, false, a);
}

}  // namespace

extern "C" {

int simsd_paged_append8(const void* qkv, int64_t ldq_b, int64_t ldq_t, int B, int L, int Hq, int Hk, int head_dim,
                        int rotary_dim, const void* q_weight, const void* k_weight, float eps, const float* cos,
                        const float* sin, int64_t n_positions, const int32_t* page_table, int64_t ld_table, int max_pages,
                        const int32_t* seq_lens, const int32_t* count, void* q_out, void* k_cache, void* v_cache,
                        float* k_scale, float* v_scale, int num_pages, int page_size, int block, int64_t ld_page,
                        int64_t ld_head, int64_t ld_tok, int64_t lds_page, int64_t lds_head, int64_t lds_block, int dtype,
                        int* err_word, void* stream) {
  if (B < 0 || L < 0 || Hq < 1 || Hk < 1 || num_pages < 1 || page_size < 1 || max_pages < 0 || n_positions < 1)
    return SIMSD_ERR_SHAPE;
  if (dtype != SIMSD_BF16 && dtype != SIMSD_F16) return SIMSD_ERR_DTYPE;
  if (head_dim != 64 && head_dim != 128) return SIMSD_ERR_UNSUPPORTED;
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16) return SIMSD_ERR_UNSUPPORTED;
  if (B == 0 || L == 0) return SIMSD_OK;
  if ((int64_t)max_pages * page_size > 0x7fff0000LL || L > 0x40000000) return SIMSD_ERR_UNSUPPORTED;
  if (!qkv || (rotary_dim > 0 && (!cos || !sin)) || (max_pages > 0 && !page_table) || ld_table < 0 || !seq_lens || !q_out ||
      !k_cache || !v_cache || !k_scale || !v_scale)
    return SIMSD_ERR_SHAPE;
  if (ldq_t < (int64_t)(Hq + 2LL * Hk) * head_dim || ldq_b < 0) return SIMSD_ERR_SHAPE;
  if (!al16(qkv) || (ldq_b & 7) || (ldq_t & 7) || !al16(q_out) || !al16(cos) || !al16(sin) || !al16(q_weight) || !al16(k_weight))
    return SIMSD_ERR_ALIGN;
  const int rc = cache8_check(k_cache, v_cache, ld_page, ld_head, ld_tok, page_size, block);
  if (rc != SIMSD_OK) return rc;
  if (!rows_apart(head_dim, {{ld_page, num_pages}, {ld_head, Hk}, {ld_tok, page_size}}) ||
      !rows_apart(1, {{lds_page, num_pages}, {lds_head, Hk}, {lds_block, page_size / block}}))
    return SIMSD_ERR_SHAPE;
  PagedAppend8Args a;
  a.qkv = qkv;
  a.qw = q_weight;
  a.kw = k_weight;
  a.cos = cos;
  a.sin = sin;
  a.page_table = page_table;
  a.seq_lens = seq_lens;
  a.count = count;
  a.q_out = q_out;
  a.k_cache = reinterpret_cast<uint8_t*>(k_cache);
  a.v_cache = reinterpret_cast<uint8_t*>(v_cache);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.err = err_word;
  a.ldq_b = ldq_b;
  a.ldq_t = ldq_t;
  a.n_pos = n_positions;
  a.ld_table = ld_table;
  a.ld_page = ld_page;
  a.ld_head = ld_head;
  a.ld_tok = ld_tok;
  a.lds_page = lds_page;
  a.lds_head = lds_head;
  a.lds_block = lds_block;
  a.B = B;
  a.L = L;
  a.Hq = Hq;
  a.Hk = Hk;
  a.R = rotary_dim;
  a.page_size = page_size;
  a.block = block;
  a.num_pages = num_pages;
  a.max_pages = max_pages;
  a.span = block < PA8_ROWS && PA8_ROWS % block == 0 ? PA8_ROWS : block;
  a.blocks = (int)(((long long)L + a.span - 2) / a.span + 1);   // that L neighbouring tokens can touch
  // queries: as many heads a task, up to 8, as leave every SM 16 warps of them
  a.q_chunks = (int)cdiv(L, 32 / (head_dim / 16));
  a.q_heads = 8;
  while (a.q_heads > 1 && (long long)B * a.q_chunks * cdiv(Hq, a.q_heads) < 16LL * sm_count()) a.q_heads /= 2;
  a.q_groups = (int)cdiv(Hq, a.q_heads);
  a.eps = eps;
  const long long kv = (long long)B * a.blocks * 2 * Hk, all = kv + (long long)B * a.q_chunks * a.q_groups;
  if (all > 0x7fffffffLL) return SIMSD_ERR_UNSUPPORTED;
  a.kv_tasks = (int)kv;
  a.tasks = (int)all;
  if (dtype == SIMSD_BF16) return head_dim == 64 ? append8<64, true>(a, stream) : append8<128, true>(a, stream);
  return head_dim == 64 ? append8<64, false>(a, stream) : append8<128, false>(a, stream);
}

size_t simsd_paged_attention8_workspace_size(int L, int Hq, int Hk, int head_dim) {
  if (L < 1 || Hq < 1 || Hk < 1 || Hq % Hk || head_dim < 1) return 256;
  return paged_plan8((long long)L * (Hq / Hk), head_dim).bytes;
}

int simsd_paged_attention8(const void* q, const void* k_cache, const void* v_cache, const float* k_scale,
                           const float* v_scale, int num_pages, int page_size, int block, int64_t ld_page, int64_t ld_head,
                           int64_t ld_tok, int64_t lds_page, int64_t lds_head, int64_t lds_block,
                           const int32_t* page_table, int64_t ld_table, int max_pages, const int32_t* seq_lens,
                           const uint8_t* tail_mask, int64_t ldm_b, int64_t ldm_t, int B, int L, int Hq, int Hk,
                           int head_dim, float scale, int window, int sinks, void* o, float* lse, int dtype,
                           void* workspace, size_t workspace_bytes, int* err_word, void* stream) {
  PagedAttn8Args t;
  std::memset(&t, 0, sizeof(t));
  PagedAttnArgs& a = t.a;
  int rc = paged_attn_request(a, q, k_cache, v_cache, num_pages, page_size, page_table, ld_table, max_pages, seq_lens, tail_mask,
                              ldm_b, ldm_t, B, L, Hq, Hk, head_dim, scale, window, sinks, o, lse, dtype, err_word);
  if (rc != SIMSD_OK || B == 0 || L == 0) return rc;
  if (!k_scale || !v_scale) return SIMSD_ERR_SHAPE;
  if ((int64_t)max_pages * page_size > PAGED_WINDOW_MAX) return SIMSD_ERR_UNSUPPORTED;
  rc = cache8_check(k_cache, v_cache, ld_page, ld_head, ld_tok, page_size, block);
  if (rc != SIMSD_OK) return rc;
  a.ld_page = ld_page;
  a.ld_head = ld_head;
  a.ld_tok = ld_tok;
  if (scale < 0.0f) a.scale_log2 = -a.scale_log2;          // the sign goes with the scale here
  t.k_scale = k_scale;
  t.v_scale = v_scale;
  t.lds_page = lds_page;
  t.lds_head = lds_head;
  t.lds_block = lds_block;
  t.block_div = paged_div(block);
  const PagedPlan pl = paged_plan8(a.rows, head_dim);
  rc = paged_attn_plan(a, pl, workspace, workspace_bytes, P8_END);
  if (rc != SIMSD_OK) return rc;
  if (dtype == SIMSD_BF16)
    return head_dim == 64 ? attend8_rows<64, true>(t, pl, stream) : attend8_rows<128, true>(t, pl, stream);
  return head_dim == 64 ? attend8_rows<64, false>(t, pl, stream) : attend8_rows<128, false>(t, pl, stream);
}

}  // extern "C"
