// extern "C" entry points around a batch's state (declared in include/simsd_b200.h): page
// tables and slot maps, and the rules on logits.
#include <cuda_runtime.h>

#include <algorithm>

#include "logit_rules.cuh"
#include "paged_tables.cuh"
#include "serving_host.cuh"
#include "simsd_b200.h"

using namespace simsd;

namespace {

template <int DT>
int adjust(const LogitRulesArgs& a, bool vec, void* stream) {
  const dim3 grid((unsigned)cdiv(a.V, LR_TOKENS * (LR_THREADS / 32)), (unsigned)a.B);
  auto launch = [&](auto kernel) { return launch_on(kernel, grid, LR_THREADS, 0, stream, false, a); };
  if (a.penal) return vec ? launch(logit_rules_kernel<DT, true, true>) : launch(logit_rules_kernel<DT, false, true>);
  return vec ? launch(logit_rules_kernel<DT, true, false>) : launch(logit_rules_kernel<DT, false, false>);
}

}  // namespace

extern "C" {

int simsd_paged_reserve(int32_t* page_table, int64_t ld_table, int max_pages, const int32_t* lens, const int32_t* count,
                        int32_t* held, int32_t* free_pages, int pool_pages, int32_t* free_count, int B, int L,
                        int page_size, int64_t* slots, int64_t* positions, int32_t* total, void* workspace,
                        size_t workspace_bytes, int* err_word, void* stream) {
  if (B < 0 || L < 0 || page_size < 1 || max_pages < 0 || pool_pages < 0 || ld_table < 0) return SIMSD_ERR_SHAPE;
  if (B == 0) return SIMSD_OK;
  if (!lens || !held || !free_count || !total || (max_pages > 0 && !page_table) || (pool_pages > 0 && !free_pages) ||
      (L > 0 && (!slots || !positions)) || !rows_apart(max_pages, {{ld_table, B}}))
    return SIMSD_ERR_SHAPE;
  // places of a block of sequences, and a grid's more, in 32 bits
  if ((int64_t)max_pages * page_size > 0x7fff0000LL || (int64_t)L * PT_THREADS > 0x7f000000LL) return SIMSD_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < SIMSD_PAGED_COUNTER_BYTES) return SIMSD_ERR_WORKSPACE;
  PagedReserveArgs a;
  a.table = page_table;
  a.lens = lens;
  a.count = count;
  a.held = held;
  a.free_pages = free_pages;
  a.free_count = free_count;
  a.slots = reinterpret_cast<long long*>(slots);
  a.positions = reinterpret_cast<long long*>(positions);
  a.total = total;
  a.err = err_word;
  a.arrived = reinterpret_cast<int*>(workspace);
  a.ld_table = ld_table;
  a.B = B;
  a.L = L;
  a.max_pages = max_pages;
  a.P = pool_pages;
  a.page_size = page_size;
  a.page_div = paged_div(page_size);
  a.l_div = paged_div(std::max(L, 1));
  const long long places = (long long)std::min(B, PT_THREADS) * L;
  const int grid = (int)std::max<long long>(1, std::min<long long>(cdiv(places, PT_THREADS), 2LL * sm_count()));
  return launch_on(paged_reserve_kernel, dim3((unsigned)grid), PT_THREADS, 0, stream, false, a);
}

int simsd_paged_release(const int32_t* page_table, int64_t ld_table, int max_pages, int32_t* held, int32_t* free_pages,
                        int pool_pages, int32_t* free_count, const int32_t* keep, int B, int page_size, void* workspace,
                        size_t workspace_bytes, int* err_word, void* stream) {
  if (B < 0 || page_size < 1 || max_pages < 0 || pool_pages < 0 || ld_table < 0) return SIMSD_ERR_SHAPE;
  if (B == 0) return SIMSD_OK;
  if (!held || !free_count || !keep || (max_pages > 0 && !page_table) || (pool_pages > 0 && !free_pages)) return SIMSD_ERR_SHAPE;
  if (workspace == nullptr || workspace_bytes < SIMSD_PAGED_COUNTER_BYTES) return SIMSD_ERR_WORKSPACE;
  PagedReleaseArgs a;
  a.table = page_table;
  a.held = held;
  a.free_pages = free_pages;
  a.free_count = free_count;
  a.keep = keep;
  a.err = err_word;
  a.arrived = reinterpret_cast<int*>(workspace);
  a.ld_table = ld_table;
  a.B = B;
  a.max_pages = max_pages;
  a.P = pool_pages;
  a.page_size = page_size;
  const int grid = (int)std::min<long long>(cdiv(std::min(B, PT_THREADS), PT_THREADS / 32), sm_count());
  return launch_on(paged_release_kernel, dim3((unsigned)grid), PT_THREADS, 0, stream, false, a);
}

int simsd_adjust_logits(const void* logits, int64_t ld_b, int64_t ld_r, void* out, int64_t ldo_b, int64_t ldo_r, int B,
                        int R, int V, int dtype, const int32_t* counts, int64_t ld_counts, const int64_t* drafts,
                        int64_t ld_drafts, const uint32_t* seen, int64_t ld_seen, const float* repetition,
                        const float* presence, const float* frequency, const int32_t* bias_ids, int64_t ld_ids,
                        const float* bias_values, int64_t ld_values, int n_bias, const uint32_t* allowed,
                        int64_t ld_allowed_b, int64_t ld_allowed_r, int* err_word, void* stream) {
  if (B < 0 || R < 0 || V < 1 || n_bias < 0) return SIMSD_ERR_SHAPE;
  if (dtype != SIMSD_BF16 && dtype != SIMSD_F16 && dtype != SIMSD_F32) return SIMSD_ERR_DTYPE;
  if (B > 65535 || V > 0x7fff0000) return SIMSD_ERR_UNSUPPORTED;
  if (B == 0 || R == 0) return SIMSD_OK;
  if (!logits || !out || (n_bias > 0 && (!bias_ids || !bias_values)) || !rows_apart(V, {{ldo_b, B}, {ldo_r, R}}))
    return SIMSD_ERR_SHAPE;
  LogitRulesArgs a;
  a.logits = logits;
  a.out = out;
  a.counts = counts;
  a.drafts = reinterpret_cast<const long long*>(drafts);
  a.seen = seen;
  a.repetition = repetition;
  a.presence = presence;
  a.frequency = frequency;
  a.bias_ids = bias_ids;
  a.bias = bias_values;
  a.allowed = allowed;
  a.err = err_word;
  a.ld_b = ld_b;
  a.ld_r = ld_r;
  a.ldo_b = ldo_b;
  a.ldo_r = ldo_r;
  a.ld_c = ld_counts;
  a.ld_d = ld_drafts;
  a.ld_s = ld_seen;
  a.ld_i = ld_ids;
  a.ld_v = ld_values;
  a.lda_b = ld_allowed_b;
  a.lda_r = ld_allowed_r;
  a.B = B;
  a.R = R;
  a.V = V;
  a.n_bias = n_bias;
  a.penal = repetition || presence || frequency;
  // 16-byte rows of logits and counts, and no row that ends inside a thread's 8 tokens
  const int e = dtype == SIMSD_F32 ? 4 : 2;
  bool vec = V % LR_EACH == 0 && al16(logits) && al16(out);
  for (int64_t ld : {ld_b, ld_r, ldo_b, ldo_r}) vec = vec && ld * e % 16 == 0;
  if (a.penal && counts) vec = vec && al16(counts) && ld_counts % 4 == 0;
  if (dtype == SIMSD_BF16) return adjust<0>(a, vec, stream);
  if (dtype == SIMSD_F16) return adjust<1>(a, vec, stream);
  return adjust<2>(a, vec, stream);
}

int simsd_count_tokens(int32_t* counts, int64_t ld_counts, const int64_t* tokens, int64_t ld_tokens, int B, int N, int V,
                       int* err_word, void* stream) {
  if (B < 0 || N < 0 || V < 1) return SIMSD_ERR_SHAPE;
  if (B == 0 || N == 0) return SIMSD_OK;
  if (!counts || !tokens || !rows_apart(V, {{ld_counts, B}})) return SIMSD_ERR_SHAPE;
  const int grid = (int)std::min<long long>(cdiv((long long)B * N, 256), 8LL * sm_count());
  return launch_on(count_tokens_kernel, dim3((unsigned)grid), 256, 0, stream, false, counts, ld_counts,
                   reinterpret_cast<const long long*>(tokens), ld_tokens, B, N, V, err_word);
}

}  // extern "C"
