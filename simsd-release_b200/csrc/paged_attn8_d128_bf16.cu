// Attention over the 8-bit cache: heads of 128 dims, bf16 queries.
#define SIMSD_PAGED_ATTN8_FORMS
#include "paged_attn8_run.cuh"

template int simsd::attend8_rows<128, true>(simsd::PagedAttn8Args&, const simsd::PagedPlan&, void*);
