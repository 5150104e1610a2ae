// The launch of attention over the 8-bit cache; its forms are compiled by paged_attn8_*.cu.
#pragma once
#include "paged_attn8_tc.cuh"
#include "serving_host.cuh"

namespace simsd {

template <int D, bool BF>
int attend8_rows(PagedAttn8Args& a, const PagedPlan& pl, void* stream);

#ifdef SIMSD_PAGED_ATTN8_FORMS
template <int D, bool BF, bool WIN, bool TMA>
int attend8(const PagedAttn8Args& a, const PagedPlan& pl, void* stream) {
  static bool done[kMaxDev];
  using S = Pat8Shape<D>;
  const int rc = allow_smem(paged_attention8_kernel<D, BF, WIN, TMA>, S::BYTES, done);
  if (rc != SIMSD_OK) return rc;
  return launch_on(paged_attention8_kernel<D, BF, WIN, TMA>, dim3((unsigned)pl.grid), S::THREADS, S::BYTES, stream, false, a);
}
template <int D, int R, bool BF>
int attend8_tc(PagedAttn8Args& a, const PagedPlan& pl, void* stream) {
  static bool done[kMaxDev];
  constexpr int smem = P8tShape<D, R>::BYTES;
  const int rc = allow_smem(paged_attention8_tc_kernel<D, R, BF>, smem, done);
  if (rc != SIMSD_OK) return rc;
  if (a.a.window == 0) a.a.window = PAGED_WINDOW_MAX, a.a.sinks = 0;       // this form has a window always
  return launch_on(paged_attention8_tc_kernel<D, R, BF>, dim3((unsigned)pl.grid), P8T_THREADS, smem, stream, false, a);
}
template <int D, bool BF>
int attend8_rows(PagedAttn8Args& a, const PagedPlan& pl, void* stream) {
  a.run = std::min(a.a.page_size & -a.a.page_size, 32);
  const CUtensorMapSwizzle swizzle = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if (a.run < 8 || !paged_cache_map(&a.k, a.a.k_cache, a.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, D, D, a.run, swizzle) ||
      !paged_cache_map(&a.v, a.a.v_cache, a.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, D, D, a.run, swizzle))
    a.run = 0;
  switch (pl.nr) {
    case 8: break;
    case 32: return attend8_tc<D, 32, BF>(a, pl, stream);
    case 64: return attend8_tc<D, 64, BF>(a, pl, stream);
    default: return attend8_tc<D, 128, BF>(a, pl, stream);
  }
  if (a.a.window) return a.run ? attend8<D, BF, true, true>(a, pl, stream) : attend8<D, BF, true, false>(a, pl, stream);
  return a.run ? attend8<D, BF, false, true>(a, pl, stream) : attend8<D, BF, false, false>(a, pl, stream);
}
#endif

}  // namespace simsd
