// The rows that a task of paged_append8 takes; compiles for the host alone too, where lengths
// next to 2^31 are tested.
#pragma once

#ifdef __CUDACC__
#define SIMSD_ROWS_FN __host__ __device__ __forceinline__
#else
#define SIMSD_ROWS_FN inline
#endif

namespace simsd {

// Rows lo .. hi - 1 of a sequence's L, at positions from `at` on (`at` itself is the position of a
// span's first token, before them where that is older); none where lo >= hi.
struct PagedRows8 {
  int at, lo, hi;
};

// Task k of a sequence of n tokens of which the last c are new (0 <= c <= min(n, L)), in spans of
// `span` tokens; positions from `top` on (top <= n) are no places.  A length comes from memory and
// may be any number up to 2^31 - 1, so a span's first position is counted in 64 bits until it is
// known to lie below top.
SIMSD_ROWS_FN PagedRows8 paged_rows8(int n, int c, int top, int L, int span, int k) {
  const int old = n - c, shift = n - L;          // shift: position of row 0
  const long long from = ((long long)(old / span) + k) * span;
  if (from >= top || c == 0) return {0, 0, 0};
  const int at = (int)from;
  return {at, (old > at ? old : at) - shift, (top - at < span ? top : at + span) - shift};
}

}  // namespace simsd
