// Where the prompt attention over the 4-bit cache finds the copies of a row's pages (cache4.cu makes them, attention_prefill_tc.cuh reads them).
#pragma once

#include "common.cuh"

namespace exl3 {

// Pages lo .. lo + count - 1 of the sequence have their copies at base, base + 1, ...; with `holes`, only those that the block table gives a page
// for, and some page that the row's queries look for has none.
struct FaRow { int lo, count, base, holes; };

// The copy of page j of a sequence whose block table is bt, or -1: beyond the table, or no page of the pool's n_pages there.
__device__ inline int row_copy(const FaRow& r, const int* bt, int n_pages, int j) {
  const int k = j - r.lo;
  if (k < 0 || k >= r.count) return -1;
  if (r.holes) {
    const int page = __ldcg(bt + j);
    if (page < 0 || page >= n_pages) return -1;
  }
  return r.base + k;
}

}  // namespace exl3
