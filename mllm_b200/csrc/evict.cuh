// What the kernels for shortened requests share: a request's numbers, checked against the tensors they point into.
#pragma once

#include "common.cuh"
#include "evict.h"

namespace mb200 {

struct Cached {
  int len, row;       // cached tokens; row of the request table
  bool bad;
};
// A request whose numbers point outside the tensors has no tokens.
__device__ __forceinline__ Cached cached_of(const CacheIndex& ix, int b) {
  Cached r;
  r.len = __ldcg(ix.seq_lens + b);
  r.row = __ldcg(ix.req_pool_indices + b);
  r.bad = r.len > 0 && (r.row < 0 || r.row >= ix.table_rows || r.len > ix.table_cols);
  if (r.len < 0 || r.bad) r.len = 0;
  return r;
}

}  // namespace mb200
