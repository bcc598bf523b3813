// What the kernels for drafted token trees share: a request's numbers, checked against the tensors they point into.
#pragma once

#include "common.cuh"
#include "tree.h"

namespace mb200 {

struct Request {
  int prefix, nodes, row, table;      // row: of node 0; table: row of the request table
};
// A request whose numbers point outside the tensors has no nodes.
__device__ __forceinline__ Request request_of(const TreeIndex& ix, int b, bool* bad) {
  Request r;
  const int seq = __ldcg(ix.seq_lens + b);
  r.prefix = __ldcg(ix.prefix_lens + b);
  r.row = __ldcg(ix.q_start + b);
  r.table = __ldcg(ix.req_pool_indices + b);
  r.nodes = seq - r.prefix;
  if (r.nodes <= 0) {
    r.nodes = 0;
  } else if (r.prefix < 0 || r.row < 0 || r.nodes > ix.rows - r.row || r.table < 0 || r.table >= ix.table_rows || seq > ix.table_cols) {
    r.nodes = 0;
    if (bad != nullptr) *bad = true;
  }
  return r;
}

}  // namespace mb200
