// Row kernels of drafted token trees: the prologue of attention, and the accepted nodes' cache rows.
#include <algorithm>

#include "tree.cuh"

namespace mb200 {
namespace {

// ---------------------------------------------------------------------------
// Prologue: per head of q and k  y = x / sqrt(mean x^2 + eps) * gain  (without a gain: y = x), then the pairs (i, i + rot / 2) of the first
// rot features turn by position * inv_freq[i], position = cached tokens + ancestors + delta; q goes out, k and v into the node's slot.
//
// A warp takes one node and some of its heads, 16 bytes a lane.  In front of the first row stand: whose node it is (a vote over the
// requests' first rows), the walk to the root (parents of up to 128 nodes in the warp's registers, a shuffle a step) and the slot; angles
// are formed once per warp, in 64 bits and reduced to one turn, since 32 lose a hundredth of a turn at positions of 10^5.  Results are
// rounded once, to the type of what they go into.
//
// Bound by the chain q_start -> lengths -> parents -> slot -> rows for small batches (8 nodes, 16 + 16 heads of 128: 3.2 us, of which a
// launch is 2) and by the rows' bytes for large ones (32 trees of 60 nodes, 32 + 16 heads of 128, e4m3 caches, 42 MB: 15.9 us, 2.7 TB/s:
// a warp's chain is paid for a few rows only).  As many warps a node as fill the card once (hsplit) halve that chain's share.
// ---------------------------------------------------------------------------
struct PrologueParams {
  TreeIndex ix;
  const void* qkv;
  const void* q_gain;
  const void* k_gain;
  const float* inv_freq;
  const int* delta;
  void* q_out;
  void* k_cache;
  void* v_cache;
  int64_t qkv_stride, kv_tok_stride, kv_head_stride, num_slots;
  int hq, hkv, half, hsplit, kv_fmt;
  float eps;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) tree_prologue_kernel(const PrologueParams p) {
  constexpr int V = 8, kLanes = D / V, kHeads = 32 / kLanes, kFreq = D / 64;      // frequencies of a lane
  constexpr int kSteps = 4;
  pdl_launch_dependents();
  pdl_wait_loads();
  const int64_t warp = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5;
  if (warp >= static_cast<int64_t>(p.ix.rows) * p.hsplit) return;
  const int t = static_cast<int>(warp / p.hsplit), part = static_cast<int>(warp - static_cast<int64_t>(t) * p.hsplit);
  const int lane = lane_id(), l = lane % kLanes;
  const int heads = p.hq + 2 * p.hkv, step = p.hsplit * kHeads;
  const T* row = static_cast<const T*>(p.qkv) + t * p.qkv_stride + l * V;
  // four steps' heads at a time, those of the next four on their way meanwhile
  uint4 next[kSteps];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int h = h0 + k * step + lane / kLanes;
      next[k] = h < heads ? __ldcg(reinterpret_cast<const uint4*>(row + static_cast<int64_t>(h) * D)) : make_uint4(0, 0, 0, 0);
    }
  };
  fetch(part * kHeads);
  const int at = l * V;                                     // the lane's first feature
  float freq[kFreq];          // lane i has those of pairs i, i + 32, ..
#pragma unroll
  for (int i = 0; i < kFreq; ++i) freq[i] = lane + 32 * i < p.half ? __ldcg(p.inv_freq + lane + 32 * i) : 0.f;
  uint4 gains[2]{};           // of queries and of keys
  if (p.q_gain != nullptr) gains[0] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.q_gain) + at));
  if (p.k_gain != nullptr) gains[1] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.k_gain) + at));

  // ---- whose node ----
  int b = -1;
  Request r{};
  bool bad = false;
  for (int b0 = 0; b0 < p.ix.batch && b < 0; b0 += 32) {
    Request mine{};
    if (b0 + lane < p.ix.batch) mine = request_of(p.ix, b0 + lane, &bad);
    const unsigned votes = __ballot_sync(0xffffffffu, mine.nodes > 0 && t >= mine.row && t < mine.row + mine.nodes);
    if (votes != 0) {
      const int from = __ffs(votes) - 1;
      b = b0 + from;
      r.prefix = __shfl_sync(0xffffffffu, mine.prefix, from);
      r.nodes = __shfl_sync(0xffffffffu, mine.nodes, from);
      r.row = __shfl_sync(0xffffffffu, mine.row, from);
      r.table = __shfl_sync(0xffffffffu, mine.table, from);
    }
  }
  if (bad && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
  if (b < 0) {                  // a row of no request: zeros
    for (int h = part * kHeads + lane / kLanes; h < p.hq; h += step)
      *reinterpret_cast<uint4*>(static_cast<T*>(p.q_out) + (static_cast<int64_t>(t) * p.hq + h) * D + at) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int node = t - r.row;
  const int slot = __ldcg(p.ix.req_to_token + r.table * p.ix.table_stride + r.prefix + node);
  const int delta = p.delta != nullptr ? __ldcg(p.delta + b) : 0;
  const bool slot_ok = slot >= 0 && slot < p.num_slots;
  // ---- the way to the root ----
  int up[4], depth = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = i * 32 + lane;
    up[i] = j <= node ? __ldcg(p.ix.parents + r.row + j) : -1;
  }
  bool tree_ok = true;
  for (int j = node;;) {
    int parent;
    if (j < 128) {
      parent = -1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int x = __shfl_sync(0xffffffffu, up[i], j & 31);
        if (j >> 5 == i) parent = x;
      }
    } else {
      parent = __ldcg(p.ix.parents + r.row + j);
    }
    if (parent < 0 || parent >= j) {
      tree_ok = tree_ok && parent == -1;
      break;
    }
    ++depth;
    j = parent;
  }
  if ((!slot_ok || !tree_ok) && part == 0 && lane == 0 && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);

  // ---- sines and cosines of the part of a turn that is left of pos * freq, in half turns ----
  float c[kFreq], s[kFreq];
  const double pos = static_cast<double>(r.prefix) + depth + delta;
#pragma unroll
  for (int i = 0; i < kFreq; ++i) {
    const double angle = pos * static_cast<double>(freq[i]) * 0.15915494309189535;         // in turns: 1 / (2 pi)
    sincospif(2.f * static_cast<float>(angle - rint(angle)), &s[i], &c[i]);
  }
  float cs[V], sn[V];
  const bool turns = at < 2 * p.half, second = at >= p.half;
  const int f0 = second ? at - p.half : at;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    cs[i] = 1.f;
    sn[i] = 0.f;
#pragma unroll
    for (int k = 0; k < kFreq; ++k) {
      const float ck = __shfl_sync(0xffffffffu, c[k], (f0 + i) & 31), sk = __shfl_sync(0xffffffffu, s[k], (f0 + i) & 31);
      if (turns && (f0 + i) >> 5 == k) {
        cs[i] = ck;
        sn[i] = second ? sk : -sk;      // first half: x cos - partner sin; second half: x cos + partner sin
      }
    }
  }
  const int partner = turns ? (second ? lane - p.half / V : lane + p.half / V) : lane;
  for (int first = part * kHeads; first < heads; first += kSteps * step) {
    uint4 now[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) now[k] = next[k];
    if (first + kSteps * step < heads) fetch(first + kSteps * step);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int h0 = first + k * step, h = h0 + lane / kLanes;
      if (h0 >= heads) break;
      uint4 raw = now[k];
      const bool is_q = h < p.hq, is_k = !is_q && h < p.hq + p.hkv;
      T* e = reinterpret_cast<T*>(&raw);
      float y[V];
  #pragma unroll
      for (int i = 0; i < V; ++i) y[i] = to_f32(e[i]);
      if (h0 < p.hq + p.hkv) {             // the warp has a head to norm and turn
        float ss = 0.f;
  #pragma unroll
        for (int i = 0; i < V; ++i) ss += y[i] * y[i];
  #pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const bool normed = (is_q ? p.q_gain : p.k_gain) != nullptr && (is_q || is_k);
        const uint4 gain = is_q ? gains[0] : gains[1];
        const T* g = reinterpret_cast<const T*>(&gain);
        const float rstd = normed ? rsqrtf(ss / static_cast<float>(D) + p.eps) : 1.f;
  #pragma unroll
        for (int i = 0; i < V; ++i) {
          const float x = normed ? y[i] * rstd * to_f32(g[i]) : y[i];
          const float other = __shfl_sync(0xffffffffu, x, partner);
          if (is_q || is_k) y[i] = turns ? x * cs[i] + other * sn[i] : x;
        }
      }
      if (is_q) {
  #pragma unroll
        for (int i = 0; i < V; ++i) e[i] = from_f32<T>(y[i]);
        *reinterpret_cast<uint4*>(static_cast<T*>(p.q_out) + (static_cast<int64_t>(t) * p.hq + h) * D + at) = raw;
      } else if (h < heads && slot_ok) {
        void* cache = is_k ? p.k_cache : p.v_cache;
        const int kvh = is_k ? h - p.hq : h - p.hq - p.hkv;
        const int64_t to = slot * p.kv_tok_stride + kvh * p.kv_head_stride + at;
        if (p.kv_fmt == kKvSame) {
  #pragma unroll
          for (int i = 0; i < V; ++i) e[i] = from_f32<T>(y[i]);
          *reinterpret_cast<uint4*>(static_cast<T*>(cache) + to) = raw;
        } else {
          uint2 o;
          o.x = pack_fp8x2(y[0], y[1], p.kv_fmt) | (pack_fp8x2(y[2], y[3], p.kv_fmt) << 16);
          o.y = pack_fp8x2(y[4], y[5], p.kv_fmt) | (pack_fp8x2(y[6], y[7], p.kv_fmt) << 16);
          *reinterpret_cast<uint2*>(static_cast<uint8_t*>(cache) + to) = o;
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Accepted nodes: row of node i of the request <- row of node path[i], for i below count, in every plane (layer, k or v, head) of the
// storage.  The path rises (path[i] >= i), so a thread that has its 16 bytes of a plane's rows in the order of i reads every row before
// it is overwritten: rows are read eight at a time, written behind that, and a later read is of a later node than all written so far.
// Bound by the chain lengths -> path -> table -> rows for few requests, by the rows' bytes for many; a thread goes through the chain once
// and then through many planes (32 requests of 3.5 accepted
// nodes, 36 layers of 8 heads of 128: 8.4 us; with a thread per plane and piece, where three waves of blocks went through it, 11.9).
// ---------------------------------------------------------------------------
struct CompactParams {
  uint8_t* store;
  const int* req_to_token;
  const int* req_pool_indices;
  const int* prefix_lens;
  const int* path;          // [batch, steps]
  const int* counts;
  int* status;
  int64_t plane_bytes, table_stride, num_slots;
  int batch, steps, table_rows, table_cols, planes, row_bytes;
};

constexpr int kCompactThreads = 256;
constexpr int kMoves = 8;                 // rows in flight per thread

__global__ void __launch_bounds__(kCompactThreads) tree_compact_kernel(const CompactParams p) {
  pdl_launch_dependents();
  pdl_wait_loads();
  const int b = blockIdx.y;
  const int* path = p.path + static_cast<int64_t>(b) * p.steps;
  int node[kMoves];
#pragma unroll
  for (int k = 0; k < kMoves; ++k) node[k] = k < p.steps ? __ldcg(path + k) : -1;
  const int count = min(__ldcg(p.counts + b), p.steps);
  const int prefix = __ldcg(p.prefix_lens + b), req = __ldcg(p.req_pool_indices + b);
  if (count <= 0) return;
  if (req < 0 || req >= p.table_rows || prefix < 0) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicExch(p.status, kStatusBadIndex);
    return;
  }
  const int lanes = p.row_bytes >> 4;
  const int items = p.planes * lanes;               // below 2^31: checked by the launcher
  const int* table = p.req_to_token + req * p.table_stride;
  bool bad = false;
  int before = -1;
  for (int i0 = 0; i0 < count; i0 += kMoves) {
    if (i0 > 0) {
      // the rows of a later part may be those that an earlier part of this thread read: all planes of a part come first
#pragma unroll
      for (int k = 0; k < kMoves; ++k) node[k] = i0 + k < count ? __ldcg(path + i0 + k) : -1;
    }
    int from[kMoves], to[kMoves];
#pragma unroll
    for (int k = 0; k < kMoves; ++k) {
      from[k] = to[k] = -1;
      if (i0 + k >= count) continue;
      const int n = node[k];
      // a path that does not rise, or leaves the table, is not followed
      if (n < i0 + k || n <= before || n >= p.table_cols - prefix) {
        bad = true;
        continue;
      }
      before = n;
      if (n == i0 + k) continue;          // in its place
      from[k] = __ldcg(table + prefix + n);
      to[k] = __ldcg(table + prefix + i0 + k);
    }
    bool any = false;
#pragma unroll
    for (int k = 0; k < kMoves; ++k) {
      if (to[k] == -1 && from[k] == -1) continue;
      if (from[k] < 0 || from[k] >= p.num_slots || to[k] < 0 || to[k] >= p.num_slots) {
        bad = true;
        to[k] = -1;
      } else {
        any = true;
      }
    }
    if (!any) continue;
    for (int item = blockIdx.x * kCompactThreads + threadIdx.x; item < items; item += gridDim.x * kCompactThreads) {
      const int plane = item / lanes;
      uint8_t* base = p.store + plane * p.plane_bytes + (item - plane * lanes) * 16;
      uint4 v[kMoves];
#pragma unroll
      for (int k = 0; k < kMoves; ++k)
        if (to[k] >= 0) v[k] = __ldcg(reinterpret_cast<const uint4*>(base + static_cast<int64_t>(from[k]) * p.row_bytes));
#pragma unroll
      for (int k = 0; k < kMoves; ++k)
        if (to[k] >= 0) *reinterpret_cast<uint4*>(base + static_cast<int64_t>(to[k]) * p.row_bytes) = v[k];
    }
  }
  if (bad && p.status != nullptr) atomicExch(p.status, kStatusBadIndex);
}

}  // namespace

int launch_tree_prologue(const TreePrologueArgs& a, cudaStream_t s) {
  if (a.index.rows <= 0 || a.index.batch <= 0) return 0;
  PrologueParams p{};
  p.ix = a.index;
  p.qkv = a.qkv;
  p.q_gain = a.q_gain;
  p.k_gain = a.k_gain;
  p.inv_freq = a.inv_freq;
  p.delta = a.position_delta;
  p.q_out = a.q_out;
  p.k_cache = a.k_cache;
  p.v_cache = a.v_cache;
  p.qkv_stride = a.qkv_stride;
  p.kv_tok_stride = a.kv_tok_stride;
  p.kv_head_stride = a.kv_head_stride;
  p.num_slots = a.num_slots;
  p.hq = a.hq;
  p.hkv = a.hkv;
  p.half = a.rotated / 2;
  p.kv_fmt = a.kv_fmt;
  p.eps = a.eps;
  const int heads = a.hq + 2 * a.hkv, per = 256 / a.head_dim, steps = (heads + per - 1) / per;
  p.hsplit = static_cast<int>(std::min<int64_t>(steps, std::max<int64_t>(1, 2048 / a.index.rows)));
  const int64_t warps = static_cast<int64_t>(a.index.rows) * p.hsplit;
  const dim3 grid(static_cast<unsigned>((warps + 3) / 4));
  cudaError_t err = cudaErrorInvalidValue;
  MB200_DISPATCH_HALF(a.dt, {
    if (a.head_dim == 64) err = launch_pdl(tree_prologue_kernel<T, 64>, grid, dim3(128), 0, s, p);
    else if (a.head_dim == 128) err = launch_pdl(tree_prologue_kernel<T, 128>, grid, dim3(128), 0, s, p);
    else if (a.head_dim == 256) err = launch_pdl(tree_prologue_kernel<T, 256>, grid, dim3(128), 0, s, p);
  });
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}

int launch_tree_compact(const TreeCompactArgs& a, cudaStream_t s) {
  if (a.batch <= 0 || a.planes <= 0 || a.steps <= 0) return 0;
  if (a.batch > 65535 || a.row_bytes <= 0 || a.row_bytes % 16 != 0) return -1;
  CompactParams p{};
  p.store = static_cast<uint8_t*>(a.store);
  p.req_to_token = a.req_to_token;
  p.req_pool_indices = a.req_pool_indices;
  p.prefix_lens = a.prefix_lens;
  p.path = a.path;
  p.counts = a.counts;
  p.status = a.status;
  p.plane_bytes = a.num_slots * a.row_bytes;
  p.table_stride = a.table_stride;
  p.num_slots = a.num_slots;
  p.batch = a.batch;
  p.steps = a.steps;
  p.table_rows = a.table_rows;
  p.table_cols = a.table_cols;
  p.planes = a.planes;
  p.row_bytes = a.row_bytes;
  const int64_t items = static_cast<int64_t>(a.planes) * (a.row_bytes / 16);
  if (items >= (int64_t(1) << 31) - (int64_t(1) << 24)) return -1;
  // about two blocks per SM in all
  const int64_t blocks = std::min<int64_t>((items + kCompactThreads - 1) / kCompactThreads, std::max<int64_t>(1, 2 * 148 / a.batch));
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(a.batch));
  const cudaError_t err = launch_pdl(tree_compact_kernel, grid, dim3(kCompactThreads), 0, s, p);
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}

}  // namespace mb200
