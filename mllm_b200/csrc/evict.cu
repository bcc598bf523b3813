// Moves the cache rows of the tokens that stay to the front: row i <- row keep[i] >= i, within one request, kv head and tensor, in place.
//
// A warp takes the rows of a (layer, request, kv head, tensor) in ascending order, up to 32 at a time: 16 bytes a lane, eight times, are on
// their way in registers.  All rows of a run are loaded before the first of them is written, and a row that a later run reads lies at or behind
// that run's own rows: nothing is overwritten before it is read.  Sources and slots are looked up in front of their run.  Rows that stay where
// they are are left out.
//
// What bounds it is memory: every moved row is read and written once.  (The copy engine takes 11 ns for every bulk copy of an SM, whatever its
// size up to 256 bytes: a row in and a row out took 340 us for 36 layers and 4 requests of 4000 tokens, a quarter kept; the bytes take 182.)
#include <algorithm>

#include "common.cuh"
#include "evict.cuh"

namespace mb200 {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kLoads = 8;                 // 16-byte pieces of a lane in a run
constexpr int kSumsPer = 8;               // sums of a lane on their way

struct EvictParams {
  CacheEvictArgs a;
  int pieces, piece;                      // of a row: how many, bytes of all but the last
  int loads, lanes_log2;                  // 16-byte pieces of a lane in a run: 32 rows or fewer; lanes of a row
  int64_t tasks, moves;                   // warps' tasks; those in front that move rows
};

__global__ void __launch_bounds__(kThreads, 6) cache_evict_kernel(const EvictParams p) {
  const CacheEvictArgs& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  const int64_t task = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (task >= p.tasks) return;
  const bool moves = task < p.moves;
  const int64_t which = moves ? task : task - p.moves;
  const int piece = moves ? static_cast<int>(which % p.pieces) : 0, tensor = moves ? static_cast<int>(which / p.pieces % 2) : 0;
  const int64_t list = moves ? which / p.pieces / 2 : which;
  const int hk = static_cast<int>(list % a.hkv), b = static_cast<int>(list / a.hkv % a.index.batch);
  const int64_t layer = list / a.hkv / a.index.batch;
  const int row = __ldcg(a.index.req_pool_indices + b), count = __ldcg(a.counts + b);
  if (count <= 0) return;
  if (row < 0 || row >= a.index.table_rows || count > a.index.table_cols || count > a.width) {
    if (lane == 0 && a.index.status != nullptr) atomicExch(a.index.status, kStatusBadIndex);
    return;
  }
  const int* keep = a.keep + list * a.width;
  bool bad = false;
  // source of row i; -1: it stays as it is
  auto checked = [&](int i, int k) {
    if (i >= count) return -1;
    if (k < i || k >= a.index.table_cols) {
      bad = true;
      return -1;
    }
    return k == i ? -1 : k;
  };
  if (!moves) {
    float* sums = a.sums + layer * a.layer_stride + row * a.row_stride + hk * a.head_stride;
    for (int base = 0; base < count; base += 32 * kSumsPer) {
      int from[kSumsPer];
      float v[kSumsPer];
#pragma unroll
      for (int u = 0; u < kSumsPer; ++u) {
        const int i = base + u * 32 + lane;
        from[u] = i < count ? __ldcg(keep + i) : -1;
      }
#pragma unroll
      for (int u = 0; u < kSumsPer; ++u) {
        from[u] = checked(base + u * 32 + lane, from[u]);
        v[u] = from[u] >= 0 ? __ldcg(sums + from[u]) : 0.f;
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < kSumsPer; ++u)
        if (from[u] >= 0) __stcg(sums + base + u * 32 + lane, v[u]);
      __syncwarp();
    }
    if (bad && a.index.status != nullptr) atomicExch(a.index.status, kStatusBadIndex);
    return;
  }

  const int* rtt = a.index.req_to_token + static_cast<int64_t>(row) * a.index.table_stride;
  const int off = piece * p.piece, bytes = min(p.piece, a.row_bytes - off), rows = p.loads * 32 >> p.lanes_log2;
  uint8_t* store = static_cast<uint8_t*>(a.store) + ((layer * 2 + tensor) * a.hkv + hk) * a.num_slots * a.row_bytes + off;
  const int runs = (count + rows - 1) / rows;
  // A run's rows, one a lane: its source (two runs ahead), the slots from and to (one ahead; nothing looks at them before their turn)
  auto kept = [&](int t) {
    const int i = t * rows + lane;
    return t < runs && lane < rows && i < count ? __ldcg(keep + i) : -1;
  };
  struct Slots {
    int from, to;
    bool moves;          // no slot's value says that a row stays
  };
  auto slots_of = [&](int t, int k) {
    const int i = t * rows + lane;
    if (t >= runs || lane >= rows || (k = checked(i, k)) < 0) return Slots{-1, -1, false};
    return Slots{__ldcg(rtt + k), __ldcg(rtt + i), true};
  };
  const int row0 = lane >> p.lanes_log2, ch = lane & ((1 << p.lanes_log2) - 1), per = 32 >> p.lanes_log2;     // of every 32 lanes' pieces
  const bool mine = ch * 16 < bytes;
  store += ch * 16;
  Slots s = slots_of(0, kept(0));
  Slots next = slots_of(1, kept(1));
  int k_next = kept(2);
  for (int t = 0; t < runs; ++t) {
    if (s.moves && (s.from < 0 || s.from >= a.num_slots || s.to < 0 || s.to >= a.num_slots)) {
      bad = true;
      s.from = s.to = -1;
    }
    uint4 x[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      if (u >= p.loads) break;
      const int from = __shfl_sync(0xffffffffu, s.from, u * per + row0);
      if (from >= 0 && mine) x[u] = __ldcg(reinterpret_cast<const uint4*>(store + static_cast<int64_t>(from) * a.row_bytes));
    }
    const int to_slot = s.to;
    s = next;
    next = slots_of(t + 2, k_next);
    k_next = kept(t + 3);
    __syncwarp();                            // all lanes have loaded what this run's stores overwrite
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      if (u >= p.loads) break;
      const int to = __shfl_sync(0xffffffffu, to_slot, u * per + row0);
      if (to >= 0 && mine) __stcg(reinterpret_cast<uint4*>(store + static_cast<int64_t>(to) * a.row_bytes), x[u]);
    }
    __syncwarp();
  }
  if (bad && a.index.status != nullptr) atomicExch(a.index.status, kStatusBadIndex);
}

}  // namespace

int launch_cache_evict(const CacheEvictArgs& a, cudaStream_t s) {
  const int64_t lists = static_cast<int64_t>(a.layers) * a.index.batch * a.hkv;
  if (lists <= 0) return 0;
  EvictParams p{};
  p.a = a;
  // Pieces of a row: no more than a warp takes at once, and half as much down to 64 bytes while there are fewer warps than 12 per SM (28 layers
  // of one request, 1200 tokens, 43 % kept: 34.1 us in pieces of 64, 36.3 of 128, some 57 of 256; 36 layers, 4 x 4000 tokens, whole rows, 231)
  p.pieces = 1;
  auto piece = [&] { return ((a.row_bytes + p.pieces - 1) / p.pieces + 15) / 16 * 16; };
  while (piece() > 512 || (lists * 2 * p.pieces < 12 * a.num_sms && piece() >= 128)) p.pieces *= 2;
  p.piece = piece();
  p.pieces = (a.row_bytes + p.piece - 1) / p.piece;
  while (16 << p.lanes_log2 < p.piece) ++p.lanes_log2;
  p.loads = std::min(kLoads, 1 << p.lanes_log2);
  p.moves = lists * 2 * p.pieces;
  p.tasks = p.moves + (a.sums != nullptr ? lists : 0);
  const int64_t grid = (p.tasks + kWarps - 1) / kWarps;
  if (grid >= (int64_t(1) << 31)) return -1;
  const cudaError_t err = launch_pdl(cache_evict_kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, s, p);
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}

}  // namespace mb200
