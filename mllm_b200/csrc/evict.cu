// Which cached tokens of a request stay, and the move of their cache rows to the front.
#include <algorithm>

#include "common.cuh"
#include "evict.cuh"

namespace mb200 {
namespace {

// ---------------------------------------------------------------------------------------------------------------------
// Selection.  Of a list of n sums (a layer, a request, a kv head) stay: the last min(recent, count) tokens, of the rest the first
// min(first, count - those), and of the rest those with the largest scores, where a score is the largest of the `pool` sums around
// the token and ties go to the lowest index; count = min(n, budget).  The list comes out in ascending order.
//
// A score's bits are turned into a number of 32 bits that rises with it (NaN is as low as minus infinity, zeros of both signs are one).
// The k-th largest is found digit by digit from histograms; a last pass over the list keeps what is larger, and of its equals the first ones.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kSelectThreads = 512;
constexpr int kDigit = 8, kBins = 1 << kDigit;

__device__ __forceinline__ uint32_t rank_of(float x) {
  if (!(x > -INFINITY)) return 0x007fffffu;                  // minus infinity's, and NaN's
  const uint32_t u = __float_as_uint(x + 0.f);               // -0 -> +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelectThreads) cache_select_kernel(const CacheSelectArgs a) {
  __shared__ int bins[kBins];
  __shared__ int warp_counts[kSelectThreads / 32][2];
  __shared__ uint32_t chosen;
  __shared__ int still;
  pdl_wait();
  const int list = blockIdx.x, hk = list % a.hkv, b = list / a.hkv % a.index.batch, layer = list / a.hkv / a.index.batch;
  const Cached r = cached_of(a.index, b);
  const int n = r.len, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int budget = __ldcg(a.budgets + b), count = max(0, min(n, min(budget, a.width)));
  if (tid == 0 && layer == 0 && hk == 0) {
    a.counts[b] = count;
    if ((r.bad || budget > a.width) && a.index.status != nullptr) atomicExch(a.index.status, kStatusBadIndex);
  }
  int* keep = a.keep + static_cast<int64_t>(list) * a.width;
  for (int i = count + tid; i < a.width; i += kSelectThreads) keep[i] = -1;
  if (count == n) {
    for (int i = tid; i < n; i += kSelectThreads) keep[i] = i;
    return;
  }
  const float* sums = a.sums + layer * a.layer_stride + r.row * a.row_stride + hk * a.head_stride;
  const int last = min(a.recent, count), first = min(a.first, count - last), rest = count - last - first;
  const int end = n - last, half = a.pool / 2;         // [first, end): what is chosen from
  auto rank = [&](int i) {
    uint32_t top = 0;
    for (int j = max(0, i - half); j <= min(n - 1, i + half); ++j) top = max(top, rank_of(sums[j]));
    return top;
  };
  // the `rest`-th largest rank, digit by digit from the top
  uint32_t prefix = 0;
  int want = rest;
  if (rest > 0)
    for (int shift = 32 - kDigit; shift >= 0; shift -= kDigit) {
      for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0;
      __syncthreads();
      for (int i = first + tid; i < end; i += kSelectThreads) {
        const uint32_t v = rank(i);
        if (shift == 32 - kDigit || v >> (shift + kDigit) == prefix >> (shift + kDigit)) atomicAdd(&bins[(v >> shift) & (kBins - 1)], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int left = want, d = kBins - 1;
        for (; d > 0 && bins[d] < left; --d) left -= bins[d];
        chosen = prefix | static_cast<uint32_t>(d) << shift;
        still = left;
      }
      __syncthreads();
      prefix = chosen;
      want = still;
    }
  // everything above `prefix`, and the first `want` of its equals, in order
  int at = 0, equals = 0;
  for (int base = 0; base < n; base += kSelectThreads) {
    const int i = base + tid;
    const bool always = i < first || (i >= end && i < n);
    const uint32_t v = i >= first && i < end && rest > 0 ? rank(i) : 0;
    const bool above = i >= first && i < end && rest > 0 && v > prefix, equal = i >= first && i < end && rest > 0 && v == prefix;
    const uint32_t eq = __ballot_sync(0xffffffffu, equal);
    __syncthreads();
    if (lane == 0) warp_counts[warp][0] = __popc(eq);
    __syncthreads();
    int eq_before = equals + __popc(eq & ((1u << lane) - 1));
    for (int w = 0; w < kSelectThreads / 32; ++w) {
      if (w < warp) eq_before += warp_counts[w][0];
      equals += warp_counts[w][0];
    }
    const bool stays = always || above || (equal && eq_before < want);
    const uint32_t st = __ballot_sync(0xffffffffu, stays);
    if (lane == 0) warp_counts[warp][1] = __popc(st);
    __syncthreads();
    int to = at + __popc(st & ((1u << lane) - 1));
    for (int w = 0; w < kSelectThreads / 32; ++w) {
      if (w < warp) to += warp_counts[w][1];
      at += warp_counts[w][1];
    }
    if (stays) keep[to] = i;
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// The move.  Row i <- row keep[i] >= i, within one request, kv head and tensor: a block takes a run of rows at a time, all loads in front
// of all stores, in ascending order.  A row that a later run reads lies at or behind that run's own rows, so nothing is overwritten
// before it is read, and a run's loads may go out in front of the stores of the run before.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 8;      // 16-byte pieces of a thread on their way

__global__ void __launch_bounds__(kMoveThreads) cache_evict_kernel(const CacheEvictArgs a) {
  pdl_wait();
  const int planes = 2 + (a.sums != nullptr ? 1 : 0);
  const int plane = blockIdx.x % planes, list = blockIdx.x / planes, tid = threadIdx.x;
  const int hk = list % a.hkv, b = list / a.hkv % a.index.batch, layer = list / a.hkv / a.index.batch;
  const int row = __ldcg(a.index.req_pool_indices + b), count = min(__ldcg(a.counts + b), a.width);
  if (count <= 0) return;
  if (row < 0 || row >= a.index.table_rows || count > a.index.table_cols) {
    if (tid == 0 && a.index.status != nullptr) atomicExch(a.index.status, kStatusBadIndex);
    return;
  }
  const int* keep = a.keep + static_cast<int64_t>(list) * a.width;
  bool bad = false;
  // source of row i; -1: it stays as it is
  auto source = [&](int i) {
    const int k = __ldcg(keep + i);
    if (k < i || k >= a.index.table_cols) {
      bad = true;
      return -1;
    }
    return k == i ? -1 : k;
  };
  if (plane == 2) {
    float* sums = a.sums + layer * a.layer_stride + row * a.row_stride + hk * a.head_stride;
    for (int base = 0; base < count; base += kMoveThreads * kMoveRows) {
      float v[kMoveRows];
      int from[kMoveRows];
#pragma unroll
      for (int u = 0; u < kMoveRows; ++u) {
        const int i = base + u * kMoveThreads + tid;
        from[u] = i < count ? source(i) : -1;
        v[u] = from[u] >= 0 ? __ldcg(sums + from[u]) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kMoveRows; ++u)
        if (from[u] >= 0) sums[base + u * kMoveThreads + tid] = v[u];
    }
  } else {
    const int* rtt = a.index.req_to_token + static_cast<int64_t>(row) * a.index.table_stride;
    uint8_t* store = static_cast<uint8_t*>(a.store) + ((static_cast<int64_t>(layer) * 2 + plane) * a.hkv + hk) * a.num_slots * a.row_bytes;
    const int pieces = a.row_bytes / 16;
    const int64_t all = static_cast<int64_t>(count) * pieces;
    for (int64_t base = 0; base < all; base += kMoveThreads * kMoveRows) {
      uint4 v[kMoveRows];
      int64_t to[kMoveRows];
#pragma unroll
      for (int u = 0; u < kMoveRows; ++u) {
        const int64_t x = base + u * kMoveThreads + tid;
        to[u] = -1;
        v[u] = make_uint4(0, 0, 0, 0);
        if (x < all) {
          const int i = static_cast<int>(x / pieces), ch = static_cast<int>(x - static_cast<int64_t>(i) * pieces), k = source(i);
          if (k >= 0) {
            const int s0 = __ldcg(rtt + i), s1 = __ldcg(rtt + k);
            if (s0 < 0 || s0 >= a.num_slots || s1 < 0 || s1 >= a.num_slots) {
              bad = true;
            } else {
              to[u] = static_cast<int64_t>(s0) * a.row_bytes + ch * 16;
              v[u] = __ldcg(reinterpret_cast<const uint4*>(store + static_cast<int64_t>(s1) * a.row_bytes + ch * 16));
            }
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kMoveRows; ++u)
        if (to[u] >= 0) *reinterpret_cast<uint4*>(store + to[u]) = v[u];
    }
  }
  if (bad && a.index.status != nullptr) atomicExch(a.index.status, kStatusBadIndex);
}

}  // namespace

int launch_cache_select(const CacheSelectArgs& a, cudaStream_t s) {
  const int64_t lists = static_cast<int64_t>(a.layers) * a.index.batch * a.hkv;
  if (lists <= 0) return 0;
  const cudaError_t err = launch_pdl(cache_select_kernel, dim3(static_cast<unsigned>(lists)), dim3(kSelectThreads), 0, s, a);
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}

int launch_cache_evict(const CacheEvictArgs& a, cudaStream_t s) {
  const int64_t lists = static_cast<int64_t>(a.layers) * a.index.batch * a.hkv;
  if (lists <= 0 || a.width <= 0) return 0;
  const cudaError_t err =
      launch_pdl(cache_evict_kernel, dim3(static_cast<unsigned>(lists * (a.sums != nullptr ? 3 : 2))), dim3(kMoveThreads), 0, s, a);
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}

}  // namespace mb200
