// Which cached tokens stay.  Of a list of n sums (a layer, a request, a kv head) stay: the last min(recent, count) tokens, of the rest the
// first min(first, count - those), and of the rest those with the largest scores, where a score is the largest of the `pool` sums around the
// token, those of the first and last tokens among them, and ties go to the lowest index; count = min(n, budget).  The list comes out in ascending order.
//
// A score's bits are turned into a number of 32 bits that rises with it, its rank (NaN is as low as minus infinity, zeros of both signs are
// one).  The k-th largest is found digit by digit, 11 bits at a time from the top: a histogram in shared memory, its bins added up from
// above until the k-th is reached.  Behind the first digit only its equals count, a few per cent of a list: they are collected, and once
// they are few enough every one is compared with every other.  Then a pass over the list, a stretch per warp, keeps what is above the k-th and
// of its equals the first ones: counts first, then indices.
//
// What bounds it is instructions, 65 to 90 per sum in three passes over shared memory, and the barriers between them, which the warps that
// shared memory leaves room for (46 %) do not cover: 60 % of the issue slots are used (2304 lists of up to 8192 sums, a quarter kept, pool 7: 71 us,
// their bytes take 14).  Eight neighbours are a thread's, so that scores are made in registers.  Lists that are too few for the SMs, or too long for a block's shared
// memory, are cut into slices for a cluster of up to 8 blocks, which add up histograms and counts through each other's shared memory
// (224 lists of 1200 sums: 6.2 us, most of it one wait behind the other).
#include <algorithm>

#include "common.cuh"
#include "evict.cuh"

namespace mb200 {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kResident = 12288;      // sums of a slice that stays in shared memory: three blocks on an SM
constexpr int kBins = 2048, kOwn = kBins / kThreads;
constexpr int kEquals = 1024;         // equals of the first digit that are collected
constexpr int kFew = 32;              // equals that are compared with each other
constexpr int kSplit = 2048;          // a list that is longer than this is worth a cluster where there are few lists
constexpr int kMaxCluster = 8;

struct SelectParams {
  CacheSelectArgs a;
  int cluster, room, split;           // blocks of a list; ranks that a block has room for; length from which on a list is cut
};

__device__ __forceinline__ float max3(float a, float b, float c) {        // NaN gives way
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// of a score that is a number; -0 counts as +0
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// what another block of the cluster has at this address
__device__ __forceinline__ uint32_t ld_other(const void* p, uint32_t rank) {
  uint32_t at, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// HALF: pool / 2 where the scores are made in registers; -1: any other.  RESIDENT: the slice's ranks stay in shared memory.
//
// The slice stands at positions sh to sh + m, so that position 0 is on a 16-byte boundary of the sums; a thread has eight neighbouring positions
// at a time.  Ranks of tokens that are not to be chosen from are 0, which is below all others.
template <int HALF, bool RESIDENT>
__device__ __forceinline__ void select_list(const CacheSelectArgs& a, int* keep, const float* sums, int n, int count, int cta, int slices, int per,
                                            uint32_t* bins, uint32_t* equals, uint32_t* ranks) {
  __shared__ uint32_t chosen;
  __shared__ int still, found, collected;
  __shared__ __align__(16) int warp_sums[2][kWarps];
  __shared__ uint32_t totals[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int last = min(a.recent, count), first = min(a.first, count - last), rest = count - last - first;
  const int end = n - last, half = HALF >= 0 ? HALF : a.pool / 2;        // [first, end): what is chosen from
  const int lo = min(n, cta * per), hi = min(n, lo + per), m = hi - lo;
  const int sh = static_cast<int>(reinterpret_cast<uintptr_t>(sums) >> 2 & 3), all = m > 0 ? sh + m : 0, shift0 = lo - sh;      // position + shift0: index

  // bits k with position p0 + k of index in [from, to)
  auto between = [&](int p0, int from, int to) {
    const int x = min(max(from - shift0 - p0, 0), 8), y = min(max(to - shift0 - p0, 0), 8);
    return (0xffu >> (8 - y)) & (0xffu << x);
  };
  auto four = [&](int p0) -> float4 {         // the sums at positions p0 ..; minus infinity outside the list
    const int i = p0 + shift0;
    if (i >= 0 && i + 3 < n) return *reinterpret_cast<const float4*>(sums + i);
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = i + k >= 0 && i + k < n ? sums[i + k] : -INFINITY;
    return make_float4(v[0], v[1], v[2], v[3]);
  };
  auto make = [&](int p0, uint32_t (&v)[8]) {        // ranks of the scores at positions p0 ..
    float y[8];
    if constexpr (HALF >= 0 && HALF <= 4) {
      constexpr int kSide = HALF == 0 ? 0 : 4;
      float x[8 + 2 * kSide];
      const bool within = p0 + shift0 >= kSide && p0 + shift0 + 8 + kSide <= n;
#pragma unroll
      for (int k = 0; k < 8 + 2 * kSide; k += 4) {
        const float4 q = within ? *reinterpret_cast<const float4*>(sums + p0 + shift0 - kSide + k) : four(p0 - kSide + k);
        x[k] = q.x;
        x[k + 1] = q.y;
        x[k + 2] = q.z;
        x[k + 3] = q.w;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        y[k] = fmaxf(x[k + kSide], -INFINITY);
#pragma unroll
        for (int d = 1; d <= HALF; ++d) y[k] = max3(y[k], x[k + kSide - d], x[k + kSide + d]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = -INFINITY;
      const int i0 = p0 + shift0;
      for (int i = max(0, i0 - half); i <= min(n - 1, i0 + 7 + half); ++i) {
        const float x = sums[i];
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = abs(i - i0 - k) <= half ? fmaxf(y[k], x) : y[k];
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = rank_of(y[k]);
    const int from = max(first, lo), to = min(end, hi);
    if (p0 + shift0 < from || p0 + shift0 + 8 > to) {
      const uint32_t open = between(p0, from, to);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = open >> k & 1 ? v[k] : 0u;
    }
  };
  auto get = [&](int p0, uint32_t (&v)[8]) {
    if constexpr (RESIDENT) {
      *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(ranks + p0);
      *reinterpret_cast<uint4*>(v + 4) = *reinterpret_cast<const uint4*>(ranks + p0 + 4);
    } else {
      make(p0, v);
    }
  };

  for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
  if (tid == 0) collected = 0;
  __syncthreads();
  uint32_t top = 0xffffffffu;
  int want = 0;
  if (rest > 0) {
    // ---- ranks of the scores, and the first digit's histogram (of ranks of 0, too: their bin is never reached) ----
#pragma unroll 1
    for (int p0 = 8 * tid; p0 < all; p0 += 8 * kThreads) {
      uint32_t v[8];
      make(p0, v);
      if constexpr (RESIDENT) {
        *reinterpret_cast<uint4*>(ranks + p0) = *reinterpret_cast<const uint4*>(v);
        *reinterpret_cast<uint4*>(ranks + p0 + 4) = *reinterpret_cast<const uint4*>(v + 4);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) atomicAdd(&bins[v[k] >> 21], 1u);
    }
    __syncthreads();
    // ---- the `rest`-th largest rank: `top`, of whose equals the first `want` stay ----
    want = rest;
    uint32_t prefix = 0;
    bool listed = false;           // the equals of the first digit have been collected
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 10 : 11;
      if (pass > 0) {
        if (slices > 1) cluster_sync();            // all have read this block's histogram
        for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
        __syncthreads();
        const uint32_t mask = (1u << width) - 1, high = prefix >> (shift + width);
        auto note = [&](uint32_t v) {
          if (v >> (shift + width) == high) atomicAdd(&bins[(v >> shift) & mask], 1u);
        };
        if (listed) {
          for (int i = tid; i < collected; i += kThreads) note(equals[i]);
        } else {
#pragma unroll 1
          for (int p0 = 8 * tid; p0 < all; p0 += 8 * kThreads) {
            uint32_t v[8];
            get(p0, v);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (v[k] != 0) note(v[k]);
          }
        }
        __syncthreads();
      }
      // a thread has eight bins, the first thread the highest
      const int bin0 = kBins - kOwn - kOwn * tid;
      int x[kOwn];
#pragma unroll
      for (int k = 0; k < kOwn; k += 4) *reinterpret_cast<uint4*>(x + k) = *reinterpret_cast<const uint4*>(bins + bin0 + k);
      if (slices > 1) {
        cluster_sync();
        for (int c = 0; c < slices; ++c)
          if (c != cta)
#pragma unroll
            for (int k = 0; k < kOwn; ++k) x[k] += ld_other(bins + bin0 + k, c);
      }
      int mine = 0;
#pragma unroll
      for (int k = 0; k < kOwn; ++k) mine += x[k];
      const int of_warp = __reduce_add_sync(0xffffffffu, mine);
      if (lane == 0) warp_sums[0][warp] = of_warp;
      __syncthreads();
      int before = 0;
#pragma unroll
      for (int w = 0; w < kWarps; w += 4) {
        const int4 s = *reinterpret_cast<const int4*>(&warp_sums[0][w]);
        before += (w < warp ? s.x : 0) + (w + 1 < warp ? s.y : 0) + (w + 2 < warp ? s.z : 0) + (w + 3 < warp ? s.w : 0);
      }
      if (before < want && want <= before + of_warp) {       // one warp has it among its bins
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
        before += incl - mine;
        if (before < want && want <= before + mine) {
          int k = kOwn - 1, in = 0, above = before;
#pragma unroll
          for (int i = kOwn - 1; i >= 0; --i)
            if (k == i) {
              in = x[i];
              if (i > 0 && above + in < want) {
                above += in;
                k = i - 1;
              }
            }
          chosen = prefix | static_cast<uint32_t>(bin0 + k) << shift;
          still = want - above;
          found = in;
        }
      }
      __syncthreads();
      prefix = chosen;
      want = still;
      const int there = found;
      if (there == want || pass == 2) {
        // Nothing is left to tell them apart, or all of them stay: those with this prefix and any digits behind it
        top = prefix - (there == want ? 1 : 0);
        want = there == want ? 0 : want;
        break;
      }
      if (pass == 0) {
#pragma unroll 1
        for (int p0 = 8 * tid; p0 < all; p0 += 8 * kThreads) {
          uint32_t v[8];
          get(p0, v);
          int mine = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) mine += (v[k] ^ prefix) < 1u << 21 ? 1 : 0;
          if (mine != 0) {
            int at = atomicAdd(&collected, mine);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if ((v[k] ^ prefix) < 1u << 21) {
                if (at < kEquals) equals[at] = v[k];
                ++at;
              }
          }
        }
        __syncthreads();
        listed = collected <= kEquals;
      }
      if (slices == 1 && listed && there <= kFew) {
        // few are left: each is compared with all others
        const int total = collected;
        uint32_t* few = bins;
        __syncthreads();                            // all have seen what was found
        if (tid == 0) found = 0;
        __syncthreads();
        for (int i = tid; i < total; i += kThreads)
          if (equals[i] >> shift == prefix >> shift) few[atomicAdd(&found, 1)] = equals[i];
        __syncthreads();
        if (tid < there) {
          const uint32_t v = few[tid];
          int above = 0, same = 0;
          for (int i = 0; i < there; ++i) {
            above += few[i] > v;
            same += few[i] == v;
          }
          if (above < want && want <= above + same) {       // the same for all equals
            const bool all = want == above + same;
            chosen = v - (all ? 1 : 0);
            still = all ? 0 : want - above;
          }
        }
        __syncthreads();
        top = chosen;
        want = still;
        break;
      }
    }
  }
  // ---- indices: what is above `top`, of its equals the first `want` (0: none of them), and the tokens that stay in any case ----
  auto classify = [&](int p0, uint32_t& above, uint32_t& equal) {
    above = equal = 0;
    if (p0 >= all) return;
    if (rest > 0) {
      uint32_t v[8];
      get(p0, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) above |= v[k] > top ? 1u << k : 0u;
      if (want > 0)
#pragma unroll
        for (int k = 0; k < 8; ++k) equal |= v[k] == top ? 1u << k : 0u;
    }
    if (p0 + shift0 < max(first, lo) || p0 + shift0 + 8 > min(end, hi)) above |= between(p0, lo, min(first, hi)) | between(p0, max(end, lo), hi);
  };
  int above_before = 0, equal_before = 0;
  if (slices > 1) {              // how many the blocks in front have
    int n_both = 0;
    if (tid < 2) totals[tid] = 0;
    __syncthreads();
    for (int p0 = 8 * tid; p0 < all; p0 += 8 * kThreads) {
      uint32_t above, equal;
      classify(p0, above, equal);
      n_both += __popc(above) | __popc(equal) << 16;       // flushed before either part runs over
      if (n_both & 0x40004000) {
        atomicAdd(&totals[0], n_both & 0xffff);
        atomicAdd(&totals[1], static_cast<uint32_t>(n_both) >> 16);
        n_both = 0;
      }
    }
    atomicAdd(&totals[0], n_both & 0xffff);
    atomicAdd(&totals[1], static_cast<uint32_t>(n_both) >> 16);
    cluster_sync();
    for (int c = 0; c < cta; ++c) {
      above_before += ld_other(&totals[0], c);
      equal_before += ld_other(&totals[1], c);
    }
  }
#pragma unroll 1
  for (int base = 0, turn = 0; base < all; base += 8 * kThreads, turn ^= 1) {
    const int p0 = base + 8 * tid;
    uint32_t above, equal;
    classify(p0, above, equal);
    const int mine = __popc(above) | __popc(equal) << 16;       // up to 2048 of each in a turn
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sums[turn][warp] = incl;
    __syncthreads();
    int before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; w += 4) {
      const int4 s = *reinterpret_cast<const int4*>(&warp_sums[turn][w]);
      before += (w < warp ? s.x : 0) + (w + 1 < warp ? s.y : 0) + (w + 2 < warp ? s.z : 0) + (w + 3 < warp ? s.w : 0);
      total += s.x + s.y + s.z + s.w;
    }
    const int my_equal = equal_before + (before >> 16);
    int to = above_before + (before & 0xffff) + min(want, my_equal);
    uint32_t stay = above;
    if (equal != 0) {            // of the equals the first that are wanted
      int left = max(0, want - my_equal);
      for (uint32_t e = equal; e != 0 && left > 0; e &= e - 1, --left) stay |= e & -e;
    }
    int* at = keep + to;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (stay >> k & 1) *at++ = p0 + shift0 + k;
    above_before += total & 0xffff;
    equal_before += total >> 16;
  }
  if (slices > 1) cluster_sync();     // no block leaves while its counts may be read
}

template <int HALF>
__global__ void __launch_bounds__(kThreads) cache_select_kernel(const SelectParams p) {
  const CacheSelectArgs& a = p.a;
  extern __shared__ __align__(16) uint32_t select_smem[];
  uint32_t* bins = select_smem;
  uint32_t* equals = bins + kBins;
  uint32_t* ranks = equals + kEquals;
  pdl_wait();
  const int cta = p.cluster > 1 ? static_cast<int>(cluster_rank()) : 0, list = blockIdx.x / p.cluster, tid = threadIdx.x;
  const int hk = list % a.hkv, b = list / a.hkv % a.index.batch, layer = list / a.hkv / a.index.batch;
  const Cached r = cached_of(a.index, b);
  const int n = r.len, count = max(0, min(n, min(__ldcg(a.budgets + b), a.width)));
  if (tid == 0 && cta == 0 && layer == 0 && hk == 0) {
    a.counts[b] = count;
    if (r.bad && a.index.status != nullptr) atomicExch(a.index.status, kStatusBadIndex);
  }
  int* keep = a.keep + static_cast<int64_t>(list) * a.width;
  for (int i = count + cta * kThreads + tid; i < a.width; i += p.cluster * kThreads) keep[i] = -1;
  if (count == n) {
    for (int i = cta * kThreads + tid; i < n; i += p.cluster * kThreads) keep[i] = i;
    return;
  }
  const int slices = n > p.split ? p.cluster : 1;
  if (cta >= slices) return;          // the cluster's barriers do not wait for blocks that have left
  const float* sums = a.sums + layer * a.layer_stride + r.row * a.row_stride + hk * a.head_stride;
  const int per = slices == 1 ? n : ((n + slices - 1) / slices + 7) / 8 * 8;
  if (per <= p.room) {
    select_list<HALF, true>(a, keep, sums, n, count, cta, slices, per, bins, equals, ranks);
  } else {
    select_list<HALF, false>(a, keep, sums, n, count, cta, slices, per, bins, equals, ranks);
  }
}

template <int HALF>
int launch_half(const SelectParams& p, unsigned lists, int smem, cudaStream_t s) {
  auto kern = cache_select_kernel<HALF>;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem) != cudaSuccess) return -3;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(lists * p.cluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, p);
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}

}  // namespace

int launch_cache_select(const CacheSelectArgs& a, cudaStream_t s) {
  const int64_t lists = static_cast<int64_t>(a.layers) * a.index.batch * a.hkv;
  if (lists <= 0) return 0;
  SelectParams p{};
  p.a = a;
  // A cluster where there are fewer lists than SMs, for lists from kSplit on, or where a list may be longer than a block has room for
  const bool few = 2 * lists <= a.num_sms;
  p.cluster = 1;
  while (p.cluster < kMaxCluster && (few ? p.cluster * 2 * lists <= a.num_sms && p.cluster * kSplit < a.index.table_cols
                                         : static_cast<int64_t>(p.cluster) * kResident < a.index.table_cols))
    p.cluster *= 2;
  p.split = few ? kSplit : kResident;
  p.room = std::min(kResident, (std::max(a.index.table_cols, 1) + 7) / 8 * 8);
  const int smem = (kBins + kEquals + p.room + 16) * 4;          // a slice may begin three places behind a 16-byte boundary
  const unsigned grid = static_cast<unsigned>(lists);
  switch (a.pool / 2) {
    case 0: return launch_half<0>(p, grid, smem, s);
    case 1: return launch_half<1>(p, grid, smem, s);
    case 2: return launch_half<2>(p, grid, smem, s);
    case 3: return launch_half<3>(p, grid, smem, s);
    case 4: return launch_half<4>(p, grid, smem, s);
    default: return launch_half<-1>(p, grid, smem, s);
  }
}

}  // namespace mb200
