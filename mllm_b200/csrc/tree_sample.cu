// Verification of drafted token trees against the target's filtered distribution, with random numbers that the caller gives.
//
// A request's walk begins at node 0.  At a node with logits l, temperature T and filters,
//   e_i = exp((l_i - max l) / T),   kept = {i: e_i >= the k-th largest, >= the smallest whose strictly larger mass is below top_p * sum e,
//   >= min_p}  (ties are kept),   p = e / sum over kept.
// The node's children are looked at in the order of their numbers: child c with token x is taken if u_c q(x) < p(x); otherwise
// p <- max(p - q, 0) / sum, where q is the distribution that the children were drawn from, or all of x (candidates without
// probabilities).  Without a child that is taken the walk ends with the first token whose running sum of p, in the order of the ids,
// passes u * sum p.  The emitted tokens are distributed as the target's own samples, whatever the draft.
//
// What a step reads is known when the step before is done, so a walk is a chain: row, maximum, sum, cut, children, row.  A cluster of up
// to 8 CTAs takes a request; each holds its part of the row in shared memory, and what they share goes through one exchange (a slot per
// CTA, one cluster barrier) per stage.  The cut needs no sort of the row and no histogram: a lower bound on it (the smallest of the
// warps' maxima for top-k, the mass that V tokens can hide below it for top-p, min_p itself) leaves a few hundred tokens, which every
// CTA collects and sorts for itself.  Where more than kList are left (flat distributions) the cut is found bit by bit, an exchange each.
//
// Whole tokens hang on sums: e is taken in 64 bits where it is above 2^-12 and sums are joined in 64 bits, so that the border of a token
// is off by some 10^-9 of the whole.
#include <algorithm>

#include "common.cuh"
#include "tree.h"

namespace mb200 {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kList = 4096;               // candidates that are sorted
constexpr int kChildren = 64;             // of a node that are looked at

struct SampleParams {
  const void* logits;
  const int64_t* tokens;
  const int* parents;
  const int* tree_lens;
  const int* q_start;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;       // or null
  const float* uniform;
  const float* uniform_final;
  const float* draft;       // [rows, vocab] or null
  int* path;
  int64_t* out;
  int* counts;
  int* status;
  int64_t logit_stride, draft_stride;
  int rows, vocab, chunk, steps, vec;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint64_t ld_cluster64(uint32_t a) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_cluster32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
// order of floats as order of whole numbers; a value that is no number is below all others
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return x != x ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ double shfl_xor_d(double v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// what the weight of a token is made of
struct Scale {
  float mx, c_hi, c_lo;     // log2(e) / T as two floats
  double inv_t, mx_d;
  __device__ __forceinline__ double operator()(float x) const {
    if (!(x == x)) return 0.0;
    if (x == mx) return 1.0;
    const float d = x - mx, t = fmaf(d, c_hi, d * c_lo);
    if (t > -12.f) return exp((static_cast<double>(x) - mx_d) * inv_t);
    return static_cast<double>(fast_exp2(t));
  }
};

struct Shared {
  uint64_t slot[2][4];          // what this CTA tells the others, alternating
  double red[kWarps][2];
  uint64_t red_key[kWarps];
  float red_min[kWarps];
  int list_n;
  int parents[512];
  int child[kChildren];         // nodes
  int child_token[kChildren];
  float child_u[kChildren], child_q[kChildren];
  double child_w[kChildren];    // e of the token, 0 where it is filtered out
  double scale[kChildren];      // rejections so far: p <- p * scale - q
  int removed[kChildren];       // tokens taken out (candidates without probabilities)
  int children, owner;
  double scan[kWarps];
};

template <typename T>
__global__ void __launch_bounds__(kThreads) tree_sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Shared sh;
  float* list = reinterpret_cast<float*>(dyn);              // this CTA's candidates
  float* sorted = list + kList;                             // all candidates
  T* xs = reinterpret_cast<T*>(sorted + kList);             // this CTA's part of the row
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int b = blockIdx.x / ranks;
  pdl_launch_dependents();
  pdl_wait_loads();
  const int nodes = __ldcg(p.tree_lens + b), row0 = __ldcg(p.q_start + b);
  const int v0 = min(p.vocab, static_cast<int>(rank) * p.chunk), n = min(p.vocab - v0, p.chunk);
  const float temp = __ldcg(p.temperature + b), top_p = __ldcg(p.top_p + b);
  const int top_k = __ldcg(p.top_k + b);
  const float min_p = p.min_p != nullptr ? __ldcg(p.min_p + b) : 0.f;
  const float u_final = __ldcg(p.uniform_final + b);
  const bool cut_k = top_k > 0 && top_k < p.vocab, cut_p = top_p < 1.f;
  int turn = 0;                 // exchanges so far
  int count = 0;

  auto finish_row = [&](int from) {        // what stands behind the walk
    if (rank == 0)
      for (int i = from + tid; i < p.steps; i += kThreads) {
        p.path[static_cast<int64_t>(b) * p.steps + i] = -1;
        p.out[static_cast<int64_t>(b) * p.steps + i] = -1;
      }
  };
  // a request without nodes, or with rows outside the tensors: nothing to walk (the same for all CTAs of the cluster)
  if (nodes <= 0 || row0 < 0 || nodes > p.rows - row0) {
    if (nodes > 0 && tid == 0 && rank == 0 && p.status != nullptr) atomicExch(p.status, kStatusBadIndex);
    finish_row(0);
    if (tid == 0 && rank == 0) p.counts[b] = 0;
    return;
  }

  // Sums over the cluster, the same bits for every thread.
  auto sum_all = [&](double& a, double& c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += shfl_xor_d(a, o);
      c += shfl_xor_d(c, o);
    }
    if (lane == 0) {
      sh.red[warp][0] = a;
      sh.red[warp][1] = c;
    }
    __syncthreads();
    if (warp == 0) {
      a = lane < kWarps ? sh.red[lane][0] : 0.0;
      c = lane < kWarps ? sh.red[lane][1] : 0.0;
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) {
        a += shfl_xor_d(a, o);
        c += shfl_xor_d(c, o);
      }
      if (lane == 0) {
        sh.slot[turn & 1][0] = static_cast<uint64_t>(__double_as_longlong(a));
        sh.slot[turn & 1][1] = static_cast<uint64_t>(__double_as_longlong(c));
      }
    }
    cluster_sync();
    double x = 0.0, y = 0.0;
    if (lane < static_cast<int>(ranks)) {
      const uint32_t from = at_rank(&sh.slot[turn & 1][0], lane);
      x = __longlong_as_double(static_cast<long long>(ld_cluster64(from)));
      y = __longlong_as_double(static_cast<long long>(ld_cluster64(from + 8)));
    }
#pragma unroll
    for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
      x += shfl_xor_d(x, o);
      y += shfl_xor_d(y, o);
    }
    a = __shfl_sync(0xffffffffu, x, 0);
    c = __shfl_sync(0xffffffffu, y, 0);
    ++turn;
  };

  for (int i = tid; i < min(nodes, 512); i += kThreads) sh.parents[i] = __ldcg(p.parents + row0 + i);
  int node = 0;
  for (;;) {
    const int row = row0 + node;
    const T* logits = static_cast<const T*>(p.logits) + row * p.logit_stride + v0;
    // ---- the row's part to shared memory; its largest value, lowest id first, and the smallest of the groups' largest ----
    float best = -INFINITY;
    uint64_t top = 0;           // key of the largest << 32 | ~id
    auto see = [&](float x, int i) {
      const uint64_t k = static_cast<uint64_t>(key_of(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(v0 + i));
      top = k > top ? k : top;
      best = fmaxf(best, x);
    };
    if (p.vec) {
      constexpr int kPer = 16 / sizeof(T);
      const int whole = n / kPer;
#pragma unroll 4
      for (int i = tid; i < whole; i += kThreads) {
        const uint4 v = __ldcg(reinterpret_cast<const uint4*>(logits) + i);
        reinterpret_cast<uint4*>(xs)[i] = v;
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int k = 0; k < kPer; ++k) see(to_f32(e[k]), i * kPer + k);
      }
      for (int i = whole * kPer + tid; i < n; i += kThreads) {
        xs[i] = logits[i];
        see(to_f32(xs[i]), i);
      }
    } else {
      for (int i = tid; i < n; i += kThreads) {
        xs[i] = logits[i];
        see(to_f32(xs[i]), i);
      }
    }
    // groups of 32 lanes (or 8, for a larger k): that many tokens are at least as large as the smallest of their maxima
    const bool by_warps = top_k <= static_cast<int>(ranks) * kWarps;
    float g_max = best;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) g_max = fmaxf(g_max, __shfl_xor_sync(0xffffffffu, g_max, o));
    if (by_warps) g_max = warp_max(g_max);
    float low = g_max;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
      const uint64_t k = __shfl_xor_sync(0xffffffffu, top, o);
      top = k > top ? k : top;
    }
    if (lane == 0) {
      sh.red_key[warp] = top;
      sh.red_min[warp] = low;
    }
    if (tid == 0) {
      sh.list_n = 0;
      sh.children = 0;
    }
    __syncthreads();
    if (warp == 0) {
      top = lane < kWarps ? sh.red_key[lane] : 0;
      low = lane < kWarps ? sh.red_min[lane] : INFINITY;
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) {
        const uint64_t k = __shfl_xor_sync(0xffffffffu, top, o);
        top = k > top ? k : top;
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
      }
      if (lane == 0) {
        sh.slot[turn & 1][0] = top;
        sh.slot[turn & 1][1] = __float_as_uint(low);
      }
      // the node's children, the same in every CTA
      if (count + 1 < p.steps) {
        int found = 0;
        for (int j0 = node + 1; j0 < nodes && found < kChildren; j0 += 32) {
          const int j = j0 + lane;
          const bool is = j < nodes && (j < 512 ? sh.parents[j] : __ldcg(p.parents + row0 + j)) == node;
          const unsigned votes = __ballot_sync(0xffffffffu, is);
          const int at = found + __popc(votes & ((1u << lane) - 1));
          if (is && at < kChildren) sh.child[at] = j;
          found += __popc(votes);
        }
        if (lane == 0) sh.children = min(found, kChildren);
      }
    }
    cluster_sync();
    {
      uint64_t k = 0;
      float m = INFINITY;
      if (lane < static_cast<int>(ranks)) {
        const uint32_t from = at_rank(&sh.slot[turn & 1][0], lane);
        k = ld_cluster64(from);
        m = __uint_as_float(static_cast<uint32_t>(ld_cluster64(from + 8)));
      }
#pragma unroll
      for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, k, o);
        k = other > k ? other : k;
        m = fminf(m, __shfl_xor_sync(0xffffffffu, m, o));
      }
      top = __shfl_sync(0xffffffffu, k, 0);
      low = __shfl_sync(0xffffffffu, m, 0);
      ++turn;
    }
    const float mx = of_key(static_cast<uint32_t>(top >> 32));
    const int first_best = static_cast<int>(0xffffffffu - static_cast<uint32_t>(top));
    const int children = sh.children;
    // the children's numbers, read side by side
    if (tid < children) {
      const int j = sh.child[tid];
      const int64_t token = __ldcg(p.tokens + row0 + j);
      const bool in = token >= 0 && token < p.vocab;      // a token outside the vocabulary is never taken
      sh.child_token[tid] = in ? static_cast<int>(token) : -1;
      sh.child_u[tid] = __ldcg(p.uniform + row0 + j);
      sh.child_q[tid] = !in || p.draft == nullptr ? 1.f : __ldcg(p.draft + row * p.draft_stride + token);
      sh.child_w[tid] = in ? static_cast<double>(to_f32(static_cast<const T*>(p.logits)[row * p.logit_stride + token])) : 0.0;
    }
    int taken = -1;
    // ---- one token has all the mass: greedy requests, and rows without a finite logit ----
    if (temp <= 1e-6f || !(mx > -INFINITY)) {
      __syncthreads();
      for (int i = 0; i < children && taken < 0; ++i)
        if (sh.child_token[i] == first_best && sh.child_u[i] * sh.child_q[i] < 1.f) taken = i;
      const int next = taken < 0 ? -1 : sh.child[taken];
      if (rank == 0 && tid == 0) {
        p.path[static_cast<int64_t>(b) * p.steps + count] = node;
        p.out[static_cast<int64_t>(b) * p.steps + count] = first_best;
      }
      ++count;
      if (next < 0) break;
      node = next;
      __syncthreads();
      continue;
    }

    Scale w;
    w.mx = mx;
    w.mx_d = mx;
    w.inv_t = 1.0 / static_cast<double>(temp);
    const double c = 1.4426950408889634 * w.inv_t;
    w.c_hi = static_cast<float>(c);
    w.c_lo = static_cast<float>(c - static_cast<double>(w.c_hi));
    constexpr int kPair = sizeof(T) == 2 ? 2 : 1;
    auto each = [&](auto&& fn) {             // fn(value, id within this part), ids far apart
      if constexpr (kPair == 2) {
        for (int i = tid; i < (n + 1) / 2; i += kThreads) {
          const uint32_t two = reinterpret_cast<const uint32_t*>(xs)[i];
          const T* e = reinterpret_cast<const T*>(&two);
          fn(to_f32(e[0]), 2 * i);
          if (2 * i + 1 < n) fn(to_f32(e[1]), 2 * i + 1);
        }
      } else {
        for (int i = tid; i < n; i += kThreads) fn(to_f32(xs[i]), i);
      }
    };
    auto sum_over = [&](auto&& weight) {     // over the cluster
      double big = 0.0, none = 0.0;
      float small = 0.f;
      each([&](float x, int i) {
        const double v = weight(x, i);
        if (v > 2.44140625e-4) big += v;
        else small += static_cast<float>(v);
      });
      big += static_cast<double>(small);
      sum_all(big, none);
      return big;
    };

    // ---- the cut: tokens from x_cut on are kept ----
    double x_cut = -INFINITY, kept = 0.0;
    if (min_p > 0.f) x_cut = static_cast<double>(mx) + static_cast<double>(temp) * log(static_cast<double>(fminf(min_p, 1.f)));
    if (!cut_k && !cut_p) {
      kept = sum_over([&](float x, int) { return static_cast<double>(x) >= x_cut ? w(x) : 0.0; });
    } else {
      const double total = cut_p ? sum_over([&](float x, int) { return w(x); }) : 0.0;
      const double want = static_cast<double>(top_p) * total;
      double bound = x_cut;
      if (cut_k && top_k <= static_cast<int>(ranks) * (by_warps ? kWarps : 4 * kWarps)) bound = fmax(bound, static_cast<double>(low));
      // below this, all tokens of the vocabulary together hold less than what top_p leaves out (and a little, for the roundings)
      if (cut_p) bound = fmax(bound, static_cast<double>(mx) + static_cast<double>(temp) * (log(fmax((1.0 - static_cast<double>(top_p)) * total / p.vocab, 1e-300)) - 1e-6));
      each([&](float x, int) {
        if (static_cast<double>(x) >= bound) {
          const int at = atomicAdd(&sh.list_n, 1);
          if (at < kList) list[at] = x;
        }
      });
      __syncthreads();
      if (tid == 0) sh.slot[turn & 1][0] = static_cast<uint64_t>(sh.list_n);
      cluster_sync();
      int have = 0;
      if (lane < static_cast<int>(ranks)) have = static_cast<int>(min(ld_cluster64(at_rank(&sh.slot[turn & 1][0], lane)), static_cast<uint64_t>(1) << 30));
      int upto = have;          // candidates of the ranks up to this lane's
#pragma unroll
      for (int o = 1; o < kMaxCluster; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto = min(upto + v, 1 << 30);
      }
      const int m = __shfl_sync(0xffffffffu, upto, static_cast<int>(ranks) - 1);
      ++turn;
      if (m <= kList) {
        // every CTA sorts all candidates, largest first
        int size = 32;
        while (size < m) size <<= 1;
        int at = 0;
        for (uint32_t r = 0; r < ranks; ++r) {
          const int c_n = __shfl_sync(0xffffffffu, have, r);
          const uint32_t from = at_rank(list, r);
          for (int i = tid; i < c_n; i += kThreads) sorted[at + i] = __uint_as_float(ld_cluster32(from + 4 * i));
          at += c_n;
        }
        for (int i = m + tid; i < size; i += kThreads) sorted[i] = -INFINITY;
        __syncthreads();
        for (int span = 2; span <= size; span <<= 1) {
          for (int step = span >> 1; step > 0; step >>= 1) {
            for (int i = tid; i < size / 2; i += kThreads) {
              const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
              const float a = sorted[lo], c2 = sorted[hi];
              const bool down = (lo & span) == 0;
              if (down ? a < c2 : a > c2) {
                sorted[lo] = c2;
                sorted[hi] = a;
              }
            }
            __syncthreads();
          }
        }
        // running mass, largest first: a thread has m / kThreads neighbours
        const int per = (m + kThreads - 1) / kThreads, i0 = min(m, tid * per), i1 = min(m, i0 + per);
        double mine = 0.0;
        for (int i = i0; i < i1; ++i) mine += w(sorted[i]);
        double incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
        if (lane == 31) sh.scan[warp] = incl;
        if (tid == 0) sh.owner = 0;
        __syncthreads();
        double before = incl - mine;
        for (int i = 0; i < warp; ++i) before += sh.scan[i];
        if (cut_p) {            // tokens with less than `want` in front of them are inside
          int inside = 0;
          double run = before;
          for (int i = i0; i < i1; ++i) {
            if (run < want) inside = i + 1;
            run += w(sorted[i]);
          }
          if (inside > 0) atomicMax(&sh.owner, inside);
        }
        __syncthreads();
        // fewer candidates (less mass) than asked for: the other filter's bound was higher, and so is its cut
        if (cut_k && top_k <= m) x_cut = fmax(x_cut, static_cast<double>(sorted[top_k - 1]));
        const int inside = max(sh.owner, 1);
        if (cut_p && m > 0) x_cut = fmax(x_cut, static_cast<double>(sorted[min(inside, m) - 1]));
        double sum = 0.0, none = 0.0;
        for (int i = i0; i < i1; ++i) sum += static_cast<double>(sorted[i]) >= x_cut ? w(sorted[i]) : 0.0;
        // the same sums in every CTA: no exchange
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += shfl_xor_d(sum, o);
        if (lane == 0) sh.red[warp][0] = sum;
        __syncthreads();
        for (int i = 0; i < kWarps; ++i) none += sh.red[i][0];
        kept = none;
        __syncthreads();
      } else {
        // flat rows: the largest key with k tokens (with the wanted mass) at or above it, bit by bit
        uint32_t at_k = 0, at_p = 0;
        for (int bit = 31; bit >= 0; --bit) {
          const uint32_t try_k = at_k | 1u << bit, try_p = at_p | 1u << bit;
          double tokens = 0.0, mass = 0.0;
          float small = 0.f;
          each([&](float x, int) {
            const uint32_t k = key_of(x);
            if (cut_k && k >= try_k) tokens += 1.0;
            if (cut_p && k >= try_p) {
              const double v = w(x);
              if (v > 2.44140625e-4) mass += v;
              else small += static_cast<float>(v);
            }
          });
          mass += static_cast<double>(small);
          sum_all(tokens, mass);
          if (cut_k && tokens >= static_cast<double>(top_k)) at_k = try_k;
          if (cut_p && mass >= want && mass > 0.0) at_p = try_p;
        }
        if (cut_k && at_k != 0) x_cut = fmax(x_cut, static_cast<double>(of_key(at_k)));
        if (cut_p && at_p != 0) x_cut = fmax(x_cut, static_cast<double>(of_key(at_p)));
        kept = sum_over([&](float x, int) { return static_cast<double>(x) >= x_cut ? w(x) : 0.0; });
      }
    }

    // ---- the children in turn ----
    __syncthreads();
    if (tid < children) {
      const float x = static_cast<float>(sh.child_w[tid]);
      sh.child_w[tid] = sh.child_token[tid] >= 0 && static_cast<double>(x) >= x_cut ? w(x) : 0.0;
    }
    __syncthreads();
    int rejected = 0;           // rejections that changed p (with probabilities), or tokens taken out
    double mass = kept;         // of what is left, before it is scaled to 1
    if (p.draft == nullptr) {
      for (int i = 0; i < children; ++i) {
        double v = sh.child_w[i];
        const int token = sh.child_token[i];
        for (int k = 0; k < rejected; ++k)
          if (sh.removed[k] == token) v = 0.0;
        if (static_cast<double>(sh.child_u[i]) * mass < v) {
          taken = i;
          break;
        }
        if (v > 0.0 && mass - v > 0.0) {
          mass -= v;
          if (tid == 0) sh.removed[rejected] = token;
          ++rejected;
          __syncthreads();
        }
      }
    } else {
      const float* draft = p.draft + row * p.draft_stride;
      // p after k rejections, of the token with weight v and draft probability q
      auto left = [&](double v, double q, int k) {
        for (int j = 0; j < k && v > 0.0; ++j) v = fmax(v * sh.scale[j] - q, 0.0);
        return v;
      };
      for (int i = 0; i < children; ++i) {
        const double q = sh.child_q[i];
        const double v = sh.child_token[i] < 0 ? 0.0 : left(sh.child_w[i], q, rejected);
        if (static_cast<double>(sh.child_u[i]) * q * mass < v) {
          taken = i;
          break;
        }
        if (sh.child_token[i] < 0) continue;
        const double scale = 1.0 / mass;
        const double rest = sum_over([&](float x, int id) {
          if (!(static_cast<double>(x) >= x_cut)) return 0.0;
          const double q_id = __ldcg(draft + v0 + id);
          return fmax(left(w(x), q_id, rejected) * scale - q_id, 0.0);
        });
        if (rest > 0.0) {
          if (tid == 0) sh.scale[rejected] = scale;
          ++rejected;
          mass = rest;
          __syncthreads();
        }
      }
    }
    if (rank == 0 && tid == 0) p.path[static_cast<int64_t>(b) * p.steps + count] = node;
    if (taken >= 0) {
      const int next = sh.child[taken];
      if (rank == 0 && tid == 0) p.out[static_cast<int64_t>(b) * p.steps + count] = sh.child_token[taken];
      ++count;
      node = next;
      __syncthreads();
      continue;
    }

    // ---- the walk's last token: the first whose running sum passes u times all ----
    {
      const float* draft = p.draft != nullptr ? p.draft + row * p.draft_stride + v0 : nullptr;
      auto weight = [&](int i) {
        const float x = to_f32(xs[i]);
        if (!(static_cast<double>(x) >= x_cut)) return 0.0;
        double v = w(x);
        if (draft != nullptr) {
          if (rejected > 0) {
            const double q = __ldcg(draft + i);
            for (int j = 0; j < rejected && v > 0.0; ++j) v = fmax(v * sh.scale[j] - q, 0.0);
          }
        } else {
          for (int k = 0; k < rejected; ++k)
            if (sh.removed[k] == v0 + i) v = 0.0;
        }
        return v;
      };
      const int per = (n + kThreads - 1) / kThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
      double mine = 0.0;
      {
        float small = 0.f;
        for (int i = i0; i < i1; ++i) {
          const double v = weight(i);
          if (v > 2.44140625e-4) mine += v;
          else small += static_cast<float>(v);
        }
        mine += static_cast<double>(small);
      }
      double incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) sh.scan[warp] = incl;
      __syncthreads();
      double before = incl - mine, here = 0.0;
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) before += sh.scan[i];
        here += sh.scan[i];
      }
      if (tid == 0) {
        sh.slot[turn & 1][0] = static_cast<uint64_t>(__double_as_longlong(here));
        sh.owner = -1;
      }
      cluster_sync();
      double part = 0.0;
      if (lane < static_cast<int>(ranks)) part = __longlong_as_double(static_cast<long long>(ld_cluster64(at_rank(&sh.slot[turn & 1][0], lane))));
      double all = 0.0, front = 0.0;
      for (uint32_t r = 0; r < ranks; ++r) all += __shfl_sync(0xffffffffu, part, r);
      const double target = static_cast<double>(u_final) * all;
      int winner = -1;          // the last part with mass that begins at or before the target
      {
        double run = 0.0;
        for (uint32_t r = 0; r < ranks; ++r) {
          const double v = __shfl_sync(0xffffffffu, part, r);
          if (v > 0.0 && run <= target) {
            winner = static_cast<int>(r);
            front = run;
          }
          run += v;
        }
      }
      ++turn;
      if (winner == static_cast<int>(rank)) {
        if (mine > 0.0 && front + before <= target) atomicMax(&sh.owner, tid);
        __syncthreads();
        if (tid == sh.owner) {
          double run = front + before;
          int pick = -1, last = -1;
          for (int i = i0; i < i1; ++i) {
            const double v = weight(i);
            if (v > 0.0) {
              run += v;
              last = i;
              if (run > target) {
                pick = i;
                break;
              }
            }
          }
          p.out[static_cast<int64_t>(b) * p.steps + count] = v0 + (pick >= 0 ? pick : last);
        }
      } else if (winner < 0 && rank == 0 && tid == 0) {
        p.out[static_cast<int64_t>(b) * p.steps + count] = first_best;      // nothing left to draw from
      }
    }
    ++count;
    break;
  }
  finish_row(count);
  if (rank == 0 && tid == 0) p.counts[b] = count;
  cluster_sync();               // no CTA leaves while its slots may be read
}

template <typename T>
int launch_type(const SampleParams& p, int cluster, int batch, cudaStream_t s) {
  auto kernel = tree_sample_kernel<T>;
  const int smem = 2 * kList * 4 + p.chunk * static_cast<int>(sizeof(T));
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem) != cudaSuccess) return -3;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(cluster * batch));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p);
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}

}  // namespace

// Bytes of shared memory that a CTA may use for its part of a row: 227 KB less the candidates and the kernel's variables.
constexpr int kPartBytes = 184 * 1024;

int tree_sample_max_vocab(DType dt) { return kMaxCluster * (kPartBytes / (dt == kF32 ? 4 : 2)); }

int launch_tree_sample(const TreeSampleArgs& a, cudaStream_t s) {
  if (a.batch <= 0 || a.steps <= 0) return 0;
  if (a.vocab <= 0 || a.vocab > tree_sample_max_vocab(a.dt)) return -1;
  SampleParams p{};
  p.logits = a.logits;
  p.tokens = a.tokens;
  p.parents = a.parents;
  p.tree_lens = a.tree_lens;
  p.q_start = a.q_start;
  p.temperature = a.temperature;
  p.top_k = a.top_k;
  p.top_p = a.top_p;
  p.min_p = a.min_p;
  p.uniform = a.uniform;
  p.uniform_final = a.uniform_final;
  p.draft = a.draft;
  p.path = a.path;
  p.out = a.out;
  p.counts = a.counts;
  p.status = a.status;
  p.logit_stride = a.logit_stride;
  p.draft_stride = a.draft_stride;
  p.rows = a.rows;
  p.vocab = a.vocab;
  p.steps = a.steps;
  // CTAs per request: about 16384 tokens each
  int cluster = 1;
  while (cluster < kMaxCluster && cluster * 16384 < a.vocab) cluster *= 2;
  const int item = a.dt == kF32 ? 4 : 2;
  p.chunk = ((a.vocab + cluster - 1) / cluster + 7) / 8 * 8;
  if (p.chunk * item > kPartBytes) return -1;
  p.vec = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.logit_stride * item % 16 == 0 ? 1 : 0;
  switch (a.dt) {
    case kBF16: return launch_type<__nv_bfloat16>(p, cluster, a.batch, s);
    case kF16: return launch_type<__half>(p, cluster, a.batch, s);
    default: return launch_type<float>(p, cluster, a.batch, s);
  }
}

}  // namespace mb200
