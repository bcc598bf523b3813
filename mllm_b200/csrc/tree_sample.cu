// Verification of drafted token trees against the target's filtered distribution, with random numbers that the caller gives.
//
// A request's walk begins at node 0.  At a node with logits l, temperature T and filters,
//   e_i = exp((l_i - max l) / T),   kept = {i: e_i >= the k-th largest, >= the smallest whose strictly larger mass is below top_p * sum e,
//   >= min_p}  (ties are kept),   p = e / sum over kept.
// The node's children are looked at in the order of their numbers: child c with token x is taken if u_c q(x) < p(x); otherwise
// p <- max(p - q, 0) / sum, where q is the distribution that the children were drawn from, each by itself, or all of x (candidates without
// probabilities).  Without a child that is taken the walk ends with the first token whose running sum of p, in the order of the ids,
// passes u * sum p.  The emitted tokens are distributed as the target's own samples, whatever the draft.
//
// What a step reads is known when the step before is done, so a walk is a chain: row, maximum, sum, cut, children, row.  A cluster of up
// to 8 CTAs takes a request; each holds its part of the row in shared memory, and what they share goes through one exchange (a slot per
// CTA, one cluster barrier) per stage.  The cut needs no sort of the row and no histogram: a lower bound on it (the k-th largest of the
// warps' maxima for top-k, a level that holds the wanted mass for top-p, min_p itself) leaves a few tokens, which every CTA collects and
// sorts for itself.  Where more than kList are left (flat distributions) the cut is closed in on, seven parts of its range an exchange.
//
// A step of a small batch takes some 9 us, nearly all of it latency: five exchanges of 1 to 1.5 us (two or three more where top-p has to
// look twice), the row (0.3 MB over 8 SMs), one way through it in shared memory.  Steps and filters follow from the random numbers: on the
// device 1 request of 8 nodes, 151936 tokens takes 31 to 70 us; 8 of 16 nodes with draft probabilities 65 to 80; 32 of 24 nodes, 128256 tokens, two
// CTAs on an SM, 90 to 137, once 174.
//
// Whole tokens hang on sums: e is taken in 64 bits where it is above 2^-12, and threads' sums are joined in 64 bits.  Smaller ones are 32-bit
// (fp64 exponentials of a whole vocabulary would bound the kernel): off by less than 2^-19 each, 2^-22 from the exponential and half a step of
// an argument of up to 32, twice; a thread adds them up in 32 bits, a rounding a term.  So a token's border is off by some 10^-9 of the whole
// where the mass is in few tokens, and by less than 2^-18 of the mass below 2^-12 (vocabularies of 151936) where it is in many.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "tree.h"

namespace mb200 {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kList = 4096;               // candidates that are sorted
constexpr int kChildren = 64;             // of a node that are looked at
constexpr int kMore = 6;                  // further sums of an exchange
constexpr float kLevelStep = 2.f;         // first guesses at the cut: so much apart below the largest logit, in units of T

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
// Order of floats as order of whole numbers; a value that is no number counts as minus infinity, and zeros are alike.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0x007fffffu;
  return x == 0.f ? 0x80000000u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
// The same for values of T: numbers without the bits that T does not have, and back.
template <typename T>
struct Keys {
  static constexpr int kDrop = std::is_same<T, __nv_bfloat16>::value ? 16 : std::is_same<T, __half>::value ? 13 : 0;
  static __device__ __forceinline__ uint32_t of(float x) { return key_of(x) >> kDrop; }
  static __device__ __forceinline__ float value(uint32_t k) {
    uint32_t u = k << kDrop;
    if (u & 0x80000000u) return __uint_as_float(u & 0x7fffffffu);
    return __uint_as_float(~(u | ((1u << kDrop) - 1)));
  }
};
__device__ __forceinline__ double shfl_xor_d(double v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// The weight e of a token: above 2^-12 in 64 bits, below in 32.
struct Scale {
  // A largest logit of infinity: infinite logits have weight 1, all others none.  Differences are then taken from the largest finite
  // number, with both parts of the factor 1: log2_of gives infinity for infinite logits, which no sum of loops over tokens has to look for.
  float mx, off, c_hi, c_lo;     // largest logit; it, or the largest finite number; log2(e) / T as two floats
  double inv_t, mx_d;
  __device__ __forceinline__ Scale(float largest, float temp)
      : mx(largest), off(fminf(largest, 3.402823466e38f)), inv_t(1.0 / static_cast<double>(temp)), mx_d(largest) {
    const double c = 1.4426950408889634 * inv_t;
    c_hi = mx == off ? static_cast<float>(c) : 1.f;
    c_lo = mx == off ? static_cast<float>(c - static_cast<double>(c_hi)) : 1.f;
  }
  __device__ __forceinline__ float log2_of(float x) const {
    const float d = fmaxf(x - off, -1e30f);      // a value that is no number, or minus infinity: no weight
    return fmaf(d, c_hi, d * c_lo);
  }
  __device__ __forceinline__ double large(float x) const { return x == mx ? 1.0 : exp((static_cast<double>(x) - mx_d) * inv_t); }
  __device__ __forceinline__ double operator()(float x) const {
    if (!(x == x)) return 0.0;
    const float t = log2_of(x);
    return t > -12.f ? large(x) : static_cast<double>(fast_exp2(t));
  }
  // adds it to a sum of two parts, for loops over all tokens
  __device__ __forceinline__ void add(float x, double& big, float& small) const {
    const float t = log2_of(x);
    if (t > -12.f) big += large(x);
    else small += fast_exp2(t);
  }
};

struct Shared {
  uint64_t slot[2][8];          // what this CTA tells the others, alternating
  double red[kWarps][2];
  double red_more[kWarps][kMore];
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
  int children, owner, found;
  double scan[kWarps];
  float group_max[kWarps];      // the warps' largest values, for the others
  alignas(16) float all_max[kMaxCluster * kWarps];
  float low;
};

template <typename T, int PER_SM>
__global__ void __launch_bounds__(kThreads, PER_SM) tree_sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Shared sh;
  float* list = reinterpret_cast<float*>(dyn);              // this CTA's candidates
  float* gathered = list + kList;                           // all candidates
  float* sorted = gathered + kList;
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

  // Sums over the cluster, the same bits for every thread: two, and kMore others where `more` is given (lane i of every warp gets the i-th).
  // `count`: a number of this CTA's (thread 0's counts), its sum in return.
  auto sum_all = [&](double& a, double& c, double (*more)[kMore] = nullptr, int* count = nullptr) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += shfl_xor_d(a, o);
      c += shfl_xor_d(c, o);
    }
    if (more != nullptr) {
#pragma unroll
      for (int i = 0; i < kMore; ++i) {
        double v = (*more)[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += shfl_xor_d(v, o);
        if (lane == 0) sh.red_more[warp][i] = v;
      }
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
        if (count != nullptr) sh.slot[turn & 1][2 + kMore - 1] = static_cast<uint64_t>(*count);
      }
      if (more != nullptr && lane < kMore) {
        double v = 0.0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) v += sh.red_more[i][lane];
        sh.slot[turn & 1][2 + lane] = static_cast<uint64_t>(__double_as_longlong(v));
      }
    }
    cluster_sync();
    double x = 0.0, y = 0.0;
    if (lane < static_cast<int>(ranks)) {
      const uint32_t from = at_rank(&sh.slot[turn & 1][0], lane);
      x = __longlong_as_double(static_cast<long long>(ld_cluster64(from)));
      y = __longlong_as_double(static_cast<long long>(ld_cluster64(from + 8)));
    }
    if (more != nullptr) {
      double v = 0.0;
      if (lane < kMore) {
        double from[kMaxCluster];
#pragma unroll
        for (uint32_t r = 0; r < kMaxCluster; ++r)
          from[r] = r < ranks ? __longlong_as_double(static_cast<long long>(ld_cluster64(at_rank(&sh.slot[turn & 1][2 + lane], r)))) : 0.0;
#pragma unroll
        for (uint32_t r = 0; r < kMaxCluster; ++r) v += from[r];
      }
      (*more)[0] = v;
    }
#pragma unroll
    for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
      x += shfl_xor_d(x, o);
      y += shfl_xor_d(y, o);
    }
    a = __shfl_sync(0xffffffffu, x, 0);
    c = __shfl_sync(0xffffffffu, y, 0);
    if (count != nullptr) {
      int v = lane < static_cast<int>(ranks) ? static_cast<int>(ld_cluster64(at_rank(&sh.slot[turn & 1][2 + kMore - 1], lane))) : 0;
      *count = __reduce_add_sync(0xffffffffu, v);
    }
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
    if (tid < 8 && n + tid < (n + 7) / 8 * 8) xs[n + tid] = from_f32<T>(-INFINITY);
    // Groups of 32 lanes (or 8, for a larger k): that many tokens are at least as large as the smallest of their maxima, and k as the k-th
    // largest.
    const bool by_warps = top_k <= static_cast<int>(ranks) * kWarps;
    float g_max = best;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) g_max = fmaxf(g_max, __shfl_xor_sync(0xffffffffu, g_max, o));
    float low = g_max;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
      g_max = fmaxf(g_max, __shfl_xor_sync(0xffffffffu, g_max, o));
      const uint64_t k = __shfl_xor_sync(0xffffffffu, top, o);
      top = k > top ? k : top;
    }
    if (lane == 0) sh.group_max[warp] = g_max;
    if (lane == 0) {
      sh.red_key[warp] = top;
      sh.red_min[warp] = low;
    }
    if (tid == 0) {
      sh.list_n = 0;
      sh.found = 0;
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
    if (cut_k && by_warps && temp > 1e-6f) {
      // up to 128 maxima: the one that k - 1 others precede
      if (tid < kMaxCluster * kWarps)
        sh.all_max[tid] = tid < static_cast<int>(ranks) * kWarps ? __uint_as_float(ld_cluster32(at_rank(&sh.group_max[tid % kWarps], tid / kWarps)))
                                                                 : -INFINITY;
      __syncthreads();
      if (tid < kMaxCluster * kWarps) {
        const float mine = sh.all_max[tid];
        int before = 0;
#pragma unroll 8
        for (int j = 0; j < kMaxCluster * kWarps; j += 4) {
          const float4 y = *reinterpret_cast<const float4*>(sh.all_max + j);
          before += (y.x > mine || (y.x == mine && j < tid)) + (y.y > mine || (y.y == mine && j + 1 < tid)) +
                    (y.z > mine || (y.z == mine && j + 2 < tid)) + (y.w > mine || (y.w == mine && j + 3 < tid));
        }
        if (before == top_k - 1) sh.low = mine;
      }
      __syncthreads();
      low = sh.low;
    }
    const float mx = Keys<float>::value(static_cast<uint32_t>(top >> 32));
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

    const Scale w(mx, temp);
    const int groups = (n + 7) / 8;          // of eight tokens; minus infinity behind the last token
    auto eight = [&](int i, float (&x)[8]) {
      if constexpr (sizeof(T) == 2) {
        const uint4 v = reinterpret_cast<const uint4*>(xs)[i];
        const T* h = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = to_f32(h[k]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; k += 4) *reinterpret_cast<float4*>(x + k) = reinterpret_cast<const float4*>(xs)[2 * i + k / 4];
      }
    };
    // x >= bound (in 64 bits) for all x of 32: x >= the next float up
    auto up = [](double v) { return __double2float_ru(v); };
    // One way through this CTA's part, eight tokens at a time: a list of the tokens from `least` on, the weights of those from `from` on and
    // of the listed ones (least >= from).
    auto sweep = [&](bool summed, float from, bool listed, float least) {
      double big = 0.0, in_list = 0.0;
      float small[4] = {};
      for (int i = tid; i < groups; i += kThreads) {
        float x[8];
        eight(i, x);
        unsigned apart = 0;            // tokens with a large weight, and those for the list
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float t = w.log2_of(x[k]);
          const bool special = (summed && t > -12.f) || (listed && x[k] >= least);
          apart |= special ? 1u << k : 0u;
          if (summed) small[k & 3] += x[k] >= from && !special ? fast_exp2(t) : 0.f;
        }
        while (apart != 0) {
          const float v = to_f32(xs[8 * i + __ffs(apart) - 1]);
          apart &= apart - 1;
          if (listed && v >= least) {
            const int at = atomicAdd(&sh.list_n, 1);
            if (at < kList) list[at] = v;
            if (summed) in_list += w(v);
          } else if (v >= from) {
            w.add(v, big, small[0]);
          }
        }
      }
      return make_double2(big + in_list + static_cast<double>((small[0] + small[1]) + (small[2] + small[3])), in_list);
    };
    auto sum_kept = [&](float from) {        // over the cluster
      double a = sweep(true, from, false, 0.f).x, none = 0.0;
      sum_all(a, none);
      return a;
    };
    // below this, all tokens of the vocabulary together hold less than top_p leaves out (and a little, for the roundings)
    auto surely_inside = [&](double total) {
      const double share = fmax((1.0 - static_cast<double>(top_p)) * total / p.vocab, 1e-300);
      return up(static_cast<double>(mx) + static_cast<double>(temp) * (log(share) - 1e-6)) - 1e-6f * fabsf(mx);
    };

    // ---- the cut: tokens from x_cut on are kept ----
    float x_cut = -INFINITY;
    double kept = 0.0;
    if (min_p > 0.f) x_cut = up(static_cast<double>(mx) + static_cast<double>(temp) * log(static_cast<double>(fminf(min_p, 1.f))));
    if (!cut_k && !cut_p) {
      kept = sum_kept(x_cut);
    } else {
      // Candidates: tokens from a bound on the cut upwards, listed on the way through the row that forms the sum.  For top_p the bound
      // is a guess, 14 T below the largest logit.
      float bound = x_cut;
      if (cut_k && top_k <= static_cast<int>(ranks) * (by_warps ? kWarps : 4 * kWarps)) bound = fmaxf(bound, low);
      const float from = fmaxf(bound, cut_p ? mx - (kMore + 1) * kLevelStep * temp : -INFINITY);
      const double2 sums = sweep(cut_p, -INFINITY, true, from);
      __syncthreads();
      double total = sums.x, mass = sums.y;
      int listed = sh.list_n > kList ? 1 << 24 : sh.list_n;
      int told = turn;            // the exchange that says how long the lists are
      sum_all(total, mass, nullptr, &listed);
      const double want = static_cast<double>(top_p) * total;
      bool have = listed <= kList;
      if (cut_p && have && listed <= 2 * kThreads && mass >= want) {
        bound = from;
      } else if (cut_p) {
        // the mass above some levels: the highest that holds what top_p wants is a better bound
        // (which tokens a full list lacks, and the order of a list, are left to chance: from the row itself then, and of whole
        // multiples of 2^-40, whose sums are exact in any order)
        double above[kMore] = {}, none = 0.0, none2 = 0.0;
        const bool in_list = sh.list_n <= kList;
        for (int i = tid; i < (in_list ? sh.list_n : n); i += kThreads) {
          const float x = in_list ? list[i] : to_f32(xs[i]);
          if (!(x >= mx - kMore * kLevelStep * temp)) continue;
          const double v = floor(w(x) * 0x1p40) * 0x1p-40;
#pragma unroll
          for (int l = 0; l < kMore; ++l)
            if (x >= mx - (l + 1) * kLevelStep * temp) above[l] += v;
        }
        sum_all(none, none2, &above);
        const unsigned enough = __ballot_sync(0xffffffffu, lane < kMore && above[0] >= want);
        if (enough != 0) {
          bound = fmaxf(bound, mx - __ffs(enough) * kLevelStep * temp);
        } else if (have && mass >= want) {
          bound = from;
        } else {
          bound = fmaxf(bound, surely_inside(total));
          have = have && bound >= from;
        }
      }
      int m = 0;
      if (!have) {            // once more, from the better bound
        __syncthreads();
        if (tid == 0) sh.list_n = 0;
        __syncthreads();
        sweep(false, 0.f, true, bound);
        __syncthreads();
        double none = 0.0, none2 = 0.0;
        int all = sh.list_n > kList ? 1 << 24 : sh.list_n;
        told = turn;
        sum_all(none, none2, nullptr, &all);
        have = all <= kList;
      }
      if (have) {
        // every CTA gathers all candidates from the bound on; how many each has was told with the sums
        int upto = 0;
        if (lane < static_cast<int>(ranks)) upto = static_cast<int>(ld_cluster64(at_rank(&sh.slot[told & 1][2 + kMore - 1], lane)));
#pragma unroll
        for (int o = 1; o < kMaxCluster; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        const int everything = __shfl_sync(0xffffffffu, upto, static_cast<int>(ranks) - 1);
        for (int i0 = warp * 32; i0 < everything; i0 += kThreads) {
          const int i = i0 + lane;
          int r = 0, front = 0;
          for (uint32_t q = 0; q + 1 < ranks; ++q) {
            const int end = __shfl_sync(0xffffffffu, upto, q);
            if (i >= end) {
              r = q + 1;
              front = end;
            }
          }
          const float x = i < everything ? __uint_as_float(ld_cluster32(at_rank(list, r) + 4 * (i - front))) : -INFINITY;
          const bool in = i < everything && x >= bound;
          const unsigned votes = __ballot_sync(0xffffffffu, in);
          int at = 0;
          if (lane == 0 && votes != 0) at = atomicAdd(&sh.found, __popc(votes));
          at = __shfl_sync(0xffffffffu, at, 0) + __popc(votes & ((1u << lane) - 1));
          if (in) gathered[at] = x;
        }
        __syncthreads();
        m = sh.found;
        // ---- largest first ----
        if (m <= 2 * kThreads) {
          // an element's place is the number of those in front of it
          for (int i = m + tid; i < (m + 3) / 4 * 4; i += kThreads) gathered[i] = -INFINITY;
          __syncthreads();
          for (int i = tid; i < m; i += kThreads) {
            const float x = gathered[i];
            int place = 0;
            for (int j = 0; j < m; j += 4) {
              const float4 y = *reinterpret_cast<const float4*>(gathered + j);
              place += (y.x > x || (y.x == x && j < i)) + (y.y > x || (y.y == x && j + 1 < i)) + (y.z > x || (y.z == x && j + 2 < i)) +
                       (y.w > x || (y.w == x && j + 3 < i));
            }
            sorted[place] = x;
          }
          __syncthreads();
        } else {
          int size = 2 * kThreads;
          while (size < m) size <<= 1;
          for (int i = tid; i < size; i += kThreads) sorted[i] = i < m ? gathered[i] : -INFINITY;
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
        }
        // running mass: a thread has m / kThreads neighbours
        const int per = (m + kThreads - 1) / kThreads, i0 = min(m, tid * per), i1 = min(m, i0 + per);
        const double w0 = i0 < i1 ? w(sorted[i0]) : 0.0;
        auto weight_at = [&](int i) { return i == i0 ? w0 : w(sorted[i]); };
        double mine = 0.0;
        for (int i = i0; i < i1; ++i) mine += weight_at(i);
        double incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
        if (lane == 31) sh.scan[warp] = incl;
        if (tid == 0) sh.owner = 0;
        __syncthreads();
        if (cut_p) {            // tokens with less than `want` in front of them are inside
          double run = incl - mine;
          for (int i = 0; i < warp; ++i) run += sh.scan[i];
          int inside = 0;
          for (int i = i0; i < i1; ++i) {
            if (run < want) inside = i + 1;
            run += weight_at(i);
          }
          inside = __reduce_max_sync(0xffffffffu, inside);
          if (lane == 0 && inside > 0) atomicMax(&sh.owner, inside);
          __syncthreads();
        }
        // fewer candidates (less mass) than asked for: the other filter's bound was higher, and so is its cut
        if (cut_k && top_k <= m) x_cut = fmaxf(x_cut, sorted[top_k - 1]);
        if (cut_p && m > 0) x_cut = fmaxf(x_cut, sorted[min(max(sh.owner, 1), m) - 1]);
        double sum = 0.0;
        for (int i = i0; i < i1; ++i) sum += sorted[i] >= x_cut ? weight_at(i) : 0.0;
        // the same sums in every CTA: no exchange
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += shfl_xor_d(sum, o);
        if (lane == 0) sh.red[warp][0] = sum;
        __syncthreads();
        for (int i = 0; i < kWarps; ++i) kept += sh.red[i][0];
        __syncthreads();
      } else {
        // Flat rows: the largest value with k tokens (with the wanted mass) at or above it, among the type's values between the bound and
        // the largest logit; six of them a sweep and an exchange.
        auto largest = [&](bool by_mass, double goal) {
          uint32_t at = Keys<T>::of(bound), span = Keys<T>::of(mx) + 1 - at;
          while (span > 1) {
            const uint32_t step = (span + kMore) / (kMore + 1);
            float test[kMore], small[kMore] = {};
            double sums[kMore] = {}, none = 0.0, none2 = 0.0;
#pragma unroll
            for (int j = 0; j < kMore; ++j) test[j] = (j + 1) * step < span ? Keys<T>::value(at + (j + 1) * step) : NAN;
            for (int i = tid; i < groups; i += kThreads) {
              float x[8], x_top = -INFINITY;
              eight(i, x);
#pragma unroll
              for (int k = 0; k < 8; ++k) x_top = fmaxf(x_top, x[k]);
              if (!(x_top >= test[0])) continue;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float lg = w.log2_of(x[k]);
                if (by_mass && lg > -12.f) {
                  const double v = w.large(x[k]);
#pragma unroll
                  for (int j = 0; j < kMore; ++j) sums[j] += x[k] >= test[j] ? v : 0.0;
                } else {
                  const float v = by_mass ? fast_exp2(lg) : 1.f;
#pragma unroll
                  for (int j = 0; j < kMore; ++j) small[j] += x[k] >= test[j] ? v : 0.f;
                }
              }
            }
#pragma unroll
            for (int j = 0; j < kMore; ++j) sums[j] += static_cast<double>(small[j]);
            sum_all(none, none2, &sums);
            const uint32_t steps = __popc(__ballot_sync(0xffffffffu, lane < kMore && sums[0] >= goal && sums[0] > 0.0));
            at += steps * step;
            span = min(step, span - steps * step);
          }
          return Keys<T>::value(at);
        };
        if (cut_k) x_cut = fmaxf(x_cut, largest(false, static_cast<double>(top_k)));
        if (cut_p) x_cut = fmaxf(x_cut, largest(true, want));
        kept = sum_kept(x_cut);
      }
    }

    // What a kept token has left after k rejections with probabilities, added to a sum of two parts: in 64 bits where the weight or the
    // draft's probability is above 2^-12.  The sums and the draw share it: a thread that has mass has a token.
    auto add_left = [&](float x, float q, int k, double& big, float& small) {
      const float t = w.log2_of(x);
      if (t > -12.f || q > 2.44140625e-4f) {
        double v = w(x);
        for (int j = 0; j < k && v > 0.0; ++j) v = fmax(v * sh.scale[j] - q, 0.0);
        big += v;
      } else {
        float v = fast_exp2(t);
        for (int j = 0; j < k && v > 0.f; ++j) v = fmaxf(fmaf(v, static_cast<float>(sh.scale[j]), -q), 0.f);
        small += v;
      }
    };
    const float* draft = p.draft != nullptr ? p.draft + row * p.draft_stride + v0 : nullptr;
    const bool wide = (reinterpret_cast<uintptr_t>(draft) & 15) == 0;
    // of eight tokens, added to `sum`
    auto left_of_eight = [&](int g, int k, double& sum) {
      float x[8], x_top = -INFINITY;
      eight(g, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x_top = fmaxf(x_top, x[e]);
      if (!(x_top >= x_cut) || x_top == -INFINITY) return;
      float q[8];
      if (wide && 8 * g + 8 <= n) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) *reinterpret_cast<float4*>(q + e) = __ldcg(reinterpret_cast<const float4*>(draft + 8 * g + e));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = 8 * g + e < n ? __ldcg(draft + 8 * g + e) : 0.f;
      }
      float small = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (x[e] >= x_cut) add_left(x[e], q[e], k, sum, small);
      sum += static_cast<double>(small);
    };

    // ---- the children in turn ----
    __syncthreads();
    if (tid < children) {
      const float x = static_cast<float>(sh.child_w[tid]);
      sh.child_w[tid] = sh.child_token[tid] >= 0 && x >= x_cut ? w(x) : 0.0;
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
        if (tid == 0) sh.scale[rejected] = scale;
        __syncthreads();
        double rest = 0.0, none = 0.0;
        for (int g = tid; g < groups; g += kThreads) left_of_eight(g, rejected + 1, rest);
        sum_all(rest, none);
        if (rest > 0.0) {
          ++rejected;
          mass = rest;
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
      auto weight = [&](int i) {
        const float x = to_f32(xs[i]);
        if (!(x >= x_cut)) return 0.0;
        if (draft != nullptr) {
          double big = 0.0;
          float small = 0.f;
          add_left(x, rejected > 0 ? __ldcg(draft + i) : 0.f, rejected, big, small);
          return big + small;
        }
        for (int k = 0; k < rejected; ++k)
          if (sh.removed[k] == v0 + i) return 0.0;
        return w(x);
      };
      // neighbouring tokens, a thread's share of them
      const int per = (groups + kThreads - 1) / kThreads, g0 = min(groups, tid * per), g1 = min(groups, g0 + per);
      const int i0 = g0 * 8, i1 = min(n, g1 * 8);
      double mine = 0.0;
      for (int g = g0; g < g1; ++g) {
        if (draft != nullptr && rejected > 0) {
          left_of_eight(g, rejected, mine);
          continue;
        }
        float x[8], small = 0.f;
        eight(g, x);
        unsigned out = 0;       // candidates that were taken out
        for (int k = 0; k < rejected; ++k) {
          const int d = sh.removed[k] - v0 - 8 * g;
          out |= d >= 0 && d < 8 ? 1u << d : 0u;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (x[e] >= x_cut && !((out >> e) & 1)) w.add(x[e], mine, small);
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
          p.out[static_cast<int64_t>(b) * p.steps + count] = last < 0 ? first_best : v0 + (pick >= 0 ? pick : last);
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
int launch_type(const SampleParams& p, int cluster, int batch, bool two, cudaStream_t s) {
  auto kernel = two ? tree_sample_kernel<T, 2> : tree_sample_kernel<T, 1>;
  const int smem = 3 * kList * 4 + p.chunk * static_cast<int>(sizeof(T));
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
constexpr int kPartBytes = 168 * 1024, kTwoBytes = 56 * 1024;      // of a row, for one CTA per SM and for two

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
  // CTAs per request: no more than 8192 tokens each, up to 8 (16 requests, 32000 tokens: 57 us; 16384 each 109, 4096 each 56; 8000 tokens: 53 / 53 /
  // 63).  Where all do not have an SM of their own, two share one, with half the registers (32 requests, 128256 tokens: 140 us; fewer CTAs
  // a request instead 168; with registers for two everywhere 1 request took 57 us instead of 54.5).
  const int item = a.dt == kF32 ? 4 : 2;
  int cluster = 1;
  while (cluster < kMaxCluster && cluster * 8192 < a.vocab) cluster *= 2;
  p.chunk = ((a.vocab + cluster - 1) / cluster + 7) / 8 * 8;
  if (p.chunk * item > kPartBytes) return -1;
  p.vec = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.logit_stride * item % 16 == 0 ? 1 : 0;
  const bool two = cluster * a.batch > a.num_sms && p.chunk * item <= kTwoBytes;
  switch (a.dt) {
    case kBF16: return launch_type<__nv_bfloat16>(p, cluster, a.batch, two, s);
    case kF16: return launch_type<__half>(p, cluster, a.batch, two, s);
    default: return launch_type<float>(p, cluster, a.batch, two, s);
  }
}

}  // namespace mb200
