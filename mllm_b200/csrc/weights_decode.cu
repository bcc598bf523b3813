// Decode attention (one query token per request) over the slot-indexed KV pool that also adds up how much every cached token is attended
// to: head sizes 64, 128 and 256, caches of the activation type or 8-bit floats.
//
//   s_hi = scale q_h . k_i (soft cap: c tanh(s / c)),   w_hi = 2^(s_hi log2 e - lse_h),   o_h = sum_i w_hi v_i,
//   sums_i <- decay sums_i + sum_h w_hi  over the heads h of the group; of the newest token: sums <- sum_h w_hi.
// A sink is one more term of a head's normaliser lse_h, without a value.
//
// Every key and value is read once, by the first kernel; lse_h is known when all keys of a request were seen.  The scores, 4 bytes per
// (token, head) beside 4 * head size / heads of a group bytes of keys and values, wait for it in a workspace that mostly stays in
// the L2 cache, and the second kernel makes weights of them, beside joining the partial results.
//   * The tokens of all (request, kv head) pairs form one line of 64-token tiles, laid out on the device from the lengths; every CTA takes
//     an equal run of it, and leaves at most two partial results.  (The same dealing as plain decode attention.)
//   * A warp owns 16 tokens of a tile and a ring that cp.async fills some tiles ahead; rows come by slot one by one.
//   * S^T = K Q^T and O^T += V^T P^T are warp-level products, tokens (features) as the 16 rows, heads as the 8 columns.
//   * 8-bit rows stay 8-bit in shared memory.  The order of the features in a contraction is free: a lane takes four neighbours of a row
//     (what ldmatrix gives it of 8-bit rows), and of the queries the same four; of the values it takes features 2 u and 2 u + 1 as rows u and
//     u + 8 of the product.  They widen to fp16, which holds every 8-bit float exactly, at one conversion for two; bf16 queries are
//     scaled by a power of two per head so that fp16 holds them: the largest has an exponent of 14, and what is 2^-25 times smaller than
//     that is rounded below fp16's last place, far below the fp32 sum's own rounding.
//   * Weights are rounded to 16 bits for the product with the values, and the output's normaliser sums the rounded ones, as in plain
//     decode attention.  The sums of weights have a normaliser of their own from the unrounded ones: a rounded weight that carries most of a
//     row would be off by 2^-9.  fp16 weights are held 2^7 up: fp16's last place is then 2^-32 of a warp's largest weight, and a tail of tens of
//     thousands of tokens that have less than 2^-25 each is not lost.
//
// What bounds it: memory while the first kernel streams, a start of some 6 us, and what shows of the second kernel (29 requests of about 1900
// tokens, 32 / 8 heads of 128, fp16: 56.3 us for 229 MB, where the bytes take 35; two chains of products per score save 0.5 us).  8-bit rows
// are bound by the latency of a warp's chain - rows, widening, product, exponential, transpose, product - with 12 warps on an SM to cover it: 41 % of
// the issue slots are used, 50 % of the ALU (32 requests of about 4096, 32 / 4 heads of 128, e4m3: 54.3 us, the bytes take 21).
#include <algorithm>

#include "common.cuh"
#include "evict.cuh"
#include "mma.cuh"

namespace mb200 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kWarpTokens = 16;
constexpr int kTile = kWarps * kWarpTokens;   // tokens of a tile
constexpr int kNoToken = -0x7fffffff;
constexpr int kSums = 4;                      // sums of a thread that are on their way while the normalisers are made
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleThreshold = 8.0f;     // the running maximum is raised when a score passes it by 2^8

struct DecodeParams {
  CacheIndex ix;
  WeightSums sums;
  const void* q;
  const void* k_cache;
  const void* v_cache;
  void* out;
  float* scores;     // [batch][hkv][tokens][group], log2 domain
  float* part_o;     // [CTAs][2][group][HD]
  float2* part_lse;  // [CTAs][2][group]: of the rounded weights, of the weights
  float* whole_lse;  // [batch][hq]: pairs that lie in one CTA
  const float* sink;
  int64_t q_stride, out_stride, num_slots, kv_tok_stride, kv_head_stride;
  int hkv, group, ctas, weight_ctas;
  int join_heads, joins;     // query heads that a CTA joins, and how many CTAs a pair has for that
  float scale_log2, cap_pre, cap_post, decay;   // cap_post 0: no soft cap
};

// The line: request by request, a request's kv heads in turn.  A (request, kv head) pair has a unit per tile, and kStart units
// behind them that hold no work: the time that a pair costs beside its tiles.
constexpr int kStart = 2;
__device__ __forceinline__ int tiles_of(int len) { return (len + kTile - 1) / kTile; }
__device__ __forceinline__ int units_of(const DecodeParams& p, int b) {
  const int n = tiles_of(cached_of(p.ix, b).len);
  return n > 0 ? n + kStart : 0;
}
// Returns the units of all requests in front of this thread's run of requests [first, last) and, in `total`, of all (per kv head).
__device__ __forceinline__ int scan_units(const DecodeParams& p, int* warp_sums, int& first, int& last, int& total) {
  const int per = (p.ix.batch + kThreads - 1) / kThreads;
  first = min(p.ix.batch, static_cast<int>(threadIdx.x) * per);
  last = min(p.ix.batch, first + per);
  int mine = 0;
  for (int b = first; b < last; ++b) mine += units_of(p, b);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if ((threadIdx.x & 31) >= o) incl += v;
  }
  if ((threadIdx.x & 31) == 31) warp_sums[threadIdx.x >> 5] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < static_cast<int>(threadIdx.x >> 5)) before += warp_sums[w];
    total += warp_sums[w];
  }
  return before + incl - mine;
}
// CTAs that share the line and where CTA c's run begins: a CTA is worth its set-up from four tiles on, up to 64 CTAs from two
__device__ __forceinline__ int ctas_used(int ctas, int64_t line) {
  const int64_t want = max(line / 4, min(line / 2, static_cast<int64_t>(64)));
  return static_cast<int>(min(static_cast<int64_t>(ctas), max(want, static_cast<int64_t>(1))));
}
// (A division of 64 bits takes some 500 cycles of the chain in front of the first copy.)
__device__ __forceinline__ bool fits_32(int64_t line, int ctas) { return line < (1ll << 31) && line * (ctas + 1) < (1ll << 32); }
__device__ __forceinline__ int64_t run_begin(int64_t line, int c, int ctas) {
  if (fits_32(line, ctas)) return static_cast<uint32_t>(line) * static_cast<uint32_t>(c) / static_cast<uint32_t>(ctas);
  return line * c / ctas;
}
// the last CTA whose run begins at or before x
__device__ __forceinline__ int owner_of(int64_t line, int64_t x, int ctas) {
  if (fits_32(line, ctas)) return min(ctas - 1, static_cast<int>((static_cast<uint32_t>(x + 1) * ctas - 1u) / static_cast<uint32_t>(line)));
  return static_cast<int>(min(static_cast<int64_t>(ctas) - 1, ((x + 1) * ctas - 1) / line));
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void cp16_l2(uint32_t dst, const void* src, bool valid) {
  const int sz = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(sz) : "memory");
}
// two 8-bit floats (low 16 bits) -> two fp16, exactly
template <int FMT>
__device__ __forceinline__ uint32_t widen(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu), FMT == kKvE5M2 ? __NV_E5M2 : __NV_E4M3);
  return static_cast<uint32_t>(h.x) | static_cast<uint32_t>(h.y) << 16;
}

template <int HD, int NT, int FMT>
struct Cfg {
  static constexpr int kItem = FMT == kKvSame ? 2 : 1;
  static constexpr int kRow = HD * kItem;                        // bytes
  static constexpr int kChunks = kRow / 16;                      // 16-byte pieces of a row
  static constexpr int kTensorBytes = kWarpTokens * kRow;        // a warp's K or V rows of one tile
  static constexpr int kStages = kRow == 64 ? 8 : kRow == 128 ? 4 : 3;
  static constexpr int kRing = kStages * 2 * kTensorBytes;
  static constexpr int kOutStride = HD + 4;                      // floats between the heads of a partial result: no bank conflicts
  static constexpr int kPart = NT * 8 * kOutStride * 4;          // a warp's partial result, where its ring was
  static constexpr int kRingBytes = kRing > kPart ? kRing : kPart;
  static constexpr int kSmem = kWarps * kRingBytes + 128;
  // three where the rings are small: 8-bit rows, which are widened on the way to the products, and heads of 64
  static constexpr int kPerSm = HD == 256 ? 1 : kRow <= 128 && NT == 1 ? 3 : 2;
  static_assert(kOutStride % 4 == 0 && kRingBytes % 128 == 0, "partial results are read four values at a time, rings begin on 128 bytes");
  static_assert(kPerSm * (kSmem + 4096) <= 227 * 1024, "shared memory");
  // 16-byte piece `ch` of row `row`: eight rows of one piece lie in eight different bank groups
  static __device__ __forceinline__ uint32_t at(int row, int ch) {
    return row * kRow + ((kRow == 64 ? ch ^ ((row >> 1) & 3) : ch ^ (row & 7)) << 4);
  }
};

template <typename T, int HD, int NT, int FMT>
__global__ void __launch_bounds__(kThreads, Cfg<HD, NT, FMT>::kPerSm) weights_decode_kernel(const DecodeParams p) {
  using C = Cfg<HD, NT, FMT>;
  using M = typename std::conditional<FMT == kKvSame, T, __half>::type;        // type of the products
  using Elem = typename std::conditional<FMT == kKvSame, T, uint8_t>::type;
  constexpr float kUp = std::is_same<M, __half>::value ? 7.f : 0.f;      // weights are 2^kUp times 2^(score - maximum): 2^15 at most, which fp16 holds
  extern __shared__ uint8_t smem_raw[];
  __shared__ int warp_sums[kWarps];
  __shared__ int start[3];                          // where the run begins: request, kv head, tile
  __shared__ Cached start_of;
  __shared__ float part_m[kWarps][NT * 8], part_l[kWarps][NT * 8], part_x[kWarps][NT * 8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = p.group;
  pdl_wait_loads();
  pdl_launch_dependents();   // the second kernel may lay out the line while this one streams

  int b, hk, t0;
  Cached r;
  int64_t left;
  {
    int first, last, total;
    const int before = scan_units(p, warp_sums, first, last, total);
    if (blockIdx.x == 0)
      for (int i = first; i < last; ++i)
        if (cached_of(p.ix, i).bad && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
    const int64_t line = static_cast<int64_t>(total) * p.hkv;
    const int used = ctas_used(p.ctas, line);
    if (static_cast<int>(blockIdx.x) >= used) return;
    const int64_t begin = run_begin(line, blockIdx.x, used);
    left = run_begin(line, blockIdx.x + 1, used) - begin;
    if (left <= 0) return;
    int64_t at = static_cast<int64_t>(before) * p.hkv;
    for (int i = first; i < last; ++i) {
      const int n = units_of(p, i);
      if (begin >= at && begin < at + static_cast<int64_t>(n) * p.hkv) {
        const int in = static_cast<int>(begin - at), h = in / n;
        start[0] = i;
        start[1] = h;
        start[2] = in - h * n;
        start_of = cached_of(p.ix, i);
      }
      at += static_cast<int64_t>(n) * p.hkv;
    }
    __syncthreads();
    b = start[0];
    hk = start[1];
    t0 = start[2];
    r = start_of;
  }

  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127)) + warp * C::kRingBytes;
  const uint32_t ring_addr = smem_u32(ring);
  float* my_part = reinterpret_cast<float*>(ring);
  bool bad = false;          // a slot of this warp's rows lies outside the cache
  bool at_run_begin = true;

  while (left > 0) {
    if (!at_run_begin) {
      if (b >= p.ix.batch) break;
      r = cached_of(p.ix, b);
    }
    const int len = r.len, n_all = tiles_of(len);
    if (t0 >= n_all) {          // behind a pair's tiles, or a request without a token
      if (n_all > 0) left -= n_all + kStart - t0;
      t0 = 0;
      if (n_all == 0 || ++hk == p.hkv) {
        hk = 0;
        ++b;
      }
      at_run_begin = false;
      continue;
    }
    const int n = static_cast<int>(min(static_cast<int64_t>(n_all - t0), left));
    const int base0 = t0 * kTile + warp * kWarpTokens;   // first token of this warp's first tile
    const int* rtt = p.ix.req_to_token + static_cast<int64_t>(r.row) * p.ix.table_stride;
    const Elem* kbase = static_cast<const Elem*>(p.k_cache) + hk * p.kv_head_stride;
    const Elem* vbase = static_cast<const Elem*>(p.v_cache) + hk * p.kv_head_stride;
    float* scores = p.scores + (static_cast<int64_t>(b) * p.hkv + hk) * p.ix.table_cols * g;

    auto slot_of = [&](int t) -> int {             // slot of token (lane & 15) of this warp's tile t; -1: outside the cache
      const int tok = base0 + t * kTile + (lane & 15);
      return (t < n && tok < len) ? max(__ldcg(rtt + tok), -1) : kNoToken;
    };
    int ahead[C::kStages - 1];              // the slots of the first tiles, in one round trip
#pragma unroll
    for (int t = 0; t < C::kStages - 1; ++t) ahead[t] = slot_of(t);
    int slot_next = slot_of(C::kStages - 1);
    auto issue = [&](int t, int s) {
      if (t < n) {
        if (s < 0 || s >= p.num_slots) {
          bad = bad || s != kNoToken;
          s = -1;
        }
        const uint32_t dst = ring_addr + (t % C::kStages) * (2 * C::kTensorBytes);
        constexpr int kRowsPerPass = 32 / C::kChunks, kPasses = kWarpTokens / kRowsPerPass;
        const int ch = lane % C::kChunks, r0 = lane / C::kChunks;
        int rs[kPasses];          // slots first, then copies: a copy does not wait for its own
#pragma unroll
        for (int i = 0; i < kPasses; ++i) rs[i] = __shfl_sync(0xffffffffu, s, i * kRowsPerPass + r0);
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          const int64_t off = static_cast<int64_t>(max(rs[i], 0)) * p.kv_tok_stride + ch * (16 / C::kItem);
          const uint32_t to = dst + C::at(i * kRowsPerPass + r0, ch);
          cp16_l2(to, kbase + off, rs[i] >= 0);
          cp16_l2(to + C::kTensorBytes, vbase + off, rs[i] >= 0);
        }
      }
      cp_commit();
    };
    // the queries of the group as the column operand: head nt * 8 + lane / 4; of every 16 features 2 c, 2 c + 1 and those 8 on
    // (c = lane % 4), of 8-bit rows 4 c to 4 c + 3
    uint32_t qf[HD / 16][NT][2];
    float scale[NT][2];       // of the scores of heads nt * 8 + 2 c + i
    {
      const T* q = static_cast<const T*>(p.q) + b * p.q_stride + static_cast<int64_t>(hk) * g * HD;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = nt * 8 + (lane >> 2);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int f = kk * 16 + (FMT == kKvSame ? i * 8 + 2 * (lane & 3) : 4 * (lane & 3) + 2 * i);
            qf[kk][nt][i] = h < g ? __ldcg(reinterpret_cast<const uint32_t*>(q + h * HD + f)) : 0u;
          }
      }
    }
#pragma unroll
    for (int t = 0; t < C::kStages - 1; ++t) issue(t, ahead[t]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      scale[nt][0] = scale[nt][1] = p.scale_log2;
      if constexpr (!std::is_same<T, M>::value) {        // bf16 queries over 8-bit rows
        float top = 0.f;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 x = unpack_bf16x2(qf[kk][nt][i]);
            top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int raise = min(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), 126);      // by 2^raise; -114 where the largest is infinite
        const float by = __uint_as_float((raise + 127) << 23);
        if (top > 0.f)
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 x = unpack_bf16x2(qf[kk][nt][i]);
              const __half2 y = __floats2half2_rn(x.x * by, x.y * by);
              qf[kk][nt][i] = *reinterpret_cast<const uint32_t*>(&y);
            }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int of = __shfl_sync(0xffffffffu, top > 0.f ? raise : 0, (2 * (lane & 3) + i) * 4);
          scale[nt][i] *= __uint_as_float((127 - of) << 23);
        }
      }
    }
    float o[HD / 16][NT][4];
    float m[NT][2], l[NT][2], x[NT][2];     // maximum less kUp, sum of the rounded weights, sum of the weights
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = x[nt][0] = x[nt][1] = 0.f;
#pragma unroll
      for (int mt = 0; mt < HD / 16; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[mt][nt][i] = 0.f;
    }

    for (int t = 0; t < n; ++t) {
      cp_wait<C::kStages - 2>();
      __syncwarp();
      issue(t + C::kStages - 1, slot_next);      // into the stage of the tile before, which every lane has left
      slot_next = slot_of(t + C::kStages);
      const int base = base0 + t * kTile;
      if (base >= len) continue;
      const uint32_t sk = ring_addr + (t % C::kStages) * (2 * C::kTensorBytes);
      const uint32_t sv = sk + C::kTensorBytes;
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[nt][i] = 0.f;
      const int row = lane & 15;
      if constexpr (FMT == kKvSame) {
        float s2[4] = {0.f, 0.f, 0.f, 0.f};       // every other product, where the heads make only one chain of them
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          uint32_t a[4];
          ldsm4(a, sk + C::at(row, kk * 2 + (lane >> 4)));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816<M>(NT == 1 && (kk & 1) ? s2 : s[nt], a[0], a[1], a[2], a[3], qf[kk][nt][0], qf[kk][nt][1]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[0][i] += s2[i];
      } else {
#pragma unroll
        for (int k2 = 0; k2 < HD / 32; ++k2) {
          uint32_t a[4];
          ldsm4(a, sk + C::at(row, k2 * 2 + (lane >> 4)));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t a0 = widen<FMT>(a[2 * i]), a1 = widen<FMT>(a[2 * i + 1]), a2 = widen<FMT>(a[2 * i] >> 16), a3 = widen<FMT>(a[2 * i + 1] >> 16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816<M>(s[nt], a0, a1, a2, a3, qf[2 * k2 + i][nt][0], qf[2 * k2 + i][nt][1]);
          }
        }
      }
      const int tok = base + (lane >> 2);
      bool ok0 = tok < len, ok1 = tok + 8 < len;
      if (__any_sync(0xffffffffu, bad)) {       // rare: tokens whose slots lie outside the cache are not seen
        const int s0 = ok0 ? __ldcg(rtt + tok) : -1, s1 = ok1 ? __ldcg(rtt + tok + 8) : -1;
        ok0 = s0 >= 0 && s0 < p.num_slots;
        ok1 = s1 >= 0 && s1 < p.num_slots;
      }
      bool raise = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[nt][i] *= scale[nt][i & 1];
        if (p.cap_post > 0.f) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[nt][i] = p.cap_post * tanhf(s[nt][i] * p.cap_pre);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[nt][i] = ok0 ? s[nt][i] : -INFINITY;
          s[nt][i + 2] = ok1 ? s[nt][i + 2] : -INFINITY;
          const float top = fmaxf(s[nt][i], s[nt][i + 2]);
          raise = raise || top > m[nt][i] + (kRescaleThreshold + kUp);   // the first tile always raises
        }
        // the scores wait for the normaliser
        const int h = nt * 8 + 2 * (lane & 3);
        float* to = scores + static_cast<int64_t>(tok) * g + h;
        if ((g & 1) == 0) {
          if (h < g && tok < len) __stcg(reinterpret_cast<float2*>(to), make_float2(s[nt][0], s[nt][1]));
          if (h < g && tok + 8 < len) __stcg(reinterpret_cast<float2*>(to + 8 * g), make_float2(s[nt][2], s[nt][3]));
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (h + i < g && tok < len) __stcg(to + i, s[nt][i]);
            if (h + i < g && tok + 8 < len) __stcg(to + 8 * g + i, s[nt][i + 2]);
          }
        }
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = fmaxf(s[nt][i], s[nt][i + 2]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float now = fmaxf(m[nt][i], top - kUp);
            const float f = m[nt][i] == -INFINITY ? 0.f : fast_exp2(m[nt][i] - now);
            m[nt][i] = now;
            l[nt][i] *= f;
            x[nt][i] *= f;
#pragma unroll
            for (int mt = 0; mt < HD / 16; ++mt) {
              o[mt][nt][i] *= f;
              o[mt][nt][i + 2] *= f;
            }
          }
        }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float e0 = fast_exp2(s[nt][2 * i] - m0), e1 = fast_exp2(s[nt][2 * i + 1] - m1);
          uint32_t w;
          float2 back;            // the sum takes what the product takes: the rounded weights
          if constexpr (std::is_same<M, __half>::value) {
            const __half2 h = __floats2half2_rn(e0, e1);
            w = *reinterpret_cast<const uint32_t*>(&h);
            back = __half22float2(h);
          } else {
            w = pack_bf16x2(e0, e1);
            back = unpack_bf16x2(w);
          }
          l[nt][0] += back.x;
          l[nt][1] += back.y;
          x[nt][0] += e0;
          x[nt][1] += e1;
          pb[nt][i] = movmatrix(w);
        }
      }
      const int vrow = (lane & 7) + ((lane >> 4) << 3);
      if constexpr (FMT == kKvSame) {
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
          uint32_t a[4];
          ldsm4_t(a, sv + C::at(vrow, mt * 2 + ((lane >> 3) & 1)));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816<M>(o[mt][nt], a[0], a[1], a[2], a[3], pb[nt][0], pb[nt][1]);
        }
      } else {
#pragma unroll
        for (int m2 = 0; m2 < HD / 32; ++m2) {
          uint32_t a[4];          // tokens 0-7 and 8-15 of 16 features, then of the next 16
          ldsm4_t(a, sv + C::at((lane & 7) + (((lane >> 3) & 1) << 3), m2 * 2 + (lane >> 4)));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            // a register has features 2 u and 2 u + 1 of two tokens: first the one, then the other
            const uint32_t lo = __byte_perm(a[2 * i], 0, 0x3120), hi = __byte_perm(a[2 * i + 1], 0, 0x3120);
            const uint32_t a0 = widen<FMT>(lo), a1 = widen<FMT>(lo >> 16), a2 = widen<FMT>(hi), a3 = widen<FMT>(hi >> 16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816<M>(o[2 * m2 + i][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
          }
        }
      }
    }
    cp_wait<0>();
    __syncwarp();

    // ---- the warps' results meet in shared memory: this warp's goes where its ring was ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sum = l[nt][i], all = x[nt][i];
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) {
          sum += __shfl_xor_sync(0xffffffffu, sum, off);
          all += __shfl_xor_sync(0xffffffffu, all, off);
        }
        const int h = nt * 8 + 2 * (lane & 3) + i;
        if (lane < 4) {
          part_m[warp][h] = m[nt][i];
          part_l[warp][h] = sum;
          part_x[warp][h] = all;
        }
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
          const int f = mt * 16 + (FMT == kKvSame ? lane >> 2 : 2 * (lane >> 2));
          my_part[h * C::kOutStride + f] = o[mt][nt][i];
          my_part[h * C::kOutStride + f + (FMT == kKvSame ? 8 : 1)] = o[mt][nt][i + 2];
        }
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && n == n_all;
    const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + (at_run_begin ? 0 : 1)) * g;
    const float* parts = reinterpret_cast<const float*>(ring - warp * C::kRingBytes);
    // a sum of 0: no key to be seen.  A NaN or infinite score makes it NaN, and that the result
    for (int i = threadIdx.x; i < g * (HD / 4); i += kThreads) {
      const int h = i / (HD / 4), d = i % (HD / 4) * 4;
      float top = part_m[0][h];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, part_m[w][h]);
      float den = 0.f, all = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = part_m[w][h] == -INFINITY ? 0.f : exp2f(part_m[w][h] - top);
        const float4 v = *reinterpret_cast<const float4*>(parts + w * (C::kRingBytes / 4) + h * C::kOutStride + d);
        den += f * part_l[w][h];
        all += f * part_x[w][h];
        acc[0] += f * v.x;
        acc[1] += f * v.y;
        acc[2] += f * v.z;
        acc[3] += f * v.w;
      }
      if (whole) {
        const float sink = p.sink != nullptr && den != 0.f ? exp2f(p.sink[hk * g + h] * kLog2e - top) : 0.f;
        den += sink;
        all += sink;
        T* out = static_cast<T*>(p.out) + b * p.out_stride + static_cast<int64_t>(hk * g + h) * HD + d;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = from_f32<T>(den == 0.f ? 0.f : acc[e] / den);
        if (d == 0) p.whole_lse[(static_cast<int64_t>(b) * p.hkv + hk) * g + h] = all == 0.f ? -INFINITY : top + log2f(all);
      } else {
        *reinterpret_cast<float4*>(p.part_o + (part + h) * HD + d) =
            den == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(acc[0] / den, acc[1] / den, acc[2] / den, acc[3] / den);
        if (d == 0) p.part_lse[part + h] = den == 0.f ? make_float2(-INFINITY, -INFINITY) : make_float2(top + log2f(den), top + log2f(all));
      }
    }
    __syncthreads();
    left -= n;
    t0 += n;
    at_run_begin = false;
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0 && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
}

// The second kernel.  Its first CTAs join the partial results of pairs that lie in several CTAs, some query heads each:
// out = sum_c w_c O_c, w_c = 2^(lse_c - max) / sum.  The others take equal runs of the line of tiles and turn scores into weights.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) weights_join_kernel(const DecodeParams p) {
  __shared__ int warp_sums[kWarps];
  __shared__ int mine[2];       // units in front of the request, and its tiles
  __shared__ int start[3];
  __shared__ __align__(16) float weight[kThreads];
  pdl_launch_dependents();
  const int g = p.group, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, all_joins = p.joins * p.hkv * p.ix.batch;
  const bool joins = static_cast<int>(blockIdx.x) < all_joins;
  int first, last, total;
  int before = scan_units(p, warp_sums, first, last, total);       // the lengths were complete when the first kernel began
  const int64_t line = static_cast<int64_t>(total) * p.hkv;
  const int used = ctas_used(p.ctas, line);
  auto owner = [&](int64_t x) { return owner_of(line, x, used); };

  if (joins) {
    const int which = blockIdx.x / p.joins, b = which / p.hkv, hk = which - b * p.hkv;
    const int h0 = (blockIdx.x - which * p.joins) * p.join_heads, h1 = min(g, h0 + p.join_heads);
    if (b >= first && b < last) {
      for (int r = first; r < b; ++r) before += units_of(p, r);
      mine[0] = before;
      mine[1] = tiles_of(cached_of(p.ix, b).len);
    }
    __syncthreads();
    const int n = mine[1];
    const int64_t begin = static_cast<int64_t>(mine[0]) * p.hkv + static_cast<int64_t>(hk) * (n + kStart);
    const int c0 = n > 0 ? owner(begin) : 0, c1 = n > 0 ? owner(begin + n - 1) : 0;
    // the first of the pair's CTAs has it in its second slot where its run begins with another pair; the others in their first
    const int first_slot = c0 * 2 + (n > 0 && run_begin(line, c0, used) < begin ? 1 : 0);
    pdl_wait_loads();
    if (n > 0 && c0 == c1) return;         // one CTA had all of it and has written the output
    constexpr int kPer = (HD + kThreads - 1) / kThreads;
    for (int h = h0; h < h1; ++h) {
      const int head = hk * g + h;
      T* out = static_cast<T*>(p.out) + b * p.out_stride + static_cast<int64_t>(head) * HD;
      auto slot = [&](int c) { return static_cast<int64_t>(c == c0 ? first_slot : c * 2) * g + h; };
      if (n == 0) {
        for (int d = threadIdx.x; d < HD; d += kThreads) out[d] = from_f32<T>(0.f);
        continue;
      }
      const float sink = p.sink != nullptr ? __ldcg(p.sink + head) * kLog2e : -INFINITY;
      float top = -INFINITY;
      for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, __ldcg(p.part_lse + slot(c)).x);
      top = warp_max(top);
      top = fmaxf(top, sink);
      // no key seen: 0, beside a sink too; a part that is no number shows
      float den = sink > -INFINITY ? exp2f(sink - top) : 0.f, acc[kPer] = {};
      for (int at = c0; at <= c1; at += kThreads) {
        const int m = min(kThreads, c1 + 1 - at);
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < m) {
          const float lse = __ldcg(p.part_lse + slot(at + threadIdx.x)).x;
          weight[threadIdx.x] = lse == -INFINITY ? 0.f : exp2f(lse - top);
        }
        __syncthreads();
#pragma unroll 8
        for (int i = 0; i < m; ++i) {
          const float w = weight[i];
          den += w;
#pragma unroll
          for (int k = 0; k < kPer; ++k) {
            const int d = threadIdx.x + k * kThreads;
            if (d < HD) acc[k] += w * __ldcg(p.part_o + slot(at + i) * HD + d);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int d = threadIdx.x + k * kThreads;
        if (d < HD) out[d] = from_f32<T>(den == 0.f ? 0.f : acc[k] / den);
      }
    }
    return;
  }

  // ---- weights ----
  const int c = blockIdx.x - all_joins;
  const int shared = static_cast<int>(min(static_cast<int64_t>(p.weight_ctas), max(line, static_cast<int64_t>(1))));
  if (c >= shared) return;
  const int64_t run0 = run_begin(line, c, shared);
  int64_t left = run_begin(line, c + 1, shared) - run0;
  if (left <= 0) return;
  {
    int64_t at = static_cast<int64_t>(before) * p.hkv;
    for (int i = first; i < last; ++i) {
      const int n = units_of(p, i);
      if (run0 >= at && run0 < at + static_cast<int64_t>(n) * p.hkv) {
        const int in = static_cast<int>(run0 - at), h = in / n;
        start[0] = i;
        start[1] = h;
        start[2] = in - h * n;
      }
      at += static_cast<int64_t>(n) * p.hkv;
    }
  }
  __syncthreads();
  int b = start[0], hk = start[1], t0 = start[2];
  int64_t pair0 = run0 - t0;         // where the pair begins on the line
  bool waited = false;
  while (left > 0 && b < p.ix.batch) {
    const Cached r = cached_of(p.ix, b);
    const int n_all = tiles_of(r.len), n = static_cast<int>(min(static_cast<int64_t>(max(n_all - t0, 0)), left));
    if (n > 0) {
      const int c0 = owner(pair0), c1 = owner(pair0 + n_all - 1);
      const int first_slot = c0 * 2 + (run_begin(line, c0, used) < pair0 ? 1 : 0);
      const int64_t pair = static_cast<int64_t>(b) * p.hkv + hk;
      const float* scores = p.scores + pair * p.ix.table_cols * g;
      float* sums = p.sums.data + r.row * p.sums.row_stride + hk * p.sums.head_stride;
      const int begin = t0 * kTile, end = min(r.len, (t0 + n) * kTile);
      // the sums so far are nothing that the first kernel writes
      float old[kSums];
#pragma unroll
      for (int k = 0; k < kSums; ++k) {
        const int tok = begin + k * kThreads + static_cast<int>(threadIdx.x);
        old[k] = tok < end && tok < r.len - 1 && p.decay != 0.f ? p.decay * __ldcg(sums + tok) : 0.f;
      }
      if (!waited) pdl_wait_loads();
      waited = true;
      __syncthreads();
      for (int h = warp; h < g; h += kWarps) {         // the heads' normalisers
        float lse;
        if (c0 == c1) {
          lse = __ldcg(p.whole_lse + pair * g + h);
        } else {
          auto part = [&](int i) { return __ldcg(p.part_lse + static_cast<int64_t>(i == c0 ? first_slot : i * 2) * g + h).y; };
          const float sink = p.sink != nullptr ? __ldcg(p.sink + hk * g + h) * kLog2e : -INFINITY;
          float top = -INFINITY, all = 0.f;
          for (int i = c0 + lane; i <= c1; i += 32) {
            const float v = part(i), most = fmaxf(top, v);
            if (most > -INFINITY) {
              all = (top == -INFINITY ? all : all * exp2f(top - most)) + (v == -INFINITY ? 0.f : exp2f(v - most));
              top = most;
            } else {
              all += v == v ? 0.f : v;
            }
          }
          const float most = warp_max(top);
          const bool none = most == -INFINITY;
          const float over = fmaxf(most, sink);
          all = warp_sum(top == -INFINITY ? all : all * exp2f(top - over));
          lse = none && all == 0.f ? -INFINITY : over + log2f(all + (p.sink != nullptr ? exp2f(sink - over) : 0.f));
        }
        if (lane == 0) weight[h] = lse;
      }
      __syncthreads();
      // scores of a token and its heads lie side by side
      auto add_up = [&](int tok) {
        const float* s = scores + static_cast<int64_t>(tok) * g;
        float add = 0.f;
        if ((g & 3) == 0) {
          for (int h = 0; h < g; h += 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(s + h)), l = *reinterpret_cast<const float4*>(&weight[h]);
            add += (l.x == -INFINITY ? 0.f : fast_exp2(v.x - l.x)) + (l.y == -INFINITY ? 0.f : fast_exp2(v.y - l.y)) +
                   (l.z == -INFINITY ? 0.f : fast_exp2(v.z - l.z)) + (l.w == -INFINITY ? 0.f : fast_exp2(v.w - l.w));
          }
        } else {
          for (int h = 0; h < g; ++h) {
            const float l = weight[h];
            add += l == -INFINITY ? 0.f : fast_exp2(__ldcg(s + h) - l);
          }
        }
        return add;
      };
#pragma unroll
      for (int k = 0; k < kSums; ++k) {
        const int tok = begin + k * kThreads + static_cast<int>(threadIdx.x);
        if (tok < end) sums[tok] = old[k] + add_up(tok);
      }
      for (int tok = begin + kSums * kThreads + static_cast<int>(threadIdx.x); tok < end; tok += kThreads)
        sums[tok] = (tok < r.len - 1 && p.decay != 0.f ? p.decay * __ldcg(sums + tok) : 0.f) + add_up(tok);
    }
    left -= n;
    t0 += n;
    if (left <= 0) break;
    if (n_all > 0) {
      left -= n_all + kStart - t0;
      pair0 += n_all + kStart;
    }
    t0 = 0;
    if (n_all == 0 || ++hk == p.hkv) {
      hk = 0;
      ++b;
    }
  }
}

template <typename T, int HD, int NT, int FMT>
int launch_one(const DecodeParams& p, cudaStream_t s) {
  auto kern = weights_decode_kernel<T, HD, NT, FMT>;
  using C = Cfg<HD, NT, FMT>;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kern), C::kSmem) != cudaSuccess) return -3;
  cudaError_t err = launch_pdl(kern, dim3(p.ctas), dim3(kThreads), C::kSmem, s, p);
  note_launch();
  if (err != cudaSuccess) return -4;
  err = launch_pdl(weights_join_kernel<T, HD>, dim3(p.joins * p.hkv * p.ix.batch + p.weight_ctas), dim3(kThreads), 0, s, p);
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}
template <typename T, int HD, int FMT>
int launch_size(const DecodeParams& p, cudaStream_t s) {
  if (p.group <= 8) return launch_one<T, HD, 1, FMT>(p, s);
  if (p.group <= 16) return launch_one<T, HD, 2, FMT>(p, s);
  if constexpr (HD <= 128) return launch_one<T, HD, 4, FMT>(p, s);
  return -1;
}
template <typename T, int HD>
int launch_format(const DecodeParams& p, int fmt, cudaStream_t s) {
  switch (fmt) {
    case kKvSame: return launch_size<T, HD, kKvSame>(p, s);
    case kKvE4M3: return launch_size<T, HD, kKvE4M3>(p, s);
    default: return launch_size<T, HD, kKvE5M2>(p, s);
  }
}

// as many as run at once (Cfg's kPerSm)
int stream_ctas(const WeightsDecodeArgs& a) {
  const int row = a.head_dim * (a.kv_fmt == kKvSame ? 2 : 1);
  return (a.head_dim == 256 ? 1 : row <= 128 && a.hq / a.hkv <= 8 ? 3 : 2) * a.num_sms;
}

}  // namespace

// groups whose heads' accumulators fit the registers
bool weights_decode_covers(int head_dim, int group) {
  return (head_dim == 64 || head_dim == 128 || head_dim == 256) && group >= 1 && group <= (head_dim == 256 ? 16 : 32);
}

int64_t weights_decode_floats(const WeightsDecodeArgs& a) {
  const int64_t group = a.hq / a.hkv, parts = static_cast<int64_t>(stream_ctas(a)) * 2 * group;
  return parts * (a.head_dim + 2) + 4 + static_cast<int64_t>(a.index.batch) * a.hq * (1 + static_cast<int64_t>(a.index.table_cols));
}

int launch_weights_decode(const WeightsDecodeArgs& a, cudaStream_t s) {
  if (a.hkv <= 0 || a.hq % a.hkv != 0 || !weights_decode_covers(a.head_dim, a.hq / a.hkv)) return -1;
  if (a.index.batch <= 0) return 0;
  DecodeParams p{};
  p.ix = a.index;
  p.sums = a.sums;
  p.q = a.q;
  p.k_cache = a.k_cache;
  p.v_cache = a.v_cache;
  p.out = a.out;
  p.group = a.hq / a.hkv;
  p.hkv = a.hkv;
  p.ctas = stream_ctas(a);
  // a CTA joins several heads where there are more heads than two per SM
  const int64_t heads = static_cast<int64_t>(a.index.batch) * a.hq;
  p.join_heads = static_cast<int>(std::min<int64_t>(p.group, std::max<int64_t>(1, heads / (2 * a.num_sms))));
  p.joins = (p.group + p.join_heads - 1) / p.join_heads;
  // No more CTAs than run at once, 9 on an SM, as long as that leaves a few for the weights (29 x 1900, 32 / 8 heads: 8 an SM for the weights
  // 58.4 us, 6 and 4 56.6; 32 x 4096, 32 / 4 heads, e4m3: 8, 6, 4 an SM 57.4, 53.4, 55.2)
  const int64_t joining = static_cast<int64_t>(p.joins) * p.hkv * a.index.batch;
  p.weight_ctas = static_cast<int>(std::min<int64_t>(6 * a.num_sms, std::max<int64_t>(4 * a.num_sms, 9 * a.num_sms - joining)));
  const int64_t parts = static_cast<int64_t>(p.ctas) * 2 * p.group;
  p.part_o = a.workspace;
  p.part_lse = reinterpret_cast<float2*>(a.workspace + parts * a.head_dim);
  p.scores = a.workspace + (parts * (a.head_dim + 2) + 3) / 4 * 4;      // on a 16-byte boundary
  p.whole_lse = p.scores + static_cast<int64_t>(a.index.batch) * a.hq * a.index.table_cols;
  p.sink = a.sink;
  p.q_stride = a.q_stride;
  p.out_stride = a.out_stride;
  p.num_slots = a.num_slots;
  p.kv_tok_stride = a.kv_tok_stride;
  p.kv_head_stride = a.kv_head_stride;
  p.scale_log2 = a.scale * kLog2e;
  p.decay = a.decay;
  if (a.logit_cap > 0.f) {      // the scores are scaled before the cap
    p.scale_log2 = a.scale;
    p.cap_pre = 1.f / a.logit_cap;
    p.cap_post = a.logit_cap * kLog2e;
  }
  int rc = -1;
  MB200_DISPATCH_HALF(a.dt, rc = a.head_dim == 64 ? launch_format<T, 64>(p, a.kv_fmt, s) : a.head_dim == 128 ? launch_format<T, 128>(p, a.kv_fmt, s)
                                                                                                             : launch_format<T, 256>(p, a.kv_fmt, s));
  return rc;
}

}  // namespace mb200
