// The attention weights of prompts that are short for certain (see weights_prompt.cuh for what is computed): one kernel, a CTA per request and
// kv head, everything between the rows of the cache and the sums in shared memory.
//
// Up to 256 tokens' keys stay in shared memory; the observed rows (query, head of the group) come 32 at a time.  S = Q K^T by warp-level
// products, 32 tokens a warp; a warp takes four rows of S, masks them, and makes weights of them; then a thread per token adds up its column.
// What bounds it is latency, one after the other: lengths, slots, rows, products, weights (160 tokens behind 16 queries, 8 kv heads: 8.5 us,
// where the two kernels for prompts of any length take 21: each of them finds its place, fills its stages and empties them).
#include <algorithm>

#include "common.cuh"
#include "evict.cuh"
#include "mma.cuh"

namespace mb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeys = kShortPromptTokens, kThreads = 256, kWarps = kThreads / 32;
constexpr int kRows = 32;                      // of S
constexpr int kStride = kKeys + 4;             // floats of a row of S
static_assert(kKeys == 32 * kWarps && kKeys == kThreads, "32 tokens a warp, one a thread");

struct ShortParams {
  WeightsPromptArgs a;
  int group;
  float scale_log2, cap_pre, cap_post;
};

template <int HD>
struct Cfg {
  static constexpr int kRow = HD * 2 + 16;     // bytes of a row of Q or K in shared memory: eight rows lie in eight different bank groups
  static constexpr int kSmem = (kKeys + kRows) * kRow + kRows * kStride * 4;
};

template <typename T, int HD, int FMT>
__global__ void __launch_bounds__(kThreads) weights_short_kernel(const ShortParams p) {
  using C = Cfg<HD>;
  using M = typename std::conditional<FMT == kKvSame, T, __half>::type;        // type of the products
  constexpr bool kScaled = !std::is_same<T, M>::value;      // bf16 queries over 8-bit rows become fp16, scaled by a power of two per row
  extern __shared__ __align__(16) uint8_t short_smem[];
  __shared__ float row_mul[kRows];
  __shared__ uint32_t seen[kWarps];        // tokens that have a slot
  uint8_t* sk = short_smem;
  uint8_t* sq = sk + kKeys * C::kRow;
  float* S = reinterpret_cast<float*>(sq + kRows * C::kRow);
  const WeightsPromptArgs& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = p.group;
  const int hk = static_cast<int>(blockIdx.x % p.a.hkv), b = static_cast<int>(blockIdx.x / p.a.hkv);
  pdl_wait();
  pdl_launch_dependents();
  const Cached c = cached_of(a.index, b);
  const int prefix = __ldcg(a.prefix_lens + b), start = __ldcg(a.q_start + b), fresh = prefix >= 0 ? c.len - prefix : 0;
  const bool any = c.len > 0 && prefix < c.len;       // new rows, and whether they are there
  const bool bad = c.bad || (any && (prefix < 0 || start < 0 || fresh > a.rows - start));
  if (bad && tid == 0 && hk == 0 && a.index.status != nullptr) atomicExch(a.index.status, kStatusBadIndex);
  if (bad || !any) return;
  const int look = a.last > 0 ? min(a.last, fresh) : fresh;
  const int len = c.len, rows = look * g, first = start + fresh - look;

  // ---- keys: a thread looks up a token's slot, a warp copies its 32 rows ----
  int slot = tid < len ? __ldcg(a.index.req_to_token + static_cast<int64_t>(c.row) * a.index.table_stride + tid) : -1;
  const bool there = slot >= 0 && slot < a.num_slots;
  if (tid < len && !there && a.index.status != nullptr) atomicExch(a.index.status, kStatusBadIndex);
  if (!there) slot = -1;
  {
    const uint32_t bits = __ballot_sync(0xffffffffu, there);
    if (lane == 0) seen[warp] = bits;
  }
  {
    constexpr int kItem = FMT == kKvSame ? 2 : 1, kPieces = HD * kItem / 16, kPer = 32 / kPieces;       // 16-byte pieces of a cached row
    const int ch = lane % kPieces, r0 = lane / kPieces;
    const uint8_t* from = static_cast<const uint8_t*>(a.k_cache) + hk * a.kv_head_stride * kItem + ch * 16;
#pragma unroll 8
    for (int k = 0; k < kPieces; ++k) {
      const int row = k * kPer + r0, rs = __shfl_sync(0xffffffffu, slot, row);
      uint8_t* to = sk + (warp * 32 + row) * C::kRow;
      const uint8_t* at = from + static_cast<int64_t>(max(rs, 0)) * a.kv_tok_stride * kItem;
      if constexpr (FMT == kKvSame) {
        cp16_zfill(smem_u32(to + ch * 16), at, rs >= 0);
      } else {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (rs >= 0) x = __ldcg(reinterpret_cast<const uint4*>(at));
        const uint32_t v[4] = {x.x, x.y, x.z, x.w};
        uint32_t y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {         // two 8-bit values -> two fp16, exactly
          const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v[i / 2] >> (16 * (i & 1)) & 0xffffu),
                                                           FMT == kKvE5M2 ? __NV_E5M2 : __NV_E4M3);
          y[i] = static_cast<uint32_t>(h.x) | static_cast<uint32_t>(h.y) << 16;
        }
        *reinterpret_cast<uint4*>(to + ch * 32) = make_uint4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<uint4*>(to + ch * 32 + 16) = make_uint4(y[4], y[5], y[6], y[7]);
      }
    }
  }
  cp_commit();
  float sum = 0.f;
  for (int row0 = 0; row0 < rows; row0 += kRows) {
    // ---- 32 rows of queries ----
    constexpr int kPieces = HD / 8;
    for (int i = tid; i < kRows * kPieces; i += kThreads) {
      const int row = i / kPieces, ch = i % kPieces, r = row0 + row;
      const uint16_t* from = static_cast<const uint16_t*>(a.q);
      if (r < rows) from += (first + r / g) * a.q_stride + static_cast<int64_t>(hk * g + r % g) * HD + ch * 8;
      uint8_t* to = sq + row * C::kRow + ch * 16;
      if constexpr (!kScaled) {
        cp16_zfill(smem_u32(to), from, r < rows);
      } else {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < rows) x = __ldcg(reinterpret_cast<const uint4*>(from));
        uint32_t v[4] = {x.x, x.y, x.z, x.w};
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = unpack_bf16x2(v[k]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
#pragma unroll
        for (int o = 1; o < kPieces; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // the largest of a row gets an exponent of 14: what is 2^-25 times smaller than that goes below fp16's last place
        const int raise = top > 0.f ? min(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), 126) : 0;
        const float by = __uint_as_float((raise + 127) << 23);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = unpack_bf16x2(v[k]);
          const __half2 h = __floats2half2_rn(f.x * by, f.y * by);
          v[k] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
        if (ch == 0) row_mul[row] = __uint_as_float((127 - raise) << 23);
      }
    }
    cp_commit();
    cp_wait<0>();
    __syncthreads();
    // ---- scores of this warp's 32 tokens ----
    if (warp * 32 < len) {
      float d[2][4][4] = {};
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        uint32_t q[2][4], k[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          ldsm4(q[i], smem_u32(sq + (i * 16 + (lane & 15)) * C::kRow + kk * 32 + (lane >> 4) * 16));
          ldsm4(k[i], smem_u32(sk + (warp * 32 + i * 16 + (lane & 7) + ((lane >> 4) << 3)) * C::kRow + kk * 32 + ((lane >> 3) & 1) * 16));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int n = 0; n < 4; ++n) mma_16816<M>(d[i][n], q[i][0], q[i][1], q[i][2], q[i][3], k[n >> 1][2 * (n & 1)], k[n >> 1][2 * (n & 1) + 1]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float2*>(S + (i * 16 + h * 8 + (lane >> 2)) * kStride + warp * 32 + n * 8 + 2 * (lane & 3)) =
                make_float2(d[i][n][2 * h], d[i][n][2 * h + 1]);
    }
    __syncthreads();
    // ---- four rows a warp: weights in the place of scores ----
#pragma unroll 1
    for (int i = 0; i < kRows / kWarps; ++i) {
      const int row = warp * (kRows / kWarps) + i, r = row0 + row;
      if (r >= rows) break;
      const int head = hk * g + r % g, place = len - look + r / g;
      const float mul = (kScaled ? row_mul[row] : 1.f) * p.scale_log2;
      float x[kKeys / 32], top = -INFINITY;
#pragma unroll
      for (int k = 0; k < kKeys / 32; ++k) {
        const int key = k * 32 + lane;
        const bool visible = key <= place && (seen[k] >> lane & 1);
        x[k] = visible ? S[row * kStride + key] * mul : -INFINITY;
        if (p.cap_post > 0.f && visible) x[k] = p.cap_post * tanhf(x[k] * p.cap_pre);
        top = fmaxf(top, x[k]);
      }
      top = warp_max(top);
      const float sink = a.sink != nullptr ? __ldcg(a.sink + head) * kLog2e : -INFINITY, at = fmaxf(top, sink);
      float all = 0.f;
#pragma unroll
      for (int k = 0; k < kKeys / 32; ++k) {
        x[k] = x[k] == -INFINITY ? 0.f : fast_exp2(x[k] - (at == -INFINITY ? 0.f : at));
        all += x[k];
      }
      all = warp_sum(all);
      if (sink > -INFINITY) all += fast_exp2(sink - at);
      const float inv = all == 0.f ? 0.f : 1.f / all;         // nothing seen: no weights
#pragma unroll
      for (int k = 0; k < kKeys / 32; ++k) S[row * kStride + k * 32 + lane] = x[k] == 0.f ? 0.f * inv : x[k] * inv;
    }
    __syncthreads();
    // ---- a thread's token ----
    const int some = min(kRows, rows - row0);
    float now = 0.f;
    // rows in front of the token's own have no weight for it, whatever they hold
    const int low = tid > len - look ? min(max((tid - (len - look)) * g - row0, 0), some) : 0;
    for (int row = low; row < some; ++row) now += S[row * kStride + tid];
    sum += now;
    __syncthreads();
  }
  if (tid < len) {
    float* to = a.sums.data + c.row * a.sums.row_stride + hk * a.sums.head_stride + tid;
    if (!there) sum = 0.f;
    *to = a.add && tid < prefix ? __ldcg(to) + sum : sum;
  }
}

template <typename T, int HD, int FMT>
int launch_one(const ShortParams& p, cudaStream_t s) {
  auto kern = weights_short_kernel<T, HD, FMT>;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kern), Cfg<HD>::kSmem) != cudaSuccess) return -3;
  const cudaError_t err = launch_pdl(kern, dim3(static_cast<unsigned>(p.a.hkv) * p.a.index.batch), dim3(kThreads), Cfg<HD>::kSmem, s, p);
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}
template <typename T, int HD>
int launch_format(const ShortParams& p, cudaStream_t s) {
  switch (p.a.kv_fmt) {
    case kKvSame: return launch_one<T, HD, kKvSame>(p, s);
    case kKvE4M3: return launch_one<T, HD, kKvE4M3>(p, s);
    default: return launch_one<T, HD, kKvE5M2>(p, s);
  }
}

}  // namespace

int launch_weights_prompt_short(const WeightsPromptArgs& a, cudaStream_t s) {
  ShortParams p{};
  p.a = a;
  p.group = a.hq / a.hkv;
  p.scale_log2 = a.scale * kLog2e;
  if (a.logit_cap > 0.f) {      // the scores are scaled before the cap
    p.scale_log2 = a.scale;
    p.cap_pre = 1.f / a.logit_cap;
    p.cap_post = a.logit_cap * kLog2e;
  }
  int rc = -1;
  MB200_DISPATCH_HALF(a.dt, rc = a.head_dim == 64 ? launch_format<T, 64>(p, s) : a.head_dim == 128 ? launch_format<T, 128>(p, s) : launch_format<T, 256>(p, s));
  return rc;
}

}  // namespace mb200
