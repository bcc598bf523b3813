// The attention weights that the last queries of prompts give to the cached tokens, added up per token and kv head: head sizes 64, 128 and
// 256, caches of the activation type or 8-bit floats.
//
// Request b has seq_lens[b] tokens in the cache, the last n = seq - prefix of them new, with queries in rows q_start[b] + j of q.  The last
// `last` of them (all, where it is 0 or more than n) are observed: query j sees the tokens i <= place_j = prefix + j, and
//   sums_i <- (add and i < prefix: sums_i +) sum_{observed j, place_j >= i} sum_h 2^(s_hji log2 e - lse_hj)   over the heads h of the group,
// s = scale q . k (soft cap: c tanh(s / c)).  A sink is one more term of a row's normaliser lse_hj, without a value.
//
// A row's normaliser needs all of its scores, a token's sum needs all normalisers: two passes over the keys, each a product and one
// exponential per (row, token).  Keeping the exponentials would take more memory traffic (4 bytes each, twice) than making them again.
//   * Rows are (query, head of the group) pairs; RT tiles of 128 make a block.  Both passes hold a block in shared memory and let copying
//     warps bring keys by slot into a ring of 128-token stages in the operand layout.  A step is KT stages: RT * KT = 2, 256 score columns in
//     tensor memory, two buffers (heads of 256: one stage, 128 columns).
//   * First pass: S = Q K^T, a row per lane.  16 warps, four to every 32 lanes of tensor memory, take a quarter of the columns each, with a
//     maximum and sum of their own; they join at the block's end.  Units (request, kv head, block) times steps form one line, dealt evenly to the
//     CTAs; a block's normaliser is written out, or a partial one per CTA.
//   * Second pass: S^T = K Q^T, a token per lane: its sum over the rows is a sum in a thread, and no two CTAs have the same token, so nothing
//     depends on their order.  Tokens are dealt by what they cost: the blocks that see them.
// What bounds it is the exponentials, 16 per cycle and SM; products take half their time.
#include <algorithm>

#include "common.cuh"
#include "evict.cuh"

namespace mb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleThreshold = 8.0f;  // the running maximum is raised when a score passes it by 2^8
constexpr int kTileRows = 128;             // MMA M
constexpr int kStart = 2;                  // steps' time that every unit of the first pass costs beside its steps
constexpr int kChunk = 8;                  // steps whose sums wait in shared memory
constexpr int kNoToken = -0x7fffffff;
constexpr int kCompute = 16;               // warps
constexpr int kThreads = 32 * (kCompute + 8), kIssueWarp = kCompute + 7;

struct PromptParams {
  CacheIndex ix;
  WeightSums sums;
  const int* prefix_lens;
  const int* q_start;
  const void* q;
  const void* k_cache;
  float* lse;        // [rows of q][hq]: normalisers of blocks that lie in one CTA
  float* part;       // [CTAs][2][block rows]
  const float* sink;
  int64_t q_stride, num_slots, kv_tok_stride, kv_head_stride;
  int rows, hkv, group, last, ctas;
  bool add;
  float scale_log2, cap_in, cap_out;     // a scaled score x becomes cap_out tanh(x cap_in ln 2 / 2); cap_out 0: no soft cap
};

struct Observed {
  int len, row, prefix, first, look;      // tokens; row of the table; cached before; row of q of the first observed query; observed ones
  bool bad;
};
__device__ __forceinline__ Observed observed_of(const PromptParams& p, int b) {
  const Cached c = cached_of(p.ix, b);
  Observed o;
  o.len = c.len;
  o.row = c.row;
  o.bad = c.bad;
  o.prefix = __ldcg(p.prefix_lens + b);
  const int start = __ldcg(p.q_start + b), n = c.len - o.prefix;
  o.look = c.len > 0 && o.prefix < c.len ? (p.last > 0 ? min(p.last, n) : n) : 0;
  if (o.look > 0 && (o.prefix < 0 || start < 0 || n > p.rows - start)) {
    o.bad = true;
    o.look = 0;
  }
  o.first = start + n - o.look;
  return o;
}

template <int NH, bool KV8, int R>
struct Cfg {
  static constexpr int RT = R, KT = NH == 4 ? 1 : 2 / R;
  static constexpr int kD = 64 * NH;
  static constexpr int kRows = RT * kTileRows;               // of a block
  static constexpr int kStepKeys = KT * 128;
  static constexpr int kCols = RT * KT * 128, kWarpCols = kCols / 4;
  static constexpr int kQBlock = kRows * 128, kQBytes = NH * kQBlock;      // 64 features of a block's rows
  static constexpr int kKBlock = 128 * 128, kStage = NH * kKBlock;
  static constexpr int kStages = NH == 4 ? 2 : NH == 2 ? (R == 2 ? 4 : 5) : 6;
  static constexpr int kTeam = KV8 || NH == 4 ? 2 : 1, kTeams = kTeam == 2 ? 2 : 4;     // warps that copy a stage; every kTeams-th each
  static constexpr int kQWarps = 7 - kTeam * kTeams;
  static constexpr int kSmem = kQBytes + kStages * kStage;
  static constexpr int kGroups = 4 / KT;                     // parts of a token's sum
  static_assert(kTeams <= kStages && kQWarps > 0 && 2 * kCols <= 512, "teams, tensor memory");
};

// What both passes do with a batch, from its numbers on.  Blocks of a request: rows r = j * group + h.
template <typename C>
struct Work {
  Observed o;
  int rows, blocks, steps;       // steps: of the second pass
  __device__ __forceinline__ void set(const PromptParams& p, int b) {
    o = observed_of(p, b);
    rows = o.look * p.group;
    blocks = (rows + C::kRows - 1) / C::kRows;
    steps = o.look > 0 ? (o.len + C::kStepKeys - 1) / C::kStepKeys : 0;
  }
  __device__ __forceinline__ int rows_of(int block) const { return min(C::kRows, rows - block * C::kRows); }
  // largest place of a block's rows
  __device__ __forceinline__ int top_of(const PromptParams& p, int block) const {
    return o.len - o.look + (min(rows, (block + 1) * C::kRows) - 1) / p.group;
  }
  __device__ __forceinline__ int steps_of(const PromptParams& p, int block) const { return top_of(p, block) / C::kStepKeys + 1; }
  // first block that sees a step of the second pass
  __device__ __forceinline__ int first_block(const PromptParams& p, int step) const {
    const int j = step * C::kStepKeys - (o.len - o.look);
    return j > 0 ? j * p.group / C::kRows : 0;
  }
  // steps, from the first one on, that all blocks see
  __device__ __forceinline__ int common(const PromptParams& p) const {
    return min(steps, (o.len - o.look + (C::kRows - 1) / p.group) / C::kStepKeys + 1);
  }
  __device__ __forceinline__ int64_t cost1(const PromptParams& p) const {      // of one kv head
    int64_t n = 0;
    for (int i = 0; i < blocks; ++i) n += steps_of(p, i) + kStart;
    return n;
  }
  __device__ __forceinline__ int64_t cost2(const PromptParams& p) const {
    if (blocks == 0) return 0;
    const int all = common(p);
    int64_t n = static_cast<int64_t>(all) * blocks;
    for (int t = all; t < steps; ++t) n += blocks - first_block(p, t);
    return n;
  }
};

// Steps t0 .. t0 + n - 1 of a block
struct Item {
  int b, hk, block, t0, n;
  bool load, release;    // the block's queries are not in shared memory yet; the next item, if any, loads others
  bool first;            // the item begins the CTA's run (first pass)
  bool flush;            // last block over these steps (second pass)
  int chunk;             // steps whose sums wait (second pass)
  int64_t at;            // where the unit begins on the first pass's line
};

__device__ __forceinline__ int used_ctas(const PromptParams& p, int64_t line) {
  return static_cast<int>(min(static_cast<int64_t>(p.ctas), max(line / 2, static_cast<int64_t>(1))));
}
__device__ __forceinline__ int64_t run_begin(int64_t line, int c, int ctas) { return line * c / ctas; }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  const int sz = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(sz) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two 32-bit operations an instruction
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves_of(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// offset of 16-byte piece `ch` of row `row` in a tile of 64-feature blocks of `block` bytes, rows of 128 bytes, 128-byte swizzle
__device__ __forceinline__ uint32_t swz(int row, int ch, int block) {
  return (ch >> 3) * block + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
}

// PASS 1: normalisers; 2: sums.  FMT: what the cache holds (kKvSame, kKvE4M3, kKvE5M2)
template <typename T, int NH, int FMT, int R, int PASS>
__global__ void __launch_bounds__(kThreads, 1) weights_prompt_kernel(const PromptParams p) {
  constexpr bool KV8 = FMT != kKvSame;
  constexpr bool kScaled = KV8 && !std::is_same<T, __half>::value;      // bf16 queries become fp16, scaled by a power of two per row
  using C = Cfg<NH, KV8, R>;
  constexpr int kD = C::kD, kStages = C::kStages, KT = C::KT;
  extern __shared__ __align__(1024) uint8_t prompt_smem[];
  __shared__ uint64_t bars[2 * kStages + 10];
  __shared__ uint32_t tmem_holder;
  __shared__ int fail_flag, holes;
  __shared__ int begin_b;
  __shared__ int64_t begin_at, begin_at1, line_of[3];       // places of the first request's first unit; run, length of the run, line of the first pass
  __shared__ int used_of;                                   // CTAs of the first pass
  __shared__ __align__(16) float neg_lse[3][C::kRows];      // -normaliser of the rows (second pass)
  __shared__ __align__(16) float row_mul[3][kScaled ? C::kRows : 4];
  __shared__ __align__(16) float cells[kChunk * 512];       // first pass: 2 x [4][128] maxima and sums; second: [parts][tokens]
  uint8_t* sQ = prompt_smem;
  uint8_t* ring = sQ + C::kQBytes;
  uint64_t* full = bars;                 // [stage] the warps of a team
  uint64_t* empty = full + kStages;      // [stage] tcgen05.commit
  uint64_t* s_full = empty + kStages;    // [buffer] tcgen05.commit
  uint64_t* s_free = s_full + 2;         // [buffer] the computing warps have read the scores
  uint64_t* q_full = s_free + 2;         // the warps that copy queries
  uint64_t* q_free = q_full + 1;         // tcgen05.commit: the last scores of a block
  uint64_t* l_full = q_free + 1;         // [3] the same warps, for the computing ones
  uint64_t* met_bar = l_full + 3;        // the computing warps among themselves

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = p.group;
  pdl_wait_loads();

  // ---- where this CTA's run begins ----
  if (warp == 0) {
    const int per = (p.ix.batch + 31) / 32;
    const int first = min(p.ix.batch, lane * per), last = min(p.ix.batch, first + per);
    int64_t mine1 = 0, mine2 = 0;
    bool bad = false;
    Work<C> w;
    for (int b = first; b < last; ++b) {
      w.set(p, b);
      bad = bad || w.o.bad;
      mine1 += w.cost1(p) * p.hkv;
      if (PASS == 2) mine2 += w.cost2(p) * p.hkv;
    }
    if (PASS == 1 && bad && blockIdx.x == 0 && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
    int64_t incl1 = mine1, incl2 = mine2;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v1 = __shfl_up_sync(0xffffffffu, incl1, o), v2 = __shfl_up_sync(0xffffffffu, incl2, o);
      if (lane >= o) {
        incl1 += v1;
        incl2 += v2;
      }
    }
    const int64_t line1 = __shfl_sync(0xffffffffu, incl1, 31), line = PASS == 1 ? line1 : __shfl_sync(0xffffffffu, incl2, 31);
    const int used1 = used_ctas(p, line1), used = PASS == 1 ? used1 : static_cast<int>(min(static_cast<int64_t>(p.ctas), max(line, static_cast<int64_t>(1))));
    const int c = blockIdx.x;
    const int64_t begin = c < used ? run_begin(line, c, used) : line, end = c < used ? run_begin(line, c + 1, used) : line;
    if (lane == 0) {
      line_of[0] = begin;
      line_of[1] = end;
      line_of[2] = line1;
      used_of = used1;
      fail_flag = 0;
      holes = 0;
    }
    int64_t at = PASS == 1 ? incl1 - mine1 : incl2 - mine2, at1 = incl1 - mine1;
    if (begin < end && begin >= at && begin < (PASS == 1 ? incl1 : incl2)) {
      for (int b = first; b < last; ++b) {
        w.set(p, b);
        const int64_t n1 = w.cost1(p) * p.hkv, n = PASS == 1 ? n1 : w.cost2(p) * p.hkv;
        if (begin >= at && begin < at + n) {
          begin_b = b;
          begin_at = at;
          begin_at1 = at1;
        }
        at += n;
        at1 += n1;
      }
    }
  } else if (warp == kIssueWarp) {
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        mbar_init(&full[i], C::kTeam);
        mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&s_free[i], kCompute);
      }
      mbar_init(q_full, C::kQWarps);
      mbar_init(q_free, 1);
      for (int i = 0; i < 3; ++i) mbar_init(&l_full[i], C::kQWarps);
      mbar_init(met_bar, kCompute);
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc(&tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_holder;
  pdl_launch_dependents();

  const bool aligned = (smem_u32(prompt_smem) & 1023) == 0;      // the swizzle counts from 1 KB boundaries
  if (!aligned && tid == 0 && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusPipelineTimeout);

  // Calls fn(request's numbers, item) for every item of the run; all roles walk the same way.
  auto items = [&](auto&& fn) {
    const int64_t begin = line_of[0], end = aligned ? line_of[1] : line_of[0];
    if (begin >= end) return;
    Work<C> w;
    Item it;
    it.b = begin_b;
    w.set(p, it.b);
    int64_t request_at = begin_at, at1 = begin_at1;        // of the request on this pass's and on the first pass's line
    int64_t unit = PASS == 1 ? w.cost1(p) : w.cost2(p), unit1 = PASS == 1 ? unit : w.cost1(p);
    it.hk = static_cast<int>((begin - request_at) / unit);
    int64_t pos = begin, rest = begin - request_at - it.hk * unit;
    it.block = 0;
    it.first = true;
    it.flush = false;
    it.chunk = 0;
    int64_t block_at = 0;
    int t = 0;
    if (PASS == 1) {
      while (rest >= w.steps_of(p, it.block) + kStart) {
        const int n = w.steps_of(p, it.block++) + kStart;
        rest -= n;
        block_at += n;
      }
      t = static_cast<int>(rest);
      while (pos < end) {
        const int all = w.steps_of(p, it.block), n = static_cast<int>(min(static_cast<int64_t>(all - t), end - pos));
        if (n > 0) {
          it.t0 = t;
          it.n = n;
          it.load = it.release = true;
          it.at = 0;
          if (!fn(w, it)) return;
          it.first = false;
          pos += n;
          t += n;
        }
        if (pos >= end) return;
        pos += all + kStart - t;
        it.first = false;
        t = 0;
        if (++it.block == w.blocks) {
          it.block = 0;
          if (++it.hk == p.hkv) {
            it.hk = 0;
            do {
              if (++it.b >= p.ix.batch) return;
              w.set(p, it.b);
            } while (w.blocks == 0);
          }
        }
      }
    } else {
      // the first step that begins at or behind the run's begin
      const int all = w.common(p);
      const int64_t level = static_cast<int64_t>(all) * w.blocks;
      if (rest <= level) {
        t = static_cast<int>((rest + w.blocks - 1) / w.blocks);
        pos += static_cast<int64_t>(t) * w.blocks - rest;
      } else {
        t = all;
        int64_t x = level;
        while (x < rest) x += w.blocks - w.first_block(p, t++);
        pos += x - rest;
      }
      int loaded = -1;        // the block whose queries are there
      while (pos < end) {
        if (t >= w.steps) {
          t = 0;
          loaded = -1;
          if (++it.hk == p.hkv) {
            it.hk = 0;
            at1 += unit1 * p.hkv;
            do {
              if (++it.b >= p.ix.batch) return;
              w.set(p, it.b);
            } while (w.blocks == 0);
            unit1 = w.cost1(p);
          }
          continue;
        }
        int n = 0;
        while (n < kChunk && t + n < w.steps && pos < end) pos += w.blocks - w.first_block(p, t + n++);
        it.t0 = t;
        it.chunk = n;
        it.block = w.first_block(p, t);
        int64_t off = 0;
        for (int i = 0; i < it.block; ++i) off += w.steps_of(p, i) + kStart;
        for (; it.block < w.blocks; ++it.block) {
          const int mine = w.steps_of(p, it.block);
          it.n = min(n, mine - t);
          it.load = loaded != it.block;
          it.flush = it.block == w.blocks - 1;
          it.release = !it.flush || t + n >= w.steps || pos >= end || w.first_block(p, t + n) != it.block;
          it.at = at1 + it.hk * unit1 + off;
          loaded = it.block;
          if (!fn(w, it)) return;
          off += mine + kStart;
        }
        t += n;
      }
    }
  };

  if (warp >= kCompute && warp < kCompute + C::kTeam * C::kTeams) {
    // =============================== keys ===============================
    const int team = (warp - kCompute) / C::kTeam, part = (warp - kCompute) % C::kTeam;
    constexpr int kPart = 128 / C::kTeam;              // rows of this warp
    constexpr int kCh = KV8 ? 4 * NH : 8 * NH;         // 16-byte pieces of a cached row
    constexpr int kRowsPer = 32 / kCh;                 // rows of a warp's copy
    using Elem = typename std::conditional<KV8, uint8_t, uint16_t>::type;
    bool bad = false, ok = true;
    uint32_t stage0 = 0;                               // stages of the items before
    items([&](const Work<C>& w, const Item& it) {
      const int* rtt = p.ix.req_to_token + static_cast<int64_t>(w.o.row) * p.ix.table_stride;
      const int base = it.t0 * C::kStepKeys + part * kPart, stages = it.n * KT;
      struct Slots {
        int s[kPart / 32];
      };
      // slots of tokens lane, lane + 32, .. of this warp's rows of stage i
      auto slots_of = [&](int i) {
        Slots s;
#pragma unroll
        for (int k = 0; k < kPart / 32; ++k) {
          const int tok = base + i * 128 + k * 32 + lane;
          s.s[k] = i < stages && tok < w.o.len ? max(__ldcg(rtt + tok), -1) : kNoToken;      // no number of the table is taken for kNoToken
        }
        return s;
      };
      const int ch = lane % kCh, r0 = lane / kCh;
      const Elem* from = static_cast<const Elem*>(p.k_cache) + it.hk * p.kv_head_stride + ch * (16 / sizeof(Elem));
      int i = (team + C::kTeams - static_cast<int>(stage0 % C::kTeams)) % C::kTeams;
      Slots next = slots_of(i);
      for (; i < stages; i += C::kTeams) {
        const uint32_t n = stage0 + i, st = n % kStages, stage = smem_u32(ring) + st * C::kStage;
        Slots s = next;
#pragma unroll
        for (int k = 0; k < kPart / 32; ++k)
          if (s.s[k] < 0 || s.s[k] >= p.num_slots) {
            bad = bad || s.s[k] != kNoToken;
            s.s[k] = -1;
          }
        next = slots_of(i + C::kTeams);
        if (n >= kStages && !mbar_wait_relaxed(&empty[st], (n / kStages - 1) & 1, 20)) ok = false;
        if (!(ok = __all_sync(0xffffffffu, ok))) return false;
        if constexpr (!KV8) {
#pragma unroll
          for (int k = 0; k < kPart / kRowsPer; ++k) {
            const int row = k * kRowsPer + r0;
            const int rs = __shfl_sync(0xffffffffu, s.s[k * kRowsPer / 32], row & 31);
            cp16(stage + swz(part * kPart + row, ch, C::kKBlock), from + max(rs, 0) * p.kv_tok_stride, rs >= 0);
          }
          cp_commit();
          cp_wait_all();
        } else {
          constexpr int kBatch = 8;
          static_assert(kPart / kRowsPer % kBatch == 0, "batches of rows");
          auto widen = [&](uint32_t two) -> uint32_t {     // two 8-bit values -> two fp16, exactly
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu), FMT == kKvE5M2 ? __NV_E5M2 : __NV_E4M3);
            return static_cast<uint32_t>(h.x) | static_cast<uint32_t>(h.y) << 16;
          };
#pragma unroll
          for (int k0 = 0; k0 < kPart / kRowsPer; k0 += kBatch) {
            uint4 x[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
              const int row = (k0 + k) * kRowsPer + r0;
              const int rs = __shfl_sync(0xffffffffu, s.s[(k0 + k) * kRowsPer / 32], row & 31);
              x[k] = rs >= 0 ? __ldcg(reinterpret_cast<const uint4*>(from + rs * p.kv_tok_stride)) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
              const int row = part * kPart + (k0 + k) * kRowsPer + r0;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t a = h ? x[k].z : x[k].x, b = h ? x[k].w : x[k].y;
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + swz(row, ch * 2 + h, C::kKBlock)), "r"(widen(a)),
                             "r"(widen(a >> 16)), "r"(widen(b)), "r"(widen(b >> 16))
                             : "memory");
              }
            }
          }
          fence_proxy_async_smem();
        }
        if (bad) holes = 1;               // the computing warps look at every step
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);
      }
      stage0 += stages;
      return true;
    });
    if (!ok) fail_flag = 1;
    if (bad && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
  } else if (warp >= kCompute && warp < kIssueWarp) {
    // =============================== queries, and in the second pass the rows' normalisers ===============================
    const int me = warp - kCompute - C::kTeam * C::kTeams;
    bool ok = true;
    uint32_t loads = 0;
    items([&](const Work<C>& w, const Item& it) {
      if (!it.load) return true;
      if (loads > 0 && !mbar_wait_relaxed(q_free, (loads - 1) & 1)) ok = false;
      if (!(ok = __all_sync(0xffffffffu, ok))) return false;
      const int rows = w.rows_of(it.block), row0 = it.block * C::kRows;
      const uint16_t* q = static_cast<const uint16_t*>(p.q) + static_cast<int64_t>(w.o.first) * p.q_stride + static_cast<int64_t>(it.hk) * g * kD;
      constexpr int kCh = 8 * NH;               // 16-byte pieces of a row
      if constexpr (!kScaled) {
        for (int c = me * 32 + lane; c < rows * kCh; c += C::kQWarps * 32) {
          const int row = c / kCh, ch = c % kCh, j = (row0 + row) / g;
          cp16(smem_u32(sQ) + swz(row, ch, C::kQBlock), q + j * p.q_stride + static_cast<int64_t>(row0 + row - j * g) * kD + ch * 8, true);
        }
        cp_commit();
      } else {
        // the largest of a row gets an exponent of 14: what is 2^-25 times smaller than that goes below fp16's last place
        constexpr int kLanes = kCh < 32 ? kCh : 32;
        for (int c0 = me * 32; c0 < rows * kCh; c0 += C::kQWarps * 32) {
          const int c = c0 + lane, row = c / kCh, ch = c % kCh;
          uint4 x = make_uint4(0, 0, 0, 0);
          if (row < rows) {
            const int j = (row0 + row) / g;
            x = __ldcg(reinterpret_cast<const uint4*>(q + j * p.q_stride + static_cast<int64_t>(row0 + row - j * g) * kD + ch * 8));
          }
          uint32_t v[4] = {x.x, x.y, x.z, x.w};
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack_bf16x2(v[i]);
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
#pragma unroll
          for (int o = 1; o < kLanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const int raise = top > 0.f ? min(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), 126) : 0;
          const float by = __uint_as_float((raise + 127) << 23);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack_bf16x2(v[i]);
            const __half2 y = __floats2half2_rn(f.x * by, f.y * by);
            v[i] = *reinterpret_cast<const uint32_t*>(&y);
          }
          if (row < rows) {
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(sQ) + swz(row, ch, C::kQBlock)), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                         : "memory");
            if (ch == 0) row_mul[loads % 3][row] = p.scale_log2 * __uint_as_float((127 - raise) << 23);
          }
        }
        fence_proxy_async_smem();
      }
      if constexpr (PASS == 2) {
        const int n = w.steps_of(p, it.block), used = used_of;
        const int64_t line = line_of[2];
        // the last CTA whose run begins at or before x
        auto owner = [&](int64_t x) { return static_cast<int>(min(static_cast<int64_t>(used) - 1, ((x + 1) * used - 1) / line)); };
        const int c0 = owner(it.at), c1 = owner(it.at + n - 1);
        const int second = run_begin(line, c0, used) < it.at ? 1 : 0;      // the first CTA has the block in its second place
        for (int row = me * 32 + lane; row < rows; row += C::kQWarps * 32) {
          const int j = (row0 + row) / g, head = it.hk * g + row0 + row - j * g;
          float lse;
          if (c0 == c1) {
            lse = __ldcg(p.lse + static_cast<int64_t>(w.o.first + j) * p.hkv * g + head);
          } else {
            auto part = [&](int c) { return __ldcg(p.part + (static_cast<int64_t>(c) * 2 + (c == c0 ? second : 0)) * C::kRows + row); };
            float top = -INFINITY;
#pragma unroll 8
            for (int c = c0; c <= c1; ++c) top = fmaxf(top, part(c));
            const bool none = top == -INFINITY;
            const float sink = p.sink != nullptr ? __ldcg(p.sink + head) * kLog2e : -INFINITY;
            top = fmaxf(top, sink);
            float sum = p.sink != nullptr ? exp2f(sink - top) : 0.f;
#pragma unroll 8
            for (int c = c0; c <= c1; ++c) {
              const float v = part(c);
              sum += v == -INFINITY ? 0.f : exp2f(v - top);
            }
            lse = none && sum == sum ? -INFINITY : top + log2f(sum);
          }
          neg_lse[loads % 3][row] = lse == -INFINITY ? -INFINITY : -lse;       // nothing seen: no weights
        }
      }
      if constexpr (!kScaled) cp_wait_all();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(q_full);
        mbar_arrive(&l_full[loads % 3]);
      }
      ++loads;
      return true;
    });
    if (!ok) fail_flag = 1;
  } else if (warp == kIssueWarp) {
    if (elect_one()) {
      // =============================== products ===============================
      bool ok = true;
      const uint64_t q_desc = umma_desc_k_sw128(smem_u32(sQ)), k_desc0 = umma_desc_k_sw128(smem_u32(ring));
      const uint32_t fmt = KV8 || std::is_same<T, __half>::value ? 0u : 1u;
      uint32_t stage = 0, step = 0, loads = 0;
      items([&](const Work<C>& w, const Item& it) {
        if (it.load) {
          if (ok && !mbar_wait(q_full, loads & 1, &fail_flag)) ok = false;
          ++loads;
        }
        const int rows = w.rows_of(it.block);
        // first pass: N is the 128 tokens of a stage; second: the block's rows
        const uint32_t idesc = umma_idesc(128, PASS == 1 ? 128 : (rows + 15) / 16 * 16, 1, fmt, fmt, 0, 0);
        for (int t = 0; t < it.n && ok; ++t, ++step) {
          const uint32_t buf = step & 1;
          if (step >= 2 && !mbar_wait(&s_free[buf], ((step >> 1) - 1) & 1, &fail_flag)) ok = false;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt, ++stage) {
            const uint32_t st = stage % kStages;
            if (ok && !mbar_wait(&full[st], (stage / kStages) & 1, &fail_flag)) ok = false;
            if (!ok) break;
            fence_proxy_async_smem();       // copies by cp.async were made in the generic proxy
            tc_fence_after_sync();
            const uint64_t k_desc = k_desc0 + st * (C::kStage >> 4);
            const uint32_t to = tmem + buf * C::kCols + kt * 128;
#pragma unroll
            for (int h = 0; h < (PASS == 1 ? C::RT : 1); ++h) {
              if (h * kTileRows >= rows) break;
#pragma unroll
              for (int kk = 0; kk < 4 * NH; ++kk) {
                const uint64_t a = q_desc + (kk >> 2) * (C::kQBlock >> 4) + h * (kTileRows * 128 >> 4) + (kk & 3) * 2;
                const uint64_t k = k_desc + (kk >> 2) * (C::kKBlock >> 4) + (kk & 3) * 2;
                umma_f16(to + h * 128, PASS == 1 ? a : k, PASS == 1 ? k : a, idesc, kk > 0 ? 1u : 0u);
              }
            }
            umma_commit(&empty[st]);
          }
          if (!ok) break;
          umma_commit(&s_full[buf]);
        }
        if (ok && it.release) umma_commit(q_free);
        return ok;
      });
      if (!ok) fail_flag = 1;
    }
  } else {
    // =============================== scores ===============================
    const int quarter = warp >> 2, in_tile = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const bool capped = p.cap_out > 0.f;
    constexpr int kWarpCols = C::kWarpCols;
    bool ok = true;
    uint32_t step = 0, loads = 0, met = 0, turn = 0;
    auto meet = [&]() {        // of all computing warps; false where one has given up
      __syncwarp();
      if (lane == 0) mbar_arrive(met_bar);
      if (!mbar_wait(met_bar, met++ & 1, &fail_flag)) ok = false;
      return ok = __all_sync(0xffffffffu, ok);
    };
    auto wait_scores = [&]() {
      if (!mbar_wait(&s_full[step & 1], (step >> 1) & 1, &fail_flag)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after_sync();
      return ok;
    };
    auto scores_read = [&]() {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_free[step & 1]);
    };
    // cap tanh(x / cap), in the log2 domain; tanh(y) = 1 - 2 / (1 + e^(2 y))
    auto cap = [&](uint32_t x, float mul) { return __float_as_uint(p.cap_out * (1.f - __fdividef(2.f, 1.f + ex2(__uint_as_float(x) * mul * p.cap_in)))); };

    items([&](const Work<C>& w, const Item& it) {
      const int rows = w.rows_of(it.block), row0 = it.block * C::kRows, least = w.o.len - w.o.look;
      if (it.load) ++loads;
      const int held = (loads - 1) % 3;
      if (PASS == 2 || kScaled) {
        if (it.load && !mbar_wait(&l_full[held], ((loads - 1) / 3) & 1, &fail_flag)) ok = false;
        if (!(ok = __all_sync(0xffffffffu, ok))) return false;
      }
      if constexpr (PASS == 1) {
        const int row = (C::RT == 2 ? (quarter >> 1) * 128 : 0) + in_tile, col0 = quarter * kWarpCols % C::kStepKeys;
        const bool valid = row < rows, any = __any_sync(0xffffffffu, valid);
        const int place = least + (row0 + min(row, rows - 1)) / g, sure = least + row0 / g;       // sure: what all rows of the block see
        float mul = p.scale_log2;
        if constexpr (kScaled)
          if (valid) mul = row_mul[held][row];
        float m = -INFINITY;
        uint64_t sums[4] = {0, 0, 0, 0};      // pairs of fp32
        for (int t = 0; t < it.n; ++t, ++step) {
          if (!wait_scores()) return false;
#pragma unroll
          for (int half = 0; half < kWarpCols / 32; ++half) {
            uint32_t raw[32];
            if (any) {
              tmem_ld_32x32(tmem + lanes + (step & 1) * C::kCols + quarter * kWarpCols + half * 32, raw);
              tmem_ld_wait();
            }
            if (half == kWarpCols / 32 - 1) scores_read();
            if (!any) continue;
            const int key = (it.t0 + t) * C::kStepKeys + col0 + half * 32;
            float by = mul;
            if (capped) {
              by = 1.f;
#pragma unroll
              for (int c = 0; c < 32; ++c) raw[c] = cap(raw[c], mul);
            }
            const bool gaps = __any_sync(0xffffffffu, *const_cast<const volatile int*>(&holes) != 0);
            if (key + 31 > sure || gaps) {
              const int seen = place + 1 - key;          // columns in front
              uint32_t there = 0xffffffffu;
              if (gaps) {      // rare: tokens whose slots lie outside the cache
                const int s = key + lane < w.o.len ? __ldcg(p.ix.req_to_token + static_cast<int64_t>(w.o.row) * p.ix.table_stride + key + lane) : -1;
                there = __ballot_sync(0xffffffffu, s >= 0 && s < p.num_slots);
              }
#pragma unroll
              for (int c = 0; c < 32; ++c) raw[c] = c < seen && ((there >> c) & 1) ? raw[c] : __float_as_uint(-INFINITY);
            }
            float mx[2] = {fmaxf(__uint_as_float(raw[0]), __uint_as_float(raw[1])), fmaxf(__uint_as_float(raw[2]), __uint_as_float(raw[3]))};
#pragma unroll
            for (int c = 4; c < 32; c += 2) mx[(c >> 1) & 1] = max3(mx[(c >> 1) & 1], __uint_as_float(raw[c]), __uint_as_float(raw[c + 1]));
            const float top = fmaxf(mx[0], mx[1]) * by;
            if (top > m + kRescaleThreshold) {        // the first tile raises; so does one behind tiles of minus infinity
              const float f = m == -INFINITY ? 0.f : exp2f(m - top);
#pragma unroll
              for (int i = 0; i < 4; ++i) sums[i] = m == -INFINITY ? sums[i] : fma2(sums[i], pair_of(f, f), 0);
              m = top;
            }
            const float neg = m == -INFINITY ? 0.f : -m;
            const uint64_t by2 = pair_of(by, by), neg2 = pair_of(neg, neg);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 x = halves_of(fma2(pair_of(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1])), by2, neg2));
              sums[i & 3] = add2(sums[i & 3], pair_of(ex2(x.x), ex2(x.y)));
            }
          }
        }
        // ---- the quarters' maxima and sums meet ----
        const float2 both = halves_of(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])));
        float2* parts = reinterpret_cast<float2*>(cells) + (turn++ & 1) * 512;
        parts[quarter * 128 + in_tile] = make_float2(m, both.x + both.y);
        if (!meet()) return false;
        if (tid < rows) {
          const int tile = C::RT == 2 ? tid >> 7 : 0;
          constexpr int kParts = C::RT == 2 ? 2 : 4;
          float2 x[kParts];
          float top = -INFINITY, sum = 0.f;
#pragma unroll
          for (int i = 0; i < kParts; ++i) {
            x[i] = parts[(tile * kParts + i) * 128 + (tid & 127)];
            top = fmaxf(top, x[i].x);
          }
          const bool none = top == -INFINITY;
#pragma unroll
          for (int i = 0; i < kParts; ++i) sum += x[i].x == -INFINITY ? x[i].y : x[i].y * exp2f(x[i].x - top);       // no score: 0, or no number
          const bool whole = it.t0 == 0 && it.n == w.steps_of(p, it.block);
          const int j = (row0 + tid) / g, head = it.hk * g + row0 + tid - j * g;
          float lse = none && sum == 0.f ? -INFINITY : top + log2f(sum);
          if (whole) {
            if (p.sink != nullptr && lse != -INFINITY) {
              const float sink = __ldcg(p.sink + head) * kLog2e, at = fmaxf(top, sink);
              lse = at + log2f(sum * exp2f(top - at) + exp2f(sink - at));
            }
            p.lse[static_cast<int64_t>(w.o.first + j) * p.hkv * g + head] = lse;
          } else {
            p.part[(static_cast<int64_t>(blockIdx.x) * 2 + (it.first ? 0 : 1)) * C::kRows + tid] = lse;
          }
        }
      } else {
        const int kt = C::RT == 1 && KT == 2 ? quarter >> 1 : 0, group = KT == 2 ? quarter & 1 : quarter;       // stage and part of the columns
        const int col0 = group * kWarpCols, chunk_keys = it.chunk * C::kStepKeys;
        const float* neg = neg_lse[held] + col0;
        const float* muls = row_mul[held] + (kScaled ? col0 : 0);
        for (int t = 0; t < it.n; ++t, ++step) {
          const int token = (it.t0 + t) * C::kStepKeys + kt * 128 + in_tile;
          // this token is seen by the block's rows from `low` on
          const int low = token > least ? min(static_cast<int64_t>(token - least) * g - row0, static_cast<int64_t>(C::kRows)) : 0;
          uint64_t sums[4] = {0, 0, 0, 0};
          if (!wait_scores()) return false;
#pragma unroll
          for (int half = 0; half < kWarpCols / 32; ++half) {
            uint32_t raw[32];
            const int col = col0 + half * 32;
            const bool any = col < rows;
            if (any) {
              tmem_ld_32x32(tmem + lanes + (step & 1) * C::kCols + quarter * kWarpCols + half * 32, raw);
              tmem_ld_wait();
            }
            if (half == kWarpCols / 32 - 1) scores_read();
            if (!any) continue;
            if (capped) {
#pragma unroll
              for (int c = 0; c < 32; ++c) raw[c] = cap(raw[c], kScaled ? muls[half * 32 + c] : p.scale_log2);
            }
            auto add_up = [&](auto masked) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 n4 = *reinterpret_cast<const float4*>(neg + half * 32 + 4 * i);
                float4 m4 = make_float4(p.scale_log2, p.scale_log2, p.scale_log2, p.scale_log2);
                if (kScaled) m4 = *reinterpret_cast<const float4*>(muls + half * 32 + 4 * i);
                if (capped) m4 = make_float4(1.f, 1.f, 1.f, 1.f);
                const float2 x = halves_of(fma2(pair_of(__uint_as_float(raw[4 * i]), __uint_as_float(raw[4 * i + 1])), pair_of(m4.x, m4.y), pair_of(n4.x, n4.y)));
                const float2 y = halves_of(fma2(pair_of(__uint_as_float(raw[4 * i + 2]), __uint_as_float(raw[4 * i + 3])), pair_of(m4.z, m4.w), pair_of(n4.z, n4.w)));
                float e[4] = {ex2(x.x), ex2(x.y), ex2(y.x), ex2(y.y)};
                if constexpr (decltype(masked)::value) {
#pragma unroll
                  for (int k = 0; k < 4; ++k) e[k] = col + 4 * i + k >= low && col + 4 * i + k < rows ? e[k] : 0.f;
                }
                sums[(2 * i) & 3] = add2(sums[(2 * i) & 3], pair_of(e[0], e[1]));
                sums[(2 * i + 1) & 3] = add2(sums[(2 * i + 1) & 3], pair_of(e[2], e[3]));
              }
            };
            if (col + 32 > rows || __any_sync(0xffffffffu, low > col)) {
              add_up(std::true_type());
            } else {
              add_up(std::false_type());
            }
          }
          const float2 both = halves_of(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])));
          float sum = both.x + both.y;
          if (*const_cast<const volatile int*>(&holes) != 0) {       // rare: a token whose slot lies outside the cache is not seen
            const int s = token < w.o.len ? __ldcg(p.ix.req_to_token + static_cast<int64_t>(w.o.row) * p.ix.table_stride + token) : -1;
            if (s < 0 || s >= p.num_slots) sum = 0.f;
          }
          float* cell = cells + group * chunk_keys + t * C::kStepKeys + kt * 128 + in_tile;
          *cell = w.first_block(p, it.t0 + t) == it.block ? sum : *cell + sum;
        }
        if (it.flush) {
          if (!meet()) return false;
          float* to = p.sums.data + w.o.row * p.sums.row_stride + it.hk * p.sums.head_stride;
          for (int i = tid; i < chunk_keys; i += 32 * kCompute) {
            const int token = it.t0 * C::kStepKeys + i;
            if (token >= w.o.len) break;
            float sum = cells[i];
#pragma unroll
            for (int k = 1; k < C::kGroups; ++k) sum += cells[k * chunk_keys + i];
            to[token] = p.add && token < w.o.prefix ? __ldcg(to + token) + sum : sum;
          }
          if (!meet()) return false;
        }
      }
      return true;
    });
    if (!ok) fail_flag = 1;
  }

  tc_fence_before_sync();
  __syncthreads();
  if (fail_flag) {
    if (tid == 0 && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusPipelineTimeout);
    for (int i = 0; i < 64; ++i) __nanosleep(1000);      // products and copies in flight land before the memory goes
    __syncthreads();
  }
  if (warp == kIssueWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int NH, int FMT, int R>
int launch_one(const PromptParams& p, cudaStream_t s) {
  using C = Cfg<NH, FMT != kKvSame, R>;
  auto first = weights_prompt_kernel<T, NH, FMT, R, 1>;
  auto second = weights_prompt_kernel<T, NH, FMT, R, 2>;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(first), C::kSmem) != cudaSuccess) return -3;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(second), C::kSmem) != cudaSuccess) return -3;
  cudaError_t err = launch_pdl(first, dim3(p.ctas), dim3(kThreads), C::kSmem, s, p);
  note_launch();
  if (err != cudaSuccess) return -4;
  err = launch_pdl(second, dim3(p.ctas), dim3(kThreads), C::kSmem, s, p);
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}
template <typename T, int NH, int R>
int launch_format(const PromptParams& p, int fmt, cudaStream_t s) {
  switch (fmt) {
    case kKvSame: return launch_one<T, NH, kKvSame, R>(p, s);
    case kKvE4M3: return launch_one<T, NH, kKvE4M3, R>(p, s);
    default: return launch_one<T, NH, kKvE5M2, R>(p, s);
  }
}
template <typename T>
int launch_type(const PromptParams& p, int head_dim, int fmt, int tiles, cudaStream_t s) {
  switch (head_dim) {
    case 64: return tiles == 2 ? launch_format<T, 1, 2>(p, fmt, s) : launch_format<T, 1, 1>(p, fmt, s);
    case 128: return tiles == 2 ? launch_format<T, 2, 2>(p, fmt, s) : launch_format<T, 2, 1>(p, fmt, s);
    default: return launch_format<T, 4, 1>(p, fmt, s);
  }
}

// Row tiles of a block: two where a request has more observed rows than one tile holds, on average; 256 features leave no room for two.
int row_tiles(const WeightsPromptArgs& a) {
  const int64_t each = a.rows / std::max(1, a.index.batch), look = a.last > 0 ? std::min<int64_t>(a.last, each) : each;
  return a.head_dim <= 128 && look * (a.hq / a.hkv) > kTileRows ? 2 : 1;
}

}  // namespace

bool weights_prompt_covers(int head_dim, int group) { return (head_dim == 64 || head_dim == 128 || head_dim == 256) && group >= 1 && group <= 32; }

int64_t weights_prompt_floats(const WeightsPromptArgs& a) { return a.rows * a.hq + static_cast<int64_t>(a.num_sms) * 2 * row_tiles(a) * kTileRows; }

int launch_weights_prompt(const WeightsPromptArgs& a, cudaStream_t s) {
  if (a.hkv <= 0 || a.hq % a.hkv != 0 || !weights_prompt_covers(a.head_dim, a.hq / a.hkv)) return -1;
  if (a.index.batch <= 0 || a.rows <= 0) return 0;
  PromptParams p{};
  p.ix = a.index;
  p.sums = a.sums;
  p.prefix_lens = a.prefix_lens;
  p.q_start = a.q_start;
  p.q = a.q;
  p.k_cache = a.k_cache;
  p.lse = a.workspace;
  p.part = a.workspace + a.rows * a.hq;
  p.sink = a.sink;
  p.q_stride = a.q_stride;
  p.num_slots = a.num_slots;
  p.kv_tok_stride = a.kv_tok_stride;
  p.kv_head_stride = a.kv_head_stride;
  p.rows = static_cast<int>(a.rows);
  p.hkv = a.hkv;
  p.group = a.hq / a.hkv;
  p.last = a.last;
  p.ctas = a.num_sms;
  p.add = a.add;
  p.scale_log2 = a.scale * kLog2e;
  if (a.logit_cap > 0.f) {
    p.cap_in = 2.f / a.logit_cap;
    p.cap_out = a.logit_cap * kLog2e;
  }
  return a.dt == kF16 ? launch_type<__half>(p, a.head_dim, a.kv_fmt, row_tiles(a), s) : launch_type<__nv_bfloat16>(p, a.head_dim, a.kv_fmt, row_tiles(a), s);
}

}  // namespace mb200
