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
//   * Rows are (query, head of the group) pairs; RT tiles of 128 make a block.  A CTA holds one operand, the block, in shared memory, and copying
//     warps bring the other through a ring of 128-row stages in the operand layout, keys by slot.  A step is KT stages: RT * KT = 2, 256 score
//     columns in tensor memory, two buffers (heads of 256: one stage, 128 columns).
//   * First pass: S = Q K^T, blocks of rows, a row per lane.  16 warps, four to every 32 lanes of tensor memory, take a quarter of the columns
//     each, with a maximum and sum of their own; they join at the block's end.  Units (request, kv head, block) times steps form one line, dealt
//     evenly to the CTAs; a row's normaliser is written out, or a partial one per CTA.
//   * Second pass: S^T = K Q^T, a token per lane: its sum over the rows is a sum in a thread.  Where the observed rows fit a block or two they
//     stay in shared memory and keys go by; tokens are dealt by what they cost, the blocks that see them, and no two CTAs have the same
//     token.  Where there are more rows, 256 tokens are the block and rows go by, in a line as in the first pass; a third kernel adds up the parts
//     of blocks that were cut.  Nothing depends on the order of CTAs.
//   * A CTA's first block is brought by the computing warps, which have nothing else to do then, later ones by a warp of its own.
// What it costs: 256 x 128 scores take 2048 cycles of exponentials (16 per cycle and SM; products take half of that), and the first pass 2750 in
// all, the second 3050.  One request of 32000 tokens behind its last 64, 32 / 8 heads of 128, has 13.5 such steps an SM: 40 of its 95 us, starts and
// ends of the passes some 18, and the rest is not explained; 2 x 1500 tokens, all queries: 132 us, of which steps without masks at these
// rates would be less than half, and a step is masked for all warps as soon as one score of it is.  Where there are few scores, two starts
// and ends count: 6 us to the first scores, 2.5 to join a block's normalisers from the first pass, 2 at the end (8 x 2048 tokens behind the
// last 32: 46.5 us).  Soft caps take the masked steps' loop and a tanhf per score (83, 195 and 250 us), 8-bit rows are widened by the
// copying warps (the three cases over e4m3: 101, 180 and 605 us; why the last one is so slow was not looked into).
#pragma once

#include <algorithm>

#include "common.cuh"
#include "evict.cuh"

namespace mb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLargest = 1e30f;          // a sum of exponentials that is not below this gets a new maximum
constexpr int kTileRows = 128;             // MMA M
constexpr int kStart = 2;                  // steps' time that every unit of the first pass costs beside its steps
constexpr int kChunk = 8;                  // steps whose sums wait in shared memory
constexpr int kNoToken = -0x7fffffff;
constexpr int kCompute = 16;               // warps
struct PromptParams {
  CacheIndex ix;
  WeightSums sums;
  const int* prefix_lens;
  const int* q_start;
  const void* q;
  const void* k_cache;
  float* lse;        // [rows of q][hq]: normalisers of blocks that lie in one CTA
  float* part;       // [CTAs][2][block rows] of the first pass
  float* part_sum;   // the same of tokens, where rows go by
  int4* jobs;        // [CTAs] of units of tokens that end in the CTA and began in another: kv head and request, block, first CTA and its place
  const float* sink;
  int64_t q_stride, num_slots, kv_tok_stride, kv_head_stride;
  int rows, hkv, group, last, ctas;
  uint32_t inv_group;      // of 16 bits: quotients of numbers below 320, exactly
  uint32_t inv_group32;    // floor(2^32 / group), 2^32 - 1 for 1
  bool add;
  float scale_log2, cap_pre, cap_post;     // a scaled score x becomes cap_post tanh(x cap_pre); cap_post 0: no soft cap
};

// n / group, n >= 0: the quotient by the reciprocal is too small by one at most
__device__ __forceinline__ int by_group(const PromptParams& p, int n) {
  int q = static_cast<int>(__umulhi(static_cast<uint32_t>(n), p.inv_group32));
  if (n - q * p.group >= p.group) ++q;
  return q;
}

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
  const int start = __ldcg(p.q_start + b), n = o.prefix >= 0 ? c.len - o.prefix : 1;
  o.look = c.len > 0 && o.prefix < c.len ? (p.last > 0 ? min(p.last, n) : n) : 0;
  if (o.look > 0 && (o.prefix < 0 || start < 0 || n > p.rows - start)) {
    o.bad = true;
    o.look = 0;
  }
  o.first = start + n - o.look;
  return o;
}

template <int NH, bool KV8, int R, int PASS>
struct Cfg {
  static constexpr int RT = R, KT = NH == 4 ? 1 : 2 / R;
  static_assert(PASS != 3 || KT == 1, "rows go by one stage a step");
  static constexpr int kD = 64 * NH;
  static constexpr int kRows = RT * kTileRows;               // of a block
  static constexpr int kStepKeys = KT * 128;
  static constexpr int kCols = RT * KT * 128, kWarpCols = kCols / 4;
  static constexpr int kBlock = kRows * 128, kBlockBytes = NH * kBlock;    // 64 features of a block's rows
  static constexpr int kPiece = 128 * 128, kStage = NH * kPiece;
  static constexpr int kStages = NH == 4 ? 2 : NH == 2 ? (R == 2 ? 4 : 5) : 6;
  // Warps: those that compute, that copy stages (kCopying of them, every kCopying-th stage each), one that walks through the CTA's run, one that
  // copies blocks, one that issues products.
  static constexpr int kCopy = 5, kCopying = kCopy < kStages ? kCopy : kStages;
  static constexpr int kWalkWarp = kCompute + kCopy, kBlockWarp = kWalkWarp + 1, kIssueWarp = kBlockWarp + 1, kThreads = 32 * (kIssueWarp + 1);
  // Registers: those of a launch, of the computing threads, of the others.  A quarter of the warps share 16384, four computing ones each.
  static constexpr int kLaunchRegs = 80, kComputeRegs = 88, kOtherRegs = 64;
  static_assert(4 * kComputeRegs + (kCopy + 3) / 4 * kOtherRegs <= (4 + (kCopy + 3) / 4) * kLaunchRegs && (kCopy + 3) % 4 == 0, "register split");
  static constexpr int kSmem = kBlockBytes + kStages * kStage;
  static constexpr int kGroups = 4 / KT;                     // parts of a token's sum
  // Normalisers and factors of rows: of the last blocks, or of the stages.  A place is written anew behind the last product of the block in
  // front, or of the stage kStages before.  That product was issued when the scores of two steps before had been read, so that the computing
  // warps were through with the step before those.
  static constexpr int kRing = PASS == 3 ? kStages + 3 : 4, kRingRows = PASS == 3 ? 128 : kRows;
  static_assert(2 * kCols <= 512, "tensor memory");
};

// What the passes do with a request.  Rows r = j * group + h, in blocks of kRows.
template <typename C, int PASS>
struct Work {
  Observed o;
  int rows, blocks, units;       // units: blocks of rows, or (third kind) of tokens
  __device__ __forceinline__ void set(const PromptParams& p, const Observed& with) {
    o = with;
    rows = o.look * p.group;
    blocks = (rows + C::kRows - 1) / C::kRows;
    units = PASS == 3 ? (rows > 0 ? (o.len + C::kRows - 1) / C::kRows : 0) : blocks;
  }
  __device__ __forceinline__ int least() const { return o.len - o.look; }        // place of the first row
  __device__ __forceinline__ int rows_of(int block) const { return min(C::kRows, rows - block * C::kRows); }
  // steps of the first pass: up to the largest place of a block's rows
  __device__ __forceinline__ int steps1(const PromptParams& p, int block) const {
    return (least() + by_group(p, min(rows, (block + 1) * C::kRows) - 1)) / C::kStepKeys + 1;
  }
  // first tile of rows that sees a block of tokens
  __device__ __forceinline__ int first_tile(const PromptParams& p, int block) const {
    const int j = block * C::kRows - least();
    return j > 0 ? j * p.group / kTileRows : 0;
  }
  __device__ __forceinline__ int steps_of(const PromptParams& p, int unit) const {
    return PASS == 3 ? (rows + kTileRows - 1) / kTileRows - first_tile(p, unit) : steps1(p, unit);
  }
  // of the second pass: steps, first block that sees one, steps from the first one on that all blocks see
  __device__ __forceinline__ int steps() const { return rows > 0 ? (o.len + C::kStepKeys - 1) / C::kStepKeys : 0; }
  __device__ __forceinline__ int first_block(const PromptParams& p, int step) const {
    const int j = step * C::kStepKeys - least();
    return j > 0 ? j * p.group / C::kRows : 0;
  }
  __device__ __forceinline__ int common(const PromptParams& p) const { return min(steps(), (least() + by_group(p, C::kRows - 1)) / C::kStepKeys + 1); }
  // of one kv head, on the first pass's line and on this one's
  __device__ __forceinline__ int64_t cost1(const PromptParams& p) const {
    int64_t n = 0;
    for (int i = 0; i < blocks; ++i) n += steps1(p, i) + kStart;
    return n;
  }
  __device__ __forceinline__ int64_t cost(const PromptParams& p) const {
    int64_t n = 0;
    if (PASS == 2) {
      if (blocks == 0) return 0;
      const int all = common(p), every = steps();
      n = static_cast<int64_t>(all) * blocks;
      for (int t = all; t < every; ++t) n += blocks - first_block(p, t);
    } else {
      for (int i = 0; i < units; ++i) n += steps_of(p, i) + kStart;
    }
    return n;
  }
};

// Steps t0 .. t0 + n - 1 of a block
struct Item {
  int b, hk, block, t0, n;
  bool load, release;    // the block is not in shared memory yet; the next item, if any, loads another
  bool first;            // the item begins the CTA's run (not in the second pass)
  bool flush;            // last block over these steps (second pass)
  int chunk;             // steps whose sums wait (second pass)
  int64_t at;            // where the unit begins: on the first pass's line (second pass), on its own (else)
  int64_t at1;           // where the request's and kv head's units begin on the first pass's line (blocks of tokens)
};
struct Record {
  Observed o;
  Item it;               // n 0: the run's end
};
constexpr int kItems = 4;      // items that the walking warp is ahead

// CTAs that share a line of units and where CTA c's run begins
__device__ __forceinline__ int used_ctas(const PromptParams& p, int64_t line) {
  return static_cast<int>(min(static_cast<int64_t>(p.ctas), max(line / 2, static_cast<int64_t>(1))));
}
// (A division of 64 bits takes some 500 cycles.)
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

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  const int sz = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(sz) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }       // all but the newest group
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// PASS 1: normalisers; 2: sums, blocks of rows; 3: sums, blocks of tokens.  FMT: what the cache holds (kKvSame, kKvE4M3, kKvE5M2)
template <typename T, int NH, int FMT, int R, int PASS>
__global__ void __launch_bounds__(Cfg<NH, FMT != kKvSame, R, PASS>::kThreads, 1) weights_prompt_kernel(const PromptParams p) {
  constexpr bool KV8 = FMT != kKvSame;
  constexpr bool kScaled = KV8 && !std::is_same<T, __half>::value;      // bf16 queries become fp16, scaled by a power of two per row
  using C = Cfg<NH, KV8, R, PASS>;
  using W = Work<C, PASS>;
  constexpr int kD = C::kD, kStages = C::kStages, KT = C::KT, kRing = C::kRing, kIssueWarp = C::kIssueWarp;
  extern __shared__ __align__(1024) uint8_t prompt_smem[];
  __shared__ uint64_t bars[2 * kStages + 8 + kRing + 2 * kItems];
  __shared__ uint32_t tmem_holder;
  __shared__ int fail_flag, holes;
  __shared__ int used_of;                                   // CTAs of the first pass
  __shared__ int64_t line_of[2];                            // lines of the first pass and of this one
  __shared__ Record records[kItems];
  __shared__ __align__(16) float neg_lse[kRing][C::kRingRows];      // -normaliser of rows (sums)
  __shared__ __align__(16) float row_mul[kRing][kScaled ? C::kRingRows : 4];
  __shared__ __align__(16) float cells[kChunk * 512];       // second pass: [parts][tokens]; else 2 x [4][128] maxima and sums
  uint8_t* sBlock = prompt_smem;
  uint8_t* ring = sBlock + C::kBlockBytes;
  uint64_t* full = bars;                 // [stage] the warps of a team
  uint64_t* empty = full + kStages;      // [stage] tcgen05.commit
  uint64_t* s_full = empty + kStages;    // [buffer] tcgen05.commit
  uint64_t* s_free = s_full + 2;         // [buffer] the computing warps have read the scores
  uint64_t* b_first = s_free + 2;        // the computing warps: the first block
  uint64_t* b_full = b_first + 1;        // the warp that copies blocks: the others
  uint64_t* b_free = b_full + 1;         // tcgen05.commit: the last scores of a block
  uint64_t* met_bar = b_free + 1;        // the computing warps among themselves
  uint64_t* l_full = met_bar + 1;        // [ring] who writes normalisers and factors (not of the first block)
  uint64_t* r_full = l_full + kRing;     // [record] the walking warp
  uint64_t* r_free = r_full + kItems;    // [record] all others: computing, copying and issuing warps

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = p.group;
  pdl_wait_loads();

  // ---- where this CTA's run begins: what one lane of the walking warp goes on with ----
  W w;
  Item it{};
  int64_t pos = 0, end = 0, rest = 0, at1 = 0, unit1 = 0;      // on this pass's line; behind the unit's first; on the first pass's line
  bool walks = false;
  if (warp == C::kWalkWarp) {
    const int per = (p.ix.batch + 31) / 32;
    const int first = min(p.ix.batch, lane * per), last = min(p.ix.batch, first + per);
    int64_t mine1 = 0, mine = 0;
    bool bad = false;
    int64_t c1 = 0, c = 0;                // of one kv head of this lane's first request
    for (int b = last - 1; b >= first; --b) {
      w.set(p, observed_of(p, b));
      bad = bad || w.o.bad;
      c = w.cost(p);
      c1 = PASS == 1 ? c : w.cost1(p);
      mine += c * p.hkv;
      mine1 += c1 * p.hkv;
    }
    if (PASS == 1 && bad && blockIdx.x == 0 && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
    int64_t incl1 = mine1, incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
      if (PASS != 1) {
        const int64_t v1 = __shfl_up_sync(0xffffffffu, incl1, o);
        if (lane >= o) incl1 += v1;
      }
    }
    if (PASS == 1) incl1 = incl;
    const int64_t line1 = __shfl_sync(0xffffffffu, incl1, 31), line = __shfl_sync(0xffffffffu, incl, 31);
    // the second pass has no cost beside its steps
    const int used = PASS == 2 ? static_cast<int>(min(static_cast<int64_t>(p.ctas), max(line, static_cast<int64_t>(1)))) : used_ctas(p, line);
    const int cta = blockIdx.x;
    pos = cta < used ? run_begin(line, cta, used) : line;
    end = cta < used ? run_begin(line, cta + 1, used) : line;
    if (lane == 0) {
      line_of[0] = line1;
      line_of[1] = line;
      used_of = used_ctas(p, line1);
      fail_flag = 0;
      holes = 0;
      if (PASS == 1) p.jobs[blockIdx.x] = make_int4(-1, 0, 0, 0);
    }
    int64_t at = incl - mine;
    at1 = incl1 - mine1;
    if (pos < end && pos >= at && pos < incl) {
      for (int b = first; b < last; ++b) {
        if (b > first) {
          w.set(p, observed_of(p, b));
          c = w.cost(p);
          c1 = PASS == 1 ? c : w.cost1(p);
        }
        if (pos < at + c * p.hkv) {
          const int64_t in = pos - at;
          it.b = b;
          it.hk = c < (1ll << 31) && in < (1ll << 31) ? static_cast<uint32_t>(in) / static_cast<uint32_t>(c) : static_cast<int>(in / c);
          rest = in - it.hk * c;
          unit1 = c1;
          walks = true;
          break;
        }
        at += c * p.hkv;
        at1 += c1 * p.hkv;
      }
    }
    if (pos >= end) walks = lane == 0;
  } else if (warp == kIssueWarp) {
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&s_free[i], kCompute);
      }
      mbar_init(b_first, kCompute);
      mbar_init(b_full, 1);
      mbar_init(b_free, 1);
      mbar_init(met_bar, kCompute);
      for (int i = 0; i < kRing; ++i) mbar_init(&l_full[i], 1);
      for (int i = 0; i < kItems; ++i) {
        mbar_init(&r_full[i], 1);
        mbar_init(&r_free[i], kCompute + C::kCopying + 2);
      }
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

  // Calls fn(request's numbers, item) for every item of the run
  auto items = [&](bool one, auto&& fn) {      // one: of a warp that is one thread
    for (uint32_t i = 0;; ++i) {
      bool there = mbar_wait(&r_full[i % kItems], (i / kItems) & 1, &fail_flag);
      if (!one) there = __all_sync(0xffffffffu, there);
      if (!there) {
        fail_flag = 1;
        return;
      }
      const Record& r = records[i % kItems];
      const Item now = r.it;
      if (now.n == 0) return;
      W v;
      v.set(p, r.o);
      if (!fn(v, now)) return;
      if (!one) __syncwarp();
      if (one || lane == 0) mbar_arrive(&r_free[i % kItems]);
    }
  };

  // ---- what is copied, by one warp or several ----
  using Elem = typename std::conditional<KV8, uint8_t, uint16_t>::type;
  constexpr int kKeyPieces = KV8 ? 4 * NH : 8 * NH, kKeyRows = 32 / kKeyPieces;      // 16-byte pieces of a cached row; rows of a warp's copy
  auto widen = [&](uint32_t two) -> uint32_t {     // two 8-bit values -> two fp16, exactly
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu), FMT == kKvE5M2 ? __NV_E5M2 : __NV_E4M3);
    return static_cast<uint32_t>(h.x) | static_cast<uint32_t>(h.y) << 16;
  };
  // 32 rows of keys whose slots the lanes have, to rows row0 .. of a tile with blocks of `block` bytes.  What stands for a token that is none, or
  // whose slot lies outside the cache, is some other row: its scores are left out where they are read.
  auto copy_keys = [&](const Elem* head, int slot, uint32_t dst, int row0, int block) {
    const int ch = lane % kKeyPieces, r0 = lane / kKeyPieces;
    const Elem* from = head + ch * (16 / sizeof(Elem));
    if constexpr (!KV8) {
      // a copy is a slot, an address and the copy itself: one warp has to keep up with the products
      uint32_t at[8 / kKeyRows];
#pragma unroll
      for (int k = 0; k < 8 / kKeyRows; ++k) at[k] = dst + swz(row0 + k * kKeyRows + r0, ch, block) - k * kKeyRows * 128;
      constexpr int kBatch = 8;          // slots first, then copies: one after the other a copy waits for its slot, 64 cycles each
#pragma unroll
      for (int k0 = 0; k0 < kKeyPieces; k0 += kBatch) {
        int rs[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) rs[k] = __shfl_sync(0xffffffffu, slot, (k0 + k) * kKeyRows + r0);
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(at[(k0 + k) % (8 / kKeyRows)] + (k0 + k) * kKeyRows * 128),
                       "l"(from + rs[k] * p.kv_tok_stride)
                       : "memory");
      }
    } else {
      constexpr int kBatch = kKeyPieces < 8 ? kKeyPieces : 8;
#pragma unroll 1
      for (int k0 = 0; k0 < kKeyPieces; k0 += kBatch) {
        uint4 x[kBatch];
        int rs[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) rs[k] = __shfl_sync(0xffffffffu, slot, (k0 + k) * kKeyRows + r0);
#pragma unroll
        for (int k = 0; k < kBatch; ++k) x[k] = __ldcg(reinterpret_cast<const uint4*>(from + rs[k] * p.kv_tok_stride));
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int row = row0 + (k0 + k) * kKeyRows + r0;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t a = h ? x[k].z : x[k].x, b = h ? x[k].w : x[k].y;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + swz(row, ch * 2 + h, block)), "r"(widen(a)), "r"(widen(a >> 16)),
                         "r"(widen(b)), "r"(widen(b >> 16))
                         : "memory");
          }
        }
      }
    }
  };
  // n rows of queries from row r0 of the request on, every `step`-th 32 pieces from the `me`-th on
  auto copy_queries = [&](const W& w, int hk, int r0, int n, uint32_t dst, int block, float* muls, int me, int step) {
    const int j0 = by_group(p, r0), h0 = r0 - j0 * g;
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + static_cast<int64_t>(w.o.first + j0) * p.q_stride + static_cast<int64_t>(hk) * g * kD;
    constexpr int kCh = 8 * NH, kRowsPer = 32 / kCh;          // 16-byte pieces of a row
    const int ch = lane % kCh;
#pragma unroll 4
    for (int row = me * kRowsPer + lane / kCh; row < (n + kRowsPer - 1) / kRowsPer * kRowsPer; row += step * kRowsPer) {
      const int x = h0 + row, j = (x * p.inv_group) >> 16;
      const uint16_t* from = q + j * p.q_stride + static_cast<int64_t>(x - j * g) * kD + ch * 8;
      if constexpr (!kScaled) {
        if (row < n) cp16(dst + swz(row, ch, block), from, true);
      } else {
        // the largest of a row gets an exponent of 14: what is 2^-25 times smaller than that goes below fp16's last place
        uint4 y = make_uint4(0, 0, 0, 0);
        if (row < n) y = __ldcg(reinterpret_cast<const uint4*>(from));
        uint32_t v[4] = {y.x, y.y, y.z, y.w};
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack_bf16x2(v[i]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
#pragma unroll
        for (int o = 1; o < kCh; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int raise = top > 0.f ? min(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), 126) : 0;
        const float by = __uint_as_float((raise + 127) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack_bf16x2(v[i]);
          const __half2 z = __floats2half2_rn(f.x * by, f.y * by);
          v[i] = *reinterpret_cast<const uint32_t*>(&z);
        }
        if (row < n) {
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + swz(row, ch, block)), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
          if (ch == 0) muls[row] = p.scale_log2 * __uint_as_float((127 - raise) << 23);
        }
      }
    }
  };
  // -normaliser of row r of the request, whose block begins at `at` on the first pass's line and has n steps
  struct Parts {
    int c0, c1, second;       // the first CTA has the block in its second place
  };
  auto parts_of = [&](int64_t at, int n) {
    const int64_t line = line_of[0];
    Parts x;
    x.c0 = owner_of(line, at, used_of);
    x.c1 = owner_of(line, at + n - 1, used_of);
    x.second = run_begin(line, x.c0, used_of) < at ? 1 : 0;
    return x;
  };
  // (`of` neighbouring lanes share a row's parts, and whole warps call)
  auto normaliser = [&](const W& w, int hk, int r, const Parts& x, int sub, int of) -> float {
    const int j = by_group(p, r), head = hk * g + r - j * g;
    float lse;
    if (x.c0 == x.c1) {
      lse = __ldcg(p.lse + static_cast<int64_t>(w.o.first + j) * p.hkv * g + head);
    } else {
      const float* part = p.part + r % C::kRows;
      const float sink = p.sink != nullptr ? __ldcg(p.sink + head) * kLog2e : -INFINITY;
      float top = -INFINITY, sum = 0.f;
      for (int c = x.c0 + sub; c <= x.c1; c += 4 * of) {
        float v[4], most = top;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int at = c + k * of;
          v[k] = at <= x.c1 ? __ldcg(part + (static_cast<int64_t>(at) * 2 + (at == x.c0 ? x.second : 0)) * C::kRows) : -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) most = fmaxf(most, v[k]);
        if (most > -INFINITY) sum = top == -INFINITY ? sum : sum * ex2(top - most);      // 0, or no number, in front of the first
        top = most;
#pragma unroll
        for (int k = 0; k < 4; ++k) sum += v[k] == -INFINITY ? 0.f : ex2(v[k] - top);
      }
      for (int o = 1; o < of; o <<= 1) {
        const float t = __shfl_xor_sync(0xffffffffu, top, o), s = __shfl_xor_sync(0xffffffffu, sum, o), most = fmaxf(top, t);
        sum = (top == -INFINITY ? sum : sum * ex2(top - most)) + (t == -INFINITY ? s : s * ex2(t - most));
        top = most;
      }
      if (top == -INFINITY && sum == 0.f) {
        lse = -INFINITY;
      } else {
        const float most = fmaxf(top, sink);
        lse = most + lg2((top == -INFINITY ? sum : sum * ex2(top - most)) + (p.sink != nullptr ? ex2(sink - most) : 0.f));
      }
    }
    return lse == -INFINITY ? -INFINITY : -lse;       // nothing seen: no weights
  };
  // an item's block, by warps `me` of `all`, and in the second pass its rows' normalisers; true where a token's slot lies outside the cache
  auto load_block = [&](const W& w, const Item& it, int held, int me, int all) {
    bool bad = false;
    if constexpr (PASS == 3) {
      const Elem* head = static_cast<const Elem*>(p.k_cache) + it.hk * p.kv_head_stride;
      const int* rtt = p.ix.req_to_token + static_cast<int64_t>(w.o.row) * p.ix.table_stride;
      for (int row0 = me * 32; row0 < C::kRows; row0 += all * 32) {
        const int tok = it.block * C::kRows + row0 + lane;
        int s = tok < w.o.len ? __ldcg(rtt + tok) : -1;
        if (s < 0 || s >= p.num_slots) {
          bad = bad || tok < w.o.len;
          s = 0;
        }
        if (p.num_slots > 0) copy_keys(head, s, smem_u32(sBlock), row0, C::kBlock);
      }
    } else {
      const int rows = w.rows_of(it.block);
      copy_queries(w, it.hk, it.block * C::kRows, rows, smem_u32(sBlock), C::kBlock, row_mul[held], me, all);
      if (PASS == 2) {
        const Parts x = parts_of(it.at, w.steps1(p, it.block));
        const int of = all * 32 > C::kRows ? all * 32 / C::kRows : 1, log2_of = 31 - __clz(of);
        for (int row0 = me * 32 >> log2_of; row0 < rows; row0 += all * 32 >> log2_of) {
          const int row = row0 + (lane >> log2_of);
          const float v = normaliser(w, it.hk, it.block * C::kRows + min(row, rows - 1), x, lane & (of - 1), of);
          if (row < rows) neg_lse[held][row] = v;
        }
      }
    }
    cp_commit();
    cp_wait_all();
    fence_proxy_async_smem();
    if (bad) holes = 1;               // the computing warps look at every step
    __syncwarp();
    return bad;
  };

  if (warp >= kCompute) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
    if (warp == C::kWalkWarp) {
      // =============================== the run ===============================
      if (walks) {
        uint32_t count = 0;
        bool ok = true;
        auto put = [&]() {
          const uint32_t place = count % kItems;
          if (count >= kItems && !mbar_wait(&r_free[place], (count / kItems - 1) & 1, &fail_flag)) ok = false;
          if (!ok) return false;
          records[place].o = w.o;
          records[place].it = it;
          mbar_arrive(&r_full[place]);
          ++count;
          return true;
        };
        auto next_request = [&]() {
          do {
            if (++it.b >= p.ix.batch) return false;
            w.set(p, observed_of(p, it.b));
          } while (w.units == 0);
          return true;
        };
        auto walk = [&]() {
          if (!aligned || pos >= end) return;
          it.first = true;
          int t = 0;
          if (PASS != 2) {
            int all = w.steps_of(p, 0);
            while (rest >= all + kStart) {
              rest -= all + kStart;
              all = w.steps_of(p, ++it.block);
            }
            t = static_cast<int>(rest);
            while (true) {
              const int n = static_cast<int>(min(static_cast<int64_t>(all - t), end - pos));
              if (n > 0) {
                it.t0 = t;
                it.n = n;
                it.load = it.release = true;
                it.at = pos - t;
                it.at1 = at1 + it.hk * unit1;
                if (!put()) return;
                pos += n;
                t += n;
              }
              if (pos >= end) return;
              pos += all + kStart - t;
              if (pos >= end) return;
              it.first = false;
              t = 0;
              if (++it.block == w.units) {
                it.block = 0;
                if (++it.hk == p.hkv) {
                  it.hk = 0;
                  at1 += unit1 * p.hkv;
                  if (!next_request()) return;
                  if (PASS == 3) unit1 = w.cost1(p);
                }
              }
              all = w.steps_of(p, it.block);
            }
          } else {
            // the first step that begins at or behind the run's begin
            const int all = w.common(p);
            const int64_t level = static_cast<int64_t>(all) * w.blocks;
            if (rest <= level && level < (1ll << 31)) {
              t = w.blocks == 1 ? static_cast<int>(rest) : static_cast<int>((static_cast<uint32_t>(rest) + w.blocks - 1) / w.blocks);
              pos += static_cast<int64_t>(t) * w.blocks - rest;
            } else {
              const bool behind = rest > level;
              t = behind ? all : 0;
              int64_t x = behind ? level : 0;
              while (x < rest) x += w.blocks - w.first_block(p, t++);
              pos += x - rest;
            }
            int loaded = -1;        // the block whose queries are there
            while (pos < end) {
              const int steps = w.steps();
              if (t >= steps) {
                t = 0;
                loaded = -1;
                if (++it.hk == p.hkv) {
                  it.hk = 0;
                  at1 += unit1 * p.hkv;
                  if (!next_request()) return;
                  unit1 = w.cost1(p);
                }
                continue;
              }
              int n = 0;
              while (n < kChunk && t + n < steps && pos < end) pos += w.blocks - w.first_block(p, t + n++);
              it.t0 = t;
              it.chunk = n;
              it.block = w.first_block(p, t);
              int64_t off = 0;
              for (int i = 0; i < it.block; ++i) off += w.steps1(p, i) + kStart;
              for (; it.block < w.blocks; ++it.block) {
                const int mine = w.steps1(p, it.block);
                it.n = min(n, mine - t);
                it.load = loaded != it.block;
                it.flush = it.block == w.blocks - 1;
                it.release = !it.flush || t + n >= steps || pos >= end || w.first_block(p, t + n) != it.block;
                it.at = at1 + it.hk * unit1 + off;
                loaded = it.block;
                if (!put()) return;
                off += mine + kStart;
              }
              t += n;
            }
          }
        };
        walk();
        it.n = 0;
        if (ok) put();
        if (!ok) fail_flag = 1;
      }
    } else if (warp < C::kWalkWarp) {
      // =============================== stages ===============================
      constexpr int kWarps = C::kCopying;
      const int me = warp - kCompute;
      bool bad = false, ok = true;
      uint32_t stage0 = 0;                               // stages of the items before
      // A stage may be on its way while the one before is waited for, unless its place waits for that one's products.  None outlives its item:
      // the next record may wait for this item's scores, and those wait for every stage.
      constexpr bool kTwo = !KV8 && kStages > kWarps;
      int pending = -1;                                  // the place of a stage that has not been waited for
      auto arrived = [&](int place) {
        fence_proxy_async_smem();
        if (bad) holes = 1;               // the computing warps look at every step
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[place]);
      };
      if (me < kWarps) items(false, [&](const W& w, const Item& it) {
        const int stages = it.n * KT;
        int i = (me + kWarps - static_cast<int>(stage0 % kWarps)) % kWarps;
        auto wait_free = [&](uint32_t n) {       // asleep in between: warps that poll take issue slots from the computing ones
          if (n >= kStages && !mbar_wait_relaxed(&empty[n % kStages], (n / kStages - 1) & 1, 20)) ok = false;
          return ok = __all_sync(0xffffffffu, ok);
        };
        if constexpr (PASS == 3) {
          const int tile0 = w.first_tile(p, it.block) + it.t0;
          // the block of the first pass that a tile of rows lies in, and where it begins on that line
          int block = tile0 * kTileRows / C::kRows;
          int64_t at = it.at1;
          for (int b = 0; b < block; ++b) at += w.steps1(p, b) + kStart;
          for (; i < stages; i += kWarps) {
            const uint32_t n = stage0 + i;
            if (!wait_free(n)) return false;
            const int r0 = (tile0 + i) * kTileRows, rows = min(kTileRows, w.rows - r0);
            for (; (block + 1) * C::kRows <= r0; ++block) at += w.steps1(p, block) + kStart;
            const uint32_t held = n % kRing;
            copy_queries(w, it.hk, r0, rows, smem_u32(ring) + n % kStages * C::kStage, C::kPiece, row_mul[held], 0, 1);
            cp_commit();
            const Parts x = parts_of(at, w.steps1(p, block));
            for (int row = lane; row < kTileRows; row += 32) neg_lse[held][row] = normaliser(w, it.hk, r0 + min(row, rows - 1), x, 0, 1);
            cp_wait_all();
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&full[n % kStages]);
              mbar_arrive(&l_full[held]);
            }
          }
        } else {
          const int* rtt = p.ix.req_to_token + static_cast<int64_t>(w.o.row) * p.ix.table_stride;
          const int base = it.t0 * C::kStepKeys;
          const Elem* head = static_cast<const Elem*>(p.k_cache) + it.hk * p.kv_head_stride;
          int next[4];          // slots of a stage's tokens lane, lane + 32, ..
          auto look = [&](int i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int tok = base + i * 128 + k * 32 + lane;
              next[k] = i < stages && tok < w.o.len ? max(__ldcg(rtt + tok), -1) : kNoToken;      // no number of the table is taken for kNoToken
            }
          };
          look(i);
          for (; i < stages; i += kWarps) {
            const uint32_t n = stage0 + i, stage = smem_u32(ring) + n % kStages * C::kStage;
            int s[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              s[k] = next[k];
              if (s[k] < 0 || s[k] >= p.num_slots) {
                bad = bad || s[k] != kNoToken;
                s[k] = 0;
              }
            }
            look(i + kWarps);
            if (!wait_free(n)) return false;
#pragma unroll 1
            for (int k = 0; k < 4 && p.num_slots > 0; ++k) {
              copy_keys(head, s[0], stage, k * 32, C::kPiece);
              s[0] = s[1];
              s[1] = s[2];
              s[2] = s[3];
            }
            cp_commit();
            if (kTwo) {
              if (pending >= 0) {
                cp_wait_one();
                arrived(pending);
              }
              pending = n % kStages;
            } else {
              cp_wait_all();
              arrived(n % kStages);
            }
          }
          if (pending >= 0) {
            cp_wait_all();
            arrived(pending);
            pending = -1;
          }
        }
        stage0 += stages;
        return true;
      });
      cp_wait_all();
      if (pending >= 0) arrived(pending);       // of an item that was given up
      if (!ok) fail_flag = 1;
      if (bad && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
    } else if (warp == C::kBlockWarp) {
      // =============================== blocks behind the first ===============================
      bool bad = false, ok = true;
      uint32_t loads = 0;
      items(false, [&](const W& w, const Item& it) {
        if (!it.load) return true;
        if (loads > 0) {
          if (!mbar_wait_relaxed(b_free, (loads - 1) & 1)) ok = false;
          if (!(ok = __all_sync(0xffffffffu, ok))) return false;
          bad = load_block(w, it, loads % kRing, 0, 1) || bad;
          if (lane == 0) {
            mbar_arrive(b_full);
            if (PASS != 3) mbar_arrive(&l_full[loads % kRing]);
          }
        }
        ++loads;
        return true;
      });
      if (!ok) fail_flag = 1;
      if (bad && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
    } else if (elect_one()) {
      // =============================== products ===============================
      bool ok = true;
      const uint64_t b_desc = umma_desc_k_sw128(smem_u32(sBlock)), r_desc0 = umma_desc_k_sw128(smem_u32(ring));
      const uint32_t fmt = KV8 || std::is_same<T, __half>::value ? 0u : 1u;
      uint32_t stage = 0, step = 0, loads = 0;
      items(true, [&](const W& w, const Item& it) {
        if (it.load) {
          if (ok && !mbar_wait(loads == 0 ? b_first : b_full, loads == 0 ? 0 : (loads - 1) & 1, &fail_flag)) ok = false;
          ++loads;
        }
        // lanes are the block's rows, a tile at a time, over the stage's 128; in the second pass the stage's over the block's
        const int rows = PASS == 3 ? min(C::kRows, w.o.len - it.block * C::kRows) : w.rows_of(it.block);
        const uint32_t idesc = umma_idesc(128, PASS == 2 ? (rows + 15) / 16 * 16 : 128, 1, fmt, fmt, 0, 0);
        for (int t = 0; t < it.n && ok; ++t, ++step) {
          const uint32_t buf = step & 1;
          if (step >= 2 && !mbar_wait(&s_free[buf], ((step >> 1) - 1) & 1, &fail_flag)) ok = false;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt, ++stage) {
            const uint32_t st = stage % kStages;
            if (ok && !mbar_wait(&full[st], (stage / kStages) & 1, &fail_flag)) ok = false;
            if (!ok) break;
            fence_proxy_async_smem();       // copies were made in the generic proxy
            tc_fence_after_sync();
            const uint64_t r_desc = r_desc0 + st * (C::kStage >> 4);
            const uint32_t to = tmem + buf * C::kCols + kt * 128;
#pragma unroll
            for (int h = 0; h < (PASS == 2 ? 1 : C::RT); ++h) {
              if (h * kTileRows >= rows) break;
#pragma unroll
              for (int kk = 0; kk < 4 * NH; ++kk) {
                const uint64_t b = b_desc + (kk >> 2) * (C::kBlock >> 4) + h * (kTileRows * 128 >> 4) + (kk & 3) * 2;
                const uint64_t r = r_desc + (kk >> 2) * (C::kPiece >> 4) + (kk & 3) * 2;
                umma_f16(to + h * 128, PASS == 2 ? r : b, PASS == 2 ? b : r, idesc, kk > 0 ? 1u : 0u);
              }
            }
            umma_commit(&empty[st]);
          }
          if (!ok) break;
          umma_commit(&s_full[buf]);
        }
        if (ok && it.release) umma_commit(b_free);
        return ok;
      });
      if (!ok) fail_flag = 1;
    }
  } else {
    // =============================== scores ===============================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kComputeRegs));
    const int quarter = warp >> 2, in_tile = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const bool capped = p.cap_post > 0.f;
    constexpr int kWarpCols = C::kWarpCols;
    bool ok = true, bad = false;
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
    // A quarter's columns of this step, 32 at a time; behind the last the buffer is free.  use(first column, scores).  Steps without masks and
    // caps have a loop of their own: with the code for the others in between a step takes a third longer.
    auto columns = [&](int count, auto&& use) {
      const uint32_t from = tmem + lanes + (step & 1) * C::kCols + quarter * kWarpCols;
      auto some = [&](int c) {
        uint32_t raw[32];
        if (c < count) {
          tmem_ld_32x32(from + c, raw);
          tmem_ld_wait();
        }
        if (c + 32 == kWarpCols) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[step & 1]);
        }
        if (c < count) use(c, raw);
      };
#pragma unroll
      for (int c = 0; c < kWarpCols; c += 32) some(c);
    };
    auto total = [&](const float (&sums)[4]) { return (sums[0] + sums[1]) + (sums[2] + sums[3]); };
    auto gaps = [&]() { return *const_cast<const volatile int*>(&holes) != 0; };
    auto slot_inside = [&](const W& w, int token) {
      const int s = token < w.o.len ? __ldcg(p.ix.req_to_token + static_cast<int64_t>(w.o.row) * p.ix.table_stride + token) : -1;
      return s >= 0 && s < p.num_slots;
    };
    // cap tanh(x / cap), in the log2 domain.  (1 - 2 / (1 + e^(2 y)) is quicker, but near 0 it keeps a score to 2^-24 of the cap only: one request of
    // 32000 tokens behind its last 64, 195 us and 164; without a cap 98.)
    auto cap = [&](uint32_t x, float mul) { return __float_as_uint(p.cap_post * tanhf(__uint_as_float(x) * mul * p.cap_pre)); };
    // What a token gets of 32 rows; where masks or caps are, of those from `low` up to `high`
    auto weights = [&](auto plain, uint32_t (&raw)[32], const float* neg, const float* muls, int low, int high, float (&sums)[4]) {
      constexpr bool kPlain = decltype(plain)::value;
      if (!kPlain && capped) {
#pragma unroll
        for (int c = 0; c < 32; ++c) raw[c] = cap(raw[c], kScaled ? muls[c] : p.scale_log2);
      }
      const float same = !kPlain && capped ? 1.f : p.scale_log2;
      if (!kPlain) {
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float e = ex2(fmaf(__uint_as_float(raw[c]), kScaled && !capped ? muls[c] : same, neg[c]));
          sum += c >= low && c < high ? e : 0.f;
        }
        sums[0] += sum;
        return;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 n4 = *reinterpret_cast<const float4*>(neg + 4 * i);
        float4 m4 = make_float4(same, same, same, same);
        if (kScaled) m4 = *reinterpret_cast<const float4*>(muls + 4 * i);
        sums[0] += ex2(fmaf(__uint_as_float(raw[4 * i]), m4.x, n4.x));
        sums[1] += ex2(fmaf(__uint_as_float(raw[4 * i + 1]), m4.y, n4.y));
        sums[2] += ex2(fmaf(__uint_as_float(raw[4 * i + 2]), m4.z, n4.z));
        sums[3] += ex2(fmaf(__uint_as_float(raw[4 * i + 3]), m4.w, n4.w));
      }
    };

    items(false, [&](const W& w, const Item& it) {
      const int least = w.least();
      if (it.load) {
        const int held = loads % kRing;
        if (loads == 0) {
          bad = load_block(w, it, 0, warp, kCompute);
          if (lane == 0) mbar_arrive(b_first);
          if ((PASS == 2 || (PASS == 1 && kScaled)) && !mbar_wait(b_first, 0, &fail_flag)) ok = false;
        } else if (PASS == 2 || (PASS == 1 && kScaled)) {
          // (the first block's place was not written by the warp that arrives here)
          if (!mbar_wait(&l_full[held], (held == 0 ? loads / kRing - 1 : loads / kRing) & 1, &fail_flag)) ok = false;
        }
        if (!(ok = __all_sync(0xffffffffu, ok))) return false;
        ++loads;
      }
      const int held = (loads - 1) % kRing;
      if constexpr (PASS == 1) {
        const int rows = w.rows_of(it.block), row0 = it.block * C::kRows;
        const int row = (C::RT == 2 ? (quarter >> 1) * 128 : 0) + in_tile, col0 = quarter * kWarpCols % C::kStepKeys;
        const bool valid = row < rows, any = __any_sync(0xffffffffu, valid);
        const int place = least + by_group(p, row0 + min(row, rows - 1)), sure = least + by_group(p, row0);       // sure: what all rows of the block see
        float mul = p.scale_log2;
        if constexpr (kScaled)
          if (valid) mul = row_mul[held][row];
        float m = -INFINITY;
        float sums[4] = {0.f, 0.f, 0.f, 0.f};
        for (int t = 0; t < it.n; ++t, ++step) {
          if (!wait_scores()) return false;
          const int key0 = (it.t0 + t) * C::kStepKeys + col0;
          const bool rare = gaps(), plain = key0 + kWarpCols - 1 <= sure && !rare && !capped;
          auto add_up = [&](auto tag, int col, uint32_t (&raw)[32]) {
            constexpr bool kPlain = decltype(tag)::value;
            const int key = key0 + col;
            const float by = !kPlain && capped ? 1.f : mul;
            if (!kPlain && capped) {
#pragma unroll
              for (int c = 0; c < 32; ++c) raw[c] = cap(raw[c], mul);
            }
            if (!kPlain) {
              const int seen = place + 1 - key;          // columns in front
              uint32_t there = seen >= 32 ? 0xffffffffu : seen > 0 ? (1u << seen) - 1 : 0u;
              if (__any_sync(0xffffffffu, rare)) there &= __ballot_sync(0xffffffffu, slot_inside(w, key + lane));        // tokens whose slots lie outside the cache
#pragma unroll
              for (int c = 0; c < 32; ++c) raw[c] = (there >> c) & 1 ? raw[c] : __float_as_uint(-INFINITY);
            }
            // The maximum of the first scores serves until a sum gets large: fp32 has the range.  (A sum that is no number raises it every time.)
            bool raise = m == -INFINITY, raised = false;
            while (true) {
              if (raise) {
                float mx[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) mx[i] = fmaxf(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1]));
#pragma unroll
                for (int c = 8; c < 32; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], __uint_as_float(raw[c]), __uint_as_float(raw[c + 1]));
                const float top = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * by, m);
                const float f = m == -INFINITY ? 1.f : ex2(m - top);      // 0, or no number, in front of the first
#pragma unroll
                for (int i = 0; i < 4; ++i) sums[i] *= f;
                m = top;
                raised = true;
              }
              const float neg = m == -INFINITY ? 0.f : -m;
              float now[4] = {sums[0], sums[1], sums[2], sums[3]};
#pragma unroll
              for (int c = 0; c < 32; ++c) now[c & 3] += ex2(fmaf(__uint_as_float(raw[c]), by, neg));
              raise = !raised && !(total(now) < kLargest);
              if (raise) continue;
#pragma unroll
              for (int i = 0; i < 4; ++i) sums[i] = now[i];
              break;
            }
          };
          columns(any ? kWarpCols : 0, [&](int col, uint32_t (&raw)[32]) {
            if (__builtin_expect(plain, 1)) {
              add_up(std::true_type(), col, raw);
            } else {
              add_up(std::false_type(), col, raw);
            }
          });
        }
        // ---- the quarters' maxima and sums meet ----
        float2* parts = reinterpret_cast<float2*>(cells) + (turn++ & 1) * 512;
        parts[quarter * 128 + in_tile] = make_float2(m, total(sums));
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
          for (int i = 0; i < kParts; ++i) sum += x[i].x == -INFINITY ? x[i].y : x[i].y * ex2(x[i].x - top);       // no score: 0, or no number
          float lse = none && sum == 0.f ? -INFINITY : top + lg2(sum);
          if (it.t0 == 0 && it.n == w.steps1(p, it.block)) {
            const int j = by_group(p, row0 + tid), head = it.hk * g + row0 + tid - j * g;
            if (p.sink != nullptr && lse != -INFINITY) {
              const float sink = __ldcg(p.sink + head) * kLog2e, at = fmaxf(top, sink);
              lse = at + lg2(sum * ex2(top - at) + ex2(sink - at));
            }
            p.lse[static_cast<int64_t>(w.o.first + j) * p.hkv * g + head] = lse;
          } else {
            p.part[(static_cast<int64_t>(blockIdx.x) * 2 + (it.first ? 0 : 1)) * C::kRows + tid] = lse;
          }
        }
      } else if constexpr (PASS == 2) {
        const int rows = w.rows_of(it.block), row0 = it.block * C::kRows;
        const int kt = C::RT == 1 && KT == 2 ? quarter >> 1 : 0, group = KT == 2 ? quarter & 1 : quarter;       // stage and part of the columns
        const int col0 = group * kWarpCols, chunk_keys = it.chunk * C::kStepKeys;
        const float* neg = neg_lse[held] + col0;
        const float* muls = row_mul[held] + (kScaled ? col0 : 0);
        for (int t = 0; t < it.n; ++t, ++step) {
          const int token = (it.t0 + t) * C::kStepKeys + kt * 128 + in_tile;
          // this token is seen by the block's rows from `low` on
          const int low = token > least ? static_cast<int>(min(static_cast<int64_t>(token - least) * g - row0, static_cast<int64_t>(C::kRows))) : 0;
          // all rows see all of the step's tokens, and this warp's columns are rows
          const bool plain = (it.t0 + t + 1) * C::kStepKeys - 1 <= least && (col0 >= rows || col0 + kWarpCols <= rows) && !capped;
          float sums[4] = {0.f, 0.f, 0.f, 0.f};
          if (!wait_scores()) return false;
          columns(rows - col0, [&](int at, uint32_t (&raw)[32]) {
            if (__builtin_expect(plain, 1)) {
              weights(std::true_type(), raw, neg + at, muls + (kScaled ? at : 0), 0, 32, sums);
            } else {
              weights(std::false_type(), raw, neg + at, muls + (kScaled ? at : 0), low - col0 - at, rows - col0 - at, sums);
            }
          });
          float sum = total(sums);
          if (gaps() && !slot_inside(w, token)) sum = 0.f;       // rare: a token whose slot lies outside the cache is not seen
          float* cell = cells + group * chunk_keys + t * C::kStepKeys + kt * 128 + in_tile;
          *cell = it.block == 0 || w.first_block(p, it.t0 + t) == it.block ? sum : *cell + sum;
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
      } else {
        const int tile = C::RT == 2 ? quarter >> 1 : 0, col0 = quarter * kWarpCols % 128;
        const int token = it.block * C::kRows + tile * 128 + in_tile, tile0 = w.first_tile(p, it.block) + it.t0;
        const bool any = __any_sync(0xffffffffu, token < w.o.len);
        float all = 0.f;
        for (int t = 0; t < it.n; ++t, ++step) {
          const uint32_t place = step % kRing;
          if (!mbar_wait(&l_full[place], (step / kRing) & 1, &fail_flag)) ok = false;
          if (!wait_scores()) return false;
          const int r0 = (tile0 + t) * kTileRows + col0, rows = w.rows - r0;
          // this token is seen by the rows from `low` on
          const int low = token > least ? static_cast<int>(min(static_cast<int64_t>(token - least) * g - r0, static_cast<int64_t>(128))) : 0;
          // all of the stage's rows see all of the block's tokens
          const bool plain = static_cast<int64_t>((it.block + 1) * C::kRows - 1 - least) * g <= (tile0 + t) * kTileRows && (rows <= 0 || rows >= kWarpCols) && !capped;
          float sums[4] = {0.f, 0.f, 0.f, 0.f};
          const float* neg = neg_lse[place] + col0;
          const float* muls = row_mul[place] + (kScaled ? col0 : 0);
          columns(any ? rows : 0, [&](int at, uint32_t (&raw)[32]) {
            if (__builtin_expect(plain, 1)) {
              weights(std::true_type(), raw, neg + at, muls + (kScaled ? at : 0), 0, 32, sums);
            } else {
              weights(std::false_type(), raw, neg + at, muls + (kScaled ? at : 0), low - at, rows - at, sums);
            }
          });
          all += total(sums);
        }
        if (gaps() && !slot_inside(w, token)) all = 0.f;       // rare: a token whose slot lies outside the cache is not seen
        float* parts = cells + (turn++ & 1) * 512;
        parts[quarter * 128 + in_tile] = all;
        if (!meet()) return false;
        constexpr int kParts = C::RT == 2 ? 2 : 4;
        const int steps = w.steps_of(p, it.block), at = it.block * C::kRows + tid;
        const bool whole = it.t0 == 0 && it.n == steps;
        if (tid < C::kRows && at < w.o.len) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < kParts; ++i) sum += parts[((tid >> 7) * kParts + i) * 128 + (tid & 127)];
          if (whole) {
            float* to = p.sums.data + w.o.row * p.sums.row_stride + it.hk * p.sums.head_stride + at;
            *to = p.add && at < w.o.prefix ? __ldcg(to) + sum : sum;
          } else {
            p.part_sum[(static_cast<int64_t>(blockIdx.x) * 2 + (it.first ? 0 : 1)) * C::kRows + tid] = sum;
          }
        }
        // the unit's last step: it began in front of this run
        if (tid == 0 && !whole && it.t0 + it.n == steps) {
          const int64_t line = line_of[1];
          const int used = used_ctas(p, line), c0 = owner_of(line, it.at, used);
          p.jobs[blockIdx.x] = make_int4(it.b, it.hk, it.block, c0 * 2 + (run_begin(line, c0, used) < it.at ? 1 : 0));
        }
      }
      return true;
    });
    if (!ok) fail_flag = 1;
    if (bad && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
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

// Adds up the parts of blocks of tokens that were cut, in the order of the CTAs; a block per CTA of the kernel above, whose note says what
// ends there (request -1: nothing).
__global__ void __launch_bounds__(256) prompt_parts_kernel(const PromptParams p, int block_rows) {
  pdl_wait_loads();
  pdl_launch_dependents();
  const int4 job = __ldcg(p.jobs + blockIdx.x);
  if (job.x < 0) return;
  const Observed o = observed_of(p, job.x);
  const int token = job.z * block_rows + threadIdx.x;
  if (static_cast<int>(threadIdx.x) >= block_rows || token >= o.len) return;
  float sum = __ldcg(p.part_sum + static_cast<int64_t>(job.w) * block_rows + threadIdx.x);
#pragma unroll 4
  for (int c = job.w / 2 + 1; c <= static_cast<int>(blockIdx.x); ++c) sum += __ldcg(p.part_sum + static_cast<int64_t>(c) * 2 * block_rows + threadIdx.x);
  float* to = p.sums.data + o.row * p.sums.row_stride + job.y * p.sums.head_stride + token;
  *to = p.add && token < o.prefix ? __ldcg(to) + sum : sum;
}

template <typename T, int NH, int FMT, int R, int PASS>
int launch_pass(const PromptParams& p, cudaStream_t s) {
  using C = Cfg<NH, FMT != kKvSame, R, PASS>;
  auto kern = weights_prompt_kernel<T, NH, FMT, R, PASS>;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kern), C::kSmem) != cudaSuccess) return -3;
  // the computing warps take registers that the others give back: together no more than the kernel is launched with
  static const int regs = [kern] {
    cudaFuncAttributes at{};
    return cudaFuncGetAttributes(&at, reinterpret_cast<const void*>(kern)) == cudaSuccess ? at.numRegs : 0;
  }();
  if (regs < C::kLaunchRegs) return -5;
  const cudaError_t err = launch_pdl(kern, dim3(p.ctas), dim3(C::kThreads), C::kSmem, s, p);
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}
template <typename T, int NH, int FMT, int R>
int launch_one(const PromptParams& p, bool rows_go_by, cudaStream_t s) {
  int rc = launch_pass<T, NH, FMT, R, 1>(p, s);
  if (rc != 0) return rc;
  if constexpr (R == 2 || NH == 4) {
    if (rows_go_by) {
      rc = launch_pass<T, NH, FMT, R, 3>(p, s);
      if (rc != 0) return rc;
      const cudaError_t err = launch_pdl(prompt_parts_kernel, dim3(p.ctas), dim3(256), 0, s, p, R * kTileRows);
      note_launch();
      return err == cudaSuccess ? 0 : -4;
    }
  }
  return launch_pass<T, NH, FMT, R, 2>(p, s);
}
template <typename T, int NH, int R>
int launch_format(const PromptParams& p, int fmt, bool rows_go_by, cudaStream_t s) {
  switch (fmt) {
    case kKvSame: return launch_one<T, NH, kKvSame, R>(p, rows_go_by, s);
    case kKvE4M3: return launch_one<T, NH, kKvE4M3, R>(p, rows_go_by, s);
    default: return launch_one<T, NH, kKvE5M2, R>(p, rows_go_by, s);
  }
}
template <typename T>
int launch_type(const PromptParams& p, int head_dim, int fmt, int tiles, bool rows_go_by, cudaStream_t s) {
  switch (head_dim) {
    case 64: return tiles == 2 ? launch_format<T, 1, 2>(p, fmt, rows_go_by, s) : launch_format<T, 1, 1>(p, fmt, rows_go_by, s);
    case 128: return tiles == 2 ? launch_format<T, 2, 2>(p, fmt, rows_go_by, s) : launch_format<T, 2, 1>(p, fmt, rows_go_by, s);
    default: return launch_format<T, 4, 1>(p, fmt, rows_go_by, s);
  }
}

// observed rows of a request and kv head, on average over the batch
int64_t rows_each(const WeightsPromptArgs& a) {
  const int64_t each = a.rows / std::max(1, a.index.batch);
  return (a.last > 0 ? std::min<int64_t>(a.last, each) : each) * (a.hq / a.hkv);
}
// Row tiles of a block: two where a request has more observed rows than one tile holds; 256 features leave no room for two.
int row_tiles(const WeightsPromptArgs& a) { return a.head_dim <= 128 && rows_each(a) > kTileRows ? 2 : 1; }

template <typename T>
int launch_prompt(const WeightsPromptArgs& a, cudaStream_t s) {
  PromptParams p{};
  p.ix = a.index;
  p.sums = a.sums;
  p.prefix_lens = a.prefix_lens;
  p.q_start = a.q_start;
  p.q = a.q;
  p.k_cache = a.k_cache;
  p.ctas = a.num_sms;
  p.jobs = reinterpret_cast<int4*>(a.workspace);       // on a 16-byte boundary
  p.lse = a.workspace + 4 * p.ctas;
  p.part = p.lse + a.rows * a.hq;
  p.part_sum = p.part + static_cast<int64_t>(p.ctas) * 2 * row_tiles(a) * kTileRows;
  p.sink = a.sink;
  p.q_stride = a.q_stride;
  p.num_slots = a.num_slots;
  p.kv_tok_stride = a.kv_tok_stride;
  p.kv_head_stride = a.kv_head_stride;
  p.rows = static_cast<int>(a.rows);
  p.hkv = a.hkv;
  p.group = a.hq / a.hkv;
  p.last = a.last;
  p.inv_group = (65536 + p.group - 1) / p.group;
  p.inv_group32 = static_cast<uint32_t>(p.group == 1 ? 0xffffffffull : (1ull << 32) / p.group);
  p.add = a.add;
  p.scale_log2 = a.scale * kLog2e;
  if (a.logit_cap > 0.f) {      // the scores are scaled before the cap
    p.scale_log2 = a.scale;
    p.cap_pre = 1.f / a.logit_cap;
    p.cap_post = a.logit_cap * kLog2e;
  }
  const int tiles = row_tiles(a);
  return launch_type<T>(p, a.head_dim, a.kv_fmt, tiles, rows_each(a) > 2 * tiles * kTileRows, s);
}

}  // namespace

}  // namespace mb200
