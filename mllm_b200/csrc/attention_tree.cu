// Attention of drafted token trees over the slot-indexed KV pool: head sizes 64, 128 and 256, caches of the activation type or 8-bit
// floats.
//
// Request b has prefix cached tokens and a tree of n nodes whose keys and values stand behind them (node j at slot
// table[prefix + j]); node j continues node parents[j] < j, or the cached text where that is -1.  It sits at position
// prefix + (its ancestors) and sees the cached tokens, its ancestors and itself:
//   o_j = sum_k softmax_k(scale q_j . k_k) v_k      over  {cached k, k >= low_j}  and  {ancestors and self at positions >= low_j},
// low_j the first position of the sliding window or of the chunk.
//
// The rows that share K and V are (node, query head of the group) pairs, n * group of them; 128 make a row tile.  Every cached key
// and value is read once per unit of one or two row tiles and meets 4 * 128 operations per element and tile: a memory stream up to 128
// rows, like decoding, with products too large for warp-level instructions (128 rows x 64 keys x 128 features twice per 32 KB).  So:
//   * work is dealt as in decoding: the 64-token tiles of all (request, kv head, rows) units form one line, laid out on the device
//     from the lengths, and every CTA takes an equal run of it.  A unit inside one CTA is written out directly; others leave at most
//     two partial results per CTA, and the CTA that has a unit's last tile leaves a note for the kernel that joins them.
//   * copying warps (4-10; 8-18 beside two row tiles) bring rows by slot with cp.async (a page of one token costs what a page of 16 does)
//     into a ring of 64-token K or V stages in the operand layout.  A warp takes whole stages in turn: what stands between two stages
//     (barriers, slots, shuffles) is a chain of some 2000 cycles, which all warps paid for every stage when they shared it.  8-bit rows
//     land as they are, and the two warps that copied them widen them.  The warps left copy Q.
//   * the last warp issues S = Q K^T (two score buffers a row tile in tensor memory) and O += P V, P from tensor memory.
//   * the first four warps (eight) hold a row per thread: online maximum and sum in fp32, P over S in place.  Masks are 64-bit words per
//     row and tile, made only in tiles that hold tree nodes or a window's edge: cached part by comparison, tree part by a walk to the
//     root over parents in shared memory.
// A token whose slot lies outside the cache is nowhere visible; a row that sees no token at all is zero.
// A value that is no number must not reach rows that do not see it (0 x NaN): in masked tiles the warps that copied V set such elements to
// zero, and they are added at the end to the rows that see them.
//
// Where the time goes (bf16, 128 features, on the device in a graph): 8 requests of 2048 tokens and 32 nodes, 72 MB, 34.6 us.  The first
// scores are there after 9 us (1.8 us for the lengths of all requests, 2 us for the slots, then the rows, all stages' at once), tiles pass
// at the rate of memory (6 TB/s), rows go out in 2 us, and the joining kernel begins 2 us behind the last CTA and takes 4.  From two
// row tiles on the softmax warps bound: 1.2 us for 256 rows and 64 keys on an SM, a chain of wait, load, maximum, exponentials and store
// with two warps a scheduler to hide it (a quarter of the exponentials by polynomial instead: 58.7 -> 63.6 us).
#include <algorithm>

#include "common.cuh"
#include "tree.cuh"

namespace mb200 {
namespace {

constexpr int kRows = 128;                 // MMA M
constexpr int kTile = 64;                  // tokens of a tile
constexpr int kStart = 4;                  // tiles' time that every unit costs beside its tiles
constexpr int kNoToken = -0x7fffffff;
constexpr int kParents = 256;              // nodes whose parents are kept in shared memory
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleThreshold = 8.0f;  // the running maximum is raised when a score passes it by 2^8

struct TreeParams {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  void* out;
  float* part_o;     // [CTAs][2][HD / 4][part_rows][4]: lanes, which hold rows, write and read neighbouring addresses
  float* part_lse;   // [CTAs][2][part_rows]
  int* job_rows;     // [CTAs]: rows to join (0: none) of the unit whose last tile the CTA has
  int4* jobs;        // [CTAs]: first row of q, first head, first CTA of the unit, whether that one has it in its second partial result
  TreeIndex ix;
  const float* sink;
  int64_t q_stride, out_stride, num_slots, kv_tok_stride, kv_head_stride;
  int hkv, group, tpt, unit_nodes, ctas, part_rows, window, chunk;   // tpt: nodes of a row tile
  float scale_log2, cap_in, cap_out;    // cap_out 0: no soft cap
  uint32_t idesc_s, idesc_o;
};
constexpr int kJobInts = 5;

// first position that a node at position i sees
__device__ __forceinline__ int first_key(const TreeParams& p, int i) {
  if (p.window > 0) return max(0, i - p.window + 1);
  return p.chunk > 0 ? i / p.chunk * p.chunk : 0;
}
// first token that is copied: the first key of the least deep position
__device__ __forceinline__ int first_token(const TreeParams& p, const Request& r) { return first_key(p, r.prefix) & ~(kTile - 1); }
// Tokens below hold keys that some node of the request may not see for the window's or the chunk's sake.
__device__ __forceinline__ int edge_of(const TreeParams& p, const Request& r) { return first_key(p, r.prefix + r.nodes - 1); }
__device__ __forceinline__ int tiles_of(const TreeParams& p, const Request& r) {
  return r.nodes == 0 ? 0 : (r.prefix + r.nodes - first_token(p, r) + kTile - 1) / kTile;
}
__device__ __forceinline__ int units_of(const TreeParams& p, const Request& r) { return (r.nodes + p.unit_nodes - 1) / p.unit_nodes; }

__device__ __forceinline__ int ctas_used(const TreeParams& p, int64_t line) {
  const int64_t want = max(line / 4, min(line / 2, static_cast<int64_t>(64)));
  return static_cast<int>(min(static_cast<int64_t>(p.ctas), max(want, static_cast<int64_t>(1))));
}
// (A division of 64 bits takes some 500 cycles.)
__device__ __forceinline__ bool fits_32(int64_t line, int ctas) { return line < (1ll << 31) && line * (ctas + 1) < (1ll << 32); }
__device__ __forceinline__ int64_t run_begin(int64_t line, int c, int ctas) {
  if (fits_32(line, ctas)) return static_cast<uint32_t>(line) * static_cast<uint32_t>(c) / static_cast<uint32_t>(ctas);
  return line * c / ctas;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  const int sz = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(sz) : "memory");
}
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
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16x2(a, b);
  }
}
// offset of 16-byte piece `ch` of row `row` in a tile of 64-feature blocks of `block` bytes, rows of 128 bytes, 128-byte swizzle
__device__ __forceinline__ uint32_t swz(int row, int ch, int block) {
  return (ch >> 3) * block + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
}

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// R: row tiles that a CTA takes through its keys and values side by side
template <int NH, bool KV8, int R>
struct Cfg {
  static_assert(R == 1 || NH == 2, "two row tiles of 256 features leave no tensor memory for scores; those of 64 lose more below 1.5 tiles than they win");
  static constexpr int kSoftmaxWarps = 4 * R, kIssueWarp = R == 1 ? 11 : 19, kThreads = 32 * (kIssueWarp + 1);
  static constexpr int kD = 64 * NH;
  static constexpr int kQBlock = kRows * 128;              // a 64-feature block of Q
  static constexpr int kQTile = NH * kQBlock, kQBytes = R * kQTile;
  static constexpr int kBlock = kTile * 128;               // a 64-feature block of a stage
  static constexpr int kStage = NH * kBlock;
  static constexpr int kStages = (NH == 1 ? (KV8 ? 6 : 10) : KV8 ? 3 : 5) * R;
  // A team of warps copies every kTeams-th item.  Never more teams than stages: a team that waits for the item kStages before its own
  // to be used has seen its item before go to the stage of the one 2 kStages before (a barrier tells a phase from the next, no more).
  static constexpr int kTeam = KV8 ? 2 : 1, kTeams = R == 1 ? (KV8 ? 3 : 5) : KV8 ? 4 : 8;
  static constexpr int kQWarps = kIssueWarp - kSoftmaxWarps - kTeam * kTeams;     // those that are left copy Q
  static_assert(kTeams <= kStages && kQWarps > 0, "teams");
  static constexpr int kRaw = KV8 ? kTile * kD : 0;        // an item as it is cached, one per team
  static constexpr int kSmem = kQBytes + kStages * kStage + kTeams * kRaw;
  static constexpr int kPerSm = NH == 4 || R == 2 ? 1 : 2;
  // registers that a CTA is launched with, those of the threads that hold rows, and what the others keep; 256 features have one CTA and need no split
  static constexpr bool kSplit = NH < 4;
  static constexpr int kLaunchRegs = R == 1 ? 80 : 96, kSoftmaxRegs = 128, kOtherRegs = R == 1 ? 56 : 72;
  static_assert(32 * (kSoftmaxWarps * kSoftmaxRegs + (kThreads / 32 - kSoftmaxWarps) * kOtherRegs) <= kThreads * kLaunchRegs, "register split");
  static_assert(kPerSm * (kSmem + 2048) <= 228 * 1024, "1 KB of each CTA is the system's, 1 KB the kernel's variables");
  // tensor memory: two score buffers of 64 columns a row tile, then O of each
  static constexpr int kScoreCols = R * 2 * kTile, kCols = NH == 4 || R == 2 ? 512 : 256;
  static_assert(kScoreCols + R * kD <= kCols, "tensor memory");
};

// Item i of a segment of n tiles, in the order in which the products need them: K0, K1, V0, K2, V1, ..
__device__ __forceinline__ bool item_is_key(int i, int n) { return i < 2 ? !(n == 1 && i == 1) : (i & 1) != 0 && i != 2 * n - 1; }
__device__ __forceinline__ int item_tile(int i, int n) {
  if (item_is_key(i, n)) return i < 2 ? i : (i + 1) / 2;
  return i == 2 * n - 1 ? n - 1 : (i - 2) / 2;
}

struct Place {          // of a segment
  int b, hk, u, t0;
  int64_t left;
};

// FMT: what the caches hold (kKvSame, kKvE4M3, kKvE5M2)
template <typename T, int NH, int FMT, int R>
__global__ void __launch_bounds__(Cfg<NH, FMT != kKvSame, R>::kThreads, Cfg<NH, FMT != kKvSame, R>::kPerSm) attn_tree_kernel(const TreeParams p) {
  constexpr bool KV8 = FMT != kKvSame, kF16 = std::is_same<T, __half>::value;
  using C = Cfg<NH, KV8, R>;
  constexpr int kD = C::kD, kStages = C::kStages, kIssueWarp = C::kIssueWarp, kSoft = C::kSoftmaxWarps;
  extern __shared__ __align__(1024) uint8_t tree_smem[];
  __shared__ uint64_t bars[2 * C::kStages + 7 + 2 * R];
  __shared__ uint32_t tmem_holder;
  __shared__ int fail_flag, poison, holes;
  __shared__ int16_t parents[kParents];
  __shared__ int begin_of[3];
  __shared__ Request begin_request;
  __shared__ int64_t line_of[3];
  __shared__ int ctas_of;
  uint8_t* sQ = tree_smem;
  uint8_t* ring = sQ + C::kQBytes;
  uint64_t* full = bars;                 // [stage] the warps of a team
  uint64_t* empty = full + kStages;      // [stage] tcgen05.commit
  uint64_t* s_full = empty + kStages;    // [buffer] tcgen05.commit: scores of a tile
  uint64_t* p_full = s_full + 2;         // [buffer][row tile] the softmax warps: P is in tensor memory, O rescaled
  // [buffer] tcgen05.commit: a tile's P V.  A wait tells a phase from the one before it and no more: the scores of tile t, which a
  // thread has seen, were issued behind P V of t - 2, so one barrier would do for neither of the two products that may be out
  uint64_t* o_done = p_full + 2 * R;
  uint64_t* q_full = o_done + 2;         // the warps that copy Q
  uint64_t* q_free = q_full + 1;         // tcgen05.commit: the segment's last scores
  uint64_t* soft = q_free + 1;           // the softmax warps among themselves; not a named barrier, which would wait for a warp that gave up

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait_loads();

  // ---- where this CTA's run begins ----
  if (warp == 0) {
    const int per = (p.ix.batch + 31) / 32;
    const int first = min(p.ix.batch, lane * per), last = min(p.ix.batch, first + per);
    int64_t mine = 0;
    bool bad = false;
    Request r{};                     // of the first of this lane's requests
    for (int b = last - 1; b >= first; --b) {
      r = request_of(p.ix, b, &bad);
      if (r.nodes > 0) mine += static_cast<int64_t>(units_of(p, r)) * (tiles_of(p, r) + kStart);
    }
    if (bad && blockIdx.x == 0 && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const int64_t line = __shfl_sync(0xffffffffu, incl, 31) * p.hkv;
    const int used = ctas_used(p, line);
    const int c = blockIdx.x;
    const int64_t begin = c < used ? run_begin(line, c, used) : line, end = c < used ? run_begin(line, c + 1, used) : line;
    if (lane == 0) {
      line_of[0] = begin;
      line_of[1] = end - begin;
      line_of[2] = line;
      ctas_of = used;
      fail_flag = 0;
      poison = 0;
      holes = 0;
    }
    int64_t at = (incl - mine) * p.hkv;
    if (begin < end && begin >= at && begin < incl * p.hkv) {
      for (int b = first; b < last; ++b) {
        if (b > first) r = request_of(p.ix, b, nullptr);
        const int n = r.nodes > 0 ? tiles_of(p, r) + kStart : 0;
        const int64_t units = static_cast<int64_t>(n) * units_of(p, r) * p.hkv;
        if (begin >= at && begin < at + units) {
          const int64_t in = begin - at;
          const int unit = in < 0x7fffffff ? static_cast<int>(in) / n : static_cast<int>(in / n);
          begin_of[0] = b;
          begin_of[1] = unit;
          begin_of[2] = static_cast<int>(in - static_cast<int64_t>(unit) * n);
          begin_request = r;
        }
        at += units;
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
        for (int h = 0; h < R; ++h) mbar_init(&p_full[i * R + h], 4);
        mbar_init(&o_done[i], 1);
      }
      mbar_init(q_full, C::kQWarps);
      mbar_init(q_free, 1);
      mbar_init(soft, kSoft);
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc(&tmem_holder, C::kCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_holder;
  pdl_launch_dependents();

  const bool aligned = (smem_u32(tree_smem) & 1023) == 0;      // the swizzle counts from 1 KB boundaries
  if (!aligned && tid == 0 && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusPipelineTimeout);

  // Calls fn(place, request, tiles of the unit, tiles of the segment, segment begins at the run's begin) for every segment of the
  // run; all roles walk the same way.
  auto segments = [&](auto&& fn) {
    Place w;
    w.left = aligned ? line_of[1] : 0;
    if (w.left <= 0) return;
    w.b = begin_of[0];
    w.t0 = begin_of[2];
    Request r = begin_request;
    int units = units_of(p, r), n_all = tiles_of(p, r);
    w.hk = begin_of[1] / units;
    w.u = begin_of[1] - w.hk * units;
    bool first = true;
    while (w.left > 0) {
      if (w.t0 >= n_all) {
        if (n_all > 0) w.left -= n_all + kStart - w.t0;
        w.t0 = 0;
        if (n_all == 0 || ++w.u == units) {
          w.u = 0;
          if (n_all == 0 || ++w.hk == p.hkv) {
            w.hk = 0;
            if (++w.b >= p.ix.batch) return;
            r = request_of(p.ix, w.b, nullptr);
            units = units_of(p, r);
            n_all = tiles_of(p, r);
          }
        }
        first = false;
        continue;
      }
      const int n = static_cast<int>(min(static_cast<int64_t>(n_all - w.t0), w.left));
      if (!fn(w, r, n_all, n, first)) return;
      w.left -= n;
      w.t0 += n;
      first = false;
    }
  };
  const int g = p.group;
  // node of a row: rows are below 128 and g is not above, where 16 bits of the reciprocal give the quotient exactly
  const uint32_t inv_g = (65536u + g - 1) / g;
  auto node_of = [&](int r) { return static_cast<int>((r * inv_g) >> 16); };

  if (warp >= kSoft) {
    if constexpr (C::kSplit) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
    if (warp < kSoft + C::kTeams * C::kTeam) {
      // =============================== keys and values ===============================
      const int team = (warp - kSoft) / C::kTeam, part = (warp - kSoft) % C::kTeam;
      constexpr int kPart = kTile / C::kTeam;            // rows of this warp
      bool bad = false, ok = true;
      uint32_t item0 = 0;                                // items of the segments before
      segments([&](const Place& w, const Request& r, int, int n, bool) {
        const int* rtt = p.ix.req_to_token + static_cast<int64_t>(r.table) * p.ix.table_stride;
        const int len = r.prefix + r.nodes, base = first_token(p, r) + w.t0 * kTile + part * kPart;
        const int items = 2 * n, edge = edge_of(p, r);
        // slots of tokens lane and lane + 32 of this warp's rows of item i; -1: nothing to read
        auto slots_of = [&](int i) -> int2 {
          int2 s = make_int2(kNoToken, kNoToken);
          if (i < items) {
            const int tok = base + item_tile(i, n) * kTile + lane;
            if (tok < len) s.x = max(__ldcg(rtt + tok), -1);          // no number of the table is taken for kNoToken
            if (kPart > 32 && tok + 32 < len) s.y = max(__ldcg(rtt + tok + 32), -1);
          }
          return s;
        };
        auto checked = [&](int s) {
          if (s >= 0 && s < p.num_slots) return s;
          bad = bad || s != kNoToken;
          return -1;
        };
        constexpr int kCh = KV8 ? 4 * NH : 8 * NH;  // 16-byte pieces of a cached row
        constexpr int kRowsPer = 32 / kCh;          // rows of a warp's copy
        const int ch = lane % kCh, r0 = lane / kCh;
        using Elem = typename std::conditional<KV8, uint8_t, uint16_t>::type;
        int i = (team + C::kTeams - static_cast<int>(item0 % C::kTeams)) % C::kTeams;
        int2 sl = slots_of(i);
        for (; i < items; i += C::kTeams) {
          const uint32_t item = item0 + i, st = item % kStages;
          const uint32_t stage = smem_u32(ring) + st * C::kStage, raw = smem_u32(ring) + kStages * C::kStage + team * C::kRaw;
          auto wait_free = [&]() {       // asleep in between: warps that poll take issue slots from the softmax (e4m3, 16 nodes: 52.9 -> 49.6 us)
            if (item >= kStages && !mbar_wait_relaxed(&empty[st], (item / kStages - 1) & 1, 20)) ok = false;
            return ok = __all_sync(0xffffffffu, ok);
          };
          if (!KV8 && !wait_free()) return false;
          const int2 s = make_int2(checked(sl.x), checked(sl.y));
          const Elem* from = static_cast<const Elem*>(item_is_key(i, n) ? p.k_cache : p.v_cache) + w.hk * p.kv_head_stride + ch * (16 / sizeof(Elem));
#pragma unroll 8
          for (int k = 0; k < kPart / kRowsPer; ++k) {
            const int row = k * kRowsPer + r0;
            const int rs = __shfl_sync(0xffffffffu, k * kRowsPer < 32 ? s.x : s.y, row & 31);
            cp16(KV8 ? raw + (part * kPart + row) * kD + ch * 16 : stage + swz(row, ch, C::kBlock), from + max(rs, 0) * p.kv_tok_stride, rs >= 0);
          }
          cp_commit();
          sl = slots_of(i + C::kTeams);
          // values of a tile that some rows do not see all of
          const int col0 = first_token(p, r) + (w.t0 + item_tile(i, n)) * kTile;
          const bool look = !item_is_key(i, n) && (col0 + kTile > r.prefix || col0 < edge);
          bool found = false;
          auto cleaned = [&](uint32_t two) -> uint32_t {       // elements that are no numbers: 0
            constexpr uint32_t kExpo = kF16 ? 0x7c00u : 0x7f80u;
            const uint32_t off = ((two & kExpo) == kExpo ? 0xffffu : 0u) | ((two & (kExpo << 16)) == (kExpo << 16) ? 0xffff0000u : 0u);
            found = found || off != 0;
            return two & ~off;
          };
          cp_wait<0>();
          if (!KV8 && look) {
#pragma unroll 1
            for (int k = 0; k < kPart / kRowsPer; ++k) {        // what this thread copied itself
              const uint32_t at = stage + swz(k * kRowsPer + r0, ch, C::kBlock);
              uint32_t x[4], y[4];
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at));
#pragma unroll
              for (int h = 0; h < 4; ++h) y[h] = cleaned(x[h]);
              if ((x[0] ^ y[0]) | (x[1] ^ y[1]) | (x[2] ^ y[2]) | (x[3] ^ y[3]))
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
            }
          }
          if constexpr (KV8) {
            // a thread widens the bytes that it copied itself
            if (!wait_free()) return false;
            auto widen = [&](uint32_t two) -> uint32_t {     // two 8-bit values -> two 16-bit ones, exactly
              const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu),
                                                               FMT == kKvE5M2 ? __NV_E5M2 : __NV_E4M3);
              if constexpr (kF16) return *reinterpret_cast<const uint32_t*>(&h);
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
              return pack_bf16x2(f.x, f.y);
            };
            // four loads side by side, then their work
            constexpr int kBatch = 4;
            static_assert(kPart / kRowsPer % kBatch == 0, "batches of rows");
#pragma unroll 1
            for (int k0 = 0; k0 < kPart / kRowsPer; k0 += kBatch) {
              uint32_t x[kBatch][4];
#pragma unroll
              for (int k = 0; k < kBatch; ++k) {
                const int row = part * kPart + (k0 + k) * kRowsPer + r0;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(x[k][0]), "=r"(x[k][1]), "=r"(x[k][2]), "=r"(x[k][3])
                             : "r"(raw + row * kD + ch * 16));
              }
#pragma unroll
              for (int k = 0; k < kBatch; ++k) {
                const int row = part * kPart + (k0 + k) * kRowsPer + r0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  uint32_t y[4] = {widen(x[k][2 * h]), widen(x[k][2 * h] >> 16), widen(x[k][2 * h + 1]), widen(x[k][2 * h + 1] >> 16)};
                  if (look)
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = cleaned(y[e]);
                  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + swz(row, ch * 2 + h, C::kBlock)), "r"(y[0]), "r"(y[1]),
                               "r"(y[2]), "r"(y[3])
                               : "memory");
                }
              }
            }
          }
          if (KV8 || look) fence_proxy_async_smem();
          if (found) poison = 1;            // for the rest of the run: the rows' ends look for themselves
          if (bad) holes = 1;               // likewise, the softmax warps at every tile
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[st]);
        }
        item0 += items;
        return true;
      });
      cp_wait<0>();
      if (!ok) fail_flag = 1;
      if (bad && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
    } else if (warp < kIssueWarp) {
      // =============================== queries ===============================
      // Rows that hold no node keep what is there: they meet only themselves.
      bool ok = true;
      uint32_t seg = 0;
      segments([&](const Place& w, const Request& r, int, int, bool) {
        if (seg > 0 && !mbar_wait_relaxed(q_free, (seg - 1) & 1)) ok = false;
        if (!(ok = __all_sync(0xffffffffu, ok))) return false;
        const int n0 = w.u * p.unit_nodes, rows = min(p.unit_nodes, r.nodes - n0) * g, half = p.tpt * g;     // half: rows of a tile
        const uint16_t* q = static_cast<const uint16_t*>(p.q) + static_cast<int64_t>(r.row + n0) * p.q_stride + static_cast<int64_t>(w.hk) * g * kD;
        constexpr int kCh = 8 * NH;               // 16-byte pieces of a row
#pragma unroll 4
        for (int c = (warp - kSoft - C::kTeams * C::kTeam) * 32 + lane; c < rows * kCh; c += C::kQWarps * 32) {
          const int all = c / kCh, ch = c % kCh, h = R > 1 && all >= half ? 1 : 0, row = all - h * half, node = node_of(row) + h * p.tpt;
          cp16(smem_u32(sQ) + h * C::kQTile + swz(row, ch, C::kQBlock), q + node * p.q_stride + static_cast<int64_t>(all - node * g) * kD + ch * 8,
               true);
        }
        cp_commit();
        cp_wait<0>();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        ++seg;
        return true;
      });
      if (!ok) fail_flag = 1;
    } else if (warp == kIssueWarp) {
      if (elect_one()) {
        // =============================== products ===============================
        bool ok = true;
        auto wait_on = [&](uint64_t* bar, uint32_t parity) {
          if (ok && !mbar_wait(bar, parity, &fail_flag)) ok = false;
          if (ok) {
            fence_proxy_async_smem();       // copies by cp.async were made in the generic proxy
            tc_fence_after_sync();
          }
        };
        const uint64_t q_desc = umma_desc_k_sw128(smem_u32(sQ)), k_desc0 = umma_desc_k_sw128(smem_u32(ring));
        const uint64_t v_desc0 = umma_desc_mn_sw128(smem_u32(ring), C::kBlock, 1024);
        const uint32_t idesc_s = p.idesc_s, idesc_o = p.idesc_o, tmem_o = tmem + C::kScoreCols;
        uint32_t item = 0, seg = 0, tile = 0;      // tile: products of values so far
        segments([&](const Place&, const Request&, int, int n, bool) {
          auto scores = [&](int t) {
            const uint32_t st = item % kStages, buf = (tile + t) & 1;
            wait_on(&full[st], (item / kStages) & 1);
            if (!ok) return;
            const uint64_t k_desc = k_desc0 + st * (C::kStage >> 4);
#pragma unroll
            for (int h = 0; h < R; ++h)
#pragma unroll
              for (int kk = 0; kk < 4 * NH; ++kk)
                umma_f16(tmem + (h * 2 + buf) * kTile, q_desc + h * (C::kQTile >> 4) + (kk >> 2) * (C::kQBlock >> 4) + (kk & 3) * 2,
                         k_desc + (kk >> 2) * (C::kBlock >> 4) + (kk & 3) * 2, idesc_s, kk > 0 ? 1u : 0u);
            umma_commit(&empty[st]);
            umma_commit(&s_full[buf]);
            if (t == n - 1) umma_commit(q_free);
            ++item;
          };
          if (ok && !mbar_wait(q_full, seg & 1, &fail_flag)) ok = false;
          scores(0);
          if (n > 1) scores(1);
          for (int t = 0; t < n && ok; ++t) {
            const uint32_t st = item % kStages, at = tile + t, buf = at & 1;
            wait_on(&full[st], (item / kStages) & 1);
            const uint64_t v_desc = v_desc0 + st * (C::kStage >> 4);
#pragma unroll
            for (int h = 0; h < R; ++h) {
              if (ok && !mbar_wait(&p_full[buf * R + h], (at >> 1) & 1, &fail_flag)) ok = false;
              tc_fence_after_sync();
              if (!ok) break;
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                umma_f16_ts(tmem_o + h * kD, tmem + (h * 2 + buf) * kTile + kk * 8, v_desc + kk * (2048 >> 4), idesc_o, t > 0 || kk > 0 ? 1u : 0u);
            }
            if (!ok) break;
            umma_commit(&empty[st]);
            umma_commit(&o_done[buf]);
            ++item;
            if (t + 2 < n) scores(t + 2);
          }
          tile += n;
          ++seg;
          return ok;
        });
        if (!ok) fail_flag = 1;
      }
    }
  } else {
    // =============================== softmax ===============================
    if constexpr (C::kSplit) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
    const int half = R > 1 ? warp >> 2 : 0, in_tile = tid & 127;      // row tile and row
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tmem_o = tmem + C::kScoreCols + half * kD + lane_base;
    const int tile_node = node_of(in_tile), row_node = half * p.tpt + tile_node, row = half * p.tpt * g + in_tile;    // row of the unit
    const bool capped = p.cap_out > 0.f;
    bool ok = true, bad = false;
    uint32_t tile = 0, met = 0;
    auto meet = [&]() {        // of all softmax warps; false where one has given up
      __syncwarp();
      if (lane == 0) mbar_arrive(soft);
      if (!mbar_wait(soft, met++ & 1, &fail_flag)) ok = false;
      return ok = __all_sync(0xffffffffu, ok);
    };
    int job_rows = 0, job_row = 0, job_head = 0, job_tiles = 0;
    segments([&](const Place& w, const Request& r, int n_all, int n, bool first) {
      const int node = w.u * p.unit_nodes + row_node;
      const bool valid = tile_node < p.tpt && node < r.nodes;
      const bool warp_valid = __any_sync(0xffffffffu, valid);
      const int key0 = first_token(p, r) + w.t0 * kTile, len = r.prefix + r.nodes;
      const bool bounded = p.window > 0 || p.chunk > 0;
      const bool masks = bounded || key0 + n * kTile > r.prefix;      // the segment has masked tiles
      auto parent_in = [&](int i) {
        const int up = __ldcg(p.ix.parents + r.row + i);
        if (up < -1 || up >= i) {
          bad = true;
          return -1;
        }
        return up;
      };
      if (masks) {        // parents to shared memory; one that is no earlier node counts as none
        if (!meet()) return false;          // the segment before has read them
        for (int i = tid; i < min(r.nodes, kParents); i += 32 * kSoft) parents[i] = static_cast<int16_t>(parent_in(i));
        if (!meet()) return false;
      }
      auto parent_of = [&](int i) { return i < kParents ? static_cast<int>(parents[i]) : parent_in(i); };
      int pos = r.prefix, low = 0;
      if (valid && bounded) {
        for (int a = parent_of(node); a >= 0; a = parent_of(a)) ++pos;
        low = first_key(p, pos);
      }
      const int edge = edge_of(p, r);
      // bit c: this row sees token col0 + c
      auto visible = [&](int col0) -> uint64_t {
        uint64_t m = 0;
        if (!valid) return m;       // no node: nothing to walk
        const int a = max(low, col0) - col0, e = min(r.prefix, col0 + kTile) - col0;      // [a, e) of the cached tokens
        if (e > a) m = (e >= 64 ? ~0ull : (1ull << e) - 1) & (~0ull << a);
        if (col0 + kTile > r.prefix) {
          int at = pos;
          const int shift = r.prefix - col0;
          auto see = [&](int j) {
            const int c = shift + j;
            if (c >= 0 && c < kTile) m |= 1ull << c;
          };
          if (!bounded && r.nodes <= kParents) {
            for (int j = node; j >= 0; j = parents[j]) see(j);
          } else {
            for (int j = node; j >= 0 && at >= low; j = parent_of(j), --at) {
              see(j);
              if (!bounded) at = low + 1;
            }
          }
        }
        return m;
      };

      // rare: bit c: token col0 + c has a slot
      auto present = [&](int col0) -> uint64_t {
        uint64_t m = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int tok = col0 + 32 * h + lane;
          const int s = tok < len ? __ldcg(p.ix.req_to_token + static_cast<int64_t>(r.table) * p.ix.table_stride + tok) : -1;
          m |= static_cast<uint64_t>(__ballot_sync(0xffffffffu, s >= 0 && s < p.num_slots)) << (32 * h);
        }
        return m;
      };

      float m_used = -INFINITY;   // maximum in use for the exponent (log2 domain)
      uint64_t sums[4] = {0, 0, 0, 0};      // pairs of fp32
      for (int t = 0; t < n; ++t) {
        const uint32_t at = tile + t, buf = at & 1;
        const int col0 = key0 + t * kTile;
        const bool masked = col0 + kTile > r.prefix || col0 < edge;
        if (!mbar_wait(&s_full[buf], (at >> 1) & 1, &fail_flag)) ok = false;
        if (!__all_sync(0xffffffffu, ok)) return ok = false;
        tc_fence_after_sync();
        if (warp_valid) {
          uint32_t raw[kTile];
          const uint32_t tmem_s = tmem + (half * 2 + buf) * kTile + lane_base;
          tmem_ld_32x32(tmem_s, *reinterpret_cast<uint32_t(*)[32]>(&raw[0]));
          tmem_ld_32x32(tmem_s + 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[32]));
          tmem_ld_wait();
          float mul = p.scale_log2;
          if (capped) {        // cap tanh(x / cap), in the log2 domain; tanh(y) = 1 - 2 / (1 + e^(2 y))
            mul = 1.f;
#pragma unroll
            for (int c = 0; c < kTile; ++c)
              raw[c] = __float_as_uint(p.cap_out * (1.f - __fdividef(2.f, 1.f + ex2(__uint_as_float(raw[c]) * p.cap_in))));
          }
          const bool gaps = __any_sync(0xffffffffu, holes != 0);
          if (masked || gaps) {
            uint64_t vis = masked ? visible(col0) : ~0ull;
            if (gaps) vis &= present(col0);
#pragma unroll
            for (int c = 0; c < kTile; ++c) raw[c] = (vis >> c) & 1 ? raw[c] : __float_as_uint(-INFINITY);
          }
          float mx[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i] = fmaxf(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1]));
#pragma unroll
          for (int c = 8; c < kTile; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], __uint_as_float(raw[c]), __uint_as_float(raw[c + 1]));
          const float m_tile = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * mul;
          float factor = 1.f;
          bool need = false;
          if (!valid || m_used == -INFINITY) {
            m_used = m_tile;      // no key seen so far: the row of O is zero
          } else if (m_tile > m_used + kRescaleThreshold) {
            factor = exp2f(m_used - m_tile);
            m_used = m_tile;
            need = true;
          }
          if (__any_sync(0xffffffffu, need)) {
            if (!mbar_wait(&o_done[buf ^ 1], ((at - 1) >> 1) & 1, &fail_flag)) ok = false;
            if (!__all_sync(0xffffffffu, ok)) return ok = false;
            tc_fence_after_sync();
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[i] = fma2(sums[i], pair_of(factor, factor), 0);
#pragma unroll 1
            for (int c = 0; c < kD; c += 16) {
              uint32_t o[16];
              tmem_ld_32x16(tmem_o + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
              tmem_st_32x16(tmem_o + c, o);
            }
          }
          const float neg = m_used == -INFINITY ? 0.f : -m_used;
          const uint64_t mul2 = pair_of(mul, mul), neg2 = pair_of(neg, neg);
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float2 x = halves_of(fma2(pair_of(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1])), mul2, neg2));
            const float p0 = ex2(x.x), p1 = ex2(x.y);
            sums[i & 3] = add2(sums[i & 3], pair_of(p0, p1));
            pk[i] = pack2<T>(p0, p1);
          }
          tmem_st_32x32(tmem_s, pk);
          tmem_st_wait();
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[buf * R + half]);
      }
      tile += n;
      if (!mbar_wait(&o_done[(tile - 1) & 1], ((tile - 1) >> 1) & 1, &fail_flag)) ok = false;
      if (!__all_sync(0xffffffffu, ok)) return ok = false;
      tc_fence_after_sync();

      // ---- the segment's rows ----
      const bool whole = w.t0 == 0 && n == n_all;
      const int head = w.hk * g + row - row_node * g;
      const float2 both = halves_of(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])));
      float l = both.x + both.y;
      if (whole && p.sink != nullptr && valid && m_used > -INFINITY) l += exp2f(p.sink[head] * kLog2e - m_used);
      const float inv = l == 0.f ? 0.f : 1.f / l;       // 0: no key seen.  A sum that is no number shows
      const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (first ? 0 : 1);
      if (masks && poison != 0) {       // rare: every masked tile's values once more, for those that are no numbers
        const int* rtt = p.ix.req_to_token + static_cast<int64_t>(r.table) * p.ix.table_stride;
#pragma unroll 1
        for (int c = 0; c < kD; c += 16) {
          uint32_t o[16];
          tmem_ld_32x16(tmem_o + c, o);
          tmem_ld_wait();
#pragma unroll 1
          for (int t = 0; t < n; ++t) {
            const int col0 = key0 + t * kTile;
            if (!(col0 + kTile > r.prefix || col0 < edge)) continue;
            const uint64_t vis = visible(col0);
#pragma unroll 1
            for (int k = 0; k < kTile && col0 + k < len; ++k) {
              if (!((vis >> k) & 1)) continue;
              const int s = __ldcg(rtt + col0 + k);
              if (s < 0 || s >= p.num_slots) continue;
              const int64_t from = s * p.kv_tok_stride + w.hk * p.kv_head_stride + c;
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float v;
                if constexpr (KV8) v = unpack_fp8x2(static_cast<const uint8_t*>(p.v_cache)[from + i], FMT).x;
                else v = to_f32(static_cast<const T*>(p.v_cache)[from + i]);
                if ((__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) o[i] = __float_as_uint(__uint_as_float(o[i]) + v);
              }
            }
          }
          __syncwarp();
          tmem_st_32x16(tmem_o + c, o);
        }
        tmem_st_wait();
      }
      if (warp_valid) {
#pragma unroll 1
        for (int c = 0; c < kD; c += 32) {
          uint32_t o[32];
          tmem_ld_32x32(tmem_o + c, o);
          tmem_ld_wait();
          if (valid) {
            float f[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(o[i]) * inv;
            if (whole) {
              uint16_t* to = static_cast<uint16_t*>(p.out) + (r.row + node) * p.out_stride + static_cast<int64_t>(head) * kD + c;
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                uint32_t v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = pack2<T>(f[i + 2 * k], f[i + 2 * k + 1]);
                *reinterpret_cast<uint4*>(to + i) = make_uint4(v[0], v[1], v[2], v[3]);
              }
            } else {
              float* to = p.part_o + slot * p.part_rows * kD + (static_cast<int64_t>(c / 4) * p.part_rows + row) * 4;
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<float4*>(to + static_cast<int64_t>(i) * p.part_rows) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
            }
          }
        }
        if (!whole && valid) p.part_lse[slot * p.part_rows + row] = l == 0.f ? -INFINITY : m_used + log2f(l);
      }
      if (!whole && w.t0 + n == n_all) {        // the unit's last tile: it began in front of this run
        job_rows = min(p.unit_nodes, r.nodes - w.u * p.unit_nodes) * g;
        job_row = r.row + w.u * p.unit_nodes;
        job_head = w.hk * g;
        job_tiles = w.t0;
      }
      tc_fence_before_sync();
      return true;
    });
    if (!ok) fail_flag = 1;
    if (bad && p.ix.status != nullptr) atomicExch(p.ix.status, kStatusBadIndex);
    if (tid == 0) {
      p.job_rows[blockIdx.x] = ok ? job_rows : 0;
      if (ok && job_rows > 0) {
        const int64_t line = line_of[2], begin = line_of[0] - job_tiles;
        const int used = ctas_of;
        // the last CTA whose run begins at or before the unit
        const int c0 = fits_32(line, used) ? static_cast<int>((static_cast<uint32_t>(begin + 1) * used - 1u) / static_cast<uint32_t>(line))
                                           : static_cast<int>(((begin + 1) * used - 1) / line);
        p.jobs[blockIdx.x] = make_int4(job_row, job_head, c0, run_begin(line, c0, used) < begin ? 1 : 0);
      }
    }
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
    tmem_dealloc(tmem, C::kCols);
  }
}

// Joins the partial results of the units that lie in several CTAs: out = sum_c w_c O_c with w_c = 2^(lse_c - max) / sum; a head's
// sink is one more term of the sum, without a value.  blockIdx.x is a note; a warp takes 32 rows (a lane each) and 16
// features, and gridDim.y blocks have a warp for every such task of the largest unit.
constexpr int kJoinWarps = 8, kJoinFeatures = 16;
template <typename T, int HD>
__global__ void __launch_bounds__(32 * kJoinWarps) attn_tree_join_kernel(const TreeParams p) {
  pdl_launch_dependents();
  pdl_wait_loads();
  const int rows = __ldcg(p.job_rows + blockIdx.x);
  const int4 job = __ldcg(p.jobs + blockIdx.x);           // anything where rows is 0
  const int row0 = job.x, head0 = job.y, c0 = job.z, second = job.w;
  const int c1 = blockIdx.x, lane = threadIdx.x & 31;
  const int groups = (rows + 31) / 32;
  for (int task = blockIdx.y * kJoinWarps + (threadIdx.x >> 5); task < groups * (HD / kJoinFeatures); task += kJoinWarps * gridDim.y) {
    const int r = task % groups * 32 + lane, d = task / groups * kJoinFeatures;
    if (r >= rows) continue;
    const int node = r / p.group, head = head0 + r - node * p.group;
    auto slot = [&](int c) { return static_cast<int64_t>(c) * 2 + (c == c0 ? second : 0); };
    const float sink = p.sink != nullptr ? p.sink[head] * kLog2e : -INFINITY;
    float top = sink;
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) top = fmaxf(top, __ldcg(p.part_lse + slot(c) * p.part_rows + r));
    float den = sink > -INFINITY ? exp2f(sink - top) : 0.f, acc[kJoinFeatures] = {};
#pragma unroll 2
    for (int c = c0; c <= c1; ++c) {
      const float lse = __ldcg(p.part_lse + slot(c) * p.part_rows + r);
      const float4* from = reinterpret_cast<const float4*>(p.part_o + slot(c) * p.part_rows * HD) + (d / 4) * p.part_rows + r;
      float4 x[kJoinFeatures / 4];
#pragma unroll
      for (int k = 0; k < kJoinFeatures / 4; ++k) x[k] = __ldcg(from + k * p.part_rows);
      if (lse == -INFINITY) continue;           // saw no key
      const float w = exp2f(lse - top);
      den += w;
#pragma unroll
      for (int k = 0; k < kJoinFeatures / 4; ++k) {
        acc[4 * k] = fmaf(w, x[k].x, acc[4 * k]);
        acc[4 * k + 1] = fmaf(w, x[k].y, acc[4 * k + 1]);
        acc[4 * k + 2] = fmaf(w, x[k].z, acc[4 * k + 2]);
        acc[4 * k + 3] = fmaf(w, x[k].w, acc[4 * k + 3]);
      }
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
    __align__(16) T o[kJoinFeatures];
#pragma unroll
    for (int k = 0; k < kJoinFeatures; ++k) o[k] = from_f32<T>(acc[k] * inv);
    uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (row0 + node) * p.out_stride + static_cast<int64_t>(head) * HD + d);
#pragma unroll
    for (int k = 0; k < kJoinFeatures / 8; ++k) to[k] = reinterpret_cast<const uint4*>(o)[k];
  }
}

template <typename T, int NH, int FMT, int R>
int launch_one(const TreeParams& p, cudaStream_t s) {
  using C = Cfg<NH, FMT != kKvSame, R>;
  auto kern = attn_tree_kernel<T, NH, FMT, R>;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kern), C::kSmem) != cudaSuccess) return -3;
  if constexpr (C::kSplit) {
    // the softmax warps take registers that the others give back: together no more than the kernel is launched with
    static const int regs = [kern] {
      cudaFuncAttributes at{};
      return cudaFuncGetAttributes(&at, reinterpret_cast<const void*>(kern)) == cudaSuccess ? at.numRegs : 0;
    }();
    if (regs < C::kLaunchRegs) return -5;
  }
  cudaError_t err = launch_pdl(kern, dim3(p.ctas), dim3(C::kThreads), C::kSmem, s, p);
  note_launch();
  if (err != cudaSuccess) return -4;
  const int join_parts = ((p.part_rows + 31) / 32 * (C::kD / kJoinFeatures) + kJoinWarps - 1) / kJoinWarps;
  err = launch_pdl(attn_tree_join_kernel<T, 64 * NH>, dim3(p.ctas, join_parts), dim3(32 * kJoinWarps), 0, s, p);
  note_launch();
  return err == cudaSuccess ? 0 : -4;
}
template <typename T, int NH, int R>
int launch_format(const TreeParams& p, int fmt, cudaStream_t s) {
  switch (fmt) {
    case kKvSame: return launch_one<T, NH, kKvSame, R>(p, s);
    case kKvE4M3: return launch_one<T, NH, kKvE4M3, R>(p, s);
    default: return launch_one<T, NH, kKvE5M2, R>(p, s);
  }
}
template <typename T>
int launch_type(const TreeParams& p, int head_dim, int fmt, cudaStream_t s) {
  switch (head_dim) {
    case 64: return launch_format<T, 1, 1>(p, fmt, s);
    case 128: return p.unit_nodes > p.tpt ? launch_format<T, 2, 2>(p, fmt, s) : launch_format<T, 2, 1>(p, fmt, s);
    default: return launch_format<T, 4, 1>(p, fmt, s);
  }
}

}  // namespace

TreePlan tree_plan(int head_dim, int group, int64_t rows, int64_t batch, int num_sms) {
  TreePlan plan;
  // Row tiles that a CTA takes side by side: two where a request has more rows than one tile on average.  Two tiles against one, 16 requests
  // of 4096 tokens, 8 query heads over a kv head, 128 features: 24 nodes (192 rows) 59.1 / 76.5 us with e4m3 caches, which are widened
  // half as often, and 58.4 / 62.5 us in bf16; 17 nodes (136 rows) 56.8 / 58.9 and 55.5 / 51.9; 16 nodes (128 rows) 56.0 / 49.6 and 54.1 / 47.2.
  // So with 16-bit caches the rule loses 7 % just above one tile and wins as much at one and a half; where that turns is not measured.
  // Heads of 64: 54.7 / 54.2 and 50.0 / 53.6 at 24 nodes, 54.0 / 42.3 and 48.8 / 42.0 at 17: always one.
  plan.row_tiles = head_dim == 128 && rows > batch * (kRows / group) ? 2 : 1;
  plan.ctas = head_dim == 256 || plan.row_tiles == 2 ? num_sms : 2 * num_sms;
  plan.part_rows = static_cast<int>(std::min<int64_t>(plan.row_tiles * (kRows / group * group), rows * group));
  plan.workspace_floats = static_cast<int64_t>(plan.ctas) * (2 * plan.part_rows * (head_dim + 1) + kJobInts) + 4;      // 4: notes on a 16-byte boundary
  return plan;
}

int launch_attention_tree(const TreeAttnArgs& a, cudaStream_t s) {
  const int g = a.hkv > 0 ? a.hq / a.hkv : 0;
  if ((a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) || a.hkv <= 0 || a.hq % a.hkv != 0 || g < 1 || g > kRows) return -1;
  if (a.index.rows <= 0 || a.index.batch <= 0) return 0;
  TreeParams p{};
  p.q = a.q;
  p.k_cache = a.k_cache;
  p.v_cache = a.v_cache;
  p.out = a.out;
  p.ctas = a.plan.ctas;
  p.part_rows = a.plan.part_rows;
  p.part_o = a.workspace;
  p.part_lse = p.part_o + static_cast<int64_t>(p.ctas) * 2 * p.part_rows * a.head_dim;
  p.jobs = reinterpret_cast<int4*>(p.part_lse + static_cast<int64_t>(p.ctas) * 2 * p.part_rows + (p.ctas * 2 * p.part_rows & 3));
  p.job_rows = reinterpret_cast<int*>(p.jobs + p.ctas);
  p.ix = a.index;
  p.sink = a.sink;
  p.q_stride = a.q_stride;
  p.out_stride = a.out_stride;
  p.num_slots = a.num_slots;
  p.kv_tok_stride = a.kv_tok_stride;
  p.kv_head_stride = a.kv_head_stride;
  p.hkv = a.hkv;
  p.group = g;
  p.tpt = kRows / g;
  p.unit_nodes = a.plan.row_tiles * p.tpt;
  p.window = a.window > 0 ? a.window : 0;
  p.chunk = a.chunk > 0 ? a.chunk : 0;
  p.scale_log2 = a.scale * kLog2e;
  if (a.logit_cap > 0.f) {
    p.cap_in = 2.f * kLog2e * a.scale / a.logit_cap;
    p.cap_out = a.logit_cap * kLog2e;
  }
  const uint32_t fmt = a.dt == kF16 ? 0u : 1u;
  p.idesc_s = umma_idesc(kRows, kTile, 1, fmt, fmt, 0, 0);
  p.idesc_o = umma_idesc(kRows, a.head_dim, 1, fmt, fmt, 0, 1);
  return a.dt == kF16 ? launch_type<__half>(p, a.head_dim, a.kv_fmt, s) : launch_type<__nv_bfloat16>(p, a.head_dim, a.kv_fmt, s);
}

}  // namespace mb200
