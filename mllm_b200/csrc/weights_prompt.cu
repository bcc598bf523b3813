// The attention weights of prompts: bf16 queries, and what the host asks for.  A type a file: there are many kernels.
#include "weights_prompt.cuh"

namespace mb200 {

static constexpr int kShortPromptRows = 64;

bool weights_prompt_covers(int head_dim, int group) { return (head_dim == 64 || head_dim == 128 || head_dim == 256) && group >= 1 && group <= 32; }

int64_t weights_prompt_floats(const WeightsPromptArgs& a) { return a.rows * a.hq + static_cast<int64_t>(a.num_sms) * (4 * row_tiles(a) * kTileRows + 4) + 4; }

int launch_weights_prompt(const WeightsPromptArgs& a, cudaStream_t s) {
  if (a.hkv <= 0 || a.hq % a.hkv != 0 || !weights_prompt_covers(a.head_dim, a.hq / a.hkv)) return -1;
  if (a.index.batch <= 0 || a.rows <= 0) return 0;
  // One kernel where no request can be long, by the sizes of the tables, and has few observed rows (256 tokens, 8 kv heads, 8 requests: 32 rows
  // 9.3 us and 22.8 by the kernels for long ones, 64 rows 16.2 and 24.1, 128 rows 30.0 and 24.5; 74 requests, 64 rows: 38.3 and 54.4).
  const int64_t rows = (a.last > 0 ? std::min<int64_t>(a.last, a.index.table_cols) : a.index.table_cols) * (a.hq / a.hkv);
  if (a.index.table_cols <= kShortPromptTokens && rows <= kShortPromptRows)
    return launch_weights_prompt_short(a, s);
  return a.dt == kF16 ? launch_weights_prompt_fp16(a, s) : launch_prompt<__nv_bfloat16>(a, s);
}

}  // namespace mb200
