// velokv_logits.cpp -- host side of vk_token_logprobs (include/velokv.h). The kernels
// are in velokv_logits.hip.
#include <cmath>

#include "velokv_internal.h"

using namespace velokv;

namespace {

constexpr int32_t kMaxVocab = 1 << 28;

struct LogprobPlan {
  int parts, part_len;
  bool whole;  // a row is one workgroup of 16 waves
  uint64_t sums_bytes, top_bytes;
};

int plan_logprobs(const vk_ctx* ctx, const vk_logprob_args* a, LogprobPlan* pl) {
  if (!a) return fail(VK_ERR_BAD_ARG, "args is null");
  if (a->dtype != VK_DT_F32 && a->dtype != VK_DT_F16) return fail(VK_ERR_BAD_ARG, "dtype %d", a->dtype);
  if (a->n_rows < 0 || a->vocab <= 0 || a->n_tokens < 0 || a->n_top < 0) return fail(VK_ERR_BAD_ARG, "bad sizes");
  if (a->row_stride != 0 && a->row_stride < a->vocab)
    return fail(VK_ERR_BAD_ARG, "row_stride %lld is less than the vocabulary (%d)", (long long)a->row_stride, a->vocab);
  if (a->vocab > kMaxVocab) return fail(VK_ERR_UNSUPPORTED, "vocabulary of %d (up to %d)", a->vocab, kMaxVocab);
  if (a->n_top > kMaxTop) return fail(VK_ERR_UNSUPPORTED, "n_top %d (up to %d)", a->n_top, kMaxTop);
  if (a->n_top > a->vocab) return fail(VK_ERR_BAD_ARG, "n_top %d exceeds the vocabulary (%d)", a->n_top, a->vocab);
  // the kernels' exponents are (x - max) * scale * log2(e), whose factor has to be finite (0 at the maximum)
  if (!(a->scale >= 0.f) || !std::isfinite(a->scale * 1.4426950408889634f))
    return fail(VK_ERR_BAD_ARG, "scale must not be negative, and finite times log2(e)");
  // Parts of 8192 values (a step of a workgroup of four waves) at least, about four
  // workgroups a CU (64 rows of 128000 fp16, 20 alternatives: 14.9 us, 16.7 with two a CU, 19.7
  // with one of 16 waves a row; one row: 8.7, 16.8 with 16 waves). Rows of 2 to 4 steps, no more
  // than the CUs, take one workgroup of 16 waves each and no join (256 of 32000 fp16: 9.2 us, 12.1
  // in parts; 256 of 20000 with 20 alternatives: 9.7, 14.9; 128 of 20000 fp32: 9.7, 10.5; one of
  // 32000 fp32: 8.6 either way; 64 of 32000 fp32: 10.0, 9.5).
  constexpr int kStep = 8192;
  const int64_t rows = std::max<int64_t>(1, a->n_rows);
  const int64_t steps = ((int64_t)a->vocab + kStep - 1) / kStep;
  pl->whole = rows <= ctx->n_cu && steps > 1 && steps <= 4;
  const int64_t want = pl->whole ? 1 : std::max<int64_t>(1, std::min({(4 * ctx->n_cu + rows - 1) / rows, steps, (int64_t)kMaxLogitParts}));
  const int64_t per = (steps + want - 1) / want;
  pl->part_len = (int)std::min<int64_t>(per * kStep, kMaxVocab);
  pl->parts = (int)((steps + per - 1) / per);
  pl->sums_bytes = pl->top_bytes = 0;
  if (pl->parts > 1) {
    pl->sums_bytes = align_up((uint64_t)a->n_rows * pl->parts * 4 * sizeof(float), 256);
    pl->top_bytes = align_up((uint64_t)a->n_rows * pl->parts * a->n_top * sizeof(uint64_t), 256);
  }
  if ((uint64_t)a->n_rows * pl->parts * (pl->whole ? 1024 : 256) >= 1ull << 32) return fail(VK_ERR_UNSUPPORTED, "grid too large");
  return VK_OK;
}

}  // namespace

std::vector<std::string> velokv::logits_kernel_names() {
  return {"vk_logprob_part_q0", "vk_logprob_part_q1", "vk_logprob_row_q0", "vk_logprob_row_q1", "vk_logprob_join_q0", "vk_logprob_join_q1"};
}

extern "C" int vk_token_logprobs_workspace(const vk_ctx* ctx, const vk_logprob_args* a, uint64_t* bytes) {
  if (!ctx || !bytes) return fail(VK_ERR_BAD_ARG, "null argument");
  LogprobPlan pl;
  if (int rc = plan_logprobs(ctx, a, &pl)) return rc;
  *bytes = pl.sums_bytes + pl.top_bytes;
  return VK_OK;
}

extern "C" int vk_token_logprobs(vk_ctx* ctx, const vk_logprob_args* a, void* stream) {
  if (!ctx) return fail(VK_ERR_NOT_WIRED, "context is null");
  LogprobPlan pl;
  int rc = plan_logprobs(ctx, a, &pl);
  if (rc) return rc;
  if (a->n_rows == 0) return VK_OK;
  if (!a->logits || (a->n_tokens && (!a->tokens || !a->token_logprobs)) || (a->n_top && (!a->top_ids || !a->top_logprobs)))
    return fail(VK_ERR_BAD_ARG, "null device pointer");
  if (reinterpret_cast<uintptr_t>(a->logits) % (a->dtype == VK_DT_F32 ? 4 : 2))
    return fail(VK_ERR_BAD_ARG, "logits are not aligned to their type");
  if ((rc = set_device(ctx))) return rc;
  const uint64_t need = pl.sums_bytes + pl.top_bytes;
  uint8_t* ws = nullptr;
  if (need) {
    if (!a->workspace && !scratch_at_hand(ctx, nullptr, 0, need, stream))
      return fail(VK_ERR_BAD_ARG, "a captured call needs %llu bytes of scratch: give it a workspace", (unsigned long long)need);
    if ((rc = split_workspace(ctx, a->workspace, a->workspace_bytes, need, &ws))) return rc;
  }
  LogprobParams p{};
  p.logits = a->logits;
  p.tokens = a->tokens;
  p.token_logprobs = a->token_logprobs;
  p.entropy = a->entropy;
  p.top_ids = a->top_ids;
  p.top_logprobs = a->top_logprobs;
  p.part_sums = reinterpret_cast<float*>(ws);
  p.part_top = reinterpret_cast<uint64_t*>(ws + pl.sums_bytes);
  p.row_stride = a->row_stride ? a->row_stride : a->vocab;
  p.n_rows = a->n_rows;
  p.vocab = a->vocab;
  p.n_tokens = a->n_tokens;
  p.n_top = a->n_top;
  p.n_parts = pl.parts;
  p.part_len = pl.part_len;
  p.scale = a->scale != 0.f ? a->scale : 1.f;
  const std::string dt = std::to_string(a->dtype);
  if (pl.whole) return launch(ctx, ("vk_logprob_row_q" + dt).c_str(), dim3((unsigned)a->n_rows), dim3(1024), p, stream);
  rc = launch(ctx, ("vk_logprob_part_q" + dt).c_str(), dim3((unsigned)((uint64_t)a->n_rows * pl.parts)), dim3(256), p, stream);
  if (rc || pl.parts == 1) return rc;
  return launch(ctx, ("vk_logprob_join_q" + dt).c_str(), dim3((unsigned)a->n_rows), dim3(256), p, stream);
}
