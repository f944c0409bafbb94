// velokv_sparse.cpp -- host side of sparse decode (include/velokv.h): the key index
// beside a pool, the choice of pages by it, and attention over listed pages. The
// kernels are in velokv_sparse.hip.
#include <cmath>

#include "velokv_internal.h"

using namespace velokv;

struct vk_key_index {
  vk_ctx* ctx = nullptr;
  vk_pool* pool = nullptr;
  uint8_t* base = nullptr;
  uint64_t bytes = 0;
  uint64_t layer_stride = 0, scales_off = 0;  // codes first, then scales
  int8_t* codes(int layer) const { return reinterpret_cast<int8_t*>(base + layer_stride * (uint64_t)layer); }
  float* scales(int layer) const { return reinterpret_cast<float*>(base + layer_stride * (uint64_t)layer + scales_off); }
};

namespace {

constexpr int kMaxGroup = 32;  // two 16-row matrix-core tiles
// The kernels hold an entry's place in an int, up to a workgroup past the list's end
constexpr int kMaxList = 1 << 30;
// HIP takes less than 2^32 threads in a grid
constexpr uint64_t kMaxThreads = (1ull << 32) - 1;

bool narrow(const vk_pool* pool) { return pool->geom.head_dim == 64; }
const char* d64(const vk_pool* pool) { return narrow(pool) ? "_d64" : ""; }
std::string update_name(const vk_pool* pool) { return "vk_index_update_kv" + std::to_string(pool->desc.kv_type) + d64(pool); }
std::string rows_tag(int group, int q_dtype) { return std::string(group > 16 ? "_r2_q" : "_r1_q") + std::to_string(q_dtype); }
std::string select_name(const char* stage, const vk_pool* pool, int group, int q_dtype) {
  return stage + std::string(d64(pool)) + rows_tag(group, q_dtype);
}
std::string sparse_name(const vk_pool* pool, int group, int q_dtype) {
  return "vk_sparse_kv" + std::to_string(pool->desc.kv_type) + d64(pool) + rows_tag(group, q_dtype);
}

int check_index(const vk_ctx* ctx, const vk_key_index* index) {
  if (!ctx) return fail(VK_ERR_NOT_WIRED, "context is null");
  if (!index) return fail(VK_ERR_NOT_WIRED, "key index is null");
  if (index->ctx != ctx) return fail(VK_ERR_BAD_ARG, "key index belongs to another context");
  return VK_OK;
}

// The block table of a call: the caller's, or the pool's slot table.
struct Table { const int32_t* bt; int32_t stride, rows; };
int resolve_table(const vk_pool* pool, const int32_t* block_tables, int32_t bt_stride, int32_t max_context_len, Table* t) {
  *t = Table{block_tables, bt_stride, 0};
  if (!t->bt) {
    if (!pool->table) return fail(VK_ERR_BAD_ARG, "no block table given and the pool has no slot table");
    *t = Table{pool->table, pool->desc.max_pages_per_slot, pool->desc.max_slots};
  }
  if (t->stride <= 0) return fail(VK_ERR_BAD_ARG, "bt_stride must be positive");
  if (max_context_len < 0) return fail(VK_ERR_BAD_ARG, "max_context_len < 0");
  if ((int64_t)max_context_len > (int64_t)t->stride * pool->desc.block_size)
    return fail(VK_ERR_BAD_ARG, "max_context_len %d exceeds the block-table row (%d pages)", max_context_len, t->stride);
  return VK_OK;
}

// How a call runs: the selection's workgroups per (sequence, KV head), the attention's
// parts of a list, and the scratch of each. They follow one another on the stream, so
// a call that does both needs the larger.
struct SparsePlan {
  Table table;
  int group, max_pages, n_chunks, n_splits, split_entries, waves;
  uint64_t units, select_bytes, acc_bytes, ml_bytes;
  uint64_t bytes(bool select, bool attend) const {
    return std::max(select ? select_bytes : 0, attend ? acc_bytes + ml_bytes : 0);
  }
};

int plan_sparse(const vk_ctx* ctx, const vk_pool* pool, const vk_sparse_args* a, SparsePlan* pl) {
  if (!a) return fail(VK_ERR_BAD_ARG, "args is null");
  const vk_pool_desc& d = pool->desc;
  if (a->layer < 0 || a->layer >= d.n_layer) return fail(VK_ERR_BAD_ARG, "layer %d out of range", a->layer);
  if (a->n_seqs < 0 || a->n_heads <= 0) return fail(VK_ERR_BAD_ARG, "bad sizes");
  if (a->n_heads % d.n_kv_heads) return fail(VK_ERR_BAD_ARG, "n_heads %d not a multiple of n_kv_heads %d", a->n_heads, d.n_kv_heads);
  pl->group = a->n_heads / d.n_kv_heads;
  if (pl->group > kMaxGroup) return fail(VK_ERR_UNSUPPORTED, "GQA group size %d (sparse decode supports up to %d)", pl->group, kMaxGroup);
  if (a->q_dtype != VK_DT_F32 && a->q_dtype != VK_DT_F16) return fail(VK_ERR_BAD_ARG, "q_dtype %d", a->q_dtype);
  if (a->n_pages <= 0) return fail(VK_ERR_BAD_ARG, "n_pages must be positive");
  if (a->n_pages > kMaxList) return fail(VK_ERR_UNSUPPORTED, "a list of %d pages (up to %d)", a->n_pages, kMaxList);
  if (a->n_first < 0 || a->n_last < 0 || (int64_t)a->n_first + a->n_last > a->n_pages)
    return fail(VK_ERR_BAD_ARG, "n_first %d and n_last %d do not fit a list of %d pages", a->n_first, a->n_last, a->n_pages);
  if (int rc = resolve_table(pool, a->block_tables, a->bt_stride, a->max_context_len, &pl->table)) return rc;
  pl->units = (uint64_t)a->n_seqs * d.n_kv_heads;
  pl->max_pages = (int)(((int64_t)a->max_context_len + d.block_size - 1) / d.block_size);
  const int64_t units = std::max<int64_t>(1, (int64_t)pl->units);
  // selection: one workgroup per (sequence, KV head), or several and a second launch past 2048
  // pages of few of them. One launch against two, us: 8 of 1024 pages 9.3 and 11.8, of 2048 13.9
  // and 12.8, of 4096 22.4 and 15.0, of 8125 38.8 and 19.6; 32 of 2560 17.2 and 14.0, of 8125
  // 48.2 and 27.2; 128 of 2560 22.5 and 28.1, of 8125 70.6 and 62.1. Between the two (64 of 4096:
  // 28.2 and 22.1, of 8125: 50.4 and 38.0) the rule takes the slower
  pl->n_chunks = 0;
  pl->select_bytes = 0;
  if (pl->max_pages > kSelPages || (pl->max_pages > 2048 && 8 * units <= ctx->n_cu)) {
    constexpr int kChunk = 64 * kSelWaves;
    pl->n_chunks = (int)std::max<int64_t>(1, std::min<int64_t>((2 * ctx->n_cu + units - 1) / units, (pl->max_pages + kChunk - 1) / kChunk));
    pl->select_bytes = align_up(pl->units * pl->max_pages * sizeof(uint32_t), 256);
  }
  // attention: eight waves a CU (more do not fit beside their registers), in one workgroup
  // per (sequence, KV head) where there are as many as CUs, in parts of the list else. Two of
  // four waves a CU where there are twice as many (512 fp16: 43.9 us, 46.7 with eight waves
  // each; 256 int8: 26.2 with eight, 26.5 with four). At most a part a CU (64 of up to 50
  // pages, fp32: 17.8 us, 23.6 with two), of a tile a wave at least (32 of 64 pages: 10.0 us,
  // 11.9 with two tiles)
  const int pt = pool->geom.page_tiles, cus = ctx->n_cu;
  pl->waves = units >= 2 * cus || pl->group > 16 ? 4 : 8;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(cus / units, (int64_t)a->n_pages * pt / 8));
  const int64_t entries = (a->n_pages + parts - 1) / parts;
  pl->split_entries = (int)std::min<int64_t>(entries, kSparseEntries);
  pl->n_splits = (a->n_pages + pl->split_entries - 1) / pl->split_entries;
  pl->acc_bytes = pl->ml_bytes = 0;
  if (pl->n_splits > 1) {
    const uint64_t rows = (uint64_t)a->n_seqs * a->n_heads * pl->n_splits;
    pl->acc_bytes = align_up(rows * pool->geom.head_dim * sizeof(float), 256);
    pl->ml_bytes = align_up(rows * 2 * sizeof(float), 256);
  }
  const uint64_t rows = ((uint64_t)a->n_seqs * a->n_heads + 3) / 4;
  if (std::max({pl->units * std::max(2, pl->n_chunks) * 64 * kSelWaves, pl->units * pl->n_splits * 64 * pl->waves, rows * 256}) > kMaxThreads)
    return fail(VK_ERR_UNSUPPORTED, "grid too large");
  return VK_OK;
}

int run_select(vk_ctx* ctx, vk_key_index* index, const vk_sparse_args* a, const SparsePlan& pl, uint8_t* ws, void* stream) {
  const vk_pool* pool = index->pool;
  SelectParams p{};
  p.codes = index->codes(a->layer);
  p.scales = index->scales(a->layer);
  p.q = a->q;
  p.pages = a->pages;
  p.keys = reinterpret_cast<uint32_t*>(ws);
  p.block_tables = pl.table.bt;
  p.bt_stride = pl.table.stride;
  p.bt_rows = pl.table.rows;
  p.seq_rows = a->seq_rows;
  p.context_lens = a->context_lens;
  p.err = ctx->err_word;
  p.n_seqs = a->n_seqs;
  p.n_heads = a->n_heads;
  p.n_kv_heads = pool->desc.n_kv_heads;
  p.n_pool_pages = pool->desc.n_blocks;
  p.page_tokens = pool->desc.block_size;
  p.cap_tokens = a->max_context_len;
  p.max_pages = pl.max_pages;
  p.n_list = a->n_pages;
  p.n_first = a->n_first;
  p.n_last = a->n_last;
  p.io_hd = pool->geom.io_hd;
  p.n_chunks = pl.n_chunks;
  const dim3 threads(64 * kSelWaves), wide(64 * kSelMaxWaves), units((unsigned)pl.units);
  if (!pl.n_chunks) {
    // by rows where the workgroups are fewer than the CUs (velokv_sparse.hip, PageTurn)
    const char* stage = pl.units < (uint64_t)ctx->n_cu ? "vk_page_select_rows" : "vk_page_select";
    return launch(ctx, select_name(stage, pool, pl.group, a->q_dtype).c_str(), units, threads, p, stream);
  }
  if (int rc = launch(ctx, select_name("vk_page_scores", pool, pl.group, a->q_dtype).c_str(),
                      dim3((unsigned)(pl.units * pl.n_chunks)), threads, p, stream))
    return rc;
  return launch(ctx, "vk_page_topk", units, wide, p, stream);
}

int run_attend(vk_ctx* ctx, vk_pool* pool, const vk_sparse_args* a, const SparsePlan& pl, uint8_t* ws, void* stream) {
  const PoolGeom& g = pool->geom;
  const uint8_t* L = pool->base + g.layer_stride * (uint64_t)a->layer;
  SparseParams p{};
  p.kc = L + g.k_off;
  p.vc = L + g.v_off;
  p.ks = g.stile_bytes ? L + g.ks_off : nullptr;
  p.vs = g.stile_bytes ? L + g.vs_off : nullptr;
  p.q = a->q;
  p.out = a->out;
  p.pages = a->pages;
  p.part_acc = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + pl.acc_bytes);
  p.block_tables = pl.table.bt;
  p.bt_stride = pl.table.stride;
  p.bt_rows = pl.table.rows;
  p.seq_rows = a->seq_rows;
  p.context_lens = a->context_lens;
  p.err = ctx->err_word;
  p.tile_bytes = g.tile_bytes;
  p.stile_bytes = g.stile_bytes;
  p.n_seqs = a->n_seqs;
  p.n_heads = a->n_heads;
  p.n_kv_heads = pool->desc.n_kv_heads;
  p.n_pages = pool->desc.n_blocks;
  p.page_tiles = g.page_tiles;
  p.cap_tokens = a->max_context_len;
  p.n_list = a->n_pages;
  p.io_hd = g.io_hd;
  p.n_splits = pl.n_splits;
  p.split_entries = pl.split_entries;
  p.scale_log2 = (a->scale != 0.f ? a->scale : 1.0f / std::sqrt((float)pool->desc.head_dim)) * 1.4426950408889634f;
  int rc = launch(ctx, sparse_name(pool, pl.group, a->q_dtype).c_str(), dim3((unsigned)(pl.units * pl.n_splits)),
                  dim3(64 * (unsigned)pl.waves), p, stream);
  if (rc || pl.n_splits == 1) return rc;
  const uint64_t rows = (uint64_t)a->n_seqs * a->n_heads;
  return launch(ctx, (std::string("vk_sparse_merge") + d64(pool)).c_str(), dim3((unsigned)((rows + 3) / 4)), dim3(256), p, stream);
}

// Selection (with an index), attention (with a pool), or both, in that order.
int run_sparse(vk_ctx* ctx, vk_key_index* index, vk_pool* pool, const vk_sparse_args* a, bool attend, void* stream) {
  SparsePlan pl;
  int rc = plan_sparse(ctx, pool, a, &pl);
  if (rc) return rc;
  if (a->n_seqs == 0) return VK_OK;
  if (!a->q || !a->pages || !a->context_lens || (attend && !a->out)) return fail(VK_ERR_BAD_ARG, "null device pointer");
  if ((rc = set_device(ctx))) return rc;
  const uint64_t need = pl.bytes(index != nullptr, attend);
  uint8_t* ws = nullptr;
  if (need) {
    if (!a->workspace && !scratch_at_hand(ctx, nullptr, 0, need, stream))
      return fail(VK_ERR_BAD_ARG, "a captured call needs %llu bytes of scratch: give it a workspace", (unsigned long long)need);
    if ((rc = split_workspace(ctx, a->workspace, a->workspace_bytes, need, &ws))) return rc;
  }
  if (index && (rc = run_select(ctx, index, a, pl, ws, stream))) return rc;
  return attend ? run_attend(ctx, pool, a, pl, ws, stream) : VK_OK;
}

}  // namespace

std::vector<std::string> velokv::sparse_kernel_names() {
  std::vector<std::string> names = {"vk_index_read", "vk_page_topk", "vk_sparse_merge", "vk_sparse_merge_d64"};
  for (const char* w : {"", "_d64"}) {
    for (int kv = 0; kv < 4; ++kv) names.push_back("vk_index_update_kv" + std::to_string(kv) + w);
    for (int group : {16, 32})
      for (int qt : {VK_DT_F32, VK_DT_F16}) {
        for (const char* stage : {"vk_page_select", "vk_page_select_rows", "vk_page_scores"}) names.push_back(stage + std::string(w) + rows_tag(group, qt));
        for (int kv = 0; kv < 4; ++kv) names.push_back("vk_sparse_kv" + std::to_string(kv) + w + rows_tag(group, qt));
      }
  }
  return names;
}

extern "C" int vk_index_create(vk_ctx* ctx, vk_pool* pool, vk_key_index** out) {
  int rc = check_pool(ctx, pool);
  if (rc) return rc;
  if (!out) return fail(VK_ERR_BAD_ARG, "out is null");
  *out = nullptr;
  if ((rc = set_device(ctx))) return rc;
  const uint64_t rows = (uint64_t)pool->desc.n_blocks * pool->desc.n_kv_heads;
  auto* x = new vk_key_index();
  x->ctx = ctx;
  x->pool = pool;
  x->scales_off = align_up(rows * 2 * pool->geom.head_dim, 256);
  x->layer_stride = x->scales_off + align_up(rows * sizeof(float), 256);
  x->bytes = x->layer_stride * (uint64_t)pool->desc.n_layer;
  hipError_t e = hipMalloc(reinterpret_cast<void**>(&x->base), x->bytes);
  if (e != hipSuccess) {
    const uint64_t bytes = x->bytes;
    delete x;
    return fail(VK_ERR_HIP, "hipMalloc of %.3f GB for the key index failed: %s", bytes / 1e9, hipGetErrorString(e));
  }
  e = hipMemset(x->base, 0, x->bytes);
  if (e == hipSuccess) e = hipDeviceSynchronize();
  if (e != hipSuccess) {
    hipFree(x->base);
    delete x;
    return fail(VK_ERR_HIP, "key index initialisation failed: %s", hipGetErrorString(e));
  }
  *out = x;
  return VK_OK;
}

extern "C" int vk_index_destroy(vk_key_index* index) {
  if (!index) return VK_OK;
  hipSetDevice(index->ctx->device);
  hipDeviceSynchronize();
  hipFree(index->base);
  delete index;
  return VK_OK;
}

extern "C" int vk_index_bytes(const vk_key_index* index, uint64_t* out) {
  if (!index || !out) return fail(VK_ERR_BAD_ARG, "null argument");
  *out = index->bytes;
  return VK_OK;
}

extern "C" int vk_index_update(vk_ctx* ctx, vk_key_index* index, int32_t layer, const int32_t* block_tables, int32_t bt_stride,
                               const int32_t* seq_rows, const int32_t* first_tokens, const int32_t* context_lens, int32_t n_seqs,
                               int32_t max_context_len, int32_t max_tokens, void* stream) {
  int rc = check_index(ctx, index);
  if (rc) return rc;
  const vk_pool* pool = index->pool;
  if (layer < 0 || layer >= pool->desc.n_layer) return fail(VK_ERR_BAD_ARG, "layer %d out of range", layer);
  if (n_seqs < 0) return fail(VK_ERR_BAD_ARG, "n_seqs < 0");
  if (max_tokens < 0) return fail(VK_ERR_BAD_ARG, "max_tokens < 0");
  Table t;
  if ((rc = resolve_table(pool, block_tables, bt_stride, max_context_len, &t))) return rc;
  if (n_seqs == 0 || max_context_len == 0) return VK_OK;
  if (!context_lens) return fail(VK_ERR_BAD_ARG, "null device pointer");
  if ((rc = set_device(ctx))) return rc;
  const PoolGeom& g = pool->geom;
  const uint8_t* L = pool->base + g.layer_stride * (uint64_t)layer;
  IndexUpdateParams p{};
  p.kc = L + g.k_off;
  p.ks = g.stile_bytes ? L + g.ks_off : nullptr;
  p.codes = index->codes(layer);
  p.scales = index->scales(layer);
  p.block_tables = t.bt;
  p.bt_stride = t.stride;
  p.bt_rows = t.rows;
  p.seq_rows = seq_rows;
  p.first_tokens = first_tokens;
  p.context_lens = context_lens;
  p.err = ctx->err_word;
  p.tile_bytes = g.tile_bytes;
  p.stile_bytes = g.stile_bytes;
  p.n_seqs = n_seqs;
  p.n_kv_heads = pool->desc.n_kv_heads;
  p.n_pages = pool->desc.n_blocks;
  p.page_tiles = g.page_tiles;
  p.cap_tokens = max_context_len;
  // n tokens in a row touch at most (n + page - 2) / page + 1 pages
  const int64_t bs = pool->desc.block_size, all = (max_context_len + bs - 1) / bs;
  p.max_pages = (int32_t)(first_tokens && max_tokens > 0 ? std::min(all, (max_tokens + bs - 2) / bs + 1) : all);
  constexpr int kWaves = 4;
  constexpr int64_t kMaxWgs = 1 << 23;  // launches of less than 2^32 threads
  const std::string name = update_name(pool);
  const int64_t units = (int64_t)p.max_pages * p.n_kv_heads, seq_wgs = (units + kWaves - 1) / kWaves, wgs = seq_wgs * n_seqs;
  if (units > 0x7FFFFFFF - kWaves || wgs > 0x7FFFFFFF) return fail(VK_ERR_UNSUPPORTED, "grid too large");
  p.seq_wgs = (int32_t)seq_wgs;
  for (int64_t w = 0; w < wgs; w += kMaxWgs) {
    p.wg0 = (int32_t)w;
    if ((rc = launch(ctx, name.c_str(), dim3((unsigned)std::min(kMaxWgs, wgs - w)), dim3(64 * kWaves), p, stream))) return rc;
  }
  return VK_OK;
}

extern "C" int vk_index_read(vk_ctx* ctx, vk_key_index* index, int32_t layer, const int32_t* pages, int32_t n_pages, float* lower,
                             float* upper, void* stream) {
  int rc = check_index(ctx, index);
  if (rc) return rc;
  const vk_pool* pool = index->pool;
  if (layer < 0 || layer >= pool->desc.n_layer) return fail(VK_ERR_BAD_ARG, "layer %d out of range", layer);
  if (n_pages < 0) return fail(VK_ERR_BAD_ARG, "n_pages < 0");
  if (n_pages == 0) return VK_OK;
  if (!pages || !lower || !upper) return fail(VK_ERR_BAD_ARG, "null device pointer");
  if ((reinterpret_cast<uintptr_t>(lower) | reinterpret_cast<uintptr_t>(upper)) & 15)
    return fail(VK_ERR_BAD_ARG, "lower and upper must be 16-byte aligned");
  if ((rc = set_device(ctx))) return rc;
  IndexReadParams p{};
  p.codes = index->codes(layer);
  p.scales = index->scales(layer);
  p.pages = pages;
  p.lower = lower;
  p.upper = upper;
  p.err = ctx->err_word;
  p.n_kv_heads = pool->desc.n_kv_heads;
  p.n_pages = pool->desc.n_blocks;
  p.io_hd = pool->geom.io_hd;
  p.tile_hd = pool->geom.head_dim;
  const uint64_t chunks = (uint64_t)n_pages * p.n_kv_heads * (p.io_hd / 4);
  if (chunks > kMaxThreads - 255) return fail(VK_ERR_UNSUPPORTED, "grid too large");
  p.n_chunks = (uint32_t)chunks;
  return launch(ctx, "vk_index_read", dim3((unsigned)((chunks + 255) / 256)), dim3(256), p, stream);
}

extern "C" int vk_sparse_workspace(const vk_pool* pool, const vk_sparse_args* a, uint64_t* bytes) {
  if (!pool || !bytes) return fail(VK_ERR_BAD_ARG, "null argument");
  SparsePlan pl;
  if (int rc = plan_sparse(pool->ctx, pool, a, &pl)) return rc;
  *bytes = pl.bytes(true, true);
  return VK_OK;
}

extern "C" int vk_select_pages(vk_ctx* ctx, vk_key_index* index, const vk_sparse_args* a, void* stream) {
  const int rc = check_index(ctx, index);
  return rc ? rc : run_sparse(ctx, index, index->pool, a, false, stream);
}

extern "C" int vk_sparse_decode(vk_ctx* ctx, vk_pool* pool, const vk_sparse_args* a, void* stream) {
  const int rc = check_pool(ctx, pool);
  return rc ? rc : run_sparse(ctx, nullptr, pool, a, true, stream);
}

extern "C" int vk_select_decode(vk_ctx* ctx, vk_key_index* index, const vk_sparse_args* a, void* stream) {
  const int rc = check_index(ctx, index);
  return rc ? rc : run_sparse(ctx, index, index->pool, a, true, stream);
}
