// What the checks of arguments answer, without a device: a context and a pool made by hand (their
// sizes alone are read), and the library's own entry points.
//   args_check scale <float>        status of vk_token_logprobs_workspace
//   args_check list <n_pages> <n_last> <context>  status of vk_sparse_workspace, one sequence and head
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "velokv_internal.h"

int main(int argc, char** argv) {
  if (argc < 3) return 2;
  vk_ctx ctx;
  uint64_t bytes = 0;
  if (!strcmp(argv[1], "scale")) {
    vk_logprob_args a{};
    a.n_rows = 2;
    a.vocab = 100000;
    a.n_top = 3;
    a.scale = strtof(argv[2], nullptr);
    const int rc = vk_token_logprobs_workspace(&ctx, &a, &bytes);
    printf("%d %llu %s\n", rc, (unsigned long long)bytes, rc ? vk_last_error() : "");
    return 0;
  }
  if (!strcmp(argv[1], "list") && argc == 5) {
    vk_pool pool;
    pool.ctx = &ctx;
    pool.desc = vk_pool_desc{1, 64, 16, 1, 128, VK_KV_F16, 0, 0};
    pool.geom.page_tiles = 1;
    pool.geom.head_dim = pool.geom.io_hd = 128;
    const int32_t table = 0;
    vk_sparse_args a{};
    a.n_seqs = a.n_heads = 1;
    a.n_pages = atoi(argv[2]);
    a.n_last = atoi(argv[3]);
    a.max_context_len = atoi(argv[4]);
    a.block_tables = &table;
    a.bt_stride = 1 << 27;
    const int rc = vk_sparse_workspace(&pool, &a, &bytes);
    printf("%d %llu %s\n", rc, (unsigned long long)bytes, rc ? vk_last_error() : "");
    return 0;
  }
  return 2;
}
