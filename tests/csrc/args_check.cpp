// What the checks of arguments answer, without a device: a context and a pool made by hand (their
// sizes alone are read), and the library's own entry points.
//   args_check scale <float>        status of vk_token_logprobs_workspace
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
  return 2;
}
