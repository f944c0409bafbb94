// What the translation units of libvelokv.so share: the context and the pool behind
// the C ABI's handles, errors, launches and scratch. Host code only.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <string>
#include <unordered_map>
#include <vector>

#include "velokv.h"
#include "velokv_params.h"
#include "velokv_plan.h"

namespace velokv {
// Sets the calling thread's vk_last_error() message and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
}  // namespace velokv

#define HIP_TRY(expr)                                                              \
  do {                                                                             \
    hipError_t _e = (expr);                                                        \
    if (_e != hipSuccess)                                                          \
      return velokv::fail(VK_ERR_HIP, "%s failed: %s", #expr, hipGetErrorString(_e));     \
  } while (0)

struct vk_ctx {
  int device = 0;
  std::string arch;
  std::vector<hipModule_t> modules;  // the code objects
  std::unordered_map<std::string, hipFunction_t> fns;
  // threads per workgroup each kernel was compiled for (__launch_bounds__), read
  // once at vk_ctx_create: a launch with more faults the device, so launch()
  // refuses it
  std::unordered_map<std::string, int> max_threads;
  std::unordered_map<std::string, std::string> unloaded;  // kernels of a code object that did not load: why
  std::mutex ws_mu;
  void* ws = nullptr;
  uint64_t ws_bytes = 0;
  // Buffers the context's workspace outgrew: a call on another host thread may
  // still have kernels queued that use one, so they are freed only by
  // vk_ctx_destroy (growth is rare: once per new largest shape).
  std::vector<void*> ws_retired;
  uint32_t* err_word = nullptr;  // device: misuse flags (VK_MISUSE_*) or-ed by the kernels
  int decode_kind = VK_DECODE_AUTO;
  int decode_sched = VK_SCHED_AUTO;
  int n_cu = 256;
  std::mutex res_mu;                                   // guards resident, wg_resident
  std::unordered_map<std::string, int64_t> resident;  // kernel -> resident waves
  std::unordered_map<std::string, velokv::WgResident> wg_resident;

  hipFunction_t fn(const std::string& name) const {
    auto it = fns.find(name);
    return it == fns.end() ? nullptr : it->second;
  }
};

struct vk_pool {
  vk_ctx* ctx = nullptr;
  vk_pool_desc desc{};
  velokv::PoolGeom geom{};
  uint8_t* base = nullptr;
  uint64_t bytes = 0;
  int32_t* table = nullptr;  // [max_slots][max_pages_per_slot]
  uint64_t table_bytes = 0;
  // I8_BLK: per block, (epoch << 32 | first token) of the last append run on it,
  // so that a call with two runs on one block is reported (VK_MISUSE_BLK_SPLIT_RUN)
  unsigned long long* claim = nullptr;
  std::atomic<uint32_t> epoch{0};
  uint32_t next_epoch() {
    uint32_t e = ++epoch;
    while (e == 0) e = ++epoch;  // 0 marks a never-claimed block
    return e;
  }
};

namespace velokv {

inline uint64_t align_up(uint64_t x, uint64_t a) { return (x + a - 1) / a * a; }

inline int set_device(const vk_ctx* ctx) {
  HIP_TRY(hipSetDevice(ctx->device));
  return VK_OK;
}

// A kernel that the context does not have.
inline int no_kernel(const vk_ctx* ctx, const char* name) {
  auto it = ctx->unloaded.find(name);
  if (it != ctx->unloaded.end()) return fail(VK_ERR_NOT_WIRED, "kernel %s: %s", name, it->second.c_str());
  return fail(VK_ERR_NOT_WIRED, "kernel %s is not in the code object", name);
}

// A workgroup shape the kernel was compiled for: at least one thread and at most
// its __launch_bounds__ (HIP_FUNC_ATTRIBUTE_MAX_THREADS_PER_BLOCK).
inline int check_launch_shape(const vk_ctx* ctx, const char* name, uint64_t threads) {
  auto it = ctx->max_threads.find(name);
  if (it == ctx->max_threads.end()) return no_kernel(ctx, name);
  if (threads == 0 || threads > (uint64_t)it->second)
    return fail(VK_ERR_BAD_ARG, "kernel %s launched with %llu threads per workgroup; it was compiled for at most %d",
                name, (unsigned long long)threads, it->second);
  return VK_OK;
}

template <typename P>
int launch(const vk_ctx* ctx, const char* name, dim3 grid, dim3 block, const P& params, void* stream) {
  hipFunction_t f = ctx->fn(name);
  if (!f) return no_kernel(ctx, name);
  int rc = check_launch_shape(ctx, name, (uint64_t)block.x * block.y * block.z);
  if (rc) return rc;
  void* args[] = {const_cast<P*>(&params)};
  HIP_TRY(hipModuleLaunchKernel(f, grid.x, grid.y, grid.z, block.x, block.y, block.z, 0,
                                reinterpret_cast<hipStream_t>(stream), args, nullptr));
  return VK_OK;
}

inline int check_pool(const vk_ctx* ctx, const vk_pool* pool) {
  if (!ctx) return fail(VK_ERR_NOT_WIRED, "context is null");
  if (!pool) return fail(VK_ERR_NOT_WIRED, "pool is null");
  if (pool->ctx != ctx) return fail(VK_ERR_BAD_ARG, "pool belongs to another context");
  return VK_OK;
}

// Split-K workspace: the caller's buffer when given (and large enough), else the
// context's own, grown on demand.
int split_workspace(vk_ctx* ctx, void* given, uint64_t given_bytes, uint64_t need, uint8_t** out);

// Whether a call can have `need` bytes of scratch: in the buffer given, or in the
// context's own, which may grow unless the stream is being captured.
bool scratch_at_hand(vk_ctx* ctx, const void* given, uint64_t given_bytes, uint64_t need, void* stream);

// The kernels of the code objects beside the main one (velokv_sparse.cpp, velokv_logits.cpp).
std::vector<std::string> sparse_kernel_names();
std::vector<std::string> logits_kernel_names();

}  // namespace velokv
