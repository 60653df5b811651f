// Shared definitions for the cascade_b200 CUDA library (sm_100a only).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <string>

#include "cascade_b200.h"

namespace cb {

// Thread-local last-error text behind cascade_last_error().
void set_error(const std::string &msg);
void clear_error();
const char *last_error();

// Kernel launches made by this library since load (cascade_diag_launch_count).
void count_launches(int k);

// Records `what` + the CUDA error text and returns CASCADE_ERR_CUDA.
int cuda_fail(cudaError_t e, const char *what);

#define CB_CUDA(call)                                                         \
  do {                                                                        \
    cudaError_t _e = (call);                                                  \
    if (_e != cudaSuccess) return ::cb::cuda_fail(_e, #call);                 \
  } while (0)

#define CB_CHECK(cond, code, msg)                                             \
  do {                                                                        \
    if (!(cond)) {                                                            \
      ::cb::set_error(msg);                                                   \
      return (code);                                                          \
    }                                                                         \
  } while (0)

// Streaming multiprocessors of the current device (148 on a B200), read
// from the device once per device and cached.
int sm_count();

// True the first time it is called with `done` on each device: for
// attributes of a kernel that hold for the life of the process.  (Setting
// them twice, as two threads' first calls may, does no harm.)
class OncePerDevice {
 public:
  bool pending() {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 63;
    bit_ = 1ull << dev;
    return !(done_->load(std::memory_order_acquire) & bit_);
  }
  void set() { done_->fetch_or(bit_, std::memory_order_release); }
  explicit OncePerDevice(std::atomic<uint64_t> *done) : done_(done) {}

 private:
  std::atomic<uint64_t> *done_;
  uint64_t bit_ = 0;
};

// Launches `kernel` so that its blocks may start while the kernel before it
// on the stream still runs; it calls wait_for_previous() before it touches
// anything that one writes.
template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, dim3 block,
                         size_t smem, cudaStream_t s, const Args &...args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

#ifdef __CUDACC__
// The kernel before this one on the stream has finished, its writes visible.
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// A kernel launched by launch_early behind this one may start.
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
#endif

// Grid size for a grid-stride kernel: a multiple of the SM count.
inline int grid_for(uint64_t work_items, int per_block, int blocks_per_sm) {
  uint64_t want = (work_items + per_block - 1) / per_block;
  uint64_t cap = (uint64_t)sm_count() * blocks_per_sm;
  if (want > cap) want = cap;
  if (want < 1) want = 1;
  return (int)want;
}

__host__ __device__ inline uint64_t div_up(uint64_t a, uint64_t b) {
  return (a + b - 1) / b;
}

}  // namespace cb
