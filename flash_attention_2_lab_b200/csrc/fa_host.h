// Host-side services that the translation units of libfa_sm100 share: the
// per-thread error message, the state of the current device, and the in-kernel
// wait limit.  Defined in fa_fwd_sm100.cu.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#define FA_HIDDEN __attribute__((visibility("hidden")))

namespace fa {
namespace host {

// Sets fa_last_error() of the calling thread and returns `code`.
FA_HIDDEN int set_error(int code, const char* fmt, ...);

struct Device {
  int index = 0;
  int sms = 0;                     // streaming multiprocessors
  unsigned int* status = nullptr;  // the device status word (fa_read_status)
};

// The current device, checked to be sm_100; FA_OK or an error code.
FA_HIDDEN int current_device(Device* out);

// Lets a kernel have that much dynamic shared memory, always the same amount: set
// once per device, which `done` (a bit each) remembers.
inline cudaError_t allow_smem(const void* kernel, int bytes, int device, std::atomic<uint64_t>& done) {
  const uint64_t bit = 1ull << (device & 63);
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// Limit of every in-kernel wait (fa_set_wait_limit_ns).
FA_HIDDEN unsigned long long wait_limit_ns();

// 128-byte-swizzled tiled map over a 16-bit tensor [slices][rows][dim], dense,
// read in boxes of box_rows x 64 elements.
FA_HIDDEN int encode_rows_map(CUtensorMap* map, const void* ptr, bool bf16, int64_t dim, int64_t rows,
                              int64_t slices, uint32_t box_rows);

}  // namespace host
}  // namespace fa
