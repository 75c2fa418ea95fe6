#include "device_error.h"

#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

namespace nvb {
namespace {
std::atomic<int*> g_word{nullptr};
}

int* device_error_word() {
  int* w = g_word.load(std::memory_order_acquire);
  if (w) return w;
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  if ((w = g_word.load(std::memory_order_acquire))) return w;
  // the first call may lie inside a stream capture, which this allocation does not concern
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
  void* m = nullptr;
  const cudaError_t e = cudaHostAlloc(&m, sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  w = static_cast<int*>(m);
  *w = 0;
  g_word.store(w, std::memory_order_release);
  return w;
}

int device_error_code(int reset) {
  int* w = g_word.load(std::memory_order_acquire);
  if (!w) return 0;  // no such kernel was ever launched
  return reset ? __atomic_exchange_n(w, 0, __ATOMIC_ACQ_REL) : __atomic_load_n(w, __ATOMIC_ACQUIRE);
}

}  // namespace nvb
