#include "waits.h"

#include <atomic>
#include <cstring>

#include "internal.h"
#include "pdl.cuh"

namespace csw {
namespace {

constexpr int kMaxDevices = 64;
uint32_t* status_words() {
  static uint32_t* const words = [] {
    // also while a stream is captured: the allocation has nothing to do with it
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    void* p = nullptr;
    if (taken(cudaThreadExchangeStreamCaptureMode(&mode)) != cudaSuccess) return (uint32_t*)nullptr;
    const size_t bytes = kMaxDevices * sizeof(uint32_t);
    const cudaError_t e = taken(cudaHostAlloc(&p, bytes, cudaHostAllocPortable | cudaHostAllocMapped));
    taken(cudaThreadExchangeStreamCaptureMode(&mode));
    if (e != cudaSuccess) return (uint32_t*)nullptr;
    return (uint32_t*)std::memset(p, 0, bytes);
  }();
  return words;
}
std::atomic<long long> limit{1ll << 32};  // some two seconds

const bool registered = (take_kernel_status = take_status, true);

}  // namespace

cudaError_t status_word(uint32_t** word) {
  int dev = 0;
  if (const cudaError_t e = taken(cudaGetDevice(&dev))) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  uint32_t* words = status_words();
  *word = words + dev;
  return words ? cudaSuccess : cudaErrorMemoryAllocation;
}

cudaError_t take_status(int* gave_up) {
  uint32_t* word;
  const cudaError_t e = status_word(&word);
  if (e == cudaSuccess) *gave_up = (int)__atomic_exchange_n(word, 0u, __ATOMIC_RELAXED);
  return e;
}

long long wait_limit() { return limit.load(std::memory_order_relaxed); }
void set_wait_limit(long long clocks) { limit.store(clocks, std::memory_order_relaxed); }

TileEncoder tile_encoder() {
  static const TileEncoder f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (taken(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r)) != cudaSuccess)
      return TileEncoder();
    return r == cudaDriverEntryPointSuccess ? reinterpret_cast<TileEncoder>(p) : TileEncoder();
  }();
  return f;
}

cudaError_t bind_context() {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  return taken(e == cudaSuccess ? cudaSetDevice(dev) : e);
}

}  // namespace csw
