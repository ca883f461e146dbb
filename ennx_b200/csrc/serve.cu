// serve.cu -- host side shared by the serving operators: the rotary table and
// the status word of their bounded waits.
#include "serve.cuh"

#include <math.h>

#include <mutex>

namespace ennx {

const RopeTable& rope_table(float theta) {
  static thread_local RopeTable t;
  static thread_local float of = -1.0f;
  if (of != theta) {
    for (int i = 0; i < 64; ++i) t.inv[i] = pow((double)theta, -2.0 * i / 128.0) / 6.283185307179586476925;
    of = theta;
  }
  return t;
}

namespace {
__device__ int g_serving_status;
struct Word {
  std::once_flag once;
  int* address = nullptr;
};
Word g_word[kMaxServingDevices];
}  // namespace

int32_t serving_device(int* device, int** status) {
  int dev = 0;
  ENNX_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev < 0 || dev >= kMaxServingDevices) return set_error(ENNX_B200_UNSUPPORTED, "device index %d out of range", dev);
  Word& w = g_word[dev];
  cudaError_t e = cudaSuccess;
  std::call_once(w.once, [&] {
    void* p = nullptr;
    e = cudaGetSymbolAddress(&p, g_serving_status);
    if (e != cudaSuccess) return;
    w.address = (int*)p;
    register_status_word(dev, w.address);
  });
  if (!w.address) return check_cuda(e, "serving status word");
  *device = dev;
  *status = w.address;
  return ENNX_B200_OK;
}

int32_t allow_shared_memory(std::once_flag& once, int32_t& result, const void* kernel, int bytes) {
  std::call_once(once, [&] {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    result = e == cudaSuccess ? ENNX_B200_OK : check_cuda(e, "shared memory of a serving kernel");
  });
  return result;
}

}  // namespace ennx
