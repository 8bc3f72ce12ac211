// Conformance probe for the GPU tests (built into tests/libjeeves_fp8_testhooks.so,
// never shipped with the product library), over the same device function as the
// product kernels (layer.h):
//   * th_inverse_sweep: every fp32 bit pattern in a range through the
//     convolution's and the gates' reciprocal, counting those that are not the
//     IEEE quotient's bits.
#include <stdint.h>

#include "layer.h"

namespace {

__global__ void inverse_sweep_kernel(uint32_t start, uint32_t n, unsigned long long* count) {
  unsigned long long c = 0;
  for (uint64_t i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
    const float d = __uint_as_float(start + (uint32_t)i);
    c += __float_as_uint(jv::inverse(d)) != __float_as_uint(1.0f / d);
  }
  atomicAdd(count, c);
}

}  // namespace

extern "C" int th_inverse_sweep(uint32_t start, uint32_t n, unsigned long long* count, void* stream) {
  inverse_sweep_kernel<<<2048, 256, 0, (hipStream_t)stream>>>(start, n, count);
  return (int)hipGetLastError();
}
