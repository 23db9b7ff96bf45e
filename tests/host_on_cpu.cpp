// The host module of the dense operators (csrc/host_ext.cpp) for CPU tensors:
// the same source with the queries of GPU, stream and allocator replaced and
// entries that count their calls in the library's place, so that its checks,
// locking and errors run where there is no GPU.
#include <Python.h>

#include <ATen/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "fgs_moe.h"

extern "C" {
int host_test_gpu = 0;      // the current GPU
int host_test_calls = 0;    // calls that reached an entry
int host_test_locked = 0;   // ... with the interpreter's lock held
int host_test_rc = 0;       // what an entry returns
}

namespace c10::hip {
inline DeviceIndex test_current_device() { return static_cast<DeviceIndex>(host_test_gpu); }
inline void test_set_device(DeviceIndex d) { host_test_gpu = d; }
inline int test_SetDevice(DeviceIndex d) { return host_test_gpu = d, 0; }
struct TestStream {
  void* stream() const { return nullptr; }
};
inline TestStream test_stream(DeviceIndex) { return {}; }
}  // namespace c10::hip
namespace at::detail {
inline TensorBase test_empty(IntArrayRef shape, ScalarType type, Device, std::nullopt_t) {
  return empty_cpu(shape, type);
}
}  // namespace at::detail

#define is_cuda is_cpu
#define empty_cuda test_empty
#define current_device test_current_device
#define set_device test_set_device
#define SetDevice test_SetDevice
#define getCurrentHIPStreamMasqueradingAsCUDA test_stream
#include "host_ext.cpp"

static int32_t entered() {
  ++host_test_calls;
  host_test_locked += PyGILState_Check();
  return host_test_rc;
}
extern "C" {
const char* host_test_last_error(void) { return "the entry's text"; }
int32_t host_test_rms_norm(const void*, int64_t, const void*, int64_t, const void*, int32_t, int32_t,
                           float, float, int64_t, int64_t, void*, void*, int64_t, int32_t, void*,
                           float*, int64_t, int64_t, void*) {
  return entered();
}
int32_t host_test_silu_and_mul_quant(const void*, int64_t, int32_t, int64_t, int64_t, int32_t,
                                     int32_t, void*, float*, int64_t, int64_t, void*) {
  return entered();
}
int32_t host_test_fp8_block_matmul(const void*, int64_t, const float*, int64_t, int64_t,
                                   const void*, int64_t, const float*, const void*, int32_t,
                                   int64_t, int64_t, int64_t, int32_t, int32_t, void*, int64_t,
                                   void*) {
  return entered();
}
}
