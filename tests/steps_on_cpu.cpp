// The host module for CPU tensors (host_on_cpu.cpp) with entries of the routed
// layer's steps that count their calls too.
#include "host_on_cpu.cpp"

extern "C" {
int64_t host_test_permute_workspace_bytes(int64_t numel, int32_t) { return 3 * numel * 4 + 256; }
int32_t host_test_permute(const void*, int64_t, int64_t, int64_t, const int32_t*, int32_t, int32_t,
                          void*, int32_t*, int32_t*, int32_t*, void*, int64_t, void*) {
  return entered();
}
int32_t host_test_permute_rows(const void*, int64_t, int64_t, int64_t, const int32_t*, int32_t,
                               const int32_t*, void*, void*) {
  return entered();
}
int32_t host_test_unpermute(const void*, int64_t, int64_t, const int32_t*, const float*, int64_t,
                            int32_t, int64_t, int32_t, void*, void*) {
  return entered();
}
int32_t host_test_unpermute_grad(const void*, int64_t, const void*, int64_t, int64_t,
                                 const int32_t*, const int32_t*, const float*, int64_t, int32_t,
                                 int64_t, int32_t, void*, float*, void*) {
  return entered();
}
int32_t host_test_topk_gating(const void*, int32_t, int64_t, int32_t, int32_t, int32_t, int32_t,
                              float*, int32_t*, void*) {
  return entered();
}
int32_t host_test_topk_gating_grad(const void*, int32_t, int64_t, int32_t, int32_t, int32_t,
                                   int32_t, const float*, const int32_t*, const float*, void*,
                                   void*) {
  return entered();
}
int32_t host_test_linear(const void*, int64_t, const void*, int64_t, int64_t, const void*,
                         const void*, int64_t, const int32_t*, int32_t, int64_t, int64_t, int64_t,
                         int32_t, int32_t, int32_t, int32_t, float*, void*, void*) {
  return entered();
}
int32_t host_test_linear_act_grad(const void*, int64_t, const float*, int64_t, int64_t, int32_t,
                                  int32_t, int32_t, void*, void*) {
  return entered();
}
int32_t host_test_linear_input_grad(const void*, int64_t, const void*, int64_t, int64_t,
                                    const int32_t*, int32_t, int64_t, int64_t, int64_t, int32_t,
                                    int32_t, void*, void*) {
  return entered();
}
int32_t host_test_linear_weight_grad(const void*, int64_t, const void*, int64_t, const int32_t*,
                                     int32_t, int64_t, int64_t, int64_t, int32_t, int32_t, void*,
                                     void*) {
  return entered();
}
int64_t host_test_linear_bias_grad_workspace_bytes(int32_t, int64_t, int64_t) { return 0; }
int32_t host_test_linear_bias_grad(const void*, int64_t, const int32_t*, int32_t, int64_t, int64_t,
                                   int32_t, void*, int64_t, void*, void*) {
  return entered();
}
}
