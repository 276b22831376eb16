// extern "C" boundary of the training-step operators: the same conventions as
// abi.cu (host-side checks, the caller's buffers, device and stream).
#include "common.cuh"

namespace fab {

size_t qk_backward_ws_bytes(int batch, int length, int q_heads, int k_heads, int dim);
int qk_impl(const fa_heads* q, const fa_heads* k, const fa_heads* gq, const fa_heads* gk,
            const fa_heads* oq, const fa_heads* ok, bool backward, const fa_qk_params* pr,
            void* ws, size_t ws_bytes, void* dqw, void* dkw, int device, cudaStream_t st);
size_t ns_ws_bytes(const fa_matrix* m, int count, int dtype);
bool ns_shape_ok(int rows, int cols);
int ns_check(const fa_matrix* m, int count, int dtype, bool update);
int ns_impl(const fa_matrix* m, int count, int dtype, const double* coef, int steps, bool update,
            double mu, int nesterov, double decay, void* ws, size_t ws_bytes, int device,
            cudaStream_t st);
int ns_wait_limit(unsigned long long limit_ns);

}  // namespace fab

using namespace fab;

extern "C" {

FA_B200_API int fa_b200_qk_norm_rotary(const fa_heads* q, const fa_heads* k,
                                       const fa_heads* q_out, const fa_heads* k_out,
                                       const fa_qk_params* params, int device, void* stream) {
  FAB_PENDING();
  FAB_DEVICE_SCOPE(device);
  return qk_impl(q, k, nullptr, nullptr, q_out, k_out, false, params, nullptr, 0, nullptr,
                 nullptr, device, static_cast<cudaStream_t>(stream));
}

FA_B200_API int fa_b200_qk_norm_rotary_backward_workspace_bytes(int batch, int length,
                                                                int q_heads, int k_heads,
                                                                int dim, size_t* out_bytes) {
  if (!out_bytes) return FA_E_ARG;
  if (batch <= 0 || length <= 0 || q_heads <= 0 || k_heads <= 0 || dim <= 0) return FA_E_SHAPE;
  *out_bytes = qk_backward_ws_bytes(batch, length, q_heads, k_heads, dim);
  return FA_OK;
}

FA_B200_API int fa_b200_qk_norm_rotary_backward(const fa_heads* q, const fa_heads* k,
                                                const fa_heads* gq, const fa_heads* gk,
                                                const fa_heads* dq, const fa_heads* dk,
                                                const fa_qk_params* params, void* dq_weight,
                                                void* dk_weight, void* workspace,
                                                size_t workspace_bytes, int device,
                                                void* stream) {
  FAB_PENDING();
  FAB_DEVICE_SCOPE(device);
  return qk_impl(q, k, gq, gk, dq, dk, true, params, workspace, workspace_bytes, dq_weight,
                 dk_weight, device, static_cast<cudaStream_t>(stream));
}

FA_B200_API int fa_b200_orthogonalize_workspace_bytes(const fa_matrix* matrices, int count,
                                                      int dtype, size_t* out_bytes) {
  if (!out_bytes || !matrices || count <= 0) return FA_E_ARG;
  if (dtype != FA_F16 && dtype != FA_BF16 && dtype != FA_F32) return FA_E_DTYPE;
  for (int i = 0; i < count; ++i)
    if (!ns_shape_ok(matrices[i].rows, matrices[i].cols)) return FA_E_SHAPE;
  *out_bytes = ns_ws_bytes(matrices, count, dtype);
  return FA_OK;
}

FA_B200_API int fa_b200_orthogonalize(const fa_matrix* matrices, int count, int dtype,
                                      const double* coefficients, int steps, void* workspace,
                                      size_t workspace_bytes, int device, void* stream) {
  FAB_PENDING();
  if (const int rc = ns_check(matrices, count, dtype, false)) return rc;
  FAB_DEVICE_SCOPE(device);
  return ns_impl(matrices, count, dtype, coefficients, steps, false, 0.0, 0, 1.0, workspace,
                 workspace_bytes, device, static_cast<cudaStream_t>(stream));
}

FA_B200_API int fa_b200_muon_step(const fa_matrix* matrices, int count, int dtype,
                                  const double* coefficients, int steps, double mu,
                                  int nesterov, double decay, void* workspace,
                                  size_t workspace_bytes, int device, void* stream) {
  FAB_PENDING();
  if (const int rc = ns_check(matrices, count, dtype, true)) return rc;
  FAB_DEVICE_SCOPE(device);
  return ns_impl(matrices, count, dtype, coefficients, steps, true, mu, nesterov, decay,
                 workspace, workspace_bytes, device, static_cast<cudaStream_t>(stream));
}

FA_B200_API int fa_b200_orthogonalize_wait_limit(unsigned long long limit_ns) {
  return ns_wait_limit(limit_ns);
}

}  // extern "C"
