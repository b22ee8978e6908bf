// C ABI of the operators that stand around the recurrences in a model (declared in include/t2fw_b200.h): the gated linear
// recurrence, the root-mean-square norm, gradient clipping.  Argument checks only; nothing here allocates, frees or synchronises.
#include <initializer_list>

#include "common.cuh"

using namespace t2fw;

extern "C" {

// Sizes whose products (elements, bytes, both halves of a projection) stay inside 62 bits.
static int check_glr(int64_t B, int64_t T, int64_t D, int dtype) {
  T2FW_CHECK_ARG(dtype_size(dtype) != 0, "unknown dtype %d", dtype);
  T2FW_CHECK_ARG(B > 0 && T > 0 && D > 0, "sizes must be positive (B=%lld T=%lld D=%lld)", (long long)B, (long long)T,
                 (long long)D);
  const int64_t most = (int64_t)1 << 40;
  T2FW_CHECK_ARG(B <= most && D <= most / B && T <= most / (B * D), "sizes out of range (B=%lld T=%lld D=%lld)",
                 (long long)B, (long long)T, (long long)D);
  return T2FW_OK;
}

int t2fw_glr_forward(const void *value, const void *forget, const void *state, void *outputs, void *next_state, int64_t B,
                     int64_t T, int64_t D, int dtype, void *stream) {
  const int rc = check_glr(B, T, D, dtype);
  if (rc != T2FW_OK) return rc;
  T2FW_CHECK_ARG(value && forget && state && outputs && next_state, "null pointer argument");
  return glr_forward(value, forget, state, outputs, next_state, B, T, D, dtype, static_cast<cudaStream_t>(stream));
}

int t2fw_glr_backward(const void *grad_output, const void *grad_state, const void *forget, const void *outputs,
                      const void *state, void *d_value, void *d_forget, void *d_state, int64_t B, int64_t T, int64_t D,
                      int dtype, void *stream) {
  const int rc = check_glr(B, T, D, dtype);
  if (rc != T2FW_OK) return rc;
  T2FW_CHECK_ARG(grad_output && forget && outputs && state && d_value && d_forget && d_state, "null pointer argument");
  return glr_backward(grad_output, grad_state, forget, outputs, state, d_value, d_forget, d_state, B, T, D, dtype,
                      static_cast<cudaStream_t>(stream));
}

int t2fw_glr_fused_forward(const void *vg, const void *state, void *outputs, void *next_state, int64_t B, int64_t T,
                           int64_t D, int dtype, void *stream) {
  const int rc = check_glr(B, T, D, dtype);
  if (rc != T2FW_OK) return rc;
  T2FW_CHECK_ARG(vg && state && outputs && next_state, "null pointer argument");
  return glr_fused_forward(vg, state, outputs, next_state, B, T, D, dtype, static_cast<cudaStream_t>(stream));
}

int t2fw_glr_fused_backward(const void *grad_output, const void *grad_state, const void *vg, const void *outputs,
                            const void *state, void *d_vg, void *d_state, int64_t B, int64_t T, int64_t D, int dtype,
                            void *stream) {
  const int rc = check_glr(B, T, D, dtype);
  if (rc != T2FW_OK) return rc;
  T2FW_CHECK_ARG(grad_output && vg && outputs && state && d_vg && d_state, "null pointer argument");
  return glr_fused_backward(grad_output, grad_state, vg, outputs, state, d_vg, d_state, B, T, D, dtype,
                            static_cast<cudaStream_t>(stream));
}

static int check_rms(int64_t rows, int64_t D, double eps, int dtype) {
  T2FW_CHECK_ARG(dtype_size(dtype) != 0, "unknown dtype %d", dtype);
  T2FW_CHECK_ARG(rows > 0 && D > 0, "sizes must be positive (rows=%lld D=%lld)", (long long)rows, (long long)D);
  T2FW_CHECK_ARG(rows < (int64_t)1 << 31 && D <= ((int64_t)1 << 40) / rows, "sizes out of range (rows=%lld D=%lld)",
                 (long long)rows, (long long)D);
  T2FW_CHECK_ARG(eps >= 0, "eps must not be negative");
  return T2FW_OK;
}

// What is written shares no byte with what is read: rows whose squares leave the range are read again after a first write, and rows
// that no registers hold are read twice.
struct Span {
  const void *p;
  int64_t bytes;
};
static int check_apart(std::initializer_list<Span> out, std::initializer_list<Span> in) {
  for (const Span &o : out)
    for (const Span &i : in) {
      const uintptr_t a = reinterpret_cast<uintptr_t>(o.p), b = reinterpret_cast<uintptr_t>(i.p);
      T2FW_CHECK_ARG(a == 0 || b == 0 || a >= b + (uint64_t)i.bytes || b >= a + (uint64_t)o.bytes,
                     "an output shares memory with an input");
    }
  return T2FW_OK;
}

int t2fw_rms_norm_forward(const void *x, const void *residual, const void *weight, void *y, void *sum, int64_t rows,
                          int64_t D, double eps, int dtype, void *stream) {
  const int rc = check_rms(rows, D, eps, dtype);
  if (rc != T2FW_OK) return rc;
  T2FW_CHECK_ARG(x && weight && y, "null pointer argument");
  T2FW_CHECK_ARG((residual == nullptr) == (sum == nullptr), "residual and sum are given together");
  const int64_t e = (int64_t)dtype_size(dtype), n = rows * D * e;
  const int apart = check_apart({{y, n}, {sum, n}}, {{x, n}, {residual, n}, {weight, D * e}});
  if (apart != T2FW_OK) return apart;
  return rms_norm_forward(x, residual, weight, y, sum, rows, D, eps, dtype, static_cast<cudaStream_t>(stream));
}

int t2fw_rms_norm_e4m3(const void *x, const void *residual, const void *weight, void *q, float *scale, void *sum,
                       int64_t rows, int64_t D, double eps, int dtype, void *stream) {
  const int rc = check_rms(rows, D, eps, dtype);
  if (rc != T2FW_OK) return rc;
  T2FW_CHECK_ARG(x && weight && q && scale, "null pointer argument");
  T2FW_CHECK_ARG((residual == nullptr) == (sum == nullptr), "residual and sum are given together");
  if (dtype == T2FW_F64) {
    set_error("rms norm with an 8-bit output: 16- and 32-bit storage only");
    return T2FW_ERR_UNSUPPORTED;
  }
  const int64_t e = (int64_t)dtype_size(dtype), n = rows * D * e;
  const int apart = check_apart({{q, rows * D}, {scale, rows * 4}, {sum, n}}, {{x, n}, {residual, n}, {weight, D * e}});
  if (apart != T2FW_OK) return apart;
  return rms_norm_e4m3(x, residual, weight, q, scale, sum, rows, D, eps, dtype, static_cast<cudaStream_t>(stream));
}

size_t t2fw_rms_norm_backward_scratch_bytes(int64_t rows, int64_t D, int dtype) {
  if (check_rms(rows, D, 0, dtype) != T2FW_OK) return 0;
  return rms_norm_backward_scratch_bytes(rows, D, dtype);
}

int t2fw_rms_norm_backward(const void *grad_y, const void *grad_sum, const void *s, const void *weight, void *d_s,
                           void *d_weight, int64_t rows, int64_t D, double eps, int dtype, void *scratch,
                           size_t scratch_bytes, void *stream) {
  const int rc = check_rms(rows, D, eps, dtype);
  if (rc != T2FW_OK) return rc;
  T2FW_CHECK_ARG(grad_y && s && weight && d_s && d_weight, "null pointer argument");
  const size_t need = rms_norm_backward_scratch_bytes(rows, D, dtype);
  if (scratch == nullptr || scratch_bytes < need) {
    set_error("rms norm backward needs %zu bytes of scratch, got %zu", need, scratch_bytes);
    return T2FW_ERR_SCRATCH;
  }
  T2FW_CHECK_ARG((reinterpret_cast<uintptr_t>(scratch) & 15) == 0, "scratch must be 16-byte aligned");
  const int64_t e = (int64_t)dtype_size(dtype), n = rows * D * e;
  const int apart = check_apart({{d_s, n}, {d_weight, D * e}, {scratch, (int64_t)need}},
                                {{grad_y, n}, {grad_sum, n}, {s, n}, {weight, D * e}});
  if (apart != T2FW_OK) return apart;
  return rms_norm_backward(grad_y, grad_sum, s, weight, d_s, d_weight, rows, D, eps, dtype, scratch,
                           static_cast<cudaStream_t>(stream));
}

size_t t2fw_grad_clip_scratch_bytes(int64_t n_tensors) { return n_tensors > 0 ? grad_clip_scratch_bytes(n_tensors) : 0; }

static int check_list(const void *const *in, const int64_t *numel, const int *dtype, int64_t n, const void *total,
                      int total_dtype, const void *scratch, size_t scratch_bytes) {
  T2FW_CHECK_ARG(n > 0 && n <= 1 << 24, "number of tensors out of range (%lld)", (long long)n);
  T2FW_CHECK_ARG(in && numel && dtype && total, "null pointer argument");
  T2FW_CHECK_ARG(total_dtype == T2FW_F32 || total_dtype == T2FW_F64, "the norm is float32 or float64 (dtype %d)",
                 total_dtype);
  int64_t left = (int64_t)1 << 44;      // elements in all
  for (int64_t i = 0; i < n; ++i) {
    T2FW_CHECK_ARG(dtype_size(dtype[i]) != 0, "tensor %lld: unknown dtype %d", (long long)i, dtype[i]);
    T2FW_CHECK_ARG(in[i] != nullptr, "tensor %lld: null pointer", (long long)i);
    T2FW_CHECK_ARG(numel[i] > 0 && numel[i] <= left, "tensor %lld: size out of range (%lld)", (long long)i,
                   (long long)numel[i]);
    left -= numel[i];
  }
  const size_t need = grad_clip_scratch_bytes(n);
  if (scratch == nullptr || scratch_bytes < need) {
    set_error("gradient norm needs %zu bytes of scratch, got %zu", need, scratch_bytes);
    return T2FW_ERR_SCRATCH;
  }
  T2FW_CHECK_ARG((reinterpret_cast<uintptr_t>(scratch) & 15) == 0, "scratch must be 16-byte aligned");
  return T2FW_OK;
}

int t2fw_grad_norm(const void *const *tensors, const int64_t *numel, const int *dtype, int64_t n, void *total,
                   int total_dtype, void *scratch, size_t scratch_bytes, void *stream) {
  const int rc = check_list(tensors, numel, dtype, n, total, total_dtype, scratch, scratch_bytes);
  if (rc != T2FW_OK) return rc;
  return grad_clip(tensors, nullptr, numel, dtype, (int)n, -1.0, total, total_dtype, scratch,
                   static_cast<cudaStream_t>(stream));
}

int t2fw_grad_clip(const void *const *tensors, void *const *out, const int64_t *numel, const int *dtype, int64_t n,
                   double max_norm, void *total, int total_dtype, void *scratch, size_t scratch_bytes, void *stream) {
  const int rc = check_list(tensors, numel, dtype, n, total, total_dtype, scratch, scratch_bytes);
  if (rc != T2FW_OK) return rc;
  T2FW_CHECK_ARG(max_norm >= 0, "max_norm must not be negative");
  T2FW_CHECK_ARG(out != nullptr, "null pointer argument");
  const bool in_place = out[0] == tensors[0];
  for (int64_t i = 0; i < n; ++i) {
    T2FW_CHECK_ARG(out[i] != nullptr, "output %lld: null pointer", (long long)i);
    T2FW_CHECK_ARG((out[i] == tensors[i]) == in_place, "either all tensors are scaled in place or none");
  }
  return grad_clip(tensors, out, numel, dtype, (int)n, max_norm, total, total_dtype, scratch,
                   static_cast<cudaStream_t>(stream));
}

}  // extern "C"
