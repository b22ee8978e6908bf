// The root-mean-square norm: choice of the storage type (kernels in rms_norm.cuh, one file per type).
#include "common.cuh"

namespace t2fw {

template <typename T, bool k8>
int rms_forward_t(const void *x, const void *r, const void *w, void *y, void *q, float *scale, void *sum, int64_t rows,
                  int64_t D, double eps, cudaStream_t st);
template <typename T>
int rms_backward_t(const void *dy, const void *dsum, const void *s, const void *w, void *ds, void *dw, int64_t rows, int64_t D,
                   double eps, void *scratch, cudaStream_t st);

// One line of partial sums of the weight gradient per block of the backward launch; there are never more than 1024 (kMostParts)
// blocks, nor more than rows.
size_t rms_norm_backward_scratch_bytes(int64_t rows, int64_t D, int dtype) {
  return (size_t)(rows < 1024 ? rows : 1024) * (size_t)D * (dtype == T2FW_F64 ? 8 : 4);
}

int rms_norm_forward(const void *x, const void *r, const void *w, void *y, void *sum, int64_t rows, int64_t D, double eps,
                     int dtype, cudaStream_t st) {
  switch (dtype) {
    case T2FW_F16: return rms_forward_t<__half, false>(x, r, w, y, nullptr, nullptr, sum, rows, D, eps, st);
    case T2FW_BF16: return rms_forward_t<__nv_bfloat16, false>(x, r, w, y, nullptr, nullptr, sum, rows, D, eps, st);
    case T2FW_F32: return rms_forward_t<float, false>(x, r, w, y, nullptr, nullptr, sum, rows, D, eps, st);
    default: return rms_forward_t<double, false>(x, r, w, y, nullptr, nullptr, sum, rows, D, eps, st);
  }
}

int rms_norm_e4m3(const void *x, const void *r, const void *w, void *q, float *scale, void *sum, int64_t rows, int64_t D,
                  double eps, int dtype, cudaStream_t st) {
  switch (dtype) {
    case T2FW_F16: return rms_forward_t<__half, true>(x, r, w, nullptr, q, scale, sum, rows, D, eps, st);
    case T2FW_BF16: return rms_forward_t<__nv_bfloat16, true>(x, r, w, nullptr, q, scale, sum, rows, D, eps, st);
    default: return rms_forward_t<float, true>(x, r, w, nullptr, q, scale, sum, rows, D, eps, st);
  }
}

int rms_norm_backward(const void *dy, const void *dsum, const void *s, const void *w, void *ds, void *dw, int64_t rows,
                      int64_t D, double eps, int dtype, void *scratch, cudaStream_t st) {
  switch (dtype) {
    case T2FW_F16: return rms_backward_t<__half>(dy, dsum, s, w, ds, dw, rows, D, eps, scratch, st);
    case T2FW_BF16: return rms_backward_t<__nv_bfloat16>(dy, dsum, s, w, ds, dw, rows, D, eps, scratch, st);
    case T2FW_F32: return rms_backward_t<float>(dy, dsum, s, w, ds, dw, rows, D, eps, scratch, st);
    default: return rms_backward_t<double>(dy, dsum, s, w, ds, dw, rows, D, eps, scratch, st);
  }
}

}  // namespace t2fw
