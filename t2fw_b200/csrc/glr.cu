// The gated linear recurrence: choice of the storage type (kernels in glr_scan.cuh, one file per type), and single steps.
#include "common.cuh"

namespace t2fw {

template <typename T, bool kFused>
int glr_forward_t(const void *x, const void *f, const void *state, void *out, void *next, int64_t B, int64_t steps, int64_t D,
                  cudaStream_t st);
template <typename T, bool kFused>
int glr_backward_t(const void *go, const void *gs, const void *x, const void *f, const void *out, const void *state, void *dx,
                   void *df, void *ds, int64_t B, int64_t steps, int64_t D, cudaStream_t st);

namespace {

// One step: every array is a flat list of n = B*D numbers.  `state` and `next` may be the same array (an element is read and
// then written by the same thread), so nothing here is declared free of aliases.
template <typename T>
__global__ void __launch_bounds__(256)
glr_step_kernel(const T *x, const T *f, const T *state, T *out, T *next, int64_t n) {
  using A = typename Elem<T>::acc;
  dependency_wait();
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const A h = (A)Elem<T>::ld(f + i) * (A)Elem<T>::ld(state + i) + (A)Elem<T>::ld(x + i);
  Elem<T>::st(out + i, h);
  Elem<T>::st(next + i, h);
}

template <typename T>
int launch_step(const void *x, const void *f, const void *state, void *out, void *next, int64_t n, cudaStream_t st) {
  T2FW_CHECK_CUDA(launch_dependent(glr_step_kernel<T>, dim3((unsigned)ceil_div64(n, 256)), dim3(256), 0, st,
                                   static_cast<const T *>(x), static_cast<const T *>(f), static_cast<const T *>(state),
                                   static_cast<T *>(out), static_cast<T *>(next), n));
  T2FW_CHECK_LAUNCH(1);
  return T2FW_OK;
}

}  // namespace

#define T2FW_GLR_TYPES(fn, fused, ...)                                     \
  switch (dtype) {                                                         \
    case T2FW_F16: return fn<__half, fused>(__VA_ARGS__);                  \
    case T2FW_BF16: return fn<__nv_bfloat16, fused>(__VA_ARGS__);          \
    case T2FW_F32: return fn<float, fused>(__VA_ARGS__);                   \
    default: return fn<double, fused>(__VA_ARGS__);                        \
  }

int glr_step(const void *x, const void *f, const void *state, void *out, void *next, int64_t n, int dtype, cudaStream_t st) {
  switch (dtype) {
    case T2FW_F16: return launch_step<__half>(x, f, state, out, next, n, st);
    case T2FW_BF16: return launch_step<__nv_bfloat16>(x, f, state, out, next, n, st);
    case T2FW_F32: return launch_step<float>(x, f, state, out, next, n, st);
    default: return launch_step<double>(x, f, state, out, next, n, st);
  }
}
int glr_forward(const void *x, const void *f, const void *state, void *out, void *next, int64_t B, int64_t T, int64_t D,
                int dtype, cudaStream_t st) {
  if (T == 1) return glr_step(x, f, state, out, next, B * D, dtype, st);
  T2FW_GLR_TYPES(glr_forward_t, false, x, f, state, out, next, B, T, D, st)
}
int glr_fused_forward(const void *vg, const void *state, void *out, void *next, int64_t B, int64_t T, int64_t D, int dtype,
                      cudaStream_t st) {
  T2FW_GLR_TYPES(glr_forward_t, true, vg, nullptr, state, out, next, B, T, D, st)
}
int glr_backward(const void *go, const void *gs, const void *f, const void *out, const void *state, void *dx, void *df,
                 void *ds, int64_t B, int64_t T, int64_t D, int dtype, cudaStream_t st) {
  T2FW_GLR_TYPES(glr_backward_t, false, go, gs, nullptr, f, out, state, dx, df, ds, B, T, D, st)
}
int glr_fused_backward(const void *go, const void *gs, const void *vg, const void *out, const void *state, void *dvg,
                       void *ds, int64_t B, int64_t T, int64_t D, int dtype, cudaStream_t st) {
  T2FW_GLR_TYPES(glr_backward_t, true, go, gs, vg, nullptr, out, state, dvg, nullptr, ds, B, T, D, st)
}

}  // namespace t2fw
