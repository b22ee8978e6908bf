// The gated linear recurrence: choice of the storage type (kernels in glr_scan.cuh, one file per type), and single steps.
#include <initializer_list>

#include "glr.cuh"

namespace t2fw {

template <typename T, bool kFused>
int glr_forward_t(const void *x, const void *f, const void *state, void *out, void *next, int64_t B, int64_t steps, int64_t D,
                  cudaStream_t st);
template <typename T, bool kFused>
int glr_backward_t(const void *go, const void *gs, const void *x, const void *f, const void *out, const void *state, void *dx,
                   void *df, void *ds, int64_t B, int64_t steps, int64_t D, cudaStream_t st);

namespace {

// One step: every array is a flat list of n = B*D numbers, V of them to a thread.  `state` and `next` may be the same array (a
// thread reads what it then writes), so nothing here is declared free of aliases.  A small call is its launch: 256 x 768 takes
// 3.7 us from Python.
template <typename T, int V>
__global__ void __launch_bounds__(256)
glr_step_kernel(const T *x, const T *f, const T *state, T *out, T *next, int64_t n) {
  using A = typename Elem<T>::acc;
  using R = typename glr::Raw<T, V>::type;
  dependency_wait();
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * V;
  if (i >= n) return;
  A h[V], fv[V], xv[V];
  glr::unpack<T, V>(*reinterpret_cast<const R *>(state + i), h);
  glr::unpack<T, V>(*reinterpret_cast<const R *>(f + i), fv);
  glr::unpack<T, V>(*reinterpret_cast<const R *>(x + i), xv);
  glr::fma_v(h, fv, h, xv);
  const R r = glr::pack<T, V>(h);
  *reinterpret_cast<R *>(out + i) = r;
  *reinterpret_cast<R *>(next + i) = r;
}

// 16 bytes to a thread where the pointers allow it and the threads are many (a small call is over sooner with more of them).  Single
// elements against vectors, fp16, us on the device: 65 536 numbers 1.0 / 1.4, 196 608 1.1 / 1.4, 262 144 1.3 / 1.4, 1 M 5.4 / 3.1; in fp32
// 0.97 / 1.25, 1.86 / 1.85, 2.24 / 2.20, 5.6 / 4.9.
template <typename T>
int launch_step(const void *x, const void *f, const void *state, void *out, void *next, int64_t n, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  uintptr_t low = 0;
  for (const void *q : {x, f, state, static_cast<const void *>(out), static_cast<const void *>(next)}) low |= reinterpret_cast<uintptr_t>(q);
  const bool wide = n % V == 0 && (low & 15) == 0 && n >= 1 << 18;
  const int64_t blocks = ceil_div64(wide ? n / V : n, 256);
  T2FW_CHECK_ARG(blocks <= 0x7fffffff, "sizes out of range");
  T2FW_CHECK_CUDA(launch_dependent(wide ? glr_step_kernel<T, V> : glr_step_kernel<T, 1>, dim3((unsigned)blocks), dim3(256), 0, st,
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
