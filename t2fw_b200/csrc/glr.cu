// The gated linear recurrence: a state of one number per channel,
//
//   h_t = f_t h_{t-1} + x_t ,   outputs_t = h_t            (h_0 = state [B,D]; x, f, outputs [B,T,D])
//
// and its gradients.  With r_t the gradient of h_t, r_T = go_T + gs and r_t = go_t + f_{t+1} r_{t+1}:
//
//   d_x_t = r_t ,   d_f_t = r_t h_{t-1} ,   d_state = f_1 r_1
//
// Fused layer form: vg [B,T,2D] = value v | gate pre-activation g, read in place: a = sigmoid(g), f = a,
// x = (1 - a) v;  d_v = (1 - a) r,  d_g = a (1 - a) r (h_{t-1} - v).
#include "common.cuh"

namespace t2fw {

namespace {

__device__ __forceinline__ float exp_neg_abs(float g) { return expf(-fabsf(g)); }
__device__ __forceinline__ double exp_neg_abs(double g) { return exp(-fabs(g)); }

// a = sigmoid(g) and 1 - a, both to full relative precision: from exp(-|g|), which does not overflow
template <typename A>
__device__ __forceinline__ void gate_pair(A g, A &a, A &rest) {
  const A e = exp_neg_abs(g), hi = A(1) / (A(1) + e), lo = e * hi;
  a = g >= A(0) ? hi : lo;
  rest = g >= A(0) ? lo : hi;
  if (!(g == g)) a = rest = g;
}

template <typename T, bool kFused>
__global__ void __launch_bounds__(128)
glr_fwd_kernel(const T *__restrict__ x, const T *__restrict__ f, const T *__restrict__ state, T *__restrict__ out,
               T *__restrict__ next, int64_t B, int64_t steps, int64_t D) {
  using A = typename Elem<T>::acc;
  dependency_wait();
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= B * D) return;
  const int64_t b = i / D, d = i - b * D, row = kFused ? 2 * D : D;
  A h = Elem<T>::ld(state + i);
  const T *px = x + b * steps * row + d, *pf = kFused ? px + D : f + b * steps * D + d;
  T *po = out + b * steps * D + d;
  for (int64_t t = 0; t < steps; ++t) {
    A xv = Elem<T>::ld(px + t * row), fv = Elem<T>::ld(pf + t * row);
    if (kFused) {
      A rest;
      gate_pair(fv, fv, rest);
      xv *= rest;
    }
    h = fv * h + xv;
    Elem<T>::st(po + t * D, h);
  }
  Elem<T>::st(next + i, h);
}

template <typename T, bool kFused>
__global__ void __launch_bounds__(128)
glr_bwd_kernel(const T *__restrict__ go, const T *__restrict__ gs, const T *__restrict__ x, const T *__restrict__ f,
               const T *__restrict__ out, const T *__restrict__ state, T *__restrict__ dx, T *__restrict__ df,
               T *__restrict__ ds, int64_t B, int64_t steps, int64_t D) {
  using A = typename Elem<T>::acc;
  dependency_wait();
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= B * D) return;
  const int64_t b = i / D, d = i - b * D, row = kFused ? 2 * D : D;
  const int64_t at = b * steps * row + d, ot = b * steps * D + d;
  A c = gs != nullptr ? (A)Elem<T>::ld(gs + i) : A(0);
  for (int64_t t = steps - 1; t >= 0; --t) {
    const A r = (A)Elem<T>::ld(go + ot + t * D) + c;
    const A before = t > 0 ? (A)Elem<T>::ld(out + ot + (t - 1) * D) : (A)Elem<T>::ld(state + i);
    if (kFused) {
      A a, rest;
      gate_pair((A)Elem<T>::ld(x + at + D + t * row), a, rest);
      Elem<T>::st(dx + at + t * row, rest * r);
      Elem<T>::st(dx + at + D + t * row, a * rest * r * (before - (A)Elem<T>::ld(x + at + t * row)));
      c = a * r;
    } else {
      Elem<T>::st(dx + ot + t * D, r);
      Elem<T>::st(df + ot + t * D, r * before);
      c = (A)Elem<T>::ld(f + ot + t * D) * r;
    }
  }
  Elem<T>::st(ds + i, c);
}

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

template <typename T, bool kFused>
int launch_fwd(const void *x, const void *f, const void *state, void *out, void *next, int64_t B, int64_t steps, int64_t D,
               cudaStream_t st) {
  T2FW_CHECK_CUDA(launch_dependent(glr_fwd_kernel<T, kFused>, dim3((unsigned)ceil_div64(B * D, 128)), dim3(128), 0, st,
                                   static_cast<const T *>(x), static_cast<const T *>(f), static_cast<const T *>(state),
                                   static_cast<T *>(out), static_cast<T *>(next), B, steps, D));
  T2FW_CHECK_LAUNCH(1);
  return T2FW_OK;
}

template <typename T, bool kFused>
int launch_bwd(const void *go, const void *gs, const void *x, const void *f, const void *out, const void *state, void *dx,
               void *df, void *ds, int64_t B, int64_t steps, int64_t D, cudaStream_t st) {
  T2FW_CHECK_CUDA(launch_dependent(glr_bwd_kernel<T, kFused>, dim3((unsigned)ceil_div64(B * D, 128)), dim3(128), 0, st,
                                   static_cast<const T *>(go), static_cast<const T *>(gs), static_cast<const T *>(x),
                                   static_cast<const T *>(f), static_cast<const T *>(out), static_cast<const T *>(state),
                                   static_cast<T *>(dx), static_cast<T *>(df), static_cast<T *>(ds), B, steps, D));
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
  T2FW_GLR_TYPES(launch_fwd, false, x, f, state, out, next, B, T, D, st)
}
int glr_fused_forward(const void *vg, const void *state, void *out, void *next, int64_t B, int64_t T, int64_t D, int dtype,
                      cudaStream_t st) {
  T2FW_GLR_TYPES(launch_fwd, true, vg, nullptr, state, out, next, B, T, D, st)
}
int glr_backward(const void *go, const void *gs, const void *f, const void *out, const void *state, void *dx, void *df,
                 void *ds, int64_t B, int64_t T, int64_t D, int dtype, cudaStream_t st) {
  T2FW_GLR_TYPES(launch_bwd, false, go, gs, nullptr, f, out, state, dx, df, ds, B, T, D, st)
}
int glr_fused_backward(const void *go, const void *gs, const void *vg, const void *out, const void *state, void *dvg,
                       void *ds, int64_t B, int64_t T, int64_t D, int dtype, cudaStream_t st) {
  T2FW_GLR_TYPES(launch_bwd, true, go, gs, vg, nullptr, out, state, dvg, nullptr, ds, B, T, D, st)
}

}  // namespace t2fw
