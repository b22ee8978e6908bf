// Root-mean-square norm over rows of D, with or without the addition of a residual, and its gradients:
//
//   s = x + residual,  rstd = 1 / sqrt(mean(s^2) + eps),  y = s rstd w
//   g = w dy:   d_s = rstd (g - s rstd^2 mean(g s)) + (gradient of s from its other use) ,   d_w = sum over rows of dy s rstd
//
// x and the residual share the gradient d_s.  The 8-bit form leaves q = e4m3(y / scale) with scale = max|y| / 448 per row.
#include <cuda_fp8.h>

#include "common.cuh"

namespace t2fw {

namespace {

constexpr float kE4m3Max = 448.f, kMinScale = 1e-30f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float inv_sqrt(float v) { return 1.f / sqrtf(v); }
__device__ __forceinline__ double inv_sqrt(double v) { return 1.0 / sqrt(v); }

// Sum over a block of 256 threads, the same in each of them.
template <typename A>
__device__ __forceinline__ A block_sum(A v, A *red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  A s = A(0);
#pragma unroll
  for (int i = 0; i < 8; ++i) s += red[i];
  return s;
}
__device__ __forceinline__ float block_max(float v, float *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) s = max_nan(s, red[i]);
  return s;
}

// A block per row.
template <typename T, bool k8>
__global__ void __launch_bounds__(256)
rms_fwd_row_kernel(const T *__restrict__ x, const T *__restrict__ r, const T *__restrict__ w, T *__restrict__ y,
                   __nv_fp8_e4m3 *__restrict__ q, float *__restrict__ scale, T *__restrict__ sum, int64_t D,
                   double eps) {
  using A = typename Elem<T>::acc;
  __shared__ A red[8];
  dependency_wait();
  const int64_t base = (int64_t)blockIdx.x * D;
  A ss = A(0);
  for (int64_t d = threadIdx.x; d < D; d += 256) {
    A s = Elem<T>::ld(x + base + d);
    if (r != nullptr) {
      s += (A)Elem<T>::ld(r + base + d);
      Elem<T>::st(sum + base + d, s);
    }
    ss += s * s;
  }
  const A rstd = inv_sqrt(block_sum(ss, red) / A(D) + A(eps));
  float top = 0.f, sc = 1.f;
  if constexpr (k8) {
    for (int64_t d = threadIdx.x; d < D; d += 256) {
      A s = Elem<T>::ld(x + base + d);
      if (r != nullptr) s += (A)Elem<T>::ld(r + base + d);
      top = max_nan(top, fabsf((float)(s * rstd * (A)Elem<T>::ld(w + d))));
    }
    sc = max_nan(block_max(top, reinterpret_cast<float *>(red)) / kE4m3Max, kMinScale);
    if (threadIdx.x == 0) scale[blockIdx.x] = sc;
  }
  for (int64_t d = threadIdx.x; d < D; d += 256) {
    A s = Elem<T>::ld(x + base + d);
    if (r != nullptr) s += (A)Elem<T>::ld(r + base + d);
    const A v = s * rstd * (A)Elem<T>::ld(w + d);
    if constexpr (k8) q[base + d] = __nv_fp8_e4m3((float)v / sc);
    else Elem<T>::st(y + base + d, v);
  }
}

// Blocks walk rows; the weight gradient of a block's rows is summed in its own line of `part`.
template <typename T>
__global__ void __launch_bounds__(256)
rms_bwd_row_kernel(const T *__restrict__ dy, const T *__restrict__ dsum, const T *__restrict__ s, const T *__restrict__ w,
                   T *__restrict__ ds, typename Elem<T>::acc *__restrict__ part, int64_t rows, int64_t D, double eps) {
  using A = typename Elem<T>::acc;
  __shared__ A red[8];
  dependency_wait();
  A *mine = part + (int64_t)blockIdx.x * D;
  for (int64_t d = threadIdx.x; d < D; d += 256) mine[d] = A(0);
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t base = row * D;
    A ss = A(0), gs = A(0);
    for (int64_t d = threadIdx.x; d < D; d += 256) {
      const A sv = Elem<T>::ld(s + base + d);
      ss += sv * sv;
      gs += sv * (A)Elem<T>::ld(w + d) * (A)Elem<T>::ld(dy + base + d);
    }
    const A rstd = inv_sqrt(block_sum(ss, red) / A(D) + A(eps));
    const A m = block_sum(gs, red) / A(D) * rstd * rstd;
    for (int64_t d = threadIdx.x; d < D; d += 256) {
      const A sv = Elem<T>::ld(s + base + d), dv = Elem<T>::ld(dy + base + d);
      A v = rstd * ((A)Elem<T>::ld(w + d) * dv - sv * m);
      if (dsum != nullptr) v += (A)Elem<T>::ld(dsum + base + d);
      Elem<T>::st(ds + base + d, v);
      mine[d] += dv * sv * rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
rms_dw_kernel(const typename Elem<T>::acc *__restrict__ part, T *__restrict__ dw, int64_t n, int64_t D) {
  using A = typename Elem<T>::acc;
  dependency_wait();
  const int64_t d = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (d >= D) return;
  A v = A(0);
  for (int64_t i = 0; i < n; ++i) v += part[i * D + d];
  Elem<T>::st(dw + d, v);
}

constexpr int64_t kMaxParts = 592;
int64_t bwd_parts(int64_t rows) { return rows < kMaxParts ? rows : kMaxParts; }

template <typename T, bool k8>
int launch_fwd(const void *x, const void *r, const void *w, void *y, void *q, float *scale, void *sum, int64_t rows,
               int64_t D, double eps, cudaStream_t st) {
  T2FW_CHECK_CUDA(launch_dependent(rms_fwd_row_kernel<T, k8>, dim3((unsigned)rows), dim3(256), 0, st,
                                   static_cast<const T *>(x), static_cast<const T *>(r), static_cast<const T *>(w),
                                   static_cast<T *>(y), static_cast<__nv_fp8_e4m3 *>(q), scale, static_cast<T *>(sum), D,
                                   eps));
  T2FW_CHECK_LAUNCH(1);
  return T2FW_OK;
}

template <typename T>
int launch_bwd(const void *dy, const void *dsum, const void *s, const void *w, void *ds, void *dw, int64_t rows, int64_t D,
               double eps, void *scratch, cudaStream_t st) {
  using A = typename Elem<T>::acc;
  const int64_t n = bwd_parts(rows);
  T2FW_CHECK_CUDA(launch_dependent(rms_bwd_row_kernel<T>, dim3((unsigned)n), dim3(256), 0, st, static_cast<const T *>(dy),
                                   static_cast<const T *>(dsum), static_cast<const T *>(s), static_cast<const T *>(w),
                                   static_cast<T *>(ds), static_cast<A *>(scratch), rows, D, eps));
  T2FW_CHECK_LAUNCH(1);
  T2FW_CHECK_CUDA(launch_dependent(rms_dw_kernel<T>, dim3((unsigned)ceil_div64(D, 256)), dim3(256), 0, st,
                                   static_cast<const A *>(scratch), static_cast<T *>(dw), n, D));
  T2FW_CHECK_LAUNCH(1);
  return T2FW_OK;
}

}  // namespace

size_t rms_norm_backward_scratch_bytes(int64_t rows, int64_t D, int dtype) {
  return (size_t)bwd_parts(rows) * (size_t)D * (dtype == T2FW_F64 ? 8 : 4);
}

int rms_norm_forward(const void *x, const void *r, const void *w, void *y, void *sum, int64_t rows, int64_t D, double eps,
                     int dtype, cudaStream_t st) {
  switch (dtype) {
    case T2FW_F16: return launch_fwd<__half, false>(x, r, w, y, nullptr, nullptr, sum, rows, D, eps, st);
    case T2FW_BF16: return launch_fwd<__nv_bfloat16, false>(x, r, w, y, nullptr, nullptr, sum, rows, D, eps, st);
    case T2FW_F32: return launch_fwd<float, false>(x, r, w, y, nullptr, nullptr, sum, rows, D, eps, st);
    default: return launch_fwd<double, false>(x, r, w, y, nullptr, nullptr, sum, rows, D, eps, st);
  }
}

int rms_norm_e4m3(const void *x, const void *r, const void *w, void *q, float *scale, void *sum, int64_t rows, int64_t D,
                  double eps, int dtype, cudaStream_t st) {
  switch (dtype) {
    case T2FW_F16: return launch_fwd<__half, true>(x, r, w, nullptr, q, scale, sum, rows, D, eps, st);
    case T2FW_BF16: return launch_fwd<__nv_bfloat16, true>(x, r, w, nullptr, q, scale, sum, rows, D, eps, st);
    default: return launch_fwd<float, true>(x, r, w, nullptr, q, scale, sum, rows, D, eps, st);
  }
}

int rms_norm_backward(const void *dy, const void *dsum, const void *s, const void *w, void *ds, void *dw, int64_t rows,
                      int64_t D, double eps, int dtype, void *scratch, cudaStream_t st) {
  switch (dtype) {
    case T2FW_F16: return launch_bwd<__half>(dy, dsum, s, w, ds, dw, rows, D, eps, scratch, st);
    case T2FW_BF16: return launch_bwd<__nv_bfloat16>(dy, dsum, s, w, ds, dw, rows, D, eps, scratch, st);
    case T2FW_F32: return launch_bwd<float>(dy, dsum, s, w, ds, dw, rows, D, eps, scratch, st);
    default: return launch_bwd<double>(dy, dsum, s, w, ds, dw, rows, D, eps, scratch, st);
  }
}

}  // namespace t2fw
