// Global norm of a list of tensors and scaling by it:
//
//   total = sqrt(sum over all tensors and elements of g^2),   c = min(1, max_norm / (total + 1e-6)),   g' = c g
//
// Two kinds of launch.  The first leaves one partial sum per block; the second adds them up in each block, in the same order,
// and scales.  The tensors' addresses and sizes travel as kernel arguments, so a call needs no table in device memory and can be
// captured.  Work is cut into pieces of 16 KB; a block takes consecutive ones.
#include "common.cuh"

namespace t2fw {

namespace {

constexpr int kTable = 512, kThreads = 256, kPieceBytes = 16384, kMaxBlocks = 592;

struct Entry {
  const void *in;
  void *out;
  int64_t n;
};
template <int N>
struct Table {
  Entry e[N];
  uint32_t first[N + 1];      // pieces before tensor i
  uint8_t type[N];
  int count;
};

__device__ __forceinline__ double block_sum(double v, double *red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) s += red[i];
  return s;
}

// The tensor that piece p lies in.
template <int N>
__device__ __forceinline__ int find(const Table<N> &t, uint32_t p) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= p) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ double squares(const T *in, int64_t from, int64_t to) {
  double s = 0;
  for (int64_t i = from + threadIdx.x; i < to; i += kThreads) {
    const double v = (double)Elem<T>::ld(in + i);
    s += v * v;
  }
  return s;
}

template <typename T, typename C>
__device__ __forceinline__ void scale(const T *in, T *out, int64_t from, int64_t to, C c) {
  using A = typename Elem<T>::acc;
  for (int64_t i = from + threadIdx.x; i < to; i += kThreads) Elem<T>::st(out + i, (A)Elem<T>::ld(in + i) * (A)c);
}

template <int N>
__global__ void __launch_bounds__(kThreads)
grad_norm_kernel(const __grid_constant__ Table<N> t, double *__restrict__ part) {
  __shared__ double red[kThreads / 32];
  dependency_wait();
  const uint32_t pieces = t.first[t.count];
  const uint32_t p0 = (uint32_t)((uint64_t)pieces * blockIdx.x / gridDim.x),
                 p1 = (uint32_t)((uint64_t)pieces * (blockIdx.x + 1) / gridDim.x);
  int k = find(t, p0);
  double s = 0;
  for (uint32_t p = p0; p < p1; ++p) {
    while (p >= t.first[k + 1]) ++k;
    const int bytes = t.type[k] == T2FW_F64 ? 8 : t.type[k] == T2FW_F32 ? 4 : 2;
    const int64_t per = kPieceBytes / bytes, from = (int64_t)(p - t.first[k]) * per;
    const int64_t to = from + per < t.e[k].n ? from + per : t.e[k].n;
    const void *in = t.e[k].in;
    switch (t.type[k]) {
      case T2FW_F16: s += squares(static_cast<const __half *>(in), from, to); break;
      case T2FW_BF16: s += squares(static_cast<const __nv_bfloat16 *>(in), from, to); break;
      case T2FW_F32: s += squares(static_cast<const float *>(in), from, to); break;
      default: s += squares(static_cast<const double *>(in), from, to); break;
    }
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// max_norm < 0: only the norm is wanted.
template <int N, typename C>
__global__ void __launch_bounds__(kThreads)
grad_scale_kernel(const __grid_constant__ Table<N> t, const double *__restrict__ part, int n_part, double max_norm,
                  C *__restrict__ total, bool in_place) {
  __shared__ double red[kThreads / 32];
  dependency_wait();
  double s = 0;
  for (int i = threadIdx.x; i < n_part; i += kThreads) s += part[i];
  const C norm = (C)sqrt(block_sum(s, red));
  if (blockIdx.x == 0 && threadIdx.x == 0) *total = norm;
  if (max_norm < 0) return;
  C c = (C)max_norm / (norm + (C)1e-6);
  if (c > C(1)) c = C(1);      // a NaN stays
  if (in_place && c == C(1)) return;
  const uint32_t pieces = t.first[t.count];
  const uint32_t p0 = (uint32_t)((uint64_t)pieces * blockIdx.x / gridDim.x),
                 p1 = (uint32_t)((uint64_t)pieces * (blockIdx.x + 1) / gridDim.x);
  if (p0 == p1) return;
  int k = find(t, p1 - 1);
  for (uint32_t p = p1; p-- > p0;) {      // backwards: what the first launch read last is still in L2
    while (p < t.first[k]) --k;
    const int bytes = t.type[k] == T2FW_F64 ? 8 : t.type[k] == T2FW_F32 ? 4 : 2;
    const int64_t per = kPieceBytes / bytes, from = (int64_t)(p - t.first[k]) * per;
    const int64_t to = from + per < t.e[k].n ? from + per : t.e[k].n;
    const void *in = t.e[k].in;
    void *out = t.e[k].out;
    switch (t.type[k]) {
      case T2FW_F16: scale(static_cast<const __half *>(in), static_cast<__half *>(out), from, to, c); break;
      case T2FW_BF16: scale(static_cast<const __nv_bfloat16 *>(in), static_cast<__nv_bfloat16 *>(out), from, to, c); break;
      case T2FW_F32: scale(static_cast<const float *>(in), static_cast<float *>(out), from, to, c); break;
      default: scale(static_cast<const double *>(in), static_cast<double *>(out), from, to, c); break;
    }
  }
}

// Tensors [at, at + N) of the list; how many there were.  (The caller has checked that their pieces can be counted in 32 bits.)
template <int N>
int fill(Table<N> &t, const void *const *in, void *const *out, const int64_t *numel, const int *dtype, int at, int n) {
  int k = 0;
  t.first[0] = 0;
  for (; k < N && at + k < n; ++k) {
    t.e[k] = {in[at + k], out != nullptr ? out[at + k] : nullptr, numel[at + k]};
    t.type[k] = (uint8_t)dtype[at + k];
    t.first[k + 1] = t.first[k] + (uint32_t)ceil_div64(numel[at + k] * (int64_t)dtype_size(dtype[at + k]), kPieceBytes);
  }
  t.count = k;
  return k;
}

template <int N>
unsigned blocks_of(const Table<N> &t) {
  const uint32_t p = t.first[t.count];
  return p < (uint32_t)kMaxBlocks ? p : (unsigned)kMaxBlocks;
}

template <int N, typename C>
int run(const void *const *in, void *const *out, const int64_t *numel, const int *dtype, int n, double max_norm, C *total,
        double *part, cudaStream_t st) {
  Table<N> t;
  int n_part = 0;
  for (int at = 0; at < n;) {
    at += fill(t, in, out, numel, dtype, at, n);
    const unsigned g = blocks_of(t);
    T2FW_CHECK_CUDA(launch_dependent(grad_norm_kernel<N>, dim3(g), dim3(kThreads), 0, st, t, part + n_part));
    T2FW_CHECK_LAUNCH(1);
    n_part += (int)g;
  }
  const bool only_norm = max_norm < 0;
  for (int at = 0; at < n;) {
    at += fill(t, in, out, numel, dtype, at, n);
    const bool in_place = out != nullptr && in[0] == out[0];
    T2FW_CHECK_CUDA(launch_dependent(grad_scale_kernel<N, C>, dim3(only_norm ? 1 : blocks_of(t)), dim3(kThreads), 0, st, t,
                                     static_cast<const double *>(part), n_part, max_norm, total, in_place));
    T2FW_CHECK_LAUNCH(1);
    if (only_norm) break;
  }
  return T2FW_OK;
}

}  // namespace

size_t grad_clip_scratch_bytes(int64_t n) { return (size_t)ceil_div64(n, kTable) * kMaxBlocks * sizeof(double); }

int grad_clip(const void *const *in, void *const *out, const int64_t *numel, const int *dtype, int n, double max_norm,
              void *total, int total_dtype, void *scratch, cudaStream_t st) {
  double *part = static_cast<double *>(scratch);
  if (total_dtype == T2FW_F64)
    return run<kTable>(in, out, numel, dtype, n, max_norm, static_cast<double *>(total), part, st);
  return run<kTable>(in, out, numel, dtype, n, max_norm, static_cast<float *>(total), part, st);
}

}  // namespace t2fw
