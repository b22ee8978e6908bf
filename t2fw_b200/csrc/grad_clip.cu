// Global norm of a list of tensors and scaling by it:
//
//   total = sqrt(sum over all tensors and elements of g^2),   c = min(1, max_norm / (total + 1e-6)),   g' = c g
//
// Two launches.  The first leaves one partial sum per block; the second adds them up in each block, in the same order, and
// scales.  The tensors' addresses and sizes travel as kernel arguments, so a call needs no table in device memory and can be
// captured.  Work is cut into pieces of 32 KB that begin at 16-byte boundaries, whatever the tensor's own address; a block takes
// consecutive ones.  Bound by memory: the sums take one conversion to fp64 per vector of 16-bit values, per value in fp32; the
// second launch walks backwards, from what is still in L2.  Measured on 70 M values: norm 26 us in 16 bits and 45 in fp32 (82 and
// 95 % of the copy bandwidth), clipped copy 71 and 145 us (three passes over the data: 90 and 89 %).
#include "glr.cuh"

namespace t2fw {

namespace {

constexpr int kTable = 512, kSmallTable = 64, kThreads = 256, kPieceBytes = 32768, kVectors = kPieceBytes / (16 * kThreads), kMaxBlocks = 592;

// At most four blocks for each of 148 SMs, as many as fit at once: 70 M bf16 values, norm and clipped copy, us: with half of them
// 32 / 84, with 592 26.3 / 71.4, with twice as many 26.4 / 69.9, but 10 M fp32 values in place 13.6 instead of 11.7.
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

// Sum of squares of a vector, in fp64.  For a total in fp32, the eight squares of 16-bit values, each of them exact, are added in
// fp32 first, in a tree: off by 3 * 2^-24 at most, so a total by half of that and its own rounding (one behind the other they
// lose up to 7 * 2^-24, always the same way, where one value in eight is large).  Where the sum is not well inside fp32's range,
// which bf16 can leave, in fp64 too.
template <typename T>
__device__ __forceinline__ double squares(const uint4 &u, bool exact) {
  if constexpr (sizeof(T) == 2) {
    float v[8], p[4];
    glr::unpack<T, 8>(u, v);
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = v[2 * k] * v[2 * k] + v[2 * k + 1] * v[2 * k + 1];
    const float q = (p[0] + p[1]) + (p[2] + p[3]);
    if (!exact && q > 0x1p-90f && q < 0x1p120f) return (double)q;
    if (((u.x | u.y | u.z | u.w) & 0x7fff7fffu) == 0) return 0.0;
    double s = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += (double)v[k] * (double)v[k];
    return s;
  } else {
    constexpr int V = 16 / sizeof(T);
    const T *p = reinterpret_cast<const T *>(&u);
    double s = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) s += (double)p[k] * (double)p[k];
    return s;
  }
}

// Where a piece lies: `at` its first byte and [from, to) the tensor's own bytes, all counted from the 16-byte boundary at or
// below the tensor's address.
struct Piece {
  const unsigned char *in;
  int64_t at, from, to;
};
template <int N>
__device__ __forceinline__ Piece piece_of(const Table<N> &t, int k, uint32_t p, int bytes) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(t.e[k].in);
  Piece r;
  r.from = (int64_t)(a & 15);
  r.in = static_cast<const unsigned char *>(t.e[k].in) - r.from;
  r.to = r.from + t.e[k].n * bytes;
  r.at = (int64_t)(p - t.first[k]) * kPieceBytes;
  return r;
}

template <typename T>
__device__ __forceinline__ double piece_squares(const Piece &r, bool exact) {
  double s = 0;
  uint4 u[kVectors];
#pragma unroll
  for (int j = 0; j < kVectors; ++j) {
    const int64_t o = r.at + (int64_t)(threadIdx.x + j * kThreads) * 16;
    u[j] = make_uint4(0, 0, 0, 0);
    if (o >= r.from && o + 16 <= r.to) {
      u[j] = *reinterpret_cast<const uint4 *>(r.in + o);
    } else if (o + 16 > r.from && o < r.to) {      // the tensor's first or last vector
      T *e = reinterpret_cast<T *>(&u[j]);
#pragma unroll
      for (int k = 0; k < 16 / (int)sizeof(T); ++k) {
        const int64_t q = o + k * (int64_t)sizeof(T);
        if (q >= r.from && q < r.to) e[k] = *reinterpret_cast<const T *>(r.in + q);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kVectors; ++j) s += squares<T>(u[j], exact);
  return s;
}

// `out` is the address that corresponds to r.in; whole vectors where it is aligned too.
template <typename T, typename C>
__device__ __forceinline__ void piece_scale(const Piece &r, unsigned char *out, C c) {
  using A = typename Elem<T>::acc;
  constexpr int V = 16 / sizeof(T), kHalf = kVectors / 2;
  const bool aligned = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  if (aligned) {
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      uint4 u[kHalf];
      const int64_t o0 = r.at + (int64_t)(threadIdx.x + h * kHalf * kThreads) * 16;
#pragma unroll
      for (int j = 0; j < kHalf; ++j) {
        const int64_t o = o0 + j * kThreads * 16;
        if (o >= r.from && o + 16 <= r.to) u[j] = __ldcs(reinterpret_cast<const uint4 *>(r.in + o));
      }
#pragma unroll
      for (int j = 0; j < kHalf; ++j) {
        const int64_t o = o0 + j * kThreads * 16;
        if (o >= r.from && o + 16 <= r.to) {
          A v[V];
          glr::unpack<T, V>(u[j], v);
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] *= (A)c;
          __stcs(reinterpret_cast<uint4 *>(out + o), glr::pack<T, V>(v));
        }
      }
    }
    if (r.at >= r.from && r.at + kPieceBytes <= r.to) return;
  }
  // the tensor's first and last vector, and outputs at another offset within 16 bytes: element by element
#pragma unroll 1
  for (int j = 0; j < kVectors; ++j) {
    const int64_t o = r.at + (int64_t)(threadIdx.x + j * kThreads) * 16;
    if (aligned && o >= r.from && o + 16 <= r.to) continue;
#pragma unroll 1
    for (int64_t q = o > r.from ? o : r.from; q < o + 16 && q < r.to; q += (int64_t)sizeof(T))
      Elem<T>::st(reinterpret_cast<T *>(out + q), (A)Elem<T>::ld(reinterpret_cast<const T *>(r.in + q)) * (A)c);
  }
}

template <int N>
__global__ void __launch_bounds__(kThreads, 4)
grad_norm_kernel(const __grid_constant__ Table<N> t, double *__restrict__ part, bool exact) {
  __shared__ double red[kThreads / 32];
  dependency_wait();
  const uint32_t pieces = t.first[t.count];
  const uint32_t p0 = (uint32_t)((uint64_t)pieces * blockIdx.x / gridDim.x),
                 p1 = (uint32_t)((uint64_t)pieces * (blockIdx.x + 1) / gridDim.x);
  int k = find(t, p0);
  double s = 0;
  for (uint32_t p = p0; p < p1; ++p) {
    while (p >= t.first[k + 1]) ++k;
    switch (t.type[k]) {
      case T2FW_F16: s += piece_squares<__half>(piece_of(t, k, p, 2), exact); break;
      case T2FW_BF16: s += piece_squares<__nv_bfloat16>(piece_of(t, k, p, 2), exact); break;
      case T2FW_F32: s += piece_squares<float>(piece_of(t, k, p, 4), exact); break;
      default: s += piece_squares<double>(piece_of(t, k, p, 8), exact); break;
    }
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// max_norm < 0: only the norm is wanted.
// Four blocks to an SM leave 64 registers, with which the element-by-element ends spill 80 bytes; with three blocks nothing spills, and
// 70 M bf16 values take 78 us instead of 71.
template <int N, typename C>
__global__ void __launch_bounds__(kThreads, 4)
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
    unsigned char *out = static_cast<unsigned char *>(t.e[k].out) - (reinterpret_cast<uintptr_t>(t.e[k].in) & 15);
    switch (t.type[k]) {
      case T2FW_F16: piece_scale<__half>(piece_of(t, k, p, 2), out, c); break;
      case T2FW_BF16: piece_scale<__nv_bfloat16>(piece_of(t, k, p, 2), out, c); break;
      case T2FW_F32: piece_scale<float>(piece_of(t, k, p, 4), out, c); break;
      default: piece_scale<double>(piece_of(t, k, p, 8), out, c); break;
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
    const int64_t lead = (int64_t)(reinterpret_cast<uintptr_t>(in[at + k]) & 15);
    t.first[k + 1] = t.first[k] + (uint32_t)ceil_div64(lead + numel[at + k] * (int64_t)dtype_size(dtype[at + k]), kPieceBytes);
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
    T2FW_CHECK_CUDA(launch_dependent(grad_norm_kernel<N>, dim3(g), dim3(kThreads), 0, st, t, part + n_part,
                                     sizeof(C) == 8));
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
  // a launch copies its whole table, 15 KB or 2: 28 small tensors 6.3 and 6.2 us on the device
  if (n <= kSmallTable) return run<kSmallTable>(in, out, numel, dtype, n, max_norm, static_cast<float *>(total), part, st);
  return run<kTable>(in, out, numel, dtype, n, max_norm, static_cast<float *>(total), part, st);
}

}  // namespace t2fw
