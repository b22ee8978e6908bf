// Root-mean-square norm over rows of D, with or without the addition of a residual, and its gradients:
//
//   s = x + residual,  rstd = 1 / sqrt(mean(s^2) + eps),  y = s rstd w
//   g = w dy:   d_s = rstd (g - s rstd^2 mean(g s)) + (gradient of s from its other use) ,   d_w = sum over rows of dy s rstd
//
// x and the residual share the gradient d_s.  The 8-bit form leaves q = e4m3(y / scale) with scale = max|y| / 448 per row;
// max|y| = rstd max|s w|, so both sums of a row are formed at once, and so are both of the gradients' (s^2 and g s).
//
// Bound by memory: a row stays in registers from its one read to its write.  y and q are computed from s before its rounding to
// the storage type; the gradients read s as it was written, and form rstd anew from it, so nothing else is saved.  Measured, with
// nothing in L2: 16384 x 2048 fp16 with the residual 45 us forward (91 % of the copy bandwidth), 40 with the 8-bit output (90 %),
// 47 backward (88 %); 8192 x 768 fp16 8.2 and 15.3 us (the weight gradient's second launch is some 3 of them).
#pragma once

#include <cuda_fp8.h>

#include <initializer_list>
#include <type_traits>

#include "glr.cuh"

namespace t2fw {
namespace rms {

using glr::Raw;
using glr::max_nan;
using glr::pack;
using glr::unpack;

constexpr float kE4m3Max = 448.f, kMinScale = 1e-30f;

__device__ __forceinline__ double max_nan(double a, double b) { return a > b || a != a ? a : b; }
__device__ __forceinline__ float inv_sqrt(float v) { return 1.f / sqrtf(v); }
__device__ __forceinline__ double inv_sqrt(double v) { return 1.0 / sqrt(v); }

// Two reductions over the GS threads of a row at once, the results in each of them; kMax: the second is a maximum.  `red`
// alternates between two halves, so a block needs one barrier per row.
template <int GS, bool kMax, typename A>
__device__ __forceinline__ void row_reduce(A &a, A &b, A (*red)[2]) {
#pragma unroll
  for (int o = (GS < 32 ? GS : 32) / 2; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    const A t = __shfl_xor_sync(0xffffffffu, b, o);
    if constexpr (kMax) b = max_nan(b, t);
    else b += t;
  }
  if constexpr (GS > 32) {
    constexpr int W = GS / 32;
    if ((threadIdx.x & 31) == 0) {
      red[threadIdx.x >> 5][0] = a;
      red[threadIdx.x >> 5][1] = b;
    }
    __syncthreads();
    a = red[0][0];
    b = red[0][1];
#pragma unroll
    for (int i = 1; i < W; ++i) {
      a += red[i][0];
      if constexpr (kMax) b = max_nan(b, red[i][1]);
      else b += red[i][1];
    }
  }
}

// Rows whose squares leave the range of A (bf16 and fp32 reach beyond 2^64, and below 2^-55 where eps is no larger) are done once
// more, with values that a power of two brings inside, when a block has been through its other rows.  Which they are is told from
// sums formed in the same order, and the sums of a row are the same in each of its threads, so all decide alike.  fp16 values and
// sums of two lie between 2^-24 and 2^17: never.  A NaN or an infinity is done again and stays.
// (In the loop over the rows the same code, skipped, cost 8 % of the 8-bit form's time at 16384 x 2048 bf16, and up to 17 %.)
template <typename T> constexpr bool kLeaves = !std::is_same<T, __half>::value;
template <typename A> struct Range;
template <> struct Range<float> {
  static constexpr float most = 0x1.fffffep127f, least = 0x1p-110f, large = 0x1p40f, down = 0x1p-100f, up = 0x1p90f;
};
template <> struct Range<double> {
  static constexpr double most = 0x1.fffffffffffffp1023, least = 0x1p-900, large = 0x1p300, down = 0x1p-600, up = 0x1p600;
};
template <typename A>
__device__ __forceinline__ bool strays(A ss, A mean) { return !(ss <= Range<A>::most) || mean < Range<A>::least; }
// a maximum of products, where zero is no stray
template <typename A>
__device__ __forceinline__ bool strays(A v) { return !(v <= Range<A>::most) || (v > A(0) && v < Range<A>::least); }
template <typename A>
__device__ __forceinline__ A power(A largest) {
  return largest >= Range<A>::large ? Range<A>::down : largest <= A(1) / Range<A>::large ? Range<A>::up : A(1);
}

// V values as e4m3, one behind the other.
template <int V> struct Raw8 { using type = uint2; };
template <> struct Raw8<4> { using type = uint32_t; };
template <> struct Raw8<2> { using type = uint16_t; };
template <> struct Raw8<1> { using type = __nv_fp8_storage_t; };
template <int V>
__device__ __forceinline__ typename Raw8<V>::type pack8(const float (&v)[V]) {
  if constexpr (V == 1) {
    return __nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
  } else {
    typename Raw8<V>::type u;
    __nv_fp8x2_storage_t *p = reinterpret_cast<__nv_fp8x2_storage_t *>(&u);
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      p[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    return u;
  }
}

template <typename T>
struct FwdArgs {
  const T *x, *r, *w;      // r: null without a residual
  T *y, *sum;
  void *q;
  float *scale;
  int64_t rows, D;
  double eps;
};
template <typename T>
struct BwdArgs {
  const T *dy, *dsum, *s, *w;      // dsum: null for zero
  T *ds;
  typename Elem<T>::acc *part;
  int64_t rows, D;
  double eps;
};

template <int GS> constexpr int block_of() { return GS <= 32 ? 256 : GS; }

// sums += a b, element by element; pairs of fp32 in one instruction
template <typename A, int V>
__device__ __forceinline__ void add_products(A (&sums)[2], const A (&a)[V], const A (&b)[V]) {
  if constexpr (V == 1) {
    sums[0] = fma(a[0], b[0], sums[0]);
  } else {
#pragma unroll
    for (int k = 0; k < V; k += 2) {
      const A x[2] = {a[k], a[k + 1]}, y[2] = {b[k], b[k + 1]};
      glr::fma_v(sums, x, y, sums);
    }
  }
}

// A row on GS threads, NV vectors of V elements each, in registers; the next row's values are on their way while a row is
// reduced.  GS <= 32: several rows in a block, a warp or a part of one each.
// The 8-bit form of 16-bit rows on 128 or 512 threads is held to the registers with which 8 or 2 blocks fit an SM: 16384 x 2048 bf16
// 44.9 -> 38.6 us, 4096 x 8192 fp16 45.7 -> 38.5.
template <typename T, int V, int NV, int GS, bool k8>
__global__ void __launch_bounds__(block_of<GS>(), k8 && sizeof(T) == 2 && NV * V == 16 ? (GS == 128 ? 8 : GS == 512 ? 2 : 0) : 0)
rms_fwd_kernel(const FwdArgs<T> p) {
  using A = typename Elem<T>::acc;
  using R = typename Raw<T, V>::type;
  constexpr int kRows = block_of<GS>() / GS;
  __shared__ A red[kLeaves<T> ? 4 : 2][GS > 32 ? GS / 32 : 1][2];
  dependency_wait();
  const int tid = threadIdx.x % GS;
  const int64_t step = (int64_t)gridDim.x * kRows;
  const A inv_d = A(1) / A(p.D), eps = (A)p.eps;
  const bool add = p.r != nullptr;
  R x[NV], r[NV], w[NV];
  bool on[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) on[i] = (int64_t)(tid + i * GS) * V < p.D;
  auto load = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t at = row * p.D + (int64_t)(tid + i * GS) * V;
      x[i] = R{};
      if (on[i]) x[i] = *reinterpret_cast<const R *>(p.x + at);
      if (add) {
        r[i] = R{};
        if (on[i]) r[i] = *reinterpret_cast<const R *>(p.r + at);
      }
    }
  };
  // all rows of a block take the same number of rounds, so that whole warps meet in the reductions
  const int64_t first = (int64_t)blockIdx.x * kRows;
  int64_t row = first + threadIdx.x / GS;
  bool valid = row < p.rows;
#pragma unroll
  for (int i = 0; i < NV; ++i) x[i] = r[i] = w[i] = R{};
  if (valid) load(row);
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (on[i]) w[i] = *reinterpret_cast<const R *>(p.w + (tid + i * GS) * V);
  bool again = false;
  for (int64_t base = first, half = 0; base < p.rows; base += step, row += step, half ^= 1) {
    A s[NV][V], sums[2] = {A(0), A(0)}, top = A(0);
    valid = row < p.rows;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      unpack<T, V>(x[i], s[i]);
      if (add) {
        A t[V];
        unpack<T, V>(r[i], t);
#pragma unroll
        for (int k = 0; k < V; ++k) s[i][k] += t[k];
        if (on[i] && valid) *reinterpret_cast<R *>(p.sum + row * p.D + (int64_t)(tid + i * GS) * V) = pack<T, V>(s[i]);
      }
    }
    if (row + step < p.rows) load(row + step);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      A wv[V];
      if constexpr (k8) unpack<T, V>(w[i], wv);
      add_products(sums, s[i], s[i]);
      if constexpr (k8) {
        glr::mul_v(wv, wv, s[i]);
#pragma unroll
        for (int k = 0; k < V; ++k) top = max_nan(top, fabsf(wv[k]));
      }
    }
    A ss = sums[0] + sums[1];
    row_reduce<GS, k8>(ss, top, red[half]);
    const A mean = ss * inv_d + eps, rstd = inv_sqrt(mean);
    if constexpr (kLeaves<T>) again |= valid && (strays(ss, mean) || (k8 && strays(top)));
    A unit = A(1);      // 1 / scale, of 1e30 at most: a factor of its own, since rstd / scale leaves the range for rows of (nearly) nothing
    if constexpr (k8) {
      const float scale = max_nan(top * rstd / kE4m3Max, kMinScale);
      if (tid == 0 && valid) p.scale[row] = scale;
      unit = 1.f / scale;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      A wv[V];
      unpack<T, V>(w[i], wv);
      A fv[V], uv[V];
#pragma unroll
      for (int k = 0; k < V; ++k) fv[k] = rstd, uv[k] = unit;
      glr::mul_v(s[i], s[i], fv);
      glr::mul_v(s[i], s[i], wv);
      if constexpr (k8) glr::mul_v(s[i], s[i], uv);
      const int64_t at = row * p.D + (int64_t)(tid + i * GS) * V;
      if (on[i] && valid) {
        if constexpr (k8) *reinterpret_cast<typename Raw8<V>::type *>(static_cast<unsigned char *>(p.q) + at) = pack8<V>(s[i]);
        else *reinterpret_cast<R *>(p.y + at) = pack<T, V>(s[i]);
      }
    }
  }
  if constexpr (kLeaves<T>) {
    if (GS <= 32 ? !__any_sync(0xffffffffu, again) : !again) return;
    int turn = 0;
#pragma unroll 1
    for (int64_t base = first; base < p.rows; base += step) {
      row = base + threadIdx.x / GS;
      valid = row < p.rows;
      const int64_t at = row * p.D;
      A none = A(0), most = A(0), sum = A(0);
      A sums[2] = {A(0), A(0)};
#pragma unroll 1
      for (int i = 0; i < NV; ++i) {
        const int64_t d = (int64_t)(tid + i * GS) * V;
        if (!valid || d >= p.D) continue;
        A s[V], t[V];
        unpack<T, V>(*reinterpret_cast<const R *>(p.x + at + d), s);
        if (add) {
          unpack<T, V>(*reinterpret_cast<const R *>(p.r + at + d), t);
#pragma unroll
          for (int k = 0; k < V; ++k) s[k] += t[k];
        }
        add_products(sums, s, s);
        if constexpr (k8) {
          unpack<T, V>(*reinterpret_cast<const R *>(p.w + d), t);
          glr::mul_v(t, t, s);
#pragma unroll
          for (int k = 0; k < V; ++k) most = max_nan(most, fabs(t[k]));
        }
      }
      sum = sums[0] + sums[1];
      row_reduce<GS, k8>(sum, most, red[2 + (turn ^= 1)]);
      const bool mine = valid && (strays(sum, sum * inv_d + eps) || (k8 && strays(most)));
      if (GS <= 32 ? !__any_sync(0xffffffffu, mine) : !mine) continue;
      const int64_t n = mine ? p.D : 0;
      auto value = [&](int64_t d) {
        A v = Elem<T>::ld(p.x + at + d);
        if (add) v += (A)Elem<T>::ld(p.r + at + d);
        return v;
      };
      most = sum = none = A(0);
#pragma unroll 1
      for (int64_t d = tid; d < n; d += GS) most = max_nan(most, fabs(value(d)));
      row_reduce<GS, true>(none, most, red[2 + (turn ^= 1)]);
      const A pre = power(most);
#pragma unroll 1
      for (int64_t d = tid; d < n; d += GS) {
        const A v = value(d) * pre;
        sum += v * v;
      }
      row_reduce<GS, false>(sum, none, red[2 + (turn ^= 1)]);
      const A rstd = inv_sqrt(sum * inv_d + eps * pre * pre);
      A unit = A(1);
      if constexpr (k8) {
        most = none = A(0);
#pragma unroll 1
        for (int64_t d = tid; d < n; d += GS) most = max_nan(most, fabs(value(d) * pre * rstd * (A)Elem<T>::ld(p.w + d)));
        row_reduce<GS, true>(none, most, red[2 + (turn ^= 1)]);
        const float scale = max_nan(most / kE4m3Max, kMinScale);
        if (tid == 0 && mine) p.scale[row] = scale;
        unit = 1.f / scale;
      }
#pragma unroll 1
      for (int64_t v0 = tid * V; v0 < n; v0 += GS * V)      // a thread writes what it has written above
#pragma unroll 1
        for (int64_t d = v0; d < v0 + V; ++d) {
          const A v[1] = {value(d) * pre * rstd * (A)Elem<T>::ld(p.w + d) * unit};
          if constexpr (k8) static_cast<__nv_fp8_storage_t *>(p.q)[at + d] = pack8<1>(v);
          else Elem<T>::st(p.y + at + d, v[0]);
        }
    }
  }
}

// The same for the gradients.  A thread sums the weight gradient of its columns over its rows in registers; a block leaves one
// line of `part`, and rms_dw_kernel adds the lines up, always in the same order.  Rows on a warp or less are not fetched ahead:
// 16 warps to an SM with a row each keep more in flight than 8 with two (the registers would not hold more).
template <typename T, int V, int NV, int GS>
__global__ void __launch_bounds__(block_of<GS>(), GS >= 512 ? 1 : GS == 128 ? 4 : 2)
rms_bwd_kernel(const BwdArgs<T> p) {
  using A = typename Elem<T>::acc;
  using R = typename Raw<T, V>::type;
  constexpr int kRows = block_of<GS>() / GS, kCols = NV * GS * V;
  constexpr bool kAhead = GS > 32, kShared = GS <= 32 && NV > 2;      // where registers are short the weights lie in shared memory
  __shared__ A red[kLeaves<T> ? 4 : 2][GS > 32 ? GS / 32 : 1][2];
  __shared__ R s_w[kShared ? NV * GS : 1];
  __shared__ A lines[kRows > 1 ? kRows / 2 : 1][kRows > 1 ? kCols : 1];
  dependency_wait();
  const int tid = threadIdx.x % GS, group = threadIdx.x / GS;
  const int64_t step = (int64_t)gridDim.x * kRows;
  const A inv_d = A(1) / A(p.D), eps = (A)p.eps;
  constexpr bool kAheadSum = kAhead && NV * sizeof(R) <= 32;      // a third array ahead, where the registers hold it
  R dy[NV], s[NV], ds_in[NV], w[kShared ? 1 : NV];
  bool on[NV];
  A dw[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    on[i] = (int64_t)(tid + i * GS) * V < p.D;
    dy[i] = s[i] = ds_in[i] = R{};
#pragma unroll
    for (int k = 0; k < V; ++k) dw[i][k] = A(0);
  }
  auto load = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t at = row * p.D + (int64_t)(tid + i * GS) * V;
      if (on[i]) {
        dy[i] = *reinterpret_cast<const R *>(p.dy + at);
        s[i] = *reinterpret_cast<const R *>(p.s + at);
        if ((kAheadSum || !kAhead) && p.dsum != nullptr) ds_in[i] = *reinterpret_cast<const R *>(p.dsum + at);
      }
    }
  };
  const int64_t first = (int64_t)blockIdx.x * kRows;
  int64_t row = first + group;
  if (kAhead && row < p.rows) load(row);
  if constexpr (kShared) {
    for (int i = threadIdx.x; i < NV * GS; i += block_of<GS>())
      s_w[i] = (int64_t)i * V < p.D ? *reinterpret_cast<const R *>(p.w + i * V) : R{};
    __syncthreads();
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      w[i] = R{};
      if (on[i]) w[i] = *reinterpret_cast<const R *>(p.w + (tid + i * GS) * V);
    }
  }
  auto weight = [&](int i, A (&v)[V]) {
    if constexpr (kShared) unpack<T, V>(s_w[tid + i * GS], v);
    else unpack<T, V>(w[i], v);
  };
  bool again = false;
  for (int64_t base = first, half = 0; base < p.rows; base += step, row += step, half ^= 1) {
    const bool valid = row < p.rows;
    if (!kAhead && valid) load(row);
    R up[NV], cdy[NV], cs[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (kAhead && !kAheadSum && p.dsum != nullptr && on[i] && valid)
        ds_in[i] = *reinterpret_cast<const R *>(p.dsum + row * p.D + (int64_t)(tid + i * GS) * V);
      up[i] = ds_in[i], cdy[i] = dy[i], cs[i] = s[i];
    }
    if (kAhead && row + step < p.rows) load(row + step);
    A s2[2] = {A(0), A(0)}, g2[2] = {A(0), A(0)};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      A sv[V], g[V], wv[V];
      unpack<T, V>(cs[i], sv);
      unpack<T, V>(cdy[i], g);
      weight(i, wv);
      add_products(s2, sv, sv);
      glr::mul_v(g, g, wv);
      add_products(g2, g, sv);
    }
    A ss = s2[0] + s2[1], gs = g2[0] + g2[1];
    row_reduce<GS, false>(ss, gs, red[half]);
    const A mean = ss * inv_d + eps;
    A rstd = inv_sqrt(mean), m = gs * inv_d * rstd * rstd * rstd;
    if constexpr (kLeaves<T>) {
      const bool stray = valid && strays(ss, mean);
      again |= stray;
      if (stray) rstd = m = A(0);      // nothing for the weight gradient yet
    }
    if (valid) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        A sv[V], g[V], wv[V], v[V], k1[V], k2[V];
        unpack<T, V>(cs[i], sv);
        unpack<T, V>(cdy[i], g);
        weight(i, wv);
#pragma unroll
        for (int k = 0; k < V; ++k) k1[k] = rstd, k2[k] = -m;
        glr::mul_v(g, g, k1);              // rstd dy
        glr::fma_v(dw[i], g, sv, dw[i]);
        glr::mul_v(v, sv, k2);
        glr::fma_v(v, g, wv, v);
        if (p.dsum != nullptr) {
          A u[V];
          unpack<T, V>(up[i], u);
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] += u[k];
        }
        if (on[i]) *reinterpret_cast<R *>(p.ds + row * p.D + (int64_t)(tid + i * GS) * V) = pack<T, V>(v);
      }
    }
  }
  if constexpr (kLeaves<T>) {
    if (GS <= 32 ? __any_sync(0xffffffffu, again) : again) {
      int turn = 0;
#pragma unroll 1
      for (int64_t base = first; base < p.rows; base += step) {
        row = base + group;
        const bool valid = row < p.rows;
        const int64_t at = row * p.D;
        A none = A(0), most = A(0), sums[2] = {A(0), A(0)}, dot = A(0);
#pragma unroll 1
        for (int i = 0; i < NV; ++i) {
          const int64_t d = (int64_t)(tid + i * GS) * V;
          if (!valid || d >= p.D) continue;
          A sv[V];
          unpack<T, V>(*reinterpret_cast<const R *>(p.s + at + d), sv);
          add_products(sums, sv, sv);
        }
        A sum = sums[0] + sums[1];
        row_reduce<GS, false>(sum, none, red[2 + (turn ^= 1)]);
        const bool mine = valid && strays(sum, sum * inv_d + eps);
        if (GS <= 32 ? !__any_sync(0xffffffffu, mine) : !mine) continue;
        const int64_t n = mine ? p.D : 0;
        sum = none = A(0);
#pragma unroll 1
        for (int64_t d = tid; d < n; d += GS) most = max_nan(most, fabs((A)Elem<T>::ld(p.s + at + d)));
        row_reduce<GS, true>(none, most, red[2 + (turn ^= 1)]);
        const A pre = power(most);
#pragma unroll 1
        for (int64_t d = tid; d < n; d += GS) {
          const A v = (A)Elem<T>::ld(p.s + at + d) * pre;
          sum += v * v;
        }
        row_reduce<GS, false>(sum, none, red[2 + (turn ^= 1)]);
        const A rstd = inv_sqrt(sum * inv_d + eps * pre * pre);
#pragma unroll 1
        for (int64_t d = tid; d < n; d += GS)
          dot += (A)Elem<T>::ld(p.dy + at + d) * (A)Elem<T>::ld(p.w + d) * ((A)Elem<T>::ld(p.s + at + d) * pre * rstd);
        row_reduce<GS, false>(dot, none, red[2 + (turn ^= 1)]);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const int64_t d = (int64_t)(tid + i * GS) * V + k;
            if (d < n) {
              const A sv = (A)Elem<T>::ld(p.s + at + d) * pre * rstd, g = Elem<T>::ld(p.dy + at + d);
              A v = (g * (A)Elem<T>::ld(p.w + d) - sv * (dot * inv_d)) * rstd * pre;
              if (p.dsum != nullptr) v += (A)Elem<T>::ld(p.dsum + at + d);
              Elem<T>::st(p.ds + at + d, v);
              dw[i][k] += g * sv;
            }
          }
      }
    }
  }
  // rows of a block: halve their number until one line is left
#pragma unroll
  for (int n = kRows / 2; n > 0; n >>= 1) {
    __syncthreads();
    if (group >= n && group < 2 * n) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) lines[group - n][(i * V + k) * GS + tid] = dw[i][k];
    }
    __syncthreads();
    if (group < n) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) dw[i][k] += lines[group][(i * V + k) * GS + tid];
    }
  }
  if (group == 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (on[i]) {
        A *to = p.part + (int64_t)blockIdx.x * p.D + (tid + i * GS) * V;
        if constexpr (V * sizeof(A) % 16 == 0) {      // 16 bytes at a time: single values of a thread lie 32 bytes from the next one's
          constexpr int W = 16 / (int)sizeof(A);
#pragma unroll
          for (int k = 0; k < V; k += W) {
            A part[W];
#pragma unroll
            for (int j = 0; j < W; ++j) part[j] = dw[i][k + j];
            *reinterpret_cast<uint4 *>(to + k) = glr::pack<A, W>(part);
          }
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k) to[k] = dw[i][k];
        }
      }
  }
}

// 32 columns of the lines that the blocks left, each warp every 32nd line.
template <typename T>
__global__ void __launch_bounds__(1024)
rms_dw_kernel(const typename Elem<T>::acc *__restrict__ part, T *__restrict__ dw, int n, int64_t D) {
  using A = typename Elem<T>::acc;
  __shared__ A sums[32][33];
  dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t d = (int64_t)blockIdx.x * 32 + lane;
  A v = A(0);
  if (d < D) {
#pragma unroll 8
    for (int i = warp; i < n; i += 32) v += part[(int64_t)i * D + d];
  }
  sums[warp][lane] = v;
  __syncthreads();
  v = warp_sum(sums[lane][warp]);      // a warp per column now
  const int64_t c = (int64_t)blockIdx.x * 32 + warp;
  if (lane == 0 && c < D) Elem<T>::st(dw + c, v);
}

// ---- rows that no registers hold: a block per row, read again for each use ------------------------------
template <typename T, bool k8>
__global__ void __launch_bounds__(512)
rms_fwd_long_kernel(const FwdArgs<T> p) {
  using A = typename Elem<T>::acc;
  __shared__ A red[4][16][2];
  dependency_wait();
  const int64_t base = (int64_t)blockIdx.x * p.D;
  auto value = [&](int64_t d) {
    A s = Elem<T>::ld(p.x + base + d);
    if (p.r != nullptr) s += (A)Elem<T>::ld(p.r + base + d);
    return s;
  };
  A ss = A(0), top = A(0), pre = A(1);
  for (int64_t d = threadIdx.x; d < p.D; d += 512) {
    const A s = value(d);
    if (p.r != nullptr) Elem<T>::st(p.sum + base + d, s);
    ss += s * s;
    if constexpr (k8) top = max_nan(top, fabsf(s * (A)Elem<T>::ld(p.w + d)));
  }
  row_reduce<512, k8>(ss, top, red[0]);
  const A mean = ss / A(p.D) + (A)p.eps;
  A rstd = inv_sqrt(mean), y_top = top * rstd;
  if constexpr (kLeaves<T>) {
    if (strays(ss, mean) || (k8 && strays(top))) {
      A sum = A(0), none = A(0), most = A(0);
      for (int64_t d = threadIdx.x; d < p.D; d += 512) most = max_nan(most, fabs(value(d)));
      row_reduce<512, true>(none, most, red[1]);
      pre = power(most);
      for (int64_t d = threadIdx.x; d < p.D; d += 512) {
        const A s = value(d) * pre;
        sum += s * s;
      }
      row_reduce<512, false>(sum, none, red[2]);
      rstd = inv_sqrt(sum / A(p.D) + (A)p.eps * pre * pre);
      if constexpr (k8) {
        y_top = A(0);
        for (int64_t d = threadIdx.x; d < p.D; d += 512) y_top = max_nan(y_top, fabsf(value(d) * pre * rstd * (A)Elem<T>::ld(p.w + d)));
        row_reduce<512, true>(none, y_top, red[3]);
      }
    }
  }
  A unit = A(1);
  if constexpr (k8) {
    const float scale = max_nan(y_top / kE4m3Max, kMinScale);
    if (threadIdx.x == 0) p.scale[blockIdx.x] = scale;
    unit = 1.f / scale;
  }
  for (int64_t d = threadIdx.x; d < p.D; d += 512) {
    A v[1] = {value(d) * pre * rstd * (A)Elem<T>::ld(p.w + d)};
    if constexpr (k8) v[0] *= unit;
    if constexpr (k8) static_cast<__nv_fp8_storage_t *>(p.q)[base + d] = pack8<1>(v);
    else Elem<T>::st(p.y + base + d, v[0]);
  }
}

// Blocks walk rows; the weight gradient of a block's rows is summed in its own line of `part`.
template <typename T>
__global__ void __launch_bounds__(512)
rms_bwd_long_kernel(const BwdArgs<T> p) {
  using A = typename Elem<T>::acc;
  __shared__ A red[5][16][2];
  dependency_wait();
  A *const mine = p.part + (int64_t)blockIdx.x * p.D;
  bool first = true;
  int half = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, half ^= 1) {
    const int64_t base = row * p.D;
    A ss = A(0), gs = A(0);
    for (int64_t d = threadIdx.x; d < p.D; d += 512) {
      const A sv = Elem<T>::ld(p.s + base + d);
      ss += sv * sv;
      gs += (A)Elem<T>::ld(p.dy + base + d) * (A)Elem<T>::ld(p.w + d) * sv;
    }
    row_reduce<512, false>(ss, gs, red[half]);
    const A ms = ss / A(p.D) + (A)p.eps;
    A pre = A(1), inner = inv_sqrt(ms), m = gs / A(p.D) * inner;
    if constexpr (kLeaves<T>) {
      if (strays(ss, ms)) {
        A sum = A(0), none = A(0), most = A(0);
        for (int64_t d = threadIdx.x; d < p.D; d += 512) most = max_nan(most, fabs((A)Elem<T>::ld(p.s + base + d)));
        row_reduce<512, true>(none, most, red[2]);
        pre = power(most);
        for (int64_t d = threadIdx.x; d < p.D; d += 512) {
          const A sv = (A)Elem<T>::ld(p.s + base + d) * pre;
          sum += sv * sv;
        }
        row_reduce<512, false>(sum, none, red[3]);
        inner = inv_sqrt(sum / A(p.D) + (A)p.eps * pre * pre);
        sum = A(0);
        for (int64_t d = threadIdx.x; d < p.D; d += 512)
          sum += (A)Elem<T>::ld(p.dy + base + d) * (A)Elem<T>::ld(p.w + d) * ((A)Elem<T>::ld(p.s + base + d) * pre * inner);
        row_reduce<512, false>(sum, none, red[4]);
        m = sum / A(p.D);
      }
    }
    const A rstd = pre * inner;
    for (int64_t d = threadIdx.x; d < p.D; d += 512) {
      const A sv = (A)Elem<T>::ld(p.s + base + d) * pre * inner, g = Elem<T>::ld(p.dy + base + d);
      A v = rstd * ((A)Elem<T>::ld(p.w + d) * g - sv * m);
      if (p.dsum != nullptr) v += (A)Elem<T>::ld(p.dsum + base + d);
      Elem<T>::st(p.ds + base + d, v);
      mine[d] = (first ? A(0) : mine[d]) + g * sv;
    }
    first = false;
  }
}

// ---- launches ---------------------------------------------------------------------------------------
// Blocks per SM that the launches below ask for: as many as keep some 100 KB of loads in flight.
template <int GS> constexpr int blocks_per_sm() { return GS <= 32 ? 4 : GS == 128 ? 8 : GS == 256 ? 4 : 2; }

template <int GS>
inline int64_t grid_of(int64_t rows, int sms, int per_sm) {
  const int64_t need = ceil_div64(rows, block_of<GS>() / GS), most = (int64_t)sms * per_sm;
  return need < most ? need : most;
}

constexpr int64_t kMostParts = 1024;      // lines of the weight gradient's partial sums; blocks of the backward launches
inline int64_t capped(int64_t n) { return n < kMostParts ? n : kMostParts; }

template <typename T, int V, int NV, int GS, bool k8>
int launch_fwd_as(const FwdArgs<T> &p, int sms, cudaStream_t st) {
  T2FW_CHECK_CUDA(launch_dependent(rms_fwd_kernel<T, V, NV, GS, k8>,
                                   dim3((unsigned)grid_of<GS>(p.rows, sms, blocks_per_sm<GS>())), dim3(block_of<GS>()), 0, st, p));
  T2FW_CHECK_LAUNCH(1);
  return T2FW_OK;
}
template <typename T, int V, int NV, int GS>
int launch_bwd_as(const BwdArgs<T> &p, int sms, int64_t *parts, cudaStream_t st) {
  constexpr int kPer = GS <= 32 && NV == 1 ? 3 : blocks_per_sm<GS>() / 2;
  *parts = capped(grid_of<GS>(p.rows, sms, kPer));
  T2FW_CHECK_CUDA(launch_dependent(rms_bwd_kernel<T, V, NV, GS>, dim3((unsigned)*parts), dim3(block_of<GS>()), 0, st, p));
  T2FW_CHECK_LAUNCH(1);
  return T2FW_OK;
}

// A row on as few threads as hold it: a part of a warp, a warp, four, eight or sixteen.  fp16, with the residual, us.  Forward, two
// vectors on a warp against one on 128 threads: 16384 x 264 8.1 / 13.6, 16384 x 512 10.1 / 13.4; against four on a warp, two of them
// empty, 10.7 and 11.5; three against one on 128 threads: 16384 x 768 15.9 / 17.9; four: 16384 x 1024 20.6 / 22.7.  Few rows would
// rather have the threads (64 x 1024 2.1 / 1.4).  Backward, two on a warp against one on 128 threads: 16384 x 264 13.8 / 23.7,
// 16384 x 512 15.3 / 25.1; one on 128 threads against two, half of them empty: 16384 x 768 28.4 / 31.6.
template <typename T, int V, bool k8>
int launch_fwd_v(const FwdArgs<T> &p, int sms, cudaStream_t st) {
  const int64_t n = ceil_div64(p.D, V);
  constexpr int M = V * sizeof(T) < 16 ? 2 : 1;      // less than 16 bytes to a vector: twice as many per thread
  if (n <= 8 * M) return launch_fwd_as<T, V, 1 * M, 8, k8>(p, sms, st);
  if (n <= 16 * M) return launch_fwd_as<T, V, 1 * M, 16, k8>(p, sms, st);
  if (n <= 32 * M) return launch_fwd_as<T, V, 1 * M, 32, k8>(p, sms, st);
  if (n <= 64 * M) return launch_fwd_as<T, V, 2 * M, 32, k8>(p, sms, st);
  if (n <= 96 * M) return launch_fwd_as<T, V, 3 * M, 32, k8>(p, sms, st);
  if (n <= 128 * M) return launch_fwd_as<T, V, 4 * M, 32, k8>(p, sms, st);
  if (n <= 256 * M) return launch_fwd_as<T, V, 2 * M, 128, k8>(p, sms, st);
  if (n <= 512 * M) return launch_fwd_as<T, V, 2 * M, 256, k8>(p, sms, st);
  if (n <= 1024 * M) return launch_fwd_as<T, V, 2 * M, 512, k8>(p, sms, st);
  if (n <= 2048 * M) return launch_fwd_as<T, V, 4 * M, 512, k8>(p, sms, st);
  T2FW_CHECK_CUDA(launch_dependent(rms_fwd_long_kernel<T, k8>, dim3((unsigned)p.rows), dim3(512), 0, st, p));
  T2FW_CHECK_LAUNCH(1);
  return T2FW_OK;
}
template <typename T, int V>
int launch_bwd_v(const BwdArgs<T> &p, int sms, int64_t *parts, cudaStream_t st) {
  const int64_t n = ceil_div64(p.D, V);
  constexpr int M = V * sizeof(T) < 16 ? 2 : 1;
  if (n <= 8 * M) return launch_bwd_as<T, V, 1 * M, 8>(p, sms, parts, st);
  if (n <= 16 * M) return launch_bwd_as<T, V, 1 * M, 16>(p, sms, parts, st);
  if (n <= 32 * M) return launch_bwd_as<T, V, 1 * M, 32>(p, sms, parts, st);
  if (n <= 64 * M) return launch_bwd_as<T, V, 2 * M, 32>(p, sms, parts, st);
  if (n <= 128 * M) return launch_bwd_as<T, V, 1 * M, 128>(p, sms, parts, st);
  if (n <= 256 * M) return launch_bwd_as<T, V, 2 * M, 128>(p, sms, parts, st);
  if (n <= 512 * M) return launch_bwd_as<T, V, 2 * M, 256>(p, sms, parts, st);
  if (n <= 1024 * M) return launch_bwd_as<T, V, 2 * M, 512>(p, sms, parts, st);
  if constexpr (V < 8)      // with eight values to a vector a thread's registers do not hold them
    if (n <= 2048 * M) return launch_bwd_as<T, V, 4 * M, 512>(p, sms, parts, st);
  *parts = capped(p.rows < 2 * sms ? p.rows : 2 * sms);
  T2FW_CHECK_CUDA(launch_dependent(rms_bwd_long_kernel<T>, dim3((unsigned)*parts), dim3(512), 0, st, p));
  T2FW_CHECK_LAUNCH(1);
  return T2FW_OK;
}

// A positive eps stays positive in A: a row of zeros has a finite 1 / sqrt(eps).
template <typename A>
inline double eps_in(double eps) {
  return std::is_same<A, float>::value && eps > 0 && eps < 0x1p-149 ? 0x1p-149 : eps;
}

inline bool aligned(int to, std::initializer_list<const void *> ps) {
  uintptr_t low = 0;
  for (const void *q : ps) low |= reinterpret_cast<uintptr_t>(q);
  return (low & (uintptr_t)(to - 1)) == 0;
}

}  // namespace rms

template <typename T, bool k8>
int rms_forward_t(const void *x, const void *r, const void *w, void *y, void *q, float *scale, void *sum, int64_t rows,
                  int64_t D, double eps, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const rms::FwdArgs<T> p = {static_cast<const T *>(x), static_cast<const T *>(r), static_cast<const T *>(w), static_cast<T *>(y),
                             static_cast<T *>(sum), q, scale, rows, D, rms::eps_in<typename Elem<T>::acc>(eps)};
  int sms = 0;
  const int rc = lfw_chunk_sm_count(&sms);
  if (rc != T2FW_OK) return rc;
  // 16 bytes per thread, else two elements, else one: 16384 x 1002 fp16, forward, 14.3 us against 31.6 with single elements
  if (D % V == 0 && rms::aligned(16, {x, r, w, y, q, sum})) return rms::launch_fwd_v<T, V, k8>(p, sms, st);
  if constexpr (sizeof(T) <= 4)
    if (D % 2 == 0 && rms::aligned(2 * (int)sizeof(T), {x, r, w, y, q, sum})) return rms::launch_fwd_v<T, 2, k8>(p, sms, st);
  return rms::launch_fwd_v<T, 1, k8>(p, sms, st);
}

template <typename T>
int rms_backward_t(const void *dy, const void *dsum, const void *s, const void *w, void *ds, void *dw, int64_t rows, int64_t D,
                   double eps, void *scratch, cudaStream_t st) {
  using A = typename Elem<T>::acc;
  constexpr int V = 16 / (int)sizeof(T);
  const rms::BwdArgs<T> p = {static_cast<const T *>(dy), static_cast<const T *>(dsum), static_cast<const T *>(s),
                             static_cast<const T *>(w), static_cast<T *>(ds), static_cast<A *>(scratch), rows, D, rms::eps_in<A>(eps)};
  int sms = 0;
  int64_t parts = 0;
  int rc = lfw_chunk_sm_count(&sms);
  if (rc != T2FW_OK) return rc;
  bool done = false;
  if (D % V == 0 && rms::aligned(16, {dy, dsum, s, w, ds})) {
    rc = rms::launch_bwd_v<T, V>(p, sms, &parts, st);
    done = true;
  }
  if constexpr (sizeof(T) <= 4)
    if (!done && D % 2 == 0 && rms::aligned(2 * (int)sizeof(T), {dy, dsum, s, w, ds})) {
      rc = rms::launch_bwd_v<T, 2>(p, sms, &parts, st);
      done = true;
    }
  if (!done) rc = rms::launch_bwd_v<T, 1>(p, sms, &parts, st);
  if (rc != T2FW_OK) return rc;
  T2FW_CHECK_CUDA(launch_dependent(rms::rms_dw_kernel<T>, dim3((unsigned)ceil_div64(D, 32)), dim3(1024), 0, st,
                                   static_cast<const A *>(scratch), static_cast<T *>(dw), (int)parts, D));
  T2FW_CHECK_LAUNCH(1);
  return T2FW_OK;
}

#define T2FW_RMS_FORWARD(T, k8)                                                                                           \
  template int rms_forward_t<T, k8>(const void *, const void *, const void *, void *, void *, float *, void *, int64_t,  \
                                    int64_t, double, cudaStream_t)
#define T2FW_RMS_BACKWARD(T)                                                                                              \
  template int rms_backward_t<T>(const void *, const void *, const void *, const void *, void *, void *, int64_t, int64_t, \
                                 double, void *, cudaStream_t)

}  // namespace t2fw
