// Pieces of the gated linear recurrence's kernels: vectors of a thread's channels, the gate, composition of maps.
#pragma once

#include "common.cuh"

namespace t2fw {
namespace glr {

// V neighbouring channels as they lie in memory: 16 bytes, or one element.
template <typename T, int V> struct Raw { using type = uint4; };
template <typename T> struct Raw<T, 1> { using type = T; };

template <typename T, int V, typename A>
__device__ __forceinline__ void unpack(const typename Raw<T, V>::type &u, A (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = (A)Elem<T>::ld(&u);
  } else if constexpr (sizeof(T) == 2) {
    using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const P *p = reinterpret_cast<const P *>(&u);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      float2 w;
      if constexpr (std::is_same<T, __half>::value) w = __half22float2(p[i]);
      else w = __bfloat1622float2(p[i]);
      v[2 * i] = w.x;
      v[2 * i + 1] = w.y;
    }
  } else {
    const T *p = reinterpret_cast<const T *>(&u);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (A)p[i];
  }
}

template <typename T, int V, typename A>
__device__ __forceinline__ typename Raw<T, V>::type pack(const A (&v)[V]) {
  typename Raw<T, V>::type u;
  if constexpr (V == 1) {
    Elem<T>::st(&u, v[0]);
  } else if constexpr (sizeof(T) == 2) {
    using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    P *p = reinterpret_cast<P *>(&u);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same<T, __half>::value) p[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      else p[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    }
  } else {
    T *p = reinterpret_cast<T *>(&u);
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = (T)v[i];
  }
  return u;
}

// a = sigmoid(g) and rest = 1 - a, both to full relative precision: from exp(-|g|), which does not overflow.  For 16-bit
// storage the exponential and the quotient are the fast ones: a few units of 2^-23, where the result is rounded to 2^-9 or
// 2^-12.  A NaN stays.
template <bool kFast>
__device__ __forceinline__ void gate_pair(float g, float &a, float &rest) {
  const float e = kFast ? __expf(-fabsf(g)) : expf(-fabsf(g));
  const float hi = kFast ? __fdividef(1.f, 1.f + e) : 1.f / (1.f + e), lo = e * hi;
  a = g >= 0.f ? hi : lo;
  rest = g >= 0.f ? lo : hi;
}
template <bool kFast>
__device__ __forceinline__ void gate_pair(double g, double &a, double &rest) {
  const double e = exp(-fabs(g)), hi = 1.0 / (1.0 + e), lo = e * hi;
  a = g >= 0.0 ? hi : lo;
  rest = g >= 0.0 ? lo : hi;
}

// A run of steps acts on the state as h -> P h + L.  A product P that left the range upwards is harmless where the state it
// meets is exactly zero, and a product that is exactly zero stays so: both are what the steps one by one would give.  (Where a
// step's own gate is infinite or NaN, L is no finite number either.)
template <typename A>
__device__ __forceinline__ A apply(A P, A L, A h) { return h == A(0) ? L : P * h + L; }
template <typename A>
__device__ __forceinline__ A product(A first, A then) { return first == A(0) ? A(0) : first * then; }

// ---- asynchronous 16-byte copies into shared memory, and a cluster's shared memory --------------------
__device__ __forceinline__ uint32_t smem_u32(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t peer_address(uint32_t own, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(own), "r"(rank));
  return r;
}
__device__ __forceinline__ void peer_store(uint32_t at, float2 v) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(v.x), "f"(v.y) : "memory");
}
__device__ __forceinline__ void peer_store(uint32_t at, double2 v) {
  asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(at), "d"(v.x), "d"(v.y) : "memory");
}
// Every thread of every block of the cluster; writes before it are seen behind it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

template <typename A> struct Pair;
template <> struct Pair<float> { using type = float2; };
template <> struct Pair<double> { using type = double2; };

}  // namespace glr
}  // namespace t2fw
