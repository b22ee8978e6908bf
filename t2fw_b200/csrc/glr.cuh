// Pieces of the gated linear recurrence's kernels: vectors of a thread's channels, the gate, composition of maps.
#pragma once

#include <type_traits>

#include "async_copy.cuh"
#include "common.cuh"
#include "steps.cuh"

namespace t2fw {
namespace glr {

// V neighbouring channels as they lie in memory: 16 bytes, two 16-bit elements, or one element.
template <typename T, int V>
struct Raw {
  using type = typename std::conditional<V * sizeof(T) == 16, uint4, typename std::conditional<V * sizeof(T) == 8, uint2, uint32_t>::type>::type;
};
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

// e = exp(-g), a = sigmoid(g) = 1 / (1 + e) and rest = 1 - a = e a, each to full relative precision.  g is held at -80 (-700):
// below that a is less than 2e-35, and e would overflow.  For 16-bit storage e = 2^(-g log2 e) and the reciprocal are the fast
// ones: some units of 2^-23, where the result is rounded to 2^-9 or 2^-12.  A NaN stays.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <bool kFast, int V>
__device__ __forceinline__ void gates(float (&g)[V], float (&rest)[V]) {      // g becomes a
  if constexpr (kFast) {
    float e[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float x = max_nan(g[k], -80.f) * -1.44269504f;      // log2 e: off by less than one unit of 2^-24 of it
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e[k]) : "f"(x));
    }
#pragma unroll
    for (int k = 0; k < V; ++k) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(g[k]) : "f"(1.f + e[k]));
#pragma unroll
    for (int k = 0; k < V; ++k) rest[k] = e[k] * g[k];
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float e = expf(-max_nan(g[k], -80.f));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(g[k]) : "f"(1.f + e));      // off by one unit of 2^-23 at most
      rest[k] = e * g[k];
    }
  }
}
template <bool kFast, int V>
__device__ __forceinline__ void gates(double (&g)[V], double (&rest)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const double e = exp(-(g[k] < -700.0 ? -700.0 : g[k]));
    g[k] = 1.0 / (1.0 + e);
    rest[k] = e * g[k];
  }
}

// A run of steps acts on the state as c -> P c + S.  Products of gates may leave the range upwards; then a state of exactly zero
// stays what S makes of it, and a product that is exactly zero stays zero, as in the steps one by one; any other state becomes
// infinite or NaN.  (Where the steps themselves meet an infinity or a NaN, S is none either.)
template <typename A>
__device__ __forceinline__ A apply(A P, A S, A c) { return c == A(0) ? S : P * c + S; }
template <typename A>
__device__ __forceinline__ A product(A first, A then) { return first == A(0) ? A(0) : first * then; }

// A sum that is rounded by itself, never merged with the product before it: two walks over the same steps agree.
__device__ __forceinline__ float add_rn(float a, float b) { return __fadd_rn(a, b); }
__device__ __forceinline__ double add_rn(double a, double b) { return __dadd_rn(a, b); }

// V products, V sums of products with one rounding each: pairs of fp32 in one instruction.
template <typename A, int V>
__device__ __forceinline__ void mul_v(A (&r)[V], const A (&a)[V], const A (&b)[V]) {
  if constexpr (std::is_same<A, float>::value && V % 2 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 2)
      steps::unpack2(steps::mul2(steps::pack2(a[k], a[k + 1]), steps::pack2(b[k], b[k + 1])), r[k], r[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) r[k] = a[k] * b[k];
  }
}
// Whether all |v| are at most 1: products of such cannot leave the range upwards.  (A NaN is not at most 1.)
template <int V>
__device__ __forceinline__ bool tame(const float (&v)[V]) {
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < V; ++k) m = max_nan(m, fabsf(v[k]));
  return m <= 1.f;
}
template <int V>
__device__ __forceinline__ bool tame(const double (&v)[V]) {
  bool ok = true;
#pragma unroll
  for (int k = 0; k < V; ++k) ok = ok && fabs(v[k]) <= 1.0;
  return ok;
}
template <typename A, int V>
__device__ __forceinline__ void fma_v(A (&r)[V], const A (&a)[V], const A (&b)[V], const A (&c)[V]) {
  if constexpr (std::is_same<A, float>::value && V % 2 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 2)
      steps::unpack2(steps::fma2(steps::pack2(a[k], a[k + 1]), steps::pack2(b[k], b[k + 1]), steps::pack2(c[k], c[k + 1])),
                     r[k], r[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) r[k] = fma(a[k], b[k], c[k]);
  }
}

// ---- asynchronous copies into shared memory, and a cluster's shared memory --------------------
using acp::smem_u32;
template <int kBytes>      // 16, 8 or 4; zeros where not ok
__device__ __forceinline__ void copy_in(uint32_t dst, const void *src, bool ok) {
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kBytes), "r"(ok ? kBytes : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t peer_address(uint32_t own, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(own), "r"(rank));
  return r;
}
// Two values into another block's shared memory; their bytes are counted on that block's barrier.
__device__ __forceinline__ void peer_send(uint32_t at, float2 v, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(at), "f"(v.x),
               "f"(v.y), "r"(bar) : "memory");
}
__device__ __forceinline__ void peer_send(uint32_t at, double2 v, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f64 [%0], {%1, %2}, [%3];" ::"r"(at), "d"(v.x),
               "d"(v.y), "r"(bar) : "memory");
}
// Bounded wait for what the blocks of the cluster send; false if it gave up.
__device__ __forceinline__ bool peer_wait(uint64_t *bar, uint32_t parity) {
#pragma unroll 1
  for (uint32_t i = 0; i < acp::kSpinLimit; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, 2000;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}
// Named barriers for n threads: `report` arrives and goes on, `meet` waits for all of them.
template <int n>
__device__ __forceinline__ void report(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(n) : "memory"); }
template <int n>
__device__ __forceinline__ void meet(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(n) : "memory"); }
// Every thread of every block of the cluster; writes before it are seen behind it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

template <typename A> struct Pair;
template <> struct Pair<float> { using type = float2; };
template <> struct Pair<double> { using type = double2; };

}  // namespace glr
}  // namespace t2fw
