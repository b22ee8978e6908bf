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
//
// A step acts on what is carried as c -> P c + L, and so does a run of steps; the maps compose.  Forward c = h, P = f, L = x;
// backward, from the last step to the first, c = f_{t+1} r_{t+1}, P = f, L = f go, r = go + c.
#include <type_traits>

#include "glr.cuh"

namespace t2fw {

namespace {

using namespace glr;

constexpr int kThreads = 256, kWarps = kThreads / 32, kMaxCluster = 8;

template <typename T>
struct ScanArgs {
  const T *x, *f, *go, *gs, *out_in, *state;      // x: value, or value | gate; out_in: the forward call's outputs
  T *out, *df, *end;                              // outputs or d_value (d_vg); d_forget; next_state or d_state
  int64_t T_, D;
  int tiles, cluster, iterations;                 // channel tiles of a row; blocks that share a tile's time axis
};

// One pass over the data.  A tile is one row b and LW * V channels; a thread holds V of them (16 bytes) over L consecutive
// steps, LW threads beside one another read a full line, and a block's part of the time axis is kRuns * L steps.  The parts of
// a round lie on the blocks of a cluster.  Per round: the threads compose their steps into one map, these are composed over
// the runs of a warp (shuffles), the warps of a block (shared memory) and the blocks of the cluster (each writes its map into
// the others' shared memory), and with the carry thus known at its start every thread walks its steps again from registers.
// Each thread copies what it alone will read, `kStages` rounds ahead, so the copies need no barrier.
template <typename T, int V, bool kFused, bool kBwd, int L, int kStages>
__global__ void __launch_bounds__(kThreads, 2)
glr_scan_kernel(const ScanArgs<T> p) {
  using A = typename Elem<T>::acc;
  using R = typename Raw<T, V>::type;
  using A2 = typename Pair<A>::type;
  constexpr bool kAsync = V > 1, kFast = sizeof(T) == 2;
  constexpr int LW = kAsync ? 8 : 32, kRuns = kThreads / LW, kPart = kRuns * L, CH = LW * V;
  constexpr int NT = kBwd ? (kFused ? 4 : 3) : 2;      // arrays read: fwd x, f; bwd go, f, h, (v)
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ __align__(16) A2 s_map[kWarps][CH];       // (P, L) of a warp's steps
  __shared__ __align__(16) A s_in[kWarps][CH];         // what is carried into a warp's steps
  __shared__ __align__(16) A2 s_peer[2][kMaxCluster][CH];
  dependency_wait();

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int col = tid % LW, run = tid / LW;
  const int C = p.cluster, rank = C > 1 ? (int)(blockIdx.x % (unsigned)C) : 0;
  const unsigned tile = blockIdx.x / (unsigned)C;
  const int64_t b = tile / (unsigned)p.tiles, d0 = (int64_t)(tile % (unsigned)p.tiles) * CH;
  const int64_t d = d0 + col * V, D = p.D, steps = p.T_, row = kFused ? 2 * D : D;
  const bool on = d < D;
  const T *const px = p.x + b * steps * row + d, *const pf = kFused ? px + D : p.f + b * steps * D + d;
  const T *const pgo = kBwd ? p.go + b * steps * D + d : nullptr, *const pho = kBwd ? p.out_in + b * steps * D + d : nullptr;
  const T *const pst = p.state + b * D + d;

  // Address of array j's values for a step; `tau` counts steps in walking order.
  auto source = [&](int j, int64_t t) -> const T * {
    if constexpr (!kBwd) return j == 0 ? px + t * row : pf + t * row;
    if (j == 0) return pgo + t * D;
    if (j == 1) return pf + t * row;
    if (j == 2) return t > 0 ? pho + (t - 1) * D : pst;
    return px + t * row;
  };
  auto fetch = [&](int it) {
    if constexpr (kAsync) {
      const int64_t tau0 = ((int64_t)it * C + rank) * kPart + run * L;
      const uint32_t slot = smem_u32(ring) + (uint32_t)(it % kStages) * (NT * L * kThreads * 16) + tid * 16;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < L; ++i) {
          const int64_t tau = tau0 + i, t = kBwd ? steps - 1 - tau : tau;
          const bool ok = on && tau < steps && it < p.iterations;
          copy16(slot + (j * L + i) * (kThreads * 16), ok ? source(j, t) : p.state, ok);
        }
      copy_commit();
    }
  };
  auto value = [&](int it, int j, int i, A (&v)[V]) {
    if constexpr (kAsync) {
      unpack<T, V>(*reinterpret_cast<const R *>(ring + (size_t)(it % kStages) * (NT * L * kThreads * 16) +
                                                (j * L + i) * (kThreads * 16) + tid * 16), v);
    } else {
      const int64_t tau = ((int64_t)it * C + rank) * kPart + run * L + i, t = kBwd ? steps - 1 - tau : tau;
      v[0] = on && tau < steps ? (A)Elem<T>::ld(source(j, t)) : A(0);
    }
  };

#pragma unroll
  for (int s = 0; s < kStages; ++s) fetch(s);
  // the thread of a channel keeps what is carried from round to round
  A carry = A(0);
  if (tid < CH && d0 + tid < D) {
    if constexpr (!kBwd) carry = (A)Elem<T>::ld(p.state + b * D + d0 + tid);
    else if (p.gs != nullptr) carry = (A)Elem<T>::ld(p.gs + b * D + d0 + tid);
  }

  if (C > 1) cluster_sync();      // the other blocks' shared memory is there to be written to
  for (int it = 0; it < p.iterations; ++it) {
    if constexpr (kAsync) copy_wait<kStages - 1>();
    const int64_t tau0 = ((int64_t)it * C + rank) * kPart + run * L;
    A u[L][V], f[L][V];      // x (or go) and the gate
    A P[V], S[V];            // the composed map of this thread's steps, then of all runs of the warp up to it
#pragma unroll
    for (int k = 0; k < V; ++k) P[k] = A(1), S[k] = A(0);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      value(it, 0, i, u[i]);
      value(it, 1, i, f[i]);
      const bool in = tau0 + i < steps;      // behind the end a step changes nothing
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if constexpr (kFused) {
          A rest;
          gate_pair<kFast>(f[i][k], f[i][k], rest);
          if constexpr (!kBwd) u[i][k] *= rest;
        }
        if (!in) f[i][k] = A(1), u[i][k] = A(0);
        S[k] = kBwd ? f[i][k] * (u[i][k] + S[k]) : f[i][k] * S[k] + u[i][k];
        P[k] *= f[i][k];
      }
    }
    A Pe[V], Se[V];          // the same without this thread's steps
    if constexpr (LW < 32) {
#pragma unroll
      for (int o = LW; o < 32; o <<= 1)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const A Pp = __shfl_up_sync(0xffffffffu, P[k], o), Sp = __shfl_up_sync(0xffffffffu, S[k], o);
          if (lane >= o) {
            S[k] = apply(P[k], S[k], Sp);
            P[k] = product(Pp, P[k]);
          }
        }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        Pe[k] = __shfl_up_sync(0xffffffffu, P[k], LW);
        Se[k] = __shfl_up_sync(0xffffffffu, S[k], LW);
        if (lane < LW) Pe[k] = A(1), Se[k] = A(0);
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) Pe[k] = A(1), Se[k] = A(0);
    }
    if (lane >= 32 - LW)
#pragma unroll
      for (int k = 0; k < V; ++k) s_map[warp][col * V + k] = A2{P[k], S[k]};
    __syncthreads();
    A2 m[kWarps];
    A start = carry;
    if (tid < CH) {
      A Pb = A(1), Sb = A(0);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        m[w] = s_map[w][tid];
        Sb = apply(m[w].x, m[w].y, Sb);
        Pb = product(Pb, m[w].x);
      }
      if (C == 1) {
        carry = apply(Pb, Sb, carry);
      } else {
        const uint32_t at = smem_u32(&s_peer[it & 1][rank][tid]);
        for (int r = 0; r < C; ++r) peer_store(peer_address(at, r), A2{Pb, Sb});
      }
    }
    // The maps of a round go into the half that the round before last has used: a block arrives here only after it has read
    // that one, so one barrier per round is enough.
    if (C > 1) {
      cluster_sync();
      if (tid < CH)
        for (int r = 0; r < C; ++r) {
          if (r == rank) start = carry;
          const A2 q = s_peer[it & 1][r][tid];
          carry = apply(q.x, q.y, carry);
        }
    }
    if (tid < CH) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        s_in[w][tid] = start;
        start = apply(m[w].x, m[w].y, start);
      }
    }
    __syncthreads();
    A c[V];
#pragma unroll
    for (int k = 0; k < V; ++k) c[k] = apply(Pe[k], Se[k], s_in[warp][col * V + k]);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int64_t tau = tau0 + i, t = kBwd ? steps - 1 - tau : tau;
      const bool write = on && tau < steps;
      if constexpr (!kBwd) {
#pragma unroll
        for (int k = 0; k < V; ++k) c[k] = f[i][k] * c[k] + u[i][k];
        if (write) *reinterpret_cast<R *>(p.out + (b * steps + t) * D + d) = pack<T, V>(c);
      } else {
        A before[V], r[V];
        value(it, 2, i, before);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          r[k] = u[i][k] + c[k];
          c[k] = f[i][k] * r[k];
        }
        if constexpr (kFused) {
          A v[V], g[V];
          value(it, 3, i, v);
          value(it, 1, i, g);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            A a, rest;
            gate_pair<kFast>(g[k], a, rest);
            r[k] *= rest;                                 // d_v
            v[k] = a * r[k] * (before[k] - v[k]);         // d_g
          }
          if (write) {
            T *to = p.out + (b * steps + t) * row + d;
            *reinterpret_cast<R *>(to) = pack<T, V>(r);
            *reinterpret_cast<R *>(to + D) = pack<T, V>(v);
          }
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k) before[k] *= r[k];
          if (write) {
            *reinterpret_cast<R *>(p.out + (b * steps + t) * D + d) = pack<T, V>(r);
            *reinterpret_cast<R *>(p.df + (b * steps + t) * D + d) = pack<T, V>(before);
          }
        }
      }
    }
    fetch(it + kStages);
  }
  if constexpr (kAsync) copy_wait<0>();
  if (rank == 0 && tid < CH && d0 + tid < D) Elem<T>::st(p.end + b * D + d0 + tid, carry);
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

int sm_count(int *n) {
  static std::atomic<int> known[64];
  int dev = 0;
  T2FW_CHECK_CUDA(cudaGetDevice(&dev));
  *n = known[dev & 63].load(std::memory_order_relaxed);
  if (*n == 0) {
    T2FW_CHECK_CUDA(cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, dev));
    known[dev & 63].store(*n, std::memory_order_relaxed);
  }
  return T2FW_OK;
}

template <typename T, int V, bool kFused, bool kBwd, int L, int kStages>
int launch_scan_v(ScanArgs<T> p, int64_t B, cudaStream_t st) {
  constexpr int LW = V > 1 ? 8 : 32, kPart = kThreads / LW * L, CH = LW * V;
  constexpr int NT = kBwd ? (kFused ? 4 : 3) : 2;
  constexpr size_t smem = V > 1 ? (size_t)kStages * NT * L * kThreads * 16 : 0;
  const auto kernel = &glr_scan_kernel<T, V, kFused, kBwd, L, kStages>;
  T2FW_ALLOW_SMEM(kernel, smem);
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc != T2FW_OK) return rc;
  const int64_t tiles = ceil_div64(p.D, CH), all = B * tiles, parts = ceil_div64(p.T_, kPart);
  int C = 1;
  while (C < kMaxCluster && C < parts && all * C < 2 * sms) C *= 2;
  T2FW_CHECK_ARG(tiles <= 0x7fffffff && all <= 0x7fffffff / C && parts <= 0x7fffffff, "sizes out of range");
  p.tiles = (int)tiles;
  p.cluster = C;
  p.iterations = (int)ceil_div64(parts, C);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(all * C));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (C > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = C;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (dependent_launch_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  T2FW_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  T2FW_CHECK_LAUNCH(1);
  return T2FW_OK;
}

// Vectors of 16 bytes where rows and pointers allow them, else single elements.
template <typename T, bool kFused, bool kBwd>
int launch_scan(const ScanArgs<T> &p, int64_t B, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const void *const ptr[] = {p.x, p.f, p.go, p.out_in, p.state, p.out, p.df};
  uintptr_t low = 0;
  for (const void *q : ptr) low |= reinterpret_cast<uintptr_t>(q);
  if (p.D % V == 0 && (low & 15) == 0)
    return launch_scan_v<T, V, kFused, kBwd, kBwd && kFused ? 2 : 4, kBwd ? 2 : 3>(p, B, st);
  return launch_scan_v<T, 1, kFused, kBwd, 8, 1>(p, B, st);
}

template <typename T, bool kFused>
int forward(const void *x, const void *f, const void *state, void *out, void *next, int64_t B, int64_t steps, int64_t D,
            cudaStream_t st) {
  ScanArgs<T> p = {};
  p.x = static_cast<const T *>(x);
  p.f = static_cast<const T *>(f);
  p.state = static_cast<const T *>(state);
  p.out = static_cast<T *>(out);
  p.end = static_cast<T *>(next);
  p.T_ = steps;
  p.D = D;
  return launch_scan<T, kFused, false>(p, B, st);
}

template <typename T, bool kFused>
int backward(const void *go, const void *gs, const void *x, const void *f, const void *out, const void *state, void *dx,
             void *df, void *ds, int64_t B, int64_t steps, int64_t D, cudaStream_t st) {
  ScanArgs<T> p = {};
  p.x = static_cast<const T *>(x);
  p.f = static_cast<const T *>(f);
  p.go = static_cast<const T *>(go);
  p.gs = static_cast<const T *>(gs);
  p.out_in = static_cast<const T *>(out);
  p.state = static_cast<const T *>(state);
  p.out = static_cast<T *>(dx);
  p.df = static_cast<T *>(df);
  p.end = static_cast<T *>(ds);
  p.T_ = steps;
  p.D = D;
  return launch_scan<T, kFused, true>(p, B, st);
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
  T2FW_GLR_TYPES(forward, false, x, f, state, out, next, B, T, D, st)
}
int glr_fused_forward(const void *vg, const void *state, void *out, void *next, int64_t B, int64_t T, int64_t D, int dtype,
                      cudaStream_t st) {
  T2FW_GLR_TYPES(forward, true, vg, nullptr, state, out, next, B, T, D, st)
}
int glr_backward(const void *go, const void *gs, const void *f, const void *out, const void *state, void *dx, void *df,
                 void *ds, int64_t B, int64_t T, int64_t D, int dtype, cudaStream_t st) {
  T2FW_GLR_TYPES(backward, false, go, gs, nullptr, f, out, state, dx, df, ds, B, T, D, st)
}
int glr_fused_backward(const void *go, const void *gs, const void *vg, const void *out, const void *state, void *dvg,
                       void *ds, int64_t B, int64_t T, int64_t D, int dtype, cudaStream_t st) {
  T2FW_GLR_TYPES(backward, true, go, gs, vg, nullptr, out, state, dvg, nullptr, ds, B, T, D, st)
}

}  // namespace t2fw
