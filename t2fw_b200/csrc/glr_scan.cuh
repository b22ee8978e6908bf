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
#pragma once

#include <cstdlib>

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
  int *status;
};

// One pass over the data.  A tile is one row b and LW * V channels; a thread holds V of them (16 bytes) over L consecutive
// steps, LW threads beside one another read a full line, and a block's part of the time axis is kRuns * L steps.  The parts of
// a round lie on the blocks of a cluster.  Per round: the threads compose their steps into one map, these are composed over
// the runs of a warp (shuffles), the warps of a block (shared memory) and the blocks of the cluster (each writes its map into
// the others' shared memory), and with the carry thus known at its start every thread walks its steps again from registers.
// Each thread copies what it alone will read, `kStages` rounds ahead, so the copies need no barrier.
template <typename T, int V, int LW, bool kFused, bool kBwd, int L, int kStages>
__global__ void __launch_bounds__(kThreads, V * sizeof(T) == 16 ? 2 : 3)
glr_scan_kernel(const ScanArgs<T> p) {
  using A = typename Elem<T>::acc;
  using R = typename Raw<T, V>::type;
  using A2 = typename Pair<A>::type;
  constexpr bool kAsync = V * sizeof(T) == 16, kFast = sizeof(T) == 2;
  constexpr int kRuns = kThreads / LW, kPart = kRuns * L, CH = LW * V;
  constexpr int NT = kBwd ? (kFused ? 4 : 3) : 2;      // arrays read: fwd x, f; bwd go, f, h, (v)
  constexpr uint32_t kSlot = NT * L * kThreads * 16;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ __align__(16) A2 s_map[kWarps][CH];       // (P, S) of a warp's steps
  __shared__ __align__(16) A s_in[kWarps][CH];         // what is carried into a warp's steps
  __shared__ __align__(8) uint64_t bar[2];
  A2 *const s_peer = reinterpret_cast<A2 *>(ring + (kAsync ? kStages * kSlot : 0));      // [2][C][CH]: maps from the cluster's blocks
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

  // Address of array j's values for step t.
  auto source = [&](int j, int64_t t) -> const T * {
    if constexpr (!kBwd) return j == 0 ? px + t * row : pf + t * row;
    if (j == 0) return pgo + t * D;
    if (j == 1) return pf + t * row;
    if (j == 2) return t > 0 ? pho + (t - 1) * D : pst;
    return px + t * row;
  };
  auto fetch = [&](int it) {
    if constexpr (kAsync) {
      const int64_t tau0 = ((int64_t)it * C + rank) * kPart + run * L;      // in walking order
      const uint32_t slot = smem_u32(ring) + (uint32_t)(it % kStages) * kSlot + tid * 16;
      if (it < p.iterations) {
#pragma unroll
        for (int i = 0; i < L; ++i) {
          const int64_t tau = tau0 + i, t = kBwd ? steps - 1 - tau : tau;
          const bool ok = on && tau < steps;
#pragma unroll
          for (int j = 0; j < NT; ++j) copy16(slot + (j * L + i) * (kThreads * 16), ok ? source(j, t) : p.state, ok);
        }
      }
      copy_commit();
    }
  };
  auto value = [&](int it, int j, int i, A (&v)[V]) {
    if constexpr (kAsync) {
      unpack<T, V>(*reinterpret_cast<const R *>(ring + (uint32_t)(it % kStages) * kSlot + (j * L + i) * (kThreads * 16) + tid * 16), v);
    } else {
      const int64_t tau = ((int64_t)it * C + rank) * kPart + run * L + i, t = kBwd ? steps - 1 - tau : tau;
      R u = {};
      if (on && tau < steps) u = *reinterpret_cast<const R *>(source(j, t));
      unpack<T, V>(u, v);
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

  bool gave_up = false;
  if (C > 1) {      // the other blocks' barriers and shared memory are there to be written to
    if (tid == 0) {
      acp::mbar_init(&bar[0], 1);
      acp::mbar_init(&bar[1], 1);
      acp::mbar_fence_init();
    }
    cluster_sync();
  }
  for (int it = 0; it < p.iterations; ++it) {
    if constexpr (kAsync) copy_wait<kStages - 1>();
    const int64_t tau0 = ((int64_t)it * C + rank) * kPart + run * L;
    A u[L][V], f[L][V], rest[kFused && kBwd ? L : 1][V];      // x (or go), the gate, 1 - gate
    const bool ragged = ((int64_t)it * C + rank + 1) * kPart > steps;
    A P[V], S[V];      // the composed map of this thread's steps, then of all runs of the warp up to it
#pragma unroll
    for (int i = 0; i < L; ++i) {
      value(it, 0, i, u[i]);
      value(it, 1, i, f[i]);
      if constexpr (kFused) {
#pragma unroll
        for (int k = 0; k < V; ++k) gate_pair<kFast>(f[i][k], f[i][k], rest[kBwd ? i : 0][k]);
        if constexpr (!kBwd) mul_v(u[i], u[i], rest[0]);
      }
      if (ragged && tau0 + i >= steps) {      // behind the end a step changes nothing
#pragma unroll
        for (int k = 0; k < V; ++k) f[i][k] = A(1), u[i][k] = A(0);
      }
      if (i == 0) {
#pragma unroll
        for (int k = 0; k < V; ++k) P[k] = f[0][k];
        // the state before the first step is zero: f * 0 keeps an infinite or NaN gate in sight
        A zero[V];
#pragma unroll
        for (int k = 0; k < V; ++k) zero[k] = A(0);
        if constexpr (kBwd) mul_v(S, f[0], u[0]);
        else fma_v(S, f[0], zero, u[0]);
      } else {
        mul_v(P, P, f[i]);
        if constexpr (kBwd) {
#pragma unroll
          for (int k = 0; k < V; ++k) S[k] += u[i][k];
          mul_v(S, S, f[i]);
        } else {
          fma_v(S, f[i], S, u[i]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) P[k] = held(P[k]);
    if constexpr (LW < 32) {
#pragma unroll
      for (int o = LW; o < 32; o <<= 1) {
        A Pp[V], Sp[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          Pp[k] = __shfl_up_sync(0xffffffffu, P[k], o);
          Sp[k] = __shfl_up_sync(0xffffffffu, S[k], o);
        }
        if (lane >= o) {
          fma_v(S, P, Sp, S);
          mul_v(P, P, Pp);
#pragma unroll
          for (int k = 0; k < V; ++k) P[k] = held(P[k]);
        }
      }
    }
    if (lane >= 32 - LW) {
#pragma unroll
      for (int k = 0; k < V; ++k) s_map[warp][col * V + k] = A2{P[k], S[k]};
    }
    __syncthreads();
    A2 m[kWarps];
    A start = carry;
    if (tid < CH) {
      A Pb = A(1), Sb = A(0);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m[w] = s_map[w][tid];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        Sb = m[w].x * Sb + m[w].y;
        Pb = held(Pb * m[w].x);
      }
      if (C == 1) {
        carry = Pb * carry + Sb;
      } else {
        // The maps of a round go into the half of the round before last.  A block sends those of this round only after it has
        // got all of the last round, and each block sent those after it had read the round before.
        if (tid == 0) acp::mbar_expect_tx(&bar[it & 1], (uint32_t)(C * CH * sizeof(A2)));
        A2 *const half = s_peer + (it & 1) * C * CH;
        const uint32_t at = smem_u32(half + rank * CH + tid), sem = smem_u32(&bar[it & 1]);
        for (int r = 0; r < C; ++r) peer_send(peer_address(at, r), A2{Pb, Sb}, peer_address(sem, r));
        if (!gave_up) gave_up = !peer_wait(&bar[it & 1], (it >> 1) & 1);
        A2 q[kMaxCluster];
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
          if (r < C) q[r] = half[r * CH + tid];
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
          if (r < C) {
            if (r == rank) start = carry;
            carry = q[r].x * carry + q[r].y;
          }
      }
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        s_in[w][tid] = start;
        start = m[w].x * start + m[w].y;
      }
    }
    __syncthreads();
    A c[V], behind[V];
#pragma unroll
    for (int k = 0; k < V; ++k) c[k] = s_in[warp][col * V + k];
    if constexpr (LW < 32) {      // what the run before leaves is what enters this one
      fma_v(behind, P, c, S);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const A q = __shfl_up_sync(0xffffffffu, behind[k], LW);
        if (lane >= LW) c[k] = q;
      }
    }
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int64_t tau = tau0 + i, t = kBwd ? steps - 1 - tau : tau;
      const bool write = on && tau < steps;
      if constexpr (!kBwd) {
        fma_v(c, f[i], c, u[i]);
        if (write) *reinterpret_cast<R *>(p.out + (b * steps + t) * D + d) = pack<T, V>(c);
      } else {
        A before[V], r[V];
        value(it, 2, i, before);
#pragma unroll
        for (int k = 0; k < V; ++k) r[k] = u[i][k] + c[k];
        mul_v(c, f[i], r);
        if constexpr (kFused) {
          A v[V];
          value(it, 3, i, v);
          mul_v(r, r, rest[i]);      // d_v
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] = f[i][k] * r[k] * (before[k] - v[k]);      // d_g
          if (write) {
            T *to = p.out + (b * steps + t) * row + d;
            *reinterpret_cast<R *>(to) = pack<T, V>(r);
            *reinterpret_cast<R *>(to + D) = pack<T, V>(v);
          }
        } else {
          mul_v(before, before, r);
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
  if (gave_up) atomicExch(p.status, 1);
  if (C > 1) cluster_sync();      // no block leaves while another may still send to it
  if (rank == 0 && tid < CH && d0 + tid < D) Elem<T>::st(p.end + b * D + d0 + tid, carry);
}

// Every thread walks V channels of a row from the first step to the last, U steps' loads at a time, the next U on their way:
// for sequences too short to be cut, and for so many channels that the walkers alone keep the memory busy.
template <typename T, int V, bool kFused, bool kBwd>
__global__ void __launch_bounds__(128)
glr_walk_kernel(const ScanArgs<T> p, int64_t n) {
  using A = typename Elem<T>::acc;
  using R = typename Raw<T, V>::type;
  constexpr bool kFast = sizeof(T) == 2;
  constexpr int U = sizeof(R) < 16 ? 8 : kBwd ? 2 : 4, NT = kBwd ? (kFused ? 4 : 3) : 2;
  dependency_wait();
  const int64_t i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i0 >= n) return;
  const int64_t at = i0 * V, D = p.D, steps = p.T_, row = kFused ? 2 * D : D, b = at / D, d = at - b * D;
  const T *const px = p.x + b * steps * row + d, *const pf = kFused ? px + D : p.f + b * steps * D + d;
  const T *const pgo = kBwd ? p.go + b * steps * D + d : nullptr, *const pho = kBwd ? p.out_in + b * steps * D + d : nullptr;
  auto raw = [](const T *q) { return *reinterpret_cast<const R *>(q); };
  const R first = raw(p.state + at);
  A c[V];
  if constexpr (!kBwd) {
    unpack<T, V>(first, c);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) c[k] = A(0);
    if (p.gs != nullptr) unpack<T, V>(raw(p.gs + at), c);
  }
  R now[U][NT], then[U][NT];
  auto load = [&](int64_t tau0, R (&to)[U][NT]) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t tau = tau0 + i, t = kBwd ? steps - 1 - tau : tau;
      if (tau < steps) {
        if constexpr (!kBwd) {
          to[i][0] = raw(px + t * row);
          to[i][1] = raw(pf + t * row);
        } else {
          to[i][0] = raw(pgo + t * D);
          to[i][1] = raw(pf + t * row);
          to[i][2] = t > 0 ? raw(pho + (t - 1) * D) : first;
          if constexpr (kFused) to[i][3] = raw(px + t * row);
        }
      }
    }
  };
  load(0, now);
  for (int64_t tau0 = 0; tau0 < steps; tau0 += U) {
    load(tau0 + U, then);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t tau = tau0 + i, t = kBwd ? steps - 1 - tau : tau;
      if (tau < steps) {
        A u[V], f[V], rest[V];
        unpack<T, V>(now[i][0], u);
        unpack<T, V>(now[i][1], f);
        if constexpr (kFused) {
#pragma unroll
          for (int k = 0; k < V; ++k) gate_pair<kFast>(f[k], f[k], rest[k]);
        }
        if constexpr (!kBwd) {
          if constexpr (kFused) mul_v(u, u, rest);
          fma_v(c, f, c, u);
          *reinterpret_cast<R *>(p.out + (b * steps + t) * D + d) = pack<T, V>(c);
        } else {
          A before[V];
          unpack<T, V>(now[i][2], before);
#pragma unroll
          for (int k = 0; k < V; ++k) u[k] += c[k];
          mul_v(c, f, u);
          if constexpr (kFused) {
            A v[V];
            unpack<T, V>(now[i][NT - 1], v);
            mul_v(u, u, rest);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = f[k] * u[k] * (before[k] - v[k]);
            T *to = p.out + (b * steps + t) * row + d;
            *reinterpret_cast<R *>(to) = pack<T, V>(u);
            *reinterpret_cast<R *>(to + D) = pack<T, V>(v);
          } else {
            mul_v(before, before, u);
            *reinterpret_cast<R *>(p.out + (b * steps + t) * D + d) = pack<T, V>(u);
            *reinterpret_cast<R *>(p.df + (b * steps + t) * D + d) = pack<T, V>(before);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) now[i][j] = then[i][j];
  }
  *reinterpret_cast<R *>(p.end + at) = pack<T, V>(c);
}

template <typename T, int V, int LW, bool kFused, bool kBwd, int L, int kStages>
int launch_scan_v(ScanArgs<T> p, int64_t B, int sms, cudaStream_t st, int forced = 0, int pad = 0) {
  constexpr bool kAsync = V * sizeof(T) == 16;
  constexpr int kPart = kThreads / LW * L, CH = LW * V;
  constexpr int NT = kBwd ? (kFused ? 4 : 3) : 2;
  constexpr size_t ring = kAsync ? (size_t)kStages * NT * L * kThreads * 16 : 0, map = CH * 2 * sizeof(typename Elem<T>::acc);
  const auto kernel = &glr_scan_kernel<T, V, LW, kFused, kBwd, L, kStages>;
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  T2FW_CHECK_CUDA(cudaGetDevice(&dev));
  if (!(ready.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    T2FW_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         pad ? 200000 : (int)(ring + 2 * kMaxCluster * map)));
    ready.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
  }
  const int64_t tiles = ceil_div64(p.D, CH), all = B * tiles, parts = ceil_div64(p.T_, kPart);
  int C = 1;
  while (C < kMaxCluster && C < parts && all * C < 2 * sms) C *= 2;
  if (forced) C = forced < parts ? forced : (int)parts;
  T2FW_CHECK_ARG(tiles <= 0x7fffffff && all <= 0x7fffffff / C && parts <= 0x7fffffff, "sizes out of range");
  p.tiles = (int)tiles;
  p.cluster = C;
  p.iterations = (int)ceil_div64(parts, C);
  const int rc = lfw_chunk_status_ptr(&p.status);
  if (rc != T2FW_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(all * C));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = ring + (C > 1 ? 2 * C * map : 0);
  if (pad) cfg.dynamicSmemBytes = 120000 > cfg.dynamicSmemBytes ? 120000 : cfg.dynamicSmemBytes;
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

template <typename T, int V, int LW, bool kFused, bool kBwd, int L, int kStages>
int launch_v(const ScanArgs<T> &p, int64_t B, cudaStream_t st) {
  int sms = 0;
  const int rc = lfw_chunk_sm_count(&sms);
  if (rc != T2FW_OK) return rc;
  const int64_t n = B * p.D / V;
  static const int walk = std::getenv("GLR_WALK") ? std::atoi(std::getenv("GLR_WALK")) : -1;
  if (walk >= 0 ? walk : p.T_ <= 32 || n >= 128 * sms) {
    T2FW_CHECK_CUDA(launch_dependent(glr_walk_kernel<T, V, kFused, kBwd>, dim3((unsigned)ceil_div64(n, 128)), dim3(128), 0, st,
                                     p, n));
    T2FW_CHECK_LAUNCH(1);
    return T2FW_OK;
  }
  return launch_scan_v<T, V, LW, kFused, kBwd, L, kStages>(p, B, sms, st);
}

// 16 bytes per thread where rows and pointers allow them, else a 32-bit word, else an element.
template <typename T, bool kFused, bool kBwd>
int launch_scan(const ScanArgs<T> &p, int64_t B, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const void *const ptr[] = {p.x, p.f, p.go, p.gs, p.out_in, p.state, p.out, p.df, p.end};
  uintptr_t low = 0;
  for (const void *q : ptr) low |= reinterpret_cast<uintptr_t>(q);
  if (p.D % V == 0 && (low & 15) == 0)
    return launch_v<T, V, 8, kFused, kBwd, kBwd && kFused ? 2 : 4, kBwd ? 2 : 3>(p, B, st);
  if constexpr (sizeof(T) == 2)
    if (p.D % 2 == 0 && (low & 3) == 0) return launch_v<T, 2, 32, kFused, kBwd, 8, 1>(p, B, st);
  return launch_v<T, 1, 32, kFused, kBwd, 8, 1>(p, B, st);
}

}  // namespace

template <typename T, bool kFused>
int glr_forward_t(const void *x, const void *f, const void *state, void *out, void *next, int64_t B, int64_t steps, int64_t D,
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
int glr_backward_t(const void *go, const void *gs, const void *x, const void *f, const void *out, const void *state, void *dx,
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

#define T2FW_GLR_INSTANTIATE(T)                                                                                            \
  template int glr_forward_t<T, false>(const void *, const void *, const void *, void *, void *, int64_t, int64_t,        \
                                       int64_t, cudaStream_t);                                                            \
  template int glr_forward_t<T, true>(const void *, const void *, const void *, void *, void *, int64_t, int64_t,         \
                                      int64_t, cudaStream_t);                                                             \
  template int glr_backward_t<T, false>(const void *, const void *, const void *, const void *, const void *,             \
                                        const void *, void *, void *, void *, int64_t, int64_t, int64_t, cudaStream_t);   \
  template int glr_backward_t<T, true>(const void *, const void *, const void *, const void *, const void *,              \
                                       const void *, void *, void *, void *, int64_t, int64_t, int64_t, cudaStream_t)

}  // namespace t2fw
