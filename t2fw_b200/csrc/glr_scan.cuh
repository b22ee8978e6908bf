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
// A step acts on what is carried as c -> P c + S, and so does a run of steps; the maps compose.  Forward c = h, P = f, S = x;
// backward, from the last step to the first, c = f_{t+1} r_{t+1}, P = f, S = f go, r = go + c.  All of it in fp32 (fp64 for fp64
// storage), rounded where it is written.
#pragma once

#include "glr.cuh"

namespace t2fw {

namespace {

using namespace glr;

constexpr int kMaxCluster = 8;

template <typename T>
struct ScanArgs {
  const T *x, *f, *go, *gs, *out_in, *state;      // x: value, or value | gate; out_in: the forward call's outputs
  T *out, *df, *end;                              // outputs or d_value (d_vg); d_forget; next_state or d_state
  int64_t T_, D;
  int tiles, cluster, iterations;                 // channel tiles of a row; blocks that share a tile's time axis
  int *status;
};

// One pass over the data.  A tile is one row b and LW * V channels; a thread holds V of them over L consecutive steps, LW threads
// beside one another read a line of memory, and a block's part of the time axis is kRuns * L steps.  The parts of a round lie on
// the blocks of a cluster.  Per round
//   A  every thread composes its steps into one map c -> P c + S, and these are composed over the runs of a warp (shuffles)
//   B  the maps are composed over the warps of a block (shared memory) and sent to the other blocks of the cluster
//   C  with the maps of all blocks, what is carried into each warp's steps is known
//   D  every thread walks its steps again and writes its results; who walks the last one writes the final state, so that it is
//      the last output, rounded from the same number
// B and C are the work of one more warp.  The others come to D of a round only after A of the next one, so that warp has the
// time of a round, and they meet it at named barriers: they report their maps and go on, and find what is carried in when they
// need it.  Maps and carried values alternate between two halves.
// Each thread copies what it alone will read, `kStages` rounds ahead, so the copies need no barrier.
//
// Measured, bf16: 64 x 1024 x 1024 forward 70 us (5.8 TB/s of the bytes that have to move, 88 % of the copy bandwidth), backward
// 124 (83 %), fused 99 and 156 (62 and 79 %); 1 x 65536 x 1024 108, 150, 146 and 202 us (57, 69, 42 and 61 %).  With many tiles
// the instructions bound it: 20 per element where 16 bits are unpacked twice (kept in registers they would halve the warps that
// fit), half of the issue slots at 15 to 20 warps per SM; fused, two special functions per gate and pass.  With one long row
// there are 256 blocks, and a round of a block takes 1.6 us, most of it the latency of A and D at two warps per scheduler.
// Not better there: clusters of 16 (128 us), quarter lines (131), eight steps to a thread in the backward pass (256: one block per
// SM), D two rounds behind A (110).
template <typename T, int V, int LW, bool kFused, bool kBwd, int L, int kStages, int kThreads, int kMin>
__global__ void __launch_bounds__(kThreads + 32, kMin)
glr_scan_kernel(const ScanArgs<T> p) {
  using A = typename Elem<T>::acc;
  using R = typename Raw<T, V>::type;
  using A2 = typename Pair<A>::type;
  constexpr int kBytes = V * (int)sizeof(T), kWarps = kThreads / 32;
  constexpr bool kAsync = kBytes >= 4, kFast = sizeof(T) == 2;
  constexpr int kRuns = kThreads / LW, kPart = kRuns * L, CH = LW * V;
  constexpr int NT = kBwd ? (kFused ? 4 : 3) : 2;      // arrays read: fwd x, f; bwd go, f, h, (v)
  constexpr uint32_t kLine = kThreads * kBytes, kSlot = NT * L * kLine;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ __align__(16) A2 s_map[2][kWarps][CH];    // (P, S) of a warp's steps
  __shared__ __align__(16) A s_in[2][kWarps][CH];      // what is carried into a warp's steps
  __shared__ __align__(8) uint64_t bar[2];
  constexpr int K = (CH + 31) / 32, kMaps = 1, kIns = 3;      // channels per thread of the last warp; numbers of named barriers
  A2 *const s_peer = reinterpret_cast<A2 *>(ring + kStages * kSlot);      // [2][C][CH]: maps from the cluster's blocks
  dependency_wait();

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int col = tid % LW, run = tid / LW;
  const int C = p.cluster, N = p.iterations, rank = C > 1 ? (int)(blockIdx.x % (unsigned)C) : 0;
  const unsigned tile = blockIdx.x / (unsigned)C;
  const int64_t b = tile / (unsigned)p.tiles, d0 = (int64_t)(tile % (unsigned)p.tiles) * CH;
  const int64_t d = d0 + col * V, D = p.D, steps = p.T_, row = kFused ? 2 * D : D;
  const bool on = d < D;
  // Steps are counted in walking order: tau = t forward, steps - 1 - t backward.  Addresses of this thread's first step in the
  // round that is fetched next and in the round that is written next; from step to step and from round to round they move by
  // the same distance.
  const int64_t hop = (int64_t)C * kPart, tau_first = (int64_t)rank * kPart + run * L, t_first = kBwd ? steps - 1 - tau_first : tau_first;
  const int64_t one = kBwd ? -1 : 1, wide = one * row, narrow = one * D;      // a step in arrays of width `row` and of width D
  const T *in[NT];
  {
    const int64_t at = (b * steps + t_first) * D + d, at_row = (b * steps + t_first) * row + d;
    if constexpr (!kBwd) {
      in[0] = p.x + at_row;
      in[1] = kFused ? p.x + at_row + D : p.f + at;
    } else {
      in[0] = p.go + at;
      in[1] = kFused ? p.x + at_row + D : p.f + at;
      in[2] = p.out_in + at - D;
      if constexpr (kFused) in[NT - 1] = p.x + at_row;
    }
  }
  T *out0 = p.out + (b * steps + t_first) * (kBwd ? row : D) + d, *out1 = nullptr;
  if constexpr (kBwd) out1 = kFused ? out0 + D : p.df + (b * steps + t_first) * D + d;
  const T *const pst = p.state + b * D + d;
  // of L steps, how many lie before the end (any number of them: no more than 2^30 is told apart)
  auto room = [&](int64_t tau) {
    const int64_t n = steps - tau;
    return !on || n < 0 ? 0 : n > (1 << 30) ? 1 << 30 : (int)n;
  };
  int64_t tau_fetch = tau_first, tau_write = tau_first;
  R held_back[kAsync ? 1 : NT][kAsync ? 1 : L];      // single 16-bit values cannot be copied asynchronously: fetched into registers
  auto fetch = [&](int it) {
    if (it < N) {
      const int left = room(tau_fetch);
      const uint32_t slot = smem_u32(ring) + (uint32_t)(it % kStages) * kSlot + tid * kBytes;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int64_t step = kFused && (!kBwd || j == 1 || j == 3) ? wide : narrow;
        const T *q = in[j];
#pragma unroll
        for (int i = 0; i < L; ++i) {
          const bool ok = i < left;
          const T *from = ok ? q : p.state;
          if (kBwd && j == 2 && i == left - 1 && left < (1 << 30)) from = pst;      // before the first step lies the state
          if constexpr (kAsync) {
            copy_in<kBytes>(slot + (j * L + i) * kLine, from, ok);
          } else {
            held_back[j][i] = R{};
            if (ok) held_back[j][i] = *reinterpret_cast<const R *>(from);
          }
          q += step;
        }
        in[j] += hop * step;
      }
      tau_fetch += hop;
    }
    copy_commit();
  };
  auto raw = [&](int it, int j, int i) -> R & {
    return *reinterpret_cast<R *>(ring + (uint32_t)(it % kStages) * kSlot + (j * L + i) * kLine + tid * kBytes);
  };
  auto put = [&](int it) {      // what `fetch` left in registers
    if constexpr (!kAsync) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < L; ++i) raw(it, j, i) = held_back[j][i];
    }
  };
  // step i of this thread in round `it`: x (or go), the gate and 1 - gate
  auto values = [&](int it, int i, A (&u)[V], A (&f)[V], A (&rest)[V]) {
    unpack<T, V>(raw(it, 0, i), u);
    unpack<T, V>(raw(it, 1, i), f);
    if constexpr (kFused) {
      gates<kFast>(f, rest);
      if constexpr (!kBwd) mul_v(u, u, rest);
    }
  };

  if (C > 1) {      // the other blocks' barriers and shared memory are there to be written to
    if (tid == 0) {
      acp::mbar_init(&bar[0], 1);
      acp::mbar_init(&bar[1], 1);
      acp::mbar_fence_init();
    }
    cluster_sync();
  }
  if (warp == kWarps) {      // B and C
    A carry[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t at = d0 + lane + 32 * k;
      carry[k] = A(0);
      if (lane + 32 * k < CH && at < D) {
        if constexpr (!kBwd) carry[k] = (A)Elem<T>::ld(p.state + b * D + at);
        else if (p.gs != nullptr) carry[k] = (A)Elem<T>::ld(p.gs + b * D + at);
      }
    }
    bool gave_up = false;
    for (int it = 0; it < N; ++it) {
      const int h = it & 1;
      meet<kThreads + 32>(kMaps + h);
      A2 m[K][kWarps];
      A start[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
          if (lane + 32 * k < CH) m[k][w] = s_map[h][w][lane + 32 * k];
      }
      if (C == 1) {
#pragma unroll
        for (int k = 0; k < K; ++k) start[k] = carry[k];
      } else {
        // The maps of a round go into the half of the round before last.  A block sends them after it has the maps of all blocks
        // of the last round, and each block sent those after it had read the half.
        if (lane == 0) acp::mbar_expect_tx(&bar[h], (uint32_t)(C * CH * sizeof(A2)));
        A2 *const half = s_peer + h * C * CH;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          A Pb = A(1), Sb = A(0);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            Sb = apply(m[k][w].x, m[k][w].y, Sb);
            Pb = product(Pb, m[k][w].x);
          }
          if (lane + 32 * k < CH) {
            const uint32_t at = smem_u32(half + rank * CH + lane + 32 * k), sem = smem_u32(&bar[h]);
            for (int r = 0; r < C; ++r) peer_send(peer_address(at, r), A2{Pb, Sb}, peer_address(sem, r));
          }
        }
        if (!gave_up) gave_up = !peer_wait(&bar[h], (it >> 1) & 1);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          start[k] = carry[k];
          A2 q[kMaxCluster];
#pragma unroll
          for (int r = 0; r < kMaxCluster; ++r)
            if (r < C && lane + 32 * k < CH) q[r] = half[r * CH + lane + 32 * k];
#pragma unroll
          for (int r = 0; r < kMaxCluster; ++r)
            if (r < C) {
              if (r == rank) start[k] = carry[k];
              carry[k] = apply(q[r].x, q[r].y, carry[k]);
            }
        }
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (lane + 32 * k < CH) s_in[h][w][lane + 32 * k] = start[k];
          start[k] = apply(m[k][w].x, m[k][w].y, start[k]);
        }
        if (C == 1) carry[k] = start[k];
      }
      report<kThreads + 32>(kIns + h);
    }
    if (gave_up) atomicExch(p.status, 1);
    if (C > 1) cluster_sync();      // no block leaves while another may still send to it
    return;
  }

  if constexpr (kAsync) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) fetch(s);
  } else {
    fetch(0);
    put(0);
    fetch(1);
  }
  A P[V], S[V], P0[V], S0[V];
  bool calm = true, calm0 = true;
  auto enter = [&](int e, A (&c)[V]) {      // what is carried into this thread's steps
#pragma unroll
    for (int k = 0; k < V; ++k) c[k] = s_in[e & 1][warp][col * V + k];
    if constexpr (LW < 32) {      // what the run before leaves is what enters this one
      A behind[V];
      if (calm0) {
        fma_v(behind, P0, c, S0);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) behind[k] = apply(P0[k], S0[k], c[k]);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const A q = __shfl_up_sync(0xffffffffu, behind[k], LW);
        if (lane >= LW) c[k] = q;
      }
    }
  };
  for (int it = 0;; ++it) {
    if (it < N) {      // A
      if constexpr (kAsync) {
        if (it == 0) copy_wait<kStages - 1>();
        else copy_wait<kStages - 2>();
      }
      const bool ragged = ((int64_t)it * C + rank + 1) * kPart > steps;
      const int64_t tau0 = ((int64_t)it * C + rank) * kPart + run * L;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        A u[V], f[V], rest[V];
        values(it, i, u, f, rest);
        if (ragged && tau0 + i >= steps) {      // behind the end a step changes nothing
#pragma unroll
          for (int k = 0; k < V; ++k) f[k] = A(1), u[k] = A(0);
        }
        if (i == 0) {
          // before the first step the state is zero: f * 0 keeps an infinite or NaN gate in sight
          A zero[V];
#pragma unroll
          for (int k = 0; k < V; ++k) P[k] = f[k], zero[k] = A(0);
          if constexpr (kBwd) mul_v(S, f, u);
          else fma_v(S, f, zero, u);
        } else {
          mul_v(P, P, f);
          if constexpr (kBwd) {
#pragma unroll
            for (int k = 0; k < V; ++k) S[k] += u[k];
            mul_v(S, S, f);
          } else {
            fma_v(S, f, S, u);
          }
        }
      }
      if constexpr (LW < 32) {
        calm = __all_sync(0xffffffffu, tame(P));      // gates of up to 1, as nearly always: nothing to look out for
#pragma unroll
        for (int o = LW; o < 32; o <<= 1) {
          A Pp[V], Sp[V];
#pragma unroll
          for (int k = 0; k < V; ++k) {
            Pp[k] = __shfl_up_sync(0xffffffffu, P[k], o);
            Sp[k] = __shfl_up_sync(0xffffffffu, S[k], o);
          }
          if (lane >= o) {
            if (calm) {
              fma_v(S, P, Sp, S);
              mul_v(P, P, Pp);
            } else {
#pragma unroll
              for (int k = 0; k < V; ++k) {
                S[k] = apply(P[k], S[k], Sp[k]);
                P[k] = product(Pp[k], P[k]);
              }
            }
          }
        }
      }
      if (lane >= 32 - LW) {
#pragma unroll
        for (int k = 0; k < V; ++k) s_map[it & 1][warp][col * V + k] = A2{P[k], S[k]};
      }
      report<kThreads + 32>(kMaps + (it & 1));
    }
    if (it > 0) {      // D, of the round before
      const int e = it - 1;
      meet<kThreads + 32>(kIns + (e & 1));
      const int left = room(tau_write);
      T *w0 = out0, *w1 = out1;
      A c[V];
      enter(e, c);
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const bool write = i < left;
        A u[V], f[V], rest[V];
        values(e, i, u, f, rest);
        if constexpr (!kBwd) {
          fma_v(c, f, c, u);
          if (write) *reinterpret_cast<R *>(w0) = pack<T, V>(c);
          w0 += D;
        } else {
          A before[V];
          unpack<T, V>(raw(e, 2, i), before);
#pragma unroll
          for (int k = 0; k < V; ++k) u[k] = add_rn(u[k], c[k]);      // r
          mul_v(c, f, u);
          if constexpr (kFused) {
            A v[V];
            unpack<T, V>(raw(e, NT - 1, i), v);
            mul_v(u, u, rest);      // d_v
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = f[k] * u[k] * (before[k] - v[k]);      // d_g
            if (write) {
              *reinterpret_cast<R *>(w0) = pack<T, V>(u);
              *reinterpret_cast<R *>(w1) = pack<T, V>(v);
            }
          } else {
            mul_v(before, before, u);
            if (write) {
              *reinterpret_cast<R *>(w0) = pack<T, V>(u);
              *reinterpret_cast<R *>(w1) = pack<T, V>(before);
            }
          }
          w0 += wide;
          w1 += wide;
        }
      }
      tau_write += hop;
      out0 += hop * (kBwd ? wide : D);
      if constexpr (kBwd) out1 += hop * wide;
      if constexpr (kAsync) fetch(e + kStages);
    }
    if (it == N) break;
    if constexpr (!kAsync) {
      put(it + 1);
      fetch(it + 2);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) P0[k] = P[k], S0[k] = S[k];
    calm0 = calm;
  }
  copy_wait<0>();
  // The final state is left by who walked the last step, in the last round.  These steps are walked once more, out here: a store in
  // the loop above cost the fused backward pass 8 to 10 %.
  const int left = room(tau_write - hop);
  if (__any_sync(0xffffffffu, left > 0 && left <= L)) {
    A c[V];
    enter(N - 1, c);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      A u[V], f[V], rest[V];
      values(N - 1, i, u, f, rest);
      if constexpr (!kBwd) {
        fma_v(c, f, c, u);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) u[k] = add_rn(u[k], c[k]);
        mul_v(c, f, u);
      }
      if (i == left - 1) *reinterpret_cast<R *>(p.end + b * D + d) = pack<T, V>(c);
    }
  }
  if (C > 1) cluster_sync();
}

// Every thread walks V channels of a row from the first step to the last, U steps' loads at a time, the next U on their way:
// for sequences too short to be cut, and for so many channels that the walkers alone keep the memory busy.  Bound by memory:
// 512 x 128 x 1024 bf16 70 us forward and 113 backward (88 and 91 % of the copy bandwidth).
template <typename T, int V, bool kFused, bool kBwd>
__global__ void __launch_bounds__(128)
glr_walk_kernel(const ScanArgs<T> p, int64_t n) {
  using A = typename Elem<T>::acc;
  using R = typename Raw<T, V>::type;
  constexpr bool kFast = sizeof(T) == 2;
  constexpr int U = sizeof(R) < 16 ? 8 : !kBwd ? 6 : kFused ? 3 : 4, NT = kBwd ? (kFused ? 4 : 3) : 2;
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
        if constexpr (kFused) gates<kFast>(f, rest);
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

template <typename T, int V, int LW, bool kFused, bool kBwd, int L, int kStages, int kThreads, int kMin>
int launch_scan_v(ScanArgs<T> p, int64_t B, int sms, cudaStream_t st) {
  constexpr int kPart = kThreads / LW * L, CH = LW * V;
  constexpr int NT = kBwd ? (kFused ? 4 : 3) : 2;
  constexpr size_t ring = (size_t)kStages * NT * L * kThreads * V * sizeof(T), map = CH * 2 * sizeof(typename Elem<T>::acc);
  const auto kernel = &glr_scan_kernel<T, V, LW, kFused, kBwd, L, kStages, kThreads, kMin>;
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  T2FW_CHECK_CUDA(cudaGetDevice(&dev));
  if (!(ready.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    T2FW_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         220 * 1024 - (int)(2 * (kThreads / 32) * (map + map / 2))));
    ready.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
  }
  const int64_t tiles = ceil_div64(p.D, CH), all = B * tiles, parts = ceil_div64(p.T_, kPart);
  // Blocks per tile: enough for every SM to have one (backward), or one and a half (forward).  Forward with clusters of 2 / 4 / 8,
  // us: 8 x 1024 x 768 15.0 / 12.3 / 15.7, 3 x 777 x 1016 10.7 / 9.4 / 8.4; backward 18.9 / 21.5 / 23.2 and 12.5 / 11.4 / 14.3.
  int C = 1;
  while (C < kMaxCluster && C < parts && all * C < (kBwd ? sms : sms + sms / 2)) C *= 2;
  T2FW_CHECK_ARG(tiles <= 0x7fffffff && all <= 0x7fffffff / C && parts <= 0x7fffffff, "sizes out of range");
  p.tiles = (int)tiles;
  p.cluster = C;
  p.iterations = (int)ceil_div64(parts, C);
  const int rc = lfw_chunk_status_ptr(&p.status);
  if (rc != T2FW_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(all * C));
  cfg.blockDim = dim3(kThreads + 32);
  // Blocks of a cluster are placed side by side, as many to an SM as fit, while other SMs stay empty: ask for so much shared
  // memory that no more fit than the launch has per SM (1 x 65536 x 1024 forward 146 -> 107 us), or two: with one, clusters of
  // eight did not all find room at once (268 us where two fit 186).
  constexpr size_t fixed = 2 * (kThreads / 32) * (map + map / 2) + 1024 + 16, per_sm = 228 * 1024;
  const size_t k = all * C > 2 * sms ? (size_t)ceil_div64(all * C, sms) : 2, spread = per_sm / (k + 1) + 1;
  cfg.dynamicSmemBytes = ring + (C > 1 ? 2 * C * map : 0);
  if (C > 1 && cfg.dynamicSmemBytes + fixed < spread) cfg.dynamicSmemBytes = (spread - fixed + 15) / 16 * 16;
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

template <typename T, int V, bool kFused, bool kBwd>
int launch_v(const ScanArgs<T> &p, int64_t B, cudaStream_t st) {
  int sms = 0;
  const int rc = lfw_chunk_sm_count(&sms);
  if (rc != T2FW_OK) return rc;
  const int64_t n = B * p.D / V;
  // Walkers need many channels or few steps.  Scan against walk, forward, bf16, us: 256 x 64 steps x 768 (24 576 walkers) 20.7 /
  // 16.7, 128 x 64 x 768 11.4 / 13.6, 512 x 128 x 1024 81.0 / 80.8 (backward 131 / 108), 256 x 16 x 768 17.7 / 5.3,
  // 64 x 40 x 768 6.1 / 9.1, 16 x 24 x 512 2.1 / 3.3.
  const int64_t full = n * V * (int64_t)sizeof(T) / 16;      // walkers of 16 bytes; narrower ones keep less in flight
  if (p.T_ <= 8 || full >= 128 * sms || (full >= 40 * sms && p.T_ <= 32)) {
    T2FW_CHECK_ARG(n <= 128 * (int64_t)0x7fffffff, "sizes out of range");
    T2FW_CHECK_CUDA(launch_dependent(glr_walk_kernel<T, V, kFused, kBwd>, dim3((unsigned)ceil_div64(n, 128)), dim3(128), 0, st,
                                     p, n));
    T2FW_CHECK_LAUNCH(1);
    return T2FW_OK;
  }
  if constexpr (V * sizeof(T) == 16) {
    // Full lines, or half lines where those tiles are so few that a cluster each leaves SMs without work.  Full against half,
    // bf16, us, forward and backward: 1 x 65536 x 1024 (16 tiles) 268 / 107 and 324 / 146, 4 x 4096 x 512 (32) 16.1 / 16.6 and
    // 20.9 / 22.0, 64 x 1024 x 1024 76 / 83 and 122 / 130.
    if (B * ceil_div64(p.D, 8 * V) * kMaxCluster >= sms + sms / 2)
      return launch_scan_v<T, V, 8, kFused, kBwd, 4, 3, 128, kBwd ? 3 : 4>(p, B, sms, st);
    return launch_scan_v<T, V, 4, kFused, kBwd, 4, 3, 128, 3>(p, B, sms, st);
  } else {
    return launch_scan_v<T, V, 32, kFused, kBwd, 8, 3, 256, 2>(p, B, sms, st);
  }
}

// 16 bytes per thread where rows and pointers allow them, else a 32-bit word, else an element.
template <typename T, bool kFused, bool kBwd>
int launch_scan(const ScanArgs<T> &p, int64_t B, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const void *const ptr[] = {p.x, p.f, p.go, p.gs, p.out_in, p.state, p.out, p.df, p.end};
  uintptr_t low = 0;
  for (const void *q : ptr) low |= reinterpret_cast<uintptr_t>(q);
  if (p.D % V == 0 && (low & 15) == 0) return launch_v<T, V, kFused, kBwd>(p, B, st);
  if constexpr (sizeof(T) == 2)
    if (p.D % 2 == 0 && (low & 3) == 0) return launch_v<T, 2, kFused, kBwd>(p, B, st);
  return launch_v<T, 1, kFused, kBwd>(p, B, st);
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
