// Short causal convolution over time (fdql_causal_conv*), channel by channel, with its SiLU:
//   pre_t = bias + sum_{j<K} w[K-1-j] x_{t-j},   y_t = SiLU(pre_t)
//
// Every value is used K times by the same channel, so a thread owns V neighbouring channels (16 bytes of x where the tensors'
// alignment allows it, else one) of one row and walks a chunk of steps with the last K inputs in registers: x is read once but for the
// K - 1 steps in front of a chunk, y written once, and memory bounds it.  A reset clears the window, which also decides the
// taps in the backward pass.  The steps are read eight (backward: four) ahead of the arithmetic.  Measured, forward: float 50 x 1024 x 1024 94 us =
// 4.5 TB/s, bf16 40 us = 5.2 TB/s; float 50 x 256 x 512 13.1 us; a single step of 32 x 512 4.2 us, of which the launch is most.
//
// Backward: dpre_t = dy_t SiLU'(pre_t), dx_t = sum_j w[K-1-j] dpre_{t+j} over the steps before the next reset, so a chunk runs K - 1
// steps past its end.  The weights' sums stay in registers over all chunks that a thread visits, are joined over the four waves of a
// workgroup in LDS and over workgroups by k_seqconv_finish: no atomics.
#include "seq.h"

#include <algorithm>

namespace fdql {
namespace {

constexpr int WPB = 4;

template <typename T, int V> struct Vec { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T, int V>
__device__ __forceinline__ void widen(const typename Vec<T, V>::type &v, float f[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f(v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void load_v(const T *p, float f[V]) {
  widen<T, V>(*reinterpret_cast<const typename Vec<T, V>::type *>(p), f);
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T *p, const float f[V]) {
  typedef T vec __attribute__((ext_vector_type(V)));
  vec v;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = from_f<T>(f[i]);
  *reinterpret_cast<vec *>(p) = v;
}

struct Args {
  fdql_causal_conv_t p;
  int blocks, chunks, len;         // channel blocks of 64 V, chunks of the time axis and their length
  int64_t units;                   // blocks * R * chunks
  float *slab;                     // [gridDim.x][K + 1][D] backward partials
};

__device__ __forceinline__ bool cut_at(const fdql_causal_conv_t &p, int t, int r) {
  return p.reset && p.reset[(int64_t)t * p.reset_st + (int64_t)r * p.reset_sr] != 0;
}

// Input of step t, t in [-(K-1), T): the carried state in front of step 0.
template <typename T, int V, int K>
__device__ __forceinline__ void input_at(const fdql_causal_conv_t &p, int t, int r, int d, float x[V]) {
  if (t >= 0) {
    load_v<T, V>(reinterpret_cast<const T *>(p.x) + (int64_t)t * p.x_st + (int64_t)r * p.x_sr + d, x);
  } else if (p.state_in) {
    load_v<T, V>(reinterpret_cast<const T *>(p.state_in) + (int64_t)r * p.state_in_sr + (int64_t)(t + K - 1) * p.D + d, x);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = 0.f;
  }
}

// The weights of V channels lie one after the other: whole 16-byte runs where V is 4 or 8.
template <int V, int K>
__device__ __forceinline__ void weights_of(const fdql_causal_conv_t &p, int d, float w[K][V], float b[V]) {
  float run[V * K];
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V * K; i += 4) load_v<float, 4>(p.weight + (int64_t)d * K + i, run + i);
  } else {
#pragma unroll
    for (int i = 0; i < V * K; ++i) run[i] = p.weight[(int64_t)d * K + i];
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][i] = run[i * K + k];
    b[i] = 0.f;
  }
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = p.bias[d + i];
  }
}

// The window moves on: win[K - 1] becomes the newest input; a reset drops the older ones.
template <int V, int K>
__device__ __forceinline__ void push(float win[K][V], const float x[V], bool cut) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int k = 0; k + 1 < K; ++k) win[k][i] = cut ? 0.f : win[k + 1][i];
    win[K - 1][i] = x[i];
  }
}

template <typename T, int V, int K>
__global__ __launch_bounds__(WPB * 64) void k_seqconv_fwd(Args a) {
  const fdql_causal_conv_t &p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned u = blockIdx.x * WPB + wave;
  if (u >= a.units) return;
  const int blk = (int)(u % a.blocks), r = (int)(u / a.blocks % p.R), ch = (int)(u / a.blocks / p.R);
  const int d = (blk * 64 + lane) * V;
  if (d >= p.D) return;
  const int t0 = ch * a.len, t1 = min(p.T, t0 + a.len);
  // U steps at a time, the next ones on their way; the first ones leave before the window's
  constexpr int U = 8;
  typedef typename Vec<T, V>::type vec;
  vec xn[U];
  uint8_t cn[U] = {};
  const T *xp = reinterpret_cast<const T *>(p.x) + (int64_t)r * p.x_sr + d;
  const uint8_t *rp = p.reset ? p.reset + (int64_t)r * p.reset_sr : nullptr;
  const auto fetch = [&](int t) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (t + i < t1) {
        xn[i] = *reinterpret_cast<const vec *>(xp + (int64_t)(t + i) * p.x_st);
        if (rp) cn[i] = rp[(int64_t)(t + i) * p.reset_st];
      }
    }
  };
  fetch(t0);
  float w[K][V], b[V], win[K][V];
  weights_of<V, K>(p, d, w, b);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) {
    float x[V];
    const int t = t0 - (K - 1) + k;
    input_at<T, V, K>(p, t, r, d, x);
    push<V, K>(win, x, t >= 0 && cut_at(p, t, r));
  }
  for (int t = t0; t < t1; t += U) {
    vec x[U];
    bool cut[U];
#pragma unroll
    for (int i = 0; i < U; ++i) x[i] = xn[i], cut[i] = cn[i] != 0;
    if (t + U < t1) fetch(t + U);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (t + i < t1) {
        float f[V], y[V];
        widen<T, V>(x[i], f);
        push<V, K>(win, f, cut[i]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float pre = b[v];
#pragma unroll
          for (int k = 0; k < K; ++k) pre = fmaf(w[k][v], win[k][v], pre);
          y[v] = p.silu ? pre * sigmoid_f<T>(pre).s : pre;
        }
        store_v<T, V>(reinterpret_cast<T *>(p.y) + ((int64_t)(t + i) * p.R + r) * p.D + d, y);
      }
    }
  }
  if (p.state_out && t1 == p.T) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) store_v<T, V>(reinterpret_cast<T *>(p.state_out) + (int64_t)r * p.state_out_sr + (int64_t)k * p.D + d, win[k + 1]);
  }
}

template <typename T, int V, int K>
__global__ __launch_bounds__(WPB * 64) void k_seqconv_bwd(Args a) {
  __shared__ float red[WPB - 1][K + 1][64 * V];
  const fdql_causal_conv_t &p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blk = blockIdx.x % a.blocks, first = blockIdx.x / a.blocks, stride = gridDim.x / a.blocks;
  const int d = (blk * 64 + lane) * V;
  const bool live = d < p.D;
  float w[K][V], b[V], dw[K][V], db[V];
  if (live) weights_of<V, K>(p, d, w, b);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    db[v] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) dw[k][v] = 0.f;
  }
  const int64_t per = (int64_t)p.R * a.chunks;      // (row, chunk) pairs of a channel block, dealt to its workgroups' waves
  for (int64_t u = (int64_t)first * WPB + wave; live && u < per; u += (int64_t)stride * WPB) {
    const int r = (int)(u % p.R), ch = (int)(u / p.R);
    const int t0 = ch * a.len, t1 = min(p.T, t0 + a.len);
    // pend[k]: gradient so far of the input K - 1 - k steps back; age: steps since the last reset, inputs older than that get nothing
    float win[K][V], pend[K][V];
    int age = K;
    // AHEAD steps in front of the arithmetic; the first ones leave before the window's
    constexpr int AHEAD = 4;
    typedef typename Vec<T, V>::type vec;
    vec xn[AHEAD], yn[AHEAD];
    bool cn[AHEAD];
    const auto fetch = [&](int t, int k) {
      cn[k] = false;
      xn[k] = yn[k] = vec{};
      if (t < min(p.T, t1 + K - 1)) {
        xn[k] = *reinterpret_cast<const vec *>(reinterpret_cast<const T *>(p.x) + (int64_t)t * p.x_st + (int64_t)r * p.x_sr + d);
        yn[k] = *reinterpret_cast<const vec *>(reinterpret_cast<const T *>(p.dy) + (int64_t)t * p.dy_st + (int64_t)r * p.dy_sr + d);
        cn[k] = cut_at(p, t, r);
      }
    };
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) fetch(t0 + k, k);
    const int from = ch ? t0 : -(K - 1);             // the first chunk also owns the carried state
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      float x[V];
      const int t = t0 - (K - 1) + k;
      input_at<T, V, K>(p, t, r, d, x);
      const bool cut = t >= 0 && cut_at(p, t, r);
      push<V, K>(win, x, cut);
      age = cut ? 0 : min(age + 1, K);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) pend[k][v] = 0.f;
    for (int tt = t0; tt < t1 + K - 1; tt += AHEAD)
#pragma unroll
    for (int ahead = 0; ahead < AHEAD; ++ahead) {
      const int t = tt + ahead;
      if (t >= t1 + K - 1) break;
      float x[V], dy[V], dp[V];
      const bool cut = cn[ahead];
      widen<T, V>(xn[ahead], x);
      widen<T, V>(yn[ahead], dy);
      fetch(t + AHEAD, ahead);
      age = cut ? 0 : min(age + 1, K);
      push<V, K>(win, x, cut);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float pre = b[v];
#pragma unroll
        for (int k = 0; k < K; ++k) pre = fmaf(w[k][v], win[k][v], pre);
        dp[v] = dy[v];
        if (p.silu) {
          const Sigmoid g = sigmoid_f<T>(pre);
          dp[v] *= g.s * fmaf(pre, g.c, 1.f);
        }
        if (t >= p.T) dp[v] = 0.f;                   // past the end only the pending gradients leave
        if (t < t1) {
          db[v] += dp[v];
#pragma unroll
          for (int k = 0; k < K; ++k) dw[k][v] = fmaf(dp[v], win[k][v], dw[k][v]);
        }
#pragma unroll
        for (int k = 0; k + 1 < K; ++k) pend[k][v] = pend[k + 1][v];
        pend[K - 1][v] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (K - 1 - k <= age) pend[k][v] = fmaf(w[k][v], dp[v], pend[k][v]);
      }
      const int done = t - (K - 1);                  // pend[0] is complete
      if (done >= from && done < t1) {
        float g[V];
#pragma unroll
        for (int v = 0; v < V; ++v) g[v] = pend[0][v];
        const int k = done - (p.T - (K - 1));        // its place in the final state, where it is one of the last inputs
        if (p.dstate_out && k >= 0) {
          bool kept = true;                          // ... and no reset came after it
          for (int q = max(done, -1) + 1; q < p.T; ++q) kept = kept && !cut_at(p, q, r);
          if (kept) {
            float ds[V];
            load_v<T, V>(reinterpret_cast<const T *>(p.dstate_out) + ((int64_t)r * (K - 1) + k) * p.D + d, ds);
#pragma unroll
            for (int v = 0; v < V; ++v) g[v] += ds[v];
          }
        }
        if (done >= 0) {
          if (p.dx) store_v<T, V>(reinterpret_cast<T *>(p.dx) + ((int64_t)done * p.R + r) * p.D + d, g);
        } else if (p.dstate_in) {
          store_v<T, V>(reinterpret_cast<T *>(p.dstate_in) + ((int64_t)r * (K - 1) + done + K - 1) * p.D + d, g);
        }
      }
    }
  }
  if (wave) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      red[wave - 1][K][lane * V + v] = db[v];
#pragma unroll
      for (int k = 0; k < K; ++k) red[wave - 1][k][lane * V + v] = dw[k][v];
    }
  }
  __syncthreads();
  if (wave || !live) return;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float sum = k < K ? dw[k < K ? k : 0][v] : db[v];
#pragma unroll
      for (int q = 0; q < WPB - 1; ++q) sum += red[q][k][lane * V + v];
      a.slab[((int64_t)first * (K + 1) + k) * p.D + d + v] = sum;
    }
  }
}

// Sums of the workgroups' slabs: 64 channels of one tap per workgroup, 16 slices of the slabs.
__global__ __launch_bounds__(1024) void k_seqconv_finish(const float *__restrict__ slab, int nslab, int D, int K, float *dweight, float *dbias) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6, k = blockIdx.y;
  const int d = blockIdx.x * 64 + lane;
  float v = 0.f;
  if (d < D)
#pragma unroll 8
    for (int q = slice; q < nslab; q += 16) v += slab[((int64_t)q * (K + 1) + k) * D + d];
  red[slice][lane] = v;
  __syncthreads();
  if (slice || d >= D) return;
  v = 0.f;
#pragma unroll
  for (int q = 0; q < 16; ++q) v += red[q][lane];
  if (k < K) {
    if (dweight) dweight[(int64_t)d * K + k] = v;
  } else if (dbias) {
    dbias[d] = v;
  }
}

struct Plan {
  int V, blocks, chunks, len, wgs;   // wgs: backward workgroups per channel block
};
// The pointers are looked at only when a call runs: the backward workspace covers either width.
Plan plan_of(const fdql_causal_conv_t &p, int V) {
  Plan q;
  q.V = V;
  q.blocks = (p.D + 64 * V - 1) / (64 * V);
  // Chunks of 64 steps, halved down to 8 while there are fewer than 2048 waves: each reads K - 1 steps of its neighbour again.  bf16 forward, 4099
  // steps of 3 x 1000: 16.7 us against 18.0 at 1024 waves and 16.7 at 4096; 16384 steps of 1 x 1024: 19.5 against 21.8 and 21.3.
  q.len = 64;
  while (q.len > 8 && (int64_t)q.blocks * p.R * ((p.T + q.len - 1) / q.len) < 2048) q.len >>= 1;
  q.chunks = std::max(1, (p.T + q.len - 1) / q.len);
  // backward: three workgroups per CU, so that the weights' partial sums stay few (1024 of them took 2-3% longer at 50 x 1024 x 1024)
  q.wgs = (int)std::min<int64_t>(((int64_t)p.R * q.chunks + WPB - 1) / WPB, std::max(1, 768 / q.blocks));
  return q;
}
int width_of(const fdql_causal_conv_t &p, bool backward) {
  const int esz = p.dtype == FDQL_F32 ? 4 : 2, V = 16 / esz;
  const auto ok = [&](const void *q) { return ((uintptr_t)q & 15) == 0; };
  bool v = p.D % V == 0 && p.x_st % V == 0 && p.x_sr % V == 0 && (!p.state_in || p.state_in_sr % V == 0) && ok(p.x) && ok(p.state_in) && ok(p.weight);
  if (backward) v = v && p.dy_st % V == 0 && p.dy_sr % V == 0 && ok(p.dy) && ok(p.dstate_out) && ok(p.dx) && ok(p.dstate_in);
  else v = v && ok(p.y) && ok(p.state_out) && (!p.state_out || p.state_out_sr % V == 0);
  return v ? V : 1;
}

template <typename T, int V, int K>
void run(const fdql_causal_conv_t &p, bool backward, hipStream_t s) {
  const Plan q = plan_of(p, V);
  Args a = {p, q.blocks, q.chunks, q.len, (int64_t)q.blocks * p.R * q.chunks, reinterpret_cast<float *>(p.workspace)};
  if (!backward) {
    hipLaunchKernelGGL((k_seqconv_fwd<T, V, K>), dim3((unsigned)((a.units + WPB - 1) / WPB)), dim3(WPB * 64), 0, s, a);
  } else {
    hipLaunchKernelGGL((k_seqconv_bwd<T, V, K>), dim3((unsigned)(q.wgs * q.blocks)), dim3(WPB * 64), 0, s, a);
    if (p.dweight || p.dbias)
      hipLaunchKernelGGL(k_seqconv_finish, dim3((unsigned)((p.D + 63) / 64), K + 1), dim3(1024), 0, s, a.slab, q.wgs, p.D, K, p.dweight, p.dbias);
  }
}
template <typename T, int V>
void run_k(const fdql_causal_conv_t &p, bool backward, hipStream_t s) {
  if (p.K == 2) run<T, V, 2>(p, backward, s);
  else if (p.K == 3) run<T, V, 3>(p, backward, s);
  else run<T, V, 4>(p, backward, s);
}
hipError_t launch(const fdql_causal_conv_t &p, bool backward, hipStream_t s) {
  const bool wide = width_of(p, backward) > 1;
  if (p.dtype == FDQL_F32) wide ? run_k<float, 4>(p, backward, s) : run_k<float, 1>(p, backward, s);
  else if (p.dtype == FDQL_BF16) wide ? run_k<bf16_t, 8>(p, backward, s) : run_k<bf16_t, 1>(p, backward, s);
  else wide ? run_k<f16_t, 8>(p, backward, s) : run_k<f16_t, 1>(p, backward, s);
  return hipGetLastError();
}

}  // namespace

int64_t seqconv_workspace_bytes(const fdql_causal_conv_t &p) {
  const int V = p.dtype == FDQL_F32 ? 4 : 8;
  const int64_t wgs = std::max(plan_of(p, 1).wgs, plan_of(p, V).wgs);
  return wgs * (p.K + 1) * p.D * 4;
}
hipError_t seqconv_fwd_launch(const fdql_causal_conv_t &p, hipStream_t s) { return launch(p, false, s); }
hipError_t seqconv_bwd_launch(const fdql_causal_conv_t &p, hipStream_t s) { return launch(p, true, s); }

}  // namespace fdql
