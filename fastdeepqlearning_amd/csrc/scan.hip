// Selective state-space scan (fdql_scan*): training over windows, prompts, single steps.
//
//   delta_t = softplus(dt_t + bias),  h_t[n] = e^(delta_t A[n]) h_{t-1}[n] + delta_t x_t B_t[n],  y_t = (C_t . h_t + skip x_t) SiLU(z_t)
//
// Layout.  A wave owns CW = 64 / S channels of one row and walks the time axis: lane = s * CW + c holds the NL states
// [s NL, s NL + NL) of channel c in registers, so the sum over n stays in a lane (S = 1) or crosses S lanes, every x / dt / z / y access
// is a run of consecutive channels, and B_t, C_t are the same for the whole wave: they pass through a small LDS tile of TS
// steps and are read back as broadcasts.  Waves of the forward kernels share nothing, so there is no barrier in them.
// Decays are e^(delta A) = exp2((delta log2 e) A): one multiply and one v_exp_f32 per state and step, which is what bounds the
// kernels at N >= 16 (about 28 cycles of a SIMD per 64 states and step forward, 60 backward).
//
// Few rows and a long time axis leave most of the card idle, so the axis is cut into segments: k_scan_carry gets each segment's
// final state from a zero start and the sum of its steps (the product of the decays is e^(A sum delta)), k_scan_combine joins
// them in order, and the main kernel runs every segment from its true start.  Backward does the same from the right.
//
// Backward.  The forward pass keeps the state in front of every TS steps (checkpoints, N floats per channel and tile).  The
// backward kernel rebuilds a tile's states from it, four states at a time (decays and states of TS steps then stay in registers), and
// walks the tile in reverse with g_t = carry + C_t dy_t, carry <- e^(delta A) g_t.  dB and dC sum over channels: 8 values per step and
// part go through a butterfly over the wave that halves the values at each step (permlane swaps, then DPP), then over the
// workgroup's waves in LDS, then over workgroups in a slab that k_scan_bc_finish adds up.  No atomics: results repeat bit by bit.
#include "seq.h"

#include <algorithm>

namespace fdql {
namespace {

constexpr int TS = 8;             // steps per tile
constexpr int WPB = 4;            // waves per workgroup

struct Args {
  fdql_scan_t p;
  int Dg, tpg;                    // channels per group, wave tiles per group
  int nseg, seglen;               // segments of the time axis; seglen is a multiple of TS when nseg > 1
  int wgt, wpw;                   // backward: workgroups per group, waves in each
  float *seg_h, *seg_d;           // [nseg][R][G][tpg][NL][64] joined states / carries; [nseg][R][G][tpg][64] sums of steps
  int *seg_f;                     // [nseg][R] a reset lies in the segment
  float *slab_b, *slab_c;         // [wgt][T][R][G][N]
  float *part_a, *part_s;         // [nseg * R][G][tpg][NL][64], [nseg * R][G][tpg][2][64]: dA; dskip, ddt_bias
};

struct Unit {
  int tile, g, r, seg;
};
__device__ __forceinline__ Unit unit_of(const Args &a, int u) {
  Unit w;
  w.tile = u % a.tpg; u /= a.tpg;
  w.g = u % a.p.G; u /= a.p.G;
  w.r = u % a.p.R;
  w.seg = u / a.p.R;
  return w;
}

__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// x + the same lane's value in the other states' lanes (S lanes CW apart hold parts of one channel's sum)
template <int S>
__device__ __forceinline__ float sum_parts(float v) {
  if constexpr (S >= 4) v += __shfl_xor(v, 16);
  if constexpr (S >= 2) v += __shfl_xor(v, 32);
  return v;
}

template <typename T>
struct Col {                      // one lane's column of a [T, R, D] tensor
  const T *base;
  int64_t st;
  __device__ __forceinline__ float at(int t) const { return to_f(base[t * st]); }
};
template <typename T>
__device__ __forceinline__ Col<T> column(const void *p, int64_t st, int64_t sr, int r, int d) {
  return {reinterpret_cast<const T *>(p) + (int64_t)r * sr + d, st};
}

// bit i: a reset at step t + i (i < nt)
__device__ __forceinline__ unsigned reset_bits(const fdql_scan_t &p, int r, int t, int nt, int lane) {
  if (!p.reset) return 0u;
  const bool on = lane < nt && p.reset[(int64_t)(t + lane) * p.reset_st + (int64_t)r * p.reset_sr] != 0;
  return (unsigned)__ballot(on);
}

// The tile's B or C rows, widened to float and padded with zeros to NP states, spread over `nthreads` threads.
template <typename T, int NP>
__device__ __forceinline__ void stage_rows(const void *src, int64_t st, int64_t sr, int64_t sg, const fdql_scan_t &p, int r, int g, int t, int nt,
                                           float *dst, int tid, int nthreads) {
  const T *b = reinterpret_cast<const T *>(src) + (int64_t)r * sr + (int64_t)g * sg;
  for (int i = tid; i < TS * NP; i += nthreads) {
    const int k = i / NP, n = i % NP;
    dst[i] = (k < nt && n < p.N) ? to_f(b[(int64_t)(t + k) * st + n]) : 0.f;
  }
}

template <int NL, int S>
__device__ __forceinline__ int64_t lane_slot(const Args &a, int64_t block, const Unit &w) {   // first float of a wave's [NL][64] block
  return (((block * a.p.R + w.r) * a.p.G + w.g) * a.tpg + w.tile) * (NL * 64);
}

// ---------------------------------------------------------------------------------------------------------------- forward
template <typename T, int NL, int S>
__global__ __launch_bounds__(WPB * 64) void k_scan_fwd(Args a) {
  constexpr int CW = 64 / S, NP = NL * S;
  __shared__ float lds[WPB][2][TS * NP];
  const fdql_scan_t &p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int u = blockIdx.x * WPB + wave;
  if (u >= a.nseg * p.R * p.G * a.tpg) return;
  const Unit w = unit_of(a, u);
  const int c = lane % CW, s = lane / CW;
  const int dc = w.tile * CW + c, d = w.g * a.Dg + min(dc, a.Dg - 1);
  const bool live = dc < a.Dg;
  const int t0 = w.seg * a.seglen, t1 = min(p.T, t0 + a.seglen);
  float *lB = lds[wave][0], *lC = lds[wave][1];

  const Col<T> X = column<T>(p.x, p.x_st, p.x_sr, w.r, d), DT = column<T>(p.dt, p.dt_st, p.dt_sr, w.r, d),
               Z = column<T>(p.z ? p.z : p.x, p.z ? p.z_st : p.x_st, p.z ? p.z_sr : p.x_sr, w.r, d);
  const float bias = p.dt_bias ? p.dt_bias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
  float h[NL], A[NL];
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int n = s * NL + j;
    A[j] = n < p.N ? p.A[(int64_t)d * p.N + n] * LOG2E : 0.f;
    if (a.nseg > 1) h[j] = a.seg_h[lane_slot<NL, S>(a, w.seg, w) + j * 64 + lane];
    else h[j] = p.state_in && n < p.N ? p.state_in[(int64_t)w.r * p.state_in_sr + (int64_t)d * p.N + n] : 0.f;
  }
  T *yp = reinterpret_cast<T *>(p.y) + (int64_t)w.r * p.D + d;
  const int64_t y_st = (int64_t)p.R * p.D;

  float xn[TS], dn[TS], zn[TS];
#pragma unroll
  for (int i = 0; i < TS; ++i) {
    const int t = min(t0 + i, t1 - 1);
    xn[i] = X.at(t); dn[i] = DT.at(t); zn[i] = Z.at(t);
  }
  for (int t = t0; t < t1; t += TS) {
    const int nt = min(TS, t1 - t);
    stage_rows<T, NP>(p.B, p.B_st, p.B_sr, p.B_sg, p, w.r, w.g, t, nt, lB, lane, 64);
    stage_rows<T, NP>(p.C, p.C_st, p.C_sr, p.C_sg, p, w.r, w.g, t, nt, lC, lane, 64);
    const unsigned rst = reset_bits(p, w.r, t, nt, lane);
    if (p.checkpoints) {
      float *ck = p.checkpoints + lane_slot<NL, S>(a, t / TS, w) + lane;
#pragma unroll
      for (int j = 0; j < NL; ++j) ck[j * 64] = h[j];
    }
    float x[TS], del[TS], z[TS];
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      x[i] = xn[i];
      z[i] = zn[i];
      del[i] = dn[i] + bias;
    }
    if (t + TS < t1) {
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        const int tn = min(t + TS + i, t1 - 1);
        xn[i] = X.at(tn); dn[i] = DT.at(tn); zn[i] = Z.at(tn);
      }
    }
    if (p.dt_softplus) {
#pragma unroll
      for (int i = 0; i < TS; ++i) del[i] = softplus_f(del[i]);
    }
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      if (i < nt) {
        if (rst >> i & 1) {
#pragma unroll
          for (int j = 0; j < NL; ++j) h[j] = 0.f;
        }
        const float dx = del[i] * x[i];
        float acc = 0.f;
#pragma unroll
        for (int j = 0; j < NL; ++j) {
          const float e = __builtin_amdgcn_exp2f(del[i] * A[j]);
          h[j] = fmaf(e, h[j], dx * lB[i * NP + s * NL + j]);
          acc = fmaf(h[j], lC[i * NP + s * NL + j], acc);
        }
        acc = sum_parts<S>(acc);
        float y = fmaf(skip, x[i], acc);
        if (p.z) y *= z[i] * sigmoid_f(z[i]);
        if (live && s == 0) yp[(int64_t)(t + i) * y_st] = from_f<T>(y);
      }
    }
    wave_lds_fence();
  }
  if (p.state_out && t1 == p.T && live) {
#pragma unroll
    for (int j = 0; j < NL; ++j)
      if (s * NL + j < p.N) p.state_out[((int64_t)w.r * p.D + d) * p.N + s * NL + j] = h[j];
  }
}

// A segment's contribution to its neighbour.  Forward (REV = 0): the state at its end from a zero start, segments [0, nseg - 1).
// Backward (REV = 1): the carry at its start from a zero carry, segments [1, nseg).
template <typename T, int NL, int S, int REV>
__global__ __launch_bounds__(WPB * 64) void k_scan_carry(Args a) {
  constexpr int CW = 64 / S, NP = NL * S;
  __shared__ float lds[WPB][TS * NP];
  const fdql_scan_t &p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int u = blockIdx.x * WPB + wave;
  if (u >= (a.nseg - 1) * p.R * p.G * a.tpg) return;
  Unit w = unit_of(a, u);
  if (REV) w.seg += 1;
  const int c = lane % CW, s = lane / CW;
  const int dc = w.tile * CW + c, d = w.g * a.Dg + min(dc, a.Dg - 1);
  const bool live = dc < a.Dg;
  const int t0 = w.seg * a.seglen, t1 = min(p.T, t0 + a.seglen);
  float *lds_w = lds[wave];
  const Col<T> DT = column<T>(p.dt, p.dt_st, p.dt_sr, w.r, d),
               V = REV ? column<T>(p.dy, p.dy_st, p.dy_sr, w.r, d) : column<T>(p.x, p.x_st, p.x_sr, w.r, d);
  const bool gate = REV && p.z;
  const Col<T> Z = gate ? column<T>(p.z, p.z_st, p.z_sr, w.r, d) : DT;
  const float bias = p.dt_bias ? p.dt_bias[d] : 0.f;
  float h[NL], A[NL], sum = 0.f;
  int any = 0;
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    h[j] = 0.f;
    A[j] = s * NL + j < p.N ? p.A[(int64_t)d * p.N + s * NL + j] * LOG2E : 0.f;
  }
  const int nt_all = t1 - t0, tiles = (nt_all + TS - 1) / TS;
  for (int k = 0; k < tiles; ++k) {
    const int t = t0 + (REV ? tiles - 1 - k : k) * TS, nt = min(TS, t1 - t);
    if (REV) stage_rows<T, NP>(p.C, p.C_st, p.C_sr, p.C_sg, p, w.r, w.g, t, nt, lds_w, lane, 64);
    else stage_rows<T, NP>(p.B, p.B_st, p.B_sr, p.B_sg, p, w.r, w.g, t, nt, lds_w, lane, 64);
    const unsigned rst = reset_bits(p, w.r, t, nt, lane);
    any |= rst != 0;
    float v[TS], del[TS];
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      const int ti = min(t + i, t1 - 1);
      del[i] = DT.at(ti) + bias;
      v[i] = V.at(ti);
      if (gate) {
        const float z = Z.at(ti);
        v[i] *= z * sigmoid_f(z);
      }
      if (p.dt_softplus) del[i] = softplus_f(del[i]);
    }
    wave_lds_fence();
#pragma unroll
    for (int ii = 0; ii < TS; ++ii) {
      const int i = REV ? TS - 1 - ii : ii;
      if (i < nt) {
        const bool cut = rst >> i & 1;
        sum += del[i];
        const float f = REV ? v[i] : del[i] * v[i];
        if (!REV && cut) {
#pragma unroll
          for (int j = 0; j < NL; ++j) h[j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < NL; ++j) {
          const float e = __builtin_amdgcn_exp2f(del[i] * A[j]);
          if (REV) h[j] = e * fmaf(f, lds_w[i * NP + s * NL + j], h[j]);
          else h[j] = fmaf(e, h[j], f * lds_w[i * NP + s * NL + j]);
        }
        if (REV && cut) {
#pragma unroll
          for (int j = 0; j < NL; ++j) h[j] = 0.f;
        }
      }
    }
    wave_lds_fence();
  }
  const int64_t o = lane_slot<NL, S>(a, w.seg, w);
#pragma unroll
  for (int j = 0; j < NL; ++j) a.seg_h[o + j * 64 + lane] = live ? h[j] : 0.f;
  a.seg_d[o / NL + lane] = sum;
  if (lane == 0 && w.tile == 0 && w.g == 0) a.seg_f[(int64_t)w.seg * p.R + w.r] = any;
}

// seg_h becomes the state every segment starts from (REV = 0) / the carry that enters every segment from the right (REV = 1).
template <int NL, int S, int REV>
__global__ __launch_bounds__(256) void k_scan_combine(Args a) {
  constexpr int CW = 64 / S;
  const fdql_scan_t &p = a.p;
  const int64_t per = (int64_t)p.R * p.G * a.tpg * NL * 64;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= per) return;
  const int lane = (int)(i & 63), j = (int)(i / 64 % NL);
  const int64_t blk = i / (64 * NL);
  const int tile = (int)(blk % a.tpg), g = (int)(blk / a.tpg % p.G), r = (int)(blk / a.tpg / p.G);
  const int dc = tile * CW + lane % CW, n = lane / CW * NL + j;
  const bool live = dc < a.Dg && n < p.N;
  const int d = g * a.Dg + min(dc, a.Dg - 1);
  const float A = live ? p.A[(int64_t)d * p.N + n] * LOG2E : 0.f;
  float cur = 0.f;
  if (live) {
    if (REV) cur = p.dstate_out ? p.dstate_out[((int64_t)r * p.D + d) * p.N + n] : 0.f;
    else cur = p.state_in ? p.state_in[(int64_t)r * p.state_in_sr + (int64_t)d * p.N + n] : 0.f;
  }
  for (int k = 0; k < a.nseg; ++k) {
    const int seg = REV ? a.nseg - 1 - k : k;
    float *at = a.seg_h + seg * per + i;
    if (k < a.nseg - 1) {
      const float own = *at, sum = a.seg_d[((int64_t)seg * p.R * p.G * a.tpg + blk) * 64 + lane];
      *at = cur;
      const float e = __builtin_amdgcn_exp2f(sum * A);
      cur = a.seg_f[(int64_t)seg * p.R + r] ? own : fmaf(e, cur, own);
    } else {
      *at = cur;
    }
  }
}

// --------------------------------------------------------------------------------------------------------------- backward
// v_permlane32_swap / v_permlane16_swap exchange half of one register's lanes with half of another's, so a swap and an add leave
// in each half the sum over both of ONE of two values; inside a row of 16 the same takes two selects and a DPP add.
__device__ __forceinline__ float dpp_ror8(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, true)); }
__device__ __forceinline__ float dpp_half_mirror(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, true)); }
__device__ __forceinline__ float dpp_xor2(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4e, 0xf, 0xf, true)); }
__device__ __forceinline__ float dpp_xor1(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xb1, 0xf, 0xf, true)); }

// lanes with BIT clear end with the sum (over lanes BIT apart) of a, the others with that of b
template <int BIT>
__device__ __forceinline__ float fold(float a, float b, int lane) {
  if constexpr (BIT == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else if constexpr (BIT == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else {
    const bool up = lane & BIT;
    const float keep = up ? b : a, give = up ? a : b;
    if constexpr (BIT == 8) return keep + dpp_ror8(give);
    else if constexpr (BIT == 4) return keep + dpp_half_mirror(give);
    else return keep + dpp_xor2(give);
  }
}
// Sums of eight values over the CW consecutive lanes of a part; value k = 4 b2 + 2 b1 + b0 ends (complete) in the lanes whose bits
// CW/2, CW/4, CW/8 are b2, b1, b0.
template <int CW>
__device__ __forceinline__ float sum8(const float v[8], int lane) {
  float u[4], q[2], o;
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = fold<CW / 2>(v[i], v[i + 4], lane);
#pragma unroll
  for (int i = 0; i < 2; ++i) q[i] = fold<CW / 4>(u[i], u[i + 2], lane);
  o = fold<CW / 8>(q[0], q[1], lane);
  if constexpr (CW >= 64) o += dpp_half_mirror(o);
  if constexpr (CW >= 32) o += dpp_xor2(o);
  o += dpp_xor1(o);
  return o;
}

template <typename T, int NL, int S>
__global__ __launch_bounds__(WPB * 64, 2) void k_scan_bwd(Args a) {
  constexpr int CW = 64 / S, NP = NL * S, PARTS = NL / 4;
  __shared__ float lB[TS * NP], lC[TS * NP];
  __shared__ float red[WPB][TS][2][NP];
  const fdql_scan_t &p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nthreads = blockDim.x;
  int u = blockIdx.x;
  Unit w;
  const int wgt = u % a.wgt; u /= a.wgt;
  w.g = u % p.G; u /= p.G;
  w.r = u % p.R;
  w.seg = u / p.R;
  w.tile = wgt * a.wpw + wave;
  const int active = min(a.wpw, a.tpg - wgt * a.wpw);
  const bool idle = w.tile >= a.tpg;            // a wave past the group's channels still takes part in staging and barriers
  if (idle) w.tile = a.tpg - 1;
  const int c = lane % CW, s = lane / CW;
  const int dc = w.tile * CW + c, d = w.g * a.Dg + min(dc, a.Dg - 1);
  const bool live = !idle && dc < a.Dg;
  const int t0 = w.seg * a.seglen, t1 = min(p.T, t0 + a.seglen);

  const Col<T> X = column<T>(p.x, p.x_st, p.x_sr, w.r, d), DT = column<T>(p.dt, p.dt_st, p.dt_sr, w.r, d),
               DY = column<T>(p.dy, p.dy_st, p.dy_sr, w.r, d), Z = p.z ? column<T>(p.z, p.z_st, p.z_sr, w.r, d) : X;
  const float bias = p.dt_bias ? p.dt_bias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
  float A[NL], carry[NL], dA[NL], dskip = 0.f, dbias = 0.f;
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int n = s * NL + j;
    A[j] = n < p.N ? p.A[(int64_t)d * p.N + n] : 0.f;
    dA[j] = 0.f;
    if (a.nseg > 1) carry[j] = a.seg_h[lane_slot<NL, S>(a, w.seg, w) + j * 64 + lane];
    else carry[j] = live && p.dstate_out && n < p.N ? p.dstate_out[((int64_t)w.r * p.D + d) * p.N + n] : 0.f;
  }
  const int64_t o_st = (int64_t)p.R * p.D, o0 = (int64_t)w.r * p.D + d;
  const int tiles = (t1 - t0 + TS - 1) / TS;
  for (int k = tiles - 1; k >= 0; --k) {
    const int t = t0 + k * TS, nt = min(TS, t1 - t);
    stage_rows<T, NP>(p.B, p.B_st, p.B_sr, p.B_sg, p, w.r, w.g, t, nt, lB, threadIdx.x, nthreads);
    stage_rows<T, NP>(p.C, p.C_st, p.C_sr, p.C_sg, p, w.r, w.g, t, nt, lC, threadIdx.x, nthreads);
    const unsigned rst = reset_bits(p, w.r, t, nt, lane);
    float x[TS], del[TS], dy[TS], yc[TS], dd[TS], gx[TS];
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      const int ti = min(t + i, t1 - 1);
      x[i] = X.at(ti);
      del[i] = DT.at(ti) + bias;
      dy[i] = DY.at(ti);
      if (p.z) {
        const float z = Z.at(ti);
        dy[i] *= z * sigmoid_f(z);
      }
      if (!live) x[i] = dy[i] = 0.f;
      if (p.dt_softplus) del[i] = softplus_f(del[i]);
      yc[i] = dd[i] = gx[i] = 0.f;
    }
    __syncthreads();
    const float *ck = p.checkpoints + lane_slot<NL, S>(a, t / TS, w) + lane;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      float h[TS + 1][4], e[TS][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[0][j] = ck[(part * 4 + j) * 64];
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        const float dl = del[i] * LOG2E, dx = del[i] * x[i];
        const bool cut = rst >> i & 1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = s * NL + part * 4 + j;
          if (i < nt) {
            e[i][j] = __builtin_amdgcn_exp2f(dl * A[part * 4 + j]);
            h[i + 1][j] = dx * lB[i * NP + n];
            if (!cut) h[i + 1][j] = fmaf(e[i][j], h[i][j], h[i + 1][j]);
            yc[i] = fmaf(h[i + 1][j], lC[i * NP + n], yc[i]);
          } else {
            e[i][j] = 0.f;
            h[i + 1][j] = h[i][j];
          }
        }
      }
#pragma unroll
      for (int ii = 0; ii < TS; ++ii) {
        const int i = TS - 1 - ii;
        if (i < nt) {
          const float dx = del[i] * x[i];
          const bool cut = rst >> i & 1;
          float v[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int n = s * NL + part * 4 + j, m = part * 4 + j;
            const float g = fmaf(dy[i], lC[i * NP + n], carry[m]);
            float ga = 0.f;
            if (!cut) {
              ga = g * e[i][j];
              const float q = ga * h[i][j];
              dd[i] = fmaf(q, A[m], dd[i]);
              dA[m] = fmaf(q, del[i], dA[m]);
            }
            gx[i] = fmaf(g, lB[i * NP + n], gx[i]);
            v[j] = g * dx;
            v[4 + j] = h[i + 1][j] * dy[i];
            carry[m] = ga;
          }
          const float o = sum8<CW>(v, lane);
          // value index: dB (first bit clear) or dC, then the state; one lane of each holding group writes
          if ((lane & (CW / 8 - 1)) == 0) {
            const int b2 = (lane / (CW / 2)) & 1, b1 = (lane / (CW / 4)) & 1, b0 = (lane / (CW / 8)) & 1;
            red[wave][i][b2][s * NL + part * 4 + 2 * b1 + b0] = o;
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      if (i < nt) {
        yc[i] = sum_parts<S>(yc[i]);
        dd[i] = sum_parts<S>(dd[i]);
        gx[i] = sum_parts<S>(gx[i]);
        const float core = fmaf(skip, x[i], yc[i]);
        float ddt = fmaf(x[i], gx[i], dd[i]);
        if (p.dt_softplus) ddt *= sigmoid_f(DT.at(t + i) + bias);
        dskip = fmaf(dy[i], x[i], dskip);
        dbias += ddt;
        if (live && s == 0) {
          const int64_t o = o0 + (int64_t)(t + i) * o_st;
          if (p.dx) reinterpret_cast<T *>(p.dx)[o] = from_f<T>(fmaf(skip, dy[i], del[i] * gx[i]));
          if (p.ddt) reinterpret_cast<T *>(p.ddt)[o] = from_f<T>(ddt);
          if (p.z && p.dz) {
            const float z = Z.at(t + i), sg = sigmoid_f(z);
            reinterpret_cast<T *>(p.dz)[o] = from_f<T>(DY.at(t + i) * core * sg * fmaf(z, 1.f - sg, 1.f));
          }
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nt * 2 * NP; i += nthreads) {
      const int n = i % NP, which = i / NP % 2, k2 = i / (2 * NP);
      if (n < p.N) {
        float v = 0.f;
        for (int q = 0; q < active; ++q) v += red[q][k2][which][n];
        float *slab = which ? a.slab_c : a.slab_b;
        slab[((((int64_t)wgt * p.T + t + k2) * p.R + w.r) * p.G + w.g) * p.N + n] = v;
      }
    }
    __syncthreads();
  }
  if (idle) return;
  if (w.seg == 0 && p.dstate_in && live) {
#pragma unroll
    for (int j = 0; j < NL; ++j)
      if (s * NL + j < p.N) p.dstate_in[((int64_t)w.r * p.D + d) * p.N + s * NL + j] = carry[j];
  }
  const int64_t o = lane_slot<NL, S>(a, w.seg, w);
#pragma unroll
  for (int j = 0; j < NL; ++j) a.part_a[o + j * 64 + lane] = dA[j];
  a.part_s[o / NL * 2 + lane] = dskip;
  a.part_s[o / NL * 2 + 64 + lane] = dbias;
}

// dB / dC: the workgroups' slabs added in order, rounded once to the tensor's type.
template <typename T>
__global__ __launch_bounds__(256) void k_scan_bc_finish(Args a) {
  const int64_t n = (int64_t)a.p.T * a.p.R * a.p.G * a.p.N;
  const float *slab = blockIdx.y ? a.slab_c : a.slab_b;
  T *out = reinterpret_cast<T *>(blockIdx.y ? a.p.dC : a.p.dB);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int k = 0; k < a.wgt; ++k) v += slab[k * n + i];
    out[i] = from_f<T>(v);
  }
}

// dA, dskip, ddt_bias: partials of the (segment, row) pairs added up; a workgroup per 64 lanes of one state, 16 slices of the pairs.
template <int NL, int S>
__global__ __launch_bounds__(1024) void k_scan_par_finish(Args a) {
  constexpr int CW = 64 / S;
  __shared__ float red[16][64];
  const fdql_scan_t &p = a.p;
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
  const int j = blockIdx.x % (NL + 2), blk = blockIdx.x / (NL + 2);
  const int64_t pairs = (int64_t)a.nseg * p.R, blocks = (int64_t)p.G * a.tpg;
  float v = 0.f;
  for (int64_t k = slice; k < pairs; k += 16)
    v += j < NL ? a.part_a[((k * blocks + blk) * NL + j) * 64 + lane] : a.part_s[((k * blocks + blk) * 2 + j - NL) * 64 + lane];
  red[slice][lane] = v;
  __syncthreads();
  if (slice) return;
  v = 0.f;
#pragma unroll
  for (int q = 0; q < 16; ++q) v += red[q][lane];
  const int g = blk / a.tpg, dc = blk % a.tpg * CW + lane % CW, n = lane / CW * NL + j;
  if (dc >= a.Dg) return;
  const int64_t d = (int64_t)g * a.Dg + dc;
  if (j < NL) {
    if (n < p.N && p.dA) p.dA[d * p.N + n] = v;
  } else if (lane < CW) {
    float *out = j == NL ? p.dskip : p.ddt_bias;
    if (out) out[d] = v;
  }
}

// ------------------------------------------------------------------------------------------------------------ single steps
// One step for every row: the state is read and written once, V = 4 states (16 bytes) per lane where the state's rows allow it.  A wave
// owns 64 channels of one row: lane = channel for delta, x and the gate; then LPC lanes share a channel and the wave passes over
// its state in LPC turns, consecutive lanes on consecutive addresses.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_scan_step(fdql_scan_t p, int Dg, int tpg, int lpc) {
  typedef float vec __attribute__((ext_vector_type(V)));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t u = (int64_t)blockIdx.x * 4 + wave;
  if (u >= (int64_t)p.R * p.G * tpg) return;
  const int tile = (int)(u % tpg), g = (int)(u / tpg % p.G), r = (int)(u / tpg / p.G);
  const int dc = tile * 64 + lane, d = g * Dg + min(dc, Dg - 1);
  const float x = to_f(reinterpret_cast<const T *>(p.x)[(int64_t)r * p.x_sr + d]);
  float del = to_f(reinterpret_cast<const T *>(p.dt)[(int64_t)r * p.dt_sr + d]) + (p.dt_bias ? p.dt_bias[d] : 0.f);
  if (p.dt_softplus) del = softplus_f(del);
  const float dx = del * x;
  float y = 0.f;
  const bool fresh = !p.state_in || (p.reset && p.reset[(int64_t)r * p.reset_sr] != 0);
  const int cpt = 64 / lpc, sub = lane % lpc, n = sub * V;       // channels per turn; this lane's part of the state
  const T *Bp = reinterpret_cast<const T *>(p.B) + (int64_t)r * p.B_sr + (int64_t)g * p.B_sg;
  const T *Cp = reinterpret_cast<const T *>(p.C) + (int64_t)r * p.C_sr + (int64_t)g * p.C_sg;
  float B[V], C[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    B[k] = n + k < p.N ? to_f(Bp[n + k]) : 0.f;
    C[k] = n + k < p.N ? to_f(Cp[n + k]) : 0.f;
  }
  for (int it = 0; it < lpc; ++it) {
    const int ch = it * cpt + lane / lpc, cc = tile * 64 + ch;     // this turn's channel
    const float del_c = __shfl(del, ch), dx_c = __shfl(dx, ch);
    float acc = 0.f;
    if (cc < Dg && n < p.N) {
      const int64_t dd = g * Dg + cc;
      const vec A = *reinterpret_cast<const vec *>(p.A + dd * p.N + n);
      vec h = {};
      if (!fresh) h = *reinterpret_cast<const vec *>(p.state_in + (int64_t)r * p.state_in_sr + dd * p.N + n);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        h[k] = fmaf(__builtin_amdgcn_exp2f(del_c * (A[k] * LOG2E)), h[k], dx_c * B[k]);
        if (fresh) h[k] = dx_c * B[k];
        acc = fmaf(h[k], C[k], acc);
      }
      if (p.state_out) *reinterpret_cast<vec *>(p.state_out + ((int64_t)r * p.D + dd) * p.N + n) = h;
    }
    for (int m = 1; m < lpc; m <<= 1) acc += __shfl_xor(acc, m);
    const float back = __shfl(acc, (lane % cpt) * lpc);            // the sum of channel it * cpt + (lane % cpt)
    if (lane / cpt == it) y = back;
  }
  y = fmaf(p.skip ? p.skip[d] : 0.f, x, y);
  if (p.z) {
    const float z = to_f(reinterpret_cast<const T *>(p.z)[(int64_t)r * p.z_sr + d]);
    y *= z * sigmoid_f(z);
  }
  if (dc < Dg) reinterpret_cast<T *>(p.y)[(int64_t)r * p.D + d] = from_f<T>(y);
}

// ------------------------------------------------------------------------------------------------------------------- host
struct Plan {
  int NL, S, tpg, Dg, nseg, seglen, wgt, wpw;
};

int cus() { return 256; }

// States per lane and lanes per channel, then segments.
Plan plan_of(const fdql_scan_t &p) {
  Plan q;
  q.Dg = p.D / p.G;
  const int64_t rows = (int64_t)p.R * p.G;
  if (p.N <= 4) q.NL = 4, q.S = 1;
  else if (p.N <= 16) {
    const bool few = rows * ((q.Dg + 63) / 64) < 512;
    q.NL = few ? 4 : p.N <= 8 ? 8 : 16;
    q.S = few ? 4 : 1;
  } else if (p.N <= 32) q.NL = 16, q.S = 2;
  else q.NL = 16, q.S = 4;
  const int CW = 64 / q.S;
  q.tpg = (q.Dg + CW - 1) / CW;
  const int64_t waves = rows * q.tpg;
  q.nseg = 1;
  q.seglen = p.T;
  if (waves > 0 && waves < 1024 && p.T >= 128) {
    const int64_t want = std::min<int64_t>((2048 + waves - 1) / waves, p.T / 64);
    if (want > 1) {
      q.seglen = (int)(((p.T + want - 1) / want + TS - 1) / TS * TS);
      q.nseg = (p.T + q.seglen - 1) / q.seglen;
    }
  }
  q.wgt = (q.tpg + WPB - 1) / WPB;
  q.wpw = (q.tpg + q.wgt - 1) / q.wgt;
  return q;
}

int64_t seg_floats(const fdql_scan_t &p, const Plan &q) {
  if (q.nseg == 1) return 0;
  const int64_t blocks = (int64_t)p.R * p.G * q.tpg;
  return q.nseg * blocks * (q.NL + 1) * 64 + ((int64_t)q.nseg * p.R + 3) / 4 * 4;
}

Args args_of(const fdql_scan_t &p, const Plan &q, bool backward) {
  Args a = {};
  a.p = p;
  a.Dg = q.Dg; a.tpg = q.tpg; a.nseg = q.nseg; a.seglen = q.seglen; a.wgt = q.wgt; a.wpw = q.wpw;
  float *f = reinterpret_cast<float *>(p.workspace);
  const int64_t blocks = (int64_t)p.R * p.G * q.tpg;
  if (q.nseg > 1) {
    a.seg_h = f; f += q.nseg * blocks * q.NL * 64;
    a.seg_d = f; f += q.nseg * blocks * 64;
    a.seg_f = reinterpret_cast<int *>(f); f += ((int64_t)q.nseg * p.R + 3) / 4 * 4;
  }
  if (backward) {
    const int64_t bc = q.wgt * (int64_t)p.T * p.R * p.G * p.N;
    a.slab_b = f; f += bc;
    a.slab_c = f; f += bc;
    a.part_a = f; f += q.nseg * blocks * q.NL * 64;
    a.part_s = f; f += q.nseg * blocks * 2 * 64;
  }
  return a;
}

template <int NL_, int S_>
struct Var { static constexpr int NL = NL_, S = S_; };

template <typename F>
hipError_t with_variant(const Plan &q, F f) {
  if (q.S == 4) return q.NL == 4 ? f(Var<4, 4>()) : f(Var<16, 4>());
  if (q.S == 2) return f(Var<16, 2>());
  return q.NL == 4 ? f(Var<4, 1>()) : q.NL == 8 ? f(Var<8, 1>()) : f(Var<16, 1>());
}

template <typename T>
hipError_t fwd(const fdql_scan_t &p, hipStream_t s) {
  const Plan q = plan_of(p);
  return with_variant(q, [&](auto v) {
    constexpr int NL = decltype(v)::NL, S = decltype(v)::S;
    const Args a = args_of(p, q, false);
    const int64_t per = (int64_t)p.R * p.G * q.tpg;
    if (q.nseg > 1) {
      hipLaunchKernelGGL((k_scan_carry<T, NL, S, 0>), dim3((unsigned)(((q.nseg - 1) * per + WPB - 1) / WPB)), dim3(WPB * 64), 0, s, a);
      hipLaunchKernelGGL((k_scan_combine<NL, S, 0>), dim3((unsigned)((per * NL * 64 + 255) / 256)), dim3(256), 0, s, a);
    }
    hipLaunchKernelGGL((k_scan_fwd<T, NL, S>), dim3((unsigned)((q.nseg * per + WPB - 1) / WPB)), dim3(WPB * 64), 0, s, a);
    return hipGetLastError();
  });
}

template <typename T>
hipError_t bwd(const fdql_scan_t &p, hipStream_t s) {
  const Plan q = plan_of(p);
  return with_variant(q, [&](auto v) {
    constexpr int NL = decltype(v)::NL, S = decltype(v)::S;
    const Args a = args_of(p, q, true);
    const int64_t per = (int64_t)p.R * p.G * q.tpg;
    if (q.nseg > 1) {
      hipLaunchKernelGGL((k_scan_carry<T, NL, S, 1>), dim3((unsigned)(((q.nseg - 1) * per + WPB - 1) / WPB)), dim3(WPB * 64), 0, s, a);
      hipLaunchKernelGGL((k_scan_combine<NL, S, 1>), dim3((unsigned)((per * NL * 64 + 255) / 256)), dim3(256), 0, s, a);
    }
    hipLaunchKernelGGL((k_scan_bwd<T, NL, S>), dim3((unsigned)((int64_t)q.nseg * p.R * p.G * q.wgt)), dim3(q.wpw * 64), 0, s, a);
    const int64_t bc = (int64_t)p.T * p.R * p.G * p.N;
    hipLaunchKernelGGL((k_scan_bc_finish<T>), dim3((unsigned)std::min<int64_t>((bc + 255) / 256, 8 * cus()), 2), dim3(256), 0, s, a);
    hipLaunchKernelGGL((k_scan_par_finish<NL, S>), dim3((unsigned)(p.G * q.tpg * (NL + 2))), dim3(1024), 0, s, a);
    return hipGetLastError();
  });
}

template <typename T>
hipError_t step(const fdql_scan_t &p, hipStream_t s) {
  const int Dg = p.D / p.G, tpg = (Dg + 63) / 64;
  const auto al = [](const void *q) { return ((uintptr_t)q & 15) == 0; };
  const bool vec = p.N % 4 == 0 && al(p.A) && al(p.state_in) && al(p.state_out) && (!p.state_in || p.state_in_sr % 4 == 0);
  int lpc = 1;
  while (lpc * (vec ? 4 : 1) < p.N) lpc <<= 1;
  const dim3 grid((unsigned)(((int64_t)p.R * p.G * tpg + 3) / 4));
  if (vec) hipLaunchKernelGGL((k_scan_step<T, 4>), grid, dim3(256), 0, s, p, Dg, tpg, lpc);
  else hipLaunchKernelGGL((k_scan_step<T, 1>), grid, dim3(256), 0, s, p, Dg, tpg, lpc);
  return hipGetLastError();
}

}  // namespace

// A single step without checkpoints has a kernel of its own; with them (a window of one step in training) it is an ordinary tile.
static bool is_step(const fdql_scan_t &p) { return p.T == 1 && !p.checkpoints; }

int64_t scan_checkpoint_floats(const fdql_scan_t &p) {
  const Plan q = plan_of(p);
  return ((int64_t)p.T + TS - 1) / TS * p.R * p.G * q.tpg * q.NL * 64;
}
int64_t scan_workspace_bytes(const fdql_scan_t &p, bool backward) {
  const Plan q = plan_of(p);
  int64_t n = seg_floats(p, q);
  if (backward) n += 2 * (q.wgt * (int64_t)p.T * p.R * p.G * p.N) + (int64_t)q.nseg * p.R * p.G * q.tpg * (q.NL + 2) * 64;
  return n * 4;
}
hipError_t scan_fwd_launch(const fdql_scan_t &p, hipStream_t s) {
  if (is_step(p)) return p.dtype == FDQL_F32 ? step<float>(p, s) : p.dtype == FDQL_BF16 ? step<bf16_t>(p, s) : step<f16_t>(p, s);
  return p.dtype == FDQL_F32 ? fwd<float>(p, s) : p.dtype == FDQL_BF16 ? fwd<bf16_t>(p, s) : fwd<f16_t>(p, s);
}
hipError_t scan_bwd_launch(const fdql_scan_t &p, hipStream_t s) {
  return p.dtype == FDQL_F32 ? bwd<float>(p, s) : p.dtype == FDQL_BF16 ? bwd<bf16_t>(p, s) : bwd<f16_t>(p, s);
}

}  // namespace fdql
