// Selective state-space scan (fdql_scan*): training over windows, prompts, single steps.
//
//   delta_t = softplus(dt_t + bias),  h_t[n] = e^(delta_t A[n]) h_{t-1}[n] + delta_t x_t B_t[n],  y_t = (C_t . h_t + skip x_t) SiLU(z_t)
//
// Layout.  A wave owns 16 channels of one row and walks the time axis: four neighbouring lanes share a channel, lane = 4 c + s holds the NL
// states [s NL, s NL + NL) of channel c in registers (NL 2, 4, 8, 16 for up to 8, 16, 32, 64 states).  The sum over n crosses a quad of lanes, and
// what a step has to do beside its states (loads, softplus, gate, store) is dealt to the quad, two of a tile's eight steps each.  B_t and
// C_t are the same for the whole wave: they pass through a small LDS tile of eight steps and are read back as broadcasts.  The next tile's
// reads are under way while one is computed.  Waves of the forward kernels share nothing, so there is no barrier in them.
// Decays are e^(delta A) = exp2(delta (A log2 e)): one multiply and one v_exp_f32 per state and step; the rounding of A log2 e is one of A's own size.
// Vector instructions bound the kernels (forward at N 16: five per state and step, of which the power takes four times as long, and some 150 per
// tile for the rest; backward 18, which are about half of its time, the rest per-tile work and scalar registers held in vector lanes).
// Measured: float 50 x 256 x 512, N 16: forward 42 us (its 213 MB with the checkpoints would take 41), backward 118; bf16 prompt 16383 x 1 x
// 1024: carries 57, join 16, outputs 76 us.
//
// Lanes without a channel and states behind the last one compute on zeros.  Zero times a step that is infinite or NaN would not stay zero: a
// tile that holds one takes the form that selects, as a tile with a reset does.  Only the kernels for other numbers of states than 8, 16, 32 and
// 64 (PAD) look for it: the masks cost registers (float windows of 12 states 161 us -> 170, of 16, without them, 168.5 against 166.5).
//
// Few rows and a long time axis leave most of the card idle, so the axis is cut into segments: k_scan_fwd<CARRY> gets each segment's
// final state from a zero start and the sum of its steps (the product of the decays is e^(A sum delta)), k_scan_combine joins
// them in order, and the main kernel runs every segment from its true start.  Backward does the same from the right.
//
// Backward.  The forward pass keeps the state in front of every eighth step (checkpoints, N floats per channel and tile).  The
// backward kernel rebuilds a tile's states from it, two states of a lane at a time (decays and states of TS steps then stay in registers), and
// walks the tile in reverse with g_t = carry + C_t dy_t, carry <- e^(delta A) g_t.  dB and dC sum over channels, 4 values per step, lane and
// pass: permlane swaps halve the values while they add (v_permlane32_swap exchanges half of one register's lanes with half of another's),
// two DPP rotations finish - a channel's parts are neighbouring lanes so that these steps need no selects; then the workgroup's waves meet in
// LDS, the workgroups in a slab that k_scan_finish adds up.  No atomics: results repeat bit by bit.  (One-hot v_mfma_f32_16x16x4 products
// for these sums measured slower, 190 us against 126 at 50 x 256 x 512 x 16: float32 matrix instructions and vector arithmetic do not overlap.)
#include "seq.h"

#include <algorithm>
#include <type_traits>

namespace fdql {
namespace {

constexpr int TS = 8;             // steps per tile
constexpr int S = 4, CW = 64 / S; // lanes that share a channel, channels of a wave
constexpr int OWN = TS / S;       // steps of a tile whose state-independent work a lane does
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

typedef float v4f __attribute__((ext_vector_type(4)));

// Nothing is read or computed ahead across this point: unrolled code would otherwise fetch every tile row into registers first, and spill.
__device__ __forceinline__ void pass_edge() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// How many of the N states lie at or behind a lane's first one, worked out where it is asked for (the compiler would hold a mask per state through the loop).
__device__ __forceinline__ int states_left(int N, int first) {
  int left = N - first;
  asm volatile("" : "+v"(left));
  return left;
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

// The value is computed by here (an accumulation put off to the end would keep every one of its terms in a register).
__device__ __forceinline__ void settle(float &v) { asm volatile("" : "+v"(v)); }

// A lane's view of a [T, R, D] tensor: one channel of one row from its part's step on (part s of a tile does the steps S q + s).
template <typename T>
struct Col {
  const T *at0;
  int64_t st;
  __device__ __forceinline__ T at(int t, int q) const { return at0[(int64_t)(t + q * S) * st]; }   // (scalar but for the last addition)
};
template <typename T>
__device__ __forceinline__ Col<T> col_of(const void *p, int64_t st, int64_t sr, int r, int s, int d) {
  return {reinterpret_cast<const T *>(p) + (int64_t)r * sr + s * st + d, st};
}

template <int NL>
__device__ __forceinline__ int64_t lane_slot(const Args &a, int64_t block, const Unit &w) {   // first float of a wave's [NL][64] block
  return (((block * a.p.R + w.r) * a.p.G + w.g) * a.tpg + w.tile) * (NL * 64);
}

// A tile's B or C rows on their way to LDS, one wave's work: element lane + 64 q is (step, state) = (/ NP, % NP), zeros behind state N.
template <typename T, int NP>
struct Rows {
  static constexpr int Q = TS * NP / 64, KQ = 64 / NP;     // elements per lane, steps that 64 of them span
  static_assert(64 % NP == 0, "a row must not straddle the lanes");
  const T *base;
  int64_t st;
  int k;
  bool on;
  T v[Q];
  __device__ __forceinline__ Rows(const void *p, int64_t st_, int64_t sr, int64_t sg, const Unit &w, int N, int lane)
      : base(reinterpret_cast<const T *>(p) + (int64_t)w.r * sr + (int64_t)w.g * sg + (lane / NP) * st_ + min(lane % NP, N - 1)), st(st_), k(lane / NP),
        on(lane % NP < N) {
#pragma unroll
    for (int q = 0; q < Q; ++q) v[q] = T(0.f);
  }
  __device__ __forceinline__ void load(int t, int t1) {
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (on && t + q * KQ + k < t1) v[q] = base[(int64_t)(t + q * KQ) * st];
  }
  __device__ __forceinline__ void put(float *dst, int lane) const {
#pragma unroll
    for (int q = 0; q < Q; ++q) dst[lane + 64 * q] = to_f(v[q]);
  }
};

// lanes with BIT clear end with the sum (over lanes BIT apart) of a, the others with that of b: v_permlane32_swap / v_permlane16_swap
// exchange half of one register's lanes with half of another's; inside a quad the same takes two selects and a DPP add.
__device__ __forceinline__ float dpp_xor2(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4e, 0xf, 0xf, true)); }
__device__ __forceinline__ float dpp_xor1(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xb1, 0xf, 0xf, true)); }
template <int N>
__device__ __forceinline__ float dpp_ror(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, true)); }
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
    return keep + (BIT == 2 ? dpp_xor2(give) : dpp_xor1(give));
  }
}
// One value per step of a tile, in parts over the S lanes of a channel: lane part s ends with the sums of its own steps S q + s.
__device__ __forceinline__ void own_sums(const float v[TS], float out[OWN], int lane) {
#pragma unroll
  for (int q = 0; q < OWN; ++q) out[q] = fold<1>(fold<2>(v[4 * q], v[4 * q + 2], lane), fold<2>(v[4 * q + 1], v[4 * q + 3], lane), lane);
}

// ---------------------------------------------------------------------------------------------------------------- forward
// CARRY: a segment's state at its end from a zero start and the sum of its steps, for segments [0, nseg - 1); no outputs.
// The S lanes of a channel share the work of a step that does not depend on the state (loads, softplus, gate, store): part s takes the
// steps S q + s of a tile and hands delta and delta x to the others through LDS.
template <typename T, int NL, bool CARRY, bool PAD>
__global__ __launch_bounds__(WPB * 64) void k_scan_fwd(Args a) {
  constexpr int NP = NL * S, VW = NL < 4 ? NL : 4;         // VW: states read from LDS at once
  typedef float vec __attribute__((ext_vector_type(VW)));
  __shared__ __align__(16) float lds[WPB][CARRY ? 1 : 2][TS * NP];
  __shared__ __align__(8) float2 lds_d[WPB][TS][CW];
  const fdql_scan_t &p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int u = blockIdx.x * WPB + wave;
  if (u >= (a.nseg - CARRY) * p.R * p.G * a.tpg) return;
  const Unit w = unit_of(a, u);
  const int c = lane / S, s = lane % S;
  const int dc = w.tile * CW + c, d = w.g * a.Dg + min(dc, a.Dg - 1);
  const bool live = dc < a.Dg;
  const int t0 = w.seg * a.seglen, t1 = min(p.T, t0 + a.seglen);
  float *lB = lds[wave][0], *lC = lds[wave][CARRY ? 0 : 1];

  const Col<T> X = col_of<T>(p.x, p.x_st, p.x_sr, w.r, s, d), DT = col_of<T>(p.dt, p.dt_st, p.dt_sr, w.r, s, d),
               Z = col_of<T>(p.z ? p.z : p.x, p.z ? p.z_st : p.x_st, p.z ? p.z_sr : p.x_sr, w.r, s, d);
  const float bias = p.dt_bias ? p.dt_bias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
  float h[NL], A[NL], sum = 0.f;
  int any = 0;
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int n = s * NL + j;
    A[j] = n < p.N ? p.A[(int64_t)d * p.N + n] * LOG2E : 0.f;
    if (CARRY) h[j] = 0.f;
    else if (a.nseg > 1) h[j] = a.seg_h[lane_slot<NL>(a, w.seg, w) + j * 64 + lane];
    else h[j] = p.state_in && live && n < p.N ? p.state_in[(int64_t)w.r * p.state_in_sr + (int64_t)d * p.N + n] : 0.f;
  }
  const int64_t y_st = (int64_t)p.R * p.D;
  T *yp = reinterpret_cast<T *>(p.y) + (int64_t)w.r * p.D + s * y_st + d;

  // the next tile, in flight while this one is computed
  T xn[OWN] = {}, dn[OWN] = {}, zn[OWN] = {};
  Rows<T, NP> Bn(p.B, p.B_st, p.B_sr, p.B_sg, w, p.N, lane), Cn(p.C, p.C_st, p.C_sr, p.C_sg, w, p.N, lane);
  uint8_t rn = 0;
  const uint8_t *rp = p.reset ? p.reset + (int64_t)w.r * p.reset_sr + (lane % TS) * p.reset_st : nullptr;
  const auto fetch = [&](int t) {
#pragma unroll
    for (int q = 0; q < OWN; ++q) {
      if (t + q * S + s < t1) {
        xn[q] = X.at(t, q);
        dn[q] = DT.at(t, q);
        if (!CARRY) zn[q] = Z.at(t, q);
      }
    }
    Bn.load(t, t1);
    if (!CARRY) Cn.load(t, t1);
    if (rp && t + lane % TS < t1) rn = rp[t * p.reset_st];
  };
  fetch(t0);
  for (int t = t0; t < t1; t += TS) {
    const int nt = min(TS, t1 - t);
    const unsigned rst = (unsigned)__ballot(lane < nt && rn != 0);
    any |= rst != 0;
    Bn.put(lB, lane);
    if (!CARRY) Cn.put(lC, lane);
    float x[OWN], del[OWN], z[OWN];
#pragma unroll
    for (int q = 0; q < OWN; ++q) {
      x[q] = live ? to_f(xn[q]) : 0.f;
      del[q] = to_f(dn[q]) + bias;
      if (!CARRY) z[q] = to_f(zn[q]);
    }
    if (t + TS < t1) fetch(t + TS);
    if (!CARRY && p.checkpoints) {
      float *ck = p.checkpoints + lane_slot<NL>(a, t / TS, w) + lane;
#pragma unroll
      for (int j = 0; j < NL; ++j) ck[j * 64] = h[j];
    }
    bool plain = true;
#pragma unroll
    for (int q = 0; q < OWN; ++q) {
      if (p.dt_softplus) del[q] = softplus_f(del[q]);
      if (!live) del[q] = 0.f;
      lds_d[wave][q * S + s][c] = make_float2(del[q], del[q] * x[q]);
      plain = plain && finite(del[q]) && finite(del[q] * x[q]);
    }
    const bool wild = PAD && __any(!plain);
    wave_lds_fence();
    float acc[TS];
    const auto tile = [&](auto whole) {              // whole: eight steps without a reset (PAD: and finite)
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        if (i % 2 == 0) pass_edge();
        acc[i] = 0.f;
        if (decltype(whole)::value || i < nt) {
          const float2 v = lds_d[wave][i][c];
          const float dl = v.x, dx = v.y;
          const int left = PAD && !decltype(whole)::value ? states_left(p.N, s * NL) : NL;
          if (CARRY) sum += dl;
          const bool cut = !decltype(whole)::value && (rst >> i & 1);
#pragma unroll
          for (int j4 = 0; j4 < NL; j4 += VW) {
            const vec B = *reinterpret_cast<const vec *>(lB + i * NP + s * NL + j4);
            vec C = {};
            if (!CARRY) C = *reinterpret_cast<const vec *>(lC + i * NP + s * NL + j4);
#pragma unroll
            for (int j = 0; j < VW; ++j) {
              const float in = dx * B[j], on = fmaf(__builtin_amdgcn_exp2f(dl * A[j4 + j]), h[j4 + j], in);
              h[j4 + j] = cut ? in : on;        // (selected: a decay beyond float's range times zero would not be nothing)
              if (j4 + j >= left) h[j4 + j] = 0.f;
              if (!CARRY) acc[i] = fmaf(h[j4 + j], C[j], acc[i]);
            }
          }
          if (!CARRY) settle(acc[i]);
        }
      }
    };
    if (rst == 0 && nt == TS && !wild) tile(std::true_type());
    else tile(std::false_type());
    if (!CARRY) {
      float own[OWN];
      own_sums(acc, own, lane);
#pragma unroll
      for (int q = 0; q < OWN; ++q) {
        const int i = q * S + s;
        float y = p.skip ? fmaf(skip, x[q], own[q]) : own[q];
        if (p.z) y *= z[q] * sigmoid_f<T>(z[q]).s;
        if (live && i < nt) yp[(int64_t)(t + q * S) * y_st] = from_f<T>(y);
      }
    }
    wave_lds_fence();
  }
  if (CARRY) {
    const int64_t o = lane_slot<NL>(a, w.seg, w);
#pragma unroll
    for (int j = 0; j < NL; ++j) a.seg_h[o + j * 64 + lane] = live ? h[j] : 0.f;
    a.seg_d[o / NL + lane] = sum;
    if (lane == 0 && w.tile == 0 && w.g == 0) a.seg_f[(int64_t)w.seg * p.R + w.r] = any;
  } else if (p.state_out && t1 == p.T && live) {
#pragma unroll
    for (int j = 0; j < NL; ++j)
      if (s * NL + j < p.N) p.state_out[(int64_t)w.r * p.state_out_sr + (int64_t)d * p.N + s * NL + j] = h[j];
  }
}

// The backward pass's segments: the carry at a segment's start from a zero carry at its end, for segments [1, nseg).
template <typename T, int NL, bool PAD>
__global__ __launch_bounds__(WPB * 64) void k_scan_carry_back(Args a) {
  constexpr int NP = NL * S, VW = NL < 4 ? NL : 4;
  typedef float vec __attribute__((ext_vector_type(VW)));
  __shared__ __align__(16) float lds[WPB][TS * NP];
  __shared__ __align__(8) float2 lds_d[WPB][TS][CW];
  const fdql_scan_t &p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int u = blockIdx.x * WPB + wave;
  if (u >= (a.nseg - 1) * p.R * p.G * a.tpg) return;
  Unit w = unit_of(a, u);
  w.seg += 1;
  const int c = lane / S, s = lane % S;
  const int dc = w.tile * CW + c, d = w.g * a.Dg + min(dc, a.Dg - 1);
  const bool live = dc < a.Dg;
  const int t0 = w.seg * a.seglen, t1 = min(p.T, t0 + a.seglen);
  float *lC = lds[wave];
  const Col<T> DT = col_of<T>(p.dt, p.dt_st, p.dt_sr, w.r, s, d), DY = col_of<T>(p.dy, p.dy_st, p.dy_sr, w.r, s, d),
               Z = p.z ? col_of<T>(p.z, p.z_st, p.z_sr, w.r, s, d) : DY;
  const float bias = p.dt_bias ? p.dt_bias[d] : 0.f;
  float h[NL], A[NL], sum = 0.f;
  int any = 0;
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    h[j] = 0.f;
    A[j] = s * NL + j < p.N ? p.A[(int64_t)d * p.N + s * NL + j] * LOG2E : 0.f;
  }
  T yn[OWN] = {}, dn[OWN] = {}, zn[OWN] = {};
  Rows<T, NP> Cn(p.C, p.C_st, p.C_sr, p.C_sg, w, p.N, lane);
  uint8_t rn = 0;
  const uint8_t *rp = p.reset ? p.reset + (int64_t)w.r * p.reset_sr + (lane % TS) * p.reset_st : nullptr;
  const auto fetch = [&](int t) {
#pragma unroll
    for (int q = 0; q < OWN; ++q) {
      if (t + q * S + s < t1) {
        yn[q] = DY.at(t, q);
        dn[q] = DT.at(t, q);
        zn[q] = Z.at(t, q);
      }
    }
    Cn.load(t, t1);
    if (rp && t + lane % TS < t1) rn = rp[t * p.reset_st];
  };
  const int last = t0 + (t1 - t0 - 1) / TS * TS;
  fetch(last);
  for (int t = last; t >= t0; t -= TS) {
    const int nt = min(TS, t1 - t);
    const unsigned rst = (unsigned)__ballot(lane < nt && rn != 0);
    any |= rst != 0;
    Cn.put(lC, lane);
    float v[OWN], del[OWN];
    bool plain = true;
#pragma unroll
    for (int q = 0; q < OWN; ++q) {
      v[q] = to_f(yn[q]);
      if (p.z) {
        const float z = to_f(zn[q]);
        v[q] *= z * sigmoid_f<T>(z).s;
      }
      del[q] = to_f(dn[q]) + bias;
      if (p.dt_softplus) del[q] = softplus_f(del[q]);
      lds_d[wave][q * S + s][c] = make_float2(del[q], v[q]);
      plain = plain && finite(del[q]) && finite(v[q]);
    }
    const bool wild = PAD && __any(!plain);
    if (t > t0) fetch(t - TS);
    wave_lds_fence();
    const auto tile = [&](auto whole) {
#pragma unroll
      for (int i = TS - 1; i >= 0; --i) {
        if (decltype(whole)::value || i < nt) {
          const float2 q = lds_d[wave][i][c];
          const float dl = q.x, dy = q.y;
          const int left = PAD && !decltype(whole)::value ? states_left(p.N, s * NL) : NL;
          sum += dl;
          const bool cut = !decltype(whole)::value && (rst >> i & 1);
#pragma unroll
          for (int j4 = 0; j4 < NL; j4 += VW) {
            const vec C = *reinterpret_cast<const vec *>(lC + i * NP + s * NL + j4);
#pragma unroll
            for (int j = 0; j < VW; ++j) {
              const float g = __builtin_amdgcn_exp2f(dl * A[j4 + j]) * fmaf(dy, C[j], h[j4 + j]);
              h[j4 + j] = cut || j4 + j >= left ? 0.f : g;
            }
          }
        }
      }
    };
    if (rst == 0 && nt == TS && !wild) tile(std::true_type());
    else tile(std::false_type());
    wave_lds_fence();
  }
  const int64_t o = lane_slot<NL>(a, w.seg, w);
#pragma unroll
  for (int j = 0; j < NL; ++j) a.seg_h[o + j * 64 + lane] = live ? h[j] : 0.f;
  a.seg_d[o / NL + lane] = sum;
  if (lane == 0 && w.tile == 0 && w.g == 0) a.seg_f[(int64_t)w.seg * p.R + w.r] = any;
}

// A zero and an infinite state pass a segment as they are, whatever the product of its decays is, as they pass its steps one by one; others are
// multiplied by its root twice, since the product may leave float's range where what it makes of a state does not.
// seg_h becomes the state every segment starts from (REV = 0) / the carry that enters every segment from the right (REV = 1).
template <int NL, int REV>
__global__ __launch_bounds__(64) void k_scan_combine(Args a) {
  const fdql_scan_t &p = a.p;
  const int64_t per = (int64_t)p.R * p.G * a.tpg * NL * 64;
  const int64_t i = (int64_t)blockIdx.x * 64 + threadIdx.x;
  const int lane = (int)(i & 63), j = (int)(i / 64 % NL);
  const int64_t blk = i / (64 * NL);
  const int tile = (int)(blk % a.tpg), g = (int)(blk / a.tpg % p.G), r = (int)(blk / a.tpg / p.G);
  const int dc = tile * CW + lane / S, n = lane % S * NL + j;
  const bool live = dc < a.Dg && n < p.N;
  const int d = g * a.Dg + min(dc, a.Dg - 1);
  const float A = live ? p.A[(int64_t)d * p.N + n] * LOG2E : 0.f;
  float cur = 0.f;
  if (live) {
    if (REV) cur = p.dstate_out ? p.dstate_out[((int64_t)r * p.D + d) * p.N + n] : 0.f;
    else cur = p.state_in ? p.state_in[(int64_t)r * p.state_in_sr + (int64_t)d * p.N + n] : 0.f;
  }
  // AHEAD segments' values are read together, the next ones before these are joined: one by one, each read behind the last one's store, 64
  // segments took 24 us
  constexpr int AHEAD = 16;
  const auto seg_of = [&](int k) { return REV ? a.nseg - 1 - k : k; };
  float own[AHEAD], sum[AHEAD];
  int any[AHEAD];
  const auto fetch = [&](int k0) {
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      const int64_t seg = seg_of(min(k0 + q, a.nseg - 2));
      own[q] = a.seg_h[seg * per + i];
      sum[q] = a.seg_d[(seg * p.R * p.G * a.tpg + blk) * 64 + lane];
      any[q] = a.seg_f[seg * p.R + r];
    }
  };
  fetch(0);
  for (int k0 = 0; k0 < a.nseg - 1; k0 += AHEAD) {
    float to[AHEAD], e[AHEAD];
    bool cut[AHEAD];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      to[q] = own[q];
      e[q] = __builtin_amdgcn_exp2f(0.5f * sum[q] * A);
      cut[q] = any[q] != 0;
    }
    if (k0 + AHEAD < a.nseg - 1) fetch(k0 + AHEAD);
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      if (k0 + q < a.nseg - 1) {
        a.seg_h[seg_of(k0 + q) * per + i] = cur;
        const float in = cur == 0.f || !finite(cur) ? cur : cur * e[q] * e[q];
        cur = cut[q] ? to[q] : in + to[q];
      }
    }
  }
  a.seg_h[seg_of(a.nseg - 1) * per + i] = cur;
}

// --------------------------------------------------------------------------------------------------------------- backward
template <typename T, int NL, bool PAD>
__global__ __launch_bounds__(WPB * 64, 2) void k_scan_bwd(Args a) {
  constexpr int NP = NL * S;
  __shared__ __align__(16) float lB[2][TS * NP], lC[2][TS * NP];
  __shared__ __align__(16) v4f lds_d[WPB][TS][CW];     // delta, delta x, gated dy of every step
  __shared__ __align__(8) float red[2][WPB][TS * 2 * NP];                       // [step][dB, dC][state]
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
  const int c = lane / S, s = lane % S;
  const int dc = w.tile * CW + c, d = w.g * a.Dg + min(dc, a.Dg - 1);
  const bool live = !idle && dc < a.Dg;
  const int t0 = w.seg * a.seglen, t1 = min(p.T, t0 + a.seglen);

  const Col<T> X = col_of<T>(p.x, p.x_st, p.x_sr, w.r, s, d), DT = col_of<T>(p.dt, p.dt_st, p.dt_sr, w.r, s, d),
               DY = col_of<T>(p.dy, p.dy_st, p.dy_sr, w.r, s, d), Z = p.z ? col_of<T>(p.z, p.z_st, p.z_sr, w.r, s, d) : X;
  const float bias = p.dt_bias ? p.dt_bias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
  float A[NL], carry[NL], dA[NL], dskip = 0.f, dbias = 0.f;
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int n = s * NL + j;
    A[j] = n < p.N ? p.A[(int64_t)d * p.N + n] * LOG2E : 0.f;
    dA[j] = 0.f;
    if (a.nseg > 1) carry[j] = a.seg_h[lane_slot<NL>(a, w.seg, w) + j * 64 + lane];
    else carry[j] = live && p.dstate_out && n < p.N ? p.dstate_out[((int64_t)w.r * p.D + d) * p.N + n] : 0.f;
  }
  const int64_t o_st = (int64_t)p.R * p.D, o0 = (int64_t)w.r * p.D + s * o_st + d;
  const int last = t0 + (t1 - t0 - 1) / TS * TS;
  const int64_t slab_st = (int64_t)p.R * p.G * p.N, slab_0 = (int64_t)wgt * p.T * slab_st + ((int64_t)w.r * p.G + w.g) * p.N;
  float *slab_b = a.slab_b + slab_0, *slab_c = a.slab_c + slab_0;

  // the tile in front of this one, in flight while this one is computed
  T xn[OWN] = {}, dn[OWN] = {}, yn[OWN] = {}, zn[OWN] = {};
  Rows<T, NP> Bn(p.B, p.B_st, p.B_sr, p.B_sg, w, p.N, lane), Cn(p.C, p.C_st, p.C_sr, p.C_sg, w, p.N, lane);   // (staged by wave 0 and, where there is one, wave 1)
  uint8_t rn = 0;
  const uint8_t *rp = p.reset ? p.reset + (int64_t)w.r * p.reset_sr + (lane % TS) * p.reset_st : nullptr;
  const int cw = blockDim.x > 64 ? 1 : 0;
  const auto fetch = [&](int t) {
#pragma unroll
    for (int q = 0; q < OWN; ++q) {
      if (t + q * S + s < t1) {
        xn[q] = X.at(t, q);
        dn[q] = DT.at(t, q);
        yn[q] = DY.at(t, q);
        zn[q] = Z.at(t, q);
      }
    }
    if (wave == 0) Bn.load(t, t1);
    if (wave == cw) Cn.load(t, t1);
    if (rp && t + lane % TS < t1) rn = rp[t * p.reset_st];
  };
  const auto put = [&](int buf) {
    if (wave == 0) Bn.put(lB[buf], lane);
    if (wave == cw) Cn.put(lC[buf], lane);
  };
  fetch(last);
  put(0);
  __syncthreads();
  int buf = 0;
  for (int t = last; t >= t0; t -= TS, buf ^= 1) {
    const int nt = min(TS, t1 - t);
    const unsigned rst = (unsigned)__ballot(lane < nt && rn != 0);
    // this lane's own steps: delta, delta x, gated dy; slope of the softplus, what dz is of the ungated output
    float x[OWN], del[OWN], dx[OWN], dy[OWN], slope[OWN], zf[OWN];
    bool plain = true;
#pragma unroll
    for (int q = 0; q < OWN; ++q) {
      x[q] = live ? to_f(xn[q]) : 0.f;
      dy[q] = to_f(yn[q]);
      if (p.z) {
        const float z = to_f(zn[q]);
        const Sigmoid g = sigmoid_f<T>(z);
        zf[q] = dy[q] * g.s * fmaf(z, g.c, 1.f);
        dy[q] *= z * g.s;
      }
      del[q] = to_f(dn[q]) + bias;
      slope[q] = 1.f;
      if (p.dt_softplus) del[q] = softplus_f(del[q], slope[q]);
      if (!live) del[q] = dy[q] = 0.f;             // (dy: behind its gate)
      dx[q] = del[q] * x[q];
      lds_d[wave][q * S + s][c] = v4f{del[q], dx[q], dy[q], 0.f};
      plain = plain && finite(del[q]) && finite(dx[q]) && finite(dy[q]);
    }
    const bool wild = PAD && __any(!plain);
    wave_lds_fence();
    if (t > t0) fetch(t - TS);
    const float *ck = p.checkpoints + lane_slot<NL>(a, t / TS, w) + lane;
    const float *tB = lB[buf] + s * NL, *tC = lC[buf] + s * NL;
    float *red_w = red[buf][wave];
    float yc[TS], dd[TS], gx[TS];
#pragma unroll
    for (int i = 0; i < TS; ++i) yc[i] = dd[i] = gx[i] = 0.f;
    const auto tile = [&](auto whole) {
      constexpr bool W = decltype(whole)::value;   // eight steps without a reset (PAD: and finite)
      float h0 = ck[0], h1 = ck[64];
#pragma unroll
      for (int m = 0; m < NL; m += 2) {
        float h[TS + 1][2], e[TS][2];
        pass_edge();
        h[0][0] = h0, h[0][1] = h1;
        if (m + 2 < NL) h0 = ck[(m + 2) * 64], h1 = ck[(m + 3) * 64];
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          if (W || i < nt) {
            const v4f st = lds_d[wave][i][c];
            const float dl = st[0], dxi = st[1];
            const float2 B = *reinterpret_cast<const float2 *>(tB + i * NP + m), C = *reinterpret_cast<const float2 *>(tC + i * NP + m);
            const bool cut = !W && (rst >> i & 1);
            const int left = PAD && !W ? states_left(p.N, s * NL) : NL;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              e[i][j] = __builtin_amdgcn_exp2f(dl * A[m + j]);
              const float in = dxi * (j ? B.y : B.x);
              h[i + 1][j] = cut ? in : fmaf(e[i][j], h[i][j], in);
              if (m + j >= left) e[i][j] = h[i + 1][j] = 0.f;
              yc[i] = fmaf(h[i + 1][j], j ? C.y : C.x, yc[i]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) e[i][j] = 0.f, h[i + 1][j] = 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < TS; ++i) settle(yc[i]);
        pass_edge();
#pragma unroll
        for (int i = TS - 1; i >= 0; --i) {
          if (W || i < nt) {
            const v4f st = lds_d[wave][i][c];
            const float dl = st[0], dxi = st[1], dyi = st[2];
            const float2 B = *reinterpret_cast<const float2 *>(tB + i * NP + m), C = *reinterpret_cast<const float2 *>(tC + i * NP + m);
            const bool cut = !W && (rst >> i & 1);
            const int left = PAD && !W ? states_left(p.N, s * NL) : NL;
            float v[4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float g = fmaf(dyi, j ? C.y : C.x, carry[m + j]);
              if (m + j >= left) g = 0.f;
              float ga = g * e[i][j], q = ga * h[i][j];
              if (cut) ga = q = 0.f;
              dd[i] = fmaf(q, A[m + j], dd[i]);        // (A log2 e: undone at the end)
              dA[m + j] = fmaf(q, dl, dA[m + j]);
              gx[i] = fmaf(g, j ? B.y : B.x, gx[i]);
              v[j] = g * dxi;
              v[2 + j] = h[i + 1][j] * dyi;
              carry[m + j] = ga;
            }
            settle(dd[i]);
            settle(gx[i]);
            settle(dA[m]);
            settle(dA[m + 1]);
            settle(carry[m]);
            settle(carry[m + 1]);
            // over the 16 channels: lane bits 5 and 4 end with dB or dC and the state of the two, bits 3 and 2 are summed as they are
            float o = fold<16>(fold<32>(v[0], v[2], lane), fold<32>(v[1], v[3], lane), lane);
            o += dpp_ror<8>(o);
            o += dpp_ror<4>(o);
            if ((lane & 12) == 0) red_w[(i * 2 + (lane >> 5)) * NP + s * NL + m + (lane >> 4 & 1)] = o;
          }
        }
      }
    };
    if (rst == 0 && nt == TS && !wild) tile(std::true_type());
    else tile(std::false_type());
    if (t > t0) put(buf ^ 1);
    __syncthreads();                             // red of this tile and the rows of the next one are there
    {
      float yo[OWN], d_o[OWN], go[OWN];
      own_sums(yc, yo, lane);
      own_sums(dd, d_o, lane);
      own_sums(gx, go, lane);
#pragma unroll
      for (int q = 0; q < OWN; ++q) {
        const int i = q * S + s;
        if (i < nt && live) {
          const float ddt = fmaf(x[q], go[q], d_o[q] * LN2) * slope[q];
          dskip = fmaf(dy[q], x[q], dskip);
          dbias += ddt;
          const int64_t o = o0 + (int64_t)(t + q * S) * o_st;
          reinterpret_cast<T *>(p.dx)[o] = from_f<T>(p.skip ? fmaf(skip, dy[q], del[q] * go[q]) : del[q] * go[q]);
          reinterpret_cast<T *>(p.ddt)[o] = from_f<T>(ddt);
          if (p.z && p.dz) reinterpret_cast<T *>(p.dz)[o] = from_f<T>(zf[q] * (p.skip ? fmaf(skip, x[q], yo[q]) : yo[q]));
        }
      }
    }
    for (int i = threadIdx.x; i < nt * 2 * NP; i += nthreads) {
      const int n = i % NP, which = i / NP % 2, k2 = i / (2 * NP);
      if (n < p.N) {
        const float *r = red[buf][0] + i;
        float v = r[0];
        for (int q = 1; q < active; ++q) v += r[q * TS * 2 * NP];
        (which ? slab_c : slab_b)[(int64_t)(t + k2) * slab_st + n] = v;
      }
    }
  }
  if (idle) return;
  if (w.seg == 0 && p.dstate_in && live) {
#pragma unroll
    for (int j = 0; j < NL; ++j)
      if (s * NL + j < p.N) p.dstate_in[((int64_t)w.r * p.D + d) * p.N + s * NL + j] = carry[j];
  }
  const int64_t o = lane_slot<NL>(a, w.seg, w);
#pragma unroll
  for (int j = 0; j < NL; ++j) a.part_a[o + j * 64 + lane] = dA[j];
  // the parts' own steps added up (each saw TS / S of a tile's)
  dskip += dpp_xor1(dskip);
  dbias += dpp_xor1(dbias);
  dskip += dpp_xor2(dskip);
  dbias += dpp_xor2(dbias);
  a.part_s[o / NL * 2 + lane] = dskip;
  a.part_s[o / NL * 2 + 64 + lane] = dbias;
}

// Joins the workgroups' parts.  blockIdx.x < nbc: dB / dC, the slabs added in order, rounded once to the tensor's type.  Behind them: dA, dskip, ddt_bias,
// partials of the (segment, row) pairs added up, a workgroup per 64 lanes of one state, 16 slices of the pairs.  (One launch: as two, one behind the
// other, 5 + 7.5 us at 50 x 256 x 512.)
template <typename T, int NL>
__global__ __launch_bounds__(1024) void k_scan_finish(Args a, int nbc) {
  __shared__ float red[16][64];
  const fdql_scan_t &p = a.p;
  if ((int)blockIdx.x < nbc) {
    const int64_t n = (int64_t)p.T * p.R * p.G * p.N;
    for (int64_t k = (int64_t)blockIdx.x * 1024 + threadIdx.x; k < 2 * n; k += (int64_t)nbc * 1024) {
      const int64_t i = k < n ? k : k - n;
      const float *slab = k < n ? a.slab_b : a.slab_c;
      float v = 0.f;
#pragma unroll 8
      for (int q = 0; q < a.wgt; ++q) v += slab[q * n + i];
      reinterpret_cast<T *>(k < n ? p.dB : p.dC)[i] = from_f<T>(v);
    }
    return;
  }
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6, u = blockIdx.x - nbc;
  const int j = u % (NL + 2), blk = u / (NL + 2);
  const int64_t pairs = (int64_t)a.nseg * p.R, blocks = (int64_t)p.G * a.tpg;
  float v = 0.f;
#pragma unroll 8
  for (int64_t k = slice; k < pairs; k += 16)
    v += j < NL ? a.part_a[((k * blocks + blk) * NL + j) * 64 + lane] : a.part_s[((k * blocks + blk) * 2 + j - NL) * 64 + lane];
  red[slice][lane] = v;
  __syncthreads();
  if (slice) return;
  v = 0.f;
#pragma unroll
  for (int q = 0; q < 16; ++q) v += red[q][lane];
  const int g = blk / a.tpg, dc = blk % a.tpg * CW + lane / S, n = lane % S * NL + j;
  if (dc >= a.Dg) return;
  const int64_t d = (int64_t)g * a.Dg + dc;
  if (j < NL) {
    if (n < p.N && p.dA) p.dA[d * p.N + n] = v;
  } else if (lane % S == 0) {
    float *out = j == NL ? p.dskip : p.ddt_bias;
    if (out) out[d] = v;
  }
}

// ------------------------------------------------------------------------------------------------------------ single steps
// One step for every row: the state is read and written once, V = 4 states (16 bytes) per lane where the state's rows allow it.  A wave
// owns 64 channels of one row: lane = channel for delta, x and the gate; then LPC lanes share a channel and the wave passes over
// its state in LPC turns, consecutive lanes on consecutive addresses.  Memory bounds it: bf16 512 x 2048 x 64 117 us = 4.7 TB/s.
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
      if (p.state_out) *reinterpret_cast<vec *>(p.state_out + (int64_t)r * p.state_out_sr + dd * p.N + n) = h;
    }
    for (int m = 1; m < lpc; m <<= 1) acc += __shfl_xor(acc, m);
    const float back = __shfl(acc, (lane % cpt) * lpc);            // the sum of channel it * cpt + (lane % cpt)
    if (lane / cpt == it) y = back;
  }
  if (p.skip) y = fmaf(p.skip[d], x, y);
  if (p.z) {
    const float z = to_f(reinterpret_cast<const T *>(p.z)[(int64_t)r * p.z_sr + d]);
    y *= z * sigmoid_f<T>(z).s;
  }
  if (dc < Dg) reinterpret_cast<T *>(p.y)[(int64_t)r * p.D + d] = from_f<T>(y);
}

// The same for few rows, whose turns one after the other would be most of the time: a wave owns the 64 / LPC channels of one turn, and the LPC lanes
// of a channel each work out its delta.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_scan_step_few(fdql_scan_t p, int Dg, int tpg, int lpc) {
  typedef float vec __attribute__((ext_vector_type(V)));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned u = blockIdx.x * 4 + wave;
  if (u >= (int64_t)p.R * p.G * tpg) return;
  const int tile = (int)(u % tpg), g = (int)(u / tpg % p.G), r = (int)(u / tpg / p.G);
  const int sub = lane % lpc, n = sub * V, c = tile * (64 / lpc) + lane / lpc, d = g * Dg + min(c, Dg - 1);
  const bool fresh = !p.state_in || (p.reset && p.reset[(int64_t)r * p.reset_sr] != 0), part = n < p.N, live = c < Dg;
  const int64_t at = (int64_t)d * p.N + (part ? n : 0);
  const vec A = *reinterpret_cast<const vec *>(p.A + at);
  vec h = {};
  if (!fresh) h = *reinterpret_cast<const vec *>(p.state_in + (int64_t)r * p.state_in_sr + at);
  const float x = to_f(reinterpret_cast<const T *>(p.x)[(int64_t)r * p.x_sr + d]);
  float del = to_f(reinterpret_cast<const T *>(p.dt)[(int64_t)r * p.dt_sr + d]) + (p.dt_bias ? p.dt_bias[d] : 0.f);
  const float z = p.z ? to_f(reinterpret_cast<const T *>(p.z)[(int64_t)r * p.z_sr + d]) : 0.f, skip = p.skip ? p.skip[d] : 0.f;
  const T *Bp = reinterpret_cast<const T *>(p.B) + (int64_t)r * p.B_sr + (int64_t)g * p.B_sg;
  const T *Cp = reinterpret_cast<const T *>(p.C) + (int64_t)r * p.C_sr + (int64_t)g * p.C_sg;
  if (p.dt_softplus) del = softplus_f(del);
  const float dx = del * x;
  float acc = 0.f;
  if (part) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float in = dx * to_f(Bp[n + k]);
      h[k] = fresh ? in : fmaf(__builtin_amdgcn_exp2f(del * (A[k] * LOG2E)), h[k], in);
      acc = fmaf(h[k], to_f(Cp[n + k]), acc);
    }
    if (p.state_out && live) *reinterpret_cast<vec *>(p.state_out + (int64_t)r * p.state_out_sr + at) = h;
  }
  for (int m = 1; m < lpc; m <<= 1) acc += __shfl_xor(acc, m);
  float y = p.skip ? fmaf(skip, x, acc) : acc;
  if (p.z) y *= z * sigmoid_f<T>(z).s;
  if (sub == 0 && live) reinterpret_cast<T *>(p.y)[(int64_t)r * p.D + d] = from_f<T>(y);
}

// ------------------------------------------------------------------------------------------------------------------- host
struct Plan {
  int NL, tpg, Dg, nseg, seglen, wgt, wpw;
};

constexpr int CUS = 256;

Plan plan_of(const fdql_scan_t &p) {
  Plan q;
  q.Dg = p.D / p.G;
  const int64_t rows = (int64_t)p.R * p.G;
  q.NL = p.N <= 8 ? 2 : p.N <= 16 ? 4 : p.N <= 32 ? 8 : 16;
  q.tpg = (q.Dg + CW - 1) / CW;
  const int64_t waves = rows * q.tpg;
  q.nseg = 1;
  q.seglen = p.T;
  // Segments: fewer than two waves per SIMD and at least three segments of 32 steps, since each is walked twice; eight waves per SIMD where the
  // length allows.  Training passes, N 16, float, cut or in one piece: 256 x 4 x 128 56 us or 181, 512 x 40 x 512 (1280 waves) 335 or 425; the
  // other way 256 x 64 x 512 (2048 waves) 270 or 237, 64 x 24 x 512 in two segments 69 or 62.  bf16 16383 x 1 x 1024: 542 us with eight waves per
  // SIMD, 575 with four, 11304 in one piece.
  if (waves > 0 && waves < 2048 && p.T >= 96) {
    const int64_t want = std::min<int64_t>((8192 + waves - 1) / waves, p.T / 32);
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

template <typename F>
hipError_t with_states(int NL, int N, F f) {
  const auto pad = [&](auto nl) { return N < nl * S ? f(nl, std::true_type()) : f(nl, std::false_type()); };
  switch (NL) {
    case 2: return pad(std::integral_constant<int, 2>());
    case 4: return pad(std::integral_constant<int, 4>());
    case 8: return pad(std::integral_constant<int, 8>());
    default: return pad(std::integral_constant<int, 16>());
  }
}

template <typename T>
hipError_t fwd(const fdql_scan_t &p, hipStream_t s) {
  const Plan q = plan_of(p);
  return with_states(q.NL, p.N, [&](auto v, auto padded) {
    constexpr int NL = decltype(v)::value;
    constexpr bool PAD = decltype(padded)::value;
    const Args a = args_of(p, q, false);
    const int64_t per = (int64_t)p.R * p.G * q.tpg;
    if (q.nseg > 1) {
      hipLaunchKernelGGL((k_scan_fwd<T, NL, true, PAD>), dim3((unsigned)(((q.nseg - 1) * per + WPB - 1) / WPB)), dim3(WPB * 64), 0, s, a);
      hipLaunchKernelGGL((k_scan_combine<NL, 0>), dim3((unsigned)(per * NL)), dim3(64), 0, s, a);
    }
    hipLaunchKernelGGL((k_scan_fwd<T, NL, false, PAD>), dim3((unsigned)((q.nseg * per + WPB - 1) / WPB)), dim3(WPB * 64), 0, s, a);
    return hipGetLastError();
  });
}

template <typename T>
hipError_t bwd(const fdql_scan_t &p, hipStream_t s) {
  const Plan q = plan_of(p);
  return with_states(q.NL, p.N, [&](auto v, auto padded) {
    constexpr int NL = decltype(v)::value;
    constexpr bool PAD = decltype(padded)::value;
    const Args a = args_of(p, q, true);
    const int64_t per = (int64_t)p.R * p.G * q.tpg;
    if (q.nseg > 1) {
      hipLaunchKernelGGL((k_scan_carry_back<T, NL, PAD>), dim3((unsigned)(((q.nseg - 1) * per + WPB - 1) / WPB)), dim3(WPB * 64), 0, s, a);
      hipLaunchKernelGGL((k_scan_combine<NL, 1>), dim3((unsigned)(per * NL)), dim3(64), 0, s, a);
    }
    hipLaunchKernelGGL((k_scan_bwd<T, NL, PAD>), dim3((unsigned)((int64_t)q.nseg * p.R * p.G * q.wgt)), dim3(q.wpw * 64), 0, s, a);
    const int64_t bc = 2ll * p.T * p.R * p.G * p.N;
    const int nbc = (int)std::min<int64_t>((bc + 1023) / 1024, 4 * CUS);
    hipLaunchKernelGGL((k_scan_finish<T, NL>), dim3((unsigned)(nbc + p.G * q.tpg * (NL + 2))), dim3(1024), 0, s, a, nbc);
    return hipGetLastError();
  });
}

template <typename T>
hipError_t step(const fdql_scan_t &p, hipStream_t s) {
  const int Dg = p.D / p.G, tpg = (Dg + 63) / 64;
  const auto al = [](const void *q) { return ((uintptr_t)q & 15) == 0; };
  const bool vec = p.N % 4 == 0 && al(p.A) && al(p.state_in) && al(p.state_out) && (!p.state_in || p.state_in_sr % 4 == 0) && (!p.state_out || p.state_out_sr % 4 == 0);
  int lpc = 1;
  while (lpc * (vec ? 4 : 1) < p.N) lpc <<= 1;
  // Below 2048 waves of 64 channels: one turn per wave, float 32 x 512 x 16 3.4 us against 4.9, 32 x 512 x 64 5.6 against 12.0; where there are more,
  // the turns share the work on delta and keep more bytes under way: bf16 512 x 2048 x 64 117 us against 188.
  if ((int64_t)p.R * p.G * tpg < 2048) {
    const int cpt = 64 / lpc, tiles = (Dg + cpt - 1) / cpt;
    const dim3 few((unsigned)(((int64_t)p.R * p.G * tiles + 3) / 4));
    if (vec) hipLaunchKernelGGL((k_scan_step_few<T, 4>), few, dim3(256), 0, s, p, Dg, tiles, lpc);
    else hipLaunchKernelGGL((k_scan_step_few<T, 1>), few, dim3(256), 0, s, p, Dg, tiles, lpc);
    return hipGetLastError();
  }
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
