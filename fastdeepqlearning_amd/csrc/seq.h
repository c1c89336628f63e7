// Sequence operators over time-major tensors [T, rows, channels]: argument checks and entry points in seq.hip, kernels in
// seqconv.hip (causal convolution), scan.hip (selective state-space scan) and gated.hip (gated linear unit).
#pragma once
#include "common.h"

namespace fdql {

hipError_t seqconv_fwd_launch(const fdql_causal_conv_t &p, hipStream_t s);
hipError_t seqconv_bwd_launch(const fdql_causal_conv_t &p, hipStream_t s);
int64_t seqconv_workspace_bytes(const fdql_causal_conv_t &p);

int64_t scan_checkpoint_floats(const fdql_scan_t &p);
int64_t scan_workspace_bytes(const fdql_scan_t &p, bool backward);
hipError_t scan_fwd_launch(const fdql_scan_t &p, hipStream_t s);
hipError_t scan_bwd_launch(const fdql_scan_t &p, hipStream_t s);

int64_t gated_workspace_bytes(const fdql_gated_t &p, bool backward);
hipError_t gated_fwd_launch(const fdql_gated_t &p, hipStream_t s);
hipError_t gated_bwd_launch(const fdql_gated_t &p, hipStream_t s);

// Pieces of the agent's state-space joiner (agent_plan.hip); T = 0: A alone
hipError_t ssm_prep_launch(const float *task_done, const float *episode_step, int T, int B, uint8_t *reset, const float *A_log, float *A, int n, hipStream_t s);
hipError_t ssm_dalog_launch(const float *dA, const float *A, int n, float *out, hipStream_t s);

#if defined(__HIPCC__)
// Element types: float, bf16 and fp16 in memory, float in registers; conversions round to nearest even.
typedef __bf16 bf16_t;
typedef _Float16 f16_t;
template <typename T> __device__ __forceinline__ float to_f(T v) { return static_cast<float>(v); }
template <typename T> __device__ __forceinline__ T from_f(float v) { return static_cast<T>(v); }

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// e^v to float precision also for large |v|: the product v log2(e) is kept in two floats (one float alone loses |v| ulps).
__device__ __forceinline__ float exp_acc(float v) {
  const float hi = v * LOG2E;
  const float lo = fmaf(v, LOG2E, -hi) + v * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(hi);
  return fabsf(hi) < 126.f ? fmaf(e, lo * LN2, e) : e;   // (infinite or vanishing: nothing to correct)
}
// s = 1 / (1 + e^-v) and c = 1 - s = 1 / (1 + e^v), each from the power w = e^-|v| that keeps its own digits where it is small (s of a negative v is
// w / (1 + w): as 1 / (1 + e^|v|) it would carry the power's error whole, c as 1 - s would have none of its digits left from v = 17 on).
// One product for the exponent is off by up to |v| float steps, 2^-17.5 of the result at most: enough for a result of 16 bits (half a step is 2^-12
// or 2^-9), not for a float one.
struct Sigmoid { float s, c; };
template <typename T>
__device__ __forceinline__ Sigmoid sigmoid_f(float v) {
  const float w = sizeof(T) == 4 ? exp_acc(-fabsf(v)) : __builtin_amdgcn_exp2f(-LOG2E * fabsf(v)), r = __builtin_amdgcn_rcpf(1.f + w), q = w * r;
  return v >= 0.f ? Sigmoid{r, q} : Sigmoid{q, r};
}
// log(1 + e^v) = max(v, 0) + log1p(w), w = e^-|v| in (0, 1]: log1p(w) = 2 atanh(w / (2 + w)), the odd series to the eighth term
// (argument at most 1/3: the first term left out is below 2e-9 of the sum).  Keeps its relative precision for small steps.
__device__ __forceinline__ float softplus_w(float v, float w) {
  const float q = w * __builtin_amdgcn_rcpf(2.f + w), q2 = q * q;
  float s = fmaf(q2, 1.f / 15.f, 1.f / 13.f);
  s = fmaf(q2, s, 1.f / 11.f);
  s = fmaf(q2, s, 1.f / 9.f);
  s = fmaf(q2, s, 1.f / 7.f);
  s = fmaf(q2, s, 1.f / 5.f);
  s = fmaf(q2, s, 1.f / 3.f);
  s = fmaf(q2, s, 1.f);
  return fmaxf(v, 0.f) + 2.f * q * s;
}
__device__ __forceinline__ float softplus_f(float v) { return softplus_w(v, exp_acc(-fabsf(v))); }
// ... and its slope 1 / (1 + e^-v) from the same power
__device__ __forceinline__ float softplus_f(float v, float &slope) {
  const float w = exp_acc(-fabsf(v)), r = __builtin_amdgcn_rcpf(1.f + w);
  slope = v >= 0.f ? r : w * r;
  return softplus_w(v, w);
}
#endif
}  // namespace fdql
