// Entry points of the sequence operators: argument checks, empty shapes, launches.
#include "seq.h"

using namespace fdql;

namespace {

constexpr int64_t MAX_THREADS = 0xffffffffll;      // threads of a launch

__global__ __launch_bounds__(256) void k_seq_zero(float *p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0.f;
}
__global__ __launch_bounds__(256) void k_seq_zero16(uint16_t *p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}
// dst [R, per] (row stride dr) = src (row stride sr) or zeros
__global__ __launch_bounds__(256) void k_seq_copy_rows(const float *src, int64_t sr, float *dst, int64_t dr, int64_t R, int64_t per) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < R * per; i += (int64_t)gridDim.x * 256) dst[i / per * dr + i % per] = src ? src[i / per * sr + i % per] : 0.f;
}
dim3 grid_for(int64_t n) { return dim3((unsigned)(n < 256 * 1024 ? (n + 255) / 256 : 1024)); }

int zero(void *p, int64_t n, int32_t dtype, hipStream_t s) {   // a kernel, not a memset: the call may be captured
  if (!p || n <= 0) return FDQL_OK;
  if (dtype == FDQL_F32) hipLaunchKernelGGL(k_seq_zero, grid_for(n), dim3(256), 0, s, (float *)p, n);
  else hipLaunchKernelGGL(k_seq_zero16, grid_for(n), dim3(256), 0, s, (uint16_t *)p, n);
  FDQL_HIP(hipGetLastError());
  return FDQL_OK;
}
int copy_rows(const float *src, int64_t sr, float *dst, int64_t dr, int64_t R, int64_t per, hipStream_t s) {
  if (!dst || R * per == 0) return FDQL_OK;
  hipLaunchKernelGGL(k_seq_copy_rows, grid_for(R * per), dim3(256), 0, s, src, sr, dst, dr, R, per);
  FDQL_HIP(hipGetLastError());
  return FDQL_OK;
}

bool type_ok(int32_t t) { return t == FDQL_F32 || t == FDQL_BF16 || t == FDQL_F16; }

int check_conv(const fdql_causal_conv_t *p) {
  FDQL_REQUIRE(p && p->size == (int32_t)sizeof(*p), "causal_conv: struct size %d, this library has %d", p ? p->size : 0, (int)sizeof(*p));
  FDQL_REQUIRE(type_ok(p->dtype), "causal_conv: dtype %d (float32, bf16 or fp16)", p->dtype);
  FDQL_REQUIRE(p->T >= 0 && p->R >= 0 && p->D >= 1, "causal_conv: T %d, R %d, D %d", p->T, p->R, p->D);
  FDQL_REQUIRE(p->K >= 2 && p->K <= 4, "causal_conv: %d taps (2 to 4)", p->K);
  FDQL_REQUIRE(((int64_t)p->D + 63) / 64 * p->R * ((p->T + 7ll) / 8 + 1) * 64 < MAX_THREADS, "causal_conv: T %d x R %d x D %d is more than one launch", p->T, p->R, p->D);
  return FDQL_OK;
}
int check_scan(const fdql_scan_t *p) {
  FDQL_REQUIRE(p && p->size == (int32_t)sizeof(*p), "scan: struct size %d, this library has %d", p ? p->size : 0, (int)sizeof(*p));
  FDQL_REQUIRE(type_ok(p->dtype), "scan: dtype %d (float32, bf16 or fp16)", p->dtype);
  FDQL_REQUIRE(p->T >= 0 && p->T <= 1 << 30 && p->R >= 0 && p->D >= 1, "scan: T %d (up to 2^30), R %d, D %d", p->T, p->R, p->D);
  FDQL_REQUIRE(p->N >= 1 && p->N <= 64, "scan: %d states (1 to 64)", p->N);
  FDQL_REQUIRE(p->G >= 1 && p->D % p->G == 0, "scan: %d groups do not divide %d channels", p->G, p->D);
  // waves of 16 channels (a time axis cut into segments: 10240 of them at most), 16 of the joining kernel's each; 18 finish workgroups of 1024 threads
  const int64_t tiles = (int64_t)p->G * ((p->D / p->G + 15) / 16);
  FDQL_REQUIRE((p->R * tiles + 10240) * 64 * 16 < MAX_THREADS && (tiles * 18 + 1024) * 1024 < MAX_THREADS, "scan: R %d x D %d is more than one launch", p->R, p->D);
  return FDQL_OK;
}
int check_gated(const fdql_gated_t *p) {
  FDQL_REQUIRE(p && p->size == (int32_t)sizeof(*p), "gated: struct size %d, this library has %d", p ? p->size : 0, (int)sizeof(*p));
  FDQL_REQUIRE(type_ok(p->dtype), "gated: dtype %d (float32, bf16 or fp16)", p->dtype);
  FDQL_REQUIRE(p->M >= 0 && p->D >= 1 && p->F >= 1 && p->D <= 1 << 24 && p->F <= 1 << 24, "gated: M %lld, D %d, F %d (D and F up to 2^24)", (long long)p->M, p->D, p->F);
  const int32_t act = p->act & ~FDQL_GATED_ROUND_GRADS;
  FDQL_REQUIRE(act >= FDQL_ACT_SILU && act <= FDQL_ACT_SIGMOID, "gated: activation %d", p->act);
  FDQL_REQUIRE(p->M <= 128ll * 65535 && (p->M / 64 + 1) * ((int64_t)(p->F > p->D ? p->F : p->D) / 64 + 1) * 256 < MAX_THREADS,
               "gated: M %lld x (D %d, F %d) is more than one launch", (long long)p->M, p->D, p->F);
  FDQL_REQUIRE(((int64_t)p->F / 128 + 1) * (p->D / 128 + 1) * 256 * 2 < MAX_THREADS / 16, "gated: weights %d x %d are more than one launch", p->F, p->D);
  return FDQL_OK;
}
int check_workspace(const char *what, const void *ws, int64_t have, int64_t need) {
  FDQL_REQUIRE(need <= 0 || (ws && have >= need && ((uintptr_t)ws & 15) == 0), "%s: workspace of %lld bytes (16-byte aligned), %lld are needed", what, (long long)have,
               (long long)need);
  return FDQL_OK;
}
// Do two sets of R rows of `len` bytes, sa and sb bytes apart, share memory?  Rows equally far apart may lie between each other (columns of one wider
// row); of others the whole ranges count.
bool rows_meet(const void *a, int64_t sa, const void *b, int64_t sb, int64_t R, int64_t len) {
  const auto lo = [&](const void *p, int64_t s) { return (int64_t)(intptr_t)p + (s < 0 ? s * (R - 1) : 0); };
  const auto hi = [&](const void *p, int64_t s) { return (int64_t)(intptr_t)p + (s > 0 ? s * (R - 1) : 0) + len; };
  if (!a || !b || lo(a, sa) >= hi(b, sb) || lo(b, sb) >= hi(a, sa)) return false;
  if (sa != sb || sa <= 0) return true;
  const int64_t off = (((int64_t)(intptr_t)b - (int64_t)(intptr_t)a) % sa + sa) % sa;
  return off < len || off > sa - len;
}
#define FDQL_TRY(call)              \
  do {                              \
    const int _rc = (call);         \
    if (_rc != FDQL_OK) return _rc; \
  } while (0)

// State-space joiner: reset[t][b] where window b breaks between t - 1 and t (the same test as is_contiguous: episode_step runs on and the step
// before was not terminal), and A = -exp(A_log).
__global__ __launch_bounds__(256) void k_ssm_prep(const float *task_done, const float *episode_step, int T, int B, uint8_t *reset, const float *A_log, float *A, int n) {
  const int64_t rows = (int64_t)T * B;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows + n; i += (int64_t)gridDim.x * 256) {
    if (i < rows) reset[i] = i >= B && !(episode_step[i] == episode_step[i - B] + 1.f && task_done[i - B] == 0.f);
    else A[i - rows] = -exp_acc(A_log[i - rows]);
  }
}
// d A_log = dA * dA/dA_log = dA * A
__global__ __launch_bounds__(256) void k_ssm_dalog(const float *dA, const float *A, int n, float *out) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) out[i] = dA[i] * A[i];
}

}  // namespace

namespace fdql {
hipError_t ssm_prep_launch(const float *task_done, const float *episode_step, int T, int B, uint8_t *reset, const float *A_log, float *A, int n, hipStream_t s) {
  hipLaunchKernelGGL(k_ssm_prep, grid_for((int64_t)T * B + n), dim3(256), 0, s, task_done, episode_step, T, B, reset, A_log, A, n);
  return hipGetLastError();
}
hipError_t ssm_dalog_launch(const float *dA, const float *A, int n, float *out, hipStream_t s) {
  hipLaunchKernelGGL(k_ssm_dalog, dim3((n + 255) / 256), dim3(256), 0, s, dA, A, n, out);
  return hipGetLastError();
}
}  // namespace fdql

extern "C" int fdql_causal_conv(const fdql_causal_conv_t *p, void *stream) {
  FDQL_TRY(check_conv(p));
  if (p->R == 0) return FDQL_OK;
  FDQL_REQUIRE(!p->state_out || p->state_out != p->state_in || (p->T == 1), "causal_conv: the state is updated in place only in a single step");
  FDQL_REQUIRE(!p->state_out || p->R == 1 || p->state_out_sr >= (p->K - 1ll) * p->D, "causal_conv: rows of state_out %lld apart overlap", (long long)p->state_out_sr);
  FDQL_REQUIRE(!p->state_out || p->state_out != p->state_in || p->state_in_sr == p->state_out_sr, "causal_conv: a state updated in place has one row stride");
  const int64_t esz = p->dtype == FDQL_F32 ? 4 : 2;
  FDQL_REQUIRE(p->state_out == p->state_in || !rows_meet(p->state_in, p->state_in_sr * esz, p->state_out, p->state_out_sr * esz, p->R, (p->K - 1ll) * p->D * esz),
               "causal_conv: state_out overlaps state_in in other places");
  FDQL_REQUIRE(p->weight && (p->T == 0 || (p->x && p->y)), "causal_conv: x, weight and y are needed");
  FDQL_HIP(seqconv_fwd_launch(*p, (hipStream_t)stream));
  return FDQL_OK;
}
extern "C" int64_t fdql_causal_conv_workspace_bytes(const fdql_causal_conv_t *p) {
  if (check_conv(p) != FDQL_OK) return FDQL_EINVAL;
  return seqconv_workspace_bytes(*p);
}
extern "C" int fdql_causal_conv_backward(const fdql_causal_conv_t *p, void *stream) {
  hipStream_t s = (hipStream_t)stream;
  FDQL_TRY(check_conv(p));
  if (p->R == 0) {
    FDQL_TRY(zero(p->dweight, (int64_t)p->D * p->K, FDQL_F32, s));
    return zero(p->dbias, p->D, FDQL_F32, s);
  }
  FDQL_REQUIRE(p->weight && (p->T == 0 || (p->x && p->dy)), "causal_conv backward: x, weight and dy are needed");
  FDQL_TRY(check_workspace("causal_conv backward", p->workspace, p->workspace_bytes, seqconv_workspace_bytes(*p)));
  FDQL_HIP(seqconv_bwd_launch(*p, s));
  return FDQL_OK;
}

extern "C" int fdql_scan(const fdql_scan_t *p, void *stream) {
  hipStream_t s = (hipStream_t)stream;
  FDQL_TRY(check_scan(p));
  if (p->R == 0) return FDQL_OK;
  FDQL_REQUIRE(!p->state_out || p->state_out != p->state_in || (p->T == 1 && !p->checkpoints), "scan: the state is updated in place only in a single step");
  FDQL_REQUIRE(!p->state_out || p->R == 1 || p->state_out_sr >= (int64_t)p->D * p->N, "scan: rows of state_out %lld apart overlap", (long long)p->state_out_sr);
  FDQL_REQUIRE(!p->state_out || p->state_out != p->state_in || p->state_in_sr == p->state_out_sr, "scan: a state updated in place has one row stride");
  FDQL_REQUIRE(p->state_out == p->state_in || !rows_meet(p->state_in, p->state_in_sr * 4, p->state_out, p->state_out_sr * 4, p->R, (int64_t)p->D * p->N * 4),
               "scan: state_out overlaps state_in in other places");
  if (p->T == 0) return copy_rows(p->state_in, p->state_in_sr, p->state_out, p->state_out_sr, p->R, (int64_t)p->D * p->N, s);
  FDQL_REQUIRE(p->x && p->dt && p->A && p->B && p->C && p->y, "scan: x, dt, A, B, C and y are needed");
  FDQL_TRY(check_workspace("scan", p->workspace, p->workspace_bytes, scan_workspace_bytes(*p, false)));
  FDQL_HIP(scan_fwd_launch(*p, s));
  return FDQL_OK;
}
extern "C" int64_t fdql_scan_checkpoint_floats(const fdql_scan_t *p) {
  if (check_scan(p) != FDQL_OK) return FDQL_EINVAL;
  return scan_checkpoint_floats(*p);
}
extern "C" int64_t fdql_scan_workspace_bytes(const fdql_scan_t *p, int32_t backward) {
  if (check_scan(p) != FDQL_OK) return FDQL_EINVAL;
  return scan_workspace_bytes(*p, backward != 0);
}
extern "C" int fdql_scan_backward(const fdql_scan_t *p, void *stream) {
  hipStream_t s = (hipStream_t)stream;
  FDQL_TRY(check_scan(p));
  if (p->R == 0 || p->T == 0) {
    FDQL_TRY(zero(p->dA, (int64_t)p->D * p->N, FDQL_F32, s));
    FDQL_TRY(zero(p->dskip, p->D, FDQL_F32, s));
    FDQL_TRY(zero(p->ddt_bias, p->D, FDQL_F32, s));
    return copy_rows(p->dstate_out, (int64_t)p->D * p->N, p->dstate_in, (int64_t)p->D * p->N, p->R, (int64_t)p->D * p->N, s);
  }
  FDQL_REQUIRE(p->x && p->dt && p->A && p->B && p->C && p->dy, "scan backward: x, dt, A, B, C and dy are needed");
  FDQL_REQUIRE(p->checkpoints, "scan backward: the forward call's checkpoints are needed");
  FDQL_REQUIRE(p->dx && p->ddt && p->dA && p->dB && p->dC, "scan backward: dx, ddt, dA, dB and dC are needed");
  FDQL_TRY(check_workspace("scan backward", p->workspace, p->workspace_bytes, scan_workspace_bytes(*p, true)));
  FDQL_HIP(scan_bwd_launch(*p, s));
  return FDQL_OK;
}

extern "C" int fdql_gated(const fdql_gated_t *p, void *stream) {
  FDQL_TRY(check_gated(p));
  if (p->M == 0) return FDQL_OK;
  FDQL_REQUIRE(p->x && p->w_gate && p->w_up && p->y, "gated: x, both weights and y are needed");
  FDQL_REQUIRE(!p->b_gate == !p->b_up, "gated: both biases or neither");
  FDQL_TRY(check_workspace("gated", p->workspace, p->workspace_bytes, gated_workspace_bytes(*p, false)));
  FDQL_HIP(gated_fwd_launch(*p, (hipStream_t)stream));
  return FDQL_OK;
}
extern "C" int64_t fdql_gated_workspace_bytes(const fdql_gated_t *p, int32_t backward) {
  if (check_gated(p) != FDQL_OK) return FDQL_EINVAL;
  return gated_workspace_bytes(*p, backward != 0);
}
extern "C" int fdql_gated_backward(const fdql_gated_t *p, void *stream) {
  hipStream_t s = (hipStream_t)stream;
  FDQL_TRY(check_gated(p));
  FDQL_REQUIRE(!p->dw_gate == !p->dw_up && !p->db_gate == !p->db_up, "gated backward: the gradients of the gate and up sides come together");
  if (p->M == 0) {
    FDQL_TRY(zero(p->dw_gate, (int64_t)p->F * p->D, p->dtype, s));
    FDQL_TRY(zero(p->dw_up, (int64_t)p->F * p->D, p->dtype, s));
    FDQL_TRY(zero(p->db_gate, p->F, p->dtype, s));
    return zero(p->db_up, p->F, p->dtype, s);
  }
  FDQL_REQUIRE(p->x && p->w_gate && p->w_up && p->dy && p->pre, "gated backward: x, both weights, dy and the forward call's pre are needed");
  FDQL_TRY(check_workspace("gated backward", p->workspace, p->workspace_bytes, gated_workspace_bytes(*p, true)));
  FDQL_HIP(gated_bwd_launch(*p, s));
  return FDQL_OK;
}
