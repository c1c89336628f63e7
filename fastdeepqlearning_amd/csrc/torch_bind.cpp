// torch binding of the sequence operators (fdql_causal_conv / fdql_scan / fdql_gated, include/fdql.h): argument checks, output and workspace
// tensors and the autograd nodes, in C++ because an acting step is a few microseconds of GPU work and a Python autograd node alone costs
// a training window 100 us of host time.  The entry points of libfdql_hip.so are handed in by bind() (fastdeepqlearning_amd/sequence.py),
// so both sides use the library that _native.py loaded.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <unordered_set>

#include "../../include/fdql.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Opt;

struct {
  const char *(*last_error)();
  int (*conv)(const fdql_causal_conv_t *, void *);
  int64_t (*conv_ws)(const fdql_causal_conv_t *);
  int (*conv_bwd)(const fdql_causal_conv_t *, void *);
  int (*scan)(const fdql_scan_t *, void *);
  int64_t (*scan_ck)(const fdql_scan_t *);
  int64_t (*scan_ws)(const fdql_scan_t *, int32_t);
  int (*scan_bwd)(const fdql_scan_t *, void *);
  int (*gated)(const fdql_gated_t *, void *);
  int64_t (*gated_ws)(const fdql_gated_t *, int32_t);
  int (*gated_bwd)(const fdql_gated_t *, void *);
} api;

struct FdqlException : std::runtime_error {
  int64_t code;
  FdqlException(int64_t c, const char *msg) : std::runtime_error(msg), code(c) {}
};
void check(int64_t rc) {
  if (rc < 0) throw FdqlException(rc, api.last_error());
}

void *ptr(const Tensor &t) {
  if (!t.defined()) return nullptr;
  void *const p = const_cast<void *>(t.const_data_ptr());
  TORCH_CHECK(p || t.numel() == 0, "sequence operators: a tensor of ", t.sizes(), " has no memory");
  return p;
}
float *fptr(const Tensor &t) { return static_cast<float *>(ptr(t)); }
uint8_t *bptr(const Tensor &t) { return static_cast<uint8_t *>(ptr(t)); }
Tensor val(const Opt &t) { return t.has_value() ? *t : Tensor(); }
Opt opt(const Tensor &t) { return t.defined() ? Opt(t) : Opt(); }        // (an autograd node takes no undefined tensor, but an empty optional)
void *stream_of(const Tensor &x) { return (void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream(); }
Tensor scratch(int64_t bytes, const Tensor &like) {
  check(bytes);
  return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
Tensor like(const Tensor &t) { return t.defined() ? at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous)) : Tensor(); }
// The values as memory holds them: a view that torch negates on reading is written out, a gradient that is a symbolic zero becomes zeros.
Tensor stored(const Tensor &t) { return t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : t.is_neg() ? t.resolve_neg() : t; }
// the last dimension dense / everything dense / everything behind the first dimension dense
Tensor dense(const Tensor &u) {
  if (!u.defined()) return u;
  const Tensor t = stored(u);
  return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
}
Tensor whole(const Tensor &t) { return t.defined() ? stored(t).contiguous() : t; }
Tensor rows_dense(const Tensor &u) {
  if (!u.defined()) return u;
  const Tensor t = stored(u);
  return t.size(0) == 0 || t.select(0, 0).is_contiguous() ? t : t.contiguous();
}

int32_t type_of(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FDQL_F32;
    case at::kBFloat16: return FDQL_BF16;
    case at::kHalf: return FDQL_F16;
    default: return -1;
  }
}
int32_t small(int64_t n) {
  TORCH_CHECK_VALUE(n <= INT32_MAX, "a dimension of ", n, " is more than one call takes");
  return (int32_t)n;
}
void head(const char *what, const Tensor &x, int64_t dims) {
  TORCH_CHECK_VALUE(x.is_cuda(), what, ": x must be a tensor on the GPU (there is no CPU path)");
  TORCH_CHECK_VALUE(type_of(x) >= 0, what, ": float32, bfloat16 or float16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() == dims, what, ": x must have ", dims, " dimensions, got ", x.sizes());
  TORCH_CHECK_VALUE(x.size(-1) >= 1, what, ": x has no channels");
}
void same(const char *what, const char *name, const Tensor &x, const Tensor &t, at::IntArrayRef shape, at::ScalarType type) {
  if (!t.defined()) return;
  TORCH_CHECK_VALUE(t.device() == x.device(), what, ": ", name, " must be on ", x.device(), ", it is on ", t.device());
  TORCH_CHECK_VALUE(t.sizes() == shape, what, ": ", name, " must be ", shape, ", got ", t.sizes());
  TORCH_CHECK_VALUE(t.scalar_type() == type, what, ": ", name, " must be ", type, ", got ", t.scalar_type());
}
void check_reset(const char *what, const Tensor &x, const Tensor &r) {
  if (!r.defined()) return;
  TORCH_CHECK_VALUE(r.device() == x.device() && (r.scalar_type() == at::kBool || r.scalar_type() == at::kByte), what, ": reset must be a bool or uint8 tensor on ", x.device());
  TORCH_CHECK_VALUE(r.sizes() == x.sizes().slice(0, x.dim() - 1), what, ": reset must be ", x.sizes().slice(0, x.dim() - 1), ", got ", r.sizes());
}
bool graded(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor &t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
void no_grad(const char *what, std::initializer_list<Tensor> ts) {
  TORCH_CHECK_VALUE(!graded(ts), what, " has no gradient: call it under torch.no_grad(), or the windowed form with T = 1");
}
// The calls go past torch's dispatcher: a trace would hold the allocation of their results and nothing that fills them.
void not_traced(const char *what) {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  bool traced = torch::jit::tracer::isTracing();
  if (TorchDispatchModeTLS::any_modes_set())
    for (const auto mode : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
      traced = traced || TorchDispatchModeTLS::get_mode(mode).has_value();
  TORCH_CHECK(!traced, what, " cannot be traced: its kernels would be missing from the trace (capture the call into a graph instead)");
}
// Tensors whose memory holds their values: a subclass that dispatches by itself or a functional transform's wrapper has none of its own, and the operators
// have no forward-mode derivative, a tangent would be dropped without a word.
void plain_one(const char *what, const Tensor &t) {
  constexpr c10::DispatchKeySet foreign({c10::DispatchKey::Python, c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::Batched,
                                         c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::ZeroTensor});
  if (!t.defined()) return;
  TORCH_CHECK_VALUE(!t.key_set().has_any(foreign), what, ": plain tensors only, one is a wrapper without memory of its own");
  TORCH_CHECK_VALUE(!t._fw_grad(0).defined(), what, " has no forward-mode derivative: a tensor carries a tangent");
}
void plain_one(const char *what, const Opt &t) {
  if (t.has_value()) plain_one(what, *t);
}
template <typename... Ts>
void plain(const char *what, const Ts &...ts) {
  (plain_one(what, ts), ...);
}
// A tensor that a kernel writes in place counts as changed: a backward pass that saved it refuses, as behind torch's own in-place operators.
void written(const Tensor &t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// Every node that the running backward pass will run behind (in its order) the node that runs now, once each, until `stop` says so: that node, or null.
// A pass for chosen inputs runs part of a graph only.
template <typename F>
torch::autograd::Node *nodes_ahead(F stop) {
  const auto node = torch::autograd::get_current_node();
  const auto *runs = torch::autograd::get_current_graph_task_exec_info();       // empty: every node does
  std::vector<torch::autograd::Node *> todo;
  std::unordered_set<torch::autograd::Node *> seen;
  if (node) todo.push_back(node.get());
  while (!todo.empty()) {
    torch::autograd::Node *n = todo.back();
    todo.pop_back();
    for (const auto &edge : n->next_edges()) {
      torch::autograd::Node *f = edge.function.get();
      if (!f || !seen.insert(f).second) continue;
      if (runs && !runs->empty()) {
        const auto it = runs->find(f);
        if (it == runs->end() || !it->second.should_execute()) continue;
      }
      if (stop(f)) return f;
      todo.push_back(f);
    }
  }
  return nullptr;
}
// A backward pass under capture that reaches a node which eager code has made on the default stream - a leaf's accumulator that an eager graph keeps
// alive, or such a graph itself - would have that stream wait for the capture, which is not allowed and ends the process.  The call refuses
// instead.  (Costs nothing outside a capture.)
void capturable(const char *what, const Tensor &x) {
  const auto stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess) {
    (void)hipGetLastError();                // (no stream that could be captured: the next launch must not find this error)
    return;
  }
  if (status == hipStreamCaptureStatusNone) return;
  const c10::Stream here = stream.unwrap(), eager = c10::hip::getDefaultHIPStreamMasqueradingAsCUDA(x.device().index()).unwrap();
  const torch::autograd::Node *bad = nodes_ahead([&](torch::autograd::Node *f) {
    const auto at = f->stream();
    return at && *at != here && *at == eager;
  });
  TORCH_CHECK(!bad, what, ": this backward pass is being captured and reaches an eager graph on the default stream (", bad->name(),
              "); delete what holds that graph (its outputs, its loss) before the capture");
}
// Gradients of a backward pass that itself is recorded (create_graph) depend on everything in `from`: differentiating them again is an error, not a silent
// zero.
variable_list once(const char *what, variable_list grads, const variable_list &from, const variable_list &incoming) {
  if (!at::GradMode::is_enabled()) return grads;
  const auto error = std::make_shared<torch::autograd::Error>(std::string(what) + " is differentiable once", torch::autograd::collect_next_edges(from, incoming));
  for (Tensor &g : grads)
    if (g.defined()) torch::autograd::create_gradient_edge(g, error);
  return grads;
}

// Which of a node's tensor arguments want a gradient: the node numbers those that are there.
struct Needs {
  bool on[12] = {};
  Needs(AutogradContext *ctx, const variable_list &args, size_t n) {
    size_t edge = 0;
    for (size_t k = 0; k < n; ++k)
      if (args[k].defined()) on[k] = ctx->needs_input_grad(edge++);
  }
};

// --------------------------------------------------------------------------------------------------------------- convolution
fdql_causal_conv_t conv_args(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &state, const Tensor &reset, bool silu) {
  fdql_causal_conv_t p = {};
  const bool win = x.dim() == 3;
  p.size = sizeof(p);
  p.dtype = type_of(x);
  p.T = win ? small(x.size(0)) : 1;
  p.R = small(x.size(-2));
  p.D = small(x.size(-1));
  p.K = (int32_t)weight.size(1);
  p.silu = silu;
  p.x = ptr(x);
  p.x_st = win ? x.stride(0) : 0;
  p.x_sr = x.stride(-2);
  p.weight = fptr(weight);
  p.bias = fptr(bias);
  p.state_in = ptr(state);
  if (state.defined()) p.state_in_sr = state.stride(0);
  if (reset.defined()) {
    p.reset = bptr(reset);
    p.reset_st = win ? reset.stride(0) : 0;
    p.reset_sr = reset.stride(-1);
  }
  return p;
}
std::pair<Tensor, Tensor> conv_run(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &state, const Tensor &reset, bool silu, bool want,
                                   Tensor out_state = {}) {
  c10::DeviceGuard guard(x.device());
  Tensor y = like(x);
  if (want && !out_state.defined()) out_state = at::empty({x.size(-2), weight.size(1) - 1, x.size(-1)}, x.options());
  fdql_causal_conv_t p = conv_args(x, weight, bias, state, reset, silu);
  p.y = ptr(y);
  p.state_out = ptr(out_state);
  if (out_state.defined()) p.state_out_sr = out_state.stride(0);
  check(api.conv(&p, stream_of(x)));
  return {y, out_state};
}
struct ConvNode : torch::autograd::Function<ConvNode> {
  static variable_list forward(AutogradContext *ctx, Tensor x, Tensor weight, Opt bias_, Opt state_, Opt reset_, bool silu, bool want) {
    const Tensor bias = val(bias_), state = val(state_), reset = val(reset_);
    ctx->set_materialize_grads(false);
    ctx->saved_data["silu"] = silu;
    ctx->save_for_backward({x, weight, bias, state, reset});
    auto r = conv_run(x, weight, bias, state, reset, silu, want);
    return want ? variable_list{r.first, r.second} : variable_list{r.first};
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    not_traced("causal_conv");
    capturable("causal_conv", s[0]);
    const Tensor &x = s[0], &weight = s[1], &bias = s[2], &state = s[3];
    c10::DeviceGuard guard(x.device());
    const Tensor dy = g[0].defined() ? dense(g[0]) : at::zeros(x.sizes(), x.options()), ds_out = g.size() > 1 ? whole(g[1]) : Tensor();
    const Needs need(ctx, s, 5);
    const Tensor dx = need.on[0] ? like(x) : Tensor(), dw = need.on[1] ? like(weight) : Tensor(), db = need.on[2] ? like(bias) : Tensor(),
                 ds = need.on[3] ? like(state) : Tensor();
    fdql_causal_conv_t p = conv_args(x, weight, bias, state, s[4], ctx->saved_data["silu"].toBool());
    p.dy = ptr(dy);
    p.dy_st = dy.stride(0);
    p.dy_sr = dy.stride(1);
    p.dstate_out = ptr(ds_out);
    p.dx = ptr(dx);
    p.dweight = fptr(dw);
    p.dbias = fptr(db);
    p.dstate_in = ptr(ds);
    const Tensor ws = scratch(api.conv_ws(&p), x);
    p.workspace = ptr(ws);
    p.workspace_bytes = ws.defined() ? ws.numel() : 0;
    check(api.conv_bwd(&p, stream_of(x)));
    return once("causal_conv", {dx, dw, db, ds, Tensor(), Tensor(), Tensor()}, s, g);
  }
};
void conv_check(const char *what, const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &state) {
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) >= 2 && weight.size(1) <= 4, what, ": weight must be [channels, 2..4 taps], got ", weight.sizes());
  const int64_t D = x.size(-1), K = weight.size(1);
  same(what, "weight", x, weight, {D, K}, at::kFloat);
  same(what, "bias", x, bias, {D}, at::kFloat);
  same(what, "state", x, state, {x.size(-2), K - 1, D}, x.scalar_type());
}
std::pair<Tensor, Opt> causal_conv(const Tensor &x, const Tensor &weight, const Opt &bias_, const Opt &reset_, const Opt &state_, bool silu, bool want) {
  const char *what = "causal_conv";
  const Tensor bias = val(bias_), reset = val(reset_), state = val(state_);
  not_traced(what);
  plain(what, x, weight, bias, state, reset);
  head(what, x, 3);
  conv_check(what, x, weight, bias, state);
  check_reset(what, x, reset);
  if (graded({x, weight, bias, state})) {
    const variable_list r = ConvNode::apply(dense(x), whole(weight), opt(whole(bias)), opt(rows_dense(state)), opt(reset), silu, want);
    return {r[0], want ? Opt(r[1]) : Opt()};
  }
  auto r = conv_run(dense(x), whole(weight), whole(bias), rows_dense(state), reset, silu, want);
  return {r.first, want ? Opt(r.second) : Opt()};
}
std::pair<Tensor, Tensor> causal_conv_step(const Tensor &x, const Opt &state_, const Tensor &weight, const Opt &bias_, const Opt &reset_, bool silu, const Opt &out_) {
  const char *what = "causal_conv_step";
  const Tensor bias = val(bias_), reset = val(reset_), state = val(state_), out = val(out_);
  not_traced(what);
  plain(what, x, state, weight, bias, out, reset);
  head(what, x, 2);
  TORCH_CHECK_VALUE(state.defined(), what, ": a state is needed");
  conv_check(what, x, weight, bias, state);
  check_reset(what, x, reset);
  no_grad(what, {x, state, weight, bias, out});
  same(what, "out_state", x, out, state.sizes(), x.scalar_type());
  TORCH_CHECK_VALUE(!out.defined() || (!out.is_neg() && (out.size(0) == 0 || out.select(0, 0).is_contiguous())), what, ": rows of out_state must be dense");
  auto r = conv_run(dense(x), whole(weight), whole(bias), rows_dense(state), reset, silu, true, out);
  written(out);
  return r;
}

// ---------------------------------------------------------------------------------------------------------------------- scan
struct ScanIn {
  Tensor x, dt, A, B, C, skip, z, dt_bias, state, reset;
  bool softplus;
};
fdql_scan_t scan_args(const ScanIn &i) {
  fdql_scan_t p = {};
  const bool win = i.x.dim() == 3;
  const auto st = [&](const Tensor &t) { return win ? t.stride(0) : 0; };
  const int64_t r = win;                                    // the row dimension
  p.size = sizeof(p);
  p.dtype = type_of(i.x);
  p.T = win ? small(i.x.size(0)) : 1;
  p.R = small(i.x.size(r));
  p.D = small(i.x.size(-1));
  p.G = small(i.B.size(-2));
  p.N = (int32_t)i.B.size(-1);
  p.dt_softplus = i.softplus;
  p.x = ptr(i.x), p.x_st = st(i.x), p.x_sr = i.x.stride(r);
  p.dt = ptr(i.dt), p.dt_st = st(i.dt), p.dt_sr = i.dt.stride(r);
  if (i.z.defined()) p.z = ptr(i.z), p.z_st = st(i.z), p.z_sr = i.z.stride(r);
  p.B = ptr(i.B), p.B_st = st(i.B), p.B_sr = i.B.stride(r), p.B_sg = i.B.stride(r + 1);
  p.C = ptr(i.C), p.C_st = st(i.C), p.C_sr = i.C.stride(r), p.C_sg = i.C.stride(r + 1);
  p.A = fptr(i.A);
  p.skip = fptr(i.skip);
  p.dt_bias = fptr(i.dt_bias);
  if (i.reset.defined()) p.reset = bptr(i.reset), p.reset_st = st(i.reset), p.reset_sr = i.reset.stride(r);
  if (i.state.defined()) p.state_in = fptr(i.state), p.state_in_sr = i.state.stride(0);
  return p;
}
std::tuple<Tensor, Tensor, Tensor> scan_run(const ScanIn &i, bool want, bool train, Tensor out_state = {}) {
  c10::DeviceGuard guard(i.x.device());
  const Tensor y = like(i.x);
  fdql_scan_t p = scan_args(i);
  if (want && !out_state.defined()) out_state = at::empty({p.R, p.D, p.N}, i.A.options());
  Tensor ck, ws;
  if (train) {
    const int64_t n = api.scan_ck(&p);
    check(n);
    ck = at::empty({n}, i.A.options());
  }
  if (p.T > 1) ws = scratch(api.scan_ws(&p, 0), i.x);
  p.y = ptr(y);
  p.state_out = fptr(out_state);
  if (out_state.defined()) p.state_out_sr = out_state.stride(0);
  p.checkpoints = fptr(ck);
  p.workspace = ptr(ws);
  p.workspace_bytes = ws.defined() ? ws.numel() : 0;
  check(api.scan(&p, stream_of(i.x)));
  return {y, out_state, ck};
}
struct ScanNode : torch::autograd::Function<ScanNode> {
  static variable_list forward(AutogradContext *ctx, Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Opt skip_, Opt z_, Opt dt_bias_, Opt state_, Opt reset_,
                               bool softplus, bool want) {
    const Tensor skip = val(skip_), z = val(z_), dt_bias = val(dt_bias_), state = val(state_), reset = val(reset_);
    ctx->set_materialize_grads(false);
    ctx->saved_data["softplus"] = softplus;
    const ScanIn i = {x, dt, A, B, C, skip, z, dt_bias, state, reset, softplus};
    auto r = scan_run(i, want, true);
    ctx->save_for_backward({x, dt, A, B, C, skip, z, dt_bias, state, reset, std::get<2>(r)});
    return want ? variable_list{std::get<0>(r), std::get<1>(r)} : variable_list{std::get<0>(r)};
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    not_traced("selective_scan");
    capturable("selective_scan", s[0]);
    const ScanIn i = {s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9], ctx->saved_data["softplus"].toBool()};
    c10::DeviceGuard guard(i.x.device());
    const Tensor dy = g[0].defined() ? dense(g[0]) : at::zeros(i.x.sizes(), i.x.options()), ds_out = g.size() > 1 ? whole(g[1]) : Tensor();
    const Needs need(ctx, s, 10);
    variable_list d;
    for (int k = 0; k < 8; ++k) d.push_back(like(s[k]));
    d.push_back(need.on[8] ? like(i.state) : Tensor());
    fdql_scan_t p = scan_args(i);
    p.checkpoints = fptr(s[10]);
    p.dy = ptr(dy);
    p.dy_st = dy.stride(0);
    p.dy_sr = dy.stride(1);
    p.dstate_out = fptr(ds_out);
    p.dx = ptr(d[0]), p.ddt = ptr(d[1]), p.dA = fptr(d[2]), p.dB = ptr(d[3]), p.dC = ptr(d[4]);
    p.dskip = fptr(d[5]), p.dz = ptr(d[6]), p.ddt_bias = fptr(d[7]), p.dstate_in = fptr(d[8]);
    const Tensor ws = scratch(api.scan_ws(&p, 1), i.x);
    p.workspace = ptr(ws);
    p.workspace_bytes = ws.defined() ? ws.numel() : 0;
    check(api.scan_bwd(&p, stream_of(i.x)));
    for (int k = 0; k < 9; ++k)
      if (!need.on[k]) d[k] = Tensor();
    d.resize(12);
    return once("selective_scan", std::move(d), s, g);
  }
};
// checks everything; B and C come back with their group dimension
ScanIn scan_check(const char *what, const Tensor &x, const Tensor &dt, const Tensor &A, Tensor B, Tensor C, const Tensor &skip, const Tensor &z, const Tensor &dt_bias,
                  const Tensor &state, const Tensor &reset, bool softplus) {
  TORCH_CHECK_VALUE(A.dim() == 2 && A.size(1) >= 1 && A.size(1) <= 64, what, ": A must be [channels, 1..64 states], got ", A.sizes());
  const int64_t D = x.size(-1), N = A.size(1), R = x.size(-2);
  same(what, "A", x, A, {D, N}, at::kFloat);
  same(what, "dt", x, dt, x.sizes(), x.scalar_type());
  TORCH_CHECK_VALUE((B.dim() == x.dim() || B.dim() == x.dim() + 1) && C.dim() == B.dim(), what, ": B and C must be [..., rows, states] or [..., rows, groups, states], got ",
                    B.sizes(), " and ", C.sizes());
  if (B.dim() == x.dim()) B = B.unsqueeze(-2), C = C.unsqueeze(-2);
  const int64_t G = B.size(-2);
  TORCH_CHECK_VALUE(G >= 1 && D % G == 0, what, ": ", G, " groups do not divide ", D, " channels");
  c10::SmallVector<int64_t, 4> bc(x.sizes().begin(), x.sizes().end() - 1);
  bc.push_back(G);
  bc.push_back(N);
  same(what, "B", x, B, bc, x.scalar_type());
  same(what, "C", x, C, bc, x.scalar_type());
  same(what, "z", x, z, x.sizes(), x.scalar_type());
  same(what, "skip", x, skip, {D}, at::kFloat);
  same(what, "dt_bias", x, dt_bias, {D}, at::kFloat);
  same(what, "state", x, state, {R, D, N}, at::kFloat);
  check_reset(what, x, reset);
  return {dense(x), dense(dt), whole(A), dense(B), dense(C), whole(skip), dense(z), whole(dt_bias), rows_dense(state), reset, softplus};
}
std::pair<Tensor, Opt> selective_scan(const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const Opt &skip, const Opt &z, const Opt &dt_bias,
                                      bool softplus, const Opt &reset, const Opt &state, bool want) {
  const char *what = "selective_scan";
  not_traced(what);
  plain(what, x, dt, A, B, C, skip, z, dt_bias, state, reset);
  head(what, x, 3);
  const ScanIn i = scan_check(what, x, dt, A, B, C, val(skip), val(z), val(dt_bias), val(state), val(reset), softplus);
  if (graded({i.x, i.dt, i.A, i.B, i.C, i.skip, i.z, i.dt_bias, i.state})) {
    const variable_list r = ScanNode::apply(i.x, i.dt, i.A, i.B, i.C, opt(i.skip), opt(i.z), opt(i.dt_bias), opt(i.state), opt(i.reset), softplus, want);
    return {r[0], want ? Opt(r[1]) : Opt()};
  }
  auto r = scan_run(i, want, false);
  return {std::get<0>(r), want ? Opt(std::get<1>(r)) : Opt()};
}
std::pair<Tensor, Tensor> selective_scan_step(const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const Opt &state_, const Opt &skip,
                                              const Opt &z, const Opt &dt_bias, bool softplus, const Opt &reset, const Opt &out_) {
  const char *what = "selective_scan_step";
  const Tensor state = val(state_), out = val(out_);
  not_traced(what);
  plain(what, x, dt, A, B, C, state, skip, z, dt_bias, out, reset);
  head(what, x, 2);
  TORCH_CHECK_VALUE(state.defined(), what, ": a state is needed");
  const ScanIn i = scan_check(what, x, dt, A, B, C, val(skip), val(z), val(dt_bias), state, val(reset), softplus);
  no_grad(what, {x, dt, A, B, C, i.skip, i.z, i.dt_bias, state, out});
  same(what, "out_state", x, out, state.sizes(), at::kFloat);
  TORCH_CHECK_VALUE(!out.defined() || (!out.is_neg() && (out.size(0) == 0 || out.select(0, 0).is_contiguous())), what, ": rows of out_state must be dense");
  auto r = scan_run(i, true, false, out);
  written(out);
  return {std::get<0>(r), std::get<1>(r)};
}

// --------------------------------------------------------------------------------------------------------------------- gated
fdql_gated_t gated_args(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &bg, const Tensor &bu, int64_t act) {
  fdql_gated_t p = {};
  p.size = sizeof(p);
  p.dtype = type_of(x);
  p.M = x.size(0);
  p.D = small(x.size(1));
  p.F = small(wg.size(0));
  p.act = (int32_t)act;
  p.x = ptr(x);
  p.x_sr = x.stride(0);
  p.w_gate = ptr(wg), p.w_up = ptr(wu), p.b_gate = ptr(bg), p.b_up = ptr(bu);
  return p;
}
std::pair<Tensor, Tensor> gated_run(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &bg, const Tensor &bu, int64_t act, bool train) {
  c10::DeviceGuard guard(x.device());
  const Tensor y = at::empty({x.size(0), wg.size(0)}, x.options()),
               pre = train ? at::empty({2, x.size(0), wg.size(0)}, x.options().dtype(at::kFloat)) : Tensor();
  fdql_gated_t p = gated_args(x, wg, wu, bg, bu, act);
  p.y = ptr(y);
  p.pre = fptr(pre);
  const Tensor ws = scratch(api.gated_ws(&p, 0), x);
  p.workspace = ptr(ws);
  p.workspace_bytes = ws.defined() ? ws.numel() : 0;
  check(api.gated(&p, stream_of(x)));
  return {y, pre};
}
struct GatedNode : torch::autograd::Function<GatedNode> {
  static Tensor forward(AutogradContext *ctx, Tensor x, Tensor wg, Tensor wu, Opt bg_, Opt bu_, int64_t act) {
    const Tensor bg = val(bg_), bu = val(bu_);
    ctx->saved_data["act"] = act;
    auto r = gated_run(x, wg, wu, bg, bu, act, true);
    ctx->save_for_backward({x, wg, wu, bg, bu, r.second});
    return r.first;
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    not_traced("gated_linear");
    capturable("gated_linear", s[0]);
    const Tensor &x = s[0];
    c10::DeviceGuard guard(x.device());
    const Tensor dy = dense(g[0]);
    const Needs need(ctx, s, 5);
    const bool w = need.on[1] || need.on[2], b = need.on[3] || need.on[4];
    variable_list d = {need.on[0] ? like(x) : Tensor(), w ? like(s[1]) : Tensor(), w ? like(s[2]) : Tensor(), b ? like(s[3]) : Tensor(),
                       b ? like(s[4]) : Tensor()};
    fdql_gated_t p = gated_args(x, s[1], s[2], s[3], s[4], ctx->saved_data["act"].toInt());
    p.pre = fptr(s[5]);
    p.dy = ptr(dy);
    p.dy_sr = dy.stride(0);
    p.dx = ptr(d[0]), p.dw_gate = ptr(d[1]), p.dw_up = ptr(d[2]), p.db_gate = ptr(d[3]), p.db_up = ptr(d[4]);
    const Tensor ws = scratch(api.gated_ws(&p, 1), x);
    p.workspace = ptr(ws);
    p.workspace_bytes = ws.defined() ? ws.numel() : 0;
    check(api.gated_bwd(&p, stream_of(x)));
    for (int k = 1; k < 5; ++k)
      if (!need.on[k]) d[k] = Tensor();
    d.resize(6);
    return once("gated_linear", std::move(d), s, g);
  }
};
Tensor gated_linear(const Tensor &x, const Tensor &wg, const Tensor &wu, const Opt &bg_, const Opt &bu_, int64_t act) {
  const char *what = "gated_linear";
  const Tensor bg = val(bg_), bu = val(bu_);
  not_traced(what);
  plain(what, x, wg, wu, bg, bu);
  TORCH_CHECK_VALUE(x.dim() >= 1, what, ": x must be [..., channels]");
  head(what, x, x.dim());
  TORCH_CHECK_VALUE(wg.dim() == 2 && wg.size(0) >= 1, what, ": w_gate must be [features, channels], got ", wg.sizes());
  const int64_t F = wg.size(0), D = x.size(-1);
  same(what, "w_gate", x, wg, {F, D}, x.scalar_type());
  same(what, "w_up", x, wu, {F, D}, x.scalar_type());
  TORCH_CHECK_VALUE(bg.defined() == bu.defined(), what, ": both biases or neither");
  same(what, "b_gate", x, bg, {F}, x.scalar_type());
  same(what, "b_up", x, bu, {F}, x.scalar_type());
  const Tensor flat = dense(x.dim() == 2 ? x : x.reshape({-1, D}));
  const Tensor y = graded({x, wg, wu, bg, bu}) ? GatedNode::apply(flat, whole(wg), whole(wu), opt(whole(bg)), opt(whole(bu)), act)
                                               : gated_run(flat, whole(wg), whole(wu), whole(bg), whole(bu), act, false).first;
  if (x.dim() == 2) return y;
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end() - 1);
  shape.push_back(F);
  return y.view(shape);
}

template <typename F>
void take(const py::dict &d, const char *name, F &f) {
  f = reinterpret_cast<F>(py::cast<uintptr_t>(d[name]));
}

}  // namespace

PYBIND11_MODULE(_seq_torch, m) {
  m.doc() = "torch binding of the sequence operators: see fastdeepqlearning_amd/sequence.py";
  m.def("bind", [](const py::dict &d, const py::object &error) {     // addresses of the library's entry points, the exception class
    take(d, "fdql_last_error", api.last_error);
    take(d, "fdql_causal_conv", api.conv);
    take(d, "fdql_causal_conv_workspace_bytes", api.conv_ws);
    take(d, "fdql_causal_conv_backward", api.conv_bwd);
    take(d, "fdql_scan", api.scan);
    take(d, "fdql_scan_checkpoint_floats", api.scan_ck);
    take(d, "fdql_scan_workspace_bytes", api.scan_ws);
    take(d, "fdql_scan_backward", api.scan_bwd);
    take(d, "fdql_gated", api.gated);
    take(d, "fdql_gated_workspace_bytes", api.gated_ws);
    take(d, "fdql_gated_backward", api.gated_bwd);
    static py::object *cls = new py::object(error);                 // (lives as long as the process, like the library)
    py::register_local_exception_translator([](std::exception_ptr p) {
      try {
        if (p) std::rethrow_exception(p);
      } catch (const FdqlException &e) {
        PyErr_SetObject(cls->ptr(), (*cls)(e.code, e.what()).ptr());
      }
    });
  });
  typedef py::call_guard<py::gil_scoped_release> free_gil;
  m.def("causal_conv", &causal_conv, free_gil());
  m.def("causal_conv_step", &causal_conv_step, free_gil());
  m.def("selective_scan", &selective_scan, free_gil());
  m.def("selective_scan_step", &selective_scan_step, free_gil());
  m.def("gated_linear", &gated_linear, free_gil());
  m.def("nodes_ahead", [] {            // names of the nodes that a captured backward pass is checked against, for the tests of that check
    std::vector<std::string> names;
    nodes_ahead([&](torch::autograd::Node *f) { return names.push_back(f->name()), false; });
    return names;
  });
}
