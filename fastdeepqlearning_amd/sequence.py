"""Sequence operators over time-major windows [T, rows, channels], on the C ABI's ``fdql_causal_conv`` / ``fdql_scan`` / ``fdql_gated``
(include/fdql.h) - the pieces of a recurrent block beside the reference's GRU (franQ/Agent/components/encoder.py:40-42, 78-94):

    from fastdeepqlearning_amd import sequence as seq
    x = seq.causal_conv(x, w, b, reset=reset)                     # short convolution + SiLU
    y = seq.selective_scan(x, dt, A, B, C, skip=d, z=z, dt_bias=bias, reset=reset)
    h = seq.gated_linear(y, w_gate, w_up, b_gate, b_up)           # SiLU(y Wg^T + bg) * (y Wu^T + bu)

Each is differentiable (once); ``causal_conv_step`` and ``selective_scan_step`` advance every acting row by one step.  Activations
may be float32, bfloat16 or float16 and any strided view (a copy is made only where the last dimension is not dense); states of the scan,
its A / skip / dt_bias and the convolution's weights are float32.  ``reset`` [T, rows] (bool or uint8) marks the steps at which a new sequence
begins: several sequences can share a row, and left padding is dropped by a reset at the first real step.  Calls run on the current
stream of the tensors' device, never synchronise, and can be captured into a graph.  All compute is in libfdql_hip.so; there is no CPU path."""
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from .core import _on_device

__all__ = ["causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "gated_linear"]

_TYPES = {torch.float32: 0, torch.bfloat16: 2, torch.float16: 3}
_ACTS = {"silu": 0, "gelu": 1, "sigmoid": 2}


def _need(ok, text):
    if not ok:
        raise ValueError(text)


def _like(x, name, t, shape, dtype=None):
    """Checks one tensor against the device of x, a shape and a type."""
    _need(isinstance(t, torch.Tensor) and t.device == x.device, f"{name} must be a tensor on {x.device}")
    _need(tuple(t.shape) == tuple(shape), f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    dtype = dtype or x.dtype
    _need(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")


def _head(what, x, dims):
    _need(isinstance(x, torch.Tensor) and x.is_cuda, f"{what}: x must be a tensor on the GPU (there is no CPU path)")
    _need(x.dtype in _TYPES, f"{what}: float32, bfloat16 or float16, got {x.dtype}")
    _need(x.dim() == dims, f"{what}: x must have {dims} dimensions, got {tuple(x.shape)}")
    _need(x.shape[-1] >= 1, f"{what}: x has no channels")


def _dense(t):
    """t with a dense last dimension."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _whole(t):
    return t if t is None else t.contiguous()


def _rows_dense(t):
    """[R, ...] with everything behind the first dimension dense (any row stride)."""
    if t is None or t.shape[0] == 0 or t[0].is_contiguous():
        return t
    return t.contiguous()


def _reset_of(x, reset, lead):
    if reset is None:
        return None
    _need(isinstance(reset, torch.Tensor) and reset.device == x.device and reset.dtype in (torch.bool, torch.uint8),
          f"reset must be a bool or uint8 tensor on {x.device}")
    _need(tuple(reset.shape) == tuple(lead), f"reset must be {tuple(lead)}, got {tuple(reset.shape)}")
    return reset


def _p(t):
    return None if t is None else t.data_ptr()


def _scratch(nbytes, device):
    if nbytes < 0:
        N.check(int(nbytes))
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _no_grad_inputs(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no gradient: call it under torch.no_grad(), or the windowed form with T = 1")


def _graded(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------------------------------------------------ convolution
def _conv_struct(x, weight, bias, state, reset, silu):
    s = N.CausalConv()
    s.size, s.dtype = C.sizeof(N.CausalConv), _TYPES[x.dtype]
    if x.dim() == 3:
        s.T, s.R, s.D = x.shape
        s.x_st, s.x_sr = x.stride(0), x.stride(1)
    else:
        s.T, (s.R, s.D) = 1, x.shape
        s.x_sr = x.stride(0)
    s.K, s.silu = weight.shape[1], int(silu)
    s.x, s.weight, s.bias, s.reset, s.state_in = _p(x), _p(weight), _p(bias), _p(reset), _p(state)
    if reset is not None:
        s.reset_st, s.reset_sr = (0,) * (2 - reset.dim()) + reset.stride()
    if state is not None:
        s.state_in_sr = state.stride(0)
    return s


def _conv_forward(x, weight, bias, state, reset, silu, want_state, out_state=None):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if want_state and out_state is None:
        out_state = torch.empty((x.shape[-2], weight.shape[1] - 1, x.shape[-1]), dtype=x.dtype, device=x.device)
    s = _conv_struct(x, weight, bias, state, reset, silu)
    s.y, s.state_out = _p(y), _p(out_state)
    with _on_device(x.device):
        N.check(N.load().fdql_causal_conv(C.byref(s), N.current_stream(x.device)))
    return y, out_state


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, reset, silu, want_state):
        ctx.set_materialize_grads(False)
        ctx.silu = silu
        ctx.save_for_backward(x, weight, bias, state, reset)
        return _conv_forward(x, weight, bias, state, reset, silu, want_state)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate):
        x, weight, bias, state, reset = ctx.saved_tensors
        need = ctx.needs_input_grad
        dev = x.device
        dy = torch.zeros_like(x, memory_format=torch.contiguous_format) if dy is None else _dense(dy)
        dstate = _whole(dstate)
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[0] else None
        dw = torch.empty_like(weight) if need[1] else None
        db = torch.empty_like(bias) if bias is not None and need[2] else None
        ds = torch.empty(state.shape, dtype=state.dtype, device=dev) if state is not None and need[3] else None
        s = _conv_struct(x, weight, bias, state, reset, ctx.silu)
        s.dy, s.dy_st, s.dy_sr, s.dstate_out = _p(dy), dy.stride(0), dy.stride(1), _p(dstate)
        s.dx, s.dweight, s.dbias, s.dstate_in = _p(dx), _p(dw), _p(db), _p(ds)
        lib = N.load()
        with _on_device(dev):
            ws = _scratch(lib.fdql_causal_conv_workspace_bytes(C.byref(s)), dev)
            s.workspace, s.workspace_bytes = _p(ws), 0 if ws is None else ws.numel()
            N.check(lib.fdql_causal_conv_backward(C.byref(s), N.current_stream(dev)))
        return dx, dw, db, ds, None, None, None


def _conv_check(what, x, weight, bias, state, R):
    _need(isinstance(weight, torch.Tensor) and weight.dim() == 2 and 2 <= weight.shape[1] <= 4, f"{what}: weight must be [channels, 2..4 taps]")
    D, K = x.shape[-1], weight.shape[1]
    _like(x, f"{what}: weight", weight, (D, K), torch.float32)
    if bias is not None:
        _like(x, f"{what}: bias", bias, (D,), torch.float32)
    if state is not None:
        _like(x, f"{what}: state", state, (R, K - 1, D))


def causal_conv(x, weight, bias=None, *, reset=None, initial_state=None, silu=True, return_state=False):
    """y_t = f(bias + sum_j weight[:, K-1-j] * x_{t-j}), f = SiLU (or identity), channel by channel.

    x [T, rows, D]; weight [D, K] (K = 2..4) and bias [D] float32; reset [T, rows]; initial_state [rows, K-1, D] in x's type, the
    inputs before step 0, oldest first (default zeros).  Returns y, or (y, state) with the last K-1 inputs when return_state."""
    _head("causal_conv", x, 3)
    _conv_check("causal_conv", x, weight, bias, initial_state, x.shape[1])
    reset = _reset_of(x, reset, x.shape[:2])
    args = (_dense(x), _whole(weight), _whole(bias), _rows_dense(initial_state), reset, bool(silu), bool(return_state))
    y, state = _Conv.apply(*args) if _graded(x, weight, bias, initial_state) else _conv_forward(*args)
    return (y, state) if return_state else y


def causal_conv_step(x, state, weight, bias=None, *, reset=None, silu=True, out_state=None):
    """One step of causal_conv for every row: x [rows, D], state [rows, K-1, D], reset [rows].  Returns (y, new state); the new state is
    written to out_state (dense; `state` itself updates it in place) or to a new tensor."""
    _head("causal_conv_step", x, 2)
    _conv_check("causal_conv_step", x, weight, bias, state, x.shape[0])
    _need(state is not None, "causal_conv_step: a state is needed")
    _no_grad_inputs("causal_conv_step", x, state, weight, bias)
    if out_state is not None:
        _like(x, "causal_conv_step: out_state", out_state, state.shape)
        _need(out_state.is_contiguous(), "causal_conv_step: out_state must be contiguous")
    return _conv_forward(_dense(x), _whole(weight), _whole(bias), _rows_dense(state), _reset_of(x, reset, x.shape[:1]), bool(silu), True, out_state)


# ------------------------------------------------------------------------------------------------------------------- scan
def _scan_struct(x, dt, A, B, Cm, skip, z, dt_bias, state, reset, softplus):
    s = N.Scan()
    s.size, s.dtype = C.sizeof(N.Scan), _TYPES[x.dtype]
    step = x.dim() == 2
    s.T, s.R, s.D = (1, *x.shape) if step else x.shape
    s.G, s.N = B.shape[-2:]
    s.dt_softplus = int(softplus)
    pad = (0,) if step else ()
    s.x, s.dt, s.z, s.B, s.C = _p(x), _p(dt), _p(z), _p(B), _p(Cm)
    s.x_st, s.x_sr, _ = pad + x.stride()
    s.dt_st, s.dt_sr, _ = pad + dt.stride()
    if z is not None:
        s.z_st, s.z_sr, _ = pad + z.stride()
    s.B_st, s.B_sr, s.B_sg, _ = pad + B.stride()
    s.C_st, s.C_sr, s.C_sg, _ = pad + Cm.stride()
    s.A, s.skip, s.dt_bias, s.reset, s.state_in = _p(A), _p(skip), _p(dt_bias), _p(reset), _p(state)
    if reset is not None:
        s.reset_st, s.reset_sr = pad + reset.stride()
    if state is not None:
        s.state_in_sr = state.stride(0)
    return s


def _scan_forward(x, dt, A, B, Cm, skip, z, dt_bias, state, reset, softplus, want_state, train=False, out_state=None):
    dev = x.device
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    s = _scan_struct(x, dt, A, B, Cm, skip, z, dt_bias, state, reset, softplus)
    if want_state and out_state is None:
        out_state = torch.empty((s.R, s.D, s.N), dtype=torch.float32, device=dev)
    lib, ck = N.load(), None
    with _on_device(dev):
        if train:
            n = lib.fdql_scan_checkpoint_floats(C.byref(s))
            if n < 0:
                N.check(int(n))
            ck = torch.empty(n, dtype=torch.float32, device=dev)
        ws = _scratch(lib.fdql_scan_workspace_bytes(C.byref(s), 0), dev) if s.T > 1 else None
        s.y, s.state_out, s.checkpoints = _p(y), _p(out_state), _p(ck)
        s.workspace, s.workspace_bytes = _p(ws), 0 if ws is None else ws.numel()
        N.check(lib.fdql_scan(C.byref(s), N.current_stream(dev)))
    return (y, out_state, ck) if train else (y, out_state)


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, Cm, skip, z, dt_bias, state, reset, softplus, want_state):
        ctx.set_materialize_grads(False)
        ctx.softplus = softplus
        y, out_state, ck = _scan_forward(x, dt, A, B, Cm, skip, z, dt_bias, state, reset, softplus, want_state, train=True)
        ctx.save_for_backward(x, dt, A, B, Cm, skip, z, dt_bias, state, reset, ck)
        return y, out_state

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate):
        x, dt, A, B, Cm, skip, z, dt_bias, state, reset, ck = ctx.saved_tensors
        need = ctx.needs_input_grad
        dev = x.device
        dy = torch.zeros_like(x, memory_format=torch.contiguous_format) if dy is None else _dense(dy)
        dstate = _whole(dstate)
        new = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=dev)  # noqa: E731
        dx, ddt, dA, dB, dC, dskip, dz, dbias = (new(t) for t in (x, dt, A, B, Cm, skip, z, dt_bias))
        ds = new(state) if need[8] else None
        s = _scan_struct(x, dt, A, B, Cm, skip, z, dt_bias, state, reset, ctx.softplus)
        s.checkpoints = _p(ck)
        s.dy, s.dy_st, s.dy_sr, s.dstate_out = _p(dy), dy.stride(0), dy.stride(1), _p(dstate)
        s.dx, s.ddt, s.dz, s.dB, s.dC = _p(dx), _p(ddt), _p(dz), _p(dB), _p(dC)
        s.dA, s.dskip, s.ddt_bias, s.dstate_in = _p(dA), _p(dskip), _p(dbias), _p(ds)
        lib = N.load()
        with _on_device(dev):
            ws = _scratch(lib.fdql_scan_workspace_bytes(C.byref(s), 1), dev)
            s.workspace, s.workspace_bytes = _p(ws), 0 if ws is None else ws.numel()
            N.check(lib.fdql_scan_backward(C.byref(s), N.current_stream(dev)))
        grads = (dx, ddt, dA, dB, dC, dskip, dz, dbias, ds)
        return tuple(g if n else None for g, n in zip(grads, need)) + (None, None, None)


def _scan_check(what, x, dt, A, B, Cm, skip, z, dt_bias, state, R):
    D = x.shape[-1]
    _need(isinstance(A, torch.Tensor) and A.dim() == 2 and 1 <= A.shape[1] <= 64, f"{what}: A must be [channels, 1..64 states]")
    n = A.shape[1]
    _like(x, f"{what}: A", A, (D, n), torch.float32)
    _like(x, f"{what}: dt", dt, x.shape)
    _need(isinstance(B, torch.Tensor) and B.dim() in (x.dim(), x.dim() + 1), f"{what}: B must be [{'T, ' if x.dim() == 3 else ''}rows, (groups,) states]")
    if B.dim() == x.dim():
        B, Cm = B.unsqueeze(-2), Cm.unsqueeze(-2)
    G = B.shape[-2]
    _need(G >= 1 and D % G == 0, f"{what}: {G} groups do not divide {D} channels")
    _like(x, f"{what}: B", B, (*x.shape[:-1], G, n))
    _like(x, f"{what}: C", Cm, (*x.shape[:-1], G, n))
    if z is not None:
        _like(x, f"{what}: z", z, x.shape)
    for name, t in (("skip", skip), ("dt_bias", dt_bias)):
        if t is not None:
            _like(x, f"{what}: {name}", t, (D,), torch.float32)
    if state is not None:
        _like(x, f"{what}: state", state, (R, D, n), torch.float32)
    return B, Cm


def selective_scan(x, dt, A, B, C, *, skip=None, z=None, dt_bias=None, dt_softplus=True, reset=None, initial_state=None, return_state=False):
    """h_t = exp(delta_t A) h_{t-1} + delta_t x_t B_t,  y_t = (C_t . h_t + skip x_t) SiLU(z_t),  delta_t = softplus(dt_t + dt_bias).

    x, dt, z [T, rows, D]; A [D, n] float32 (1..64 states); B, C [T, rows, n] or [T, rows, groups, n], group g serving the
    channels [g D / groups, (g + 1) D / groups); skip, dt_bias [D] float32; reset [T, rows]; initial_state [rows, D, n] float32 (default zeros).
    Returns y, or (y, state after the last step) when return_state."""
    _head("selective_scan", x, 3)
    B, C = _scan_check("selective_scan", x, dt, A, B, C, skip, z, dt_bias, initial_state, x.shape[1])
    reset = _reset_of(x, reset, x.shape[:2])
    args = (_dense(x), _dense(dt), _whole(A), _dense(B), _dense(C), _whole(skip), _dense(z), _whole(dt_bias), _rows_dense(initial_state), reset,
            bool(dt_softplus), bool(return_state))
    graded = _graded(x, dt, A, B, C, skip, z, dt_bias, initial_state)
    y, state = _Scan.apply(*args) if graded else _scan_forward(*args)
    return (y, state) if return_state else y


def selective_scan_step(x, dt, A, B, C, state, *, skip=None, z=None, dt_bias=None, dt_softplus=True, reset=None, out_state=None):
    """One step of selective_scan for every row: x, dt, z [rows, D], B, C [rows, (groups,) n], state [rows, D, n], reset [rows].  Returns
    (y, new state); the new state is written to out_state (dense; `state` itself updates it in place) or to a new tensor."""
    _head("selective_scan_step", x, 2)
    B, C = _scan_check("selective_scan_step", x, dt, A, B, C, skip, z, dt_bias, state, x.shape[0])
    _need(state is not None, "selective_scan_step: a state is needed")
    _no_grad_inputs("selective_scan_step", x, dt, A, B, C, skip, z, dt_bias, state)
    if out_state is not None:
        _like(x, "selective_scan_step: out_state", out_state, state.shape, torch.float32)
        _need(out_state.is_contiguous(), "selective_scan_step: out_state must be contiguous")
    return _scan_forward(_dense(x), _dense(dt), _whole(A), _dense(B), _dense(C), _whole(skip), _dense(z), _whole(dt_bias), _rows_dense(state),
                         _reset_of(x, reset, x.shape[:1]), bool(dt_softplus), True, False, out_state)


# ------------------------------------------------------------------------------------------------------------------ gated
def _gated_struct(x, w_gate, w_up, b_gate, b_up, act):
    s = N.Gated()
    s.size, s.dtype = C.sizeof(N.Gated), _TYPES[x.dtype]
    s.M, s.D = x.shape
    s.F, s.act = w_gate.shape[0], act
    s.x, s.x_sr = _p(x), x.stride(0)
    s.w_gate, s.w_up, s.b_gate, s.b_up = _p(w_gate), _p(w_up), _p(b_gate), _p(b_up)
    return s


def _gated_forward(x, w_gate, w_up, b_gate, b_up, act, train=False):
    dev = x.device
    y = torch.empty((x.shape[0], w_gate.shape[0]), dtype=x.dtype, device=dev)
    pre = torch.empty((2, *y.shape), dtype=torch.float32, device=dev) if train else None
    s = _gated_struct(x, w_gate, w_up, b_gate, b_up, act)
    s.y, s.pre = _p(y), _p(pre)
    lib = N.load()
    with _on_device(dev):
        ws = _scratch(lib.fdql_gated_workspace_bytes(C.byref(s), 0), dev)
        s.workspace, s.workspace_bytes = _p(ws), 0 if ws is None else ws.numel()
        N.check(lib.fdql_gated(C.byref(s), N.current_stream(dev)))
    return (y, pre) if train else y


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        ctx.act = act
        y, pre = _gated_forward(x, w_gate, w_up, b_gate, b_up, act, train=True)
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up, pre)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w_gate, w_up, b_gate, b_up, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dev = x.device
        dy = _dense(dy)
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[0] else None
        dwg, dwu = (torch.empty_like(w_gate), torch.empty_like(w_up)) if need[1] or need[2] else (None, None)
        dbg, dbu = (torch.empty_like(b_gate), torch.empty_like(b_up)) if need[3] or need[4] else (None, None)
        s = _gated_struct(x, w_gate, w_up, b_gate, b_up, ctx.act)
        s.pre, s.dy, s.dy_sr = _p(pre), _p(dy), dy.stride(0)
        s.dx, s.dw_gate, s.dw_up, s.db_gate, s.db_up = _p(dx), _p(dwg), _p(dwu), _p(dbg), _p(dbu)
        lib = N.load()
        with _on_device(dev):
            ws = _scratch(lib.fdql_gated_workspace_bytes(C.byref(s), 1), dev)
            s.workspace, s.workspace_bytes = _p(ws), 0 if ws is None else ws.numel()
            N.check(lib.fdql_gated_backward(C.byref(s), N.current_stream(dev)))
        return tuple(g if n else None for g, n in zip((dx, dwg, dwu, dbg, dbu), need)) + (None,)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, *, activation="silu"):
    """f(x w_gate^T + b_gate) * (x w_up^T + b_up), f = "silu", "gelu" (erf form) or "sigmoid".

    x [..., D], weights [F, D], biases [F] (both or neither), all of one type; returns [..., F].  Sums are float32; the backward pass rounds
    the two pre-activation gradients once to the type before its products."""
    _need(isinstance(x, torch.Tensor) and x.dim() >= 1, "gated_linear: x must be a tensor [..., channels]")
    _head("gated_linear", x, x.dim())
    _need(activation in _ACTS, f"gated_linear: activation must be one of {sorted(_ACTS)}, got {activation!r}")
    _need(isinstance(w_gate, torch.Tensor) and w_gate.dim() == 2 and w_gate.shape[0] >= 1, "gated_linear: w_gate must be [features, channels]")
    F, D = w_gate.shape[0], x.shape[-1]
    _like(x, "gated_linear: w_gate", w_gate, (F, D))
    _like(x, "gated_linear: w_up", w_up, (F, D))
    _need((b_gate is None) == (b_up is None), "gated_linear: both biases or neither")
    for name, t in (("b_gate", b_gate), ("b_up", b_up)):
        if t is not None:
            _like(x, f"gated_linear: {name}", t, (F,))
    lead = x.shape[:-1]
    args = (_dense(x.reshape(-1, D)), _whole(w_gate), _whole(w_up), _whole(b_gate), _whole(b_up), _ACTS[activation])
    y = _Gated.apply(*args) if _graded(x, w_gate, w_up, b_gate, b_up) else _gated_forward(*args)
    return y.view(*lead, F)
