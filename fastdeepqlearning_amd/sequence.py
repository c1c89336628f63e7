"""Sequence operators over time-major windows [T, rows, channels], on the C ABI's ``fdql_causal_conv`` / ``fdql_scan`` / ``fdql_gated``
(include/fdql.h) - the pieces of a recurrent block beside the reference's GRU (franQ/Agent/components/encoder.py:40-42, 78-94):

    from fastdeepqlearning_amd import sequence as seq
    x = seq.causal_conv(x, w, b, reset=reset)                     # short convolution + SiLU
    y = seq.selective_scan(x, dt, A, B, C, skip=d, z=z, dt_bias=bias, reset=reset)
    h = seq.gated_linear(y, w_gate, w_up, b_gate, b_up)           # SiLU(y Wg^T + bg) * (y Wu^T + bu)

Each is differentiable (once, in reverse mode: a second derivative and a forward-mode tangent raise); ``causal_conv_step`` and ``selective_scan_step`` advance every acting row by one step.  Activations
may be float32, bfloat16 or float16 and any strided view (a copy is made only where the last dimension is not dense); states of the scan,
its A / skip / dt_bias and the convolution's weights are float32.  ``reset`` [T, rows] (bool or uint8) marks the steps at which a new sequence
begins: several sequences can share a row, and left padding is dropped by a reset at the first real step.  Calls run on the current
stream of the tensors' device, never synchronise, and can be captured into a graph (a captured backward pass raises while an eager graph of the same
leaves is alive on the default stream); tracers (torch.jit.trace, make_fx, fake tensors) cannot see them, and the calls raise there.  Wrong types, shapes or devices raise ValueError, a failed
launch FdqlError.  All compute is in libfdql_hip.so; there is no CPU path."""
import ctypes as C

from . import _native as N

__all__ = ["causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "gated_linear"]

_ACTS = {"silu": 0, "gelu": 1, "sigmoid": 2}
_ROUND_GRADS = 0x100
_bound = None


def _ops():
    """The torch binding (csrc/torch_bind.cpp) on the loaded library; raises NativeLibraryMissing."""
    global _bound
    if _bound is None:
        lib = N.load()
        try:
            from . import _seq_torch
        except ImportError as e:
            raise N.NativeLibraryMissing("fastdeepqlearning_amd/_seq_torch.so is missing or does not load: build it with "
                                         "`make -C fastdeepqlearning_amd/csrc`. There is no Python fallback.") from e
        names = [n for n in N.SIGNATURES if n.startswith(("fdql_causal_conv", "fdql_scan", "fdql_gated", "fdql_last_error"))]
        _seq_torch.bind({n: C.cast(getattr(lib, n), C.c_void_p).value for n in names}, N.FdqlError)
        _bound = _seq_torch
    return _bound


def causal_conv(x, weight, bias=None, *, reset=None, initial_state=None, silu=True, return_state=False):
    """y_t = f(bias + sum_j weight[:, K-1-j] * x_{t-j}), f = SiLU (or identity), channel by channel.

    x [T, rows, D]; weight [D, K] (K = 2..4) and bias [D] float32; reset [T, rows]; initial_state [rows, K-1, D] in x's type, the
    inputs before step 0, oldest first (default zeros).  Returns y, or (y, state) with the last K-1 inputs when return_state."""
    y, state = (_bound or _ops()).causal_conv(x, weight, bias, reset, initial_state, silu, return_state)
    return (y, state) if return_state else y


def causal_conv_step(x, state, weight, bias=None, *, reset=None, silu=True, out_state=None):
    """One step of causal_conv for every row: x [rows, D], state [rows, K-1, D], reset [rows].  Returns (y, new state); the new state is
    written to out_state (rows dense, any distance apart; `state` itself updates it in place, rows that overlap in another way are
    refused) or to a new tensor."""
    return (_bound or _ops()).causal_conv_step(x, state, weight, bias, reset, silu, out_state)


def selective_scan(x, dt, A, B, C, *, skip=None, z=None, dt_bias=None, dt_softplus=True, reset=None, initial_state=None, return_state=False):
    """h_t = exp(delta_t A) h_{t-1} + delta_t x_t B_t,  y_t = (C_t . h_t + skip x_t) SiLU(z_t),  delta_t = softplus(dt_t + dt_bias).

    x, dt, z [T, rows, D]; A [D, n] float32 (1..64 states); B, C [T, rows, n] or [T, rows, groups, n], group g serving the
    channels [g D / groups, (g + 1) D / groups); skip, dt_bias [D] float32; reset [T, rows]; initial_state [rows, D, n] float32 (default zeros).
    Returns y, or (y, state after the last step) when return_state."""
    y, state = (_bound or _ops()).selective_scan(x, dt, A, B, C, skip, z, dt_bias, dt_softplus, reset, initial_state, return_state)
    return (y, state) if return_state else y


def selective_scan_step(x, dt, A, B, C, state, *, skip=None, z=None, dt_bias=None, dt_softplus=True, reset=None, out_state=None):
    """One step of selective_scan for every row: x, dt, z [rows, D], B, C [rows, (groups,) n], state [rows, D, n], reset [rows].  Returns
    (y, new state); the new state is written to out_state (rows dense, any distance apart; `state` itself
    updates it in place, rows that overlap in another way are refused) or to a new tensor."""
    return (_bound or _ops()).selective_scan_step(x, dt, A, B, C, state, skip, z, dt_bias, dt_softplus, reset, out_state)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, *, activation="silu", rounded_grads=False):
    """f(x w_gate^T + b_gate) * (x w_up^T + b_up), f = "silu", "gelu" (erf form) or "sigmoid".

    x [..., D], weights [F, D], biases [F] (both or neither), all of one type; returns [..., F].  Sums are float32.  The backward pass of
    the 16-bit types keeps the two pre-activation gradients in two parts of the type, so that the gradients are rounded once, at the end;
    rounded_grads=True rounds them before its products too, which halves the products' work and makes the gradients' error about sqrt(2) times as
    large.  In float16 a pre-activation gradient beyond 65504 counts as infinite (choose the loss scale for it)."""
    act = _ACTS.get(activation)
    if act is None:
        raise ValueError(f"gated_linear: activation must be one of {sorted(_ACTS)}, got {activation!r}")
    return (_bound or _ops()).gated_linear(x, w_gate, w_up, b_gate, b_up, act | (_ROUND_GRADS if rounded_grads else 0))
