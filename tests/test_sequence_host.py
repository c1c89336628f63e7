"""The sequence operators without a GPU: their 64-bit definitions against differences, and every refusal that the host makes."""
import ctypes as C

import pytest
import torch

from fastdeepqlearning_amd import _native as nat
from fastdeepqlearning_amd import sequence as seq
from oracle import sequence as osq


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float64)


def _difference_check(fn, inputs, grads, seed):
    """Directional derivatives of sum(outputs * cotangents) against the hand-written adjoints."""
    g = torch.Generator().manual_seed(seed)
    for name, t in inputs.items():
        d = _rand(g, *t.shape)
        eps = 1e-6
        up, down = fn({**inputs, name: t + eps * d}), fn({**inputs, name: t - eps * d})
        num = (up - down) / (2 * eps)
        ana = float((grads[name] * d).sum())
        assert abs(num - ana) <= 1e-6 * max(1.0, abs(ana)), (name, num, ana)


@pytest.mark.parametrize("T,K,reset", [(1, 2, False), (2, 4, False), (7, 3, True), (6, 4, True)])
def test_conv_definition_against_differences(T, K, reset):
    g = torch.Generator().manual_seed(T * 10 + K)
    R, D = 2, 3
    inp = dict(x=_rand(g, T, R, D), weight=_rand(g, D, K), bias=_rand(g, D), state=_rand(g, R, K - 1, D))
    rst = (torch.rand(T, R, generator=g) < 0.3) if reset else None
    dy, ds = _rand(g, T, R, D), _rand(g, R, K - 1, D)
    o = osq.causal_conv(**inp, reset=rst, dy=dy, dstate=ds)

    def fn(i):
        r = osq.causal_conv(**i, reset=rst)
        return float((r["y"] * dy).sum() + (r["state"] * ds).sum())
    _difference_check(fn, inp, {"x": o["dx"], "weight": o["dweight"], "bias": o["dbias"], "state": o["dstate"]}, 1)


@pytest.mark.parametrize("T,G,reset,softplus", [(1, 1, False, True), (5, 2, True, True), (6, 1, True, False)])
def test_scan_definition_against_differences(T, G, reset, softplus):
    g = torch.Generator().manual_seed(T * 10 + G)
    R, D, N = 2, 4, 3
    inp = dict(x=_rand(g, T, R, D), dt=_rand(g, T, R, D), A=-torch.rand(D, N, generator=g, dtype=torch.float64) - 0.1, B=_rand(g, T, R, G, N),
               C=_rand(g, T, R, G, N), skip=_rand(g, D), z=_rand(g, T, R, D), dt_bias=_rand(g, D), state=_rand(g, R, D, N))
    rst = (torch.rand(T, R, generator=g) < 0.3) if reset else None
    dy, ds = _rand(g, T, R, D), _rand(g, R, D, N)
    o = osq.selective_scan(**inp, softplus=softplus, reset=rst, dy=dy, dstate=ds)

    def fn(i):
        r = osq.selective_scan(**i, softplus=softplus, reset=rst)
        return float((r["y"] * dy).sum() + (r["state"] * ds).sum())
    _difference_check(fn, inp, {k: o["d" + k] for k in inp}, 2)


@pytest.mark.parametrize("kind", ["silu", "gelu", "sigmoid"])
def test_gated_definition_against_differences(kind):
    g = torch.Generator().manual_seed(3)
    inp = dict(x=_rand(g, 5, 4), w_gate=_rand(g, 3, 4), w_up=_rand(g, 3, 4), b_gate=_rand(g, 3), b_up=_rand(g, 3))
    dy = _rand(g, 5, 3)
    o = osq.gated_linear(**inp, kind=kind, dy=dy)
    _difference_check(lambda i: float((osq.gated_linear(**i, kind=kind)["y"] * dy).sum()), inp, {k: o["d" + k] for k in inp}, 4)


def test_calls_refuse_cpu_tensors():
    """No CPU path: the calls raise on host tensors."""
    x, w = torch.zeros(2, 1, 4), torch.zeros(4, 2)
    with pytest.raises(ValueError, match="GPU"):
        seq.causal_conv(x, w)
    with pytest.raises(ValueError, match="GPU"):
        seq.causal_conv_step(x[0], torch.zeros(1, 1, 4), w)
    with pytest.raises(ValueError, match="GPU"):
        seq.selective_scan(x, x, torch.zeros(4, 2), torch.zeros(2, 1, 2), torch.zeros(2, 1, 2))
    with pytest.raises(ValueError, match="GPU"):
        seq.selective_scan_step(x[0], x[0], torch.zeros(4, 2), torch.zeros(1, 2), torch.zeros(1, 2), torch.zeros(1, 4, 2))
    with pytest.raises(ValueError, match="GPU"):
        seq.gated_linear(x, torch.zeros(3, 4), torch.zeros(3, 4))


def _conv(**kw):
    s = nat.CausalConv()
    s.size, s.dtype, s.T, s.R, s.D, s.K = C.sizeof(s), 0, 4, 2, 8, 4
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _scan(**kw):
    s = nat.Scan()
    s.size, s.dtype, s.T, s.R, s.D, s.N, s.G = C.sizeof(s), 0, 4, 2, 8, 4, 1
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _gated(**kw):
    s = nat.Gated()
    s.size, s.dtype, s.M, s.D, s.F = C.sizeof(s), 0, 4, 8, 8
    for k, v in kw.items():
        setattr(s, k, v)
    return s


P = 4096    # a pointer that the refused call never follows


@pytest.mark.parametrize("entry,make,bad,word", [
    ("fdql_causal_conv", _conv, dict(size=8), "size"), ("fdql_causal_conv", _conv, dict(dtype=1), "dtype"), ("fdql_causal_conv", _conv, dict(K=1), "taps"),
    ("fdql_causal_conv", _conv, dict(K=5), "taps"), ("fdql_causal_conv", _conv, dict(T=-1), "T -1"), ("fdql_causal_conv", _conv, dict(D=0), "D 0"),
    ("fdql_causal_conv", _conv, dict(), "needed"), ("fdql_causal_conv", _conv, dict(T=2**31 - 1, R=2**20, D=4096), "one launch"),
    ("fdql_causal_conv", _conv, dict(x=P, weight=P, y=P, state_in=P, state_out=P), "in place"),
    ("fdql_causal_conv_backward", _conv, dict(x=P, weight=P, dy=P), "workspace"), ("fdql_causal_conv_backward", _conv, dict(x=P, dy=P), "needed"),
    ("fdql_scan", _scan, dict(size=8), "size"), ("fdql_scan", _scan, dict(dtype=7), "dtype"), ("fdql_scan", _scan, dict(N=65), "states"),
    ("fdql_scan", _scan, dict(N=0), "states"), ("fdql_scan", _scan, dict(G=3), "groups"), ("fdql_scan", _scan, dict(R=-1), "R -1"), ("fdql_scan", _scan, dict(), "needed"),
    ("fdql_scan", _scan, dict(R=2**30), "one launch"), ("fdql_scan", _scan, dict(state_in=P, state_out=P), "in place"),
    ("fdql_scan", _scan, dict(T=4096, x=P, dt=P, A=P, B=P, C=P, y=P), "workspace"),
    ("fdql_scan_backward", _scan, dict(x=P, dt=P, A=P, B=P, C=P, dy=P), "checkpoints"),
    ("fdql_scan_backward", _scan, dict(x=P, dt=P, A=P, B=P, C=P, dy=P, checkpoints=P), "dx, ddt"),
    ("fdql_scan_backward", _scan, dict(x=P, dt=P, A=P, B=P, C=P, dy=P, checkpoints=P, dx=P, ddt=P, dA=P, dB=P, dC=P, workspace=8, workspace_bytes=1 << 30), "workspace"),
    ("fdql_gated", _gated, dict(size=8), "size"), ("fdql_gated", _gated, dict(dtype=1), "dtype"), ("fdql_gated", _gated, dict(act=3), "activation"),
    ("fdql_gated", _gated, dict(M=-1), "M -1"), ("fdql_gated", _gated, dict(M=1 << 40), "one launch"), ("fdql_gated", _gated, dict(), "needed"),
    ("fdql_gated", _gated, dict(x=P, w_gate=P, w_up=P, y=P, b_up=P), "biases"), ("fdql_gated_backward", _gated, dict(dw_up=P), "together"),
    ("fdql_gated_backward", _gated, dict(x=P, w_gate=P, w_up=P, dy=P), "pre"), ("fdql_gated_backward", _gated, dict(x=P, w_gate=P, w_up=P, dy=P, pre=P), "workspace"),
])
def test_c_abi_refuses(entry, make, bad, word):
    """A refused call returns FDQL_EINVAL with a message before anything reaches the device."""
    lib = nat.load()
    rc = getattr(lib, entry)(C.byref(make(**bad)), None)
    assert rc == nat.FDQL_EINVAL
    assert word in lib.fdql_last_error().decode()


def test_workspace_queries():
    """Sizes grow with the problem, need no pointers, take empty problems and refuse bad ones."""
    lib = nat.load()
    assert lib.fdql_scan_checkpoint_floats(C.byref(_scan(T=0))) == 0
    assert lib.fdql_scan_checkpoint_floats(C.byref(_scan(T=9))) == 2 * lib.fdql_scan_checkpoint_floats(C.byref(_scan(T=8)))
    assert lib.fdql_scan_workspace_bytes(C.byref(_scan()), 0) == 0 < lib.fdql_scan_workspace_bytes(C.byref(_scan()), 1)
    assert lib.fdql_scan_workspace_bytes(C.byref(_scan(T=4096)), 0) > 0
    for s in (_scan(R=0, T=500), _scan(T=0)):
        assert lib.fdql_scan_workspace_bytes(C.byref(s), 1) >= 0
    assert lib.fdql_causal_conv_workspace_bytes(C.byref(_conv())) > 0
    assert lib.fdql_causal_conv_workspace_bytes(C.byref(_conv(R=0))) >= 0
    assert lib.fdql_gated_workspace_bytes(C.byref(_gated()), 0) == 0 < lib.fdql_gated_workspace_bytes(C.byref(_gated()), 1)
    assert lib.fdql_gated_workspace_bytes(C.byref(_gated(M=0)), 1) >= 0
    assert lib.fdql_scan_workspace_bytes(C.byref(_scan(N=99)), 1) == nat.FDQL_EINVAL
    assert lib.fdql_causal_conv_workspace_bytes(C.byref(_conv(K=9))) == nat.FDQL_EINVAL
    assert lib.fdql_gated_workspace_bytes(C.byref(_gated(F=0)), 1) == nat.FDQL_EINVAL


@pytest.mark.parametrize("entry,make,kw,least", [("fdql_causal_conv", _conv, dict(x=P, weight=P, y=P, T=1), 24), ("fdql_scan", _scan, dict(x=P, dt=P, A=P, B=P, C=P, y=P, T=1), 32)])
def test_state_rows_that_would_overlap_are_refused(entry, make, kw, least):
    """A row stride of state_out below a row's length (0: every row in one place) would let rows overwrite each other."""
    lib = nat.load()
    for sr in (0, least - 1, -least):
        assert getattr(lib, entry)(C.byref(make(state_out=P, state_out_sr=sr, **kw)), None) == nat.FDQL_EINVAL
        assert "overlap" in lib.fdql_last_error().decode()


def test_more_channels_than_the_finish_kernels_take_are_refused():
    lib = nat.load()
    assert lib.fdql_scan_workspace_bytes(C.byref(_scan(R=1, D=1 << 22)), 1) == nat.FDQL_EINVAL
    assert "one launch" in lib.fdql_last_error().decode()
    assert lib.fdql_scan_workspace_bytes(C.byref(_scan(R=1, D=1 << 21)), 1) > 0


def test_windows_longer_than_the_step_index_are_refused():
    lib = nat.load()
    assert lib.fdql_scan_workspace_bytes(C.byref(_scan(T=2**31 - 1, R=1, D=1, N=1)), 0) == nat.FDQL_EINVAL
    assert "2^30" in lib.fdql_last_error().decode()
    assert lib.fdql_scan_workspace_bytes(C.byref(_scan(T=2**30, R=1, D=1, N=1)), 0) > 0
