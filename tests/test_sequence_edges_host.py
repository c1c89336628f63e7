"""The sequence operators without a GPU: options, refusals and bookkeeping that their callers rely on at the edges."""
import ctypes as C

import pytest
import torch

from fastdeepqlearning_amd import _native as nat
from fastdeepqlearning_amd import sequence as seq
from test_sequence_host import P, _conv, _gated, _scan

ROUND = 0x100      # FDQL_GATED_ROUND_GRADS


def test_gated_gradient_parts_are_the_callers_choice():
    """16-bit types hold the gradients in front of the products in two parts at every size, in one where the caller says so; float has one part."""
    lib = nat.load()
    need = lambda **kw: lib.fdql_gated_workspace_bytes(C.byref(_gated(**kw)), 1)  # noqa: E731
    for M, D, F in ((4, 8, 8), (60, 128, 136), (70, 128, 136), (5000, 136, 1032), (8192, 1024, 4096)):
        for dtype in (2, 3):
            assert need(dtype=dtype, M=M, D=D, F=F) - need(dtype=dtype, M=M, D=D, F=F, act=ROUND) == 2 * 2 * M * F     # dg and du once more
        assert need(dtype=0, M=M, D=D, F=F) == need(dtype=0, M=M, D=D, F=F, act=ROUND)
    for act in (ROUND | 3, ROUND << 1, -1):
        assert lib.fdql_gated(C.byref(_gated(act=act, x=P, w_gate=P, w_up=P, y=P)), None) == nat.FDQL_EINVAL
        assert "activation" in lib.fdql_last_error().decode()


def _calls(seq, lift=lambda t: t):
    """name -> the five calls on small CPU tensors, every floating-point argument in turn passed through `lift`."""
    z = lambda *s: torch.ones(*s)  # noqa: E731
    forms = {
        "causal_conv": ([z(2, 1, 4), z(4, 2), z(4)], lambda a: seq.causal_conv(*a)),
        "causal_conv with a state": ([z(2, 1, 4), z(4, 2), z(1, 1, 4)], lambda a: seq.causal_conv(a[0], a[1], initial_state=a[2])),
        "causal_conv_step": ([z(1, 4), z(1, 1, 4), z(4, 2), z(4), z(1, 1, 4)], lambda a: seq.causal_conv_step(*a[:4], out_state=a[4])),
        "selective_scan": ([z(2, 1, 4), z(2, 1, 4), z(4, 2), z(2, 1, 2), z(2, 1, 2), z(4), z(2, 1, 4), z(4), z(1, 4, 2)],
                           lambda a: seq.selective_scan(*a[:5], skip=a[5], z=a[6], dt_bias=a[7], initial_state=a[8])),
        "selective_scan_step": ([z(1, 4), z(1, 4), z(4, 2), z(1, 2), z(1, 2), z(1, 4, 2), z(4), z(1, 4), z(4), z(1, 4, 2)],
                                lambda a: seq.selective_scan_step(*a[:6], skip=a[6], z=a[7], dt_bias=a[8], out_state=a[9])),
        "gated_linear": ([z(2, 4), z(3, 4), z(3, 4), z(3), z(3)], lambda a: seq.gated_linear(*a)),
    }
    for name, (args, call) in forms.items():
        for k in range(len(args)):
            yield f"{name}, argument {k}", lambda: call([lift(t) if j == k else t for j, t in enumerate(args)])  # noqa: B023


def test_forward_mode_tangents_are_refused():
    """A dual tensor in any place raises; the result would have no tangent."""
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        for name, call in _calls(seq, lambda t: fwad.make_dual(t, torch.ones_like(t))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
                pytest.fail(name)


def test_tracing_is_refused():
    """A trace would hold uninitialised results: jit and fx tracers and fake tensors raise."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    seen = set()
    for name, call in _calls(seq):
        if name.split(",")[0] in seen:
            continue
        seen.add(name.split(",")[0])
        for trace in (lambda f: torch.jit.trace(f, torch.ones(1), check_trace=False), lambda f: make_fx(f)(torch.ones(1)),
                      lambda f: make_fx(f, tracing_mode="fake")(torch.ones(1))):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                trace(lambda a: call())  # noqa: B023
        with FakeTensorMode(), pytest.raises(RuntimeError, match="cannot be traced"):
            call()
    assert len(seen) == 6


class _Wrapped(torch.Tensor):
    """A tensor without memory of its own, as distributed and quantised tensors are."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} was called")


def test_wrapper_tensors_are_refused():
    """In any place: their data pointer is null.  A plain subclass, which has memory, gets as far as every other tensor."""
    for name, call in _calls(seq, _Wrapped):
        with pytest.raises(ValueError, match="plain tensors"):
            call()
            pytest.fail(name)
    with pytest.raises(ValueError, match="GPU"):
        seq.gated_linear(torch.nn.Parameter(torch.ones(2, 4)), torch.ones(3, 4), torch.ones(3, 4))


def test_functional_transforms_are_refused():
    w = torch.ones(3, 4)
    for transform in (torch.vmap, torch.func.grad):
        with pytest.raises(ValueError, match="plain tensors"):
            transform(lambda a: seq.gated_linear(a, w, w).sum())(torch.ones(2, 2, 4))


class _Looks(torch.autograd.Function):
    """Identity whose backward pass notes what the binding sees ahead of it."""
    seen = []

    @staticmethod
    def forward(ctx, *xs):
        return sum(x.sum() for x in xs)

    @staticmethod
    def backward(ctx, g):
        _Looks.seen.append(sorted(seq._ops().nodes_ahead()))
        return tuple(g.expand(6) for _ in ctx.needs_input_grad)


def _ahead(run):
    _Looks.seen = []
    run()
    return _Looks.seen[0]


def test_nodes_that_a_backward_pass_will_run():
    """What a captured backward pass is checked against: leaves behind views and behind other operators, each once, nothing that the pass leaves out."""
    leaf, other = torch.ones(2, 3, requires_grad=True), torch.ones(6, requires_grad=True)
    acc = "torch::autograd::AccumulateGrad"
    assert _ahead(lambda: _Looks.apply(other).backward()) == [acc]                                                            # a leaf itself
    assert _ahead(lambda: _Looks.apply(leaf.view(6)).backward()) == sorted(["ViewBackward0", acc])                            # a leaf behind a view
    deep = (leaf * 2).view(6).exp()
    assert _ahead(lambda: _Looks.apply(deep, deep).backward()) == sorted(["ExpBackward0", "ViewBackward0", "MulBackward0", acc])      # node -> node -> leaf, met twice
    both = lambda: _Looks.apply(leaf.view(6), other.exp())  # noqa: E731
    assert _ahead(lambda: both().backward()) == sorted(["ViewBackward0", "ExpBackward0", acc, acc])
    assert _ahead(lambda: torch.autograd.grad(both(), [leaf])) == sorted(["ViewBackward0", acc])                              # chosen inputs: their way only
    assert _ahead(lambda: torch.autograd.grad(both(), [other])) == sorted(["ExpBackward0", acc])
    middle = leaf.view(6)
    assert _ahead(lambda: torch.autograd.grad(_Looks.apply(middle.exp()), [middle])) == ["ExpBackward0", "ViewBackward0"]     # (stops at the input's own node)
    assert seq._ops().nodes_ahead() == []                                                                                     # outside a pass


@pytest.mark.parametrize("entry,make,kw,row", [("fdql_causal_conv", _conv, dict(x=P, weight=P, y=P), 24 * 4), ("fdql_causal_conv", _conv, dict(x=P, weight=P, y=P, dtype=2), 24 * 2),
                                               ("fdql_scan", _scan, dict(x=P, dt=P, A=P, B=P, C=P, y=P), 32 * 4)])
def test_states_that_share_memory_are_refused(entry, make, kw, row):
    """Rows of the new state on top of other rows or of parts of rows of the old one; columns side by side in one buffer get past this check (and are
    refused for what else this struct lacks, before anything is launched)."""
    lib, esz = nat.load(), 2 if kw.get("dtype") else 4
    base = 1 << 20

    def call(off, so, si, T=1, **more):
        s = make(state_in=base, state_in_sr=si // esz, state_out=base + off, state_out_sr=so // esz, T=T, **{**kw, **more})
        assert getattr(lib, entry)(C.byref(s), None) == nat.FDQL_EINVAL
        return lib.fdql_last_error().decode()
    for off, so, si in ((esz, row, row), (-esz, row, row), (row, row, row), (esz, 3 * row, 3 * row), (2 * row + esz, 3 * row, 3 * row), (row, 2 * row, row), (0, row, 0), (row - esz, row, 0)):
        if off == 0 and so != si:
            assert "row stride" in call(off, so, si)
        else:
            assert "overlaps" in call(off, so, si) and "overlaps" in call(off, so, si, T=4), (off, so, si)
    missing = {"fdql_causal_conv": dict(x=None), "fdql_scan": dict(x=None)}[entry]
    for off, so, si in ((2 * row, row, row), (row, 3 * row, 3 * row), (-row, 3 * row, 3 * row), (2 * row, 3 * row, 3 * row), (row, row, 0)):
        assert "overlap" not in call(off, so, si, **missing), (off, so, si)
