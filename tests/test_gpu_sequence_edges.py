"""The sequence operators on the GPU at the edges of what their documentation allows, against the 64-bit definitions of oracle/sequence.py."""
import pytest
import torch

from oracle import sequence as osq
from test_gpu_sequence import TYPES, U32, _gated_inputs, _gen, _near, _scan_call, _scan_inputs, dev, seq   # noqa: F401  (dev, seq: fixtures)

pytestmark = pytest.mark.gpu


def _norm_ratio(got, want):
    """Error's norm over that of rounding the exact values once."""
    once = (want.to(got.dtype).double() - want).norm()
    return float((got.detach().cpu().double() - want).norm() / once)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=["bf16", "f16"])
@pytest.mark.parametrize("M,D,F", [(60, 128, 136), (70, 128, 136), (300, 101, 99), (2000, 136, 200), (5000, 136, 1030), (1200, 776, 2050)])
def test_gated_gradients_round_once_at_every_size(dev, seq, M, D, F, dtype):
    """The gradients' error is that of one rounding whatever the size.  The error's mean square over n values scatters by 1 / sqrt(n) (a rounding error is
    uniform), n at least 7680 here: six of these are 7% of it, 3.5% of the norm; the float sums are off by 2^-24 sqrt(terms) of the terms' norm, at
    most 2^-18 against a rounding of 2^-9 / 2 and 2^-12 / 2 (and fp16's smallest step, 2^-24, against values near 1).  1.05 holds both.  With one part
    for d the products' terms are off by as much again: sqrt(2), within the same scatter and what fp16's subnormal numbers add."""
    x, wg, wu, _, _, dy = _gated_inputs(dev, M, D, F, dtype, False, seed=M)
    o = osq.gated_linear(x, wg, wu, None, None, "silu", dy)
    ratio = {}
    for rounded in (False, True):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
        y = seq.gated_linear(*leaves, rounded_grads=rounded)
        grads = torch.autograd.grad(y, leaves, dy)
        ratio[rounded] = [_norm_ratio(got, o[name]) for name, got in zip(("dx", "dw_gate", "dw_up"), grads)]
    print(M, D, F, dtype, ratio)
    assert max(ratio[False]) <= 1.05, ratio
    assert max(ratio[True]) <= 1.6 and min(ratio[True]) > 1.1, ratio


def _graded_calls(dev, seq):
    """(operator, output, leaves) of the three operators on small inputs."""
    g = _gen(3)
    r = lambda *s: torch.randn(*s, generator=g).to(dev).requires_grad_()  # noqa: E731
    x, w, b, st = r(5, 2, 8), r(8, 4), r(8), r(2, 3, 8)
    yield "causal_conv", seq.causal_conv(x, w, b, initial_state=st), [x, w, b, st]
    x, dt, A, B, C, h = r(5, 2, 8), r(5, 2, 8), (-torch.rand(8, 4, generator=g)).to(dev).requires_grad_(), r(5, 2, 4), r(5, 2, 4), r(2, 8, 4)
    yield "selective_scan", seq.selective_scan(x, dt, A, B, C, initial_state=h), [x, dt, A, B, C, h]
    x, wg, wu = r(6, 8), r(5, 8), r(5, 8)
    yield "gated_linear", seq.gated_linear(x, wg, wu), [x, wg, wu]


def test_differentiating_a_gradient_raises(dev, seq):
    """A gradient taken with create_graph carries an error, by itself and beside the output in one loss; its values are the ordinary ones."""
    for name, y, leaves in _graded_calls(dev, seq):
        plain = torch.autograd.grad(y.sum(), leaves, retain_graph=True)
        grads = torch.autograd.grad(y.sum(), leaves, create_graph=True)
        for g, p in zip(grads, plain):
            assert g.requires_grad and not p.requires_grad and torch.equal(g.detach(), p)
            with pytest.raises(RuntimeError, match=f"{name} is differentiable once"):
                (y.sum() + g.pow(2).sum()).backward(retain_graph=True)
            with pytest.raises(RuntimeError, match=f"{name} is differentiable once"):
                torch.autograd.grad(g.sum(), leaves, retain_graph=True, allow_unused=True)


def test_views_that_torch_negates_on_reading(dev, seq):
    """The imaginary part of a conjugate view is stored with the other sign: inputs, gradients and states of that kind count with their values."""
    neg = lambda t: torch.complex(torch.zeros_like(t), -t).conj().imag  # noqa: E731
    g = _gen(12)
    r = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    x, w, b, st, dt, A, B, h, wg, wu = r(5, 2, 8), r(8, 4), r(8), r(2, 3, 8), r(5, 2, 8), -r(8, 4).abs(), r(5, 2, 4), r(2, 8, 4), r(6, 8), r(6, 8)
    assert neg(x).is_neg() and torch.equal(neg(x), x)
    calls = [([x, w, b, st], lambda a: seq.causal_conv(a[0], a[1], a[2], initial_state=a[3])), ([x, dt, A, B, h], lambda a: seq.selective_scan(a[0], a[1], a[2], a[3], a[3], initial_state=a[4])),
             ([x, wg, wu], lambda a: seq.gated_linear(*a))]
    for args, call in calls:
        want = call(args)
        assert torch.equal(call([neg(t) for t in args]), want)
        leaves, dy = [t.clone().requires_grad_() for t in args], torch.randn(want.shape, generator=g).to(dev)
        plain = torch.autograd.grad(call(leaves), leaves, dy)
        for a, c in zip(plain, torch.autograd.grad(call([neg(t) for t in leaves]), leaves, neg(dy))):
            assert torch.equal(a, c)
    y, s = seq.causal_conv_step(x[0], st, w, b)
    y2, s2 = seq.causal_conv_step(neg(x[0]), neg(st), w, b)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    with pytest.raises(ValueError, match="out_state"):
        seq.causal_conv_step(x[0], st, w, b, out_state=neg(st))
    with pytest.raises(ValueError, match="out_state"):
        seq.selective_scan_step(x[0], dt[0], A, B[0], B[0], h, out_state=neg(h))


def _relative(name, got, want, steps):
    """Every value within `steps` roundings of float, 2^-24 each, of its own size."""
    off = (got.detach().cpu().double() - want).abs() / want.abs()
    assert off.max() <= steps * U32, f"{name}: {float(off.max() / U32):.1f} roundings at {int(off.argmax())}"


def _sig(v):
    """1 / (1 + e^-v) and 1 / (1 + e^v) in 64 bits, both with all their digits"""
    return torch.where(v >= 0, 1 / (1 + torch.exp(-v)), torch.exp(v) / (1 + torch.exp(v))), torch.where(v >= 0, torch.exp(-v) / (1 + torch.exp(-v)), 1 / (1 + torch.exp(v)))


# float activations far from zero, relative to their own size.  e^-|v| to one step (2 roundings of 2^-24) and its correction's 2, 1 + w 1, the reciprocal 2, the
# product with w 1, two or three more products: 11; the slope's 1 + v c another 2 and the cancellation left at v <= -10 (1 + v c is at least 9 |c| of terms 11 |c|) 1.3 of
# those.  16 holds them.  GELU adds the complementary error function's own error, up to 4 steps = 8 roundings: 24.
@pytest.mark.parametrize("T", [1, 40])
def test_small_conv_outputs_keep_their_digits(dev, seq, T):
    v = -torch.logspace(1, 1.92, T * 3 * 64).view(T, 3, 64)
    x = v.to(dev).requires_grad_()
    w = torch.tensor([[0.0, 1.0]]).expand(64, 2).to(dev)
    y = seq.causal_conv(x, w)
    s, c = _sig(v.double())
    _relative("y", y, v.double() * s, 16)
    _relative("dx", torch.autograd.grad(y, x, torch.ones_like(y))[0], s * (1 + v.double() * c), 16)
    _relative("step", seq.causal_conv_step(x[0].detach(), torch.zeros(3, 1, 64, device=dev), w)[0], (v.double() * s)[0], 16)


@pytest.mark.parametrize("T", [1, 40, 200])
def test_small_scan_gates_keep_their_digits(dev, seq, T):
    v = -torch.logspace(1, 1.92, T * 64).view(T, 1, 64)
    z, one = v.to(dev).requires_grad_(), torch.ones(T, 1, 64, device=dev)
    A, B, skip = -torch.ones(64, 4, device=dev), torch.zeros(T, 1, 4, device=dev), torch.ones(64, device=dev)
    y = seq.selective_scan(one, one, A, B, B, skip=skip, z=z)
    s, c = _sig(v.double())
    _relative("y", y, v.double() * s, 16)
    dz, dx = torch.autograd.grad(seq.selective_scan(one.requires_grad_(), one, A, B, B, skip=skip, z=z), [z, one], torch.ones_like(y))
    _relative("dz", dz, s * (1 + v.double() * c), 16)
    _relative("dx", dx, v.double() * s, 16)
    state = torch.zeros(1, 64, 4, device=dev)
    _relative("step", seq.selective_scan_step(one[0].detach(), one[0].detach(), A, B[0], B[0], state, skip=skip, z=v[0].to(dev))[0], (v.double() * s)[0], 16)


@pytest.mark.parametrize("M", [5, 32, 33, 4000])
@pytest.mark.parametrize("kind", ["silu", "sigmoid", "gelu"])
def test_small_gated_outputs_keep_their_digits(dev, seq, M, kind):
    """One channel is the gate's value, another the constant 1 that the up side reads; sigmoid's slope on both sides."""
    v = -torch.logspace(0.3 if kind == "gelu" else 1, 1.08 if kind == "gelu" else 1.92, M)
    if kind == "sigmoid":
        v[::2] *= -1
    x = torch.stack([v, torch.ones(M), torch.zeros(M), torch.zeros(M)], 1).to(dev).requires_grad_()
    wg, wu = torch.tensor([[1.0, 0, 0, 0]]).to(dev), torch.tensor([[0.0, 1, 0, 0]]).to(dev)
    y = seq.gated_linear(x, wg, wu, activation=kind)
    g = v.double()
    s, c = _sig(g)
    cdf, pdf = 0.5 * torch.erfc(-g / 2 ** 0.5), torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    f, df = {"silu": (g * s, s * (1 + g * c)), "sigmoid": (s, s * c), "gelu": (g * cdf, cdf + g * pdf)}[kind]
    _relative("y", y[:, 0], f, 24 if kind == "gelu" else 16)
    _relative("dx", torch.autograd.grad(y, x, torch.ones_like(y))[0][:, 0], df, 24 if kind == "gelu" else 16)


def _same(name, got, want, rel=1e-3):
    """Infinities and NaN where the definition has them, the rest near (a check of special values: errors are measured elsewhere)."""
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), want.isnan()), f"{name}: NaN in {int((got.isnan() != want.isnan()).sum())} wrong places"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]) and not got[~inf & ~want.isnan()].isinf().any(), f"{name}: infinities"
    ok = want.isfinite()
    assert torch.allclose(got[ok], want[ok], rtol=rel, atol=rel * float(want[ok].abs().max() if ok.any() else 1.0)), name


@pytest.mark.parametrize("T,R,D,G", [(9, 2, 21, 1), (160, 2, 38, 2)])
@pytest.mark.parametrize("N", [1, 3, 4, 5, 7, 8, 12, 16, 20, 32, 33, 64])
@pytest.mark.parametrize("form", ["x", "dt", "dy", "carried", "bare", "nan"])
def test_scan_infinite_values_stay_where_they_are(dev, seq, T, R, D, N, G, form):
    """An infinite input, step, gradient or carried state gives the infinities of the definition and no NaN beside them, in windows (whole and cut into
    segments) and in steps, for every number of states and with channels that leave a wave part empty; a NaN stays in its channel."""
    i, _, dy, _ = _scan_inputs(dev, T, R, D, N, G, torch.float32, "dense", seed=N)
    for k in ("x", "dt", "B", "C", "state"):
        i[k] = i[k].abs() + 0.1
    i["dt"], dy, inf = i["dt"] * 0.2, dy.abs() + 0.1, float("inf")
    i["z"] = None
    i["skip"] = None if form == "bare" else i["skip"].abs() + 0.1
    at = T // 2
    for d in (1, D - 1):         # the last channel is the one that lanes without a channel look at
        if form in ("x", "bare"):
            i["x"][at, 1, d] = inf
        elif form == "dt":
            i["dt"][at, 1, d] = inf
        elif form == "dy":
            dy[at, 1, d] = inf
        elif form == "carried":
            i["state"][1, d] = inf
        else:
            i["x"][at, 1, d] = float("nan")
    o = osq.selective_scan(**i, dy=None if form == "dt" else dy)
    with torch.no_grad():
        y, st = _scan_call(seq, i, None, True, return_state=True)
        h = i["state"]
        for t in range(T if T < 20 else 0):
            yt, h = seq.selective_scan_step(i["x"][t], i["dt"][t], i["A"], i["B"][t], i["C"][t], h, skip=i["skip"], dt_bias=i["dt_bias"])
            _same("step y", yt, o["y"][t])
        _same("y", y, o["y"])
        _same("state", st, o["state"])
        assert T >= 20 or torch.equal(h.isnan(), st.isnan())
    if form == "dt":             # (0 * inf in the definition's own gradients)
        return
    leaves = {k: v.detach().requires_grad_() for k, v in i.items() if v is not None}
    y = _scan_call(seq, {k: leaves.get(k) for k in i}, None, True)
    for k, g in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)):
        _same("d" + k, g, o["d" + k])


@pytest.mark.parametrize("T,N", [(6, 4), (6, 5), (9, 16), (170, 4), (170, 16), (170, 33)])
@pytest.mark.parametrize("form", ["positive A", "negative step"])
def test_scan_growth_beyond_floats_range_ends_at_a_reset(dev, seq, T, N, form):
    """A decay that overflows (positive A, or negative steps without the softplus) is dropped with the state it would multiply: the step that begins a sequence
    has its own input alone, in windows, their segments and backward, and in single steps."""
    R, D = 2, 20
    i, _, dy, _ = _scan_inputs(dev, T, R, D, N, 1, torch.float32, "dense", seed=4)
    i.update(state=None, dt_bias=None, dt=torch.full((T, R, D), 1e-3, device=dev), A=-torch.ones(D, N, device=dev))
    at = [3, T - 2] if T < 20 else [3, 60, T - 2]
    rst = torch.zeros(T, R, dtype=torch.bool, device=dev)
    for t in at:                             # e^(delta A) = e^200 there
        rst[t, 1] = True
        i["dt"][t, 1] = 200.0 if form == "positive A" else -200.0
    if form == "positive A":
        i["A"] = -i["A"]
    args = dict(i, softplus=False, reset=rst, dy=dy)
    o = osq.selective_scan(**args)
    assert all(v.isfinite().all() for v in o.values())
    leaves = {k: v.detach().requires_grad_() for k, v in i.items() if v is not None}
    li = {k: leaves.get(k) for k in i}
    y, st = _scan_call(seq, li, rst, False, return_state=True)
    _same("y", y, o["y"])
    _same("state", st, o["state"])
    for k, g in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)):
        _same("d" + k, g, o["d" + k])
    with torch.no_grad():
        h = torch.zeros(R, D, N, device=dev)
        for t in range(T if T < 20 else 0):
            yt, h = seq.selective_scan_step(i["x"][t], i["dt"][t], i["A"], i["B"][t], i["C"][t], h, skip=i["skip"], z=i["z"][t], dt_softplus=False, reset=rst[t])
            _same("step", yt, o["y"][t])


def test_join_of_segments_whose_decays_leave_floats_range(dev, seq):
    """32 steps of e^3.125: e^100 in one piece is beyond float's range, a state of 2e-38 reaches 5e5 by it and one of zeros stays zeros."""
    T, D, N = 192, 4, 4
    dt = torch.zeros(T, 2, D, device=dev)
    dt[:32] = 3.125
    h0 = torch.full((2, D, N), 2e-38, device=dev)
    h0[1] = 0.0
    x, B, C = torch.zeros(T, 2, D, device=dev), torch.zeros(T, 2, N, device=dev), torch.ones(T, 2, N, device=dev)
    y, st = seq.selective_scan(x, dt, torch.ones(D, N, device=dev), B, C, dt_softplus=False, initial_state=h0, return_state=True)
    o = osq.selective_scan(x, dt, torch.ones(D, N), B[:, :, None], C[:, :, None], softplus=False, state=h0)
    _same("y", y, o["y"])
    _same("state", st, o["state"])


@pytest.mark.parametrize("form", ["view", "operators"])
def test_capturing_beside_an_eager_graph_further_ahead_is_refused(dev, seq, form):
    """The leaf whose accumulator an eager graph keeps on the default stream lies behind a view (gated_linear of a 3-dimensional x), or behind two more
    operators: the call raises, and works once the eager graph is gone.  (What the check walks over is tested without a GPU: nodes_ahead.)"""
    g = _gen(7)
    leaf = torch.randn(6, 2, 8, generator=g).to(dev).requires_grad_()
    w, B, wg, A = torch.randn(8, 4, generator=g).to(dev), torch.randn(6, 2, 4, generator=g).to(dev), torch.randn(5, 8, generator=g).to(dev), -torch.rand(8, 4, generator=g).to(dev)

    def call():
        x = leaf
        if form == "operators":
            x = seq.causal_conv(x, w)
            x = seq.selective_scan(x, torch.ones_like(x), A, B, B)
        return seq.gated_linear(x, wg, wg)
    step = lambda: torch.autograd.grad(call().sum(), [leaf])[0]  # noqa: E731
    want = step()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    alive = call()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    del alive
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize(dev)
        assert torch.equal(got, want) and torch.equal(step(), want)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,R,D,N,G", [(50, 16, 512, 16, 1), (50, 2, 128, 16, 2), (16, 4, 200, 64, 1), (9, 30, 65, 5, 1), (300, 2, 72, 33, 2), (1100, 1, 96, 8, 1)])
def test_scan_errors_are_a_few_roundings(dev, seq, T, R, D, N, G, dtype):
    """Error norms.  A step adds about five roundings of the state's size (the decay's exponent and power, the input, the sum), each of variance u^2 / 3, u =
    2^-24; a state of m remembered steps is itself a sum of m terms, so against its own size they add up to u sqrt(5 m / 3), m at most T.  A's own
    rounding is the same at every step, but a state forgets it by the rate that it is off by: it, the sum over states, the gate and the step size add a
    few u, 4 here.  The whole is allowed twice (resets and decays shorten the memory: a lost digit shows below 100 steps); 16-bit results add one rounding of their own (5% for its scatter
    over 500 values and more, as a norm)."""
    i, rst, dy, ds = _scan_inputs(dev, T, R, D, N, G, dtype, "dense", seed=T + D)
    leaves = {k: v.detach().requires_grad_() for k, v in i.items()}
    y, state = _scan_call(seq, leaves, rst, True, return_state=True)
    got = dict(zip(("d" + k for k in leaves), torch.autograd.grad([y, state], list(leaves.values()), [dy, ds])), y=y, state=state)
    o = osq.selective_scan(**i, reset=rst, dy=dy, dstate=ds)
    own = 2 * ((5 * T / 3) ** 0.5 + 4) * U32
    worst = {}
    for k, v in got.items():
        once = float((o[k].to(v.dtype).double() - o[k]).norm())
        off = float((v.detach().cpu().double() - o[k]).norm())
        worst[k] = off / (own * float(o[k].norm()) + (1.05 * once if v.dtype != torch.float32 else 0.0))
    print(T, R, D, N, dtype, {k: round(v, 3) for k, v in worst.items()})
    assert max(worst.values()) <= 1.0, worst


def test_offsets_past_32_bits(dev, seq):
    """Tensors of more than 2^31 elements: the last steps, rows and channels against a call on those alone (the same kernels' bits where each value has its own
    sums, the definition's neighbourhood for the weights' sums)."""
    if torch.cuda.mem_get_info(dev)[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    T, D, last = 66000, 32768, 40
    bf, g = torch.bfloat16, torch.Generator(device=dev).manual_seed(1)
    x = torch.empty(T, 1, D, dtype=bf, device=dev).normal_(generator=g)
    assert x.numel() > 2 ** 31
    w = torch.randn(D, 4, device=dev, generator=g) * 0.5
    tail, state = x[-last:], x[-last - 3:-last].transpose(0, 1)
    leaf, tail_leaf = x.requires_grad_(), tail.detach().clone().requires_grad_()
    y, want = seq.causal_conv(leaf, w), seq.causal_conv(tail_leaf, w, initial_state=state.detach())
    assert torch.equal(y[-last:], want)
    dy = torch.empty_like(x).normal_(generator=g)
    dx, = torch.autograd.grad(y, leaf, dy)
    assert torch.equal(dx[-last:], torch.autograd.grad(want, tail_leaf, dy[-last:])[0])
    del y, dx, leaf, tail_leaf, want
    x = x.detach()
    A, B = -torch.rand(D, 4, device=dev, generator=g) - 0.5, torch.randn(T, 1, 4, device=dev, generator=g).to(bf)
    reset = torch.zeros(T, 1, dtype=torch.bool, device=dev)
    reset[-last] = True
    with torch.no_grad():
        y, st = seq.selective_scan(x, dy, A, B, B, reset=reset, return_state=True)
        want, wst = seq.selective_scan(x[-last:], dy[-last:], A, B[-last:], B[-last:], return_state=True)
    assert torch.equal(y[-last:], want) and torch.allclose(st, wst, rtol=1e-5, atol=1e-6)
    del y, dy
    rows = x.view(-1, 512)                                    # 4.2 million rows
    M, F, k = rows.shape[0], 40, 3000
    wg, wu = (torch.randn(F, 512, device=dev, generator=g).mul(0.05).to(bf).requires_grad_() for _ in range(2))
    leaf, tail_leaf = rows.requires_grad_(), rows[-k:].detach().clone().requires_grad_()
    y, want = seq.gated_linear(leaf, wg, wu), seq.gated_linear(tail_leaf, wg, wu)
    assert torch.allclose(y[-k:].float(), want.float(), rtol=2 ** -7, atol=1e-5)
    dy = torch.zeros_like(y)
    dy[-k:] = torch.randn(k, F, device=dev, generator=g).to(bf)          # only the last rows add to the weights' sums
    got, ref = torch.autograd.grad(y, [leaf, wg, wu], dy), torch.autograd.grad(want, [tail_leaf, wg, wu], dy[-k:])
    assert torch.allclose(got[0][-k:].float(), ref[0].float(), rtol=2 ** -7, atol=1e-5) and not got[0][:-k].any()
    for a, b in zip(got[1:], ref[1:]):
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -6, atol=2 ** -8 * float(b.abs().max()))


@pytest.mark.parametrize("dtype", TYPES[1:], ids=["bf16", "f16"])
def test_gated_weights_of_the_widest_tiles(dev, seq, dtype):
    """Weights large enough for 256 x 256 tiles in the weight gradients (512 of them, two for each CU) and few rows behind them, in two parts and in one: the bounds of
    test_gated_gradients_round_once_at_every_size, a last row tile that is not whole."""
    M, D, F = 200, 4096, 4090
    x, wg, wu, bg, bu, dy = _gated_inputs(dev, M, D, F, dtype, True, seed=2)
    o = osq.gated_linear(x, wg, wu, bg, bu, "silu", dy)
    for rounded, low, high in ((False, 0.0, 1.05), (True, 1.1, 1.6)):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu, bg, bu)]
        grads = torch.autograd.grad(seq.gated_linear(*leaves, rounded_grads=rounded), leaves, dy)
        ratio = {n: _norm_ratio(g, o[n]) for n, g in zip(("dx", "dw_gate", "dw_up", "db_gate", "db_up"), grads)}
        print(dtype, ratio)
        assert all((r <= high) for r in ratio.values()) and all(ratio[n] >= low for n in ("dx", "dw_gate", "dw_up")), ratio
        assert max(ratio["db_gate"], ratio["db_up"]) <= 1.05                    # (sums of the unrounded values either way)


def test_threads_at_once(dev, seq):
    """Training passes of four threads, each on a stream of its own, have the bits of lone ones; an error in one of them is that thread's own."""
    import threading
    jobs = []
    for k in range(4):
        g = _gen(40 + k)
        i, rst, dy, _ = _scan_inputs(dev, 130 + k, 2, 40 + 8 * k, 12 + k, 1, torch.float32, "dense", seed=k)
        w, wg = torch.randn(40 + 8 * k, 4, generator=g).to(dev), torch.randn(24, 40 + 8 * k, generator=g).to(dev).to(torch.bfloat16)

        def job(i=i, rst=rst, dy=dy, w=w, wg=wg):
            li = {n: v.detach().requires_grad_() for n, v in i.items()}
            y = _scan_call(seq, dict(li, x=seq.causal_conv(li["x"], w, reset=rst)), rst, True)
            out = seq.gated_linear(y.to(torch.bfloat16), wg, wg)
            return [out.detach()] + list(torch.autograd.grad(out.float().sum() + (y * dy).sum(), list(li.values())))
        jobs.append(job)
    want = [job() for job in jobs]
    torch.cuda.synchronize(dev)
    got, errors = [None] * 4, []

    def run(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream(dev)):
                for _ in range(5):
                    got[k] = jobs[k]()
                    with pytest.raises(ValueError, match="weight must be"):
                        seq.causal_conv(torch.zeros(2, 1, 8 + k, device=dev), torch.zeros(3, 4, device=dev))
                torch.cuda.current_stream(dev).synchronize()
        except BaseException as e:      # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        for p, q in zip(a, b):
            assert torch.equal(p, q)
