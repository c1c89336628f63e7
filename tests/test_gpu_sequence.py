"""The sequence operators on the GPU against their 64-bit definitions (oracle/sequence.py).

Tolerances.  A result of type t is allowed half a step of t (finfo(t).eps / 2 relative to its value) plus K 2^-24 times the sum of the
magnitudes of its terms, K the number of float32 roundings a term can meet: taps and epilogue for the convolution; for the scan
at most six per step the term is carried through, the sums over states and rows, and the exponent's own error (3 roundings of
delta |A| log2 e, which the decay e^-(delta |A|) caps at 150 before the term is gone); contraction length and epilogue for the gated unit,
whose backward pass also rounds dg and du once to the type."""
import pytest
import torch

from oracle import sequence as osq

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def seq():
    from fastdeepqlearning_amd import sequence
    return sequence


def _near(name, got, want, mag, K, extra=None):
    half = torch.finfo(got.dtype).eps / 2
    tiny = 0.0 if got.dtype != torch.float16 else 2.0 ** -25          # half a step among fp16's subnormal numbers
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{name} is not finite"
    # a value near a rounding border may go either way: half a step of the slightly moved value too
    err = K * U32 * mag
    tol = (half * (want.abs() + err) + err) * 1.0001 + tiny + 1e-37 + (0 if extra is None else extra)
    worst = ((got - want).abs() - tol).max() if got.numel() else torch.tensor(-1.0)
    assert worst <= 0, f"{name}: {float(worst):.3g} over the tolerance, off by {float((got - want).abs().max()):.3g}"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _place(t, dev, layout):
    """The same values in another place: "dense", a "slice" of wider rows that starts off alignment, or row-major "swapped" memory."""
    t = t.to(dev)
    if layout == "slice":
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 5, dtype=t.dtype, device=dev)
        wide[..., 3:3 + t.shape[-1]] = t
        return wide[..., 3:3 + t.shape[-1]]
    if layout == "swapped" and t.dim() >= 3:
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    return t


# ------------------------------------------------------------------------------------------------------------ convolution
CONV = [(1, 1, 1, 2), (2, 3, 5, 4), (3, 2, 64, 4), (9, 2, 66, 3), (17, 3, 260, 4), (50, 4, 512, 4), (130, 1, 96, 2), (65, 7, 1000, 3)]


def _conv_inputs(dev, T, R, D, K, dtype, layout, seed=0, resets=0.2):
    g = _gen(seed)
    x = _place(torch.randn(T, R, D, generator=g).to(dtype), dev, layout)
    w, b = (torch.randn(D, K, generator=g) * K ** -0.5).to(dev), (torch.randn(D, generator=g) * 0.3).to(dev)
    rst = (torch.rand(T, R, generator=g) < resets).to(dev)
    st = torch.randn(R, K - 1, D, generator=g).to(dtype).to(dev)
    dy = _place(torch.randn(T, R, D, generator=g).to(dtype), dev, layout)
    ds = torch.randn(R, K - 1, D, generator=g).to(dtype).to(dev)
    return x, w, b, rst, st, dy, ds


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,R,D,K", CONV)
@pytest.mark.parametrize("form", ["plain", "full", "slice", "swapped"])
def test_conv(dev, seq, T, R, D, K, dtype, form):
    layout = form if form in ("slice", "swapped") else "dense"
    x, w, b, rst, st, dy, ds = _conv_inputs(dev, T, R, D, K, dtype, layout)
    if form == "plain":
        b = rst = st = ds = None
    silu = form != "swapped"
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, st)]
    y, state = seq.causal_conv(leaves[0], leaves[1], leaves[2], reset=rst, initial_state=leaves[3], silu=silu, return_state=True)
    outs, cots = [y], [dy]
    if ds is not None:
        outs.append(state)
        cots.append(ds)
    used = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(outs, used, cots))
    args = (x, w, b, st, rst, silu, dy, ds)
    o, m = osq.causal_conv(*args), osq.causal_conv(*args, mag=True)
    Kf = K + 12
    _near("y", y, o["y"], m["y"], Kf)
    assert torch.equal(state.detach().cpu().double(), o["state"])
    _near("dx", next(grads), o["dx"], m["dx"], 2 * Kf)
    _near("dweight", next(grads), o["dweight"], m["dweight"], 2 * Kf + T * R)
    if b is not None:
        _near("dbias", next(grads), o["dbias"], m["dbias"], 2 * Kf + T * R)
    if st is not None:
        _near("dstate", next(grads), o["dstate"], m["dstate"], 2 * Kf)
    with torch.no_grad():
        assert torch.equal(seq.causal_conv(x, w, b, reset=rst, initial_state=st, silu=silu), y)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", ["dense", "slice"])
def test_conv_steps_are_the_window(dev, seq, dtype, layout):
    """Single steps, in place, give the window's bits and state."""
    T, R, D, K = 11, 5, 72, 4
    x, w, b, rst, st, _, _ = _conv_inputs(dev, T, R, D, K, dtype, layout, seed=3)
    y, last = seq.causal_conv(x, w, b, reset=rst, initial_state=st, return_state=True)
    state = st.clone()
    for t in range(T):
        yt, new = seq.causal_conv_step(x[t], state, w, b, reset=rst[t], out_state=state)
        assert new is state and torch.equal(yt, y[t])
    assert torch.equal(state, last)
    yt, new = seq.causal_conv_step(x[0], st, w, b, reset=rst[0])
    assert torch.equal(yt, y[0]) and not torch.equal(new, st)


# ------------------------------------------------------------------------------------------------------------------- scan
# every (states per lane, lanes per channel) form, whole and cut into segments, channels that leave a wave part empty, groups
SCAN = [(1, 1, 1, 1, 1), (2, 3, 5, 4, 1), (7, 2, 130, 3, 1), (8, 1, 64, 16, 1), (9, 3, 65, 5, 1), (50, 2, 128, 16, 2), (33, 2, 40, 24, 2), (16, 2, 20, 64, 1),
        (5, 260, 70, 16, 1), (6, 520, 33, 8, 3), (200, 1, 70, 16, 1), (300, 2, 36, 33, 2), (150, 1, 33, 3, 3), (131, 2, 300, 20, 1), (129, 300, 40, 7, 1)]


def _scan_inputs(dev, T, R, D, N, G, dtype, layout, seed=0, resets=0.1):
    g = _gen(seed)
    p = lambda *s: _place(torch.randn(*s, generator=g).to(dtype), dev, layout)  # noqa: E731
    A = (-(0.05 + 3 * torch.rand(D, N, generator=g))).to(dev)
    i = dict(x=p(T, R, D), dt=p(T, R, D), A=A, B=p(T, R, G, N), C=p(T, R, G, N), skip=torch.randn(D, generator=g).to(dev), z=p(T, R, D),
             dt_bias=(torch.randn(D, generator=g) - 2).to(dev), state=torch.randn(R, D, N, generator=g).to(dev))
    rst = (torch.rand(T, R, generator=g) < resets).to(dev)
    return i, rst, p(T, R, D), torch.randn(R, D, N, generator=g).to(dev)


def _scan_call(seq, i, rst, softplus, **kw):
    return seq.selective_scan(i["x"], i["dt"], i["A"], i["B"], i["C"], skip=i["skip"], z=i["z"], dt_bias=i["dt_bias"], dt_softplus=softplus, reset=rst,
                              initial_state=i["state"], **kw)


def _scan_check(seq, i, rst, dy, ds, softplus=True):
    T, R, D = i["x"].shape
    N = i["A"].shape[1]
    leaves = {k: v.detach().requires_grad_() for k, v in i.items() if v is not None}
    li = {k: leaves.get(k) for k in i}
    y, state = _scan_call(seq, li, rst, softplus, return_state=True)
    outs, cots = ([y, state], [dy, ds]) if ds is not None else ([y], [dy])
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), cots)))
    args = dict(i, softplus=softplus, reset=rst, dy=dy, dstate=ds)
    o, m = osq.selective_scan(**args), osq.selective_scan(**args, mag=True)
    Kf = 6 * T + N + 40 + 450
    _near("y", y, o["y"], m["y"], Kf)
    _near("state", state, o["state"], m["state"], Kf)
    for k, v in grads.items():
        many = {"A": T * R, "skip": T * R, "dt_bias": T * R, "B": D, "C": D}.get(k, 0)
        _near("d" + k, v, o["d" + k], m["d" + k], 2 * Kf + many)
    with torch.no_grad():
        y2, s2 = _scan_call(seq, i, rst, softplus, return_state=True)
        if T > 1:
            assert torch.equal(y2, y) and torch.equal(s2, state)


@pytest.mark.parametrize("T,R,D,N,G", SCAN)
def test_scan_f32(dev, seq, T, R, D, N, G):
    i, rst, dy, ds = _scan_inputs(dev, T, R, D, N, G, torch.float32, "dense", seed=T + N)
    _scan_check(seq, i, rst, dy, ds)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=["bf16", "f16"])
@pytest.mark.parametrize("T,R,D,N,G", [s for s in SCAN if s[0] * s[1] * s[2] < 60000])
def test_scan_16_bit(dev, seq, T, R, D, N, G, dtype):
    i, rst, dy, ds = _scan_inputs(dev, T, R, D, N, G, dtype, "dense", seed=T + N)
    _scan_check(seq, i, rst, dy, ds)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,R,D,N,G", [(9, 3, 65, 5, 1), (40, 2, 72, 16, 2), (140, 2, 40, 24, 1)])
@pytest.mark.parametrize("form", ["slice", "swapped", "bare", "nosoftplus", "all_reset"])
def test_scan_forms(dev, seq, T, R, D, N, G, dtype, form):
    i, rst, dy, ds = _scan_inputs(dev, T, R, D, N, G, dtype, form if form in ("slice", "swapped") else "dense", seed=5)
    softplus = True
    if form == "bare":          # only what is needed
        i.update(skip=None, z=None, dt_bias=None, state=None)
        rst = ds = None
    elif form == "nosoftplus":
        i["dt"] = i["dt"].abs() * 0.3
        i["dt_bias"] = None
        softplus = False
    elif form == "all_reset":   # every step begins a sequence
        rst = torch.ones_like(rst)
    _scan_check(seq, i, rst, dy, ds, softplus)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("R,D,N,G", [(1, 1, 1, 1), (3, 65, 5, 1), (5, 128, 16, 2), (2, 200, 64, 1), (4, 96, 33, 3)])
def test_scan_steps_follow_the_definition(dev, seq, R, D, N, G, dtype):
    """Steps from a state, to a new tensor and in place, against the definition; a reset row drops even a NaN state."""
    i, rst, _, _ = _scan_inputs(dev, 3, R, D, N, G, dtype, "dense", seed=7, resets=0.4)
    o, m = osq.selective_scan(**i, reset=rst), osq.selective_scan(**i, reset=rst, mag=True)
    state, kept = i["state"].clone(), i["state"].clone()
    kw = dict(skip=i["skip"], dt_bias=i["dt_bias"])
    for t in range(3):
        first = (i["x"][t], i["dt"][t], i["A"], i["B"][t], i["C"][t])
        y, kept = seq.selective_scan_step(*first, kept, z=i["z"][t], reset=rst[t], **kw)
        y2, same = seq.selective_scan_step(*first, state, z=i["z"][t], reset=rst[t], out_state=state, **kw)
        assert same is state and torch.equal(y, y2) and torch.equal(kept, state)
        _near("y", y, o["y"][t], m["y"][t], 6 * 3 + N + 490)
    _near("state", state, o["state"], m["state"], 6 * 3 + N + 490)
    bad = torch.full_like(state, float("nan"))
    y, _ = seq.selective_scan_step(*first, bad, z=i["z"][2], reset=torch.ones(R, dtype=torch.bool, device=dev), **kw)
    assert torch.isfinite(y).all()


@pytest.mark.parametrize("T", [20, 150])
def test_reset_drops_nan_and_inf(dev, seq, T):
    """What lies before a reset - a NaN state, NaN and infinite steps - leaves no trace behind it; packing equals separate calls."""
    R, D, N, K = 2, 40, 16, 4
    i, _, _, _ = _scan_inputs(dev, T, R, D, N, 1, torch.float32, "dense", seed=9)
    cut = T // 2 + 1
    rst = torch.zeros(T, R, dtype=torch.bool, device=dev)
    rst[cut] = True
    w, b = torch.randn(D, K, device=dev), torch.randn(D, device=dev)
    want = _scan_call(seq, {k: (v[cut:] if v.dim() >= 3 and k != "state" else None if k == "state" else v) for k, v in i.items()}, None, True, return_state=True)
    wconv = seq.causal_conv(i["x"][cut:], w, b, return_state=True)
    for k in ("x", "dt", "B", "z"):
        i[k] = i[k].clone()
        i[k][:cut] = float("nan")
        i[k][1] = float("inf")
    i["state"] = torch.full_like(i["state"], float("-inf"))
    y, st = _scan_call(seq, i, rst, True, return_state=True)
    o = osq.selective_scan(**{k: (v[cut:] if v.dim() >= 3 and k != "state" else None if k == "state" else v) for k, v in i.items()}, mag=True)
    _near("y", y[cut:], want[0].cpu().double(), o["y"], 12 * T + 2 * 506)
    _near("state", st, want[1].cpu().double(), o["state"], 12 * T + 2 * 506)
    yc, sc = seq.causal_conv(i["x"], w, b, reset=rst, initial_state=torch.full((R, K - 1, D), float("nan"), device=dev), return_state=True)
    assert torch.equal(yc[cut:], wconv[0]) and torch.equal(sc, wconv[1])


def test_state_carries_over_a_split(dev, seq):
    """A window in two calls, the state handed over, gives the whole window's outputs and gradients."""
    T, R, D, N = 60, 3, 48, 16
    i, rst, dy, ds = _scan_inputs(dev, T, R, D, N, 1, torch.float32, "dense", seed=11)
    li = {k: v.detach().requires_grad_() for k, v in i.items()}
    part = lambda a, b, st: {k: (v[a:b] if v.dim() >= 3 and k != "state" else v) for k, v in li.items()} | {"state": st}  # noqa: E731
    y1, s1 = _scan_call(seq, part(0, 23, li["state"]), rst[:23], True, return_state=True)
    y2, s2 = _scan_call(seq, part(23, T, s1), rst[23:], True, return_state=True)
    got = dict(zip(li, torch.autograd.grad([y1, y2, s2], list(li.values()), [dy[:23], dy[23:], ds])))
    args = dict(i, reset=rst, dy=dy, dstate=ds)
    o, m = osq.selective_scan(**args), osq.selective_scan(**args, mag=True)
    Kf = 6 * T + N + 490
    _near("y", torch.cat([y1, y2]), o["y"], m["y"], Kf)
    _near("state", s2, o["state"], m["state"], Kf)
    for k, v in got.items():
        _near("d" + k, v, o["d" + k], m["d" + k], 2 * Kf + T * R)


# ------------------------------------------------------------------------------------------------------------------ gated
GATED = [(1, 1, 1), (5, 16, 16), (17, 40, 50), (32, 256, 256), (33, 64, 48), (64, 130, 66), (100, 72, 100), (300, 200, 136), (129, 96, 130), (1000, 64, 64)]


def _gated_inputs(dev, M, D, F, dtype, bias, seed=0):
    g = _gen(seed)
    r = lambda *s, k=1.0: (torch.randn(*s, generator=g) * k).to(dtype).to(dev)  # noqa: E731
    x, wg, wu = r(M, D), r(F, D, k=D ** -0.5), r(F, D, k=D ** -0.5)
    return [x, wg, wu] + ([r(F, k=0.3), r(F, k=0.3)] if bias else [None, None]) + [r(M, F)]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,D,F", GATED)
@pytest.mark.parametrize("form", ["silu", "gelu", "sigmoid_bare", "slice"])
def test_gated(dev, seq, M, D, F, dtype, form):
    bias, kind = form != "sigmoid_bare", {"sigmoid_bare": "sigmoid", "slice": "silu"}.get(form, form)
    x, wg, wu, bg, bu, dy = _gated_inputs(dev, M, D, F, dtype, bias, seed=M)
    if form == "slice":
        x, dy = _place(x, dev, "slice"), _place(dy, dev, "slice")
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, wg, wu, bg, bu)]
    y = seq.gated_linear(*leaves, activation=kind)
    used = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, used, dy)
    o = osq.gated_linear(x, wg, wu, bg, bu, kind, dy)
    _near("y", y, o["y"], o["m_y"] + o["y"].abs() * 8 / (D + 1), 2 * D + 8)
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0                # dg, du among fp16's subnormal numbers
    for name, got in zip(("x", "w_gate", "w_up", "b_gate", "b_up"), grads):
        n = 2 * F if name == "x" else M
        full = sub * (2 * F * float(wg.detach().abs().max()) + M * float(x.detach().abs().max())) if name[0] != "b" else 0.0
        rounded = half * o["r_d" + name] * (0 if name[0] == "b" else 1.001) + full
        _near("d" + name, got, o["d" + name], o["r_d" + name] * (2 * n + 16) + o["e_d" + name] * (2 * D + 8), 1, rounded * (1 + half))
    with torch.no_grad():
        assert torch.equal(seq.gated_linear(x, wg, wu, bg, bu, activation=kind), y)


# many rows, many features, many channels: every tile shape of every product, edges on all sides
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,D,F", [(5000, 136, 1030), (9000, 72, 1030), (13000, 520, 40), (22000, 776, 72), (200, 2000, 1600), (100, 2104, 4200)])
def test_gated_many_tiles(dev, seq, M, D, F, dtype):
    """Enough tiles for the large tile shapes, edges on every side, rows split over workgroups for the weights' gradients."""
    x, wg, wu, bg, bu, dy = _gated_inputs(dev, M, D, F, dtype, True, seed=1)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    y = seq.gated_linear(*leaves, activation="silu")
    grads = torch.autograd.grad(y, leaves, dy)
    o = osq.gated_linear(x, wg, wu, bg, bu, "silu", dy)
    _near("y", y, o["y"], o["m_y"] + o["y"].abs() * 8 / (D + 1), 2 * D + 8)
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for name, got in zip(("x", "w_gate", "w_up", "b_gate", "b_up"), grads):
        n = 2 * F if name == "x" else M
        full = sub * (2 * F * float(wg.detach().abs().max()) + M * float(x.detach().abs().max())) if name[0] != "b" else 0.0
        rounded = (half * o["r_d" + name] * 1.001 if name[0] != "b" else 0.0) + full
        _near("d" + name, got, o["d" + name], o["r_d" + name] * (2 * n + 16) + o["e_d" + name] * (2 * D + 8), 1, rounded)


def test_gated_leading_dimensions(dev, seq):
    x, wg, wu, bg, bu, _ = _gated_inputs(dev, 24, 40, 50, torch.float32, True)
    y = seq.gated_linear(x, wg, wu, bg, bu)
    assert torch.equal(seq.gated_linear(x.view(2, 3, 4, 40), wg, wu, bg, bu), y.view(2, 3, 4, 50))
    assert torch.equal(seq.gated_linear(x[0], wg, wu, bg, bu), y[0])
    swapped = x.view(4, 6, 40).transpose(0, 1)
    assert torch.equal(seq.gated_linear(swapped, wg, wu, bg, bu), y.view(4, 6, 50).transpose(0, 1))


# --------------------------------------------------------------------------------------------------------------- together
class _Block:
    """A recurrent block over windows: projections by torch, the three operators, one step at a time or all at once."""

    def __init__(self, dev, din=24, inner=72, n=16, out=40, dtype=torch.float32):
        g = _gen(21)
        r = lambda *s, k=1.0, t=dtype: (torch.randn(*s, generator=g) * k).to(t).to(dev)  # noqa: E731
        self.w_in, self.w_sel = r(2 * inner, din, k=din ** -0.5), r(inner + 2 * n, inner, k=inner ** -0.5)
        self.conv_w, self.conv_b = r(inner, 4, k=0.5, t=torch.float32), r(inner, k=0.1, t=torch.float32)
        self.A = (-(0.1 + 2 * torch.rand(inner, n, generator=g))).to(dev)
        self.skip, self.dt_bias = r(inner, t=torch.float32), r(inner, t=torch.float32) - 2
        self.wg, self.wu, self.bg, self.bu = r(out, inner, k=inner ** -0.5), r(out, inner, k=inner ** -0.5), r(out, k=0.1), r(out, k=0.1)
        self.inner, self.n = inner, n

    def params(self):
        return [self.w_in, self.w_sel, self.conv_w, self.conv_b, self.A, self.skip, self.dt_bias, self.wg, self.wu, self.bg, self.bu]

    def window(self, seq, e, reset=None, conv_state=None, state=None):
        x, z = (e @ self.w_in.t()).chunk(2, -1)
        x, cs = seq.causal_conv(x, self.conv_w, self.conv_b, reset=reset, initial_state=conv_state, return_state=True)
        dt, B, C = (x @ self.w_sel.t()).split([self.inner, self.n, self.n], -1)
        y, hs = seq.selective_scan(x, dt, self.A, B, C, skip=self.skip, z=z, dt_bias=self.dt_bias, reset=reset, initial_state=state, return_state=True)
        return seq.gated_linear(y, self.wg, self.wu, self.bg, self.bu), cs, hs

    def step(self, seq, e, cs, hs, reset=None):
        x, z = (e @ self.w_in.t()).chunk(2, -1)
        x, cs = seq.causal_conv_step(x, cs, self.conv_w, self.conv_b, reset=reset)
        dt, B, C = (x @ self.w_sel.t()).split([self.inner, self.n, self.n], -1)
        y, hs = seq.selective_scan_step(x, dt, self.A, B, C, hs, skip=self.skip, z=z, dt_bias=self.dt_bias, reset=reset)
        return seq.gated_linear(y, self.wg, self.wu, self.bg, self.bu), cs, hs


def test_block_prompt_then_steps(dev, seq):
    """A prompt and the steps after it give what the whole window gives (the sums run in other orders: float32's error times the depth)."""
    blk = _Block(dev)
    e = torch.randn(30, 5, 24, generator=_gen(4)).to(dev)
    rst = (torch.rand(30, 5, generator=_gen(5)) < 0.1).to(dev)
    want, wcs, whs = blk.window(seq, e, rst)
    y, cs, hs = blk.window(seq, e[:19], rst[:19])
    assert torch.allclose(y, want[:19], rtol=1e-4, atol=1e-4)
    for t in range(19, 30):
        y, cs, hs = blk.step(seq, e[t], cs, hs, rst[t])
        assert torch.allclose(y, want[t], rtol=1e-4, atol=1e-4)
    assert torch.allclose(cs, wcs, rtol=1e-4, atol=1e-4) and torch.allclose(hs, whs, rtol=1e-4, atol=1e-4)


def test_block_gradients_against_differences(dev, seq):
    """One training pass of the block: every parameter's gradient against a central difference of the float64 definition."""
    blk = _Block(dev, din=8, inner=12, n=4, out=6)
    e = torch.randn(7, 3, 8, generator=_gen(4)).to(dev)
    rst = (torch.rand(7, 3, generator=_gen(5)) < 0.2).to(dev)
    dy = torch.randn(7, 3, 6, generator=_gen(6)).to(dev)
    for p in blk.params():
        p.requires_grad_()
    grads = torch.autograd.grad(blk.window(seq, e, rst)[0], blk.params(), dy)

    def value(ps):
        w_in, w_sel, cw, cb, A, skip, bias, wg, wu, bg, bu = ps
        x, z = (e.cpu().double() @ w_in.t()).chunk(2, -1)
        x = osq.causal_conv(x, cw, cb, reset=rst)["y"]
        dt, B, C = (x @ w_sel.t()).split([12, 4, 4], -1)
        y = osq.selective_scan(x, dt, A, B.unsqueeze(2), C.unsqueeze(2), skip, z, bias, reset=rst)["y"]
        out = osq.gated_linear(y.reshape(-1, 12), wg, wu, bg, bu)["y"]
        return float((out * dy.cpu().double().reshape(-1, 6)).sum())
    base = [p.detach().cpu().double() for p in blk.params()]
    g = _gen(8)
    for k, (p, grad) in enumerate(zip(base, grads)):
        d = torch.randn(p.shape, generator=g, dtype=torch.float64)
        num = (value(base[:k] + [p + 1e-6 * d] + base[k + 1:]) - value(base[:k] + [p - 1e-6 * d] + base[k + 1:])) / 2e-6
        ana = float((grad.cpu().double() * d).sum())
        scale = float((grad.cpu().double() * d).abs().sum())
        assert abs(num - ana) <= 1e-4 * scale + 1e-7, (k, num, ana)


def test_block_trains_in_a_replayed_graph(dev, seq):
    """Forward and backward captured once and replayed on new inputs, with eager work between: every replay has the eager bits."""
    blk = _Block(dev)
    leaves = [p.detach().clone().requires_grad_() for p in blk.params()]
    names = ["w_in", "w_sel", "conv_w", "conv_b", "A", "skip", "dt_bias", "wg", "wu", "bg", "bu"]
    for n, p in zip(names, leaves):
        setattr(blk, n, p)
    e, dy = torch.zeros(140, 2, 24, device=dev), torch.zeros(140, 2, 40, device=dev)
    rst = torch.zeros(140, 2, dtype=torch.bool, device=dev)

    def one():
        y, cs, hs = blk.window(seq, e, rst)
        return [y.detach(), cs.detach(), hs.detach()] + list(torch.autograd.grad(y, leaves, dy))   # (no autograd graph outlives the call)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        for _ in range(2):
            one()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = one()
    g = _gen(31)
    for k in range(4):
        e.copy_(torch.randn(e.shape, generator=g))
        dy.copy_(torch.randn(dy.shape, generator=g))
        rst.copy_(torch.rand(rst.shape, generator=g) < 0.1 * k)
        graph.replay()
        got = [o.detach().clone() for o in outs]
        torch.cuda.synchronize(dev)
        want = one()
        for a, b in zip(got, want):
            assert torch.equal(a, b.detach())


def test_steps_in_a_replayed_graph(dev, seq):
    """An acting step captured with its states in place: replays follow the eager steps."""
    blk = _Block(dev)
    e = torch.zeros(4, 24, device=dev)
    cs, hs = torch.zeros(4, 3, 72, device=dev), torch.zeros(4, 72, 16, device=dev)

    def one():
        x, z = (e @ blk.w_in.t()).chunk(2, -1)
        x, _ = seq.causal_conv_step(x, cs, blk.conv_w, blk.conv_b, out_state=cs)
        dt, B, C = (x @ blk.w_sel.t()).split([72, 16, 16], -1)
        y, _ = seq.selective_scan_step(x, dt, blk.A, B, C, hs, skip=blk.skip, z=z, dt_bias=blk.dt_bias, out_state=hs)
        return seq.gated_linear(y, blk.wg, blk.wu, blk.bg, blk.bu)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        one()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one()
    cs.zero_()
    hs.zero_()
    steps = torch.randn(5, 4, 24, generator=_gen(2)).to(dev)
    ref_c, ref_h = torch.zeros_like(cs), torch.zeros_like(hs)
    for k in range(5):
        e.copy_(steps[k])
        graph.replay()
        y, ref_c, ref_h = blk.step(seq, steps[k], ref_c, ref_h)
        assert torch.equal(out, y) and torch.equal(cs, ref_c) and torch.equal(hs, ref_h)


def test_two_streams_at_once(dev, seq):
    """Calls on two streams do not share anything: both give the bits of a lone call."""
    i, rst, dy, _ = _scan_inputs(dev, 200, 2, 70, 16, 1, torch.float32, "dense", seed=2)

    def one():
        li = {k: v.detach().requires_grad_() for k, v in i.items()}
        y = _scan_call(seq, li, rst, True)
        return [y.detach()] + list(torch.autograd.grad(y, list(li.values()), dy))
    want = one()
    torch.cuda.synchronize(dev)
    streams, got = [torch.cuda.Stream(dev) for _ in range(2)], [None, None]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = one()
    torch.cuda.synchronize(dev)
    for r in got:
        for a, b in zip(r, want):
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ empty shapes, refusals
def test_empty_shapes(dev, seq):
    z = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    st, h0 = torch.randn(2, 3, 8, device=dev), torch.randn(2, 8, 4, device=dev)
    for T, R in ((0, 2), (4, 0), (0, 0)):
        x, w, b = z(T, R, 8).requires_grad_(), z(8, 4).requires_grad_(), z(8).requires_grad_()
        s0 = st[:R].clone().requires_grad_()
        y, s1 = seq.causal_conv(x, w, b, initial_state=s0, return_state=True)
        assert y.shape == (T, R, 8) and (T > 0 or torch.equal(s1, s0))
        g = torch.autograd.grad([y, s1], [x, w, b, s0], [torch.ones_like(y), torch.ones_like(s1)])
        assert not g[1].any() and not g[2].any() and (T > 0 or (g[3] == 1).all())
        A, B = z(8, 4).requires_grad_(), z(T, R, 4).requires_grad_()
        i0 = h0[:R].clone().requires_grad_()
        y, s1 = seq.selective_scan(x, x, A, B, B, dt_bias=b, initial_state=i0, return_state=True)
        assert y.shape == (T, R, 8) and (T > 0 or torch.equal(s1, i0))
        g = torch.autograd.grad([y, s1], [A, b, i0], [torch.ones_like(y), torch.ones_like(s1)])
        assert not g[0].any() and not g[1].any() and (T > 0 or (g[2] == 1).all())
    assert seq.causal_conv_step(z(0, 8), z(0, 3, 8), z(8, 4))[0].shape == (0, 8)
    assert seq.selective_scan_step(z(0, 8), z(0, 8), z(8, 4), z(0, 4), z(0, 4), z(0, 8, 4))[0].shape == (0, 8)
    for dtype in TYPES:
        wg = torch.ones(6, 8, device=dev, dtype=dtype).requires_grad_()
        x = torch.zeros(0, 8, device=dev, dtype=dtype).requires_grad_()
        bias = torch.ones(6, device=dev, dtype=dtype).requires_grad_()
        y = seq.gated_linear(x, wg, wg, bias, bias)
        g = torch.autograd.grad(y, [x, wg, bias], torch.ones_like(y))
        assert y.shape == (0, 6) and g[0].shape == (0, 8) and not g[1].any() and not g[2].any()


def test_refusals(dev, seq):
    """Wrong types, shapes and devices raise before anything is launched."""
    z = lambda *s, t=torch.float32: torch.zeros(*s, device=dev, dtype=t)  # noqa: E731
    x, w = z(4, 2, 8), z(8, 4)
    bad = [
        lambda: seq.causal_conv(x.double(), w), lambda: seq.causal_conv(x[0], w), lambda: seq.causal_conv(x, z(8, 5)), lambda: seq.causal_conv(x, z(7, 4)),
        lambda: seq.causal_conv(x, w.half()), lambda: seq.causal_conv(x, w.cpu()), lambda: seq.causal_conv(x, w, z(7)),
        lambda: seq.causal_conv(x, w, reset=z(4, 2)), lambda: seq.causal_conv(x, w, reset=z(2, 4, t=torch.bool)),
        lambda: seq.causal_conv(x, w, initial_state=z(2, 4, 8)), lambda: seq.causal_conv(x, w, initial_state=z(2, 3, 8, t=torch.float16)),
        lambda: seq.causal_conv_step(x[0], z(2, 3, 8), w, out_state=z(2, 8, 3).transpose(1, 2)), lambda: seq.causal_conv_step(x[0], None, w),
        lambda: seq.causal_conv_step(x[0].requires_grad_(), z(2, 3, 8), w),
        lambda: seq.selective_scan(x, x, z(8, 65), z(4, 2, 65), z(4, 2, 65)), lambda: seq.selective_scan(x, x, z(8, 4), z(4, 2, 3, 4), z(4, 2, 3, 4)),
        lambda: seq.selective_scan(x, x[:3], z(8, 4), z(4, 2, 4), z(4, 2, 4)), lambda: seq.selective_scan(x, x, z(8, 4), z(4, 2, 4), z(4, 2, 5)),
        lambda: seq.selective_scan(x, x, z(8, 4, t=torch.bfloat16), z(4, 2, 4), z(4, 2, 4)), lambda: seq.selective_scan(x, x, z(8, 4), z(4, 2, 4), z(4, 2, 4), z=z(4, 2, 7)),
        lambda: seq.selective_scan(x, x, z(8, 4), z(4, 2, 4), z(4, 2, 4), initial_state=z(2, 8, 5)),
        lambda: seq.selective_scan_step(x[0], x[0], z(8, 4), z(2, 4), z(2, 4), None),
        lambda: seq.selective_scan_step(x[0], x[0], z(8, 4).requires_grad_(), z(2, 4), z(2, 4), z(2, 8, 4)),
        lambda: seq.gated_linear(x, z(5, 8), z(6, 8)), lambda: seq.gated_linear(x, z(5, 8), z(5, 8), z(5)), lambda: seq.gated_linear(x, z(5, 8), z(5, 8), activation="tanh"),
        lambda: seq.gated_linear(x, z(5, 8, t=torch.float16), z(5, 8, t=torch.float16)), lambda: seq.gated_linear(x, z(5, 7), z(5, 7)),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_second_derivative_is_refused(dev, seq):
    x = torch.randn(3, 8, device=dev, requires_grad=True)
    w = torch.randn(4, 8, device=dev, requires_grad=True)
    g, = torch.autograd.grad(seq.gated_linear(x, w, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("D,N,pad", [(64, 16, 0), (37, 5, 0), (64, 16, 1), (40, 64, 4)])
@pytest.mark.parametrize("inplace", [False, True])
def test_states_as_columns_of_one_row(dev, seq, D, N, pad, inplace):
    """Both states of a row side by side in one buffer (rows of 3 D + D N + pad floats): read from and written to strided views, in place and
    into another buffer; the columns between and behind stay as they were; equal to dense states bit for bit."""
    R, W = 5, 3 * D + D * N + pad
    g = _gen(D + N)
    buf = torch.randn(R, W, generator=g).to(dev)
    out = buf if inplace else torch.full((R, W), 7.0, device=dev)
    views = lambda t: (t[:, :3 * D].view(R, 3, D), t[:, 3 * D:3 * D + D * N].view(R, D, N))  # noqa: E731
    x, w = torch.randn(R, D, generator=g).to(dev), torch.randn(D, 4, generator=g).to(dev)
    A, bc = -torch.rand(D, N, generator=g).to(dev), torch.randn(2, R, N, generator=g).to(dev)
    (cs, hs), (co, ho) = views(buf), views(out)
    rest = out[:, 3 * D + D * N:].clone()
    want_y, want_c = seq.causal_conv_step(x, cs.clone(), w)
    want_v, want_h = seq.selective_scan_step(want_y, x, A, bc[0], bc[1], hs.contiguous().clone())
    y, c = seq.causal_conv_step(x, cs, w, out_state=co)
    v, h = seq.selective_scan_step(y, x, A, bc[0], bc[1], hs, out_state=ho)
    assert c.data_ptr() == co.data_ptr() and h.data_ptr() == ho.data_ptr()
    for got, want in ((y, want_y), (co, want_c), (ho, want_h)):
        assert torch.equal(got, want)
    terms = (want_h.double() * bc[1].double()[:, None]).abs().sum(-1)
    assert ((v.double() - want_v.double()).abs() <= 2.02 * (N + 1) * 2.0 ** -24 * terms).all()
    assert torch.equal(out[:, 3 * D + D * N:], rest)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("M,D,F", [(1, 358, 316), (3, 61, 22), (5, 64, 64), (40, 17, 19), (473, 42, 18), (1417, 48, 16), (16, 18, 98), (9, 800, 112), (200, 8, 8)])
@pytest.mark.parametrize("kind", ["silu", "gelu", "sigmoid"])
def test_gated_small_gradients_round_once(dev, seq, M, D, F, kind, dtype):
    """Few values: the gradients in front of the products are kept in two 16-bit parts.  Two parts leave at most u^2 of a value (u: half a step;
    the second part's own rounding; fp16's smallest step, 2^-24, bounds it from below), the float products and the activation's slope a few
    dozen 2^-24 of the terms' magnitudes, and the result is rounded once: in one part the terms themselves would be off by u."""
    g = _gen(M + D + F)
    x, wg, wu = torch.randn(M, D, generator=g), torch.randn(F, D, generator=g) * D ** -0.5, torch.randn(F, D, generator=g) * D ** -0.5
    dy = torch.randn(M, F, generator=g)
    x, wg, wu, dy = (t.to(dtype) for t in (x, wg, wu, dy))
    leaves = [t.to(dev).requires_grad_() for t in (x, wg, wu)]
    got = torch.autograd.grad(seq.gated_linear(*leaves, activation=kind), leaves, dy.to(dev))
    o = osq.gated_linear(x, wg, wu, None, None, kind, dy)
    u, e = torch.finfo(dtype).eps / 2, 2.0 ** -24
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for name, have, n, other in (("dx", got[0], 2 * F, torch.stack([wg, wu])), ("dw_gate", got[1], M, x), ("dw_up", got[2], M, x)):
        want = o[name]
        exact = o["r_" + name] * (1.01 * u * u + (2 * n + 32) * e) + o["e_" + name] * (2 * D + 32) * e + tiny * n * float(other.abs().max())
        bound = (want.abs() + exact) * u * 1.01 + exact + tiny
        off = (have.cpu().double() - want).abs()
        assert (off <= bound).all(), (name, float((off / bound.clamp_min(1e-300)).max()))


def test_a_state_updated_in_place_counts_as_changed(dev, seq):
    """A window that saved the state for its backward pass refuses to run it once a step has written that state; out_state rows that share
    memory, and one that wants a gradient, are refused."""
    g = _gen(5)
    x = torch.randn(3, 2, 8, generator=g).to(dev)
    w, A = torch.randn(8, 4, generator=g).to(dev).requires_grad_(), -torch.rand(8, 4, generator=g).to(dev)
    B = torch.randn(3, 2, 4, generator=g).to(dev)
    cs, hs = torch.randn(2, 3, 8, generator=g).to(dev), torch.randn(2, 8, 4, generator=g).to(dev)
    y = seq.causal_conv(x, w, initial_state=cs)
    v = seq.selective_scan(y, x, A, B, B, initial_state=hs)
    kept = [seq.causal_conv(x, w, initial_state=cs.clone()).sum(), v.sum()]
    with torch.no_grad():
        seq.causal_conv_step(x[0], cs, w, out_state=cs)
        seq.selective_scan_step(x[0], x[0], A, B[0], B[0], hs, out_state=hs)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="inplace"):
        kept[1].backward()
    kept[0].backward()
    with torch.no_grad():
        with pytest.raises(Exception, match="overlap"):
            seq.causal_conv_step(x[0], cs, w, out_state=cs[:1].expand(2, 3, 8))
        with pytest.raises(Exception, match="overlap"):
            seq.selective_scan_step(x[0], x[0], A, B[0], B[0], hs, out_state=hs[:1].expand(2, 8, 4))
    with pytest.raises(ValueError, match="no gradient"):
        seq.selective_scan_step(x[0], x[0], A, B[0], B[0], hs, out_state=torch.zeros(2, 8, 4, device=dev, requires_grad=True))
    with torch.inference_mode():
        s = torch.zeros(2, 3, 8, device=dev)
        seq.causal_conv_step(x[0], s, w, out_state=s)
        assert s.any()


@pytest.mark.parametrize("op", ["conv", "scan", "gated", pytest.param("gated view", marks=pytest.mark.skip(
    reason="a 3-dimensional x reaches its leaf through a view: ended the process when only direct leaves were looked at; not run again since"))])
def test_capturing_beside_an_eager_graph_of_the_same_leaves_is_refused(dev, seq, op):
    """The call raises instead of letting the leaf's accumulator, which lives on the default stream, end the process; once the eager graph is gone
    the same capture works and its replay has the eager bits."""
    g = _gen(7)
    leaf = torch.randn(6, 2, 8, generator=g).to(dev).requires_grad_()
    w, B, wg = torch.randn(8, 4, generator=g).to(dev), torch.randn(6, 2, 4, generator=g).to(dev), torch.randn(5, 8, generator=g).to(dev)
    A = -torch.rand(8, 4, generator=g).to(dev)
    call = {"conv": lambda: seq.causal_conv(leaf, w), "scan": lambda: seq.selective_scan(leaf, torch.ones_like(leaf), A, B, B),
            "gated": lambda: seq.gated_linear(flat, wg, wg), "gated view": lambda: seq.gated_linear(leaf, wg, wg)}[op]
    flat = torch.randn(12, 8, generator=g).to(dev).requires_grad_()
    step = lambda: torch.autograd.grad(call().sum(), [flat if op == "gated" else leaf])[0]  # noqa: E731
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
        assert torch.equal(got, want)
        assert torch.equal(step(), want)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("R,D,N,G", [(700, 192, 16, 1), (1100, 65, 5, 1), (2050, 7, 33, 1), (360, 258, 64, 2), (2048, 64, 4, 1), (2047, 64, 4, 1)])
def test_scan_steps_of_many_rows(dev, seq, R, D, N, G, dtype):
    """Both sides of the rule that gives few rows a kernel of their own."""
    test_scan_steps_follow_the_definition(dev, seq, R, D, N, G, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,D,F", [(70, 64, 40), (200, 136, 72), (40, 24, 130), (33, 101, 99), (300, 37, 61)])
@pytest.mark.parametrize("off", ["x", "weights", "both"])
def test_gated_tensors_that_start_inside_a_chunk(dev, seq, M, D, F, dtype, off):
    """Whole rows whose first element is not 16-byte aligned, and rows that are not whole chunks: outputs and gradients against the definition.  With u
    half a step of the type and e = 2^-24: a product of n float terms is off by (2 n + 32) e of its terms, what D roundings move in the gate and the
    up side enters through e_*, a 16-bit d (dg, du) by u of its terms (twice u^2 where it is kept in two parts: not more), the result by u."""
    g = _gen(M + D)

    def place(t, shifted):
        t = t.to(dtype)
        buf = torch.zeros(t.numel() + 1, dtype=dtype, device=dev)
        out = buf[1:] if shifted else torch.zeros(t.numel(), dtype=dtype, device=dev)
        return out.copy_(t.reshape(-1)).view(t.shape)
    x, wg, wu = torch.randn(M, D, generator=g), torch.randn(F, D, generator=g) * D ** -0.5, torch.randn(F, D, generator=g) * D ** -0.5
    dy = torch.randn(M, F, generator=g).to(dtype)
    leaves = [place(x, off != "weights").requires_grad_()] + [place(w, off != "x").requires_grad_() for w in (wg, wu)]
    assert off == "weights" or leaves[0].data_ptr() % 16
    y = seq.gated_linear(*leaves)
    got = torch.autograd.grad(y, leaves, dy.to(dev))
    o = osq.gated_linear(*(t.to(dtype) for t in (x, wg, wu)), None, None, "silu", dy)
    u, e = (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2), 2.0 ** -24
    out_u = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    checks = [("y", y.detach(), o["m_y"] * (2 * D + 32) * e)]
    for name, have, n in (("dx", got[0], 2 * F), ("dw_gate", got[1], M), ("dw_up", got[2], M)):
        checks.append((name, have, o["r_" + name] * (1.01 * u + (2 * n + 32) * e) + o["e_" + name] * (2 * D + 32) * e + tiny * n))
    for name, have, exact in checks:
        bound = (o[name].abs() + exact) * out_u * 1.01 + exact + tiny
        off_by = (have.cpu().double() - o[name]).abs()
        assert (off_by <= bound).all(), (name, float((off_by / bound.clamp_min(1e-300)).max()))
