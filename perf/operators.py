"""The sequence operators that are measured: the causal convolution, the selective state-space scan and the gated linear unit of
fastdeepqlearning_amd.sequence, each as a training step over replay windows, as a prompt and as one step for every acting row.

`run` computes them in plain torch operations in 32 bits; with `own` set it calls the framework.  Tensors are time-major,
[T, rows, channels], as the replay samples its windows."""
import math

import torch
import torch.nn.functional as F

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # the update's replay windows (50 steps of 256 rows, 512 inner channels): forward and every gradient
        {"name": "conv windows train f32", "op": "conv_train", "type": "f32", "T": 50, "R": 256, "D": 512, "K": 4, "reset": 0.02},
        # three ragged prompts of a few thousand steps, an inner width that is no power of two, going on from a carried state
        {"name": "conv prompt bf16", "op": "conv", "type": "bf16", "T": 4099, "R": 3, "D": 1000, "K": 4, "reset": 0.001},
        # one acting step of 32 environments: latency
        {"name": "conv step f32", "op": "conv_step", "type": "f32", "R": 32, "D": 512, "K": 4, "reset": 0.05},
        # the same windows through the scan: forward and every gradient
        {"name": "scan windows train f32", "op": "scan_train", "type": "f32", "T": 50, "R": 256, "D": 512, "N": 16, "G": 1, "reset": 0.02},
        # few long sequences in training: the time axis has to be split to fill the card
        {"name": "scan long train bf16", "op": "scan_train", "type": "bf16", "T": 4096, "R": 2, "D": 1024, "N": 16, "G": 1, "reset": 0.001},
        # one long prompt of odd length, the state kept for the steps that follow
        {"name": "scan prompt bf16", "op": "scan", "type": "bf16", "T": 16383, "R": 1, "D": 1024, "N": 16, "G": 2, "reset": 0.0},
        # one acting step of 32 environments: latency
        {"name": "scan step f32", "op": "scan_step", "type": "f32", "R": 32, "D": 512, "N": 16, "G": 1, "reset": 0.05},
        # one step of many served rows with a wide state: the state's traffic
        {"name": "scan step wide bf16", "op": "scan_step", "type": "bf16", "R": 512, "D": 2048, "N": 64, "G": 1, "reset": 0.0},
        # one acting step of 32 environments: the weights' traffic and latency
        {"name": "gated rows f32", "op": "gated", "type": "f32", "M": 32, "D": 256, "F": 256, "act": "silu", "bias": True},
        # all rows of the replay windows in the update's own type: forward and every gradient
        {"name": "gated windows train f32", "op": "gated_train", "type": "f32", "M": 12800, "D": 512, "F": 256, "act": "silu", "bias": True},
        # a training batch of a wide block
        {"name": "gated train bf16", "op": "gated_train", "type": "bf16", "M": 8192, "D": 1024, "F": 4096, "act": "silu", "bias": False},
        # a forward pass with no size a multiple of a tile
        {"name": "gated ragged f16", "op": "gated", "type": "f16", "M": 4097, "D": 1000, "F": 2730, "act": "gelu", "bias": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv_train", "conv", "conv_step", "scan_train", "scan", "scan_step", "gated", "gated_train"])
    c = {"op": op, "type": rng.choice(["f32", "bf16", "f16"])}
    if op in ("conv_train", "conv"):
        c.update(R=_log(rng, 1, 300), D=_log(rng, 16, 2100), K=rng.choice([2, 3, 4]), reset=rng.choice([0.0, 0.01, 0.2]))
        c["T"] = _log(rng, 1, max(2, min(5000, 6500000 // (c["R"] * c["D"]))))
    elif op in ("scan_train", "scan"):
        c.update(R=_log(rng, 1, 300), N=rng.choice([4, 7, 8, 16, 24, 32]), G=rng.choice([1, 1, 2]), reset=rng.choice([0.0, 0.01, 0.2]))
        c["D"] = c["G"] * _log(rng, 16, 1024 // c["G"])
        c["T"] = _log(rng, 1, max(2, min(16000, 100000000 // (c["R"] * c["D"] * c["N"]))))
    elif op == "conv_step":
        c.update(R=_log(rng, 1, 512), D=_log(rng, 16, 2100), K=rng.choice([2, 3, 4]), reset=rng.choice([0.0, 0.1]))
    elif op == "scan_step":
        c.update(R=_log(rng, 1, 512), N=rng.choice([4, 7, 8, 16, 32, 64]), G=rng.choice([1, 1, 2]), reset=rng.choice([0.0, 0.1]))
        c["D"] = c["G"] * _log(rng, 16, 2048 // c["G"])
    else:
        c.update(D=_log(rng, 16, 1030), F=_log(rng, 16, 4100), act=rng.choice(["silu", "gelu", "sigmoid"]), bias=rng.choice([True, False]))
        most = (1 << 35) if c["type"] != "f32" else (1 << 32)
        c["M"] = _log(rng, 1, max(2, min(13000, most // (c["D"] * c["F"]) // (2 if op == "gated_train" else 1))))
    return c


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda").manual_seed(int(seed))
    dt = TYPES[c["type"]]
    op = c["op"]

    def normal(*shape, scale=1.0, to=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(to)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = {"case": dict(c)}
    if op.startswith("gated"):
        s["x"] = normal(c["M"], c["D"])
        s["w_gate"], s["w_up"] = (normal(c["F"], c["D"], scale=c["D"] ** -0.5) for _ in range(2))
        if c["bias"]:
            s["b_gate"], s["b_up"] = (normal(c["F"], scale=0.1) for _ in range(2))
        lead, out = [k for k in ("x", "w_gate", "w_up", "b_gate", "b_up") if k in s], (c["M"], c["F"])
    elif op.startswith("conv"):
        step = op == "conv_step"
        s["x"] = normal(*([] if step else [c["T"]]), c["R"], c["D"])
        s["weight"], s["bias"] = normal(c["D"], c["K"], scale=c["K"] ** -0.5, to=torch.float32), normal(c["D"], scale=0.1, to=torch.float32)
        s["reset"] = uniform(*s["x"].shape[:-1]) < c["reset"]
        s["state"] = normal(c["R"], c["K"] - 1, c["D"])
        lead, out = ["x", "weight", "bias"], tuple(s["x"].shape)
    else:
        step = op == "scan_step"
        t = [] if step else [c["T"]]
        s["x"], s["z"] = F.silu(normal(*t, c["R"], c["D"], to=torch.float32)).to(dt), normal(*t, c["R"], c["D"])
        s["dt"] = normal(*t, c["R"], c["D"], scale=0.5)
        s["A"] = -(1.0 + torch.arange(c["N"], device="cuda")).expand(c["D"], c["N"]) * (0.9 + 0.2 * uniform(c["D"], c["N"]))
        s["B"], s["C"] = (normal(*t, c["R"], c["G"], c["N"]) for _ in range(2))
        s["skip"] = 1.0 + normal(c["D"], scale=0.1, to=torch.float32)
        first = torch.exp(uniform(c["D"]) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        s["dt_bias"] = torch.log(torch.expm1(first))      # softplus of it is the first step size
        s["reset"] = uniform(*s["x"].shape[:-1]) < c["reset"]
        s["state"] = normal(c["R"], c["D"], c["N"], to=torch.float32)
        lead, out = ["x", "dt", "A", "B", "C", "skip", "z", "dt_bias"], tuple(s["x"].shape)
    s["train"] = lead if op.endswith("train") else []
    for k in s["train"]:
        s[k].requires_grad_()
    if s["train"]:
        s["d_out"] = normal(*out)
    if op.endswith("step"):
        s["out_state"] = torch.empty_like(s["state"])
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _act(g, kind):
    if kind == "silu":
        return g * torch.sigmoid(g)
    return torch.sigmoid(g) if kind == "sigmoid" else 0.5 * g * (1.0 + torch.erf(g * 0.5 ** 0.5))


def _gated(s):
    g, u = s["x"] @ s["w_gate"].t(), s["x"] @ s["w_up"].t()
    if "b_gate" in s:
        g, u = g + s["b_gate"], u + s["b_up"]
    return _act(g, s["case"]["act"]) * u


def _conv(s, state):
    """Output and the last K - 1 inputs; an input before a reset is as good as zero."""
    x, w, K = s["x"], s["weight"], s["weight"].shape[1]
    T = x.shape[0]
    full = torch.cat([state.transpose(0, 1), x])                                   # row t + K - 1 is step t
    runs = F.pad(torch.cumsum(s["reset"].long(), 0), (0, 0, K - 1, 0))             # sequences begun up to a step
    taps = [torch.where((runs[j:j + T] == runs[K - 1:]).unsqueeze(-1), full[j:j + T], 0.0) * w[:, j] for j in range(K)]
    pre = sum(taps) + s["bias"]
    kept = torch.where((runs[T:] == runs[-1]).unsqueeze(-1), full[T:], 0.0)
    return pre * torch.sigmoid(pre), kept.transpose(0, 1)


def _softplus(v):
    return v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))


def _terms(s):
    """Decay and input of the recurrence h <- decay * h + inp, [..., rows, channels, N]."""
    per = s["x"].shape[-1] // s["B"].shape[-2]
    B, C = (s[k].repeat_interleave(per, -2) for k in ("B", "C"))
    delta = _softplus(s["dt"] + s["dt_bias"])
    decay = torch.exp(delta.unsqueeze(-1) * s["A"])
    decay = torch.where(s["reset"][..., None, None], 0.0, decay)
    return decay, (delta * s["x"]).unsqueeze(-1) * B, C


def _gate(s, h, C):
    return ((h * C).sum(-1) + s["skip"] * s["x"]) * (s["z"] * torch.sigmoid(s["z"]))


def _scan(s, state):
    a, b, C = _terms(s)
    b = torch.cat([torch.addcmul(b[:1], a[:1], state), b[1:]])
    span = 1
    while span < b.shape[0]:        # after it, b holds the state of each step from the 2 * span steps up to it
        b = torch.cat([b[:span], torch.addcmul(b[span:], a[span:], b[:-span])])
        a = torch.cat([a[:span], a[span:] * a[:-span]])
        span *= 2
    return _gate(s, b, C), b[-1]


def _plain(s):
    op, dt = s["case"]["op"], TYPES[s["case"]["type"]]
    keep = {k: v for k, v in s.items() if not (isinstance(v, torch.Tensor) and v.is_floating_point())}
    p = dict(keep, **{k: v.detach().float().requires_grad_(k in s["train"]) for k, v in s.items() if k not in keep})
    with torch.set_grad_enabled(bool(s["train"])):
        if op.startswith("gated"):
            outs = {"y": _gated(p)}
        elif op == "conv_train":
            outs = {"y": _conv(p, torch.zeros_like(p["state"]))[0]}
        elif op == "conv":
            outs = dict(zip(("y", "state"), _conv(p, p["state"])))
        elif op == "conv_step":
            y, kept = _conv(dict(p, x=p["x"][None], reset=p["reset"][None]), p["state"])
            outs = {"y": y[0], "state": kept}
        elif op == "scan_train":
            outs = {"y": _scan(p, torch.zeros_like(p["state"]))[0]}
        elif op == "scan":
            outs = dict(zip(("y", "state"), _scan(p, p["state"])))
        else:
            a, b, C = _terms(p)
            h = a * p["state"] + b
            outs = {"y": _gate(p, h, C), "state": h}
    if s["train"]:
        grads = torch.autograd.grad(outs["y"], [p[k] for k in s["train"]], p["d_out"])
        outs.update({"d_" + k: v.to(s[k].dtype) for k, v in zip(s["train"], grads)})
    return {k: v.detach().to(s["state"].dtype if k == "state" else dt if k == "y" else v.dtype) for k, v in outs.items()}


# ---------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    from fastdeepqlearning_amd import sequence as seq
    c = s["case"]
    op = c["op"]
    outs = {}
    if op.startswith("gated"):
        outs["y"] = seq.gated_linear(s["x"], s["w_gate"], s["w_up"], s.get("b_gate"), s.get("b_up"), activation=c["act"])
    elif op == "conv_train":
        outs["y"] = seq.causal_conv(s["x"], s["weight"], s["bias"], reset=s["reset"])
    elif op == "conv":
        outs["y"], outs["state"] = seq.causal_conv(s["x"], s["weight"], s["bias"], reset=s["reset"], initial_state=s["state"], return_state=True)
    elif op == "conv_step":
        outs["y"], outs["state"] = seq.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], reset=s["reset"], out_state=s["out_state"])
    else:
        args = (s["x"], s["dt"], s["A"], s["B"], s["C"])
        kw = dict(skip=s["skip"], z=s["z"], dt_bias=s["dt_bias"], reset=s["reset"])
        if op == "scan_train":
            outs["y"] = seq.selective_scan(*args, **kw)
        elif op == "scan":
            outs["y"], outs["state"] = seq.selective_scan(*args, initial_state=s["state"], return_state=True, **kw)
        else:
            outs["y"], outs["state"] = seq.selective_scan_step(*args, s["state"], out_state=s["out_state"], **kw)
    if s["train"]:
        grads = torch.autograd.grad(outs["y"], [s[k] for k in s["train"]], s["d_out"])
        outs.update({"d_" + k: v for k, v in zip(s["train"], grads)})
    return {k: v.detach() for k, v in outs.items()}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    c, e = case, SIZE[case["type"]]
    op = c["op"]
    if op.startswith("gated"):
        w, x, h = 2 * c["D"] * c["F"], c["M"] * c["D"], c["M"] * c["F"]
        if op == "gated":
            return {"bytes": e * (w + x + h), "flops": 4 * c["M"] * c["D"] * c["F"]}
        return {"bytes": e * (2 * w + 2 * x + 2 * h), "flops": 12 * c["M"] * c["D"] * c["F"]}
    rows = c["R"] * c.get("T", 1)
    n = rows * c["D"]
    if op.startswith("conv"):
        K, st = c["K"], c["R"] * (c["K"] - 1) * c["D"]
        if op == "conv_train":
            return {"bytes": e * 4 * n + rows + 8 * c["D"] * (K + 1), "flops": n * (6 * K + 12)}
        return {"bytes": e * (2 * n + 2 * st) + rows + 4 * c["D"] * (K + 1), "flops": n * (2 * K + 4)}
    N, bc = c["N"], 2 * rows * c["G"] * c["N"]
    par = 4 * c["D"] * (N + 2)
    if op == "scan_train":
        return {"bytes": e * (8 * n + 2 * bc) + rows + 2 * par, "flops": n * (24 * N + 30)}
    return {"bytes": e * (4 * n + bc) + rows + par + 8 * c["R"] * c["D"] * N, "flops": n * (7 * N + 12)}


# ---------------------------------------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    train, op = s["train"], case["op"]
    v = {k: (t.detach().double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t) for k, t in s.items()}
    if op.startswith("gated"):
        return _exact_gated(v, train)
    if op.startswith("conv"):
        return _exact_conv(v, train, op)
    return _exact_scan(v, train, op)


def _exact_gated(v, train):
    kind = v["case"]["act"]
    zero = torch.zeros(v["w_gate"].shape[0], dtype=torch.float64, device="cuda")
    g = torch.addmm(v.get("b_gate", zero), v["x"], v["w_gate"].T)
    u = torch.addmm(v.get("b_up", zero), v["x"], v["w_up"].T)
    sg = 1 / (1 + torch.exp(-g))
    cdf = 0.5 * torch.erfc(-g / math.sqrt(2))
    f = {"silu": g * sg, "sigmoid": sg, "gelu": g * cdf}[kind]
    out = {"y": f * u}
    if train:
        df = {"silu": sg + g * sg * (1 - sg), "sigmoid": sg * (1 - sg), "gelu": cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)}[kind]
        dg, du = v["d_out"] * u * df, v["d_out"] * f
        out.update(d_x=dg @ v["w_gate"] + du @ v["w_up"], d_w_gate=dg.T @ v["x"], d_w_up=du.T @ v["x"])
        if "b_gate" in train:
            out.update(d_b_gate=dg.sum(0), d_b_up=du.sum(0))
    return out


def _exact_conv(v, train, op):
    x, w, K = v["x"], v["weight"], v["case"]["K"]
    x, reset = (x[None], v["reset"][None]) if op == "conv_step" else (x, v["reset"])
    window = torch.zeros_like(v["state"]) if train else v["state"].clone()
    window = torch.cat([torch.zeros_like(window[:, :1]), window], 1)
    y, pres, seen = torch.empty_like(x), [], []
    for t in range(x.shape[0]):
        window = torch.cat([window[:, 1:].masked_fill(reset[t][:, None, None], 0.0), x[t][:, None]], 1)
        pre = (window * w.T).sum(1) + v["bias"]
        y[t] = pre / (1 + torch.exp(-pre))
        if train:
            pres.append(pre)
            seen.append(window)
    if not train:
        return {"y": y[0] if op == "conv_step" else y, "state": window[:, 1:]}
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(v["bias"])
    for t in range(x.shape[0]):
        sg = 1 / (1 + torch.exp(-pres[t]))
        d = v["d_out"][t] * sg * (1 + pres[t] * (1 - sg))
        db += d.sum(0)
        dw += (d[:, None] * seen[t]).sum(0).T
        alive = torch.ones_like(reset[t])
        for back in range(K):
            if t - back < 0:
                break
            dx[t - back] += torch.where(alive[:, None], d * w[:, K - 1 - back], 0.0)
            alive = alive & ~reset[t - back]
    return {"y": y, "d_x": dx, "d_weight": dw, "d_bias": db}


def _exact_scan(v, train, op):
    one = op == "scan_step"
    x, dt, z, B, C, reset = ((v[k][None] if one else v[k]) for k in ("x", "dt", "z", "B", "C", "reset"))
    T, R, D = x.shape
    G, N = B.shape[-2:]
    A, skip = v["A"], v["skip"]
    raw = dt + v["dt_bias"]
    delta = torch.where(raw > 30, raw, torch.log1p(torch.exp(raw.clamp(max=30))))
    wide = lambda m: m.view(R, G, 1, N).expand(R, G, D // G, N).reshape(R, D, N)  # noqa: E731
    h = torch.zeros_like(v["state"]) if train else v["state"]
    core, hs = torch.empty_like(x), [h]
    for t in range(T):
        h = torch.exp(delta[t][..., None] * A) * h.masked_fill(reset[t][:, None, None], 0.0) + (delta[t] * x[t])[..., None] * wide(B[t])
        core[t] = (h * wide(C[t])).sum(-1)
        if train:
            hs.append(h)
    sz = 1 / (1 + torch.exp(-z))
    core = core + skip * x
    y = core * z * sz
    if not train:
        return {"y": y[0] if one else y, "state": h}
    dy = v["d_out"] * z * sz
    out = {"y": y, "d_z": v["d_out"] * core * sz * (1 + z * (1 - sz)), "d_skip": (dy * x).sum((0, 1)), "d_x": dy * skip,
           "d_dt": torch.empty_like(x), "d_A": torch.zeros_like(A), "d_B": torch.empty_like(B), "d_C": torch.empty_like(C)}
    carry = torch.zeros_like(h)
    for t in reversed(range(T)):
        g = carry + dy[t][..., None] * wide(C[t])
        ga = g * torch.exp(delta[t][..., None] * A)
        carry = ga.masked_fill(reset[t][:, None, None], 0.0)
        past = carry * hs[t]
        gb = (g * wide(B[t])).sum(-1)
        out["d_x"][t] += gb * delta[t]
        out["d_dt"][t] = (past * A).sum(-1) + gb * x[t]
        out["d_A"] += (past * delta[t][..., None]).sum(0)
        out["d_B"][t] = (g * (delta[t] * x[t])[..., None]).view(R, G, D // G, N).sum(2)
        out["d_C"][t] = (hs[t + 1] * dy[t][..., None]).view(R, G, D // G, N).sum(2)
    out["d_dt"] = out["d_dt"] / (1 + torch.exp(-raw))
    out["d_dt_bias"] = out["d_dt"].sum((0, 1))
    return out
