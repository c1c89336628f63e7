"""State-space joiner without a GPU: configuration, refusals, tensor layout, the CPU definition against the operators' 64-bit ones."""
import ctypes as C

import pytest
import torch

from fastdeepqlearning_amd import _native as N
from fastdeepqlearning_amd.core import make_config
from oracle import sequence as os_
from oracle import update as oup


def _create(cfg):
    lib = N.load()
    h = C.c_void_p()
    rc = lib.fdql_agent_create(C.byref(h), C.byref(cfg))
    return lib, h, rc


def _config(**kw):
    base = dict(obs_dim=5, act_dim=2, T=4, B=6, latent=16, enc_features=12, enc_hidden=(8,), pi_hidden=(8,), critic_hidden=(8,), joiner_ssm=True,
                ssm_inner=20, ssm_state=6)
    base.update(kw)
    return make_config(**base)


def test_layout_and_state_width():
    lib, h, rc = _create(_config())
    assert rc == 0
    try:
        assert lib.fdql_agent_state_floats(h) == 20 * 3 + 20 * 6
        name, arena, off, shape = C.create_string_buffer(256), C.c_int32(), C.c_int64(), (C.c_int32 * 2)()
        got = {}
        for i in range(lib.fdql_agent_tensor_info(h, -1, None, 0, None, None, None)):
            lib.fdql_agent_tensor_info(h, i, name, 256, C.byref(arena), C.byref(off), shape)
            got[name.value.decode()] = tuple(s for s in shape if s)
        spec = oup.Spec(obs=5, act=2, C=2, Q=10, T=4, B=6, latent=16, enc_features=12, enc_hidden=(8,), pi_hidden=(8,), critic_hidden=(8,),
                        ssm="zero", ssm_inner=20, ssm_state=6)
        for n, s in oup.net_shapes(spec, "encoder.joiner"):
            assert got[n] == s, n
    finally:
        lib.fdql_agent_destroy(h)
    for kw, width in ((dict(joiner_ssm=False), 0), (dict(joiner_ssm=False, joiner_gru=True), 16)):
        lib, h, rc = _create(_config(**kw))
        assert rc == 0 and lib.fdql_agent_state_floats(h) == width
        lib.fdql_agent_destroy(h)


@pytest.mark.parametrize("field,value", [("joiner_gru", 1), ("ssm_inner", 0), ("ssm_inner", -3), ("ssm_state", 0), ("ssm_state", 65),
                                         ("gru_state_mode", 2), ("gru_state_mode", -1), ("ssm_inner", 1 << 17)])
def test_refusals(field, value):
    cfg = _config()
    setattr(cfg, field, value)
    lib, h, rc = _create(cfg)
    assert rc != 0 and lib.fdql_last_error()


def test_defaults():
    c = make_config(5, 2, 4, 6, enc_features=48, joiner_ssm=True, gru_state_mode="store")
    assert (c.joiner_ssm, c.ssm_inner, c.ssm_state, c.gru_state_mode, c.joiner_gru) == (1, 96, 16, 1, 0)
    c = make_config(5, 2, 4, 6)
    assert (c.joiner_ssm, c.ssm_inner, c.gru_state_mode) == (0, 0, 0)


def test_definition_agrees_with_the_operators():
    """oracle/update.py's step loop against the operators' own 64-bit definitions (hand-written adjoints): output, state, gradients."""
    spec = oup.Spec(obs=5, act=2, C=2, Q=2, T=7, B=3, latent=6, enc_features=8, ssm="store", ssm_inner=10, ssm_state=4)
    D, S = spec.ssm_dims
    g = torch.Generator().manual_seed(1)
    p = {n: torch.randn(s, generator=g, dtype=torch.float64) * 0.4 for n, s in oup.net_shapes(spec, "encoder.joiner")}
    for v in p.values():
        v.requires_grad_()
    e = torch.randn(7, 3, 8, generator=g, dtype=torch.float64)
    h0 = torch.randn(3, 3 * D + D * S, generator=g, dtype=torch.float64)
    reset = torch.rand(7, 3, generator=g) < 0.3
    out, state = oup.ssm_joiner(p, spec, e, h0, reset)
    dout = torch.randn(out.shape, generator=g, dtype=torch.float64)
    (out * dout).sum().backward()
    w = {k.split(".", 2)[2]: v.detach() for k, v in p.items()}
    xz = e @ w["in_proj.weight"].t() + w["in_proj.bias"]
    u, z = xz.chunk(2, -1)
    cv = os_.causal_conv(u, w["conv.weight"], w["conv.bias"], h0[:, :3 * D].view(3, 3, D), reset)
    sel = cv["y"] @ w["sel_proj.weight"].t()
    dt, Bt, Ct = sel.split([D, S, S], -1)
    A = -w["A_log"].exp()
    args = (cv["y"], dt, A, Bt[:, :, None], Ct[:, :, None], w["skip"], z, w["dt_bias"], True, h0[:, 3 * D:].view(3, D, S), reset)
    sc = os_.selective_scan(*args)
    y = sc["y"].reshape(21, D)
    gl = os_.gated_linear(y, w["gate_proj.weight"], w["up_proj.weight"], w["gate_proj.bias"], w["up_proj.bias"], "silu", dout.reshape(21, 6))
    close = lambda a, b: torch.allclose(a, b, rtol=1e-10, atol=1e-12)
    assert close(out.detach(), gl["y"].view(7, 3, 6))
    assert close(state.detach(), torch.cat([cv["state"].reshape(3, -1), sc["state"].reshape(3, -1)], 1))
    sc = os_.selective_scan(*args, dy=gl["dx"].view(7, 3, D))
    dx = sc["dx"] + torch.cat([sc["ddt"], sc["dB"].squeeze(2), sc["dC"].squeeze(2)], -1) @ w["sel_proj.weight"]
    cv = os_.causal_conv(u, w["conv.weight"], w["conv.bias"], h0[:, :3 * D].view(3, 3, D), reset, dy=dx)
    for name, want in (("gate_proj.weight", gl["dw_gate"]), ("up_proj.bias", gl["db_up"]), ("skip", sc["dskip"]), ("dt_bias", sc["ddt_bias"]),
                       ("A_log", sc["dA"] * A), ("conv.weight", cv["dweight"]), ("conv.bias", cv["dbias"])):
        assert close(p["encoder.joiner." + name].grad, want), name


def test_sizes_past_the_operators_limits_are_refused():
    """What fdql_scan would refuse as more than one launch is refused when the agent is made."""
    lib, h, rc = _create(_config(T=2, B=1 << 20, ssm_inner=1 << 16, latent=4, enc_features=4))
    assert rc != 0 and b"one launch" in lib.fdql_last_error()
