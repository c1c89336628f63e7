"""The state-space joiner (EncoderConf.JoinerModeEnum.ssm): causal convolution, selective scan and gated output layer inside the agent's
update step and act(), against the CPU oracle (oracle/update.py::ssm_joiner, autograd)."""
import numpy as np
import pytest
import torch

from test_gpu_facade import _conf
from test_gpu_parity import Report, _check_step, _snapshot, dev, logp_cond   # noqa: F401  (dev: fixture)

pytestmark = pytest.mark.gpu


def _agent(spec, device):
    from fastdeepqlearning_amd.core import NativeAgent, make_config
    cfg = make_config(spec.obs, spec.act, spec.T, spec.B, goal_dim=spec.goal, discrete=spec.discrete, n_critics=spec.C, n_quantiles=spec.Q,
                      latent=spec.latent, enc_features=spec.enc_features, enc_hidden=spec.enc_hidden, joint_hidden=spec.joint_hidden,
                      pi_hidden=spec.pi_hidden, critic_hidden=spec.critic_hidden, gamma=spec.gamma, tau=spec.tau, lr=spec.lr,
                      init_log_alpha=spec.init_log_alpha, drop_frac=spec.drop, burn_in_steps=spec.burn_in, joiner_ssm=True,
                      ssm_inner=spec.ssm_inner, ssm_state=spec.ssm_state, gru_state_mode=spec.ssm)
    return NativeAgent(cfg, device)


def _batch(spec, g):
    T, B, A = spec.T, spec.B, spec.act
    xp = {"obs_1d": torch.randn(T, B, spec.obs, generator=g), "action": torch.rand(T, B, A, generator=g) * 2 - 1,
          "reward": torch.randn(T, B, 1, generator=g), "mc_return": torch.randn(T, B, 1, generator=g) * 2,
          "task_done": (torch.rand(T, B, 1, generator=g) < 0.1).float(),
          "episode_step": (torch.arange(T).view(T, 1, 1) + torch.randint(0, 50, (1, B, 1), generator=g)).float()}
    if spec.discrete:
        xp["action"] = torch.randint(0, A, (T, B, 1), generator=g).float()
    xp["episode_step"][T // 2:, ::5] = 0.0
    if spec.ssm == "store":
        D, S = spec.ssm_dims
        xp["agent_state"] = torch.randn(T, B, 3 * D + D * S, generator=g) * 0.5
    noise = (torch.rand if spec.discrete else torch.randn)
    return xp, noise(T - 1, B, A, generator=g), noise(T - 1, B, A, generator=g)


NETS = dict(latent=64, enc_features=48, enc_hidden=(64,), joint_hidden=(64,), pi_hidden=(64,), critic_hidden=(64, 64))
CASES = [
    ("windows from zeros", dict(obs=9, act=3, C=2, Q=3, T=12, B=40, ssm="zero", **NETS)),
    ("stored start states, burn-in rows", dict(obs=9, act=3, C=2, Q=3, T=12, B=40, ssm="store", burn_in=2, **NETS)),
    ("two steps (one gradient step)", dict(obs=9, act=3, C=2, Q=3, T=2, B=33, ssm="store", **NETS)),
    ("odd widths: 21 latent, 18 features, 37 channels, 5 states", dict(obs=3, act=2, C=2, Q=3, T=5, B=7, ssm="store", ssm_inner=37, ssm_state=5,
                                                                       latent=21, enc_features=18, enc_hidden=(18,), joint_hidden=(33,),
                                                                       pi_hidden=(21,), critic_hidden=(33, 18))),
    ("64 states, discrete head", dict(obs=9, act=5, discrete=True, C=2, Q=3, T=9, B=24, ssm="zero", ssm_inner=64, ssm_state=64, **NETS)),
    ("windows of 50 steps, several gradient slabs", dict(obs=17, act=6, C=3, Q=2, T=50, B=128, ssm="zero", ssm_inner=128, **NETS)),
    ("long windows: the time axis in segments", dict(obs=9, act=3, C=2, Q=3, T=200, B=4, ssm="store", ssm_inner=40, **NETS)),
]


@pytest.mark.parametrize("name,kw", CASES, ids=[c[0] for c in CASES])
def test_update_matches_oracle(dev, name, kw):
    """One step: states, losses, every gradient, Adam."""
    from oracle import update as oup
    spec = oup.Spec(**kw)
    params = oup.init_params(spec, seed=5)
    st = oup.new_state(spec, params)
    ag = _agent(spec, dev)
    ag.load_tensors(params)
    xp, nt, na = _batch(spec, torch.Generator().manual_seed(9))
    alpha, log_alpha = st.alpha, float(st.params["actor_critic.log_alpha"])
    loss, aux = oup.train_step(st, spec, xp, nt, na)
    before = _snapshot(ag)
    ag.update({k: v.to(dev) for k, v in xp.items()}, nt.to(dev), na.to(dev))
    rep = Report("state-space joiner: " + name)
    ref = {k: (v.detach().numpy() if isinstance(v, torch.Tensor) else v) for k, v in aux.items() if k != "grad"}
    ref["loss"], ref["grad"] = float(loss), aux["grad"]
    ref["after"] = {n: st.params[n] for n in ag.tensors if "_frozen." not in n}
    _check_step(rep, 0, ag, spec, ref, before, alpha, log_alpha, 1)
    rep.finish()


@pytest.mark.parametrize("mode", ["zero", "store"])
def test_graph_mode_equals_eager(dev, mode):
    """The whole step captured into a graph and replayed, with other work on the stream between the replays: bit for bit the eager steps'
    parameters."""
    from oracle import update as oup
    spec = oup.Spec(obs=9, act=3, C=2, Q=3, T=16, B=24, ssm=mode, **NETS)
    params = oup.init_params(spec, seed=3)
    out = []
    xp, nt, na = _batch(spec, torch.Generator().manual_seed(4))
    xp, nt, na = {k: v.to(dev) for k, v in xp.items()}, nt.to(dev), na.to(dev)
    for graph in (False, True):
        ag = _agent(spec, dev)
        ag.load_tensors(params)
        ag.set_launch_mode(graph)
        for _ in range(5):
            ag.update(xp, nt, na)
            (torch.randn(64, 64, device=dev) @ torch.randn(64, 64, device=dev)).sum().item()
        if graph:
            assert ag.stats()["graph_launches"] >= 3
        out.append(ag.params.clone())
    assert torch.equal(out[0], out[1])


@pytest.mark.parametrize("rows,kw", [(1, {}), (5, {}), (33, {}), (300, {}), (9, dict(ssm_inner=37, ssm_state=5)), (40, dict(ssm_inner=37, ssm_state=5)), (17, dict(discrete=True, act=5)),
                                     (3, dict(ssm_inner=600, ssm_state=64, latent=256))])
def test_act_matches_oracle(dev, rows, kw):
    from oracle import update as oup
    base = dict(obs=17, act=6, C=3, Q=2, latent=64, enc_features=48, enc_hidden=(64,), joint_hidden=(48,), pi_hidden=(64,), critic_hidden=(32,),
                T=2, B=4, ssm="zero")
    base.update(kw)
    spec = oup.Spec(**base)
    params = oup.init_params(spec, seed=rows)
    gen = torch.Generator().manual_seed(rows)
    for k in params:
        params[k] = params[k] + 0.05 * torch.randn(params[k].shape, generator=gen)
    ag = _agent(spec, dev)
    ag.load_tensors(params)
    D, S = spec.ssm_dims
    assert ag.state_floats() == 3 * D + D * S
    xp = {"obs_1d": torch.randn(rows, spec.obs, generator=gen), "agent_state": torch.randn(rows, 3 * D + D * S, generator=gen) * 0.5,
          "exploit_mask": torch.rand(rows, 1, generator=gen) < 0.4}
    noise = torch.rand(rows, spec.act, generator=gen) if spec.discrete else torch.randn(rows, spec.act, generator=gen)
    rep = Report(f"state-space joiner act rows={rows} {kw}")
    for state in (xp["agent_state"], None):
        if state is None:
            xp.pop("agent_state")
        want = oup.act(params, spec, xp, noise)
        got = ag.act(xp["obs_1d"], None, None, xp["exploit_mask"], noise=noise, agent_state=state)
        rep.check("hidden_state", got[4], want[4])
        if spec.discrete:
            for i in (0, 2, 3):
                assert np.array_equal(got[i].cpu().numpy().astype(np.int64), want[i].numpy())
            rep.check("log_prob", got[1], want[1])
        else:
            for i, key in ((0, "action"), (2, "explore"), (3, "exploit")):
                rep.check(key, got[i], want[i])
            rep.check("log_prob", got[1], want[1], extra=logp_cond(want[2].numpy()))
    rep.finish()
    with pytest.raises(ValueError, match="agent_state"):
        ag.act(xp["obs_1d"], agent_state=torch.zeros(rows, 5))


def test_acting_step_by_step_gives_the_windows_states(dev):
    """The training pass over a window and act() carried through the same steps see the same states: the action's mean of every step
    (exploit action) equals the one computed from the window's latent states."""
    from oracle import update as oup
    spec = oup.Spec(obs=9, act=3, C=2, Q=3, T=12, B=6, ssm="zero", **NETS)
    params = oup.init_params(spec, seed=8)
    ag = _agent(spec, dev)
    ag.load_tensors(params)
    xp, nt, na = _batch(spec, torch.Generator().manual_seed(2))
    xp["task_done"].zero_()
    xp["episode_step"] = torch.arange(spec.T).view(-1, 1, 1).expand(spec.T, spec.B, 1).float().contiguous()
    state, seen = None, []
    for t in range(spec.T):
        r = ag.act(xp["obs_1d"][t], exploit_mask=torch.ones(spec.B, 1, dtype=torch.bool), agent_state=state)
        seen.append(r[3])
        state = r[4]
    with torch.no_grad():
        latent = oup.encoder(params, spec, xp)
        mean = oup.skip_head_mlp(params, "actor_critic.actor", latent, len(spec.pi_hidden)).chunk(2, -1)[0]
    rep = Report("state-space joiner: acting step by step")
    rep.check("exploit", torch.stack(seen), torch.tanh(mean))
    ag.update({k: v.to(dev) for k, v in xp.items()}, nt.to(dev), na.to(dev))
    rep.check("state", ag.debug("state", (spec.T, spec.B, spec.latent)), latent)
    rep.finish()


def test_agent_life_cycle(dev):
    """Through the facade: act() carries the state, the replay stores it, train_step starts its windows from the stored states."""
    from fastdeepqlearning_amd import Agent, Replay
    conf = _conf(dev, T=4, B=16)
    conf.num_instances = 1
    ec = conf.encoder_conf
    ec.joiner_mode = ec.JoinerModeEnum.ssm
    ec.ssm_inner_dim, ec.ssm_state_dim = 24, 4
    ec.rnn_latent_state_training_mode = ec.RnnLatentStateTrainMode.store
    try:
        read_heads, write_heads = Replay.make(conf)
        agent = Agent.make(conf)
        assert tuple(agent.state_dict()["encoder.joiner.sel_proj.weight"].shape) == (32, 24)
        h = agent.get_random_hidden()
        assert tuple(h.shape) == (24 * 7,) and not h.any()
        rng = np.random.RandomState(1)
        hidden = h.view(1, -1).to(dev)
        for ep in range(3):
            for i in range(60):
                obs = rng.standard_normal(5).astype(np.float32)
                action, hidden_next, info = agent.act({"obs_1d": torch.tensor(obs).view(1, -1), "agent_state": hidden,
                                                       "exploit_mask": torch.zeros(1, 1, dtype=torch.bool)})
                assert tuple(hidden_next.shape) == (1, 24 * 7) and not torch.equal(hidden_next, hidden)
                write_heads[0].add({"obs_1d": obs, "action": action[0].cpu().numpy(), "reward": float(rng.standard_normal()),
                                    "task_done": False, "episode_done": i == 59, "episode_step": i, "idx": 0,
                                    "agent_state": hidden[0].cpu().numpy()})
                hidden = hidden_next
        agent.enable_training(read_heads)
        before = {k: v.clone() for k, v in agent.state_dict().items()}
        for _ in range(2):
            agent.train_step()
        sc = agent.native.scalars()
        assert np.isfinite(sc["loss"]) and sc["step"] == 2
        after = agent.state_dict()
        for k in after:
            if k.startswith("encoder.joiner."):
                assert torch.isfinite(after[k]).all() and not torch.equal(before[k], after[k]), k
    finally:
        ec.joiner_mode = ec.JoinerModeEnum.feedforward      # EncoderConf attributes are class-level defaults
        ec.ssm_inner_dim, ec.ssm_state_dim = 0, 16
        ec.rnn_latent_state_training_mode = ec.RnnLatentStateTrainMode.zero


def test_stored_states_of_another_width_are_refused(dev):
    from oracle import update as oup
    spec = oup.Spec(obs=9, act=3, C=2, Q=3, T=4, B=8, ssm="store", **NETS)
    ag = _agent(spec, dev)
    ag.load_tensors(oup.init_params(spec, seed=1))
    xp, nt, na = _batch(spec, torch.Generator().manual_seed(1))
    xp = {k: v.to(dev) for k, v in xp.items()}
    for bad in (torch.zeros(4, 8, spec.latent, device=dev), xp["agent_state"][:, :3].contiguous()[:1]):
        with pytest.raises(ValueError, match="agent_state"):
            ag.update(dict(xp, agent_state=bad), nt.to(dev), na.to(dev))
    del xp["agent_state"]
    with pytest.raises(Exception, match="agent_state"):
        ag.update(xp, nt.to(dev), na.to(dev))
