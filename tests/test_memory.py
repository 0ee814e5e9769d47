"""The policy with memory (qqt_b200/memory.py): its operators run together.

Acting tick by tick gives what the unrolled rollout gives; the loss's
gradient with respect to every parameter equals that of the same network in
float64, written in elementary torch operations; a rollout and its update run
on the simulator.  Linear layers run in float32 (TF32 off), so activations of
order 1 carry about 1e-6, and the parameters' gradients, sums over a few
thousand rows, about 1e-5 of their largest value; 1e-4 is allowed.
"""

from __future__ import annotations

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from qqt_b200 import _capi
    from qqt_b200.memory import (HEADS, MemoryActorCritic, collect_memory, local_features,
                                 update_memory)
    from qqt_b200.policy_loss import policy_logp, policy_loss


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    yield
    torch.cuda.synchronize()
    assert _capi.device_error() == 0


def _case(t, n, f, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    torch.manual_seed(seed)
    model = MemoryActorCritic(f, 96).cuda()
    x = torch.randn((t, n, f), generator=g, device="cuda")
    state = torch.randn((n, 96), generator=g, device="cuda")
    reset = torch.rand((t, n), generator=g, device="cuda") < 0.05
    return model, x, state, reset, g


def test_ticks_equal_the_unrolled_rollout():
    model, x, state, reset, _ = _case(70, 33, 40)
    with torch.no_grad():
        logits, value, last = model.unroll(x, state, reset)
        s = state.clone()
        for t in range(70):
            lt, vt = model.step(x[t], s, reset[t])
            assert (lt - logits[t]).abs().max().item() <= 1e-4
            assert (vt - value[t]).abs().max().item() <= 1e-4
    assert (s - last).abs().max().item() <= 1e-4


def _plain_loss(m, x, state, reset, legal, act, old, adv, opt):
    """The same network and loss in elementary operations."""
    def norm(v, ln):
        c = v - v.mean(-1, keepdim=True)
        return c / ((c * c).mean(-1, keepdim=True) + ln.eps).sqrt() * ln.weight + ln.bias

    both = m.mix(norm(m.encode(x), m.norm_in))
    cand, gate = both.split(m.width, -1)
    f, h, hs = torch.sigmoid(gate), state, []
    for t in range(x.shape[0]):
        h = torch.where(reset[t][:, None], torch.zeros_like(h), h)
        h = f[t] * h + (1 - f[t]) * cand[t]
        hs.append(h)
    out = m.heads(norm(torch.stack(hs), m.norm_out)).flatten(0, 1)
    z = torch.where(legal, out[:, :-1], torch.full_like(out[:, :-1], -1e30))
    logp, ent = 0, 0
    for k, part in enumerate(z.split(HEADS, 1)):
        lp = torch.log_softmax(part, 1)
        logp = logp + lp.gather(1, act[:, k:k + 1])[:, 0]
        ent = ent - (lp.exp() * lp).sum(1)
    r = (logp - old).exp()
    pg = -torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv)
    q = old - logp
    return (pg + opt["kl_coef"] * (torch.expm1(q) - q) - opt["entropy_coef"] * ent).mean(), \
        out[:, -1]


def test_gradients_match_the_network_in_float64():
    t, n, f = 90, 20, 30
    model, x, state, reset, g = _case(t, n, f, 3)
    legal = torch.rand((t * n, 7), generator=g, device="cuda") < 0.7
    legal[:, [0, 5]] = True
    act = torch.zeros((t * n, 2), dtype=torch.int64, device="cuda")
    opt = dict(kl_coef=0.05, entropy_coef=0.02)
    with torch.no_grad():
        logits = model.unroll(x, state, reset)[0].flatten(0, 1)
        logp, _ = policy_logp(logits, act, legal, HEADS)
    step = torch.randn(t * n, generator=g, device="cuda")
    old = logp - torch.where(step.abs() < 1, 0.05 * step, 0.4 * torch.sign(step))
    adv = torch.randn(t * n, generator=g, device="cuda")
    w = torch.randn(t * n, generator=g, device="cuda") / (t * n)
    logits, value, _ = model.unroll(x, state, reset)
    loss, stats = policy_loss(logits.flatten(0, 1), act, old, adv, old, legal, heads=HEADS, **opt)
    (loss + (value.reshape(-1) * w).sum()).backward()
    wide = copy.deepcopy(model).double()
    wide.zero_grad()
    want, v64 = _plain_loss(wide, x.double(), state.double(), reset, legal, act, old.double(),
                            adv.double(), opt)
    (want + (v64 * w.double()).sum()).backward()
    assert abs(loss.item() - want.item()) <= 1e-5
    for (name, p), q in zip(model.named_parameters(), wide.parameters()):
        err = (p.grad.double() - q.grad).abs().max().item()
        assert err <= 1e-4 * q.grad.abs().max().item(), (name, err)


def test_rollout_and_update_on_the_simulator():
    from qqt_b200 import scenarios
    from qqt_b200.bots import make_bot
    from qqt_b200.config import SimConfig
    from qqt_b200.ppo import PPOConfig
    from qqt_b200.sim import B200Sim
    torch.manual_seed(0)
    n, T = 96, 40
    cfg = SimConfig(**scenarios.CFG2)
    sim = B200Sim(cfg, n, seed=1, template=scenarios.corridor_template(cfg, n, 1))
    bot = make_bot(sim, "random")
    sim.observe_and_mask()
    model = MemoryActorCritic(local_features(sim, 0).shape[1]).cuda()
    opt = torch.optim.Adam(model.parameters(), lr=1e-3)
    before = [p.detach().clone() for p in model.parameters()]
    data = collect_memory(sim, model, bot, T)
    # the log-probabilities of acting are those of the unrolled rollout
    with torch.no_grad():
        logits, value, last = model.unroll(data["features"], data["start"], data["reset"])
        logp, _ = policy_logp(logits.flatten(0, 1), data["act"].flatten(0, 1),
                              data["legal"].flatten(0, 1), HEADS)
    assert (logp - data["logp"].reshape(-1)).abs().max().item() <= 1e-3
    assert (value - data["val"]).abs().max().item() <= 1e-3
    assert (last - data["state"]).abs().max().item() <= 1e-3
    assert data["legal"].gather(2, data["act"][..., :1]).all()
    stats = update_memory(model, opt, data, PPOConfig(epochs=2, minibatches=3), kl_coef=0.02)
    assert all(torch.isfinite(torch.tensor(v)) for v in stats.values())
    assert stats["ent"] > 0 and any(not torch.equal(a, b) for a, b in zip(before, model.parameters()))
    data = collect_memory(sim, model, bot, T, data["state"], data["fresh"])
    assert torch.isfinite(data["logp"]).all()


def test_a_rollout_keeps_its_state_when_the_next_goes_on_from_it():
    """What collect_memory was given and has returned stays as it is: the same
    state can be collected from twice, and a rollout's last state is that of its
    own unroll after the next rollout too."""
    from qqt_b200 import scenarios
    from qqt_b200.bots import make_bot
    from qqt_b200.config import SimConfig
    from qqt_b200.sim import B200Sim
    torch.manual_seed(0)
    n = 64
    cfg = SimConfig(**scenarios.CFG2)
    sim = B200Sim(cfg, n, seed=1, template=scenarios.corridor_template(cfg, n, 1))
    bot = make_bot(sim, "random")
    sim.observe_and_mask()
    model = MemoryActorCritic(local_features(sim, 0).shape[1], 32).cuda()
    first = collect_memory(sim, model, bot, 5)
    kept = {k: v.clone() for k, v in first.items()}
    for _ in range(2):
        again = collect_memory(sim, model, bot, 5, first["state"], first["fresh"])
        assert torch.equal(again["start"], kept["state"])
        assert not torch.equal(again["state"], kept["state"])
    for k, v in kept.items():
        assert torch.equal(first[k], v), k
