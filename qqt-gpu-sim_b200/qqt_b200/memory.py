"""A policy with memory over the local-view features, its rollout and its PPO
update.  It takes the place of the reference's recurrent policy (ActorCritic
arch="lstm" and its windowed update, train/ppo.py:440-535) with a gated
linear recurrence, whose whole rollout is one call in training:

    features -> Linear -> layer_norm -> Linear -> gated_recurrence
             -> layer_norm -> move, bomb and value heads

Acting advances the state one tick at a time (`gated_recurrence_step`);
training unrolls the rollout at once from the state that entered it, with
resets where an episode began, and takes the clipped loss with its KL term
straight from the logits (`policy_loss`).
"""

from __future__ import annotations

import torch
import torch.nn as nn

from .norm import LayerNorm
from .policy_loss import policy_logp, policy_loss
from .ppo import PPOConfig, gae
from .recurrence import gated_recurrence, gated_recurrence_step

HEADS = (5, 2)        # moves, bomb


def local_features(sim, pid: int, obs=None) -> torch.Tensor:
    """(N, F) float32: seat pid's local view, bomb and global features, side
    by side (sim/obs.py:241-340)."""
    parts = sim.local_view_features(obs, only_p0=pid == 0)
    return torch.cat([p[:, pid].reshape(sim.num_envs, -1) for p in parts], 1).float()


class MemoryActorCritic(nn.Module):
    """Actor-critic whose memory is a gated linear recurrence of `width`
    channels; the state is (N, width) float32, zero at an episode's start."""

    def __init__(self, n_features: int, width: int = 128):
        super().__init__()
        self.width = width
        self.encode = nn.Linear(n_features, width)
        self.norm_in = LayerNorm(width)
        self.mix = nn.Linear(width, 2 * width)         # candidate, gate
        self.norm_out = LayerNorm(width)
        self.heads = nn.Linear(width, sum(HEADS) + 1)  # move, bomb, value
        with torch.no_grad():
            self.mix.bias[width:] = 2.0                # remembers about eight ticks at first

    def initial_state(self, n: int) -> torch.Tensor:
        return torch.zeros((n, self.width), device=self.heads.weight.device)

    def _gates(self, features):
        both = self.mix(self.norm_in(self.encode(features)))
        return both[..., :self.width], both[..., self.width:]

    def _out(self, h):
        out = self.heads(self.norm_out(h))
        return out[..., :-1], out[..., -1]

    def unroll(self, features, state, reset):
        """(logits (T, N, 7), values (T, N), last state) for features (T, N, F),
        the state entering the first tick and reset (T, N): an episode begins."""
        h, last = gated_recurrence(*self._gates(features), state, reset)
        return (*self._out(h), last)

    @torch.no_grad()
    def step(self, features, state, reset):
        """(logits (N, 7), values (N,)) of one tick; `state` advances in place."""
        h, _ = gated_recurrence_step(*self._gates(features), state, reset, state_out=state)
        return self._out(h)


@torch.no_grad()
def sample(logits: torch.Tensor, legal: torch.Tensor, generator=None) -> torch.Tensor:
    """(N, 2) actions drawn from the legal places of both heads."""
    u = torch.rand(logits.shape, device=logits.device, generator=generator).clamp_(1e-7, 1 - 1e-7)
    z = logits.masked_fill(~legal, -torch.inf) - torch.log(-torch.log(u))
    return torch.stack([part.argmax(1) for part in z.split(HEADS, 1)], 1)


@torch.no_grad()
def collect_memory(sim, model: MemoryActorCritic, opponent, T: int, state=None, fresh=None,
                   pid: int = 0) -> dict:
    """A T-tick rollout of seat pid against `opponent` (a bot, on every other
    seat).  state, fresh: what the rollout before left under "state" and
    "fresh" (an episode has just begun); None starts anew."""
    n, dev = sim.num_envs, sim.device
    # (the ticks advance a state of this rollout's own in place)
    state = model.initial_state(n) if state is None else state.clone()
    fresh = torch.ones(n, dtype=torch.bool, device=dev) if fresh is None else fresh
    rows, start = [], state.clone()
    for _ in range(T):
        obs, mm, bm = sim.observe_and_mask()
        x = local_features(sim, pid, obs)
        legal = torch.cat([mm[:, pid], bm[:, pid]], 1).bool()
        logits, value = model.step(x, state, fresh)
        act = sample(logits, legal)
        logp, _ = policy_logp(logits, act, legal, HEADS)
        acts = torch.empty((n, sim.cfg.n_players, 2), dtype=torch.int64, device=dev)
        for p in range(sim.cfg.n_players):
            acts[:, p] = act if p == pid else opponent.act(obs, mm[:, p], bm[:, p], p)
        rew, done, _ = sim.step(acts, auto_reset=True)
        done = done.bool().clone()
        rows.append((x, legal, act, logp, value, rew[:, pid].clone(), done, fresh))
        fresh = done
    names = ("features", "legal", "act", "logp", "val", "rew", "done", "reset")
    data = {k: torch.stack(v) for k, v in zip(names, zip(*rows))}
    # the value after the last tick, without advancing the state
    x = local_features(sim, pid, sim.observe_and_mask()[0])
    data.update(start=start, state=state, fresh=fresh,
                last_val=model.step(x, state.clone(), fresh)[1])
    return data


def update_memory(model: MemoryActorCritic, opt, data: dict, cfg: PPOConfig,
                  entropy_coef: float = 0.03, kl_coef: float = 0.0, perm_fn=None) -> dict:
    """PPO over a rollout of `collect_memory`: every epoch goes through the
    sequences in minibatches, each unrolled over all ticks.  kl_coef weighs
    the KL term against the policy that collected.  Returns the means of the
    statistics."""
    adv, ret = gae(data["rew"].contiguous(), data["done"], data["val"].contiguous(),
                   data["last_val"], cfg.gamma, cfg.gae_lambda)
    adv = (adv - adv.mean()) / (adv.std() + 1e-8)
    T, n = adv.shape
    mb = max(1, -(-n // cfg.minibatches))
    dev = adv.device
    perm_fn = perm_fn or (lambda k: torch.randperm(k, device=dev))
    total, count = torch.zeros(6, device=dev), 0
    params = list(model.parameters())
    for _ in range(cfg.epochs):
        perm = perm_fn(n)
        for at in range(0, n, mb):
            s = perm[at:at + mb]
            # (kept as (T, rows, ...): a sequence's ticks stay together)
            d = {k: data[k][:, s] for k in ("features", "legal", "act", "logp", "val", "reset")}
            logits, value, _ = model.unroll(d["features"], data["start"][s], d["reset"])
            old = d["logp"].reshape(-1)
            pg, stats = policy_loss(logits.flatten(0, 1), d["act"].flatten(0, 1), old,
                                    adv[:, s].reshape(-1), old if kl_coef else None,
                                    d["legal"].flatten(0, 1), heads=HEADS, clip=cfg.clip_eps,
                                    kl_coef=kl_coef, entropy_coef=entropy_coef)
            r = ret[:, s]
            clipped = d["val"] + (value - d["val"]).clamp(-cfg.clip_eps, cfg.clip_eps)
            vf = 0.5 * torch.max((value - r) ** 2, (clipped - r) ** 2).mean()
            opt.zero_grad(set_to_none=True)
            (pg + cfg.value_coef * vf).backward()
            torch.nn.utils.clip_grad_norm_(params, cfg.max_grad_norm)
            opt.step()
            total += torch.cat([stats, vf.detach()[None]])
            count += 1
    names = ("loss", "pg", "kl", "ent", "clipfrac", "vf")
    return {k: float(v) / count for k, v in zip(names, total.tolist())}
