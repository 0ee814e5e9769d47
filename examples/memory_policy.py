"""Trains a policy with memory against the random bot for a few rollouts:

    python examples/memory_policy.py [--envs 1024] [--ticks 128] [--rollouts 5]

Each rollout steps the simulator and the policy's memory tick by tick; each
update unrolls all ticks at once (layer norm, gated recurrence and the
clipped policy loss with its KL term on the package's kernels).
"""

import argparse
import os
import sys
import time

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..",
                                "qqt-gpu-sim_b200"))

import torch  # noqa: E402

from qqt_b200 import scenarios  # noqa: E402
from qqt_b200.bots import make_bot  # noqa: E402
from qqt_b200.config import SimConfig  # noqa: E402
from qqt_b200.memory import (MemoryActorCritic, collect_memory, local_features,  # noqa: E402
                             update_memory)
from qqt_b200.ppo import PPOConfig  # noqa: E402
from qqt_b200.sim import B200Sim  # noqa: E402


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__,
                                 formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--envs", type=int, default=1024)
    ap.add_argument("--ticks", type=int, default=128)
    ap.add_argument("--rollouts", type=int, default=5)
    a = ap.parse_args()
    torch.manual_seed(0)
    cfg = SimConfig(**scenarios.CFG2)
    sim = B200Sim(cfg, a.envs, seed=1, template=scenarios.corridor_template(cfg, a.envs, 1))
    bot = make_bot(sim, "random")
    sim.observe_and_mask()
    model = MemoryActorCritic(local_features(sim, 0).shape[1]).cuda()
    opt = torch.optim.Adam(model.parameters(), lr=1e-3)
    state = fresh = None
    for k in range(a.rollouts):
        t0 = time.perf_counter()
        data = collect_memory(sim, model, bot, a.ticks, state, fresh)
        state, fresh = data["state"], data["fresh"]
        stats = update_memory(model, opt, data, PPOConfig(), kl_coef=0.02)
        print(f"rollout {k}: reward per tick {data['rew'].mean().item():+.4f}  "
              + "  ".join(f"{n} {v:.4f}" for n, v in stats.items())
              + f"  ({time.perf_counter() - t0:.2f} s)")


if __name__ == "__main__":
    main()
