"""A recurrent policy on Ant: act in every environment on the GPU, keep the rollout, learn from it.

    python examples/memory_policy.py [--envs 4096] [--horizon 32] [--updates 10]

Each update steps the world ``horizon`` times (the policy reads the observations where the world
wrote them, and the world reads the actions where the policy wrote them), then takes one
policy-gradient step through the whole rollout, memory included.  The learning rule is
the plainest one (returns-to-go against their mean, Gaussian actions of fixed width); the point is
how the pieces fit.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import zeno_b200
from zeno_b200 import scenes
from zeno_b200.policy import MemoryPolicy, Muon

NOISE = 0.2  # standard deviation of the actions around the policy's
DISCOUNT = 0.99


def run(envs: int = 4096, horizon: int = 32, updates: int = 10, seed: int = 0, log=print):
    torch.manual_seed(seed)
    device = torch.device("cuda")
    world = zeno_b200.ZenoWorld(mjcf_string=scenes.ant(), num_envs=envs, substeps=4)
    world.set_task(body=1, z_min=0.2, z_max=1.0, auto_reset=True, noise=0.1, seed=seed)
    stream = torch.cuda.Stream()
    world.set_stream(stream.cuda_stream)
    obs, rewards, dones = (torch.as_tensor(world.device_array(k), device=device) for k in ("observations", "rewards", "dones"))
    policy = MemoryPolicy(world.obs_dim, world.action_dim).to(device)
    optimiser = Muon(policy.parameters(), lr=0.01)
    state = policy.initial_state(envs)
    means = []
    # everything on the world's stream: a step is ordered behind the actions it reads
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        # time-major storage: the operators read its transposed views without a copy
        kept_obs = torch.empty((horizon, envs, world.obs_dim), device=device)
        kept_actions = torch.empty((horizon, envs, world.action_dim), device=device)
        kept_rewards = torch.empty((horizon, envs), device=device)
        begins = torch.zeros((horizon, envs), dtype=torch.uint8, device=device)
        ended = torch.zeros((horizon, envs), dtype=torch.uint8, device=device)
        last = torch.zeros(envs, dtype=torch.uint8, device=device)
        for update in range(updates):
            first_state = state.clone()
            for t in range(horizon):
                kept_obs[t], begins[t] = obs, last
                mean = policy.act(kept_obs[t], state, last)
                kept_actions[t] = mean + NOISE * torch.randn_like(mean)
                world.step_async(kept_actions[t])
                kept_rewards[t], ended[t] = rewards, dones
                last.copy_(dones)
            returns = torch.empty_like(kept_rewards)
            ahead = torch.zeros(envs, device=device)
            for t in reversed(range(horizon)):
                ahead = kept_rewards[t] + DISCOUNT * ahead * (ended[t] == 0)
                returns[t] = ahead
            advantage = (returns - returns.mean()) / (returns.std() + 1e-6)
            mean, _ = policy(kept_obs.transpose(0, 1), first_state, begins.transpose(0, 1))
            log_prob = -(kept_actions.transpose(0, 1) - mean).square().sum(-1) / (2 * NOISE ** 2)
            loss = -(advantage.T * log_prob).mean()
            optimiser.zero_grad()
            loss.backward()
            optimiser.step()
            means.append(float(kept_rewards.mean()))
            if log:
                log(f"update {update}: mean reward {means[-1]:.4f}, episodes ended {int(ended.sum())}")
    torch.cuda.synchronize()
    return policy, means


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--envs", type=int, default=4096)
    ap.add_argument("--horizon", type=int, default=32)
    ap.add_argument("--updates", type=int, default=10)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    run(a.envs, a.horizon, a.updates, a.seed)
