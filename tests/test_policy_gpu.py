"""The recurrent policy on the operators (zeno_b200/policy.py) and its example on a world."""
import sys
from pathlib import Path

import pytest
import torch

from zeno_b200.policy import MemoryPolicy, Muon

import operators_plain as plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 1e-2)])
def test_acting_and_learning_give_the_same_actions(dtype, tol):
    # bfloat16: the two forms round the same memory reads to 8 bits, a few times 2^-8 of the action at most
    torch.manual_seed(0)
    E, T = 37, 45
    policy = MemoryPolicy(29, 8, hidden=64, heads=2, width=32, dtype=dtype).cuda()
    obs = torch.randn(E, T, 29, device="cuda")
    begins = (torch.rand(E, T, device="cuda") < 0.1).to(torch.uint8)
    state = policy.initial_state(E)
    acted = torch.stack([policy.act(obs[:, t], state, begins[:, t]) for t in range(T)], 1)
    actions, last = policy(obs, None, begins)
    assert plain.off(acted, actions) <= tol and plain.off(state, last) <= tol
    time_major = obs.transpose(0, 1).contiguous().transpose(0, 1)
    assert plain.off(policy(time_major, policy.initial_state(E), begins)[0], actions) <= tol


def test_learns_to_remember():
    """The target at the end of an episode is its first observation: no memory, no success."""
    torch.manual_seed(0)
    E, T = 256, 12
    policy = MemoryPolicy(4, 2, hidden=64, heads=2, width=32).cuda()
    optimiser = Muon(policy.parameters(), lr=0.02)
    losses = []
    for _ in range(150):
        obs = torch.randn(E, T, 4, device="cuda") * 0.3
        cue = torch.sign(torch.randn(E, 2, device="cuda"))
        obs[:, 0, :2], obs[:, 0, 2] = cue, 2.0
        actions, _ = policy(obs)
        loss = (actions[:, -1] - 0.5 * cue).square().mean()
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        losses.append(float(loss.detach()))
    # without the memory the best is the mean, a loss of 0.25
    assert sum(losses[-10:]) / 10 < 0.05, losses[-10:]


def test_muon_refuses():
    with pytest.raises(ValueError):
        Muon([torch.zeros(2, 2, device="cuda", requires_grad=True)], lr=-1.0)


def test_example_runs_on_a_world():
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    import memory_policy
    policy, means = memory_policy.run(envs=64, horizon=8, updates=2, log=None)
    assert len(means) == 2 and all(m == m for m in means)
    assert all(torch.isfinite(p).all() for p in policy.parameters())
