"""The policy on linear attention and layer norms (zeno_b200/policy.py): the operators together, as they are used."""
import sys
from pathlib import Path

import pytest
import torch

from zeno_b200.policy import MemoryPolicy, Muon

import memory_plain as plain
from operators_plain import off

pytestmark = pytest.mark.gpu


def exact(policy, obs, state, begins):
    """The policy's formulas in 64 bits on its parameters: actions and the memory behind them."""
    f = {name: p.detach().double().requires_grad_(True) for name, p in policy.named_parameters()}
    x = torch.tanh(obs.double() @ f["encode.weight"].T + f["encode.bias"])
    y = plain.layer_norm(x, f["norm.weight"], f["norm.bias"])
    q, k, v = (y @ f["qkv.weight"].T).unflatten(-1, (3, policy.heads, policy.width)).unbind(-3)
    memory, last = plain.linear_attention(q, k, v, torch.nn.functional.logsigmoid(f["decay"]), begins, state)
    read = plain.layer_norm(memory, f["read_norm.weight"], f["read_norm.bias"]).flatten(-2)
    return torch.tanh(torch.cat([x, read], -1) @ f["out.weight"].T + f["out.bias"]), last, f


def rollout(E=37, T=45, seed=0):
    torch.manual_seed(seed)
    return torch.randn(E, T, 29, device="cuda"), (torch.rand(E, T, device="cuda") < 0.1).to(torch.uint8)


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 1e-2)])
def test_acting_and_learning_give_the_same_actions(dtype, tol):
    # 32 bits: TF32 is off in the projections, which sum 256 terms at most; bfloat16: queries, keys, values and reads are rounded to 8 bits, a few
    # times 2^-8 of an action at most
    obs, begins = rollout()
    policy = MemoryPolicy(29, 8, hidden=64, heads=2, width=32, dtype=dtype, memory="decay").cuda()
    state = policy.initial_state(37)
    acted = torch.stack([policy.act(obs[:, t], state, begins[:, t]) for t in range(45)], 1)
    actions, last = policy(obs, None, begins)
    want, memory, _ = exact(policy, obs, None, begins)
    assert off(acted, actions) <= tol and off(state, last) <= tol
    assert off(actions, want) <= tol and off(last, memory) <= tol
    time_major = obs.transpose(0, 1).contiguous().transpose(0, 1)
    assert off(policy(time_major, policy.initial_state(37), begins)[0], actions) <= tol


def test_gradients_of_every_parameter():
    obs, begins = rollout(E=21, T=40, seed=1)
    policy = MemoryPolicy(29, 8, hidden=64, heads=2, width=32, dtype=torch.float32, memory="decay").cuda()
    state = torch.randn(21, 2, 32, 32, device="cuda")
    d_actions, d_last = torch.randn(21, 40, 8, device="cuda"), torch.randn(21, 2, 32, 32, device="cuda") * 0.01
    actions, last = policy(obs, state, begins)
    names = [name for name, _ in policy.named_parameters()]
    got = torch.autograd.grad([actions, last], [p for _, p in policy.named_parameters()], [d_actions, d_last])
    want_actions, want_last, f = exact(policy, obs, state, begins)
    want = torch.autograd.grad([want_actions, want_last], [f[n] for n in names], [d_actions.double(), d_last.double()])
    for name, a, b in zip(names, got, want):
        # 32-bit sums over 840 tokens through five layers of them
        assert off(a, b) <= 1e-4, (name, off(a, b))


def test_in_a_cuda_graph():
    """A training step captured after an eager one of the same parameters, replayed on another rollout."""
    obs, begins = rollout(E=700, T=20, seed=2)
    policy = MemoryPolicy(29, 8, hidden=64, heads=2, width=32, memory="decay").cuda()
    parameters = list(policy.parameters())

    def step(obs, begins):
        actions, _ = policy(obs, None, begins)
        return torch.autograd.grad(actions.square().mean(), parameters)
    other = rollout(E=700, T=20, seed=3)
    want = step(*other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(obs, begins)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(obs, begins)
    obs.copy_(other[0]), begins.copy_(other[1])
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert off(a, b) <= 1e-5  # (the projections' library products may choose another order in the graph)


def test_learns_with_muon():
    obs, begins = rollout(E=64, T=12, seed=4)
    policy = MemoryPolicy(29, 8, hidden=64, heads=2, width=32, memory="decay").cuda()
    optimiser = Muon(policy.parameters(), lr=0.02)
    before = [p.detach().clone() for p in policy.parameters()]
    for _ in range(3):
        loss = (policy(obs, None, begins)[0] - 0.5).square().mean()
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
    for p, b in zip(policy.parameters(), before):
        assert torch.isfinite(p).all() and not torch.equal(p, b)


def test_refusals_and_defaults():
    with pytest.raises(ValueError, match="memory"):
        MemoryPolicy(4, 2, memory="none")
    names = [name for name, _ in MemoryPolicy(4, 2).named_parameters()]
    assert names == ["encode.weight", "encode.bias", "qkv.weight", "gates.weight", "gates.bias", "out.weight", "out.bias"]


def test_example_runs_on_a_world():
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    import memory_policy
    policy, means = memory_policy.run(envs=64, horizon=8, updates=2, log=None, memory="decay")
    assert policy.memory == "decay" and len(means) == 2 and all(m == m for m in means)
    assert all(torch.isfinite(p).all() for p in policy.parameters())
