"""A recurrent policy over a world's observations, built on the operators: the gated delta rule, or linear attention with a
decay for each head between layer norms, as its memory of the episode, Newton-Schulz orthogonalised updates for its matrices.

``MemoryPolicy.act`` takes one observation of every environment and updates their memories in
place; ``MemoryPolicy.forward`` runs a stored rollout with gradients.  Both give the same
actions for the same observations.  ``Muon`` is the optimiser step for the policy's
matrices.  ``examples/memory_policy.py`` runs them on a world.
"""
from __future__ import annotations

import math
from typing import Iterable, Optional, Tuple

import torch
from torch import nn

from .operators import delta_rule, delta_rule_step, layer_norm, linear_attention, linear_attention_step, orthogonalize


class LayerNorm(nn.Module):
    """``operators.layer_norm`` over the last axis of ``width`` values, with a float32 weight and bias."""

    def __init__(self, width: int, eps: float = 1e-5):
        super().__init__()
        self.eps = eps
        self.weight, self.bias = nn.Parameter(torch.ones(width)), nn.Parameter(torch.zeros(width))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, eps=self.eps)


class MemoryPolicy(nn.Module):
    """Observations to action means: a hidden layer, a memory of ``heads`` heads
    of ``width`` x ``width``, and a bounded linear output.

    ``memory``: "delta", a gated delta rule (takes back what it holds under a key, gates for each token), or "decay",
    linear attention with a learned decay for each head, from memories of 4 tokens to ones of 256; its keys and values come from normalised
    features, what it returns is normalised head by head.
    ``dtype`` is that of the memory's queries, keys and values (bfloat16 or float32); parameters, gates and the memory
    itself are float32."""

    def __init__(self, obs_dim: int, action_dim: int, hidden: int = 256, heads: int = 4, width: int = 64,
                 dtype: torch.dtype = torch.bfloat16, memory: str = "delta"):
        super().__init__()
        if memory not in ("delta", "decay"):
            raise ValueError(f'memory must be "delta" or "decay", got {memory!r}')
        self.heads, self.width, self.dtype, self.memory = heads, width, dtype, memory
        self.encode = nn.Linear(obs_dim, hidden)
        self.qkv = nn.Linear(hidden, 3 * heads * width, bias=False)
        if memory == "delta":
            self.gates = nn.Linear(hidden, 2 * heads)
        else:
            # of the log decay -log(1 + exp(-x)): memories of 2^x tokens and one more
            self.decay = nn.Parameter(torch.linspace(2.0, 8.0, heads) * math.log(2.0))
            self.norm, self.read_norm = LayerNorm(hidden), LayerNorm(width)
        self.out = nn.Linear(hidden + heads * width, action_dim)

    def initial_state(self, num_envs: int, device=None) -> torch.Tensor:
        """An empty memory for every environment."""
        device = self.encode.weight.device if device is None else device
        return torch.zeros((num_envs, self.heads, self.width, self.width), device=device)

    def _inputs(self, obs: torch.Tensor):
        """Features, what the memory reads and writes, and its gates."""
        x = torch.tanh(self.encode(obs))
        q, k, v = self.qkv(x if self.memory == "delta" else self.norm(x)).to(self.dtype).unflatten(-1, (3, self.heads, self.width)).unbind(-3)
        if self.memory == "decay":
            return x, (q, k, v, nn.functional.logsigmoid(self.decay))
        decay, write = self.gates(x).unflatten(-1, (2, self.heads)).unbind(-2)
        # log decay of a sigmoid gate, biased to remember
        return x, (q, k, v, nn.functional.logsigmoid(decay + 4.0), torch.sigmoid(write))

    def _actions(self, x: torch.Tensor, memory: torch.Tensor) -> torch.Tensor:
        if self.memory == "decay":
            memory = self.read_norm(memory)
        return torch.tanh(self.out(torch.cat([x, memory.flatten(-2).to(x.dtype)], -1)))

    @torch.no_grad()
    def act(self, obs: torch.Tensor, state: torch.Tensor, begins: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Actions [E, action_dim] for observations [E, obs_dim].  ``state`` is updated in place (keep
        a clone for ``forward`` to start from); ``begins`` [E] marks environments whose observation
        is the first of an episode (the ``dones`` of the step that returned it, with automatic
        resets)."""
        x, inputs = self._inputs(obs)
        step = delta_rule_step if self.memory == "delta" else linear_attention_step
        return self._actions(x, step(*inputs, state, begins))

    def forward(self, obs: torch.Tensor, state: Optional[torch.Tensor] = None,
                begins: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Actions [E, T, action_dim] of a rollout [E, T, obs_dim] from ``state`` on, and the memory behind it."""
        x, inputs = self._inputs(obs)
        rule = delta_rule if self.memory == "delta" else linear_attention
        memory, last = rule(*inputs, begins, state)
        return self._actions(x, memory), last


class Muon(torch.optim.Optimizer):
    """Momentum whose update of each matrix is orthogonalised (``operators.orthogonalize``); other parameters take a plain
    momentum step.  ``params`` are the parameters or groups of them, as for any optimiser."""

    def __init__(self, params: Iterable, lr: float = 0.02, momentum: float = 0.95, steps: int = 5):
        if lr < 0 or not 0 <= momentum < 1:
            raise ValueError(f"lr must not be negative and momentum in [0, 1), got {lr} and {momentum}")
        super().__init__(params, dict(lr=lr, momentum=momentum, steps=steps))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state["momentum"] = torch.zeros_like(p)
                m = state["momentum"]
                m.mul_(group["momentum"]).add_(p.grad)
                update = p.grad.add(m, alpha=group["momentum"])
                if p.dim() >= 2:
                    rows, cols = p.shape[-2:]
                    update = orthogonalize(update, group["steps"]).mul_(max(1.0, rows / cols) ** 0.5)
                p.add_(update, alpha=-group["lr"])
        return loss
