"""A recurrent policy over a world's observations, built on the operators: the gated delta rule
as its memory of the episode, Newton-Schulz orthogonalised updates for its matrices.

``MemoryPolicy.act`` takes one observation of every environment and updates their memories in
place; ``MemoryPolicy.forward`` runs a stored rollout with gradients.  Both give the same
actions for the same observations.  ``Muon`` is the optimiser step for the policy's
matrices.  ``examples/memory_policy.py`` runs them on a world.
"""
from __future__ import annotations

from typing import Iterable, Optional, Tuple

import torch
from torch import nn

from .operators import delta_rule, delta_rule_step, orthogonalize


class MemoryPolicy(nn.Module):
    """Observations to action means: a hidden layer, a gated delta-rule memory of ``heads`` heads
    of ``width`` x ``width``, and a bounded linear output.

    ``dtype`` is that of the memory's queries, keys and values (bfloat16 or float32); parameters, gates and the memory
    itself are float32."""

    def __init__(self, obs_dim: int, action_dim: int, hidden: int = 256, heads: int = 4, width: int = 64,
                 dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.heads, self.width, self.dtype = heads, width, dtype
        self.encode = nn.Linear(obs_dim, hidden)
        self.qkv = nn.Linear(hidden, 3 * heads * width, bias=False)
        self.gates = nn.Linear(hidden, 2 * heads)
        self.out = nn.Linear(hidden + heads * width, action_dim)

    def initial_state(self, num_envs: int, device=None) -> torch.Tensor:
        """An empty memory for every environment."""
        device = self.encode.weight.device if device is None else device
        return torch.zeros((num_envs, self.heads, self.width, self.width), device=device)

    def _inputs(self, obs: torch.Tensor):
        x = torch.tanh(self.encode(obs))
        q, k, v = self.qkv(x).to(self.dtype).unflatten(-1, (3, self.heads, self.width)).unbind(-3)
        decay, write = self.gates(x).unflatten(-1, (2, self.heads)).unbind(-2)
        # log decay of a sigmoid gate, biased to remember
        return x, q, k, v, nn.functional.logsigmoid(decay + 4.0), torch.sigmoid(write)

    def _actions(self, x: torch.Tensor, memory: torch.Tensor) -> torch.Tensor:
        return torch.tanh(self.out(torch.cat([x, memory.flatten(-2).to(x.dtype)], -1)))

    @torch.no_grad()
    def act(self, obs: torch.Tensor, state: torch.Tensor, begins: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Actions [E, action_dim] for observations [E, obs_dim].  ``state`` is updated in place (keep
        a clone for ``forward`` to start from); ``begins`` [E] marks environments whose observation
        is the first of an episode (the ``dones`` of the step that returned it, with automatic
        resets)."""
        x, q, k, v, g, beta = self._inputs(obs)
        return self._actions(x, delta_rule_step(q, k, v, g, beta, state, begins))

    def forward(self, obs: torch.Tensor, state: Optional[torch.Tensor] = None,
                begins: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Actions [E, T, action_dim] of a rollout [E, T, obs_dim] from ``state`` on, and the memory behind it."""
        x, q, k, v, g, beta = self._inputs(obs)
        memory, last = delta_rule(q, k, v, g, beta, begins, state)
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
