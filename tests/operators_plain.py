"""The policy operators in 64 bits, token by token, for the tests (plain torch, autograd)."""
import torch


def delta_rule(q, k, v, g, beta, reset=None, initial=None, scale=None, normalize=True):
    """(out, final state) in float64; q [B, T, Hk, dk], v [B, T, H, dv], g and beta [B, T, H]."""
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    B, T, H, dv = v.shape
    dk = q.shape[-1]
    if normalize:
        q = q / (q.square().sum(-1, keepdim=True) + 1e-6).sqrt()
        k = k / (k.square().sum(-1, keepdim=True) + 1e-6).sqrt()
    q = q.repeat_interleave(H // q.shape[2], 2) * (dk ** -0.5 if scale is None else scale)
    k = k.repeat_interleave(H // k.shape[2], 2)
    S = torch.zeros((B, H, dk, dv), dtype=torch.float64, device=v.device) if initial is None else initial.double()
    out = []
    for t in range(T):
        drop = torch.zeros((B, H), dtype=torch.bool, device=v.device)
        if reset is not None:
            drop = drop | (reset[:, t] != 0)[:, None]
        # a decay to nothing drops the state too; the unused branch stays finite for autograd
        gone = drop | (g[:, t].exp().float() == 0)
        alpha = torch.where(gone, torch.zeros_like(g[:, t]), torch.where(gone, torch.zeros_like(g[:, t]), g[:, t]).exp())
        S = torch.where(gone[..., None, None], torch.zeros_like(S), S) * alpha[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - torch.einsum("bhkv,bhk->bhv", S, k[:, t]))
        S = S + k[:, t, :, :, None] * u[:, :, None, :]
        out.append(torch.einsum("bhkv,bhk->bhv", S, q[:, t]))
    return (torch.stack(out, 1) if out else v.new_zeros(B, 0, H, dv)), S


def orthogonalize(m, steps=5):
    x = m.double()
    wide = x.shape[-2] <= x.shape[-1]
    x = x if wide else x.mT
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + 1e-7)
    a, b, c = 3.4445, -4.7750, 2.0315
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x if wide else x.mT


def off(x, y):
    """2-norm of the difference over that of y (over 1 where y is zero)."""
    x, y = x.detach().double(), y.detach().double()
    n = float(y.norm())
    return float((x - y).norm()) / (n if n else 1.0)
