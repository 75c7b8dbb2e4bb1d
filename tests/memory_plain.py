"""Linear attention and layer norm in 64 bits, for the tests (plain torch, autograd)."""
import torch


def linear_attention(q, k, v, g, reset=None, initial=None, scale=None):
    """(out, final state) in float64, token by token; q [B, T, Hk, dk], v [B, T, H, dv], g [H] or [B, T, H]."""
    q, k, v, g = (x.double() for x in (q, k, v, g))
    B, T, H, dv = v.shape
    dk = q.shape[-1]
    q = q.repeat_interleave(H // q.shape[2], 2) * (dk ** -0.5 if scale is None else scale)
    k = k.repeat_interleave(H // k.shape[2], 2)
    g = g.expand(B, T, H)
    S = torch.zeros((B, H, dk, dv), dtype=torch.float64, device=v.device) if initial is None else initial.double()
    out = []
    for t in range(T):
        gone = g[:, t].exp().float() == 0  # a decay to nothing drops the state too
        if reset is not None:
            gone = gone | (reset[:, t] != 0)[:, None]
        # the unused branch stays finite for autograd
        alpha = torch.where(gone, torch.zeros_like(g[:, t]), torch.where(gone, torch.zeros_like(g[:, t]), g[:, t]).exp())
        S = torch.where(gone[..., None, None], torch.zeros_like(S), S) * alpha[..., None, None]
        S = S + k[:, t, :, :, None] * v[:, t, :, None, :]
        out.append(torch.einsum("bhkv,bhk->bhv", S, q[:, t]))
    return (torch.stack(out, 1) if out else v.new_zeros(B, 0, H, dv)), S


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    x = x.double()
    x = x - x.mean(-1, keepdim=True)
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    y = y if weight is None else y * weight.double()
    return y if bias is None else y + bias.double()
