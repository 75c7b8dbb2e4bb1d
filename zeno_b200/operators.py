"""Operators of policies that act in batched worlds, on PyTorch CUDA tensors.

``delta_rule_step`` acts: one token for every environment, the memory of each updated in
place, cleared where the world reports the end of an episode.  ``delta_rule`` runs the
same recurrence over a stored rollout in chunks, with gradients, for learning.
``linear_attention_step`` and ``linear_attention`` are the same pair for a memory that adds and decays only,
``layer_norm`` normalises what such a memory returns and what is fed to it.
``orthogonalize`` is the Newton-Schulz step of the Muon optimiser for the matrices around
them.  The kernels are in libzeno.so and run on the current stream of the tensors' device;
there is no fallback.
"""
from __future__ import annotations

import struct
import threading
from contextlib import nullcontext
from importlib.machinery import ExtensionFileLoader
from importlib.util import module_from_spec, spec_from_loader
from pathlib import Path
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from ._ffi import _lib, ffi


_binding_lock = threading.Lock()
_torch = None


def _binding():
    """The compiled functions of the memory operators (csrc/torch_binding.cpp), loaded at the first call of one: the others need
    libzeno.so alone."""
    global _torch
    with _binding_lock:
        if _torch is not None:
            return _torch
        path = Path(__file__).resolve().parent / "lib" / "zeno_torch.so"
        if not path.exists():
            raise ImportError(f"{path} is missing: build it with `python -m zeno_b200.build` (it needs a PyTorch with CUDA and Python's headers)")
        try:
            loader = ExtensionFileLoader("zeno_torch", str(path))
            module = module_from_spec(spec_from_loader("zeno_torch", loader))
            loader.exec_module(module)
        except ImportError as e:
            raise ImportError(f"{path} does not load with PyTorch {torch.__version__}: build it again with `python -m zeno_b200.build` ({e})") from e
        _torch = module
        return module


_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_FLAGS = (torch.uint8, torch.bool)
_MAX_DIM = 128

Tensor = torch.Tensor

# The C structs as flat records: a call writes one in a single pack, a third of the time of
# filling it field by field.  ZenoTensor is a pointer and three strides.
_RULE = struct.Struct("@8IfI" + "P3q" * 6 + "2P" + "P3q" + "P")
_GRADS = struct.Struct("@P3qP" + "P3q" * 5 + "P")
assert _RULE.size == ffi.sizeof("ZenoDeltaRule") and _GRADS.size == ffi.sizeof("ZenoDeltaRuleGrads")
_RULE_PTR, _GRADS_PTR = ffi.typeof("ZenoDeltaRule*"), ffi.typeof("ZenoDeltaRuleGrads*")
_ADDRESS, _NO_TENSOR = ffi.typeof("void*"), (0, 0, 0, 0)


def _check(code: int, what: str) -> None:
    if code != 0:
        raise RuntimeError(f"{what} failed with error code {code}: {ffi.string(_lib.zeno_last_error()).decode()}")


def _stream(index: int):
    """The current stream of a device, as the C entries take it."""
    return ffi.cast(_ADDRESS, torch._C._cuda_getCurrentRawStream(index))


def _on(index: int):
    """A context in which the device is the current one."""
    return nullcontext() if torch.cuda.current_device() == index else torch.cuda.device(index)


def _refuse_tangents(what: str, *tensors: Optional[Tensor]) -> None:
    """The kernels see values alone: a tangent would be lost without a word."""
    if forward_ad._current_level >= 0 and any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivatives")


def _expect(name: str, x: Tensor, shape: Tuple[int, ...], dtypes, device: torch.device) -> None:
    if x.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(x.shape)}")
    if x.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {x.dtype}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, q on {device}")


def _check_inputs(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, reset: Optional[Tensor], lead: int):
    """``lead``: the axes in front of the heads (2: batch and tokens, 1: batch).  Returns the
    state's shape."""
    qs, vs, dtype, device = q.shape, v.shape, q.dtype, q.device
    if len(qs) != lead + 2 or len(vs) != lead + 2:
        axes = "[batch, tokens, heads, width]" if lead == 2 else "[batch, heads, width]"
        raise ValueError(f"q, k and v must be {axes}, got {tuple(qs)} and {tuple(vs)}")
    if device.type != "cuda":
        raise ValueError(f"expected CUDA tensors, got q on {device}")
    if dtype not in _DTYPES:
        raise TypeError(f"q must be float32 or bfloat16, got {dtype}")
    key_heads, dk = qs[lead:]
    heads, dv = vs[lead:]
    if not (1 <= dk <= _MAX_DIM and 1 <= dv <= _MAX_DIM):
        raise ValueError(f"head widths must be 1 to {_MAX_DIM}, got {dk} and {dv}")
    if key_heads < 1 or heads < 1 or heads % key_heads:
        raise ValueError(f"the {heads} value heads must be a multiple of the {key_heads} key heads")
    front = qs[:lead]
    gates = vs[:-1]
    _expect("k", k, qs, (dtype,), device)
    _expect("v", v, front + vs[lead:], (dtype,), device)
    _expect("g", g, gates, (torch.float32,), device)
    _expect("beta", beta, gates, (torch.float32,), device)
    if reset is not None:
        _expect("reset", reset, front, _FLAGS, device)
    return (qs[0], heads, dk, dv)


def _rows(x: Tensor) -> Tensor:
    """x, or a copy of it where its last axis is not contiguous."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _tokens(x: Optional[Tensor]):
    """A ZenoTensor of [batch, tokens, ...]."""
    if x is None:
        return _NO_TENSOR
    s = x.stride()
    return x.data_ptr(), s[0], s[1], s[2] if len(s) > 2 else 0


def _one_token(x: Optional[Tensor]):
    """A ZenoTensor of [batch, ...], a single token."""
    if x is None:
        return _NO_TENSOR
    s = x.stride()
    return x.data_ptr(), s[0], 0, s[1] if len(s) > 1 else 0


def _address(x: Optional[Tensor]) -> int:
    return 0 if x is None else x.data_ptr()


def _rule(tensor, q, k, v, g, beta, reset, initial, final, out, scale, normalize, saved=None):
    qs, vs = q.shape, v.shape
    return ffi.from_buffer(_RULE_PTR, _RULE.pack(
        qs[0], qs[1] if tensor is _tokens else 1, qs[-2], vs[-2], qs[-1], vs[-1], _DTYPES[q.dtype], bool(normalize), scale, 0,
        *tensor(q), *tensor(k), *tensor(v), *tensor(g), *tensor(beta), *tensor(reset), _address(initial), _address(final),
        *tensor(out), _address(saved)))


def _workspace(p, which: int, device: torch.device) -> Tuple[object, int, Optional[Tensor]]:
    n = _lib.zeno_delta_rule_workspace_bytes(p, which)
    if not n:
        return ffi.NULL, 0, None
    w = torch.empty(n, dtype=torch.uint8, device=device)
    return ffi.cast(_ADDRESS, w.data_ptr()), n, w


def _forward(q, k, v, g, beta, reset, initial, scale, normalize, save):
    out = torch.empty_like(v)
    if out.stride(-1) != 1:
        out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    device = q.device
    final = torch.empty((v.shape[0], v.shape[2], q.shape[3], v.shape[3]), dtype=torch.float32, device=device)
    p = _rule(_tokens, q, k, v, g, beta, reset, initial, final, out, scale, normalize)
    saved = None
    with _on(device.index):
        if save:
            saved = torch.empty(_lib.zeno_delta_rule_saved_bytes(p) // 4, dtype=torch.float32, device=device)
            p = _rule(_tokens, q, k, v, g, beta, reset, initial, final, out, scale, normalize, saved)
        at, n, _keep = _workspace(p, 0, device)
        _check(_lib.zeno_delta_rule_forward(p, at, n, _stream(device.index)), "delta_rule")
    return out, final, saved


class _DeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, reset, initial, scale, normalize):
        out, final, saved = _forward(q, k, v, g, beta, reset, initial, scale, normalize, True)
        ctx.save_for_backward(q, k, v, g, beta, reset, initial, saved)
        ctx.scale, ctx.normalize = scale, normalize
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out, d_final):
        q, k, v, g, beta, reset, initial, saved = ctx.saved_tensors
        if d_out is None:
            d_out = torch.zeros(v.shape, dtype=v.dtype, device=v.device)
        d_out = _rows(d_out)
        if d_final is not None:
            d_final = d_final.contiguous()
        p = _rule(_tokens, q, k, v, g, beta, reset, initial, None, d_out, ctx.scale, ctx.normalize, saved)
        grads = [torch.empty_like(x) for x in (q, k, v, g, beta)]
        grads = [y if i > 2 or y.stride(-1) == 1 else torch.empty(y.shape, dtype=y.dtype, device=y.device)
                 for i, y in enumerate(grads)]
        d_initial = torch.empty_like(initial) if initial is not None and ctx.needs_input_grad[6] else None
        d = ffi.from_buffer(_GRADS_PTR, _GRADS.pack(*_tokens(d_out), _address(d_final), *(x for y in grads for x in _tokens(y)),
                                                    _address(d_initial)))
        index = q.device.index
        with _on(index):
            at, n, _keep = _workspace(p, 1, q.device)
            _check(_lib.zeno_delta_rule_backward(p, d, at, n, _stream(index)), "delta_rule backward")
        return (*grads, None, d_initial, None, None)


def delta_rule(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, reset: Optional[Tensor] = None,
               initial_state: Optional[Tensor] = None, *, scale: Optional[float] = None,
               normalize: bool = True) -> Tuple[Tensor, Tensor]:
    """Gated delta rule over a rollout: ``(out [B, T, H, dv], final_state [B, H, dk, dv])``.

    For each environment and value head a state S [dk, dv] walks over the tokens::

        S = exp(g) * S          # zero where an episode begins
        u = beta * (v - S^T k)
        S = S + k u^T
        out = scale * S^T q

    ``q``, ``k`` [B, T, Hk, dk] and ``v`` [B, T, H, dv] are float32 or bfloat16 (one type),
    H a multiple of Hk (value head h reads key head h // (H // Hk)), widths up to 128.
    ``g`` (log decay) and ``beta`` [B, T, H] are float32.  ``reset`` [B, T] (uint8 or bool)
    marks the first token of an episode: the state in front of it is dropped, whatever it
    held.  ``initial_state`` [B, H, dk, dv] float32 is the state in front of the rollout
    (None: zero).  ``normalize`` divides q and k by sqrt(|x|^2 + 1e-6).  ``scale``
    defaults to dk ** -0.5.

    Any strides are taken (a time-major buffer's transposed view needs no copy) as long as
    the last axis is contiguous.  The state is held in 32 bits.  Gradients flow to q, k, v,
    g, beta and initial_state; they are sums in a fixed order, so they repeat bit for bit.
    (Once, and in reverse mode only.)  g's is a difference of sums over q, k and the state and
    carries their 32-bit error, which may exceed it where decays leave next to nothing.
    For the gradients a call keeps the state in front of every 32 tokens but the first,
    widths rounded up to 32, 64 or 128: 0.8 GB for 4096 x 128 tokens and 4 heads of 64 x 64.
    """
    state = _check_inputs(q, k, v, g, beta, reset, 2)
    if initial_state is not None:
        _expect("initial_state", initial_state, state, (torch.float32,), q.device)
        initial_state = initial_state.contiguous()
    _refuse_tangents("delta_rule", q, k, v, g, beta, initial_state)
    scale = q.shape[3] ** -0.5 if scale is None else float(scale)
    q, k, v = _rows(q), _rows(k), _rows(v)
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, g, beta, initial_state)):
        return _DeltaRule.apply(q, k, v, g, beta, reset, initial_state, scale, normalize)
    out, final, _ = _forward(q, k, v, g, beta, reset, initial_state, scale, normalize, False)
    return out, final


def delta_rule_step(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, state: Tensor, reset: Optional[Tensor] = None,
                    *, scale: Optional[float] = None, normalize: bool = True) -> Tensor:
    """One token of ``delta_rule`` for every environment, without gradients: returns out [B, H, dv].

    ``q``, ``k`` [B, Hk, dk], ``v`` [B, H, dv], ``g``, ``beta`` [B, H], ``reset`` [B] (a
    world's ``dones`` buffer can be passed as it is).  ``state`` [B, H, dk, dv] float32,
    contiguous, is updated in place, and autograd knows: a rollout that was given the same
    tensor as its initial state and is yet to be differentiated needs a clone of it."""
    _expect("state", state, _check_inputs(q, k, v, g, beta, reset, 1), (torch.float32,), q.device)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is updated in place")
    if torch.is_grad_enabled() and any(x.requires_grad for x in (q, k, v, g, beta, state)):
        raise RuntimeError("delta_rule_step has no gradients: call it under torch.no_grad(), and delta_rule to learn")
    _refuse_tangents("delta_rule_step", q, k, v, g, beta, state)
    scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    q, k, v = _rows(q), _rows(k), _rows(v)
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    p = _rule(_one_token, q, k, v, g, beta, reset, state, state, out, scale, normalize)
    index = q.device.index
    with _on(index):
        _check(_lib.zeno_delta_rule_step(p, _stream(index)), "delta_rule_step")
    if not state.is_inference():  # (those have no version, and are never saved for a backward pass)
        increment_version(state)
    return out


def linear_attention(q: Tensor, k: Tensor, v: Tensor, g: Tensor, reset: Optional[Tensor] = None,
                     initial_state: Optional[Tensor] = None, *, scale: Optional[float] = None) -> Tuple[Tensor, Tensor]:
    """Linear attention with a decay for each head over a rollout: ``(out [B, T, H, dv], final_state [B, H, dk, dv])``.

    For each environment and value head a state S [dk, dv] walks over the tokens::

        S = exp(g) * S          # zero where an episode begins
        S = S + k v^T
        out = scale * S^T q

    ``q``, ``k`` [B, T, Hk, dk] and ``v`` [B, T, H, dv] are float32 or bfloat16 (one type),
    H a multiple of Hk (value head h reads key head h // (H // Hk)), widths up to 128.  They are taken as they are: what
    bounds the keys (a norm, a feature map) is the caller's.
    ``g`` (log decay, float32) is [H], one for each head, or [B, T, H], a gate's.  ``reset`` [B, T] (uint8 or bool)
    marks the first token of an episode: the state in front of it is dropped, whatever it
    held.  ``initial_state`` [B, H, dk, dv] float32 is the state in front of the rollout
    (None: zero).  ``scale`` defaults to dk ** -0.5.

    Any strides are taken (a time-major buffer's transposed view needs no copy) as long as
    the last axis is contiguous.  The state and all sums are held in 32 bits.  Products with 32-bit values keep 24 bits of them where the result is 32-bit, 17
    where it is bfloat16, which its rounding covers 512 times.  Gradients flow to q, k, v, g and initial_state
    (once, and in reverse mode only); they are sums in a fixed order, so they repeat bit for bit.
    For the gradients a call keeps the state in front of every 64 tokens but the first (32 in float32, and of heads
    of up to 32 channels): 0.27 GB for 4096 x 128 tokens and 4 heads of 64 x 64 in bfloat16.
    """
    return (_torch or _binding()).linear_attention(q, k, v, g, reset, initial_state, scale)


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, g: Tensor, state: Tensor, reset: Optional[Tensor] = None,
                          *, scale: Optional[float] = None) -> Tensor:
    """One token of ``linear_attention`` for every environment, without gradients: returns out [B, H, dv].

    ``q``, ``k`` [B, Hk, dk], ``v`` [B, H, dv], ``g`` [H] or [B, H], ``reset`` [B] (a
    world's ``dones`` buffer can be passed as it is).  ``state`` [B, H, dk, dv] float32,
    contiguous, is updated in place, and autograd knows: a rollout that was given the same
    tensor as its initial state and is yet to be differentiated needs a clone of it."""
    return (_torch or _binding()).linear_attention_step(q, k, v, g, state, reset, scale)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, *, eps: float = 1e-5) -> Tensor:
    """Layer norm over the last axis: ``(x - mean) / sqrt(variance + eps) * weight + bias``, of x's type and shape.

    ``x`` [..., n] is float32 or bfloat16, of any strides (up to three leading axes need no copy while the last axis is
    contiguous; the result keeps a time-major order).  ``weight`` and ``bias`` [n] are float32 or of x's type, both of one
    type; None: 1 and 0.  Mean, variance and all sums are held in 32 bits; a row whose squares leave their range is taken in other
    units, so a finite row of any spread has a finite result (a row of no spread and ``eps`` 0 is 0 / 0).  Gradients flow to x, weight and bias (once,
    and in reverse mode only); they are sums in a fixed order, so they repeat bit for bit."""
    return (_torch or _binding()).layer_norm(x, weight, bias, eps)


def orthogonalize(update: Tensor, steps: int = 5) -> Tensor:
    """Newton-Schulz orthogonalisation of a matrix [..., m, n] (or a stack of them), as the
    Muon optimiser applies it to its momentum: ``X = M / |M|``, then ``steps`` times
    ``X = a X + (b A + c A A) X`` with ``A = X X^T`` and (a, b, c) = (3.4445, -4.7750,
    2.0315), on the transposed matrix where m > n.  float32 or bfloat16, any strides; the
    result is contiguous and of the same type, without a gradient."""
    if update.dim() < 2:
        raise ValueError(f"expected a matrix or a stack of matrices, got shape {tuple(update.shape)}")
    if update.device.type != "cuda":
        raise ValueError(f"expected a CUDA tensor, got one on {update.device}")
    if update.dtype not in _DTYPES:
        raise TypeError(f"update must be float32 or bfloat16, got {update.dtype}")
    if not 0 <= steps <= 100:
        raise ValueError(f"steps must be 0 to 100, got {steps}")
    _refuse_tangents("orthogonalize", update)
    m, n = update.shape[-2:]
    x = update.detach()
    x = x.unsqueeze(0) if x.dim() == 2 else x if x.dim() == 3 else x.reshape(-1, m, n)
    out = torch.empty(update.shape, dtype=update.dtype, device=update.device)
    if not update.numel():
        return out
    index = update.device.index
    with _on(index):
        dtype = _DTYPES[update.dtype]
        need = _lib.zeno_orthogonalize_workspace_bytes(x.shape[0], m, n, dtype)
        work = torch.empty(need, dtype=torch.uint8, device=update.device) if need else None
        _check(_lib.zeno_orthogonalize(ffi.cast(_ADDRESS, x.data_ptr()), x.stride(), ffi.cast(_ADDRESS, out.data_ptr()), x.shape[0], m, n,
                                       dtype, steps, ffi.cast(_ADDRESS, _address(work)), need, _stream(index)), "orthogonalize")
    return out
