"""What the C entries of linear attention and layer norm refuse, and the sizes they give (no GPU is touched before the
checks)."""
import re

import pytest
import torch

import zeno_b200
from zeno_b200._ffi import _lib, ffi

INVALID = -6
AT = 4096  # an address that is never read: each call is refused, or has no rows


def message():
    return ffi.string(_lib.zeno_last_error()).decode()


def attention(**kw):
    p = ffi.new("ZenoLinearAttention*")
    p.batch = p.tokens = p.key_heads = p.value_heads = 1
    p.key_dim = p.value_dim = 8
    for name in ("q", "k", "v", "g", "out"):
        getattr(p, name).data = ffi.cast("void*", AT)
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def attention_grads():
    d = ffi.new("ZenoLinearAttentionGrads*")
    for name in ("d_out", "d_q", "d_k", "d_v"):
        getattr(d, name).data = ffi.cast("void*", AT)
    return d


def norm(**kw):
    p = ffi.new("ZenoLayerNorm*")
    p.rows = (1, 1, 4)
    p.width = 8
    p.x.data = p.out.data = ffi.cast("void*", AT)
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def test_cpu_tensors_are_refused():
    x, g = torch.zeros(1, 2, 1, 8), torch.zeros(1)
    with pytest.raises(ValueError, match="CUDA"):
        zeno_b200.linear_attention(x, x, x, g)
    with pytest.raises(ValueError, match="CUDA"):
        zeno_b200.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], g, torch.zeros(1, 1, 8, 8))
    with pytest.raises(ValueError, match="CUDA"):
        zeno_b200.layer_norm(torch.zeros(3, 8))


@pytest.mark.parametrize("change,why", [
    (dict(dtype=7), "dtype"), (dict(key_dim=0), "key_dim"), (dict(key_dim=129), "key_dim"), (dict(value_dim=200), "value_dim"),
    (dict(key_heads=0), "heads"), (dict(key_heads=2, value_heads=3), "multiple"), (dict(batch=1 << 28), "2\\^27"),
    (dict(initial_state=ffi.cast("float*", AT + 2)), "aligned")])
def test_attention_entries_refuse(change, why):
    p, d = attention(**change), attention_grads()
    for call in (lambda: _lib.zeno_linear_attention_step(p, ffi.NULL), lambda: _lib.zeno_linear_attention_forward(p, ffi.NULL, 0, ffi.NULL),
                 lambda: _lib.zeno_linear_attention_backward(p, d, ffi.cast("void*", AT), 1 << 20, ffi.NULL)):
        assert call() == INVALID
        assert re.search(why, message()), message()


def test_attention_entries_refuse_missing_and_misaligned_data():
    for name in ("q", "k", "v", "g", "out"):
        for address, why in ((0, name), (AT + 1, "aligned")):
            p = attention()
            getattr(p, name).data = ffi.cast("void*", address)
            for call in (_lib.zeno_linear_attention_step, lambda p, s: _lib.zeno_linear_attention_forward(p, ffi.NULL, 0, s)):
                assert call(p, ffi.NULL) == INVALID and why in message()
    for name in ("d_out", "d_q", "d_k", "d_v"):
        d = attention_grads()
        getattr(d, name).data = ffi.NULL
        assert _lib.zeno_linear_attention_backward(attention(), d, ffi.cast("void*", AT), 1 << 20, ffi.NULL) == INVALID and name in message()
    for name in ("d_final", "d_initial", "d_decay"):
        d = attention_grads()
        setattr(d, name, ffi.cast("float*", AT + 1))
        assert _lib.zeno_linear_attention_backward(attention(), d, ffi.cast("void*", AT), 1 << 20, ffi.NULL) == INVALID and "aligned" in message()
    assert _lib.zeno_linear_attention_step(ffi.NULL, ffi.NULL) == INVALID
    assert _lib.zeno_linear_attention_forward(ffi.NULL, ffi.NULL, 0, ffi.NULL) == INVALID
    assert _lib.zeno_linear_attention_backward(attention(), ffi.NULL, ffi.NULL, 0, ffi.NULL) == INVALID
    for tokens in (0, 2):
        assert _lib.zeno_linear_attention_step(attention(tokens=tokens), ffi.NULL) == INVALID and "tokens" in message()


def test_attention_workspaces():
    p, d = attention(tokens=4096, value_heads=2), attention_grads()
    need = _lib.zeno_linear_attention_workspace_bytes(p, 0)
    assert need > 0
    assert _lib.zeno_linear_attention_forward(p, ffi.cast("void*", AT), need - 1, ffi.NULL) == INVALID and "too small" in message()
    assert _lib.zeno_linear_attention_forward(p, ffi.NULL, need, ffi.NULL) == INVALID and "NULL" in message()
    assert _lib.zeno_linear_attention_forward(p, ffi.cast("void*", AT + 4), need, ffi.NULL) == INVALID and "16 bytes" in message()
    need = _lib.zeno_linear_attention_workspace_bytes(p, 1)
    assert _lib.zeno_linear_attention_backward(p, d, ffi.cast("void*", AT), need, ffi.NULL) == INVALID and "saved is NULL" in message()
    p.saved = ffi.cast("float*", AT)
    assert _lib.zeno_linear_attention_backward(p, d, ffi.cast("void*", AT), need - 1, ffi.NULL) == INVALID and "too small" in message()
    assert _lib.zeno_linear_attention_backward(p, d, ffi.NULL, need, ffi.NULL) == INVALID and "NULL" in message()
    # the states in front of every 64 tokens but the first, of 32 in 32-bit calls and heads of up to 32 channels
    assert _lib.zeno_linear_attention_saved_bytes(attention(batch=3, tokens=130, value_heads=2, key_dim=37, dtype=1)) == 3 * 2 * 2 * 37 * 8 * 4
    assert _lib.zeno_linear_attention_saved_bytes(attention(batch=3, tokens=130, value_heads=2, key_dim=7, dtype=1)) == 3 * 2 * 4 * 7 * 8 * 4
    assert _lib.zeno_linear_attention_saved_bytes(attention(tokens=65)) == 2 * 8 * 8 * 4
    assert _lib.zeno_linear_attention_saved_bytes(attention(tokens=32)) == 0
    assert _lib.zeno_linear_attention_saved_bytes(attention(key_dim=0)) == 0
    assert _lib.zeno_linear_attention_workspace_bytes(attention(dtype=9), 1) == 0


def test_no_rows_is_not_an_error():
    assert _lib.zeno_linear_attention_step(attention(batch=0), ffi.NULL) == 0
    assert _lib.zeno_linear_attention_forward(attention(batch=0), ffi.NULL, 0, ffi.NULL) == 0
    assert _lib.zeno_linear_attention_backward(attention(batch=0), attention_grads(), ffi.NULL, 0, ffi.NULL) == 0
    assert _lib.zeno_layer_norm_forward(norm(rows=(3, 0, 1 << 40)), ffi.NULL) == 0
    assert _lib.zeno_layer_norm_backward(norm(rows=(3, 0, 4)), ffi.new("ZenoLayerNormGrads*"), ffi.NULL, 0, ffi.NULL) == 0


@pytest.mark.parametrize("change,why", [
    (dict(dtype=7), "dtype"), (dict(affine_dtype=1), "affine_dtype"), (dict(dtype=1, affine_dtype=2), "affine_dtype"), (dict(width=0), "width"),
    (dict(width=(1 << 30) + 1), "width"), (dict(rows=(1 << 16, 1 << 15, 2)), "rows"), (dict(rows=(1 << 63, 2, 1)), "rows"),
    (dict(weight=ffi.cast("void*", AT + 2)), "aligned"), (dict(bias=ffi.cast("void*", AT + 1)), "aligned"), (dict(saved=ffi.cast("float*", AT + 1)), "aligned")])
def test_norm_entries_refuse(change, why):
    p, d = norm(**change), ffi.new("ZenoLayerNormGrads*")
    d.d_out.data = ffi.cast("void*", AT)
    for call in (lambda: _lib.zeno_layer_norm_forward(p, ffi.NULL), lambda: _lib.zeno_layer_norm_backward(p, d, ffi.NULL, 0, ffi.NULL)):
        assert call() == INVALID
        assert re.search(why, message()), message()


def test_norm_entries_refuse_missing_data():
    p, d = norm(), ffi.new("ZenoLayerNormGrads*")
    assert _lib.zeno_layer_norm_forward(ffi.NULL, ffi.NULL) == INVALID
    assert _lib.zeno_layer_norm_backward(p, ffi.NULL, ffi.NULL, 0, ffi.NULL) == INVALID
    assert _lib.zeno_layer_norm_backward(p, d, ffi.NULL, 0, ffi.NULL) == INVALID and "d_out is NULL" in message()
    d.d_out.data = ffi.cast("void*", AT)
    assert _lib.zeno_layer_norm_backward(p, d, ffi.NULL, 0, ffi.NULL) == INVALID and "saved is NULL" in message()
    p.saved, d.d_weight = ffi.cast("float*", AT), ffi.cast("void*", AT)
    need = _lib.zeno_layer_norm_workspace_bytes(p)
    assert need >= 2 * 8 * 4
    assert _lib.zeno_layer_norm_backward(p, d, ffi.cast("void*", AT), need - 1, ffi.NULL) == INVALID and "too small" in message()
    assert _lib.zeno_layer_norm_backward(p, d, ffi.NULL, need, ffi.NULL) == INVALID and "NULL" in message()
    assert _lib.zeno_layer_norm_backward(p, d, ffi.cast("void*", AT + 4), need, ffi.NULL) == INVALID and "16 bytes" in message()
    d.d_x.data = ffi.cast("void*", AT + 1)
    assert _lib.zeno_layer_norm_backward(p, d, ffi.cast("void*", AT), need, ffi.NULL) == INVALID and "d_x" in message()
    p.out.data = ffi.NULL
    assert _lib.zeno_layer_norm_forward(p, ffi.NULL) == INVALID and "out is NULL" in message()
