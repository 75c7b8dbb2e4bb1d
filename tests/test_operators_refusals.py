"""What the policy operators refuse: arguments in Python (checked before anything runs) and
at the C entries (no GPU is touched before the checks)."""
import pytest
import torch

import zeno_b200
from zeno_b200._ffi import _lib, ffi

INVALID = -6


def fake(shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    x = fake((1, 2, 1, 8))
    with pytest.raises(ValueError, match="CUDA"):
        zeno_b200.delta_rule(x, x, x, fake((1, 2, 1)), fake((1, 2, 1)))
    y = fake((1, 1, 8))
    with pytest.raises(ValueError, match="CUDA"):
        zeno_b200.delta_rule_step(y, y, y, fake((1, 1)), fake((1, 1)), fake((1, 1, 8, 8)))
    with pytest.raises(ValueError, match="CUDA"):
        zeno_b200.orthogonalize(fake((4, 4)))
    with pytest.raises(ValueError, match="matrix"):
        zeno_b200.orthogonalize(fake((4,)))


def arguments(**kw):
    p = ffi.new("ZenoDeltaRule*")
    p.batch = p.tokens = p.key_heads = p.value_heads = 1
    p.key_dim = p.value_dim = 8
    for name in ("q", "k", "v", "g", "beta", "out"):  # never read: each call below is refused, or has no rows
        getattr(p, name).data = ffi.cast("void*", 4096)
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def message():
    return ffi.string(_lib.zeno_last_error()).decode()


@pytest.mark.parametrize("change,why", [
    (dict(dtype=7), "dtype"), (dict(key_dim=0), "key_dim"), (dict(key_dim=129), "key_dim"), (dict(value_dim=200), "value_dim"),
    (dict(key_heads=0), "heads"), (dict(key_heads=2, value_heads=3), "multiple"), (dict(batch=1 << 28), "2\\^27"),
    (dict(initial_state=ffi.cast("float*", 4098)), "aligned")])
def test_c_entries_refuse(change, why):
    p = arguments(**change)
    d = ffi.new("ZenoDeltaRuleGrads*")
    for call in (lambda: _lib.zeno_delta_rule_step(p, ffi.NULL),
                 lambda: _lib.zeno_delta_rule_forward(p, ffi.NULL, 0, ffi.NULL),
                 lambda: _lib.zeno_delta_rule_backward(p, d, ffi.NULL, 0, ffi.NULL)):
        assert call() == INVALID
        import re
        assert re.search(why, message()), message()


def test_c_entries_refuse_missing_and_misaligned_data():
    for name in ("q", "k", "v", "g", "beta", "out"):
        p = arguments()
        getattr(p, name).data = ffi.NULL
        assert _lib.zeno_delta_rule_forward(p, ffi.NULL, 0, ffi.NULL) == INVALID and name in message()
        p = arguments()
        getattr(p, name).data = ffi.cast("void*", 4097)
        assert _lib.zeno_delta_rule_step(p, ffi.NULL) == INVALID and "aligned" in message()
    assert _lib.zeno_delta_rule_step(ffi.NULL, ffi.NULL) == INVALID
    assert _lib.zeno_delta_rule_forward(ffi.NULL, ffi.NULL, 0, ffi.NULL) == INVALID
    assert _lib.zeno_delta_rule_backward(arguments(), ffi.NULL, ffi.NULL, 0, ffi.NULL) == INVALID
    d = ffi.new("ZenoDeltaRuleGrads*")
    d.d_out.data = ffi.cast("void*", 4096)
    assert _lib.zeno_delta_rule_backward(arguments(), d, ffi.NULL, 0, ffi.NULL) == INVALID and "d_q" in message()


def test_sizes_are_known_without_a_gpu():
    p = arguments(batch=3, tokens=100, key_heads=2, value_heads=4, key_dim=64, value_dim=64)
    # the states in front of the chunks after the first: 3 of 4 chunks of 32 tokens
    assert _lib.zeno_delta_rule_saved_bytes(p) == 3 * 4 * 3 * 64 * 64 * 4
    assert _lib.zeno_delta_rule_saved_bytes(arguments(tokens=32)) == 0
    assert _lib.zeno_delta_rule_saved_bytes(arguments(key_dim=0)) == 0
    assert _lib.zeno_orthogonalize_workspace_bytes(1, 100, 290, 0) > 0
    assert _lib.zeno_orthogonalize_workspace_bytes(1, 100, 290, 9) == 0


def test_no_rows_is_not_an_error():
    assert _lib.zeno_delta_rule_step(arguments(batch=0), ffi.NULL) == 0
    assert _lib.zeno_delta_rule_forward(arguments(batch=0), ffi.NULL, 0, ffi.NULL) == 0


def test_orthogonalize_entry_refuses():
    s = ffi.new("int64_t[3]", [64, 8, 1])
    at = ffi.cast("void*", 4096)
    big = 1 << 30
    call = _lib.zeno_orthogonalize
    assert call(at, s, at, 1, 8, 8, 5, 5, at, big, ffi.NULL) == INVALID and "dtype" in message()
    assert call(at, s, at, 1, 8, 8, 0, 101, at, big, ffi.NULL) == INVALID and "steps" in message()
    assert call(at, s, at, 70000, 8, 8, 0, 5, at, big, ffi.NULL) == INVALID and "matrices" in message()
    assert call(ffi.NULL, s, at, 1, 8, 8, 0, 5, at, big, ffi.NULL) == INVALID
    assert call(at, s, at, 1, 100, 100, 0, 5, at, 16, ffi.NULL) == INVALID and "workspace" in message()
    assert call(at, s, ffi.cast("void*", 4097), 1, 8, 8, 0, 5, at, big, ffi.NULL) == INVALID and "aligned" in message()
    assert call(ffi.NULL, ffi.NULL, ffi.NULL, 0, 8, 8, 0, 5, ffi.NULL, 0, ffi.NULL) == 0


@pytest.mark.gpu
def test_python_refusals_on_the_gpu():
    def t(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype, device="cuda")
    q, v, g = t(2, 3, 2, 8), t(2, 3, 4, 16), t(2, 3, 4)
    zeno_b200.delta_rule(q, q, v, g, g)
    rule = zeno_b200.delta_rule
    with pytest.raises(ValueError, match="k must have shape"):
        rule(q, t(2, 3, 2, 9), v, g, g)
    with pytest.raises(TypeError, match="k must be"):
        rule(q, q.bfloat16(), v, g, g)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        rule(q.half(), q.half(), v.half(), g, g)
    with pytest.raises(TypeError, match="g must be"):
        rule(q, q, v, g.bfloat16(), g)
    with pytest.raises(ValueError, match="beta must have shape"):
        rule(q, q, v, g, t(2, 3, 2))
    with pytest.raises(ValueError, match="multiple"):
        rule(t(2, 3, 3, 8), t(2, 3, 3, 8), v, g, g)
    with pytest.raises(ValueError, match="widths"):
        rule(t(2, 3, 2, 136), t(2, 3, 2, 136), v, g, g)
    with pytest.raises(ValueError, match="reset must have shape"):
        rule(q, q, v, g, g, t(2, 4, dtype=torch.uint8))
    with pytest.raises(TypeError, match="reset must be"):
        rule(q, q, v, g, g, t(2, 3))
    with pytest.raises(ValueError, match="initial_state must have shape"):
        rule(q, q, v, g, g, None, t(2, 4, 16, 8))
    with pytest.raises(ValueError, match="batch, tokens, heads"):
        rule(q[0], q[0], v[0], g[0], g[0])
    with pytest.raises(ValueError, match="on cpu"):
        rule(q, q.cpu(), v, g, g)
    step = zeno_b200.delta_rule_step
    one = (q[:, 0], q[:, 0], v[:, 0], g[:, 0], g[:, 0])
    with pytest.raises(ValueError, match="contiguous"):
        step(*one, t(2, 4, 16, 8).mT)
    with pytest.raises(TypeError, match="state must be"):
        step(*one, t(2, 4, 8, 16, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="no gradients"):
        step(*one, t(2, 4, 8, 16).requires_grad_(True))
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        zeno_b200.orthogonalize(t(3, 3, dtype=torch.float64))
    with pytest.raises(ValueError, match="steps"):
        zeno_b200.orthogonalize(t(3, 3), steps=-1)
