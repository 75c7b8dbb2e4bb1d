"""The C entries of the policy operators refuse a workspace that is not there, whatever its stated size (no GPU is
touched before the checks)."""
from zeno_b200._ffi import _lib, ffi
from test_operators_refusals import INVALID, arguments, message


def test_delta_rule_refuses_a_missing_workspace():
    p = arguments(tokens=4096, value_heads=2)
    for pass_ in (0, 1):
        need = _lib.zeno_delta_rule_workspace_bytes(p, pass_)
        assert need > 0
        if pass_ == 0:
            assert _lib.zeno_delta_rule_forward(p, ffi.NULL, need, ffi.NULL) == INVALID
        else:
            d = ffi.new("ZenoDeltaRuleGrads*")
            for name in ("d_out", "d_q", "d_k", "d_v", "d_g", "d_beta"):
                getattr(d, name).data = ffi.cast("void*", 4096)
            p.saved = ffi.cast("float*", 4096)
            assert _lib.zeno_delta_rule_backward(p, d, ffi.NULL, need, ffi.NULL) == INVALID
        assert "workspace is NULL" in message()
