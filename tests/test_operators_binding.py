"""The operators on libzeno.so alone do not need the compiled PyTorch functions."""
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("how,message", [("raise ImportError('undefined symbol: x')", "does not load with PyTorch"), ("missing", "is missing")])
def test_without_the_binding(how, message):
    program = textwrap.dedent("""
        import importlib.machinery, pathlib
        import torch, zeno_b200
        if HOW == "missing":
            exists = pathlib.Path.exists
            pathlib.Path.exists = lambda self, **kw: self.name != "zeno_torch.so" and exists(self, **kw)
        else:
            load = importlib.machinery.ExtensionFileLoader.create_module
            def create_module(self, spec):
                if "zeno_torch" in spec.name:
                    exec(HOW)
                return load(self, spec)
            importlib.machinery.ExtensionFileLoader.create_module = create_module
        import zeno_b200.policy
        x = torch.zeros(1, 2, 1, 8)
        for f in (lambda: zeno_b200.delta_rule(x, x, x, x[..., 0], x[..., 0]), lambda: zeno_b200.orthogonalize(x)):
            try:
                f()
            except ValueError as e:
                assert "CUDA" in str(e)
            else:
                raise AssertionError
        for f in (lambda: zeno_b200.layer_norm(x), lambda: zeno_b200.linear_attention(x, x, x, torch.zeros(1)),
                  lambda: zeno_b200.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], torch.zeros(1), torch.zeros(1, 1, 8, 8))):
            try:
                f()
            except ImportError as e:
                assert MESSAGE in str(e) and "zeno_b200.build" in str(e), e
            else:
                raise AssertionError
    """)
    r = subprocess.run([sys.executable, "-c", f"HOW, MESSAGE = {how!r}, {message!r}\n{program}"], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
