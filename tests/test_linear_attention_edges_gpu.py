"""Linear attention where its parts meet: chunks within a segment of a long rollout.

Tolerances and the plain implementation are those of test_linear_attention_gpu.py."""
import pytest
import torch

import zeno_b200
from test_linear_attention_gpu import NAMES, check, exact, gradients, inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bad", ["nan gate", "growing gates", "nan key", "inf value"])
@pytest.mark.parametrize("dtype,d,segment", [(torch.bfloat16, 64, 256), (torch.float32, 64, 224), (torch.bfloat16, 32, 224), (torch.bfloat16, 128, 512),
                                             (torch.bfloat16, 100, 512), (torch.float32, 128, 224)])
def test_a_reset_in_another_chunk_of_a_segment(dtype, d, segment, bad):
    """32 rollouts of 2000 tokens are cut into segments of several chunks.  In one of them an episode holds a gate that is not a number, gates whose
    product is past a float, or rows that are not finite, and a reset in a chunk in front of it and in one behind it ends that: every other
    episode, the state behind the rollout and the gradient of the one in front are what they are without it."""
    B, T, H = 16, 2000, 2
    begin, at, end = 2 * segment + 4, 2 * segment + 68, 2 * segment + 135  # three chunks of one segment, of 32 tokens or of 64
    assert end < 3 * segment
    x = inputs(B, T, H, H, d, d, dtype, reset=None)
    x[4] = torch.zeros(B, T, device=DEV, dtype=torch.uint8)
    x[4][:, begin] = x[4][:, end] = 1
    d_out, d_final = torch.randn(B, T, H, d, device=DEV).to(dtype), torch.randn(B, H, d, d, device=DEV)
    two = [t[:2] for t in x]
    want = exact(two, d_out[:2], d_final[:2])
    y = [t.clone() for t in x]
    if bad == "nan gate":
        y[3][0, at, 1] = float("nan")
    elif bad == "growing gates":
        y[3][0, at:at + 24, 1] = 4.0  # exp(96)
    elif bad == "nan key":
        y[1][0, at, 1, 5] = float("nan")
    else:
        y[2][0, at, 1, 5] = float("inf")
    got = [t[:2] for t in gradients(zeno_b200.linear_attention, y, d_out, d_final)]
    outside = [t for t in range(T) if not begin <= t < end]
    for name, a, b in zip(NAMES, got, want):
        if name in ("state", "d_initial"):
            check(a, b, name)
            continue
        check(a[1], b[1], name), check(a[0, :, 0], b[0, :, 0], name)
        check(a[0, outside, 1], b[0, outside, 1], name)
