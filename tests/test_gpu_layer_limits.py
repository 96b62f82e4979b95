"""GPU: the operators round the recurrence where their numbers get hard."""
import pytest
import torch

import flashkda_b200 as F
import layer_ref as R
from test_gpu_conv_norm import norm_bound, randn

pytestmark = pytest.mark.gpu
bf16, fp32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("gate_first", [False, True])
@pytest.mark.parametrize("D", [64, 128, 1032])
def test_gated_norm_where_x_times_gate_overflows(act, gate_first, D):
    """|x gate| beyond the largest fp32 while the activation is 0, or in rows that are large throughout."""
    x, g, w = randn(1, 6, 3, D, seed=1), randn(1, 6, 3, D, seed=2, std=2.0), randn(D, dtype=fp32, seed=3)
    x[0, 0, :, 5], g[0, 0, :, 5] = 1e25, -1e25                      # (alone in its row, which has the rest to show that it counts as 0 with the gate first)
    x[0, 1] *= 1e8
    g[0, 1, :, ::3] = -3e38
    x[0, 2, :, ::2], g[0, 2, :, ::2] = -2e15, -2e30
    g[0, 3] = -3e38
    out = torch.full_like(x, float("nan"))
    want = R.gated(x, g, w, 1e-5, act, gate_first)
    F.gated_norm(x, g, w, out, eps=1e-5, act=act, gate_first=gate_first)
    if not gate_first:                                              # the square of 1e25 is beyond fp32 itself, whatever the gate
        out, want = out[:, 1:], want[:, 1:]
    assert R.off(out, want, norm_bound(want)) <= 1
