"""The trunk operators in a process that has loaded libmarl_torch.so and not bound it: an error, not a call of nothing."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import torch
torch.ops.load_library("marl_amd/libmarl_torch.so")
ops = torch.ops.marl_amd
x = torch.ones(4, 8, device="cuda")
calls = [lambda: ops.gated_linear(x, x, x), lambda: ops.residual_norm(x, x, x[0], x[0]), lambda: ops.keyed_dropout(x, 0.5, 1),
         lambda: ops.sample_logits(x, x[:, 0].contiguous())]
calls += [lambda: ops.gated_linear_backward(x[:, :4], x, x, x, x[:, :4].contiguous(), x[:, :4].contiguous(), True, True),
          lambda: ops.residual_norm_backward(x, x, x, x, x[0], x[0], None, x[:, :4].contiguous(), 1.0, "rms")]
for call in calls:
    try:
        call()
    except RuntimeError as e:
        assert "bound" in str(e), e
    else:
        raise SystemExit("not refused")
print("fine")
"""


def test_operators_that_are_not_bound_are_refused():
    out = subprocess.run([sys.executable, "-c", SCRIPT], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and "fine" in out.stdout, out.stderr[-2000:]
