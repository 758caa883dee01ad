"""marl_amd.ops without the libraries: the module imports, what needs no library works, what needs one says which."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import os, torch
from marl_amd import _lib
exists = os.path.exists
os.path.exists = lambda p: False if str(p).endswith({missing!r}) else exists(p)
import marl_amd.ops
ops = torch.ops.marl_amd
m = lambda *s, dtype=torch.float64: torch.empty(*s, dtype=dtype, device="meta")
assert ops.adjacency_bits(m(2, 40), m(2, 40), m(2, dtype=torch.int32)).shape == (2, 40, 2)
x = torch.zeros(2, 3)
for call in (lambda: ops.gated_linear(x, x, x), lambda: ops.residual_norm(x, x, x[0], x[0]), lambda: ops.keyed_dropout(x, 0.5, 1),
             lambda: ops.sample_logits(x, x[:, 0]), lambda: _lib.load_torch()):
    try:
        call()
    except _lib.MarlError as e:
        assert {missing!r} in str(e) and "build" in str(e), e
    else:
        raise SystemExit("not refused")
print("fine")
"""


@pytest.mark.parametrize("missing", ["libmarl_torch.so", "libmarl_env.so"])
def test_ops_import_without_a_library(missing):
    out = subprocess.run([sys.executable, "-c", SCRIPT.format(missing=missing)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "fine" in out.stdout, out.stderr[-2000:]
