"""GPU tests of the trunk operators' place in autograd beside their gradients."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import marl_amd.ops  # noqa: F401  registers torch.ops.marl_amd

pytestmark = pytest.mark.gpu
ops = torch.ops.marl_amd


@pytest.mark.parametrize("name,call", [
    ("x", lambda x, w, v: ops.gated_linear(x, w, w)),
    ("x", lambda x, w, v: ops.residual_norm(x, x, v, v)[1]),
    ("x", lambda x, w, v: ops.keyed_dropout(x, 0.5, 1)),
    ("v", lambda x, w, v: ops.residual_norm(x, x, v, v)[0]),
    ("v", lambda x, w, v: ops.residual_norm(x, x, v.detach(), v.detach(), v)[0]),
])
def test_forward_mode_derivatives_are_refused(name, call):
    """Tangents would be lost without a word: the operators have gradients only."""
    t = dict(x=torch.randn(4, 24, device="cuda"), w=torch.randn(8, 24, device="cuda"), v=torch.randn(24, device="cuda"))
    with fwd.dual_level():
        t[name] = fwd.make_dual(t[name], torch.ones_like(t[name]))
        with pytest.raises(RuntimeError, match="jvp|forward"):
            call(t["x"], t["w"], t["v"])
