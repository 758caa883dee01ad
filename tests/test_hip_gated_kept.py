"""What gated_linear keeps between forward and backward: f = act(a) and p = b act'(a) are not rounded to the element type.

Tolerances: a gradient with a single term, dW[j][k] = da[j] x[k], has two roundings to the type (da, which is a matrix operand,
and the result), half a step each, besides float32 errors: a and b are sums of d terms, off by (d + 8) 2^-24 of their
magnitudes; act and act' are off by 2^-20 of 1 + |a|."""
import pytest
import torch

import marl_amd.ops  # noqa: F401  registers torch.ops.marl_amd
from test_hip_trunk_ops import BF16, F16, U, act64, close, gen, half_step, tiny

pytestmark = pytest.mark.gpu
ops = torch.ops.marl_amd


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("kind", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("T,d,h", [(1, 64, 1024), (100, 72, 1000)])
def test_gradients_are_rounded_once_as_operands_and_once_as_results(T, d, h, kind, dt):
    rn = gen(d + h)
    x, wg, wu, gy = rn(T, d).to(dt), (rn(h, d) / d ** 0.5).to(dt), (rn(h, d) / d ** 0.5).to(dt), rn(T, h).to(dt)
    row = T // 2
    gy[torch.arange(T) != row] = 0.0                   # one term in every sum over rows
    leaves = [t.cuda().requires_grad_(True) for t in (x, wg, wu)]
    _, dwg, dwu = torch.autograd.grad(ops.gated_linear(*leaves, kind), leaves, gy.cuda())
    x1, wg, wu, g = x[row].double(), wg.double(), wu.double(), gy[row].double()
    a, b = wg @ x1, wu @ x1
    ea, eb = ((d + 8) * U * (w.abs() @ x1.abs()) for w in (wg, wu))
    f, df, dmax, d2max = act64(a, kind)
    ef, edf = dmax * ea + 2.0 ** -20 * (1 + a.abs()), d2max * ea + 2.0 ** -20 * (1 + a.abs())
    ep = b.abs() * edf + df.abs() * eb + eb * edf
    e = half_step(dt)
    for name, got, v, ev in (("dw_gate", dwg, g * b * df, g.abs() * ep), ("dw_up", dwu, g * f, g.abs() * ef)):
        want = v[:, None] * x1[None, :]
        ev = ev + e * (v.abs() + ev) + 4 * U * v.abs() + tiny(dt)
        close(name, got, want, (e + 2 * U) * want.abs() + 1.01 * ev[:, None] * x1.abs()[None, :] + tiny(dt))


@pytest.mark.parametrize("T", [3, 90])
def test_what_is_kept_may_exceed_the_range_of_float16(T):
    """b = 2 10^5 fits no float16, y = act(a) b and the gradients do."""
    d, h = 64, 40
    x = torch.full((T, d), 50.0, dtype=F16)
    wg, wu = torch.full((h, d), 0.01 / (50 * d), dtype=F16), torch.full((h, d), 64.0, dtype=F16)
    gy = torch.zeros(T, h, dtype=F16)
    gy[0] = 2.0 ** -10                                 # rows without a gradient: 0, not 0 times infinity
    leaves = [t.cuda().requires_grad_(True) for t in (x, wg, wu)]
    y = ops.gated_linear(*leaves, "silu")
    assert bool(y.isfinite().all())
    dx, dwg, dwu = torch.autograd.grad(y, leaves, gy.cuda())
    a, b = x[0].double() @ wg.double().t(), x[0].double() @ wu.double().t()
    f, df, *_ = act64(a, "silu")
    da, db = gy[0].double() * b * df, gy[0].double() * f
    e = half_step(F16)
    # a and b are sums of 64 equal signs, off by 72 2^-24 of themselves, act and act' by a few 2^-22: together below 2^-16.
    # da ~ 100 and db ~ 5 10^-6 are rounded to float16 (db to its subnormal step), then the result
    eda, edb = (e + 2.0 ** -16) * da.abs(), (e + 2.0 ** -16) * db.abs() + tiny(F16)
    for name, got, want, tol in (("dx", dx[0], da @ wg.double() + db @ wu.double(), eda @ wg.double().abs() + edb @ wu.double().abs()),
                                 ("dw_gate", dwg, da[:, None] * x[:1].double(), eda[:, None] * 50.0),
                                 ("dw_up", dwu, db[:, None] * x[:1].double(), edb[:, None] * 50.0)):
        close(name, got, want, e * want.abs() + 1.01 * tol + tiny(F16))
    assert bool((dx[1:] == 0).all())
