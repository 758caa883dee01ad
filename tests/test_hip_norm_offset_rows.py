"""Gradients of residual_norm on rows whose mean is large against their spread: the normalised row of the backward pass is
that of the forward pass, computed from y before it is rounded.

Tolerances as in test_hip_trunk_ops.py, without any term for a rounded y: a result rounded to type t is off by half a step, a
float32 sum of n terms by at most (n + 16) 2^-24 of the sum of their magnitudes, carried through the formulas."""
import pytest
import torch

import marl_amd.ops  # noqa: F401  registers torch.ops.marl_amd
from test_hip_trunk_ops import BF16, F16, F32, U, close, gen, half_step, tiny

pytestmark = pytest.mark.gpu
ops = torch.ops.marl_amd


def oracle(x, b, wpost, wpre, gate, scale, kind, gy, gn):
    dt, (T, d) = x.dtype, x.shape
    x, b, wpost, wpre, gy, gn = (t.double() for t in (x, b, wpost, wpre, gy, gn))
    g = torch.ones(1, dtype=torch.float64) if gate is None else gate.double()
    e, E, layer = half_step(dt), (d + 16) * U, kind == "layer"
    mean = lambda t: t.mean(1, keepdim=True)

    def norm(v):
        m = mean(v) if layer else torch.zeros(T, 1, dtype=torch.float64)
        r = 1 / torch.sqrt(mean((v - m) ** 2) + 1e-5)
        hat = (v - m) * r
        return r, hat, E * (2 * hat.abs() + 2 * v.abs().max(1, keepdim=True).values * r)

    rb, bh, ebh = norm(b)
    o = bh * wpost
    y = scale * x + g * o
    ey = (g * wpost).abs() * ebh + 4 * U * ((scale * x).abs() + (g * o).abs())
    ry, yh, eyh = norm(y)
    worst = ey.max(1, keepdim=True).values
    eyh = eyh + ry * (ey + worst) + yh.abs() * ry * worst

    def back(q, eq, hat, ehat, r):
        p, s = mean(q * hat), mean(q) if layer else 0.0
        ep = mean(eq * hat.abs() + q.abs() * ehat) + E * mean((q * hat).abs())
        es = (mean(eq) + E * mean(q.abs())) if layer else 0.0
        t = r * (q - s - hat * p)
        return t, 1.01 * r * (eq + es + ehat * p.abs() + hat.abs() * ep) + E * r * (q.abs() + mean(q.abs()) + (hat * p).abs())

    t, et = back(gn * wpre, 2 * U * (gn * wpre).abs(), yh, eyh, ry)
    t, et = t + gy, et + 2 * U * (t.abs() + 2 * gy.abs())
    q = t * g * wpost
    db, edb = back(q, (g * wpost).abs() * et + 4 * U * q.abs(), bh, ebh, rb)
    S = (T + 16) * U
    out = {"dx": (scale * t, abs(scale) * et), "dblock": (db, edb),
           "dw_post": ((t * g * bh).sum(0), (g.abs() * (et * bh.abs() + t.abs() * ebh)).sum(0) * 1.01 + S * (t * g * bh).abs().sum(0)),
           "dw_pre": ((gn * yh).sum(0), (gn.abs() * eyh).sum(0) * 1.01 + S * (gn * yh).abs().sum(0))}
    if gate is not None:
        gg, eg = t * o, 1.01 * (o.abs() * et + (t * wpost).abs() * ebh) + 4 * U * (t * o).abs()
        if gate.dim() == 1:
            gg, eg = gg.sum(0), eg.sum(0) + S * gg.abs().sum(0)
        out["dgate"] = (gg, eg)
    return {k: (v, (e + 2 * U) * v.abs() + tol + tiny(dt)) for k, (v, tol) in out.items()}


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate", ["none", "channel", "row"])
@pytest.mark.parametrize("T,d,offset", [(1, 128, 64.0), (3, 256, 16.0), (2, 1001, 64.0), (5, 33, -40.0), (2, 2050, 30.0)])
def test_gradients_of_rows_with_a_large_mean(T, d, offset, gate, kind, dt):
    rn = gen(T + d)
    x, b = (rn(T, d) + offset).to(dt), (0.7 * rn(T, d) + 0.2).to(dt)
    wpost, wpre = (1 + 0.2 * rn(d)).to(dt), (1 + 0.2 * rn(d)).to(dt)
    g = None if gate == "none" else (0.5 + 0.3 * (rn(d) if gate == "channel" else rn(T, d))).to(dt)
    gy, gn = rn(T, d).to(dt), rn(T, d).to(dt)
    want = oracle(x, b, wpost, wpre, g, 0.75, kind, gy, gn)
    on = [t.cuda().requires_grad_(True) if t is not None else None for t in (x, b, wpost, wpre, g)]
    y, n = ops.residual_norm(*on, 0.75, 1e-5, kind)
    grads = torch.autograd.grad((y, n), [t for t in on if t is not None], (gy.cuda(), gn.cuda()))
    for (name, (w, tol)), got in zip(want.items(), grads):
        close(name, got, w, tol)


def test_gradients_of_a_strided_stream():
    """x as a slice of columns (its rows are taken as they are) and as a transposed view (copied)."""
    rn = gen(4)
    x, b, w, v, gy, gn = (rn(6, 72) + 50).to(BF16), rn(6, 72).to(BF16), (1 + 0.1 * rn(72)).to(BF16), (1 + 0.1 * rn(72)).to(BF16), rn(6, 72).to(BF16), rn(6, 72).to(BF16)
    want = oracle(x, b, w, v, None, 0.5, "layer", gy, gn)
    wide = torch.full((6, 90), float("nan"), dtype=BF16, device="cuda")
    wide[:, 5:77] = x
    for view in (wide[:, 5:77], x.cuda().t().contiguous().t()):
        on = [t.detach().cuda().requires_grad_(True) for t in (view, b, w, v)]
        y, n = ops.residual_norm(*on, None, 0.5, 1e-5, "layer")
        for (name, (wt, tol)), got in zip(want.items(), torch.autograd.grad((y, n), on, (gy.cuda(), gn.cuda()))):
            close(name, got, wt, tol)
