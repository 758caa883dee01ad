"""GPU tests of gated_linear, residual_norm, keyed_dropout and sample_logits against their definitions in 64 bits.

Tolerances are bounds, worked out per element before the comparison: a result rounded to type t is off by at most half a
step (eps(t) / 2 of its value); a float32 sum of n terms by at most (n + 8) 2^-24 of the sum of their magnitudes; values
kept in t between forward and backward (f, p, y) and matrix operands (da, db) by half a step each, carried through the formulas."""
import numpy as np
import pytest
import torch

import marl_amd.ops  # noqa: F401  registers torch.ops.marl_amd

pytestmark = pytest.mark.gpu
ops = torch.ops.marl_amd
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps      # a step of the subnormal numbers


def gen(seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g)


def close(name, got, want, tol):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = int(torch.nonzero(bad.reshape(-1))[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off; first {i}: {got.reshape(-1)[i]} for {want.reshape(-1)[i]} "
                             f"+- {tol.expand_as(want).reshape(-1)[i]}")


# -- gated_linear ------------------------------------------------------------------------------------------------------
def act64(a, kind):
    """act(a), its derivative, bounds of the derivative's size and of the second derivative."""
    if kind == "relu":
        return a.clamp(min=0), (a > 0).double(), 1.0, 0.0
    if kind == "gelu":
        cdf = torch.special.ndtr(a)
        return a * cdf, cdf + a * torch.exp(-a * a / 2) / (2 * np.pi) ** 0.5, 1.13, 0.8
    s = torch.sigmoid(a)
    if kind == "sigmoid":
        return s, s * (1 - s), 0.25, 0.1
    return a * s, s * (1 + a * (1 - s)), 1.1, 0.5


def gated_oracle(x, wg, wu, gy, kind):
    dt, K = x.dtype, x.shape[1]
    x, wg, wu, gy = (t.double() for t in (x, wg, wu, gy))
    e = half_step(dt)
    a, b = x @ wg.t(), x @ wu.t()
    ea, eb = ((K + 8) * U * (x.abs() @ w.abs().t()) for w in (wg, wu))
    f, df, dmax, d2max = act64(a, kind)
    # act evaluated in float32: a few steps of its parts (2^-20 covers the hardware exponential over |a| < 16)
    ef = dmax * ea + 2.0 ** -20 * (1 + a.abs())
    y = f * b
    ty = e * y.abs() + (b.abs() * ef + f.abs() * eb + ef * eb) * 1.01 + 2 * U * y.abs() + tiny(dt)
    # backward works from f = act(a) and p = b act'(a), rounded to the type
    edf = d2max * ea + 2.0 ** -20 * (1 + a.abs())
    if kind == "relu":
        edf = edf + (a.abs() <= ea).double()                         # the step of the derivative at 0
    p = b * df
    ep = b.abs() * edf + df.abs() * eb + eb * edf + (e + 2 * U) * p.abs() + tiny(dt)
    ef = ef + e * f.abs() + tiny(dt)
    da, db = gy * b * df, gy * f
    eda, edb = gy.abs() * ep * 1.01, gy.abs() * ef * 1.01
    eda, edb = eda + (e + 4 * U) * (da.abs() + eda) + tiny(dt), edb + (e + 4 * U) * (db.abs() + edb) + tiny(dt)
    dx, dwg, dwu = da @ wg + db @ wu, da.t() @ x, db.t() @ x
    n, T = 2 * wg.shape[0], x.shape[0]
    mag = da.abs() @ wg.abs() + db.abs() @ wu.abs()
    tx = e * dx.abs() + 1.01 * (eda @ wg.abs() + edb @ wu.abs()) + (n + 72) * U * mag + tiny(dt)      # + up to 64 slices of the sum
    tg = e * dwg.abs() + 1.01 * (eda.t() @ x.abs()) + (T + 72) * U * (da.abs().t() @ x.abs()) + tiny(dt)
    tu = e * dwu.abs() + 1.01 * (edb.t() @ x.abs()) + (T + 72) * U * (db.abs().t() @ x.abs()) + tiny(dt)
    return (y, dx, dwg, dwu), (ty, tx, tg, tu)


def gated_check(T, d, h, dt, kind, seed=0, prepare=lambda t: t, name=""):
    rn = gen(seed)
    x, wg, wu, gy = rn(T, d).to(dt), (rn(h, d) / d ** 0.5).to(dt), (rn(h, d) / d ** 0.5).to(dt), rn(T, h).to(dt)
    want, tol = gated_oracle(x, wg, wu, gy, kind)
    xd, gd, ud = (prepare(t.cuda()).requires_grad_(True) for t in (x, wg, wu))
    y = ops.gated_linear(xd, gd, ud, kind)
    with torch.no_grad():
        assert torch.equal(y, ops.gated_linear(xd, gd, ud, kind))                    # with and without kept f, p
    grads = torch.autograd.grad(y, (xd, gd, ud), gy.cuda())
    for n_, g, w, t in zip(("y", "dx", "dw_gate", "dw_up"), (y,) + grads, want, tol):
        close(f"{name} {n_}", g, w, t)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("T,d,h", [
    (1, 1, 1), (1, 64, 32), (1, 200, 100), (3, 7, 5), (31, 33, 65), (32, 64, 64), (33, 128, 96), (64, 40, 48),       # few rows
    (65, 64, 64), (65, 1, 1), (100, 72, 136), (129, 65, 33), (200, 257, 131), (256, 128, 128), (300, 200, 520),       # tiles
    (1024, 96, 64), (2000, 24, 40),                                                                                # long sums over rows
])
def test_gated_linear_and_gradients(T, d, h, dt):
    gated_check(T, d, h, dt, "silu", seed=T + d + h)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("T,d,h", [(5, 48, 40), (130, 72, 50)])
def test_gated_linear_activations(T, d, h, dt, kind):
    gated_check(T, d, h, dt, kind, seed=11)


@pytest.mark.parametrize("dt,T,d,h", [(BF16, 3600, 520, 3592), (BF16, 3601, 517, 3591), (F32, 3600, 64, 3592), (F16, 1030, 8200, 40),
                                      (BF16, 4100, 3590, 64)])
def test_gated_linear_large_tiles(dt, T, d, h):
    """Sizes that fill the chip with the large tiles in at least one of the products, whole and ragged."""
    gated_check(T, d, h, dt, "silu", seed=5)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("T,d,h", [(1, 1024, 33), (5, 3337, 80), (40, 2050, 7), (64, 1536, 2016), (2, 4096, 1)])
def test_gated_linear_few_rows_over_narrow_weights(T, d, h, dt):
    """The slices of d over blocks, and both sides of where they begin."""
    gated_check(T, d, h, dt, "silu", seed=d)


def test_gated_linear_weights_of_different_strides():
    """Rows of w_gate and w_up spaced differently: the gradient of x moves through both."""
    rn = gen(12)
    x, wg, wu, gy = rn(150, 64), rn(72, 64) / 8, rn(72, 64) / 8, rn(150, 72)
    want, tol = gated_oracle(x, wg, wu, gy, "silu")
    wide = torch.full((72, 96), float("nan"), device="cuda")
    wide[:, :64] = wu
    leaves = [x.cuda().requires_grad_(True), wg.cuda().requires_grad_(True), wide[:, :64].detach().requires_grad_(True)]
    y = ops.gated_linear(*leaves)
    for g, w, t in zip((y,) + torch.autograd.grad(y, leaves, gy.cuda()), want, tol):
        close("strides", g, w, t)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("T", [7, 140])
def test_gated_linear_strided_and_shifted_operands(dt, T):
    def columns(t):                                  # every tensor a slice of columns of a wider one
        wide = torch.full((t.shape[0], t.shape[1] + 24), float("nan"), dtype=t.dtype, device="cuda")
        wide[:, 8:8 + t.shape[1]] = t
        return wide[:, 8:8 + t.shape[1]].detach()

    def shifted(t):                                  # rows that start one element behind a 16-byte border
        buf = torch.full((t.numel() + 17,), float("nan"), dtype=t.dtype, device="cuda")
        buf[1:1 + t.numel()] = t.reshape(-1)
        return buf[1:1 + t.numel()].view(t.shape).detach()

    def transposed(t):
        return t.t().contiguous().t().detach()

    for name, prep in (("columns", columns), ("shifted", shifted), ("transposed", transposed)):
        gated_check(T, 64, 72, dt, "silu", seed=2, prepare=prep, name=name)


def test_gated_linear_gradient_against_differences():
    rn = gen(3)
    x, wg, wu, gy = rn(70, 9), rn(5, 9) / 3, rn(5, 9) / 3, rn(70, 5)
    leaves = [t.cuda().requires_grad_(True) for t in (x, wg, wu)]
    grads = torch.autograd.grad(ops.gated_linear(*leaves, "gelu"), leaves, gy.cuda())
    f = lambda *t: float((act64(t[0] @ t[1].t(), "gelu")[0] * (t[0] @ t[2].t()) * gy.double()).sum())
    vals = [t.double() for t in (x, wg, wu)]
    for which, g in enumerate(grads):
        for at in ((0, 0), (2, 3), (4, 8)):
            step = 1e-4
            up, dn = [v.clone() for v in vals], [v.clone() for v in vals]
            up[which][at] += step
            dn[which][at] -= step
            # difference quotient: off by step^2 |f'''| / 6 (below 1e-5 here); the gradient by float32 steps of sums near 10
            assert abs((f(*up) - f(*dn)) / (2 * step) - float(g[at])) < 5e-5


def test_gated_linear_leading_dimensions_empty_rows_and_partial_gradients():
    rn = gen(4)
    x, wg, wu = rn(4, 5, 16).cuda(), rn(24, 16).cuda(), rn(24, 16).cuda()
    y = ops.gated_linear(x, wg, wu)
    assert y.shape == (4, 5, 24) and torch.equal(y.reshape(20, 24), ops.gated_linear(x.reshape(20, 16), wg, wu))
    assert torch.equal(ops.gated_linear(x[0, 0], wg, wu), y[0, 0])
    one = wg.clone().requires_grad_(True)
    e = ops.gated_linear(x[:0], one, wu)
    assert e.shape == (0, 5, 24)
    assert torch.equal(torch.autograd.grad(e.sum(), one)[0], torch.zeros_like(one))
    full = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
    want = torch.autograd.grad(ops.gated_linear(*full).sum(), full)               # gy: an expanded scalar
    for i in range(3):
        part = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, wg, wu))]
        assert torch.equal(torch.autograd.grad(ops.gated_linear(*part).sum(), part[i])[0], want[i])


@pytest.mark.parametrize("T", [3, 100])
def test_gated_linear_keeps_infinities_and_nan_in_their_rows(T):
    rn = gen(6)
    x, wg, wu = rn(T, 40).to(BF16).cuda(), rn(48, 40).to(BF16).cuda(), rn(48, 40).to(BF16).cuda()
    clean = ops.gated_linear(x, wg, wu)
    x[1, 3], x[2, 0] = float("nan"), float("inf")
    y = ops.gated_linear(x, wg, wu)
    rest = [i for i in range(T) if i not in (1, 2)]
    assert torch.equal(y[rest], clean[rest]) and bool(y[1].isnan().all()) and not bool(y[2].isfinite().all())


# -- residual_norm -----------------------------------------------------------------------------------------------------
def norm_oracle(x, b, wpost, wpre, gate, scale, eps, kind, gy, gn):
    dt, (T, d) = x.dtype, x.shape
    x, b, wpost, wpre, gy, gn = (t.double() for t in (x, b, wpost, wpre, gy, gn))
    g = torch.ones(1, dtype=torch.float64) if gate is None else gate.double()
    e, E = half_step(dt), (d + 16) * U
    layer = kind == "layer"
    mean = lambda t: t.mean(1, keepdim=True)

    def norm(v):
        m = mean(v) if layer else torch.zeros(T, 1, dtype=torch.float64)
        r = 1 / torch.sqrt(mean((v - m) ** 2) + eps)
        hat = (v - m) * r
        return m, r, hat, E * (2 * hat.abs() + 2 * v.abs().max(1, keepdim=True).values * r)      # value, bound of its float32 error

    mb, rb, bh, ebh = norm(b)
    o = bh * wpost
    y = scale * x + g * o
    ey = (g * wpost).abs() * ebh + 4 * U * ((scale * x).abs() + (g * o).abs())
    my, ry, yh, eyh = norm(y)
    worst = ey.max(1, keepdim=True).values
    eyh = eyh + ry * (ey + worst) + yh.abs() * ry * worst
    n = yh * wpre
    out, tol = [y, n], [e * y.abs() + ey + tiny(dt), e * n.abs() + wpre.abs() * eyh + 2 * U * n.abs() + tiny(dt)]
    # backward: y rounded to the type
    eyh = eyh + ry * e * y.abs() + tiny(dt)

    def back(q, eq, hat, ehat, r):
        p, s = mean(q * hat), mean(q) if layer else 0.0
        ep = mean(eq * hat.abs() + q.abs() * ehat) + E * mean((q * hat).abs())
        es = (mean(eq) + E * mean(q.abs())) if layer else 0.0
        t = r * (q - s - hat * p)
        return t, 1.01 * r * (eq + es + ehat * p.abs() + hat.abs() * ep) + E * r * (q.abs() + mean(q.abs()) + (hat * p).abs())

    t, et = back(gn * wpre, 2 * U * (gn * wpre).abs(), yh, eyh, ry)
    t = t + gy
    et = et + 2 * U * (t.abs() + gy.abs())
    q = t * g * wpost
    db, edb = back(q, (g * wpost).abs() * et + 4 * U * q.abs(), bh, ebh, rb)
    dx = scale * t
    S = (T + 16) * U
    dpost, dpre = (t * g * bh).sum(0), (gn * yh).sum(0)
    tpost = (g.abs() * (et * bh.abs() + t.abs() * ebh)).sum(0) * 1.01 + S * (t * g * bh).abs().sum(0)
    tpre = (gn.abs() * eyh).sum(0) * 1.01 + S * (gn * yh).abs().sum(0)
    out += [dx, db, dpost, dpre]
    tol += [e * dx.abs() + abs(scale) * et + 2 * U * dx.abs() + tiny(dt), e * db.abs() + edb + tiny(dt), e * dpost.abs() + tpost + tiny(dt),
            e * dpre.abs() + tpre + tiny(dt)]
    if gate is not None:
        gg = t * o
        eg = 1.01 * (o.abs() * et + (t * wpost).abs() * ebh) + 4 * U * gg.abs()
        if gate.dim() == 1:
            eg, gg = eg.sum(0) + S * gg.abs().sum(0), gg.sum(0)
        out.append(gg)
        tol.append(e * gg.abs() + eg + tiny(dt))
    return out, tol


def norm_check(T, d, dt, kind, gate, seed=0, prepare=lambda t: t, scale=0.75):
    rn = gen(seed)
    x, b = rn(T, d).to(dt), (0.7 * rn(T, d) + 0.2).to(dt)
    wpost, wpre = (1 + 0.2 * rn(d)).to(dt), (1 + 0.2 * rn(d)).to(dt)
    g = None if gate == "none" else (0.5 + 0.3 * (rn(d) if gate == "channel" else rn(T, d))).to(dt)
    gy, gn = rn(T, d).to(dt), rn(T, d).to(dt)
    want, tol = norm_oracle(x, b, wpost, wpre, g, scale, 1e-5, kind, gy, gn)
    on = [prepare(t.cuda()).requires_grad_(True) if t is not None else None for t in (x, b, wpost, wpre, g)]
    y, n = ops.residual_norm(*on, scale, 1e-5, kind)
    with torch.no_grad():
        y2, n2 = ops.residual_norm(*on, scale, 1e-5, kind)
    assert torch.equal(y, y2) and torch.equal(n, n2)
    leaves = [t for t in on if t is not None]
    grads = torch.autograd.grad((y, n), leaves, (prepare(gy.cuda()), prepare(gn.cuda())))
    names = ("y", "n", "dx", "dblock", "dw_post", "dw_pre", "dgate")
    for name, got, w, t in zip(names, (y, n) + grads, want, tol):
        close(name, got, w, t)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("kind,gate", [("rms", "none"), ("layer", "channel"), ("rms", "row"), ("layer", "row"), ("rms", "channel")])
@pytest.mark.parametrize("T,d", [(1, 2), (1, 128), (3, 63), (67, 128), (130, 100), (33, 1001), (5, 2050)])
def test_residual_norm_and_gradients(T, d, dt, kind, gate):
    norm_check(T, d, dt, kind, gate, seed=T + d)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("d", [64, 65, 256, 257, 512, 513, 1024, 1025, 2048, 4096, 4097, 8192, 8193, 16384])
def test_residual_norm_every_width(d, dt):
    """Both sides of every width at which the kernel changes its threads per row."""
    norm_check(9, d, dt, "layer", "channel", seed=d)


def test_residual_norm_many_rows():
    norm_check(3000, 96, F32, "layer", "channel", seed=1)
    norm_check(2501, 520, BF16, "rms", "row", seed=2)


@pytest.mark.parametrize("dt", [F32, F16])
def test_residual_norm_strided_operands(dt):
    def columns(t):
        if t.dim() == 1:
            buf = torch.full((2 * t.shape[0],), float("nan"), dtype=t.dtype, device="cuda")
            buf[::2] = t
            return buf[::2].detach()
        wide = torch.full((t.shape[0], t.shape[1] + 5), float("nan"), dtype=t.dtype, device="cuda")
        wide[:, 3:3 + t.shape[1]] = t
        return wide[:, 3:3 + t.shape[1]].detach()

    norm_check(21, 72, dt, "layer", "row", seed=3, prepare=columns)
    norm_check(21, 72, dt, "rms", "channel", seed=3, prepare=columns)


def test_residual_norm_constant_and_zero_rows():
    """A constant row has variance 0: eps alone; nothing may turn into NaN."""
    x, b, w = torch.zeros(4, 96).cuda(), torch.full((4, 96), 3.0).cuda(), torch.ones(96).cuda()
    leaves = [t.requires_grad_(True) for t in (x, b)]
    y, n = ops.residual_norm(x, b, w, w, None, 1.0, 1e-5, "layer")
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(n, torch.zeros_like(n))
    for g in torch.autograd.grad((y, n), leaves, (torch.ones_like(y), torch.ones_like(n))):
        assert bool(g.isfinite().all())


def test_residual_norm_one_gradient_at_a_time_and_leading_dimensions():
    rn = gen(8)
    x, b, w, v = rn(3, 4, 40).cuda(), rn(3, 4, 40).cuda(), rn(40).cuda(), rn(40).cuda()
    leaves = [t.requires_grad_(True) for t in (x, b, w, v)]
    y, n = ops.residual_norm(x, b, w, v)
    zero, one = torch.zeros_like(y), torch.ones_like(y)
    both = lambda gy, gn: torch.autograd.grad((y, n), leaves, (gy, gn), retain_graph=True)
    only_n = torch.autograd.grad(n, leaves, one, retain_graph=True)
    only_y = torch.autograd.grad(y, leaves[:3], one, retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(only_n, both(zero, one)))
    assert all(torch.equal(p, q) for p, q in zip(only_y, both(one, zero)))
    assert ops.residual_norm(x[:0], b[:0], w, v)[0].shape == (0, 4, 40)


def test_residual_norm_gradient_against_differences():
    rn = gen(9)
    vals = [rn(3, 10).double(), rn(3, 10).double(), 1 + 0.2 * rn(10).double(), 1 + 0.2 * rn(10).double(), rn(10).double()]
    gy, gn = rn(3, 10).double(), rn(3, 10).double()

    def f(x, b, wpost, wpre, g):
        def norm(v):
            v = v - v.mean(1, keepdim=True)
            return v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5)
        y = 0.5 * x + g * norm(b) * wpost
        return float((y * gy).sum() + (norm(y) * wpre * gn).sum())

    leaves = [v.float().cuda().requires_grad_(True) for v in vals]
    vals = [v.detach().double().cpu() for v in leaves]
    y, n = ops.residual_norm(*leaves, 0.5, 1e-5, "layer")
    grads = torch.autograd.grad((y, n), leaves, (gy.float().cuda(), gn.float().cuda()))
    gy, gn = gy.float().double(), gn.float().double()
    for which, g in enumerate(grads):
        for at in ((0, 1), (2, 7)) if g.dim() == 2 else ((0,), (9,)):
            up, dn = [v.clone() for v in vals], [v.clone() for v in vals]
            up[which][at] += 1e-5
            dn[which][at] -= 1e-5
            # quotient: off by 1e-10 |f'''| / 6 + rounding 1e-15 |f| / 1e-5; the gradient by float32 steps of sums of tens
            assert abs((f(*up) - f(*dn)) / 2e-5 - float(g[at])) < 1e-4 * (1 + abs(float(g[at])))


# -- keyed_dropout -----------------------------------------------------------------------------------------------------
def draws(keys, d, seed):
    """16-bit draws by Philox4x32-10 on Python integers' terms (numpy uint64 holds the 64-bit products)."""
    keys = np.asarray(keys, dtype=np.int64).astype(np.uint64)[:, None]
    nb = -(-d // 8)
    m = np.uint64(0xFFFFFFFF)
    c = [np.broadcast_to(np.arange(nb, dtype=np.uint64), (len(keys), nb)), np.full((len(keys), nb), 6, np.uint64),
         np.broadcast_to(keys & m, (len(keys), nb)), np.broadcast_to(keys >> np.uint64(32), (len(keys), nb))]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), q & m, (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return torch.from_numpy(np.stack(c, 2).astype("<u4").view("<u2").reshape(len(keys), nb * 8)[:, :d].astype(np.int64))


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("T,d", [(1, 1), (1, 8), (3, 7), (65, 9), (40, 512), (33, 1537), (2, 40000)])
def test_keyed_dropout_and_gradient(T, d, dt):
    rn = gen(T + d)
    x, gy = rn(T, d).to(dt), rn(T, d).to(dt)
    seed = -5 if d == 9 else (1 << 62) + 12345
    for keys in (None, torch.randperm(T, generator=torch.Generator().manual_seed(1)) + (5 << 33), torch.full((T,), -7)):
        for p in (0.0, 0.1, 0.5, 1.0):
            thr = int(p * 65536 + 0.5)
            keep = draws(np.arange(T) if keys is None else keys.numpy(), d, seed & 0xFFFFFFFFFFFFFFFF) >= thr
            s = 65536 / (65536 - thr) if thr < 65536 else 0.0
            xd = x.cuda().requires_grad_(True)
            y = ops.keyed_dropout(xd, p, seed, None if keys is None else keys.cuda())
            g, = torch.autograd.grad(y, xd, gy.cuda())
            for name, got, v in (("y", y, x), ("dx", g, gy)):
                want = torch.where(keep, v.double() * s, torch.zeros((), dtype=torch.float64))
                # scale and product round in float32, the result to the type
                close(name, got, want, (half_step(dt) + 3 * U) * want.abs() + tiny(dt))
                assert torch.equal(got.cpu()[~keep], torch.zeros(int((~keep).sum()), dtype=dt))


def test_keyed_dropout_rows_are_named_by_their_keys():
    rn = gen(1)
    x = rn(50, 70).cuda()
    keys = torch.arange(1000, 1050, device="cuda")
    y = ops.keyed_dropout(x, 0.3, 9, keys)
    perm = torch.randperm(50, device="cuda")
    assert torch.equal(ops.keyed_dropout(x[perm], 0.3, 9, keys[perm]), y[perm])       # a shuffled minibatch
    assert torch.equal(ops.keyed_dropout(x[7], 0.3, 9, keys[7]), y[7])                # one row alone
    assert torch.equal(ops.keyed_dropout(x.view(5, 10, 70), 0.3, 9, keys.view(5, 10)).view(50, 70), y)
    assert not torch.equal(ops.keyed_dropout(x, 0.3, 10, keys), y) and not torch.equal(ops.keyed_dropout(x, 0.3, 9, keys + 1), y)
    wide = torch.full((50, 90), float("nan"), device="cuda")
    wide[:, 11:81] = x
    assert torch.equal(ops.keyed_dropout(wide[:, 11:81], 0.3, 9, keys), y)
    bad = x.clone()
    bad[y == 0] = float("nan")                                                        # dropped whatever it held
    assert torch.equal(ops.keyed_dropout(bad, 0.3, 9, keys), y)
    assert ops.keyed_dropout(x[:0], 0.3, 9).shape == (0, 70) and ops.keyed_dropout(x[:, :0], 0.3, 9).shape == (50, 0)


def test_keyed_dropout_rate():
    y = ops.keyed_dropout(torch.ones(4096, 1024, device="cuda"), 0.25, 3)
    # 2^22 draws: the share kept has a standard deviation of sqrt(.25 .75 / 2^22) = 2.1e-4; five of them
    assert abs(float((y > 0).double().mean()) - 0.75) < 1.1e-3
    # columns and rows: 4096 and 1024 draws, standard deviations 6.8e-3 and 1.4e-2; six of them
    kept = (y > 0).double()
    assert float((kept.mean(0) - 0.75).abs().max()) < 0.041 and float((kept.mean(1) - 0.75).abs().max()) < 0.082


# -- sample_logits -----------------------------------------------------------------------------------------------------
def sample_oracle(logits, u, t, k, p, m):
    l = np.asarray(logits, dtype=np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    top = l.max()
    if top == -np.inf:
        return -1, -np.inf
    if t <= 0:
        return int(np.argmax(l)), 0.0
    with np.errstate(invalid="ignore"):
        z = np.where(l == top, 0.0, (l - top) / t)
    w = np.where(np.isneginf(l), 0.0, np.exp(z))
    order = np.argsort(-l, kind="stable")
    n = len(l) if k < 1 else min(k, len(l))
    ws = w[order[:n]]
    if p < 1:
        before = np.cumsum(ws) - ws
        inside = before < p * ws.sum()
        inside[0] = True
        n = int(inside.sum())
    w[order[n:]] = 0
    w[w < m] = 0
    cum = np.cumsum(w)
    i = int(np.searchsorted(cum, u * cum[-1], side="right"))
    i = min(i, int(np.nonzero(w)[0][-1]))
    return i, float(z[i] - np.log(cum[-1]))


def sample_check(logits, u, t=1.0, k=0, p=1.0, m=0.0, settings=None):
    V = logits.shape[-1]
    if settings is None:
        index, lp = ops.sample_logits(logits.cuda(), u.cuda(), t, k, p, m)
    else:
        index, lp = ops.sample_logits(logits.cuda(), u.cuda(), settings=settings.cuda())
    index, lp = index.cpu(), lp.cpu()
    f32 = lambda v: float(np.float32(v))
    for r in range(logits.shape[0]):
        s = (f32(t), k, f32(p), f32(m)) if settings is None else (float(settings[r, 0]), int(settings[r, 1]), float(settings[r, 2]), float(settings[r, 3]))
        i, want = sample_oracle(logits[r].double().numpy(), float(u[r]), *s)
        assert int(index[r]) == i, (r, int(index[r]), i, s)
        # weights are held in units of 2^-42 of the largest, each off by half of one; the result is rounded to float32
        assert lp[r] == want if np.isinf(want) else abs(float(lp[r]) - want) <= U * abs(want) + V * 2.0 ** -43 + 1e-12, (r, float(lp[r]), want)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 3, 1.0, 0.0), (1.3, 0, 0.8, 0.0), (1.0, 0, 1.0, 0.2), (0.9, 40, 0.9, 0.05),
            (2.0, 1, 1.0, 0.0), (1.0, 0, 1e-6, 0.0), (1.0, 10 ** 6, 0.999, 1.0), (5.0, 700, 0.97, 0.0)]


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 2, 3, 4, 5, 8, 16, 17, 33, 64, 65, 100, 255, 1000, 4096, 4097, 9000, 50001])
def test_sample_logits(V, dt):
    rn = gen(V)
    R = 40 if V < 3000 else 6
    logits = (3 * rn(R, V)).to(dt)
    u = torch.rand(R, generator=torch.Generator().manual_seed(V))
    for s in SETTINGS:
        sample_check(logits, u, *s)
    settings = torch.tensor([SETTINGS[r % len(SETTINGS)] for r in range(R)])
    sample_check(logits, u, settings=settings)


@pytest.mark.parametrize("V", [4, 50, 300, 6000])
def test_sample_logits_ties_masks_and_special_values(V):
    rn = gen(V)
    inf, low = float("inf"), torch.finfo(F32).min
    base = rn(V)
    rows = [torch.zeros(V), torch.full((V,), -inf), torch.full((V,), low), torch.full((V,), float("nan")), base.round(),
            torch.where(torch.arange(V) == V - 1, 1.0, -inf), torch.where(torch.arange(V) % 2 == 0, base, low), base.clone(), base.clone(),
            torch.where(torch.arange(V) % 3 == 0, -inf, base), torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0), base * 1e30]
    rows[7][V // 2], rows[7][1] = inf, inf
    rows[8][0], rows[8][V // 2] = float("nan"), -inf
    logits = torch.stack(rows)
    for u in (0.0, 0.3, 0.999999, 1.0):
        for s in SETTINGS:
            sample_check(logits, torch.full((len(rows),), u), *s)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_sample_logits_crowded_bins(dt):
    """More elements between two borders than are sorted at once: thousands of equal logits, thousands within 2^-17."""
    V, g = 20000, torch.Generator().manual_seed(7)
    near = 1 + 1e-4 * torch.rand(V, generator=g)
    rows = [torch.zeros(V), (torch.rand(V, generator=g) < 0.5).float(), near, torch.where(torch.rand(V, generator=g) < 0.3, near, torch.zeros(V)),
            torch.randint(0, 5, (V,), generator=g).float(), -3 + 0 * near]
    rows[5][123] = 2.0
    logits = torch.stack(rows).to(dt)
    for k, p in ((5000, 1.0), (0, 0.37), (9000, 0.61), (1, 0.5), (19999, 0.9999)):
        sample_check(logits, torch.rand(6, generator=g), 0.8, k, p, 0.0)


def test_sample_logits_largest_row_and_refused_settings_are_made_safe():
    V = 1 << 20
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(2, V, generator=g)
    u = torch.tensor([0.25, 0.875])
    sample_check(logits, u)
    sample_check(logits, u, 0.9, 100, 0.9, 0.0)
    nan = float("nan")
    odd = torch.tensor([[nan, nan, nan, nan], [-1.0, -3.0, -1.0, 7.0], [1.0, 1e9, 2.0, -1.0], [1.0, 0.5, 0.0, 2.0]])
    l4 = torch.randn(4, 300, generator=g)
    u4 = torch.tensor([0.1, 0.5, 0.7, 0.9])
    index, _ = ops.sample_logits(l4.cuda(), u4.cuda(), settings=odd.cuda())
    plain = ops.sample_logits(l4.cuda(), u4.cuda())[0].cpu()
    top = l4.argmax(1)
    assert index.cpu().tolist() == [int(plain[0]), int(top[1]), int(plain[2]), int(top[3])]


def test_sample_logits_frequencies_follow_the_weights():
    p = torch.tensor([0.1, 0.2, 0.3, 0.4])
    R = 200000
    index, lp = ops.sample_logits(p.log().expand(R, 4).contiguous().cuda(), torch.rand(R, generator=torch.Generator().manual_seed(0)).cuda())
    share = torch.bincount(index.cpu(), minlength=4).double() / R
    assert float((share - p).abs().max()) < 5 * (0.25 / R) ** 0.5                 # five standard deviations
    assert float((lp.cpu() - p.log()[index.cpu()]).abs().max()) < 1e-6            # float32 logs of the weights


def test_sample_logits_more_rows_than_one_launch_takes():
    R = (1 << 21) + 3
    u = torch.rand(R, device="cuda")
    logits = torch.zeros(R, 2, device="cuda")
    logits[:, 1] = torch.where(torch.arange(R, device="cuda") % 3 == 0, float("-inf"), 0.0)
    index, lp = ops.sample_logits(logits, u)
    open_ = logits[:, 1] == 0.0
    assert torch.equal(index, (open_ & (u >= 0.5)).long())          # u 2 is exact: 1 exceeds it below a half
    half = torch.tensor(0.5).log().item()
    assert float((lp - torch.where(open_, half, 0.0)).abs().max()) < 1e-7


def test_second_gradients():
    """keyed_dropout is linear and differentiable again; the others say that they are not."""
    x = torch.randn(5, 24, device="cuda", requires_grad=True)
    c = torch.randn(5, 24, device="cuda", requires_grad=True)
    g, = torch.autograd.grad((ops.keyed_dropout(x, 0.5, 3) * c).sum(), x, create_graph=True)
    gg, = torch.autograd.grad((g * 2.0).sum(), c)
    assert torch.equal(gg, ops.keyed_dropout(torch.full_like(x, 2.0), 0.5, 3))
    w = torch.randn(8, 24, device="cuda", requires_grad=True)
    for f in (lambda: ops.gated_linear(x, w, w), lambda: ops.residual_norm(x, x, c[0], c[1])[1]):
        g, = torch.autograd.grad(f().pow(2).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            g.sum().backward()


def test_sample_logits_strides_and_shapes():
    rn = gen(2)
    big = rn(6, 5, 700).cuda()
    u = torch.rand(6, 5, generator=torch.Generator().manual_seed(2)).cuda()
    i, lp = ops.sample_logits(big, u, 0.8, 20, 0.9)
    assert i.shape == lp.shape == (6, 5)
    view = big.reshape(30, 700)[::2]
    j, _ = ops.sample_logits(view, u.reshape(30)[::2], 0.8, 20, 0.9)
    assert torch.equal(j, i.reshape(30)[::2])
    cols = ops.sample_logits(big.reshape(30, 700)[:, 3:403], u.reshape(30), 0.8, 20, 0.9)[0]
    assert torch.equal(cols, ops.sample_logits(big.reshape(30, 700)[:, 3:403].contiguous(), u.reshape(30), 0.8, 20, 0.9)[0])
    assert ops.sample_logits(big[:0], u[:0])[0].shape == (0, 5)


# -- all of them: streams, graphs, a run as they are used -----------------------------------------------------------------
def trunk_step(x, block_w, norm_w, keys, u, out_w):
    """One residual block as a policy trunk uses it, down to the draw."""
    wg, wu, wd = block_w
    y0, n0 = ops.residual_norm(x, x, norm_w, norm_w, None, 0.5, 1e-5, "layer")
    h = ops.keyed_dropout(ops.gated_linear(n0, wg, wu), 0.2, 77, keys)
    y1, n1 = ops.residual_norm(y0, h @ wd.t(), norm_w, norm_w, None, 1.0, 1e-5, "layer")
    logits = n1 @ out_w.t()
    return y1, logits, ops.sample_logits(logits.detach(), u, 0.9, 3, 0.95)


def trunk_inputs(T, d, h, seed):
    rn = gen(seed)
    x = rn(T, d).cuda().requires_grad_(True)
    w = [(rn(h, d) / d ** 0.5).cuda().requires_grad_(True), (rn(h, d) / d ** 0.5).cuda().requires_grad_(True),
         (rn(d, h) / h ** 0.5).cuda().requires_grad_(True)]
    nw = (1 + 0.1 * rn(d)).cuda().requires_grad_(True)
    return x, w, nw, torch.arange(T, device="cuda") + 99, torch.rand(T, generator=torch.Generator().manual_seed(seed)).cuda(), \
        (rn(6, d) / d ** 0.5).cuda().requires_grad_(True)


def test_a_block_as_it_is_used_against_float64():
    T, d, h = 150, 48, 120
    x, w, nw, keys, u, ow = trunk_inputs(T, d, h, 1)
    y, logits, (index, lp) = trunk_step(x, w, nw, keys, u, ow)
    gl = torch.randn(T, 6, generator=torch.Generator().manual_seed(5)).cuda()
    leaves = [x, *w, nw, ow]
    grads = torch.autograd.grad(logits, leaves, gl)
    # the same in float64 on the CPU, by autograd
    c = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    cx, cg, cu, cd, cn, co = c

    def norm(v):
        v = v - v.mean(1, keepdim=True)
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5) * cn

    y0 = 0.5 * cx + norm(cx)
    n0 = norm(y0)
    a = n0 @ cg.t()
    hid = a * torch.sigmoid(a) * (n0 @ cu.t())
    keep = draws(keys.cpu().numpy(), h, 77) >= int(0.2 * 65536 + 0.5)
    hid = hid * keep * (65536 / (65536 - int(0.2 * 65536 + 0.5)))
    y1 = y0 + norm(hid @ cd.t())
    want = norm(y1) @ co.t()
    want_grads = torch.autograd.grad(want, c, gl.double().cpu())
    # float32 throughout: a chain of eight stages of sums of at most 150 terms, each off by at most 158 2^-24 = 1e-5 of its
    # magnitudes; 8 x 1e-5 of the largest value
    for got, ref in zip((logits,) + grads, (want.detach(),) + want_grads):
        assert float((got.detach().cpu().double() - ref).abs().max()) <= 8e-5 * float(ref.abs().max())
    for r in range(T):
        i, l = sample_oracle(logits[r].detach().cpu().double().numpy(), float(u[r]), float(np.float32(0.9)), 3, float(np.float32(0.95)), 0.0)
        assert int(index[r]) == i and abs(float(lp[r]) - l) < 1e-6


def test_side_stream_equals_the_default_stream():
    args = trunk_inputs(200, 64, 160, 2)
    want = trunk_step(*args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = trunk_step(*args)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2][0], want[2][0])


def test_captured_forward_and_backward_replay_with_new_inputs():
    """Two graphs of different sizes, captured with their backward passes (torch.autograd.grad: no accumulation into leaves),
    replayed in turn with eager work in between; every replay against the eager result on the same values."""
    made = []
    for T, h, seed in ((96, 160, 3), (40, 72, 4)):
        x, w, nw, keys, u, ow = trunk_inputs(T, 64, h, seed)
        gl = torch.randn(T, 6, generator=torch.Generator().manual_seed(seed)).cuda()
        leaves = [x, *w, nw]

        def step(x=x, w=w, nw=nw, keys=keys, u=u, ow=ow, gl=gl, leaves=leaves):
            y, logits, (i, lp) = trunk_step(x, w, nw, keys, u, ow)
            return [logits.detach(), i, lp] + list(torch.autograd.grad(logits, leaves, gl))

        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            step()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        made.append((g, out, step, x, keys, u))
    for turn in range(4):
        for g, out, step, x, keys, u in made:
            with torch.no_grad():
                x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(turn)))
                keys.add_(1000)
                u.copy_(torch.rand(u.shape, generator=torch.Generator().manual_seed(turn)))
        for g, *_ in made:
            g.replay()
        torch.cuda.synchronize()
        for g, out, step, *_ in made:
            kept = [t.clone() for t in out]
            want = step()
            # library products (h @ wd, the head) may differ from eager ones in their order of adding; the rest is ours
            for p, q in zip(kept, want):
                if p.dtype == torch.int64:
                    assert float((p != q).float().mean()) < 0.02
                else:
                    assert torch.allclose(p, q, rtol=1e-4, atol=1e-4)


def test_results_do_not_vary_from_run_to_run():
    args = trunk_inputs(700, 96, 200, 6)
    x, w, nw = args[0], args[1], args[2]

    def once():
        n = ops.residual_norm(x, x, nw, nw)[1]
        hdn = ops.gated_linear(n, w[0], w[1])
        return [hdn] + list(torch.autograd.grad(hdn.sum(), [x, w[0], w[1], nw])) + list(ops.sample_logits(hdn.detach(), torch.rand(700, generator=torch.Generator().manual_seed(1)).cuda(), 1.0, 20, 0.9))

    first = once()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, once()))


@pytest.mark.parametrize("dt", [torch.float32, torch.float16], ids=str)
def test_sample_logits_many_long_rows(dt):
    # many rows above 8192 logits take smaller workgroups than a few: the draws are those of the definition, and a row drawn
    # among many is the row drawn among few, bit for bit (integer weights), on both sides of the limits of top-k
    R, V = 516, 8203
    g = torch.Generator().manual_seed(11)
    logits = (3 * torch.randn(R, V, generator=g)).to(dt)
    logits[torch.rand(R, V, generator=g) < 0.1] = float("-inf")
    logits[5] = 1.0                                    # one value
    logits[6] = float("-inf")                          # nothing
    logits[7, 2:] = float("-inf")                      # fewer than k
    logits[8, 4000:4300] = 20.0                        # ties across every limit below
    logits[9, 77] = float("inf")
    u = torch.rand(R, generator=g)
    ks = torch.tensor([0, 1, 64, 255, 256, 257, 511, 512, 513, 1025])
    settings = torch.stack([0.5 + torch.rand(R, generator=g), ks[torch.arange(R) % len(ks)].float(), torch.where(torch.rand(R, generator=g) < 0.5, 0.9, 1.0),
                            torch.where(torch.rand(R, generator=g) < 0.3, 0.01, 0.0)], 1).contiguous()
    dev = [t.cuda() for t in (logits, u, settings)]
    many = ops.sample_logits(dev[0], dev[1], settings=dev[2])
    for first in range(0, R, 129):
        s = slice(first, first + 129)
        few = ops.sample_logits(dev[0][s], dev[1][s], settings=dev[2][s])
        assert torch.equal(many[0][s], few[0]) and torch.equal(many[1][s], few[1])
    pick = torch.cat([torch.arange(0, 40), torch.arange(40, R, 7)])
    index, lp = many[0].cpu(), many[1].cpu()
    for r in pick.tolist():
        i, want = sample_oracle(logits[r].double().numpy(), float(u[r]), float(settings[r, 0]), int(settings[r, 1]), float(settings[r, 2]), float(settings[r, 3]))
        assert int(index[r]) == i, (r, int(index[r]), i, settings[r])
        assert float(lp[r]) == want if np.isinf(want) else abs(float(lp[r]) - want) <= U * abs(want) + V * 2.0 ** -43 + 1e-12, (r, float(lp[r]), want)
