"""Refusals of the trunk operators (gated_linear, residual_norm, keyed_dropout, sample_logits), their shapes on the meta
device and the argument checks of their C entry points.  No kernel is launched here."""
import pytest
import torch

import marl_amd.ops  # noqa: F401  registers torch.ops.marl_amd
from marl_amd import _lib

ops = torch.ops.marl_amd
Z = torch.zeros


@pytest.mark.parametrize("call", [
    lambda: ops.gated_linear(Z(2, 3), Z(4, 3), Z(4, 3)),                                  # not on the device
    lambda: ops.gated_linear(Z(2, 3), Z(4, 3), Z(4, 3), "tanh"),
    lambda: ops.gated_linear(Z(2, 3), Z(4, 5), Z(4, 5)),
    lambda: ops.gated_linear(Z(2, 3), Z(4, 3), Z(5, 3)),
    lambda: ops.gated_linear(Z(2, 3), Z(4, 3).half(), Z(4, 3)),
    lambda: ops.gated_linear(Z(2, 3).double(), Z(4, 3).double(), Z(4, 3).double()),
    lambda: ops.gated_linear(Z(2, 0), Z(4, 0), Z(4, 0)),
    lambda: ops.residual_norm(Z(2, 3), Z(2, 3), Z(3), Z(3)),
    lambda: ops.residual_norm(Z(2, 3), Z(2, 4), Z(3), Z(3)),
    lambda: ops.residual_norm(Z(2, 3), Z(2, 3), Z(4), Z(3)),
    lambda: ops.residual_norm(Z(2, 3), Z(2, 3), Z(3), Z(3), Z(2, 1)),
    lambda: ops.residual_norm(Z(2, 3), Z(2, 3), Z(3), Z(3), None, 1.0, -1.0),
    lambda: ops.residual_norm(Z(2, 3), Z(2, 3), Z(3), Z(3), None, 1.0, 1e-5, "batch"),
    lambda: ops.residual_norm(Z(1, 16385), Z(1, 16385), Z(16385), Z(16385)),
    lambda: ops.residual_norm(Z(2, 3), Z(2, 3).half(), Z(3), Z(3)),
    lambda: ops.keyed_dropout(Z(2, 3), 0.5, 1),
    lambda: ops.keyed_dropout(Z(2, 3), 1.5, 1),
    lambda: ops.keyed_dropout(Z(2, 3), -0.1, 1),
    lambda: ops.keyed_dropout(Z(2, 3), float("nan"), 1),
    lambda: ops.keyed_dropout(Z(2, 3), 0.5, 1, Z(2)),
    lambda: ops.keyed_dropout(Z(2, 3), 0.5, 1, Z(3, dtype=torch.int64)),
    lambda: ops.keyed_dropout(Z(2, 3, dtype=torch.int32), 0.5, 1),
    lambda: ops.sample_logits(Z(2, 3), Z(2)),
    lambda: ops.sample_logits(Z(2, 3), Z(3)),
    lambda: ops.sample_logits(Z(2, 3), Z(2).double()),
    lambda: ops.sample_logits(Z(2, 0), Z(2)),
    lambda: ops.sample_logits(Z(1, (1 << 20) + 1), Z(1)),
    lambda: ops.sample_logits(Z(2, 3), Z(2), -1.0),
    lambda: ops.sample_logits(Z(2, 3), Z(2), float("nan")),
    lambda: ops.sample_logits(Z(2, 3), Z(2), 1.0, -1),
    lambda: ops.sample_logits(Z(2, 3), Z(2), 1.0, 0, 0.0),
    lambda: ops.sample_logits(Z(2, 3), Z(2), 1.0, 0, 1.0, 1.5),
    lambda: ops.sample_logits(Z(2, 3), Z(2), settings=Z(2, 3)),
    lambda: ops.sample_logits(Z(2, 3), Z(2), settings=Z(2, 4).half()),
    lambda: ops.sample_logits(Z(2, 3, dtype=torch.int64), Z(2)),
])
def test_bad_arguments_are_refused(call):
    with pytest.raises(ValueError):
        call()


def test_shapes_on_the_meta_device():
    m = lambda *s, dtype=torch.float32: torch.empty(*s, device="meta", dtype=dtype)
    assert ops.gated_linear(m(3, 5, 8), m(16, 8), m(16, 8), "gelu").shape == (3, 5, 16)
    assert [t.shape for t in ops.residual_norm(m(4, 8), m(4, 8), m(8), m(8), m(8))] == [(4, 8), (4, 8)]
    assert ops.keyed_dropout(m(3, 4, dtype=torch.bfloat16), 0.1, 1).dtype == torch.bfloat16
    i, lp = ops.sample_logits(m(3, 2, 7), m(3, 2))
    assert i.shape == lp.shape == (3, 2) and i.dtype == torch.int64 and lp.dtype == torch.float32
    with pytest.raises(ValueError):
        ops.gated_linear(m(3, 5), m(16, 8), m(16, 8))


def test_entry_points_check_their_arguments():
    lib, P = _lib.load(), 1 << 12                     # P: a pointer that is never followed
    E, U = _lib.MARL_EINVAL, _lib.MARL_EUNSUPPORTED
    gf = lambda dt=0, act=0, rows=2, d=8, h=8, x=P, ldx=8, wg=P, ldg=8, y=P, a=None, b=None, ws=None: \
        lib.marl_gated_forward(dt, act, rows, d, h, x, ldx, wg, ldg, P, 8, y, a, b, ws, None)
    for bad in (dict(dt=3), dict(dt=-1), dict(act=4), dict(rows=0), dict(d=0), dict(h=0), dict(x=None), dict(wg=None), dict(y=None),
                dict(ldx=7), dict(ldg=7), dict(a=P), dict(ws=P + 8), dict(rows=100, x=P + 4)):
        assert gf(**bad) == E, bad
    assert gf(rows=1 << 31) == U and gf(d=(1 << 24) + 1, ldx=1 << 25, ldg=1 << 25) == U
    gb = lambda rows=2, d=8, h=8, a=P, gy=P, ldgy=8, dx=P, dwg=P, dwu=P, ws=P: \
        lib.marl_gated_backward(0, rows, d, h, P, 8, P, 8, P, 8, a, P, gy, ldgy, dx, dwg, dwu, ws, None)
    for bad in (dict(rows=0), dict(a=None), dict(gy=None), dict(ldgy=7), dict(dwu=None), dict(ws=None), dict(ws=P + 8)):
        assert gb(**bad) == E, bad
    ws = lambda dt, rows, d, h, x=P, ldx=8, backward=0: lib.marl_gated_workspace_bytes(dt, rows, d, h, x, ldx, P, ldx, P, ldx, backward)
    assert ws(0, 0, 8, 8, backward=1) == 0 and ws(1, 100, 8, 16, backward=1) >= 100 * 32 * 2
    assert ws(1, 100, 8, 16) == 0 and ws(1, 64, 7, 16, ldx=7) == 0 and ws(1, 100, 8, 16, x=P + 2) >= 100 * 8 * 2
    assert ws(1, 100, 7, 16, ldx=7) >= 100 * 8 * 2 + 2 * 16 * 8 * 2
    nf = lambda dt=0, kind=0, rows=2, d=8, x=P, ldx=8, gate=None, ldg=0, eps=1e-5, stats=None: \
        lib.marl_residual_norm(dt, kind, rows, d, x, ldx, P, 8, P, P, gate, ldg, 1.0, eps, P, P, stats, None)
    for bad in (dict(dt=3), dict(kind=2), dict(rows=0), dict(d=0), dict(x=None), dict(ldx=7), dict(gate=P, ldg=7), dict(eps=-1.0),
                dict(eps=float("nan")), dict(stats=P + 4)):
        assert nf(**bad) == E, bad
    assert nf(d=_lib.MAX_NORM_WIDTH + 1) == U
    nb = lambda stats=P, gate=None, dgate=None, gy=P, ldgy=8, ws=P: \
        lib.marl_residual_norm_backward(0, 0, 2, 8, P, P, 8, P, P, gate, 0, stats, gy, ldgy, None, 0, 1.0, P, P, P, P, dgate, ws, None)
    for bad in (dict(stats=None), dict(stats=P + 4), dict(gate=P), dict(dgate=P), dict(ldgy=7), dict(ws=None), dict(ws=P + 4)):
        assert nb(**bad) == E, bad
    assert lib.marl_residual_norm_workspace_bytes(0) == lib.marl_residual_norm_workspace_bytes(16385) == 0
    kd = lambda dt=0, rows=2, d=8, x=P, ldx=8, p=0.5: lib.marl_keyed_dropout(dt, rows, d, x, ldx, P, None, p, 1, None)
    for bad in (dict(dt=3), dict(rows=0), dict(d=0), dict(x=None), dict(ldx=7), dict(p=1.5), dict(p=-0.5), dict(p=float("nan"))):
        assert kd(**bad) == E, bad
    sl = lambda dt=0, rows=2, V=8, lg=P, ld=8, t=1.0, k=0, p=1.0, m=0.0: lib.marl_sample_logits(dt, rows, V, lg, ld, P, t, k, p, m, None, P, P, None)
    for bad in (dict(dt=3), dict(rows=0), dict(V=0), dict(lg=None), dict(ld=7), dict(t=-1.0), dict(t=float("nan")), dict(k=-1), dict(p=0.0),
                dict(m=-0.1), dict(m=1.1)):
        assert sl(**bad) == E, bad
    assert sl(V=(1 << 20) + 1, ld=1 << 21) == U


def test_gated_trunk_is_refused_on_the_cpu_and_the_default_networks_are_unchanged():
    from marl_amd.agents import Actor, Critic, PPOAgent
    for bad in (dict(trunk="gated"), dict(trunk="conv"), dict(trunk_dropout=0.1), dict(trunk="gated", trunk_dropout=1.0)):
        with pytest.raises(ValueError):
            PPOAgent(device="cpu", **bad)
    assert [k for k in Actor().state_dict()][:2] == ["trunk.0.weight", "trunk.0.bias"] and "network.4.bias" in Critic().state_dict()
    agent = PPOAgent(device="cpu", seed=1)
    assert set(agent._config()) & {"trunk", "trunk_blocks", "trunk_dropout"} == set()


def M(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


# x [2, 3], weights [4, 3], what forward keeps [2, 4]
GATED = dict(gy=(2, 4), x=(2, 3), w_gate=(4, 3), w_up=(4, 3), f=(2, 4), p=(2, 4))
NORM = dict(gy=(2, 3), gn=(2, 3), y=(2, 3), block=(2, 3), w_post=(3,), w_pre=(3,), gate=(3,), stats=(2, 4))


def gated_backward(**other):
    t = {k: M(*s) for k, s in GATED.items()}
    t.update(other)
    return ops.gated_linear_backward(*t.values(), True, True)


def norm_backward(**other):
    t = {k: M(*s) for k, s in NORM.items()}
    t.update(other)
    return ops.residual_norm_backward(*t.values(), 1.0, "rms")


def test_backward_shapes():
    assert [tuple(g.shape) for g in gated_backward()] == [(2, 3), (4, 3), (4, 3)]
    assert [tuple(g.shape) for g in norm_backward()] == [(2, 3), (2, 3), (3,), (3,), (3,)]
    assert len(norm_backward(gy=None, gate=None)) == 5


@pytest.mark.parametrize("name", ["gy", "f", "p"])
def test_gated_backward_refuses_what_forward_did_not_keep(name):
    bad = [M(1, 4), M(2, 3), M(2, 4, dtype=torch.float16)] + ([] if name == "gy" else [M(4, 2).t()])
    for t in bad:
        with pytest.raises(ValueError):
            gated_backward(**{name: t})


@pytest.mark.parametrize("name", ["gy", "gn", "y", "block", "w_post", "w_pre", "gate", "stats"])
def test_norm_backward_refuses_what_forward_did_not_keep(name):
    bad = [M(1, 3), M(2, 2), M(*NORM[name], dtype=torch.float16)] + ([M(3, 2).t()] if name == "y" else [M(4, 2).t()] if name == "stats" else [])
    for t in bad:
        with pytest.raises(ValueError):
            norm_backward(**{name: t})


BEYOND = (1 << 32) + 1          # cut to 32 bits this is 1


@pytest.mark.parametrize("call", [
    lambda: ops.gated_linear(M(1, 1), M(BEYOND, 1), M(BEYOND, 1)),
    lambda: ops.gated_linear(M(1, BEYOND), M(1, BEYOND), M(1, BEYOND)),
    lambda: ops.keyed_dropout(M(1, BEYOND), 0.5, 1),
])
def test_sizes_beyond_32_bits_are_refused(call):
    with pytest.raises(ValueError):
        call()
