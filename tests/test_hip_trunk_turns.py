"""GPU tests of the trunk operators at sizes where a workgroup takes more than one turn of its loop over rows (rows beyond what
the chip holds at once, with a ragged last turn) or a tile takes all of a long k."""
import pytest
import torch

import marl_amd.ops  # noqa: F401  registers torch.ops.marl_amd
from test_hip_trunk_ops import BF16, F16, F32, U, close, draws, gated_check, gen, half_step, norm_check, tiny

pytestmark = pytest.mark.gpu
ops = torch.ops.marl_amd


# rows at once: 256 (2048 / threads) workgroups of threads / lanes rows
@pytest.mark.parametrize("T,d,dt,kind,gate", [
    (33001, 64, F32, "layer", "channel"),        # 16 lanes a row: 32768 at once
    (16411, 128, F32, "layer", "channel"),       # 32: 16384
    (8203, 500, F16, "rms", "row"),              # 64: 8192
    (4099, 1021, BF16, "layer", "none"),         # 128: 4096
    (2053, 1024, F32, "rms", "channel"),         # 256: 2048
    (1031, 4096, F16, "layer", "row"),           # 512: 1024
    (1100, 4097, F16, "rms", "row"),             # 512, two chunks a thread
    (1100, 8192, BF16, "layer", "channel"),
    (530, 8191, F32, "layer", "channel"),        # 1024, two chunks: 512
    (530, 16384, F32, "layer", "channel"),       # 1024, four chunks
    (530, 16384, F32, "rms", "row"),
])
def test_residual_norm_more_rows_than_the_chip_holds(T, d, dt, kind, gate):
    norm_check(T, d, dt, kind, gate, seed=d)


def columns(t):
    """A slice of columns that begins one element behind a 16-byte border."""
    wide = torch.full((t.shape[0], t.shape[1] + 3), float("nan"), dtype=t.dtype, device="cuda")
    wide[:, 1:1 + t.shape[1]] = t
    return wide[:, 1:1 + t.shape[1]].detach()


@pytest.mark.parametrize("T,d,h,dt,prepare", [(65539, 8, 16, BF16, lambda t: t), (66001, 9, 7, F32, lambda t: t), (65600, 16, 9, F16, columns)])
def test_gated_linear_more_rows_than_a_grid_dimension(T, d, h, dt, prepare):
    gated_check(T, d, h, dt, "silu", seed=d, prepare=prepare)


@pytest.mark.parametrize("T,d", [((1 << 21) + 777, 16), ((1 << 22) + 1301, 5)])
def test_keyed_dropout_more_groups_than_threads(T, d):
    x = torch.randn(T, d, device="cuda").to(BF16).requires_grad_(True)
    gy = torch.randn(T, d, device="cuda").to(BF16)
    keys = torch.arange(T, device="cuda") * 3 + (7 << 32)
    y = ops.keyed_dropout(x, 0.25, 21, keys)
    g, = torch.autograd.grad(y, x, gy)
    rows = torch.cat([torch.arange(0, 1000), torch.arange(T // 2, T // 2 + 1000), torch.arange(T - 3000, T)])
    keep = draws((rows * 3 + (7 << 32)).numpy(), d, 21) >= 16384
    at = rows.cuda()
    for got, v in ((y, x), (g, gy)):
        want = torch.where(keep, v.detach()[at].double().cpu() * (65536 / 49152), torch.zeros((), dtype=torch.float64))
        close("dropout", got[at], want, (half_step(BF16) + 3 * U) * want.abs() + tiny(BF16))
    # every row was written, by the same rule: the mask of the gradient is that of the value
    assert torch.equal(y.detach() == 0, (g == 0) | (x.detach() == 0)) or bool(((y.detach() == 0) == (g == 0))[(x.detach() != 0) & (gy != 0)].all())


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("T,d,h", [(64, 4096, 128), (65, 4096, 128), (64, 2500, 512), (65, 2500, 512), (300, 4096, 130)])
def test_gated_linear_narrow_weights_of_long_rows(T, d, h, dt):
    """Both sides of the number of rows up to which k is sliced in forward."""
    gated_check(T, d, h, dt, "silu", seed=T + h)
