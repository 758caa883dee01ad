"""sample_logits at its borders: of bins (a logit on the border but for less than the rounding of the distance to the maximum), of
the row lengths and row counts at which another kernel is taken."""
import pytest
import torch

import marl_amd.ops  # noqa: F401  registers torch.ops.marl_amd
from test_hip_trunk_ops import sample_check

pytestmark = pytest.mark.gpu
ops = torch.ops.marl_amd


@pytest.mark.parametrize("V", [3000, 8192, 20000])
@pytest.mark.parametrize("temperature", [1.2434278726577759, 2.829232692718506, 2.944525480270386, 0.7, 1.0])
@pytest.mark.parametrize("low", [-1e-17, 1e-17, -1e-16, 0.0])
def test_logits_next_to_zero_below_a_maximum_of_the_temperature(V, temperature, low):
    """(low - top) / temperature rounds to a number on one side of -1, the border itself to one on the other."""
    t = torch.tensor(temperature)
    logits = torch.full((8, V), low)
    for r in range(8):
        logits[r, (r * 997) % V] = t * 2.0 ** (r % 3)
        logits[r, (r * 331 + 5) % V] = -t
    u = torch.tensor([0.01, 0.2, 0.35, 0.5, 0.65, 0.8, 0.95, 0.9999])
    for k, p in ((64, 1.0), (64, 0.9), (0, 0.5), (1500, 1.0), (200, 0.7)):
        sample_check(logits, u, float(t), k, p, 0.0)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 3, 1.0, 0.0), (1.3, 0, 0.8, 0.0), (0.9, 40, 0.9, 0.05), (0.8, 100, 0.95, 0.0), (5.0, 700, 0.97, 0.0)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("V", [127, 128, 129, 256, 257, 511, 512, 513, 1023, 1024, 1025, 2047, 2048, 2049, 8191, 8192, 8193])
def test_both_sides_of_every_length_at_which_the_kernel_changes(V, dt):
    g = torch.Generator().manual_seed(V)
    logits = (3 * torch.randn(6, V, generator=g)).to(dt)
    logits[5, V // 3:] = float("-inf")
    u = torch.rand(6, generator=g)
    for s in SETTINGS:
        sample_check(logits, u, *s)


@pytest.mark.parametrize("R,V", [(511, 9001), (512, 9001), (512, 131072), (512, 131073)])
def test_both_sides_of_the_rule_for_many_long_rows(R, V):
    """A row drawn among many is the row drawn among few; the first ones against the definition."""
    g = torch.Generator(device="cuda").manual_seed(R + V)
    logits = (3 * torch.randn(R, V, device="cuda", generator=g)).to(torch.float16)
    u = torch.rand(R, device="cuda", generator=g)
    for s in SETTINGS:
        many = ops.sample_logits(logits, u, *s)
        for at in (slice(0, 3), slice(R - 3, R)):
            few = ops.sample_logits(logits[at], u[at], *s)
            assert torch.equal(many[0][at], few[0]) and torch.equal(many[1][at], few[1])
        if V < 10000:
            sample_check(logits[:3].cpu(), u[:3].cpu(), *s)
