"""sample_logits where a logit lies on the border of a bin but for less than the rounding of the distance to the maximum."""
import pytest
import torch

import marl_amd.ops  # noqa: F401  registers torch.ops.marl_amd
from test_hip_trunk_ops import sample_check

pytestmark = pytest.mark.gpu


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
