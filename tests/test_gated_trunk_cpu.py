"""Parts of the gated trunk that need no GPU."""
import pytest
import torch

from marl_amd.agents import Critic, _dropout_seed


def test_an_unknown_trunk_of_the_critic_is_refused():
    with pytest.raises(ValueError):
        Critic(trunk="conv")
    assert "network.4.bias" in Critic(trunk="mlp").state_dict()


@pytest.mark.parametrize("seed", [0, 1, -1, (1 << 55) - 1, 1 << 55, (1 << 64) - 1, None])
def test_dropout_seeds_are_int64_and_leave_room_for_the_blocks(seed):
    s = _dropout_seed(seed)
    assert 0 <= s and s + 255 < 1 << 63 and s % 256 == 0
    if seed is not None and 0 <= seed < 1 << 55:
        assert s == seed << 8


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_what_gated_linear_keeps_is_float32(dtype):
    import marl_amd.ops  # noqa: F401  registers torch.ops.marl_amd
    ops = torch.ops.marl_amd
    m = lambda *s, dtype=dtype: torch.empty(*s, dtype=dtype, device="meta")
    y, f, p = ops.gated_linear_saved(m(2, 3), m(4, 3), m(4, 3), "gelu")
    assert y.dtype == dtype and f.dtype == p.dtype == torch.float32 and f.shape == p.shape == (2, 4)
    assert all(g.dtype == dtype for g in ops.gated_linear_backward(m(2, 4), m(2, 3), m(4, 3), m(4, 3), f, p, True, True))
    if dtype != torch.float32:
        for kept in ((m(2, 4), p), (f, m(2, 4))):
            with pytest.raises(ValueError):
                ops.gated_linear_backward(m(2, 4), m(2, 3), m(4, 3), m(4, 3), *kept, True, True)
