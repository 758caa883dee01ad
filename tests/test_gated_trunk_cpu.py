"""Parts of the gated trunk that need no GPU."""
import pytest

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
