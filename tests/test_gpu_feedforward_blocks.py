"""GPU tests of topologies that have blocks in both directions (tests/test_feedforward_blocks.py says which have)."""
import pytest

from test_feedforward_blocks import SHARED
from test_gpu_feedforward import BF16, F16, Shared, check_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("sets", [1, 2])
@pytest.mark.parametrize("tokens, scattered", [(17, True), (64, False), (150, True)])
@pytest.mark.parametrize("inputs, outputs, slots, group, blocks", SHARED[:-2])
def test_steps_of_blocks_in_both_directions(inputs, outputs, slots, group, blocks, tokens, scattered, sets, dtype):
    p = Shared(tokens, inputs, outputs, slots, dtype, sets, group, scattered)
    assert p.top.blocks == blocks
    check_step(p, "silu")


@pytest.mark.parametrize("sets", [1, 2])
def test_a_step_of_more_than_a_thousand_scattered_blocks(sets):
    inputs, outputs, slots, group, blocks = SHARED[-2]
    p = Shared(70, inputs, outputs, slots, BF16, sets, group, True)
    assert p.top.blocks == blocks
    check_step(p, "gelu")
