"""CPU tests of which topologies go to the tensor cores: neurons that share their connections, in blocks of up to 16."""
import ctypes as C

import numpy as np
import pytest

from graphchallenge21_b200 import SparseTopology, _lib
from graphchallenge21_b200.generator import SyntheticNetwork
from test_gpu_feedforward import shared_rows

# inputs, outputs, slots, group; blocks forward and backward
SHARED = [(256, 320, 32, 16, (20, 16)), (1024, 1024, 32, 16, (64, 64)), (300, 333, 45, 15, (23, 20)), (64, 33, 32, 32, (3, 4)),
          (96, 1600, 48, 16, (100, 6)), (192, 480, 64, 12, (40, 22)), (128, 80, 64, 16, (5, 8)), (512, 333, 96, 16, (21, 32)),
          (17600, 17600, 32, 16, (1100, 1100)), (32768, 32768, 32, 16, (2048, 2048))]


@pytest.mark.parametrize("scattered", [False, True])
@pytest.mark.parametrize("inputs, outputs, slots, group, blocks", SHARED)
def test_blocks_do_not_depend_on_the_numbering(inputs, outputs, slots, group, blocks, scattered):
    """As many where neighbours share their connections as where both sides are renumbered at random."""
    top = SparseTopology.from_rows(shared_rows(inputs, outputs, slots, group, scattered), inputs, device=None)
    assert top.blocks == blocks


@pytest.mark.parametrize("inputs, outputs, slots, group, blocks", [(128, 96, 20, 10, (0, 0)), (96, 1600, 8, 8, (0, 0)), (512, 100, 48, 16, (7, 0)),
                                                                  (360, 350, 30, 12, (30, 0)), (640, 77, 64, 16, (5, 0))])
def test_small_groups_and_short_lists_are_not_worth_blocks(inputs, outputs, slots, group, blocks):
    top = SparseTopology.from_rows(shared_rows(inputs, outputs, slots, group, False), inputs, device=None)
    assert top.blocks == blocks


def test_random_and_challenge_networks():
    rng = np.random.default_rng(1)
    assert SparseTopology.from_rows(rng.integers(0, 4096, (4096, 32)), 4096, device=None).blocks == (0, 0)
    cp, ri, _ = SyntheticNetwork(4096, 3, "radix16").layer_csc(2)
    assert SparseTopology(4096, 4096, cp, ri, device=None).blocks == (256, 256)
    assert SparseTopology(5, 3, np.zeros(4), np.zeros(0), device=None).blocks == (0, 0)
    n = C.c_int(7)
    assert _lib.load().spdnn_topology_blocks(None, C.byref(n), None) == -1 and n.value == 7
