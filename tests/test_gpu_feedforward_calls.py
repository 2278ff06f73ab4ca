"""GPU tests of how the feed-forward operators are called: what they refuse, and first calls."""
import pytest

from test_gpu_feedforward import BF16, Problem, torch

pytestmark = pytest.mark.gpu


def test_saved_pre_activations_of_another_type_or_layout_are_refused():
    from graphchallenge21_b200 import Saved, SpDNNError
    p = Problem(5, 40, 30, 4, BF16, 2)
    y, saved = p.forward("silu", save=True)
    want = p.backward(saved, "silu")
    wide = torch.empty(2, 5, 32, device="cuda")[:, :, :30].copy_(saved.z)
    for z in (saved.z.bfloat16(), saved.z.half(), saved.z.transpose(1, 2).contiguous().transpose(1, 2), wide, saved.z[:1].expand(2, 5, 30)):
        with pytest.raises(SpDNNError, match="contiguous float32"):
            p.backward(Saved(z), "silu")
    got = p.backward(Saved(saved.z.clone()), "silu")
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1] + got[2], want[1] + want[2]))
