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


@pytest.mark.parametrize("tokens", [1, 200])
def test_the_first_call_comes_from_another_stream_at_once(tokens):
    from graphchallenge21_b200 import SparseTopology
    p = Problem(tokens, 4000, 5000, 48, BF16, 1)
    want = p.forward("none")
    torch.cuda.synchronize()
    for _ in range(8):
        top = SparseTopology.from_rows(p.rows_given, 4000)
        with torch.cuda.stream(torch.cuda.Stream()):
            y = top.linear(p.x, p.w[0], p.b[0])
            torch.cuda.current_stream().synchronize()
        assert torch.equal(y, want)
        top.close()
