"""CPU tests of what the binding of the feed-forward operators checks before a pointer reaches the library."""
import pytest

from graphchallenge21_b200 import Saved, SparseTopology, SpDNNError
from graphchallenge21_b200 import feedforward

torch = pytest.importorskip("torch")


def on_the_host():
    """A topology of 6 outputs whose device is where CPU tensors are: for checks that need no library."""
    feedforward._torch()
    top = SparseTopology.__new__(SparseTopology)
    top.device, top.outputs = torch.zeros(1).get_device(), 6
    return top


def test_saved_pre_activations_of_another_type_or_layout_are_refused():
    """The kernels read [sets, tokens, outputs] float32 from the first element on: halved types and views with gaps or overlaps would
    be read beyond their end, or in the wrong order."""
    top = on_the_host()
    z = torch.zeros(2, 5, 6)
    assert top._pre_activations(Saved(z), 2, 5) is z
    for other in (z.bfloat16(), z.half(), z.double(), z.int()):
        with pytest.raises(SpDNNError, match="contiguous float32"):
            top._pre_activations(Saved(other), 2, 5)
    for view in (torch.zeros(2, 6, 5).transpose(1, 2), torch.zeros(2, 5, 7)[:, :, :6], torch.zeros(1, 5, 6).expand(2, 5, 6),
                 torch.zeros(2, 1, 6).expand(2, 5, 6), torch.zeros(4, 5, 6)[::2]):
        assert view.shape == (2, 5, 6)
        with pytest.raises(SpDNNError, match="contiguous float32"):
            top._pre_activations(Saved(view), 2, 5)
    for wrong in (None, Saved(z[:1]), Saved(torch.zeros(2, 5, 7)), Saved(torch.zeros(2, 4, 6))):
        with pytest.raises(SpDNNError, match="what the forward call returned"):
            top._pre_activations(wrong, 2, 5)
