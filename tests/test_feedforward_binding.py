"""CPU tests of what the binding of the feed-forward operators checks before a pointer reaches the library."""
import os
import subprocess

import numpy as np
import pytest

from graphchallenge21_b200 import MX4, Saved, SparseTopology, SpDNNError, mx4_quantize
from graphchallenge21_b200 import build, feedforward

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


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    """tests/topology_device_harness.cpp, built with the host compiler against the headers of the CUDA runtime."""
    cxx, nvcc = build._host_cxx()[1:] or ["g++"], build._nvcc()
    exe = str(tmp_path_factory.mktemp("harness") / "topology_device")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")
    subprocess.run([*cxx, "-std=c++17", "-O1", "-pthread", "-I", build.CSRC, "-I", include, "-o", exe,
                    os.path.join(os.path.dirname(os.path.abspath(__file__)), "topology_device_harness.cpp")], check=True)
    return lambda *args: subprocess.run([exe, *map(str, args)], check=True, capture_output=True, text=True, timeout=120).stdout.split()


def test_a_topology_is_on_the_gpu_when_its_creation_returns(harness):
    """Copies from pageable memory may return before they are done, and a call on another stream than theirs does not wait for them."""
    assert harness("ordered") == ["0"]


def test_a_topology_that_cannot_be_created_leaves_no_device_memory(harness):
    device, host = map(int, harness("calls"))
    assert device == 18 and host >= 1
    for where, times in (("device", device), ("host", host)):
        for n in range(1, times + 1):
            assert harness(where, n) == ["1", "0"], (where, n)


@pytest.mark.parametrize("rows", [[2 ** 32 + 3], [2 ** 31], [-2 ** 32 + 1], [3.9], [float("nan")], [float("inf")], [2.0 ** 40], [2 ** 64], [1j],
                                  np.array([2 ** 63 + 1], dtype=np.uint64)])
def test_indices_that_are_not_32_bit_integers_are_refused(rows):
    """A cast would make another index of them that the library cannot tell from the one that was meant."""
    with pytest.raises(SpDNNError, match="row_idx"):
        SparseTopology(8, 1, [0, 1], rows, device=None)
    with pytest.raises(SpDNNError, match="col_ptr"):
        SparseTopology(8, 1, [0, rows[0]], [0], device=None)


def test_rows_that_are_not_a_matrix_of_indices_are_refused():
    for rows, says in (([[2 ** 32 + 3]], "beyond 32 bits"), ([[3.9]], "integers"), ([[float("nan"), 1]], "integers"), ([[-0.5, 1]], "integers"),
                       ([3, 4], "matrix"), (3, "matrix")):
        with pytest.raises(SpDNNError, match=says):
            SparseTopology.from_rows(rows, 8, device=None)
    # whole numbers of other types, and any negative number for a connection that is not there, are what they were
    for t in (np.int8, np.uint16, np.int64, np.float32):
        assert SparseTopology.from_rows(np.array([[3, 1]], dtype=t), 8, device=None).rows().tolist() == [[1, 3]]
    assert SparseTopology.from_rows([[3, -2 ** 40], [1, -1]], 8, device=None).rows().tolist() == [[3, -1], [1, -1]]


def test_sizes_beyond_32_bits_are_refused():
    """They would reach the library modulo 2^32."""
    for sizes in (dict(inputs=2 ** 32 + 4), dict(inputs=4 - 2 ** 32), dict(inputs=4, slots=2 ** 32 + 2), dict(inputs=4, device=2 ** 32)):
        with pytest.raises(SpDNNError, match="out of range"):
            SparseTopology(outputs=1, col_ptr=[0, 1], row_idx=[0], **{"device": None, **sizes})
    with pytest.raises(SpDNNError, match="inputs and outputs"):
        SparseTopology(2 ** 31 - 1, 1, [0, 1], [0], device=None)


class Shape:
    """What the binding looks at of a tensor that is too large for this test."""
    is_cuda, dtype = True, torch.float16

    def __init__(self, *shape):
        self.shape = shape

    def dim(self):
        return len(self.shape)


def test_matrices_of_more_rows_or_columns_than_a_call_takes_are_refused():
    top = on_the_host()
    top.inputs, top.slots, top._top = 1, 1, True
    for tokens in (2 ** 26 + 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5):
        with pytest.raises(SpDNNError, match="tokens a call"):
            top._begin(Shape(tokens, 1), (), "none")
    for cols in (2 ** 30 + 1, 2 ** 32 + 32):
        with pytest.raises(SpDNNError, match="columns"):
            mx4_quantize(Shape(1, cols))
        with pytest.raises(SpDNNError, match="columns"):
            MX4(Shape(1, cols // 32, 16), Shape(1, cols // 32), cols)


def test_tensors_that_require_grad_are_refused_in_grad_mode():
    top = on_the_host()
    bias = torch.zeros(6, requires_grad=True)

    class Parameter:
        """A matrix on the GPU as far as the binding looks."""
        is_cuda, dtype, requires_grad, shape = True, torch.float32, True, (3, 4)
        stride, data_ptr, get_device = (lambda self: (4, 1)), (lambda self: 0), (lambda self: 0)

    with pytest.raises(SpDNNError, match="weights requires grad"):
        feedforward._operand(Parameter(), 3, 4, 0, "weights")
    with pytest.raises(SpDNNError, match="a bias requires grad"):
        top._bias(bias)
    with torch.no_grad():
        feedforward._operand(Parameter(), 3, 4, 0, "weights")
        assert top._bias(bias) == bias.data_ptr()
    assert top._bias(bias.detach()) == bias.data_ptr()
