"""CPU tests of the feed-forward operators: the host analysis of topologies and the refusals that need no GPU."""
import ctypes as C

import numpy as np
import pytest

from graphchallenge21_b200 import SparseTopology, SpDNNError, _lib
from graphchallenge21_b200.generator import SyntheticNetwork


def err_of(fn, *args):
    err = C.create_string_buffer(256)
    return fn(*args, err, 256), err.value.decode()


def test_operand_struct_matches_header_size():
    assert C.sizeof(_lib.Operand) == 32      # two pointers, int64, two int32


def test_canonical_order_of_a_ragged_topology():
    rows = np.array([[7, 2, -1, 4], [-1, -1, -1, -1], [0, 0, 5, -1], [9, 8, 1, 3]])
    top = SparseTopology.from_rows(rows, 10, device=None)
    assert (top.inputs, top.outputs, top.slots, top.connections) == (10, 4, 4, 10)
    assert top.fan_out == 2                                   # input 0, twice in one neuron
    assert np.array_equal(top.rows(), [[2, 4, 7, -1], [-1, -1, -1, -1], [0, 0, 5, -1], [1, 3, 8, 9]])
    packed = top.pack(np.arange(10, 20))                      # in the order of the rows above, -1 left out
    assert np.array_equal(packed, [[11, 12, 10, 0], [0, 0, 0, 0], [13, 14, 15, 0], [18, 19, 17, 16]])


def test_no_connections_at_all():
    top = SparseTopology(5, 3, np.zeros(4), np.zeros(0), device=None)
    assert top.slots == 1 and top.connections == 0 and top.fan_out == 0
    assert np.array_equal(top.rows(), -np.ones((3, 1)))


def test_layers_of_a_generated_network():
    net = SyntheticNetwork(1024, 3, "radix16")
    cp, ri, _ = net.layer_csc(1)
    top = SparseTopology(1024, 1024, cp, ri, device=None)
    assert top.slots == 32 and top.fan_out == 32 and top.connections == 32 * 1024
    assert np.array_equal(top.rows(), np.sort(np.asarray(ri).reshape(1024, 32), axis=1))


@pytest.mark.parametrize("inputs, outputs, col_ptr, row_idx, says", [
    (0, 2, [0, 1, 2], [0, 0], "inputs and outputs"),
    (1 << 26, 1, [0, 1], [0], "inputs and outputs"),
    (4, 2, [1, 1, 2], [0, 0], "col_ptr[0]"),
    (4, 2, [0, 2, 1], [0, 1], "non-decreasing"),
    (4, 2, [0, 1, 2], [0, 4], "out of range in column 1"),
    (4, 2, [0, 1, 2], [-1, 0], "out of range in column 0"),
    (4, 1, [0, 4097], [0] * 4097, "4096"),
])
def test_malformed_topologies_are_refused(inputs, outputs, col_ptr, row_idx, says):
    lib = _lib.load()
    cp, ri = np.array(col_ptr, np.int32), np.array(row_idx, np.int32)
    top = C.c_void_p(1)
    rc, msg = err_of(lib.spdnn_topology_create, C.byref(top), -1, inputs, outputs, 0, cp.ctypes.data, ri.ctypes.data)
    assert rc == -1 and says in msg and not top.value


def test_null_arguments_are_refused():
    lib = _lib.load()
    top = C.c_void_p()
    assert err_of(lib.spdnn_topology_create, None, -1, 4, 4, 0, None, None)[0] == -1
    assert err_of(lib.spdnn_topology_create, C.byref(top), -1, 4, 4, 0, None, None)[0] == -1
    cp = np.array([0, 1], np.int32)
    rc, msg = err_of(lib.spdnn_topology_create, C.byref(top), -1, 4, 1, 0, cp.ctypes.data, None)
    assert rc == -1 and "row_idx" in msg
    assert lib.spdnn_topology_info(None, None, None, None, None, None) == -1
    assert lib.spdnn_topology_rows(None, None, 0) == -1
    lib.spdnn_topology_destroy(None)
    n = C.c_int64()
    assert lib.spdnn_layer_workspace(None, 1, 1, 0, 0, 0, C.byref(n)) == -1


def operand(type=0, data=4096, scales=None, stride=1 << 20):
    return _lib.Operand(data, scales, stride, type, 0)


@pytest.fixture(scope="module")
def analysis():
    top = SparseTopology.from_rows(np.array([[0, 1], [2, 3], [1, -1]]), 4, device=None)
    yield top
    top.close()


def linear(top, tokens=2, x=operand(), w=operand(), act=0, clip=32.0, y=operand(), z=None):
    ref = lambda o: None if o is None else C.byref(o)  # noqa: E731
    return err_of(_lib.load().spdnn_linear, top and top._top, tokens, ref(x), ref(w), None, act, clip, ref(y), ref(z), 4096, 1 << 20, None)


@pytest.mark.parametrize("case, says", [
    (dict(tokens=-1), "tokens"), (dict(tokens=(1 << 26) + 1), "tokens"), (dict(act=6), "activation"), (dict(act=-1), "activation"),
    (dict(act=2, clip=0.0), "clip"), (dict(act=2, clip=float("nan")), "clip"),
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"),
    (dict(x=operand(type=7)), "type"), (dict(w=operand(type=-1)), "type"), (dict(y=operand(type=3)), "type"),
    (dict(x=operand(data=None)), "no data"), (dict(w=operand(data=None)), "no data"), (dict(y=operand(data=None)), "no data"),
    (dict(x=operand(stride=3)), "stride"), (dict(w=operand(stride=1)), "stride"), (dict(y=operand(stride=2)), "stride"),
    (dict(x=operand(data=4098)), "aligned"), (dict(x=operand(type=1, data=4097), w=operand(type=1)), "aligned"),
    (dict(x=operand(type=3, scales=4096, data=4098), w=operand(type=3, scales=4096)), "aligned"),
    (dict(w=operand(type=2)), "activations' type"), (dict(x=operand(type=3, scales=4096)), "activations' type"),
    (dict(w=operand(type=3)), "scales"), (dict(z=operand(type=1)), "pre-activations are saved as fp32"),
    (dict(), "analysis only"),
])
def test_refusals_of_a_layer(analysis, case, says):
    rc, msg = linear(analysis, **case)
    assert says in msg and rc == (-4 if says == "analysis only" else -1)


def test_refusals_of_the_gated_block_and_of_backward_calls(analysis):
    lib = _lib.load()
    o, f16, mx = operand(), operand(type=1), operand(type=3, scales=4096)
    r = C.byref
    tail = (4096, 1 << 20, None)
    gated = lambda x, wg, wu, y, zg, zu: err_of(lib.spdnn_gated, analysis._top, 2, r(x), r(wg), r(wu), None, None, 3, 32.0, r(y),  # noqa: E731
                                                zg, zu, *tail)
    assert "one type" in gated(o, o, f16, o, None, None)[1]
    assert "both pre-activations" in gated(o, o, o, o, r(o), None)[1]
    assert "one stride" in gated(o, o, o, o, r(o), r(operand(stride=77)))[1]
    back = lambda dy, x, w, z, dx, dw, db, act=3: err_of(lib.spdnn_linear_backward, analysis._top, 2, r(dy), r(x), r(w), z, act, 32.0, dx,  # noqa: E731
                                                         dw, db, *tail)
    assert "dy must have" in back(f16, o, o, r(o), None, None, None)[1]
    assert "type" in back(o, mx, mx, r(o), None, None, None)[1]
    assert "null" in back(o, o, o, None, None, None, None)[1]
    assert "dx must have" in back(o, o, o, r(o), r(f16), None, None)[1]
    assert "biases" in back(o, o, o, r(o), r(o), None, 4096)[1]
    assert "aligned" in back(o, o, o, r(o), r(o), 4098, None)[1] and "aligned" in back(o, o, o, r(o), r(o), 4096, 4097)[1]
    assert "aligned" in err_of(lib.spdnn_linear, analysis._top, 2, r(o), r(o), 4097, 0, 32.0, r(o), None, *tail)[1]
    assert back(o, o, o, None, r(o), 4096, 4096, act=0)[0] == -4        # nothing saved is needed without an activation
    rc, msg = err_of(lib.spdnn_gated_backward, analysis._top, 2, r(o), r(o), r(o), r(o), r(o), r(o), 3, 32.0, None, 4096, None, None, None,
                     *tail)
    assert rc == -1 and "both sets" in msg


def test_refusals_of_microscaled_matrices():
    lib = _lib.load()
    q = lambda x, rows, cols, codes=4096, scales=4096: err_of(lib.spdnn_mx4_quantize, C.byref(x), rows, cols, codes, scales, None)  # noqa: E731
    assert q(operand(), 2, 0)[0] == -1 and q(operand(), -1, 4)[0] == -1 and q(operand(), 1 << 40, 32)[0] == -1
    assert "null" in q(operand(), 2, 4, codes=None)[1] and "null" in q(operand(), 2, 4, scales=None)[1]
    assert "aligned" in q(operand(), 2, 4, codes=4098)[1] and "stride" in q(operand(stride=3), 2, 4)[1]
    assert "type" in q(operand(type=3, scales=4096), 2, 4)[1]
    assert q(operand(data=None), 0, 4, None, None)[0] == 0              # no rows: nothing to do
    rc, msg = err_of(lib.spdnn_mx4_dequantize, 4096, None, 2, 4, C.byref(operand()), None)
    assert rc == -1 and "null" in msg


def test_python_refusals_without_a_gpu(analysis):
    import torch
    x, w = torch.zeros(2, 4), torch.zeros(3, 2)
    with pytest.raises(SpDNNError, match="analysis only"):
        analysis.linear(x, w)
    with pytest.raises(SpDNNError, match="col_ptr must have"):
        SparseTopology(4, 3, [0, 1], [0], device=None)
    with pytest.raises(SpDNNError, match="row_idx size"):
        SparseTopology(4, 1, [0, 2], [0], device=None)
    with pytest.raises(SpDNNError, match="val size"):
        analysis.pack([1.0])
    from graphchallenge21_b200 import MX4, mx4_quantize
    with pytest.raises(SpDNNError, match="CUDA tensor"):
        mx4_quantize(x)
    with pytest.raises(SpDNNError, match="codes must be"):
        MX4(torch.zeros(2, 1, 8, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8), 4)
    closed = SparseTopology(4, 1, [0, 1], [0], device=None)
    closed.close()
    with pytest.raises(SpDNNError, match="closed"):
        closed.rows()
    with pytest.raises(SpDNNError, match="closed"):
        closed.linear(x, w)


def test_microscaled_reference_of_the_tests():
    """The definition itself, on values worked out by hand."""
    from feedforward_reference import mx4_reference
    v = np.zeros((5, 33))
    v[0, :9] = [6, 5, -5.1, 2.5, 3.5, 0.25, 0.75, -0.26, 7.9]     # max 7.9: scale 1
    v[1, 0] = 2.0 ** -140                                          # below the smallest scale
    v[2, 3] = np.inf
    v[3, 32] = 3.0                                                 # the second block, one column long: scale 2^-1
    codes, scales, values = mx4_reference(v)
    assert np.array_equal(values[0, :9], [6, 4, -6, 2, 4, 0, 1, -0.5, 6])
    assert scales[:, 0].tolist() == [127, 0, 255, 0, 0] and scales[3, 1] == 126
    assert np.isnan(values[2, :32]).all() and values[2, 32] == 0 and values[3, 32] == 3.0 and codes[3, 1, 0] == 7
    assert codes[0, 0, 0] == 7 | 6 << 4 and codes[0, 0, 1] == (8 | 7) | 4 << 4


def test_slots_are_the_width_that_was_asked_for():
    """A table of rows keeps its width where no neuron uses all of it; CSC takes the longest, or what it is given."""
    rows = np.array([[3, -1, 1], [2, -1, -1]])
    top = SparseTopology.from_rows(rows, 4, device=None)
    assert top.slots == 3 and np.array_equal(top.rows(), [[1, 3, -1], [2, -1, -1]])
    assert np.array_equal(top.pack([5, 6, 7]), [[6, 5, 0], [7, 0, 0]])
    csc = ([0, 2, 3], [3, 1, 2])
    assert SparseTopology(4, 2, *csc, device=None).slots == 2 and SparseTopology(4, 2, *csc, device=None, slots=7).slots == 7
    for bad in (1, -1, 4097):
        with pytest.raises(SpDNNError, match="slots"):
            SparseTopology(4, 2, *csc, device=None, slots=bad)
