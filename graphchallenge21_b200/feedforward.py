"""Feed-forward operators on torch CUDA tensors, over the C ABI (include/spdnn_b200.h).

``SparseTopology`` holds which inputs every output neuron is connected to, on one GPU; its methods run the plain layer
``act(x W + b)`` and the gated block ``act(x Wg + bg) * (x Wu + bu)`` on activations ``[tokens, neurons]`` with the
weights given to each call, and their gradients.  ``mx4_quantize`` makes microscaled 4-bit matrices (``MX4``) of weights or
activations, which the forward calls take in place of tensors.

Calls enqueue on torch's current stream of the tensors' device and return at once; they may be captured into CUDA graphs.
Nothing here is differentiated by autograd: the gradients are the ``*_backward`` calls.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from .network import SpDNNError

ACTIVATIONS = {"none": 0, "relu": 1, "clip": 2, "silu": 3, "gelu": 4, "gelu_tanh": 5}
F32, F16, BF16, MX4_TYPE = 0, 1, 2, 3
_ERR_LEN = 256


def _type_of(dtype):
    import torch
    t = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}.get(dtype)
    if t is None:
        raise SpDNNError(-1, f"type {dtype} is not float32, float16 or bfloat16")
    return t


def _call(fn, *args):
    err = C.create_string_buffer(_ERR_LEN)
    rc = fn(*args, err, _ERR_LEN)
    if rc != 0:
        raise SpDNNError(rc, err.value.decode())


def _stream(device):
    import torch
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _ref(operand):
    return None if operand is None else C.byref(operand)


def _data(t):
    return None if t is None else C.c_void_p(t.data_ptr())


class MX4:
    """A matrix of microscaled 4-bit floats: ``codes`` uint8 [rows, blocks, 16], ``scales`` uint8 [rows, blocks], blocks of 32
    of its ``cols`` columns (include/spdnn_b200.h says what the bytes mean)."""

    def __init__(self, codes, scales, cols: int):
        import torch
        blocks = (int(cols) + 31) // 32
        if (codes.dim() != 3 or codes.dtype != torch.uint8 or codes.shape[2] != 16 or codes.shape[1] != blocks or cols < 1
                or scales.dtype != torch.uint8 or tuple(scales.shape) != tuple(codes.shape[:2])):
            raise SpDNNError(-1, f"codes must be uint8 [rows, {blocks}, 16] and scales uint8 [rows, {blocks}]")
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.device != scales.device or not codes.is_cuda:
            raise SpDNNError(-1, "codes and scales must be contiguous and on one GPU")
        self.codes, self.scales, self.cols = codes, scales, int(cols)

    @property
    def shape(self):
        return (int(self.codes.shape[0]), self.cols)

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=None, out=None):
        """The values as a tensor (float32 unless ``dtype`` or ``out`` says otherwise)."""
        import torch
        if out is None:
            out = torch.empty(self.shape, dtype=dtype or torch.float32, device=self.device)
        elif out.device != self.device:
            raise SpDNNError(-1, "out lives on another device")
        operand = _operand(out, self.shape, "out")
        with torch.cuda.device(self.device):
            _call(_lib.load().spdnn_mx4_dequantize, _data(self.codes), _data(self.scales), self.shape[0], self.cols,
                  C.byref(operand), _stream(self.device))
        return out


def _operand(t, shape, name):
    if isinstance(t, MX4):
        if t.shape != tuple(shape):
            raise SpDNNError(-1, f"{name} must be {tuple(shape)}, not {t.shape}")
        return _lib.Operand(t.codes.data_ptr(), t.scales.data_ptr(), int(t.codes.shape[1]), MX4_TYPE, 0)
    if not hasattr(t, "is_cuda") or not t.is_cuda:
        raise SpDNNError(-1, f"{name} must be a CUDA tensor")
    if tuple(t.shape) != tuple(shape):
        raise SpDNNError(-1, f"{name} must be {tuple(shape)}, not {tuple(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise SpDNNError(-1, f"{name} must have adjacent elements in a row (stride 1)")
    stride = int(t.stride(0)) if t.shape[0] > 1 else int(t.shape[1])
    return _lib.Operand(t.data_ptr(), None, stride, _type_of(t.dtype), 0)


def mx4_quantize(x) -> MX4:
    """``x`` [rows, cols] (float32, float16 or bfloat16, rows of any stride) as microscaled 4-bit floats."""
    import torch
    if not hasattr(x, "is_cuda") or x.dim() != 2 or x.shape[1] < 1:
        raise SpDNNError(-1, "x must be a matrix with at least one column")
    operand = _operand(x, x.shape, "x")
    rows, cols = int(x.shape[0]), int(x.shape[1])
    blocks = (cols + 31) // 32
    codes = torch.empty((rows, blocks, 16), dtype=torch.uint8, device=x.device)
    scales = torch.empty((rows, blocks), dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _call(_lib.load().spdnn_mx4_quantize, C.byref(operand), rows, cols, _data(codes), _data(scales), _stream(x.device))
    return MX4(codes, scales, cols)


class Saved(tuple):
    """What a forward call with ``save=True`` keeps for its backward call: one pre-activation matrix (float32) per set of weights."""


class SparseTopology:
    """The connections between ``inputs`` and ``outputs`` neurons, as CSC: output c is connected to inputs
    ``row_idx[col_ptr[c]:col_ptr[c + 1]]``.  ``device=None``: analysis only (``rows``, ``pack``), no GPU needed."""

    def __init__(self, inputs: int, outputs: int, col_ptr, row_idx, device: int | None = 0):
        self._top = C.c_void_p()
        self._lib = _lib.load()
        col_ptr = np.ascontiguousarray(col_ptr, dtype=np.int32)
        row_idx = np.ascontiguousarray(row_idx, dtype=np.int32)
        if col_ptr.shape != (outputs + 1,):
            raise SpDNNError(-1, f"col_ptr must have {outputs + 1} entries")
        if row_idx.ndim != 1 or row_idx.size != int(col_ptr[-1]):
            raise SpDNNError(-1, "row_idx size must equal col_ptr[-1]")
        self._col_ptr, self._row_idx = col_ptr, row_idx
        self.device = None if device is None else int(device)
        _call(self._lib.spdnn_topology_create, C.byref(self._top), -1 if device is None else self.device, inputs, outputs,
              C.c_void_p(col_ptr.ctypes.data), C.c_void_p(row_idx.ctypes.data))
        slots, fan_out, connections = C.c_int(), C.c_int(), C.c_int64()
        self._lib.spdnn_topology_info(self._top, None, None, C.byref(slots), C.byref(fan_out), C.byref(connections))
        self.inputs, self.outputs = int(inputs), int(outputs)
        self.slots, self.fan_out, self.connections = slots.value, fan_out.value, connections.value

    @classmethod
    def from_rows(cls, rows, inputs: int, device: int | None = 0):
        """``rows`` int [outputs, K]: the inputs of every output (entries < 0 are skipped), as ``SpDNN.set_layer_rows``."""
        rows = np.asarray(rows)
        keep = rows >= 0
        col_ptr = np.concatenate([[0], np.cumsum(keep.sum(axis=1))])
        return cls(inputs, rows.shape[0], col_ptr, rows[keep], device)

    def close(self):
        """Frees the device tables.  No call on the topology may be in flight."""
        if getattr(self, "_top", None):
            self._lib.spdnn_topology_destroy(self._top)
            self._top = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def rows(self) -> np.ndarray:
        """[outputs, slots]: the inputs of every output ascending, -1 behind the last: the canonical order of weights."""
        out = np.empty((self.outputs, self.slots), dtype=np.int32)
        if self._lib.spdnn_topology_rows(self._top, C.c_void_p(out.ctypes.data), out.size) != 0:
            raise SpDNNError(-4, "the topology is closed")
        return out

    def pack(self, val) -> np.ndarray:
        """Values in the order of the ``row_idx`` given at creation -> float32 [outputs, slots], zero where there is no connection."""
        val = np.asarray(val, dtype=np.float32).reshape(-1)
        if val.size != self._row_idx.size:
            raise SpDNNError(-1, "val size must equal row_idx size")
        count = np.diff(self._col_ptr)
        column = np.repeat(np.arange(self.outputs), count)
        order = np.lexsort((self._row_idx, column))       # stable: repeated entries keep their order
        out = np.zeros((self.outputs, self.slots), dtype=np.float32)
        out[column, np.arange(val.size) - np.repeat(self._col_ptr[:-1], count)] = val[order]
        return out

    # -- calls -----------------------------------------------------------------------
    def _prepare(self, x, weights, biases, activation):
        if not self._top:
            raise SpDNNError(-4, "the topology is closed")
        if self.device is None:
            raise SpDNNError(-4, "the topology was created for analysis only (device None)")
        if activation not in ACTIVATIONS:
            raise SpDNNError(-1, f"activation must be one of {sorted(ACTIVATIONS)}")
        if len(x.shape) != 2:
            raise SpDNNError(-1, f"x must be [tokens, {self.inputs}]")
        tokens = int(x.shape[0])
        ops = [_operand(x, (tokens, self.inputs), "x")] + [_operand(w, (self.outputs, self.slots), "weights") for w in weights]
        self._same_device(x, *weights, *biases)
        import torch
        for b in biases:
            if b is not None and (b.dtype != torch.float32 or tuple(b.shape) != (self.outputs,) or not b.is_contiguous()):
                raise SpDNNError(-1, f"a bias must be contiguous float32 [{self.outputs}]")
        return tokens, ops

    def _same_device(self, *tensors):
        for t in tensors:
            if t is not None and t.device.index != self.device:
                raise SpDNNError(-1, "a tensor lives on another device than the topology")

    def _workspace(self, tokens, sets, x_type, w_type, backward, device):
        import torch
        n = C.c_int64()
        rc = self._lib.spdnn_layer_workspace(self._top, tokens, sets, x_type, w_type, int(backward), C.byref(n))
        if rc != 0:
            raise SpDNNError(rc, "these types of activations and weights do not go together")
        return torch.empty(n.value, dtype=torch.uint8, device=device), n.value

    def _forward(self, x, weights, biases, activation, clip, save, out_dtype, out):
        import torch
        tokens, ops = self._prepare(x, weights, biases, activation)
        if out is None:
            if out_dtype is None:
                if isinstance(x, MX4):
                    raise SpDNNError(-1, "out_dtype is needed for microscaled activations")
                out_dtype = x.dtype
            out = torch.empty((tokens, self.outputs), dtype=out_dtype, device=x.device)
        self._same_device(out)
        y = _operand(out, (tokens, self.outputs), "out")
        saved = None
        if save:
            if isinstance(x, MX4):
                raise SpDNNError(-1, "microscaled activations have no backward pass: nothing to save")
            saved = Saved(torch.empty((tokens, self.outputs), dtype=torch.float32, device=x.device) for _ in weights)
        z = [_operand(s, (tokens, self.outputs), "saved") for s in saved] if save else [None] * len(weights)
        ws, size = self._workspace(tokens, len(weights), ops[0].type, ops[1].type, False, x.device)
        fn = self._lib.spdnn_gated if len(weights) == 2 else self._lib.spdnn_linear
        _call(fn, self._top, tokens, *map(_ref, ops), *map(_data, biases), ACTIVATIONS[activation], float(clip), _ref(y),
              *map(_ref, z), _data(ws), size, _stream(x.device))
        return (out, saved) if save else out

    def linear(self, x, w, bias=None, activation: str = "none", clip: float = 32.0, save: bool = False, out_dtype=None, out=None):
        """``act(x W + bias)``: x [tokens, inputs], w [outputs, slots] (of x's type, or ``MX4``), bias float32 [outputs].
        ``save``: also return what ``linear_backward`` needs."""
        return self._forward(x, [w], [bias], activation, clip, save, out_dtype, out)

    def gated(self, x, w_gate, w_up, bias_gate=None, bias_up=None, activation: str = "silu", clip: float = 32.0,
              save: bool = False, out_dtype=None, out=None):
        """``act(x Wg + bg) * (x Wu + bu)``, both projections in one pass; ``save`` as in ``linear``."""
        return self._forward(x, [w_gate, w_up], [bias_gate, bias_up], activation, clip, save, out_dtype, out)

    def _backward(self, dy, x, weights, saved, activation, clip, need_dx, need_dw):
        import torch
        tokens, ops = self._prepare(x, weights, [], activation)
        shape = (tokens, self.outputs)
        if not isinstance(saved, Saved) or len(saved) != len(weights):
            raise SpDNNError(-1, "saved must be what the forward call returned")
        self._same_device(dy, *saved)
        dy_op = _operand(dy, shape, "dy")
        z = [_operand(s, shape, "saved") for s in saved]
        dx = torch.empty((tokens, self.inputs), dtype=x.dtype, device=x.device) if need_dx else None
        dw = [torch.empty((self.outputs, self.slots), dtype=torch.float32, device=x.device) if need_dw else None for _ in weights]
        db = [torch.empty(self.outputs, dtype=torch.float32, device=x.device) if need_dw else None for _ in weights]
        dx_op = _operand(dx, (tokens, self.inputs), "dx") if need_dx else None
        ws, size = self._workspace(tokens, len(weights), ops[0].type, ops[1].type, True, x.device)
        fn = self._lib.spdnn_gated_backward if len(weights) == 2 else self._lib.spdnn_linear_backward
        _call(fn, self._top, tokens, _ref(dy_op), *map(_ref, ops), *map(_ref, z), ACTIVATIONS[activation], float(clip), _ref(dx_op),
              *map(_data, dw), *map(_data, db), _data(ws), size, _stream(x.device))
        return (dx, *dw, *db)

    def linear_backward(self, dy, x, w, saved, activation: str = "none", clip: float = 32.0, need_dx: bool = True, need_dw: bool = True):
        """Gradients ``(dx, dw, dbias)`` of ``linear(..., save=True)`` for dL/dy = ``dy`` (of x's type): dx of x's type, dw
        [outputs, slots] and dbias in float32; what is not needed is None."""
        return self._backward(dy, x, [w], saved, activation, clip, need_dx, need_dw)

    def gated_backward(self, dy, x, w_gate, w_up, saved, activation: str = "silu", clip: float = 32.0, need_dx: bool = True,
                       need_dw: bool = True):
        """Gradients ``(dx, dw_gate, dw_up, dbias_gate, dbias_up)`` of ``gated(..., save=True)``."""
        return self._backward(dy, x, [w_gate, w_up], saved, activation, clip, need_dx, need_dw)
