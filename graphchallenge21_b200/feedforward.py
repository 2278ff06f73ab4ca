"""Feed-forward operators on torch CUDA tensors, over the C ABI (include/spdnn_b200.h).

``SparseTopology`` holds which inputs every output neuron is connected to, on one GPU; its methods run the plain layer
``act(x W + b)`` and the gated block ``act(x Wg + bg) * (x Wu + bu)`` on activations ``[tokens, neurons]`` with the
weights given to each call, and their gradients.  ``mx4_quantize`` makes microscaled 4-bit matrices (``MX4``) of weights or
activations, which the forward calls take in place of tensors.

Calls enqueue on torch's current stream of the tensors' device and return at once; they may be captured into CUDA graphs.
Nothing here is differentiated by autograd: the gradients are the ``*_backward`` calls, and tensors that require grad are refused
unless grad mode is off (``torch.no_grad()``, the forward and backward of an ``autograd.Function``), as torch's own ``out=`` does.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from .network import SpDNNError

ACTIVATIONS = {"none": 0, "relu": 1, "clip": 2, "silu": 3, "gelu": 4, "gelu_tanh": 5}
F32, F16, BF16, MX4_TYPE = 0, 1, 2, 3
_ERR_LEN = 256


_TYPES = {}          # torch type -> SPDNN_F32 ..., filled with what follows when torch is first needed
_F32 = _U8 = _raw_stream = _grad_enabled = None
_byref, _Operand = C.byref, _lib.Operand


def _torch():
    import torch
    global _F32, _U8, _raw_stream, _grad_enabled
    if not _TYPES:
        _F32, _U8, _grad_enabled = torch.float32, torch.uint8, torch.is_grad_enabled
        # torch.cuda.current_stream makes an object for the handle, in twenty times the time
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
        _TYPES.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
    return torch


MAX_TOKENS, MAX_COLUMNS = 1 << 26, 1 << 30      # of one call; of a microscaled matrix: checked here, where they are not yet C ints
_Error = C.c_char * _ERR_LEN


def _call(fn, *args):
    err = _Error()
    rc = fn(*args, err, _ERR_LEN)
    if rc != 0:
        raise SpDNNError(rc, err.value.decode())


def _stream(device: int) -> int:
    """The handle of torch's current stream."""
    if not _TYPES:
        _torch()
    return _raw_stream(device)


class MX4:
    """A matrix of microscaled 4-bit floats: ``codes`` uint8 [rows, blocks, 16], ``scales`` uint8 [rows, blocks], blocks of 32
    of its ``cols`` columns (include/spdnn_b200.h says what the bytes mean)."""

    def __init__(self, codes, scales, cols: int):
        if not _TYPES:
            _torch()
        cols = int(cols)
        if cols > MAX_COLUMNS:
            raise SpDNNError(-1, f"a matrix has at most {MAX_COLUMNS} columns")
        blocks = (cols + 31) // 32
        shape = codes.shape
        if len(shape) != 3 or shape[1] != blocks or shape[2] != 16 or scales.shape != shape[:2] or cols < 1 or not (
                codes.dtype is _U8 and scales.dtype is _U8):
            raise SpDNNError(-1, f"codes must be uint8 [rows, {blocks}, 16] and scales uint8 [rows, {blocks}]")
        if not codes.is_cuda or codes.get_device() != scales.get_device() or not codes.is_contiguous() or not scales.is_contiguous():
            raise SpDNNError(-1, "codes and scales must be contiguous and on one GPU")
        self.codes, self.scales, self.cols = codes, scales, cols
        self.shape = (shape[0], cols)

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=None, out=None):
        """The values as a tensor (float32 unless ``dtype`` or ``out`` says otherwise)."""
        torch = _torch()
        device = self.codes.get_device()
        given = out
        if out is None:
            out = self.codes.new_empty(self.shape, dtype=dtype or torch.float32)
        operand = _operand(out, *self.shape, device, "out")
        _on(device, _lib.load().spdnn_mx4_dequantize, self.codes.data_ptr(), self.scales.data_ptr(), self.shape[0], self.cols,
            _byref(operand), _stream(device))
        if given is not None:
            _written(given)
        return out


def _on(device, fn, *args):
    """``_call`` with ``device`` as the current one."""
    cuda = _torch().cuda
    if cuda.current_device() == device:
        _call(fn, *args)
    else:
        with cuda.device(device):
            _call(fn, *args)


def _written(t):
    """A tensor of the caller has new values: autograd must notice if it was kept for a gradient."""
    _torch().autograd.graph.increment_version(t)


def _refuse_grad(name):
    """For a tensor that requires grad: its result would have no graph, and the gradient would be lost without a word."""
    if _grad_enabled():
        raise SpDNNError(-1, f"{name} requires grad, which these calls do not record: pass it detached, or call under torch.no_grad() and "
                             "use the backward call")


def _operand(t, rows, cols, device, name):
    """The C operand of a matrix [rows, cols] on GPU ``device`` (None: any)."""
    if isinstance(t, MX4):
        if t.shape != (rows, cols):
            raise SpDNNError(-1, f"{name} must be {(rows, cols)}, not {t.shape}")
        on, operand = t.codes.get_device(), _Operand(t.codes.data_ptr(), t.scales.data_ptr(), (cols + 31) // 32, MX4_TYPE, 0)
    else:
        if not getattr(t, "is_cuda", False):
            raise SpDNNError(-1, f"{name} must be a CUDA tensor")
        if t.shape != (rows, cols):
            raise SpDNNError(-1, f"{name} must be {(rows, cols)}, not {tuple(t.shape)}")
        if t.requires_grad:
            _refuse_grad(name)
        stride, step = t.stride()
        if step != 1 and cols > 1:
            raise SpDNNError(-1, f"{name} must have adjacent elements in a row (stride 1)")
        kind = _TYPES.get(t.dtype)
        if kind is None:
            raise SpDNNError(-1, f"{name} is {t.dtype}, not float32, float16 or bfloat16")
        on, operand = t.get_device(), _Operand(t.data_ptr(), None, stride if rows > 1 else cols, kind, 0)
    if on != device and device is not None:
        raise SpDNNError(-1, f"{name} lives on another device than the topology or matrix")
    return operand


def mx4_quantize(x) -> MX4:
    """``x`` [rows, cols] (float32, float16 or bfloat16, rows of any stride) as microscaled 4-bit floats."""
    torch = _torch()
    if not hasattr(x, "is_cuda") or x.dim() != 2 or x.shape[1] < 1:
        raise SpDNNError(-1, "x must be a matrix with at least one column")
    rows, cols = x.shape
    if cols > MAX_COLUMNS:
        raise SpDNNError(-1, f"a matrix has at most {MAX_COLUMNS} columns")
    operand = _operand(x, rows, cols, None, "x")
    blocks = (cols + 31) // 32
    codes = x.new_empty((rows, blocks, 16), dtype=torch.uint8)
    scales = x.new_empty((rows, blocks), dtype=torch.uint8)
    device = x.get_device()
    _on(device, _lib.load().spdnn_mx4_quantize, _byref(operand), rows, cols, codes.data_ptr(), scales.data_ptr(), _stream(device))
    q = MX4.__new__(MX4)                 # what __init__ would check holds
    q.codes, q.scales, q.cols, q.shape = codes, scales, cols, (rows, cols)
    return q


class Saved:
    """What a forward call with ``save=True`` keeps for its backward call: the pre-activations, float32 [sets, tokens, outputs]
    without gaps (a backward call refuses any other type or layout)."""

    def __init__(self, z):
        self.z = z

    def __len__(self):
        return self.z.shape[0]

    def __iter__(self):
        return iter(self.z)


def _whole(a, name):
    """``a`` as an array of integers; floats only where they are whole numbers."""
    a = np.asarray(a)
    if a.dtype.kind not in "iufb":
        raise SpDNNError(-1, f"{name} must hold integers")
    if a.dtype.kind == "f":
        with np.errstate(invalid="ignore"):
            whole = a.astype(np.int64)
        if not np.array_equal(whole, a):
            raise SpDNNError(-1, f"{name} must hold integers")
        return whole
    return a


def _int32(a, name):
    """``a`` as contiguous int32, refused where a value does not fit (a cast would wrap around to another index)."""
    a = _whole(a, name)
    if a.dtype != np.int32 and a.size and not (a.min() >= -(1 << 31) and a.max() < 1 << 31):
        raise SpDNNError(-1, f"{name} holds values beyond 32 bits")
    return np.ascontiguousarray(a, dtype=np.int32)


class SparseTopology:
    """The connections between ``inputs`` and ``outputs`` neurons, as CSC: output c is connected to inputs
    ``row_idx[col_ptr[c]:col_ptr[c + 1]]``.  ``slots``: columns of a weight matrix (0: as many as the output with most
    connections has).  ``device=None``: analysis only (``rows``, ``pack``), no GPU needed.  ``blocks``: how many groups of up to 16
    neurons with equal connections the tensor cores take, forward and backward (0: none, too few neurons share theirs)."""

    def __init__(self, inputs: int, outputs: int, col_ptr, row_idx, device: int | None = 0, slots: int = 0):
        self._top = C.c_void_p()
        self._lib = _lib.load()
        self._sizes = {}                 # workspaces: a function of these arguments and the topology
        col_ptr, row_idx = _int32(col_ptr, "col_ptr"), _int32(row_idx, "row_idx")
        if col_ptr.shape != (outputs + 1,):
            raise SpDNNError(-1, f"col_ptr must have {outputs + 1} entries")
        if row_idx.ndim != 1 or row_idx.size != int(col_ptr[-1]):
            raise SpDNNError(-1, "row_idx size must equal col_ptr[-1]")
        for v, name in ((inputs, "inputs"), (outputs, "outputs"), (slots, "slots"), (-1 if device is None else device, "device")):
            if not -(1 << 31) <= v < 1 << 31:
                raise SpDNNError(-1, f"{name} is out of range")
        self._col_ptr, self._row_idx = col_ptr, row_idx
        self.device = None if device is None else int(device)
        _call(self._lib.spdnn_topology_create, C.byref(self._top), -1 if device is None else self.device, inputs, outputs, slots,
              C.c_void_p(col_ptr.ctypes.data), C.c_void_p(row_idx.ctypes.data))
        slots, fan_out, connections = C.c_int(), C.c_int(), C.c_int64()
        self._lib.spdnn_topology_info(self._top, None, None, C.byref(slots), C.byref(fan_out), C.byref(connections))
        forward, backward = C.c_int(), C.c_int()
        self._lib.spdnn_topology_blocks(self._top, C.byref(forward), C.byref(backward))
        self.blocks = forward.value, backward.value
        self.inputs, self.outputs = int(inputs), int(outputs)
        self.slots, self.fan_out, self.connections = slots.value, fan_out.value, connections.value

    @classmethod
    def from_rows(cls, rows, inputs: int, device: int | None = 0):
        """``rows`` int [outputs, K]: the inputs of every output (entries < 0 are skipped), as ``SpDNN.set_layer_rows``; weight
        matrices are [outputs, K]."""
        rows = _whole(rows, "rows")
        if rows.ndim != 2:
            raise SpDNNError(-1, "rows must be a matrix [outputs, connections]")
        if rows.size and rows.min() >= 0:
            return cls(inputs, rows.shape[0], np.arange(rows.shape[0] + 1, dtype=np.int64) * rows.shape[1], rows.reshape(-1), device,
                       rows.shape[1])
        keep = rows >= 0
        col_ptr = np.concatenate([[0], np.cumsum(keep.sum(axis=1))])
        return cls(inputs, rows.shape[0], col_ptr, rows[keep], device, rows.shape[1])

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
    def _begin(self, x, weights, activation):
        """(tokens, the activation's number, operands of x and the weights, their types) of a call."""
        if self.device is None or not self._top:
            raise SpDNNError(-4, "the topology was created for analysis only (device None)" if self._top else "the topology is closed")
        kind = ACTIVATIONS.get(activation)
        if kind is None:
            raise SpDNNError(-1, f"activation must be one of {sorted(ACTIVATIONS)}")
        if not _TYPES:
            _torch()
        if len(x.shape) != 2:
            raise SpDNNError(-1, f"x must be [tokens, {self.inputs}]")
        tokens, device = x.shape[0], self.device
        if tokens > MAX_TOKENS:
            raise SpDNNError(-1, f"at most {MAX_TOKENS} tokens a call")
        xo = _operand(x, tokens, self.inputs, device, "x")
        ops = [xo]
        for w in weights:
            ops.append(_operand(w, self.outputs, self.slots, device, "weights"))
        return tokens, kind, [_byref(o) for o in ops], xo.type, ops[1].type

    def _bias(self, b):
        if b is None:
            return None
        if b.dtype is not _F32 or b.get_device() != self.device or b.shape != (self.outputs,) or not b.is_contiguous():
            raise SpDNNError(-1, f"a bias must be contiguous float32 [{self.outputs}] on the topology's device")
        if b.requires_grad:
            _refuse_grad("a bias")
        return b.data_ptr()

    def _workspace(self, x, *key):
        """(pointer, bytes, what keeps it alive) of a call's workspace; ``key``: tokens, sets, types of x and w, backward."""
        size = self._sizes.get(key)
        if size is None:
            n = C.c_int64()
            rc = self._lib.spdnn_layer_workspace(self._top, *key, _byref(n))
            if rc != 0:
                raise SpDNNError(rc, "these types of activations and weights do not go together")
            if len(self._sizes) > 4096:
                self._sizes.clear()
            size = self._sizes[key] = n.value
        if not size:
            return None, 0, None
        ws = x.new_empty(size, dtype=_U8)
        return ws.data_ptr(), size, ws

    def _pre_activations(self, saved, sets, tokens):
        """The tensor of ``saved``, which the kernels read as float32 without gaps."""
        z = getattr(saved, "z", None)
        if z is None or z.shape != (sets, tokens, self.outputs) or z.get_device() != self.device:
            raise SpDNNError(-1, "saved must be what the forward call returned")
        if z.dtype is not _F32 or not z.is_contiguous():
            raise SpDNNError(-1, "saved pre-activations must be contiguous float32, as the forward call returned them")
        return z

    def _saved_operands(self, z, tokens):
        at, step = z.data_ptr(), tokens * self.outputs * 4
        return [_byref(_Operand(at + s * step, None, self.outputs, F32, 0)) for s in range(z.shape[0])]

    def _forward(self, fn, x, weights, biases, activation, clip, save, out_dtype, out):
        tokens, kind, refs, x_type, w_type = self._begin(x, weights, activation)
        refs += [self._bias(b) for b in biases]
        like = x.codes if x_type == MX4_TYPE else x
        given = out
        if out is None:
            if out_dtype is None and like is not x:
                raise SpDNNError(-1, "out_dtype is needed for microscaled activations")
            out = like.new_empty((tokens, self.outputs), dtype=out_dtype)
            y_type = x_type if out_dtype is None else _TYPES.get(out_dtype)
            if y_type is None:
                raise SpDNNError(-1, f"out is {out_dtype}, not float32, float16 or bfloat16")
            y = _Operand(out.data_ptr(), None, self.outputs, y_type, 0)
        else:
            y = _operand(out, tokens, self.outputs, self.device, "out")
        if save:
            if like is not x:
                raise SpDNNError(-1, "microscaled activations have no backward pass: nothing to save")
            saved = Saved(x.new_empty((len(weights), tokens, self.outputs), dtype=_F32))
            z = self._saved_operands(saved.z, tokens)
        else:
            z = (None,) * len(weights)
        ws, size, keep = self._workspace(like, tokens, len(weights), x_type, w_type, 0)
        _call(fn, self._top, tokens, *refs, kind, clip, _byref(y), *z, ws, size, _stream(self.device))
        if given is not None:
            _written(given)
        return (out, saved) if save else out

    def linear(self, x, w, bias=None, activation: str = "none", clip: float = 32.0, save: bool = False, out_dtype=None, out=None):
        """``act(x W + bias)``: x [tokens, inputs], w [outputs, slots] (of x's type, or ``MX4``), bias float32 [outputs].
        ``save``: also return what ``linear_backward`` needs."""
        return self._forward(self._lib.spdnn_linear, x, [w], [bias], activation, clip, save, out_dtype, out)

    def gated(self, x, w_gate, w_up, bias_gate=None, bias_up=None, activation: str = "silu", clip: float = 32.0,
              save: bool = False, out_dtype=None, out=None):
        """``act(x Wg + bg) * (x Wu + bu)``, both projections in one pass; ``save`` as in ``linear``."""
        return self._forward(self._lib.spdnn_gated, x, [w_gate, w_up], [bias_gate, bias_up], activation, clip, save, out_dtype, out)

    def _backward(self, fn, dy, x, weights, saved, activation, clip, need_dx, need_dw):
        tokens, kind, refs, x_type, w_type = self._begin(x, weights, activation)
        if x_type == MX4_TYPE:
            raise SpDNNError(-1, "microscaled activations have no backward pass")
        z = self._pre_activations(saved, len(weights), tokens)
        dy_ref = _byref(_operand(dy, tokens, self.outputs, self.device, "dy"))
        dx = dx_ref = None
        if need_dx:
            dx = x.new_empty((tokens, self.inputs))
            dx_ref = _byref(_Operand(dx.data_ptr(), None, self.inputs, x_type, 0))
        grads = pointers = (None,) * (2 * len(weights))
        if need_dw:
            grads = [x.new_empty((self.outputs, self.slots), dtype=_F32) for _ in weights] + [x.new_empty(self.outputs, dtype=_F32) for _ in weights]
            pointers = [t.data_ptr() for t in grads]
        ws, size, keep = self._workspace(x, tokens, len(weights), x_type, w_type, 1)
        _call(fn, self._top, tokens, dy_ref, *refs, *self._saved_operands(z, tokens), kind, clip, dx_ref, *pointers, ws, size,
              _stream(self.device))
        return (dx, *grads)

    def linear_backward(self, dy, x, w, saved, activation: str = "none", clip: float = 32.0, need_dx: bool = True, need_dw: bool = True):
        """Gradients ``(dx, dw, dbias)`` of ``linear(..., save=True)`` for dL/dy = ``dy`` (of x's type): dx of x's type, dw
        [outputs, slots] and dbias in float32; what is not needed is None."""
        return self._backward(self._lib.spdnn_linear_backward, dy, x, [w], saved, activation, clip, need_dx, need_dw)

    def gated_backward(self, dy, x, w_gate, w_up, saved, activation: str = "silu", clip: float = 32.0, need_dx: bool = True,
                       need_dw: bool = True):
        """Gradients ``(dx, dw_gate, dw_up, dbias_gate, dbias_up)`` of ``gated(..., save=True)``."""
        return self._backward(self._lib.spdnn_gated_backward, dy, x, [w_gate, w_up], saved, activation, clip, need_dx, need_dw)
