"""GPU tests of how the feed-forward operators are called: what they refuse, and first calls."""
import pytest

from test_gpu_feedforward import BF16, F16, F32, Problem, Shared, torch

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


def test_tensors_that_require_grad_are_refused_in_grad_mode():
    from graphchallenge21_b200 import SpDNNError, mx4_quantize
    p = Problem(7, 40, 30, 4, F32, 2)
    y, saved = p.forward("silu", save=True)
    grads = p.backward(saved, "silu")
    out = torch.empty_like(y)
    for t in (p.x, *p.w, *p.b, p.dy, out):
        t.requires_grad_()
        with pytest.raises(SpDNNError, match="requires grad"):
            p.backward(saved, "silu") if t is p.dy else p.forward("silu", out=out)
        if t is p.x:
            with pytest.raises(SpDNNError, match="requires grad"):
                mx4_quantize(t)
        with torch.no_grad():
            assert torch.equal(p.forward("silu", out=out), y) and torch.equal(p.backward(saved, "silu")[0], grads[0])
        t.requires_grad_(False)


def test_inside_an_autograd_function():
    """As a training program uses the calls: grad mode is off in both directions."""
    p = Problem(20, 40, 30, 4, F32, 2)

    class Block(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, wg, wu, bg, bu):
            y, ctx.saved = p.top.gated(x, wg, wu, bg, bu, save=True)
            ctx.save_for_backward(x, wg, wu)
            return y

        @staticmethod
        def backward(ctx, dy):
            dx, dwg, dwu, dbg, dbu = p.top.gated_backward(dy.contiguous(), *ctx.saved_tensors, ctx.saved)
            return dx, dwg, dwu, dbg, dbu

    leaves = [t.requires_grad_() for t in (p.x, *p.w, *p.b)]
    got = torch.autograd.grad((Block.apply(*leaves) * p.dy).sum(), leaves)
    for t in leaves:
        t.requires_grad_(False)
    dx, dw, db = p.backward(p.forward("silu", save=True)[1], "silu")
    assert all(torch.equal(a, b) for a, b in zip(got, [dx, *dw, *db]))


def test_results_in_tensors_of_the_caller_count_as_changes_of_them():
    """A tensor that autograd has kept for a gradient and that a call writes to is found out, as with torch's own operations."""
    from graphchallenge21_b200 import mx4_quantize
    p = Problem(7, 40, 30, 4, F32, 1)
    q = mx4_quantize(p.w[0])
    for write, shape in ((lambda t: p.forward("silu", out=t), (7, 30)), (lambda t: q.dequantize(out=t), (30, 4))):
        out = torch.ones(shape, device="cuda")
        w = torch.ones(shape, device="cuda", requires_grad=True)
        loss = (w * out).sum()
        before = out._version
        write(out)
        assert out._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        with torch.inference_mode():
            kept = torch.ones(shape, device="cuda")
            write(kept)                                    # has no version to count
        assert torch.equal(kept, out)


@pytest.mark.parametrize("shared", [False, True])
def test_fp16_gradients_of_other_sizes_in_a_replayed_graph(shared):
    """What dx is scaled by is found again in every replay, and by every stream for itself."""
    make = lambda: Shared(150, 256, 320, 32, F16, 2, 16, True) if shared else Problem(150, 256, 320, 16, F16, 2, "ragged")  # noqa: E731
    p = make()
    y, saved = p.forward("silu", save=True)
    base = p.dy.clone()
    want = {}
    for e in (0, -12, 6):
        p.dy.copy_((base.float() * 2.0 ** e).to(F16))
        want[e] = p.backward(saved, "silu")
    assert not torch.equal(want[0][0], want[6][0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = p.backward(saved, "silu")
    side = torch.cuda.Stream()
    for e in (6, -12, 0, 6):
        p.dy.copy_((base.float() * 2.0 ** e).to(F16))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = p.backward(saved, "silu")
        torch.cuda.synchronize()
        for a in (got, other):
            assert torch.equal(a[0], want[e][0]) and all(torch.equal(u, v) for u, v in zip(a[1] + a[2], want[e][1] + want[e][2]))
    del graph


@pytest.mark.parametrize("tokens", [1, 5, 64, 65, 257])
def test_fp16_gradients_leave_what_is_behind_them_alone(tokens):
    """dx and the saved pre-activations as parts of larger buffers, by the C entry point; the workspace exactly as large as asked for."""
    import ctypes as C
    from graphchallenge21_b200 import _lib
    lib, p = _lib.load(), Problem(tokens, 90, 75, 11, F16, 2)
    y, saved = p.forward("gelu", save=True)
    want = p.backward(saved, "gelu")
    n = C.c_int64()
    assert lib.spdnn_layer_workspace(p.top._top, tokens, 2, 1, 1, 1, C.byref(n)) == 0
    ws = torch.full((n.value + 512,), 0xA5, dtype=torch.uint8, device="cuda")
    assert ws.data_ptr() % 256 == 0
    z = torch.full((2, tokens + 3, 80), float("nan"), device="cuda")
    z[:, :tokens, 2:77] = saved.z
    dx = torch.full((tokens + 4, 99), 5.0, dtype=F16, device="cuda")
    o = lambda t, kind: C.byref(_lib.Operand(t.data_ptr(), None, t.stride(-2), kind, 0))  # noqa: E731
    dw = [torch.full((75 * p.top.slots + 8,), 7.0, device="cuda") for _ in range(2)]
    db = [torch.full((75 + 8,), 7.0, device="cuda") for _ in range(2)]
    err = C.create_string_buffer(256)
    torch.cuda.synchronize()
    rc = lib.spdnn_gated_backward(p.top._top, tokens, o(p.dy, 1), o(p.x, 1), o(p.w[0], 1), o(p.w[1], 1), o(z[0, :, 2:], 0), o(z[1, :, 2:], 0), 4,
                                  32.0, o(dx[:, 3:], 1), dw[0].data_ptr(), dw[1].data_ptr(), db[0].data_ptr(), db[1].data_ptr(), ws.data_ptr(),
                                  n.value, None, err, 256)
    torch.cuda.synchronize()
    assert rc == 0, err.value
    assert torch.equal(dx[:tokens, 3:93], want[0]) and (dx[:, :3] == 5).all() and (dx[:, 93:] == 5).all() and (dx[tokens:] == 5).all()
    for got, w, size in ((dw[0], want[1][0], 75 * p.top.slots), (dw[1], want[1][1], 75 * p.top.slots), (db[0], want[2][0], 75), (db[1], want[2][1], 75)):
        assert torch.equal(got[:size], w.reshape(-1)) and (got[size:] == 7).all()
    assert (ws[n.value:] == 0xA5).all()


def test_result_types_that_do_not_exist_are_refused():
    from graphchallenge21_b200 import SpDNNError
    p = Problem(7, 40, 30, 4, BF16, 1)
    for t in (torch.float64, torch.int32, torch.uint8):
        with pytest.raises(SpDNNError, match="not float32"):
            p.forward("silu", out_dtype=t)
        with pytest.raises(SpDNNError, match="not float32"):
            p.forward("silu", out=torch.empty(7, 30, dtype=t, device="cuda"))
