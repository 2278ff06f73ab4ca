"""GPU tests of how the feed-forward operators are called: what they refuse, and first calls."""
import pytest

from test_gpu_feedforward import BF16, F32, Problem, torch

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
