"""GPU tests of the feed-forward operators against 64-bit plain forms (tests/feedforward_reference.py), within bounds that count
roundings."""
import numpy as np
import pytest

import feedforward_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def topology_rows(inputs, outputs, slots, net, seed=0):
    """[outputs, slots]: random; ragged (a third missing, one neuron without connections); hub (input 0 feeds every output)."""
    rng = np.random.default_rng(seed)
    if slots > inputs:
        raise ValueError("slots > inputs")
    if inputs > 4 * slots:
        rows = np.sort(rng.integers(0, inputs - slots + 1, (outputs, slots)), axis=1) + np.arange(slots)
    else:
        rows = np.sort(np.argsort(rng.random((outputs, inputs)), axis=1)[:, :slots], axis=1)
    if net == "ragged":
        rows = np.where(rng.random(rows.shape) < 1 / 3, -1, rows)
        rows[outputs // 2] = -1
    if net == "hub":
        rows[:, 0] = 0
    return rows


class Problem:
    def __init__(self, tokens, inputs, outputs, slots, dtype, sets, net="random", seed=0, bias=True):
        from graphchallenge21_b200 import SparseTopology
        self.rows_given = topology_rows(inputs, outputs, slots, net, seed)
        self.top = SparseTopology.from_rows(self.rows_given, inputs)
        self.rows = self.top.rows()
        g = torch.Generator("cuda").manual_seed(seed + 1)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.x = rand(tokens, inputs).to(dtype)
        self.w = [(rand(outputs, self.top.slots) / slots ** 0.5).to(dtype) for _ in range(sets)]
        self.b = [0.3 * rand(outputs) if bias else None for _ in range(sets)]
        self.dy = rand(tokens, outputs).to(dtype)
        self.inputs, self.sets = inputs, sets

    def forward(self, kind, **kw):
        x, w = kw.pop("x", self.x), kw.pop("w", self.w)
        if self.sets == 2:
            return self.top.gated(x, w[0], w[1], self.b[0], self.b[1], activation=kind, **kw)
        return self.top.linear(x, w[0], self.b[0], activation=kind, **kw)

    def backward(self, saved, kind, **kw):
        if self.sets == 2:
            dx, d0, d1, b0, b1 = self.top.gated_backward(self.dy, self.x, *self.w, saved, activation=kind, **kw)
            return dx, [d0, d1], [b0, b1]
        dx, d0, b0 = self.top.linear_backward(self.dy, self.x, self.w[0], saved, activation=kind, **kw)
        return dx, [d0], [b0]

    def reference(self, kind, **kw):
        return ref.Forward(self.rows, self.inputs, kw.pop("x", self.x), kw.pop("w", self.w), self.b, kind, **kw)


def check(got, want, bound, what):
    ok, worst = ref.within(got, want, bound)
    assert ok, f"{what}: {worst:.3g} times its bound"


def check_step(p, kind):
    y, saved = p.forward(kind, save=True)
    f = p.reference(kind)
    check(y, f.y, f.bound, "y")
    for s, z, e in zip(saved, f.z, f.dz):
        check(s, z, e + ref.U * z.abs(), "z")
    dx, dw, db = p.backward(saved, kind)
    (wdx, bdx), wdw, wdb = ref.backward(f, p.dy)
    check(dx, wdx, bdx, "dx")
    for s in range(p.sets):
        check(dw[s], *wdw[s], f"dw[{s}]")
        check(db[s], *wdb[s], f"db[{s}]")


# token counts around every width of an image (1, 2, 4, 8, 16, 32, 64 tokens) and of the packing blocks
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9, 17, 31, 33, 64, 65, 130, 257])
def test_gated_step_over_token_counts(tokens, dtype):
    check_step(Problem(tokens, 100, 70, 9, dtype, 2, seed=tokens), "silu")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens, inputs, outputs, slots, net", [
    (7, 1, 1, 1, "random"), (70, 1, 40, 1, "random"), (70, 300, 1, 300, "random"), (33, 65, 129, 37, "ragged"),
    (20, 513, 257, 32, "hub"), (40, 64, 2000, 5, "ragged"), (40, 2000, 64, 5, "ragged"), (3, 31, 33, 31, "random"),
])
@pytest.mark.parametrize("sets", [1, 2])
def test_steps_over_shapes(tokens, inputs, outputs, slots, net, sets, dtype):
    check_step(Problem(tokens, inputs, outputs, slots, dtype, sets, net), "gelu")


@pytest.mark.parametrize("kind", ["none", "relu", "clip", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("sets", [1, 2])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_activations(kind, sets, dtype):
    check_step(Problem(50, 200, 150, 16, dtype, sets, "ragged"), kind)


# images of 4, 2 and 1 tokens (many neurons), and neurons that do not fit on an SM at all
@pytest.mark.parametrize("dtype, inputs", [(BF16, 20000), (F16, 40000), (BF16, 70000), (F16, 120000), (F32, 20000), (F32, 40000), (F32, 60000)])
@pytest.mark.parametrize("tokens", [1, 21])
def test_many_neurons(dtype, inputs, tokens):
    check_step(Problem(tokens, inputs, 90, 32, dtype, 2), "silu")
    check_step(Problem(tokens, 90, inputs, 8, dtype, 2), "silu")


def test_no_tokens_and_no_bias():
    p = Problem(0, 40, 30, 4, BF16, 2)
    y, saved = p.forward("silu", save=True)
    dx, dw, db = p.backward(saved, "silu")
    assert y.shape == (0, 30) and dx.shape == (0, 40)
    assert all((t == 0).all() for t in dw + db)
    p = Problem(6, 40, 30, 4, F32, 2, bias=False)
    check_step(p, "gelu_tanh")


def test_repeated_connections_count_twice():
    from graphchallenge21_b200 import SparseTopology
    rows = np.array([[3, 3, 1], [0, 0, 0]])
    top = SparseTopology.from_rows(rows, 5)
    x = torch.arange(10, dtype=F32, device="cuda").view(2, 5)
    w = torch.tensor([[1.0, 10.0, 100.0], [1.0, 2.0, 4.0]], device="cuda")
    y, saved = top.linear(x, w, save=True)
    assert y.tolist() == [[331.0, 0.0], [886.0, 35.0]]
    dx, dw, db = top.linear_backward(torch.ones_like(y), x, w, saved)
    assert dx.tolist() == [[7.0, 1.0, 0.0, 110.0, 0.0]] * 2
    assert dw.tolist() == [[7.0, 11.0, 11.0], [5.0, 5.0, 5.0]] and db.tolist() == [2.0, 2.0]


def test_weights_without_connection_and_infinities():
    """What a weight matrix holds where there is no connection is never read; an infinity or NaN of an activation reaches the
    outputs that are connected to it, and no others."""
    p = Problem(9, 50, 40, 6, BF16, 1, "ragged")
    want = p.forward("none")
    hole = torch.as_tensor(p.rows < 0).cuda()
    p.w[0] = p.w[0].masked_fill(hole, float("nan"))
    y, saved = p.forward("none", save=True)
    assert torch.equal(y, want)
    dx, dw, _ = p.backward(saved, "none")
    assert torch.isfinite(dx).all() and (dw[0][hole] == 0).all()
    p.x[4, 7] = float("inf")
    p.x[5, 9] = float("nan")
    y = p.forward("none")
    touched = torch.zeros_like(y, dtype=torch.bool)
    touched[4] = torch.as_tensor((p.rows == 7).any(1)).cuda()
    touched[5] = torch.as_tensor((p.rows == 9).any(1)).cuda()
    assert touched.any() and not torch.isfinite(y[touched]).any() and torch.equal(y[~touched], want[~touched])
    assert torch.isnan(p.forward("relu")[5][touched[5]]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_strides_and_alignment(dtype):
    p = Problem(37, 90, 75, 11, dtype, 2)
    want, saved = p.forward("silu", save=True)
    gx, gw, gb = p.backward(saved, "silu")
    odd = lambda t, at, extra: torch.full((t.shape[0], t.shape[1] + extra), 7.0, dtype=t.dtype, device="cuda")[:, at:at + t.shape[1]].copy_(t)  # noqa: E731
    q = Problem(37, 90, 75, 11, dtype, 2)
    q.x, q.w, q.dy = odd(p.x, 3, 5), [odd(w, 1, 2) for w in p.w], odd(p.dy, 5, 9)
    out = torch.full((37, 80), 5.0, dtype=dtype, device="cuda")
    y, saved2 = q.forward("silu", save=True, out=out[:, 3:78])
    assert torch.equal(y, want) and (out[:, :3] == 5).all() and (out[:, 78:] == 5).all()
    hx, hw, hb = q.backward(saved2, "silu")
    assert torch.equal(hx, gx) and all(torch.equal(a, b) for a, b in zip(gw + gb, hw + hb))


def test_outputs_of_other_types():
    p = Problem(20, 60, 50, 8, BF16, 2)
    for t in (F32, F16, BF16):
        f = p.reference("silu", out_dtype=t)
        y = p.forward("silu", out_dtype=t)
        assert y.dtype == t
        check(y, f.y, f.bound, f"y in {t}")


def test_gradients_against_differences():
    """Central differences of the operator's own forward pass in float32: sum(y * dy) as a function of one operand."""
    p = Problem(12, 30, 25, 5, F32, 2)
    y, saved = p.forward("gelu", save=True)
    dx, dw, db = p.backward(saved, "gelu")
    g = torch.Generator("cuda").manual_seed(9)
    loss = lambda: float((p.forward("gelu").double() * p.dy.double()).sum())  # noqa: E731
    hole = torch.as_tensor(p.rows < 0).cuda()
    h = 2.0 ** -6
    for t, grad in [(p.x, dx), (p.w[0], dw[0]), (p.w[1], dw[1]), (p.b[0], db[0]), (p.b[1], db[1])]:
        step = torch.randn(t.shape, device="cuda", generator=g)
        if t.shape == hole.shape:
            step = step.masked_fill(hole, 0.0)
        was = t.clone()
        t.copy_(was + h * step); up = loss()
        t.copy_(was - h * step); down = loss()
        t.copy_(was + 2 * h * step); up2 = loss()
        t.copy_(was - 2 * h * step); down2 = loss()
        t.copy_(was)
        # fourth order: (8 (f(h) - f(-h)) - (f(2h) - f(-2h))) / 12 h; what remains is h^4 f'''''/30 and the roundings of f
        slope = (8 * (up - down) - (up2 - down2)) / (12 * h)
        want = float((grad.double() * step.double()).sum())
        # f is a sum of 300 terms of order 1 along a direction of length up to 19: its fifth derivative along it is of order
        # 300 * 3^5 / 30 h^4 < 2e-4 of |f'| ~ 30; roundings 300 * 2^-22 / h < 0.005
        assert abs(slope - want) < 0.02 + 1e-3 * abs(want), (slope, want)


def test_same_call_same_bits():
    p = Problem(333, 700, 900, 32, BF16, 2, "ragged")
    y, saved = p.forward("silu", save=True)
    a = p.backward(saved, "silu")
    b = p.backward(saved, "silu")
    assert torch.equal(y, p.forward("silu"))
    assert torch.equal(a[0], b[0]) and all(torch.equal(u, v) for u, v in zip(a[1] + a[2], b[1] + b[2]))
    only_x = p.backward(saved, "silu", need_dw=False)
    only_w = p.backward(saved, "silu", need_dx=False)
    assert torch.equal(only_x[0], a[0]) and only_x[1] == [None, None] and only_w[0] is None
    assert all(torch.equal(u, v) for u, v in zip(a[1] + a[2], only_w[1] + only_w[2]))


# ---- microscaled 4-bit floats -----------------------------------------------------------------

def mx4_input(rows, cols, dtype, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    v = torch.randn(rows, cols, device="cuda", generator=g) * torch.exp2(3 * torch.randn(rows, 1, device="cuda", generator=g))
    if rows > 3:
        v[1] = 0
        v[2] = torch.round(v[2] * 4) / 4                  # ties
        v[3] = torch.exp2(torch.floor(torch.log2(v[3].abs() + 1e-3)))
    return v.to(dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows, cols", [(1, 1), (5, 31), (5, 32), (7, 33), (4, 100), (300, 64), (33, 1000), (2, 4099)])
def test_quantize(rows, cols, dtype):
    from graphchallenge21_b200 import mx4_quantize
    x = mx4_input(rows, cols, dtype, rows * 31 + cols)
    codes, scales, values = ref.mx4_reference(x.double().cpu().numpy())
    q = mx4_quantize(x)
    assert np.array_equal(q.scales.cpu().numpy(), scales) and np.array_equal(q.codes.cpu().numpy(), codes)
    assert np.array_equal(q.dequantize().cpu().numpy(), values.astype(np.float32))
    wide = torch.full((rows, cols + 3), 1e4 if dtype == F16 else 1e9, device="cuda").to(dtype)
    wide[:, 2:2 + cols] = x
    r = mx4_quantize(wide[:, 2:2 + cols])
    assert torch.equal(r.codes, q.codes) and torch.equal(r.scales, q.scales)


def test_quantize_extremes():
    from graphchallenge21_b200 import MX4, mx4_quantize
    x = torch.zeros(8, 64, device="cuda")
    x[0, 3], x[0, 40] = float("inf"), 1.0
    x[1, 5], x[1, 33] = float("nan"), -0.0
    x[2, 0], x[2, 32] = 3.4e38, -3.4e38
    x[3, :8] = torch.tensor([2.0 ** -149, 2.0 ** -126, 2.0 ** -127, 1.5 * 2.0 ** -126, -2.0 ** -128, 2.0 ** -130, 0.0, -0.0])
    x[4, :3] = torch.tensor([2.0 ** -149, -2.0 ** -140, 0.0])
    x[5, :2] = torch.tensor([2.0 ** -125, 2.0 ** -129])
    x[6, :2] = torch.tensor([2.0 ** -124, 7.0 * 2.0 ** -127])
    codes, scales, values = ref.mx4_reference(x.double().cpu().numpy())
    q = mx4_quantize(x)
    assert np.array_equal(q.scales.cpu().numpy(), scales) and np.array_equal(q.codes.cpu().numpy(), codes)
    assert np.array_equal(q.dequantize().cpu().numpy(), values.astype(np.float32), equal_nan=True)
    # every code at every scale, and into the 16-bit types
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")[:, None, None].expand(256, 1, 16).contiguous()
    for s in (0, 1, 100, 127, 140, 252, 255):
        m = MX4(codes, torch.full((256, 1), s, dtype=torch.uint8, device="cuda"), 32)
        c = np.stack([np.arange(256) & 15, np.arange(256) >> 4], 1)
        want = ref.E2M1[c & 7] * np.where(c >= 8, -1, 1) * (2.0 ** (s - 127.0) if s < 255 else np.nan)
        got = m.dequantize()[:, :2].cpu().double().numpy()
        assert np.array_equal(got, want, equal_nan=True)
        for t in (F16, BF16):
            assert torch.equal(m.dequantize(t).nan_to_num(9.0), m.dequantize().to(t).nan_to_num(9.0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("sets", [1, 2])
@pytest.mark.parametrize("tokens, inputs, outputs, slots, net", [(1, 500, 300, 32, "random"), (3, 90, 70, 37, "ragged"), (70, 257, 129, 64, "random"),
                                                                  (130, 1000, 65, 20, "ragged"), (9, 70000, 60, 33, "random")])
def test_product_with_microscaled_weights(tokens, inputs, outputs, slots, net, sets, dtype):
    from graphchallenge21_b200 import mx4_quantize
    p = Problem(tokens, inputs, outputs, slots, dtype, sets, net)
    q = [mx4_quantize(w) for w in p.w]
    f = p.reference("silu", w=[m.dequantize() for m in q])
    check(p.forward("silu", w=q), f.y, f.bound, "y")
    # microscaled activations too: their values are exact in the image
    x4 = mx4_quantize(p.x)
    for t in (F32, BF16):
        f = p.reference("silu", x=x4.dequantize(), w=[m.dequantize() for m in q], out_dtype=t)
        y = p.forward("silu", x=x4, w=q, out_dtype=t)
        assert y.dtype == t
        check(y, f.y, f.bound, f"y of microscaled activations in {t}")


def test_product_at_extreme_scales():
    """Weights far below what fp16 holds keep their values beside fp16 activations."""
    from graphchallenge21_b200 import mx4_quantize
    p = Problem(20, 60, 50, 32, F16, 1, bias=False)
    w = (p.w[0].float() * 2.0 ** -40)
    q = mx4_quantize(w)
    f = p.reference("none", w=[q.dequantize()], out_dtype=F32)
    check(p.forward("none", w=[q], out_dtype=F32), f.y, f.bound, "y")


# ---- as they are used ---------------------------------------------------------------------------

def test_a_feedforward_block_is_trained_and_served():
    """Gated block, down projection, gradients through both, a step of descent; then both layers' weights to 4 bits and the
    same block served from them, token by token and all at once."""
    from graphchallenge21_b200 import SparseTopology, mx4_quantize
    d, hidden, tokens = 128, 320, 77
    up = SparseTopology.from_rows(topology_rows(d, hidden, 16, "random", 1), d)
    down = SparseTopology.from_rows(topology_rows(hidden, d, 32, "ragged", 2), hidden)
    g = torch.Generator("cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    wg, wu, wd = rand(hidden, 16) / 4, rand(hidden, 16) / 4, rand(d, down.slots) / 5
    bg, bd = 0.1 * rand(hidden), 0.1 * rand(d)
    x, dy = rand(tokens, d), rand(tokens, d)
    h, s1 = up.gated(x, wg, wu, bg, None, save=True)
    y, s2 = down.linear(h, wd, bd, save=True)
    dh, dwd, dbd = down.linear_backward(dy, h, wd, s2)
    dx, dwg, dwu, dbg, dbu = up.gated_backward(dh, x, wg, wu, s1)
    # the same in 64 bits by autograd over dense matrices
    leaves = [t.double().requires_grad_() for t in (x, wg, wu, wd, bg, bd)]
    X, Wg, Wu, Wd, Bg, Bd = leaves
    def mat(rows, w, n):
        rows = torch.as_tensor(rows).cuda().long()
        keep = rows >= 0
        out = torch.arange(rows.shape[0], device="cuda")[:, None].expand_as(rows)[keep]
        return torch.zeros(n, rows.shape[0], dtype=torch.float64, device="cuda").index_put((rows[keep], out), w[keep], accumulate=True)
    gate = X @ mat(up.rows(), Wg, d) + Bg
    H = gate * torch.sigmoid(gate) * (X @ mat(up.rows(), Wu, d))
    Y = H @ mat(down.rows(), Wd, hidden) + Bd
    want = torch.autograd.grad((Y * dy.double()).sum(), leaves)
    # float32 throughout: sums of at most 77 terms twice over, so a few hundred half steps of the largest element
    for got, exact in [(y, Y.detach()), *zip((dx, dwg, dwu, dwd, dbg, dbd), want)]:
        assert float((got.double() - exact).abs().max()) <= 400 * ref.U * float(exact.abs().max())
    for w, grad in ((wg, dwg), (wu, dwu), (wd, dwd)):
        w -= 0.01 * grad
    qg, qu, qd = (mx4_quantize(w) for w in (wg, wu, wd))
    xb = x.bfloat16()
    serve = lambda t: down.linear(up.gated(t, qg, qu, bg), qd, bd)  # noqa: E731
    whole = serve(xb)
    f = ref.Forward(up.rows(), d, xb, [qg.dequantize(), qu.dequantize()], [bg, None], "silu")
    hb = up.gated(xb, qg, qu, bg)
    check(hb, f.y, f.bound, "hidden")
    f = ref.Forward(down.rows(), hidden, hb, [qd.dequantize()], [bd], "none")
    check(whole, f.y, f.bound, "served")
    for t in (0, 40, 76):
        one = serve(xb[t:t + 1])
        h1 = up.gated(xb[t:t + 1], qg, qu, bg)
        f = ref.Forward(down.rows(), hidden, h1, [qd.dequantize()], [bd], "none")
        check(one, f.y, f.bound, "one token")


def test_captured_and_replayed():
    p = Problem(40, 300, 200, 16, BF16, 2)
    y, saved = p.forward("silu", save=True)
    grads = p.backward(saved, "silu")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y2, saved2 = p.forward("silu", save=True)
        grads2 = p.backward(saved2, "silu")
    x = p.x.clone()
    p.x.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(y2, y)
    p.x.copy_(x)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y2, y) and torch.equal(grads2[0], grads[0])
    assert all(torch.equal(a, b) for a, b in zip(grads[1] + grads[2], grads2[1] + grads2[2]))
    del graph


def test_two_streams_and_two_threads_at_once():
    import threading
    problems = [Problem(500, 400, 300, 24, BF16, 2, seed=s) for s in (1, 1)]
    problems[1].top = problems[0].top                      # one topology, two callers
    problems[1].x = problems[1].x * 0.5
    want = [p.forward("silu").clone() for p in problems]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i].append(problems[i].forward("silu"))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                             # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for i in (0, 1):
        assert len(got[i]) == 20 and all(torch.equal(y, want[i]) for y in got[i])


def test_refusals_on_the_gpu():
    from graphchallenge21_b200 import MX4, SparseTopology, SpDNNError, mx4_quantize
    p = Problem(5, 40, 30, 4, BF16, 2)
    top, (w0, w1), x = p.top, p.w, p.x
    y, saved = p.forward("silu", save=True)
    for call, says in [
        (lambda: top.gated(x.float(), w0, w1), "go together"),
        (lambda: top.gated(x[:, :39], w0, w1), "must be"),
        (lambda: top.gated(x, w0, w1[:, :3]), "must be"),
        (lambda: top.gated(x, w0, w1.float()), "one type"),
        (lambda: top.gated(x.double(), w0, w1), "not float32"),
        (lambda: top.gated(x.t().contiguous().t(), w0, w1), "stride 1"),
        (lambda: top.gated(x[0], w0, w1), "tokens"),
        (lambda: top.gated(x, w0, w1, activation="tanh"), "activation must be"),
        (lambda: top.gated(x, w0, w1, p.b[0].double()), "bias"),
        (lambda: top.gated(x.cpu(), w0, w1), "CUDA"),
        (lambda: top.gated(x, w0, w1, out=torch.empty(5, 31, device="cuda")), "must be"),
        (lambda: top.gated(mx4_quantize(x), w0.half(), w1.half(), out_dtype=BF16), "go together"),
        (lambda: top.gated(mx4_quantize(x), mx4_quantize(w0), mx4_quantize(w1)), "out_dtype"),
        (lambda: top.gated(mx4_quantize(x), mx4_quantize(w0), mx4_quantize(w1), save=True, out_dtype=BF16), "nothing to save"),
        (lambda: top.gated_backward(p.dy, x, w0, w1, None), "saved"),
        (lambda: top.gated_backward(p.dy.float(), x, w0, w1, saved), "dy must have"),
        (lambda: top.gated_backward(p.dy, x, mx4_quantize(w0), mx4_quantize(w1), saved), "go together"),
        (lambda: top.linear_backward(p.dy, x, w0, saved), "saved"),
    ]:
        with pytest.raises(SpDNNError, match=says):
            call()
    with pytest.raises(SpDNNError):
        SparseTopology.from_rows(p.rows, 40, device=99)
    codes = torch.zeros(30, 1, 16, dtype=torch.uint8, device="cuda")
    with pytest.raises(SpDNNError, match="codes must be"):
        MX4(codes, torch.zeros(30, 2, dtype=torch.uint8, device="cuda"), 4)
    # the calls before left nothing behind
    assert torch.equal(p.forward("silu"), y)


def test_a_workspace_that_is_too_small_is_refused():
    import ctypes as C
    from graphchallenge21_b200 import _lib
    p = Problem(300, 40, 30, 4, F32, 1)
    lib = _lib.load()
    n = C.c_int64()
    assert lib.spdnn_layer_workspace(p.top._top, 1, 1, 0, 0, 0, C.byref(n)) == 0 and n.value == 0      # one token needs none
    assert lib.spdnn_layer_workspace(p.top._top, 300, 1, 0, 0, 0, C.byref(n)) == 0 and n.value > 0
    ws = torch.empty(n.value + 256, dtype=torch.uint8, device="cuda")
    y = torch.empty(300, 30, device="cuda")
    o = lambda t: C.byref(_lib.Operand(t.data_ptr(), None, t.stride(0), 0, 0))  # noqa: E731
    err = C.create_string_buffer(256)
    call = lambda at, size: lib.spdnn_linear(p.top._top, 300, o(p.x), o(p.w[0]), None, 0, 32.0, o(y), None, ws.data_ptr() + at, size, None,  # noqa: E731
                                             err, 256)
    assert call(0, n.value - 1) == -1 and b"workspace" in err.value
    assert call(16, n.value) == -1 and b"aligned" in err.value
    assert call(0, n.value) == 0
    torch.cuda.synchronize()


# ---- neurons that share their inputs -------------------------------------------------------------

def shared_rows(inputs, outputs, slots, group, scattered, seed=0):
    """[outputs, slots]: groups of `group` outputs read the same inputs, every input is read by whole groups of inputs too where the
    sizes allow it (a butterfly); scattered: both sides renumbered at random.  One group reads nothing."""
    rng = np.random.default_rng(seed)
    groups = (outputs + group - 1) // group
    base = np.stack([np.sort(rng.permutation(inputs // group)[: (slots + group - 1) // group]) for _ in range(groups)])
    rows = (base[:, :, None] * group + np.arange(group)).reshape(groups, -1)[:, :slots]
    rows[groups // 2] = -1
    rows = np.repeat(rows, group, axis=0)[:outputs]
    if scattered:
        renumber = rng.permutation(inputs)
        rows = np.where(rows < 0, -1, renumber[rows])
        rows = rows[rng.permutation(outputs)]
    return rows


class Shared(Problem):
    def __init__(self, tokens, inputs, outputs, slots, dtype, sets, group, scattered, seed=0):
        from graphchallenge21_b200 import SparseTopology
        super().__init__(tokens, inputs, outputs, slots, dtype, sets)
        self.top = SparseTopology.from_rows(shared_rows(inputs, outputs, slots, group, scattered, seed), inputs)
        self.rows = self.top.rows()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("sets", [1, 2])
@pytest.mark.parametrize("tokens, inputs, outputs, slots, group, scattered", [
    (17, 256, 320, 32, 16, False), (64, 256, 320, 32, 16, True), (65, 512, 100, 48, 16, False), (200, 128, 96, 20, 10, True),
    (130, 1024, 1024, 32, 16, True), (77, 300, 333, 45, 15, False), (64, 64, 33, 32, 32, False), (31, 96, 1600, 8, 8, False),
    (130, 360, 350, 30, 12, True), (18, 640, 77, 64, 16, True),
])
def test_steps_of_neurons_that_share_their_inputs(tokens, inputs, outputs, slots, group, scattered, sets, dtype):
    check_step(Shared(tokens, inputs, outputs, slots, dtype, sets, group, scattered), "gelu")


def test_the_challenge_networks_butterfly():
    from graphchallenge21_b200 import SparseTopology, mx4_quantize
    from graphchallenge21_b200.generator import SyntheticNetwork
    p = Problem(150, 1024, 1024, 32, BF16, 2)
    cp, ri, _ = SyntheticNetwork(1024, 3, "radix16").layer_csc(2)
    p.top = SparseTopology(1024, 1024, cp, ri)
    p.rows = p.top.rows()
    check_step(p, "silu")
    q = [mx4_quantize(w) for w in p.w]
    x4 = mx4_quantize(p.x)
    for x, t in ((p.x, BF16), (x4, F32)):
        f = p.reference("silu", x=x if x is p.x else x4.dequantize(), w=[m.dequantize() for m in q], out_dtype=t)
        check(p.forward("silu", x=x, w=q, out_dtype=t), f.y, f.bound, "y")
    out = torch.full((150, 1030), 5.0, dtype=BF16, device="cuda")
    p.forward("silu", out=out[:, 1:1025])
    assert torch.equal(out[:, 1:1025], p.forward("silu")) and (out[:, 0] == 5).all() and (out[:, 1025:] == 5).all()


@pytest.mark.parametrize("shared", [False, True])
def test_holes_and_infinities_of_many_tokens(shared):
    """As test_weights_without_connection_and_infinities, for the images' and the blocks' way."""
    p = Shared(200, 256, 320, 32, F16, 2, 16, False) if shared else Problem(200, 256, 320, 32, F16, 2, "ragged")
    want, saved = p.forward("silu", save=True)
    grads = p.backward(saved, "silu")
    hole = torch.as_tensor(p.rows < 0).cuda()
    assert hole.any()
    p.w = [w.masked_fill(hole, float("nan")) for w in p.w]
    y, saved = p.forward("silu", save=True)
    again = p.backward(saved, "silu")
    assert torch.equal(y, want) and torch.equal(again[0], grads[0])
    assert all(torch.equal(a, b) for a, b in zip(again[1] + again[2], grads[1] + grads[2]))
    assert all((d[hole] == 0).all() for d in again[1])
    p.x[150, 7] = float("nan")
    y = p.forward("silu")
    touched = torch.zeros_like(y, dtype=torch.bool)
    touched[150] = torch.as_tensor((p.rows == 7).any(1)).cuda()
    assert touched.any() and torch.isnan(y[touched]).all() and torch.equal(y[~touched], want[~touched])


@pytest.mark.parametrize("shared", [False, True])
def test_large_images_captured_and_replayed(shared):
    """Kernels with more shared memory than a launch has by default, and a gradient that is cleared first, inside a capture that is
    the first call on its topology."""
    make = lambda: Shared(150, 4096, 4100, 32, BF16, 2, 16, False) if shared else Problem(150, 4096, 4100, 32, BF16, 2, "ragged")  # noqa: E731
    p, q = make(), make()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, saved = p.forward("silu", save=True)
        grads = p.backward(saved, "silu")
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    want, kept = q.forward("silu", save=True)
    wants = q.backward(kept, "silu")
    assert torch.equal(y, want) and torch.equal(grads[0], wants[0])
    assert all(torch.equal(a, b) for a, b in zip(grads[1] + grads[2], wants[1] + wants[2]))
    del graph


def test_two_graphs_of_one_topology_replayed_in_turn():
    """Each graph has a workspace of its own: replays of one do not disturb the other's results."""
    p = Problem(300, 500, 400, 20, BF16, 2)
    x2 = (p.x.float() * -0.5).to(BF16)
    want = [p.forward("silu").clone(), p.forward("silu", x=x2).clone()]
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g, x in zip(graphs, (p.x, x2)):
        with torch.cuda.graph(g):
            outs.append(p.forward("silu", x=x))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    del graphs


def test_large_values():
    """Pre-activations far out: the activations' limits, no overflow on the way."""
    p = Problem(40, 64, 48, 8, F32, 1, bias=False)
    p.x *= 1e3
    for kind in ("silu", "gelu", "gelu_tanh"):
        y, saved = p.forward(kind, save=True)
        f = p.reference(kind)
        check(y, f.y, f.bound, kind)
        assert all(torch.isfinite(t).all() for t in p.backward(saved, kind)[1])
    h = Problem(300, 64, 48, 8, BF16, 1, bias=False)
    h.x = (h.x.float() * 1e3).to(BF16)
    for kind in ("silu", "gelu", "gelu_tanh"):
        y, saved = h.forward(kind, save=True)
        f = h.reference(kind)
        check(y, f.y, f.bound, kind)
        assert all(torch.isfinite(t).all() for t in h.backward(saved, kind)[1])


def test_two_threads_with_images_of_different_sizes():
    """The same kernel launched from two threads with different amounts of shared memory."""
    import threading
    a = Problem(40, 4000, 300, 16, BF16, 2)
    b = Problem(60, 6900, 300, 16, BF16, 2)
    want = [p.forward("silu", save=True) for p in (a, b)]
    grads = [p.backward(s, "silu")[0] for p, (_, s) in zip((a, b), want)]
    torch.cuda.synchronize()
    errors = []

    def work(p, y, g):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(150):
                    got, saved = p.forward("silu", save=True)
                    dx = p.backward(saved, "silu", need_dw=False)[0]
                torch.cuda.current_stream().synchronize()
                assert torch.equal(got, y) and torch.equal(dx, g)
        except Exception as e:                             # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(p, y, g)) for p, (y, _), g in zip((a, b), want, grads)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors


@pytest.mark.parametrize("shared", [False, True])
def test_offsets_beyond_32_bits(shared):
    """More than 2^31 activations in one call: its last tokens as a call of their own gives them."""
    tokens, inputs, outputs = 140001, 16384, 32
    p = (Shared(1, inputs, outputs, 16, BF16, 1, 16, False) if shared else Problem(1, inputs, outputs, 16, BF16, 1))
    x = torch.zeros(tokens, inputs, dtype=BF16, device="cuda")
    assert x.numel() > 2 ** 31
    g = torch.Generator("cuda").manual_seed(5)
    tail = torch.randn(500, inputs, device="cuda", generator=g).to(BF16)
    x[-500:] = tail
    dy = torch.zeros(tokens, outputs, dtype=BF16, device="cuda")
    dy[-500:] = torch.randn(500, outputs, device="cuda", generator=g).to(BF16)
    y, saved = p.top.linear(x, p.w[0], p.b[0], activation="silu", save=True)
    small, kept = p.top.linear(tail, p.w[0], p.b[0], activation="silu", save=True)
    assert torch.equal(y[-500:], small) and torch.equal(y[0], y[70000])
    dx, dw, db = p.top.linear_backward(dy, x, p.w[0], saved, activation="silu")
    dx2, dw2, db2 = p.top.linear_backward(dy[-500:], tail, p.w[0], kept, activation="silu")
    assert torch.equal(dx[-500:], dx2) and not dx[:-500].any()
    # the same products, added up in another order: 500 terms and their zeros
    bound = 2 * 510 * ref.U * (tail.double().abs().t() @ dy[-500:].double().abs()).max()
    assert float((dw - dw2).abs().max()) <= bound and float((db - db2).abs().max()) <= bound
    del x, dx, y, saved
    from graphchallenge21_b200 import mx4_quantize
    big = torch.zeros(70000, 33000, dtype=BF16, device="cuda")
    big[-3:] = torch.randn(3, 33000, device="cuda", generator=g).to(BF16)
    q = mx4_quantize(big)
    last = mx4_quantize(big[-3:])
    assert torch.equal(q.codes[-3:], last.codes) and torch.equal(q.scales[-3:], last.scales) and not q.codes[:-3].any()
    values = q.dequantize(BF16)
    assert torch.equal(values[-3:], last.dequantize(BF16)) and not values[:-3].any()


@pytest.mark.parametrize("tokens", [3, 200])
def test_weights_wider_than_any_neuron(tokens):
    p = Problem(tokens, 90, 40, 12, BF16, 2, "random")
    from graphchallenge21_b200 import SparseTopology
    rows = p.rows_given.copy()
    rows[:, -3:] = -1                                      # nine of twelve are used
    p.top = SparseTopology.from_rows(rows, 90)
    assert p.top.slots == 12
    p.rows = p.top.rows()
    check_step(p, "silu")
