"""The feed-forward operators this framework is measured on: whole calls on ``SparseTopology`` as a training step or a
serving program makes them, and the same in elementary torch operations (``own = False``).

A topology connects every output neuron to at most ``slots`` input neurons (32 in the challenge networks); activations are
[tokens, neurons] matrices, the weights of a set are [outputs, slots].  ``op`` names the operator:

  gated    y = act(x Wg + bg) * (x Wu + bu): gated feed-forward block, gate and up projection over one topology
  train    the same (or, with sets = 1, y = act(x W + b)) and its gradients: dx, dw and db for every set
  quantize a matrix to microscaled 4-bit floats (E2M1, blocks of 32 along a row, one power-of-two scale each)
  product  the layer with microscaled weights, sets = 1 plain, 2 gated; x4: the activations are quantised on the way too

``net`` names the topology: "random" draws a neuron's inputs at random, "radix16" is the butterfly of 16-wide blocks of the
challenge networks (a block's 16 outputs read the same two blocks of inputs), "general" is random with a tenth of the
connections missing."""
import math

import torch

own = False

FORMATS = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, op, tokens, inputs, outputs=0, slots=32, net="random", dtype="bf16", sets=2, act="silu", x4=False):
    return {"name": name, "op": op, "tokens": tokens, "inputs": inputs, "outputs": outputs, "slots": slots, "net": net,
            "dtype": dtype, "sets": sets, "act": act, "x4": x4}


def listed():
    return [
        # one token of a decoding loop through the widest block: the latency of a call, weights read once
        _case("gated_one_token", "gated", 1, 4096, 16384),
        # a few hundred rows in full precision, ragged neurons, sizes that no vector width divides
        _case("gated_ragged", "gated", 301, 1000, 2500, slots=37, net="general", dtype="fp32", act="gelu"),
        # a long prompt through the up half of a feed-forward block
        _case("gated_prompt", "gated", 4096, 4096, 16384),
        # the challenge's butterfly at N = 16384 with trained (unequal) weights
        _case("gated_butterfly", "gated", 1024, 16384, 16384, net="radix16", dtype="fp16", act="gelu_tanh"),
        # fine-tuning steps: a small batch in full precision, a full one, the down projection, the widest block
        _case("train_small", "train", 97, 1024, 4096, dtype="fp32"),
        _case("train_block", "train", 4096, 1024, 4096, net="radix16"),
        _case("train_down", "train", 2048, 4096, 1024, slots=64, sets=1, act="none"),
        _case("train_wide", "train", 1024, 16384, 16384, dtype="fp16", act="gelu"),
        # weights after training, and a prompt's activations, to 4 bits
        _case("quantize_weights", "quantize", 16384, 32, dtype="fp32"),
        _case("quantize_tokens", "quantize", 8191, 4100),
        # decoding and prompt with 4-bit weights
        _case("product_one_token", "product", 1, 16384, 4096, sets=1, act="none"),
        _case("product_prompt", "product", 2000, 4096, 16384, x4=True),
    ]


def draw(rng):
    def size(lo, hi, step=1):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step) * step))

    op = rng.choice(["gated", "train", "quantize", "product"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op == "quantize":
        cols = size(20, 16384)
        return {k: v for k, v in _case("", op, size(1, min(65536, 2**26 // cols)), cols, dtype=dtype).items() if k != "name"}
    net = rng.choice(["random", "radix16", "general"])
    step = rng.choice([16, 1]) if net != "radix16" else 16
    inputs, outputs = size(256, 16384, step), size(256, 16384, step)
    slots = 32 if net == "radix16" else rng.choice([8, 20, 32, 32, 37, 64])
    sets = 2 if op == "gated" else rng.choice([1, 2])
    act = rng.choice(["silu", "gelu", "gelu_tanh"]) if sets == 2 or op == "train" else rng.choice(["none", "relu", "clip", "silu"])
    # as many connections times tokens as the largest listed case of the kind at most
    most = (2**31 if op != "train" else 2**29) // (outputs * slots)
    c = _case("", op, size(1, max(2, min(8192, most))), inputs, outputs, slots, net, dtype, sets, act,
              op == "product" and rng.choice([True, False]))
    return {k: v for k, v in c.items() if k != "name"}


# ---- inputs --------------------------------------------------------------------------------

def _rows(case, gen):
    """[outputs, slots] input neurons, ascending; missing connections (-1) behind them."""
    n, m, k = case["inputs"], case["outputs"], case["slots"]
    if case["net"] == "radix16":
        block, at = torch.arange(m, device="cuda") // 16, torch.arange(16, device="cuda")
        a, b = block * 16 % n, (block * 16 + 16 * (n // 32)) % n
        return torch.cat([a[:, None] + at, b[:, None] + at], 1).sort(1).values
    r = (torch.rand(m, k, device="cuda", generator=gen) * (n - k + 1)).long().sort(1).values + torch.arange(k, device="cuda")
    if case["net"] == "general":
        gone = torch.rand(m, k, device="cuda", generator=gen) < 0.1
        r = r.masked_fill(gone, n).sort(1).values
        r = r.masked_fill(r == n, -1)
    return r


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    n, m, k, dt = case["inputs"], case["outputs"], case["slots"], FORMATS[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    state = dict(case)
    if case["op"] == "quantize":
        # rows of different magnitudes, a few of them zero
        x = randn(case["tokens"], n) * torch.exp2(2 * randn(case["tokens"], 1))
        state["x"] = (x * (torch.rand(case["tokens"], 1, device="cuda", generator=gen) > 0.01)).to(dt)
        return state
    rows = _rows(case, gen)
    state["rows"] = rows
    state["x"] = randn(case["tokens"], n).to(dt)
    state["w"] = [(randn(m, k) / math.sqrt(k)).masked_fill(rows < 0, 0.0).to(dt) for _ in range(case["sets"])]
    state["b"] = [0.1 * randn(m) for _ in range(case["sets"])]
    if case["op"] == "train":
        state["dy"] = randn(case["tokens"], m).to(dt)
    if case["op"] == "product":
        state["w"] = [_quantize(w) for w in state["w"]]
    if own:
        from graphchallenge21_b200 import SparseTopology
        state["top"] = SparseTopology.from_rows(rows.cpu().numpy(), n)
    return state


# ---- plain form ----------------------------------------------------------------------------

def _act(z, kind):
    if kind == "none":
        return z
    if kind == "relu":
        return z.clamp(min=0)
    if kind == "clip":
        return z.clamp(0, 32)
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)))


def _slope(z, kind):
    if kind == "none":
        return torch.ones_like(z)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z**3))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)


def _quantize(v):
    """Codes [rows, blocks, 16] (two to a byte, the even one in the low half) and scale bytes [rows, blocks]."""
    v = v.float()
    rows, cols = v.shape
    blocks = (cols + 31) // 32
    v = torch.nn.functional.pad(v, (0, blocks * 32 - cols)).view(rows, blocks, 32)
    top = v.abs().amax(2)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 127)          # floor(log2 top) - 2
    e = torch.where(top == 0, -127, e)
    # by an exact power of two, in two steps: 2^127 times 2^-e may pass the range of one factor
    a = v.double().abs() * torch.exp2(-e.double())[:, :, None]
    # round half to even on the grid of E2M1: steps of 1/2 below 2, of 1 below 4, of 2 up to 6
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)
    code = (a[..., None] > torch.tensor(E2M1[:-1], device=v.device, dtype=a.dtype)).sum(-1) + 8 * torch.signbit(v).long()
    return (code[:, :, 0::2] | (code[:, :, 1::2] << 4)).to(torch.uint8), (e + 127).to(torch.uint8)


def _values(codes, scales, cols):
    """The fp32 values a microscaled matrix stands for."""
    code = torch.stack([codes & 15, codes >> 4], 3).flatten(2).long()
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device, dtype=torch.float64)
    return (table[code] * torch.exp2(scales.double() - 127)[:, :, None]).flatten(1)[:, :cols].float()


def _plain(state):
    dt = FORMATS[state["dtype"]]
    if state["op"] == "quantize":
        codes, scales = _quantize(state["x"])
        return {"values": _values(codes, scales, state["inputs"]), "scales": scales}
    rows, x, act, k = state["rows"], state["x"].float(), state["act"], state["slots"]
    at = rows.clamp(min=0)
    if state["x4"]:
        x = _values(*_quantize(x), state["inputs"])
    w = [_values(*q, k) if state["op"] == "product" else q.float() for q in state["w"]]
    w = torch.stack(w, 1).masked_fill((rows < 0)[:, None, :], 0.0)                # [outputs, sets, slots]
    xg = x.t()[at]                                                                # [outputs, slots, tokens]
    z = torch.bmm(w, xg) + torch.stack(state["b"], 1)[:, :, None]                 # [outputs, sets, tokens]
    y = _act(z[:, 0], act) * z[:, 1] if state["sets"] == 2 else _act(z[:, 0], act)
    if state["op"] != "train":
        return {"y": y.t().to(dt)}
    dy = state["dy"].float().t()
    d = [dy * _slope(z[:, 0], act)]
    if state["sets"] == 2:
        d = [d[0] * z[:, 1], dy * _act(z[:, 0], act)]
    d = torch.stack(d, 1)                                                         # [outputs, sets, tokens]
    dw = torch.bmm(d, xg.transpose(1, 2)).masked_fill((rows < 0)[:, None, :], 0.0)
    dx = torch.zeros_like(x.t()).index_add_(0, at.flatten(), torch.bmm(w.transpose(1, 2), d).flatten(0, 1))
    return {"y": y.t().to(dt), "dx": dx.t().to(dt), "dw": [dw[:, s] for s in range(state["sets"])],
            "db": [d[:, s].sum(1) for s in range(state["sets"])]}


# ---- the framework's calls -----------------------------------------------------------------

def _framework(state):
    from graphchallenge21_b200 import MX4, mx4_quantize
    dt, x = FORMATS[state["dtype"]], state["x"]
    if state["op"] == "quantize":
        q = mx4_quantize(x)
        return {"values": q.dequantize(), "scales": q.scales}
    top, act, sets = state["top"], state["act"], state["sets"]
    w, b = state["w"], state["b"]
    if state["op"] == "product":
        w = [MX4(codes, scales, state["slots"]) for codes, scales in w]
        if state["x4"]:
            x = mx4_quantize(x)
    forward = (lambda **kw: top.gated(x, w[0], w[1], b[0], b[1], activation=act, **kw)) if sets == 2 else (
        lambda **kw: top.linear(x, w[0], b[0], activation=act, **kw))
    if state["op"] != "train":
        return {"y": forward(out_dtype=dt)}
    y, saved = forward(save=True)
    if sets == 2:
        dx, dwg, dwu, dbg, dbu = top.gated_backward(state["dy"], x, w[0], w[1], saved, activation=act)
        return {"y": y, "dx": dx, "dw": [dwg, dwu], "db": [dbg, dbu]}
    dx, dw, db = top.linear_backward(state["dy"], x, w[0], saved, activation=act)
    return {"y": y, "dx": dx, "dw": [dw], "db": [db]}


def run(state):
    return _framework(state) if own else _plain(state)


# ---- the definition in 64 bits -------------------------------------------------------------

def _exact_quantize(v):
    """The nearest representable value of every element: all 16 candidates at the block's scale, ties to the even code."""
    rows, cols = v.shape
    v = torch.nn.functional.pad(v, (0, -cols % 32)).view(rows, -1, 32)
    top = v.abs().amax(2, keepdim=True)
    e = torch.where(top > 0, torch.floor(torch.log2(top)) - 2, -127.0)
    # log2 is rounded: near a power of two its floor may be one off either way
    e = torch.where((top > 0) & (torch.exp2(e + 2) > top), e - 1, e)
    e = torch.where((top > 0) & (torch.exp2(e + 3) <= top), e + 1, e).clamp(-127, 127)
    scale = torch.exp2(e)
    best, gap = torch.zeros_like(v), v.abs().clone()
    for code, m in enumerate(E2M1):
        if code:
            off = (v.abs() - m * scale).abs()
            take = (off < gap) | ((off == gap) & (code % 2 == 0))
            best, gap = torch.where(take, m * scale, best), torch.where(take, off, gap)
    return (best * torch.sign(v)).flatten(1)[:, :cols], (e + 127).squeeze(2)


def exact(case, seed):
    if case["op"] != "quantize" and case["inputs"] * case["outputs"] * 8 > 3e9:
        return None
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "quantize":
        if x.numel() > 2**28:
            return None
        values, _ = _exact_quantize(x)
        return {"values": values, "scales": None}
    rows, n, m, act = s["rows"], case["inputs"], case["outputs"], case["act"]
    if case["x4"]:
        x = _exact_quantize(x)[0]
    out = torch.arange(m, device="cuda")[:, None].expand_as(rows)[rows >= 0]
    inp = rows[rows >= 0]
    z, dense = [], []
    for q, b in zip(s["w"], s["b"]):
        if case["op"] == "product":
            codes, scales = q
            code = torch.stack([codes & 15, codes >> 4], 3).flatten(2).long()
            mag, man = (code >> 1) & 3, code & 1
            v = torch.where(mag == 0, 0.5 * man, torch.exp2(mag.double() - 1) * (1 + 0.5 * man))
            v = torch.where(code >= 8, -v, v) * torch.exp2(scales.double() - 127)[:, :, None]
            q = v.flatten(1)[:, : case["slots"]]
        W = torch.zeros(n, m, device="cuda", dtype=torch.float64)
        W.index_put_((inp, out), q.double()[rows >= 0], accumulate=True)
        dense.append(W)
        z.append(x @ W + b.double())
    g = z[0].requires_grad_()
    a = {"none": lambda v: v * 1, "relu": torch.relu, "clip": lambda v: torch.minimum(torch.relu(v), torch.full_like(v, 32)),
         "silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: v * torch.special.ndtr(v),
         "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v**3))}[act](g)
    y = a.detach() * z[1] if case["sets"] == 2 else a.detach()
    if case["op"] != "train":
        return {"y": y}
    slope, = torch.autograd.grad(a.sum(), g)
    dy = s["dy"].double()
    d = [dy * slope * z[1], dy * a.detach()] if case["sets"] == 2 else [dy * slope]
    dx = sum(v @ W.t() for v, W in zip(d, dense))
    dw = []
    for v in d:
        D = x.t() @ v
        full = torch.zeros(rows.shape, device="cuda", dtype=torch.float64)
        full[rows >= 0] = D[inp, out]
        dw.append(full)
    return {"y": y, "dx": dx, "dw": dw, "db": [v.sum(0) for v in d]}


def work(case):
    t, n, m, k, sets = case["tokens"], case["inputs"], case["outputs"], case["slots"], case["sets"]
    s = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "quantize":
        return {"bytes": t * n * (s + 4) + t * ((n + 31) // 32 * 17), "flops": 4 * t * n}
    index = m * k * (2 if n < 65536 else 4)
    fma = 2 * sets * t * m * k
    if case["op"] == "product":
        return {"bytes": s * t * (n + m) + index + sets * m * ((k + 31) // 32 * 17 + 4), "flops": fma}
    forward = s * t * (n + m) + index + sets * m * (k * s + 4)
    if case["op"] == "gated":
        return {"bytes": forward, "flops": fma}
    # the gradients: dy and x read once more than the forward's output and input, dx, dw and db written
    return {"bytes": forward + s * t * (m + n) + sets * m * (k + 1) * 4, "flops": 3 * fma}
