"""GPU tests of the feed-forward operators where values leave the ordinary: gradients beyond fp16's range, infinities, activations far
from zero.  References and the meaning of U and half_step: tests/feedforward_reference.py."""
import math

import numpy as np
import pytest

import feedforward_reference as ref
from test_gpu_feedforward import BF16, F16, F32, Problem, Shared, check, torch

pytestmark = pytest.mark.gpu


# ---- dL/dz on its way to dx in fp16 ---------------------------------------------------------------

def scaled_dx(f, dy):
    """dx and its bound where the gathered dL/dz of a token are held in fp16 at a power of two of their own: a value is off by half
    a step, or by half the smallest subnormal at that scale, where the token's largest value lies in [2^14, 2^15): 2^-25 2^-14 of it (twice
    that where the kernel's largest value is below a power of two and the exact one is not)."""
    h, u = ref.half_step(F16), ref.U
    dyd = dy.double()
    off = [e + u * z.abs() for z, e in zip(f.z, f.dz)]
    s, ds = ref.slope(f.z[0], f.kind, f.clip), 0.85 * off[0] + 32 * u * (1 + f.z[0].abs())
    if f.kind in ("none", "relu", "clip"):
        ds = ref.corners(f.z[0], f.dz[0], f.kind, f.clip)
    if len(f.ws) == 1:
        d, dd = [dyd * s], [dyd.abs() * ds]
    else:
        a, da = ref.act(f.z[0], f.kind, f.clip), 1.13 * off[0] + 16 * u * f.z[0].abs()
        d = [dyd * s * f.z[1], dyd * a]
        dd = [dyd.abs() * (ds * (f.z[1].abs() + off[1]) + s.abs() * off[1]), dyd.abs() * da]
    top = torch.stack([v.abs() for v in d]).nan_to_num(0, 0, 0).amax((0, 2))
    rows = torch.as_tensor(f.rows, device=dy.device).long()
    fan = int(torch.bincount(rows[rows >= 0]).max())
    dx, bound = torch.zeros(dy.shape[0], f.inputs, dtype=torch.float64, device=dy.device), 0
    for v, e, w in zip(d, dd, f.ws):
        W, A = ref.dense(f.rows, w, f.inputs), ref.dense(f.rows, w.double().abs(), f.inputs)
        es = (e + 4 * u * v.abs()) * (1 + h) + h * v.abs() + 2.0 ** -38 * top[:, None]
        dx = dx + v @ W.t()
        bound = bound + es @ A.t() + (fan * len(f.ws) + 2) * u * ((v.abs() + es) @ A.t())
    return dx, bound * (1 + h) + ref.stored(dx, F16), d


@pytest.mark.parametrize("kind, sets", [("silu", 2), ("gelu", 2), ("relu", 2), ("none", 2), ("gelu_tanh", 1), ("clip", 1)])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("tokens", [1, 6, 40, 200])
def test_fp16_gradients_beyond_the_types_range(tokens, shared, kind, sets):
    """dL/dz above 65504 and below 2^-24 where dx itself is well inside: both by the token."""
    p = Shared(tokens, 256, 320, 32, F16, sets, 16, False) if shared else Problem(tokens, 256, 320, 16, F16, sets, "ragged")
    # small weights and large activations: pre-activations of order 30, gradients of order 3000 of most tokens ...
    p.w = [(0.01 * w.float()).to(F16) for w in p.w]
    p.x = (3000 * p.x.float()).clamp(-6e4, 6e4).to(F16)
    p.dy = (3000 * p.dy.float()).to(F16)
    # ... and tiny ones of every third, whose dL/dz are subnormal or gone in fp16
    p.dy[2::3] = (p.dy[2::3].float() * 2.0 ** -36).to(F16)
    y, saved = p.forward(kind, save=True)
    f = p.reference(kind)
    dx, dw, db = p.backward(saved, kind)
    want, bound, d = scaled_dx(f, p.dy)
    assert want.abs().max() < 6e4
    if sets == 2:
        assert max(float(v.abs().max()) for v in d) > 65504
    check(dx, want, bound, "dx")
    assert all(torch.isfinite(t).all() for t in dw + db)
    only = p.backward(saved, kind, need_dw=False)[0]
    assert torch.equal(only, dx)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("sets", [1, 2])
def test_fp16_small_gradients_meet_large_weights(sets, shared):
    """dL/dz around fp16's smallest numbers, weights of order 100: what dx loses is half a step of a term, not of the subnormals."""
    p = Shared(70, 256, 320, 32, F16, sets, 16, True) if shared else Problem(70, 300, 200, 16, F16, sets)
    p.w = [(100 * w.float()).to(F16) for w in p.w]
    p.x = (0.01 * p.x.float()).to(F16)
    p.dy = (2.0 ** -22 * p.dy.float()).to(F16)
    y, saved = p.forward("silu", save=True)
    want, bound, d = scaled_dx(p.reference("silu"), p.dy)
    check(p.backward(saved, "silu")[0], want, bound, "dx")


@pytest.mark.parametrize("tokens", [5, 90])
def test_fp16_infinite_gradients_stay_with_their_connections(tokens):
    p = Problem(tokens, 256, 320, 16, F16, 2)
    y, saved = p.forward("silu", save=True)
    f = p.reference("silu")
    want, bound, _ = scaled_dx(f, p.dy)
    clean = p.backward(saved, "silu")[0]
    check(clean, want, bound, "dx")
    p.dy[3, 11], p.dy[4, 200] = float("inf"), float("nan")
    dx = p.backward(saved, "silu")[0]
    touched = torch.zeros_like(dx, dtype=torch.bool)
    touched[3, torch.as_tensor(p.rows[11]).cuda().long()] = True
    touched[4, torch.as_tensor(p.rows[200]).cuda().long()] = True
    assert not torch.isfinite(dx[touched]).any()
    # what else these two tokens hold is scaled by their largest finite value, which may have been one of the two
    check(dx[~touched], want[~touched], (2 * bound)[~touched], "the others")


# ---- infinities in gradients of weights --------------------------------------------------------------

def check_with_infinities(got, want, bound, what):
    odd = ~torch.isfinite(want)
    assert odd.any()
    assert torch.equal(got[odd].double().nan_to_num(7.0, posinf=5.0, neginf=3.0), want[odd].nan_to_num(7.0, posinf=5.0, neginf=3.0)), what
    check(got[~odd], want[~odd], bound[~odd], what)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("tokens", [20, 63, 64, 100, 129, 300])
def test_infinities_in_gradients_of_weights(tokens, shared, dtype):
    """An infinite activation or gradient of one token gives infinities of the definition's sign, and NaN only where the definition
    has 0 times infinity or a difference of two."""
    p = Shared(tokens, 256, 320, 32, dtype, 1, 16, False) if shared else Problem(tokens, 256, 320, 16, dtype, 1, "ragged")
    p.dy = torch.where(p.dy.float().abs() < 0.1, torch.ones_like(p.dy), p.dy)
    p.dy[1, ::5] = 1.0                                   # few bits, and gradients of zero
    p.dy[1, 4::5] = 0.0
    p.x[1, 7], p.x[tokens - 1, 30] = float("inf"), -float("inf")
    p.dy[2, 9], p.dy[12, 21] = -float("inf"), float("inf")
    p.x[2, ::3] = 0.0
    y, saved = p.forward("none", save=True)
    dx, dw, db = p.backward(saved, "none")
    rows = torch.as_tensor(p.rows).cuda().long()
    xd, v, at = p.x.double(), p.dy.double(), rows.clamp(min=0)
    want = torch.gather((xd.t() @ v).t(), 1, at).masked_fill(rows < 0, 0.0)
    size = torch.gather((xd.abs().t() @ v.abs()).t(), 1, at).masked_fill(rows < 0, 0.0)
    bound = (tokens + 8 + 4) * ref.U * size + 2.0 ** -140
    assert (want == float("inf")).any() and (want == -float("inf")).any() and torch.isnan(want).any()
    check_with_infinities(dw[0], want, bound, "dw")
    check_with_infinities(db[0], v.sum(0), (tokens + 8) * ref.U * v.abs().sum(0), "db")


# ---- activations far from zero -----------------------------------------------------------------------

def activation_of(values, dtype, kind, tokens, shared, out_dtype):
    """The activation of `values` [tokens], through a layer whose first connection has the weight one and the others zero."""
    from graphchallenge21_b200 import SparseTopology
    n = 32
    rows = np.tile(np.arange(n), (n, 1)) if shared else np.arange(n)[:, None]
    top = SparseTopology.from_rows(rows, n)
    x = torch.zeros(tokens, n, dtype=dtype, device="cuda")
    x[:, 0] = values
    w = torch.zeros(n, rows.shape[1], dtype=dtype, device="cuda")
    w[:, 0] = 1.0
    y, saved = top.linear(x, w, activation=kind, save=True, out_dtype=out_dtype)
    assert torch.equal(saved.z[0, :, 0], values.float())
    return top, x, w, y, saved


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens, shared", [(3, False), (700, False), (700, True)])
def test_gelu_keeps_its_digits_far_below_zero(tokens, shared, dtype):
    """v Phi(v) for v down to -12: a relative bound.  In the tail Phi is e^(-v^2 / 2) times what changes slowly: three roundings of the exponent
    put it off by 1.5 v^2 u; the exponential and the reciprocal (4 u each), the polynomial and the products by less than 20 u."""
    v = torch.linspace(-12, 4, tokens, device="cuda").to(dtype)
    y = activation_of(v, dtype, "gelu", tokens, shared, F32)[3][:, 0]
    z = v.double()
    want = 0.5 * z * torch.erfc(-z * math.sqrt(0.5))         # (torch.special.ndtr(-12.0) is 0)
    check(y, want, (2 * z * z + 4 * z.abs() + 20) * ref.U * want.abs() + 2.0 ** -140, "gelu")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("shared", [False, True])
def test_slopes_of_huge_pre_activations(kind, dtype, shared):
    """1 above zero and 0 below, to the largest numbers there are."""
    v = torch.tensor([1e5, 1e13, 1e18, 1.8e19, 2e19, 1e25, 1e30, 3e38], device="cuda").repeat(4)
    v = torch.cat([v, -v]).to(dtype)
    top, x, w, y, saved = activation_of(v, dtype, kind, 64, shared, None)
    assert torch.equal(y[:, 0], v.clamp(min=0))
    dx, dw, db = top.linear_backward(torch.ones_like(y), x, w, saved, activation=kind)
    assert torch.isfinite(dx).all() and torch.isfinite(db).all()
    reads = top.outputs if shared else 1
    assert torch.equal(dx[:, 0], (v > 0).to(dtype) * reads)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("tokens, shared", [(4, False), (999, False), (999, True)])
def test_activations_to_a_relative_bound(tokens, shared, kind, dtype):
    """(20 + 12 |z| + 2 z^2 + |z|^3) u of the value: the exponent w of SILU is z, of the tanh form 1.6 z + 0.072 z^3; five roundings of w and two of
    the exponential's argument make 7 u |w| of the exponential at most, GELU's v^2 / 2 less than 2 z^2 u; the rest is below 20 u."""
    v = torch.linspace(-20, 20, tokens, device="cuda").to(dtype)
    y = activation_of(v, dtype, kind, tokens, shared, F32)[3][:, 0]
    z = v.double()
    w = z if kind == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    want = 0.5 * z * torch.erfc(-z * math.sqrt(0.5)) if kind == "gelu" else z / (1 + torch.exp(-w))
    check(y, want, (20 + 12 * z.abs() + 2 * z * z + z.abs() ** 3) * ref.U * want.abs() + 2.0 ** -120, kind)
