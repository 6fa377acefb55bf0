"""The trainable block pieces where values are not finite, sides are short or a
call comes first: what the header promises holds in every form that a call can
take (few queries, tiles on the CUDA cores, tensor cores), and one form's
results are another's.

Tolerances are those of test_gpu_train.py, derived there."""
import math
import os
import subprocess
import sys

import pytest
import torch
from test_gpu_train import (EPS, HALF, TYPES, U32, attention_case, backward_reference, forward_reference, gen, hat_error, lens, make,
                            norm_backward_reference, norm_inputs, run_backward, run_forward, run_norm, run_norm_backward,
                            standard64, within)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def vk():
    import vestra_kernels

    return vestra_kernels


# dtype, sequences, heads, queries, keys, head_dim: every form of the backward pass
FORMS = [
    # few queries, the keys in one block and split
    ("f32", 2, 3, 1, 300, 64), ("f32", 2, 3, 4, 70, 64), ("f32", 2, 3, 2, 900, 16), ("bf16", 2, 3, 1, 300, 64),
    ("bf16", 2, 3, 1, 40, 8), ("bf16", 2, 2, 3, 200, 64), ("bf16", 2, 2, 4, 150, 64),
    # tiles on the CUDA cores, split and not
    ("f32", 2, 3, 20, 300, 32), ("f32", 2, 40, 130, 200, 64), ("bf16", 2, 2, 30, 50, 64), ("bf16", 2, 3, 70, 600, 32),
    # tensor cores: one block, several, the last full and not
    ("bf16", 2, 40, 100, 70, 64), ("bf16", 2, 3, 300, 385, 64), ("bf16", 2, 3, 256, 384, 64), ("bf16", 2, 30, 3, 200, 64),
]


@pytest.mark.parametrize("dtype,b,h,nq,nk,d", FORMS)
@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("where", ["d_out", "q"])
def test_attention_gradients_past_the_lengths_are_zeros(vk, dtype, b, h, nq, nk, d, bad, where):
    """A value that is not finite in a valid row of d_out or q (an overflowed gradient) leaves the rows past the
    lengths zeros, and the other heads as they are without it."""
    t = TYPES[dtype]
    q, k, v, _, _, _, _ = attention_case(t, b, h, nq, nk, d, "head", False, 80)
    g = make((b, h, nq, d), t, gen(81))
    ql, kl = lens([nq, max(1, nq // 2)]), lens([max(1, nk - 9), nk // 3])
    out, lse = run_forward(vk, q, k, v, ql, kl)
    clean = run_backward(vk, q, k, v, out, lse, g, ql, kl)
    (g if where == "d_out" else q)[0, 0, 0, 3] = bad
    out, lse = run_forward(vk, q, k, v, ql, kl)
    dq, dk, dv = run_backward(vk, q, k, v, out, lse, g, ql, kl)
    for i in range(b):
        assert (dq[i, :, int(ql[i]):] == 0).all()
        assert (dk[i, :, int(kl[i]):] == 0).all() and (dv[i, :, int(kl[i]):] == 0).all()
    for x, y in zip((dq, dk, dv), clean):
        assert torch.equal(x[1:], y[1:]) and torch.equal(x[:1, 1:], y[:1, 1:])


@pytest.mark.parametrize("dtype,b,h,nq,nk,d", FORMS)
@pytest.mark.parametrize("ragged", [False, True])
def test_attention_gradients_of_scores_far_below_zero(vk, dtype, b, h, nq, nk, d, ragged):
    """Scores so low that exp(-lse) is beyond f32: what a block reads past its keys must not count."""
    t = TYPES[dtype]
    q, k, v, _, _, _, _ = attention_case(t, b, h, nq, nk, d, "head", False, 86)
    q, k = (q.abs() + 4).to(t), (-k.abs() - 4).to(t)
    g = make((b, h, nq, d), t, gen(87))
    scale = 8.0 / d  # (sums of d products near -23: -184 at any head size)
    ql, kl = ([nq, max(1, nq // 2)], [max(1, nk - 9), max(1, nk // 3)]) if ragged else ([nq] * b, [nk] * b)
    qt, kt = (lens(ql), lens(kl)) if ragged else (None, None)
    out, lse = run_forward(vk, q, k, v, qt, kt, scale=scale)
    want, bound, lse_want, lse_bound = forward_reference(q, k, v, ql, kl, scale)
    within(out, want, bound, "out")
    live = lse_want != -math.inf
    assert lse_want[live].max() < -95
    within(lse[live], lse_want[live], lse_bound[live], "lse")
    dq, dk, dv = torch.full_like(q, 7.0), torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    vk.attention_backward(q, k, v, out, lse, g, dq, dk, dv, scale=scale, q_lens=qt, kv_lens=kt)
    for name, x, (w, e) in zip(("dq", "dk", "dv"), (dq, dk, dv), backward_reference(q, k, v, out, lse, g, ql, kl, scale)):
        within(x, w, e, name)


# queries, keys, ragged: the last block of keys full and not
SIDES = [(140, 300, False), (140, 256, False), (256, 100, False), (3, 300, False), (1, 300, False), (70, 70, False), (260, 300, True)]


def infinite_query(vk, dtype, nq, nk, ragged):
    """Inputs whose middle query scores -inf with every key, and those without it."""
    t, b, h, row = TYPES[dtype], 2, 20, nq // 2
    q, k, v, _, _, _, _ = attention_case(t, b, h, nq, nk, 64, "head", False, 82)
    k = (k.abs() + 0.1).to(t)
    q[:, :, row, 5] = -math.inf
    ql, kl = ([nq, nq - 9], [nk, nk - 7]) if ragged else ([nq] * b, [nk] * b)
    out, lse = run_forward(vk, q, k, v, *((lens(ql), lens(kl)) if ragged else (None, None)))
    return q, k, v, out, lse, ql, kl, row, [i for i in range(nq) if i != row]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq,nk,ragged", SIDES)
def test_attention_query_of_minus_infinity(vk, dtype, nq, nk, ragged):
    """A query that scores -inf with every key is a row without values: out 0, lse -inf; the others are as without it."""
    q, k, v, out, lse, ql, kl, row, rest = infinite_query(vk, dtype, nq, nk, ragged)
    assert (out[:, :, row] == 0).all() and (lse[:, :, row] == -math.inf).all()
    if rest:
        want, bound, _, _ = forward_reference(q[:, :, rest], k, v, [n - 1 for n in ql], kl, 0.125)
        within(out[:, :, rest], want, bound, "out")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq,nk,ragged", SIDES)
def test_attention_gradients_of_a_query_of_minus_infinity(vk, dtype, nq, nk, ragged):
    """Its gradient is 0, the other queries' and the keys' are as without it (its infinite column of dk apart: 0 * inf)."""
    q, k, v, out, lse, ql, kl, row, rest = infinite_query(vk, dtype, nq, nk, ragged)
    g = make(q.shape, q.dtype, gen(83))
    grads = run_backward(vk, q, k, v, out, lse, g, *((lens(ql), lens(kl)) if ragged else (None, None)))
    assert (grads[0][:, :, row] == 0).all()
    if not rest:
        return
    ql = [n - 1 for n in ql]
    (dq, bq), (dk, bk), (dv, bv) = backward_reference(q[:, :, rest], k, v, out[:, :, rest], lse[:, :, rest], g[:, :, rest], ql, kl, 0.125)
    finite = [i for i in range(64) if i != 5]
    within(grads[0][:, :, rest], dq, bq, "dq")
    within(grads[1][..., finite], dk[..., finite], bk[..., finite], "dk")
    within(grads[2], dv, bv, "dv")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nk,nq,ragged", SIDES)
def test_attention_key_of_minus_infinity(vk, dtype, nk, nq, ragged):
    """A key that every query scores -inf with has no weight: its gradients are 0, the other keys' those of a batch
    without it, and so are the queries' (its own infinite column of dq apart: 0 * inf)."""
    t = TYPES[dtype]
    b, h, row = 2, 20, nk // 2
    q, k, v, _, _, _, _ = attention_case(t, b, h, nq, nk, 64, "head", False, 84)
    q = (q.abs() + 0.1).to(t)
    k[:, :, row, 5] = -math.inf
    g = make(q.shape, t, gen(85))
    ql, kl = ([nq, nq - 9], [nk, nk - 7]) if ragged else ([nq] * b, [nk] * b)
    qt, kt = (lens(ql), lens(kl)) if ragged else (None, None)
    out, lse = run_forward(vk, q, k, v, qt, kt)
    grads = run_backward(vk, q, k, v, out, lse, g, qt, kt)
    assert (grads[1][:, :, row] == 0).all() and (grads[2][:, :, row] == 0).all()
    rest = [i for i in range(nk) if i != row]
    if not rest:
        assert (out == 0).all() and (lse == -math.inf).all()
        return
    kr, vr = k[:, :, rest], v[:, :, rest]
    kl = [n - 1 for n in kl]
    want, bound, _, _ = forward_reference(q, kr, vr, ql, kl, 0.125)
    within(out, want, bound, "out")
    (dq, bq), (dk, bk), (dv, bv) = backward_reference(q, kr, vr, out, lse, g, ql, kl, 0.125)
    finite = [i for i in range(64) if i != 5]
    within(grads[0][..., finite], dq[..., finite], bq[..., finite], "dq")
    within(grads[1][:, :, rest], dk, bk, "dk")
    within(grads[2][:, :, rest], dv, bv, "dv")


@pytest.mark.parametrize("dtype,piece", [("f32", "attention"), ("bf16", "attention"), ("bf16", "rope"), ("f32", "norm")])
def test_first_call_of_a_process_captured(dtype, piece):
    """The first call on a device may be a captured one: nothing has to run before it."""
    here = os.path.dirname(os.path.abspath(__file__))
    run = subprocess.run([sys.executable, "-c", FIRST, dtype, piece], cwd=os.path.dirname(here), capture_output=True, text=True,
                         env={**os.environ, "PYTHONPATH": os.path.join(os.path.dirname(here), "vestra-kernels_b200")}, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


FIRST = """
import sys, torch, vestra_kernels as vk
t, piece = {"f32": torch.float32, "bf16": torch.bfloat16}[sys.argv[1]], sys.argv[2]
x = torch.randn(2, 3, 200, 64, device="cuda").to(t)
pos = torch.arange(200, device="cuda")[:, None].contiguous()
vec = torch.ones(64, device="cuda")

def run():
    if piece == "attention":
        out, lse = torch.empty_like(x), torch.empty(2, 3, 200, device="cuda")
        grads = [torch.empty_like(x) for _ in range(3)]
        vk.attention_forward(x, x, x, out, lse)
        vk.attention_backward(x, x, x, out, lse, x, *grads)
        return [out, lse, *grads]
    if piece == "rope":
        out = torch.empty_like(x)
        vk.rope_axes(x, None, pos, (64,), 100.0, out, None)
        return [out]
    rows = x.view(6, 200, 64)
    h, y, stats = torch.empty_like(rows), torch.empty_like(rows), torch.empty(6, 200, 2, device="cuda")
    d_x, d_branch, d_gamma, d_beta = torch.empty_like(rows), torch.empty_like(rows), torch.empty_like(vec), torch.empty_like(vec)
    vk.residual_norm_forward(rows, rows, vec, vec, 1e-6, h, y, stats)
    vk.residual_norm_backward(rows, rows, h, rows, stats, vec, d_x, d_branch, d_gamma, d_beta)
    return [h, y, stats, d_x, d_branch, d_gamma, d_beta]

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    held = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(held, run()))
vk.synchronize()
"""


def test_residual_norm_of_as_many_rows_as_are_taken(vk):
    """2^31 - 1 rows, of one column: h = x + branch, whose norm is beta."""
    rows = 2 ** 31 - 1
    x = torch.zeros(1, rows, 1, dtype=torch.bfloat16, device="cuda")
    branch, y = torch.ones_like(x), torch.zeros_like(x)
    stats = torch.zeros(1, rows, 2, device="cuda")
    x[0, -9:] = 2
    gamma, beta = torch.ones(1, device="cuda"), torch.full((1,), 3.0, device="cuda")
    vk.residual_norm_forward(x, branch, gamma, beta, 1e-2, x, y, stats)
    assert (x[0, :9] == 1).all() and (x[0, -9:] == 3).all()
    assert (stats[0, -9:, 0] == 3).all() and (stats[0, :9, 0] == 1).all()
    within(stats[0, -9:, 1], torch.full((9,), 10.0, device="cuda"), 10 * 2.0 ** -22, "rstd")
    assert (y == 3).all()


@pytest.mark.parametrize("side", [False, True])
def test_synchronize_waits_for_the_last_call(vk, side):
    """Of the default stream and of another one."""
    x = make((64, 12, 3000, 64), torch.bfloat16, gen(88))
    pos, out = torch.arange(3000, device="cuda")[:, None].contiguous(), torch.empty_like(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream() if side else torch.cuda.default_stream()):
        for _ in range(20):
            vk.rope_axes(x, None, pos, (64,), 100.0, out, None)
        done = torch.cuda.Event()
        done.record()
    vk.synchronize()
    assert done.query()


# bf16 of 64 where few queries or few keys meet a long other side on the tensor cores, and few scores off them
SHORT_SIDES = [(8, 3, 2, 1500), (8, 12, 2, 700), (8, 12, 3, 300), (8, 12, 7, 500), (8, 12, 500, 5), (4, 12, 900, 2), (4, 30, 60, 60),
               (3, 5, 130, 3), (1, 2, 3, 300), (2, 2, 4, 150), (1, 1, 60, 60), (1, 2, 865, 3)]


@pytest.mark.parametrize("b,h,nq,nk", SHORT_SIDES)
@pytest.mark.parametrize("ragged", [False, True])
def test_attention_with_a_short_side(vk, b, h, nq, nk, ragged):
    q, k, v, ql, kl, qt, kt = attention_case(torch.bfloat16, b, h, nq, nk, 64, "token", ragged, 89)
    out, lse = run_forward(vk, q, k, v, qt, kt)
    want, bound, lse_want, lse_bound = forward_reference(q, k, v, ql, kl, 0.125)
    within(out, want, bound, "out")
    live = lse_want != -math.inf
    assert torch.equal(lse != -math.inf, live)
    within(lse[live], lse_want[live], lse_bound[live], "lse")
    g = make(q.shape, q.dtype, gen(90), "token")
    if ragged:
        for i in range(b):
            g[i, :, ql[i]:] = math.nan
    grads = run_backward(vk, q, k, v, out, lse, g, qt, kt)
    for name, x, (w, e) in zip(("dq", "dk", "dv"), grads, backward_reference(q, k, v, out, lse, g, ql, kl, 0.125)):
        within(x, w, e, name)


@pytest.mark.parametrize("b,h,n,m,lengths", [(8, 12, 865, 2, None), (8, 12, 865, 8, None), (8, 12, 3, 865, None), (8, 12, 300, 300, (200, 3)),
                                             (8, 12, 865, 865, None)])
def test_attention_gradients_keep_their_error_on_short_sides(vk, b, h, n, m, lengths):
    """The tensor cores round P and dS to bf16, and that costs a gradient as much as its own rounding whether a row has two
    keys or many: of terms of random signs the squares add up to the square of their sum, on average, so roundings of the
    terms and one of the sum, of the same relative size, make sqrt(2) of the latter alone as a root mean square; 1.6 is an eighth above it, for averages over ten thousand values and more."""
    q, k, v, _, _, _, _ = attention_case(torch.bfloat16, b, h, n, m, 64, "head", False, 91)
    g = make(q.shape, q.dtype, gen(92))
    x, y = lengths or (n, m)
    qt, kt = (lens([x] * b), lens([y] * b)) if lengths else (None, None)
    out, lse = run_forward(vk, q, k, v, qt, kt)
    grads = run_backward(vk, q, k, v, out, lse, g, qt, kt)
    q, k, v, g, out = (t[:, :, :c].double() for t, c in ((q, x), (k, y), (v, y), (g, x), (out, x)))
    p = torch.softmax(q @ k.mT * 0.125, -1)
    ds = p * (g @ v.mT - (g * out).sum(-1, keepdim=True))
    for got, want in zip(grads, (ds @ k * 0.125, ds.mT @ q * 0.125, p.mT @ g)):
        got = got[:, :, :want.shape[2]].double()
        one = (want.bfloat16().double() - want).norm()
        assert (got - want).norm() <= 1.6 * one


def test_residual_norm_at_odd_addresses(vk):
    """Every output of matrices that start 4 or 2 bytes off, against 64 bits."""
    s = norm_inputs("f32", "bf16", 3, 401, 136, True, True, True, 50)

    def off(t):  # the same values, one element further
        return None if t is None else torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

    h, y, stats, post_stats = run_norm(vk, s)
    g = gen(51)
    d_h, d_y = torch.randn(h.shape, device="cuda", generator=g), torch.randn(y.shape, device="cuda", generator=g).bfloat16()
    s = {n: off(t) for n, t in s.items()}
    x, y3, h3 = off(s["x"]), off(torch.zeros_like(y)), off(torch.zeros_like(h))
    st3, post3 = torch.zeros_like(stats), torch.zeros_like(post_stats)
    vk.residual_norm_forward(x, s["branch"], s["gamma"], s["beta"], EPS, h3, y3, st3, scale=s["scale"], gate=s["gate"],
                             post_gamma=s["post_gamma"], post_beta=s["post_beta"], post_stats=post3)
    n = s["branch"].double()
    hat, mean, rstd = standard64(n)
    e, e_mean, e_rstd = hat_error(n, mean, rstd, 0 * n)
    within(post3[..., :1], mean, e_mean, "post mean")
    within(post3[..., 1:], rstd, e_rstd, "post rstd")
    pg = s["post_gamma"].double()
    n = hat * pg + s["post_beta"].double()
    n_err = e * pg.abs() + 2 * U32 * (n.abs() + (hat * pg).abs())
    f = s["scale"].double() * s["gate"].double()[:, None]
    want_h = s["x"].double() + f * n
    h_err = f.abs() * (n_err + 2 * U32 * n.abs()) * 1.01 + U32 * want_h.abs()
    within(h3, want_h, h_err + U32 * 1.01 * want_h.abs(), "h")
    hat, mean, rstd = standard64(want_h)
    e, e_mean, e_rstd = hat_error(want_h, mean, rstd, h_err)
    within(st3[..., :1], mean, e_mean + 1e-12, "mean")
    within(st3[..., 1:], rstd, e_rstd, "rstd")
    want_y = hat * s["gamma"].double() + s["beta"].double()
    y_err = e * s["gamma"].double().abs() + 2 * U32 * (want_y.abs() + (hat * s["gamma"].double()).abs())
    within(y3, want_y, y_err + HALF[torch.bfloat16] * 1.01 * want_y.abs(), "y")
    got = run_norm_backward(vk, s, h3, st3, post3, off(d_h), off(d_y), d_x=off(d_h), d_branch=off(d_y))
    want, bound = norm_backward_reference(s, h3, st3, post3, d_h, d_y)
    assert set(got) == set(want)
    for name in want:
        within(got[name], want[name], bound[name] + 1e-30, name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [1e-38, 1e-40, 2.0 ** -100])
def test_attention_of_a_tiny_scale(vk, dtype, scale):
    """Every score next to 0: the mean of the values, and gradients that keep it."""
    q, k, v, ql, kl, _, _ = attention_case(TYPES[dtype], 2, 12, 200, 300, 64, "head", False, 93)
    g = make(q.shape, q.dtype, gen(94))
    out, lse = run_forward(vk, q, k, v, None, None, scale=scale)
    want, bound, lse_want, lse_bound = forward_reference(q, k, v, ql, kl, scale)
    within(out, want, bound, "out")
    within(lse, lse_want, lse_bound, "lse")
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    vk.attention_backward(q, k, v, out, lse, g, dq, dk, dv, scale=scale)
    for name, x, (w, e) in zip(("dq", "dk", "dv"), (dq, dk, dv), backward_reference(q, k, v, out, lse, g, ql, kl, scale)):
        within(x, w, e, name)
