"""The trainable block pieces (attention with row statistics and its backward
pass, rotary positions over several axes, the residual step between two norms)
against plain implementations in 64 bits, their refusals, and a run of them
together against 64-bit automatic differentiation.

Tolerances are bounds, element by element, from the roundings each operator
makes: a rounding is off by at most half a step, eps / 2 relative to the value
(f32 2^-24, bf16 2^-8), a sum of n products in f32 by at most n 2^-24 of the
sum of their absolute values."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def vk():
    import vestra_kernels

    return vestra_kernels


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(shape, dtype, g, layout="head", spread=1.0):
    b, h, n, d = shape
    if layout == "token":  # the middle slice of a token-major product
        return torch.randn(b, n, 3, h, d, device="cuda", generator=g).mul_(spread).to(dtype)[:, :, 1].transpose(1, 2)
    return torch.randn(b, h, n, d, device="cuda", generator=g).mul_(spread).to(dtype)


def within(got, want, bound, what):
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"{what}: {over.max().item():.3e} over its bound at {over.argmax().item()}"


# ------------------------------------------------------------------ attention
def lens(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def attention_case(dtype, b, h, nq, nk, d, layout, ragged, seed):
    """Inputs with NaN and infinity wherever the lengths say nothing is."""
    g = gen(seed)
    q, k, v = make((b, h, nq, d), dtype, g, layout), make((b, h, nk, d), dtype, g, layout), make((b, h, nk, d), dtype, g, layout)
    ql = kl = None
    if ragged:
        ql = [nq] + [(nq * (i * 37 % 101)) // 101 for i in range(1, b)]
        kl = [max(1, nk // 2)] + [(nk * ((i - 1) * 53 % 101)) // 101 for i in range(1, b)]  # sequence 1 has no keys
        for i in range(b):
            q[i, :, ql[i]:] = math.nan
            k[i, :, kl[i]:] = math.inf
            v[i, :, kl[i]:] = math.nan
    return q, k, v, ql or [nq] * b, kl or [nk] * b, (lens(ql) if ragged else None), (lens(kl) if ragged else None)


def score_error(q, k, scale):
    """Bound of the error of a score (absolute), which is the relative error of its exponential: d products and the
    scaling; then the exponential itself and its argument's rounding (|s| log2 e at most 2^-23 off), 2^-18 covering
    the coarsest exponential that is used."""
    d = q.shape[-1]
    most = torch.einsum("hnd,hmd->hnm", q.abs(), k.abs()).amax() * scale
    return float((d + 4) * U32 * most + 2.0 ** -18)


ATTENTION = [
    ("f32", 1, 1, 1, 1, 8, "head", False), ("f32", 2, 3, 5, 70, 16, "token", True), ("f32", 1, 2, 64, 64, 32, "head", False),
    ("f32", 2, 2, 65, 129, 64, "token", False), ("f32", 4, 6, 197, 197, 64, "head", True), ("f32", 1, 2, 1, 300, 64, "head", False),
    ("f32", 1, 2, 130, 1, 64, "token", False),
    # few rows, whose long side is split over blocks (shares that are empty among them); many rows, 128 to a block
    ("f32", 1, 1, 1, 3457, 64, "head", False), ("f32", 3, 2, 20, 700, 32, "token", True), ("f32", 2, 6, 100, 1000, 64, "head", True),
    ("f32", 1, 1, 3, 600, 8, "head", False), ("f32", 3, 2, 40, 900, 16, "token", True), ("f32", 1, 2, 500, 500, 64, "head", False),
    ("bf16", 2, 1, 70, 600, 32, "head", True), ("f32", 37, 8, 128, 70, 8, "head", True), ("f32", 37, 8, 128, 70, 16, "token", False),
    ("f32", 37, 8, 127, 130, 32, "head", True), ("f32", 3, 12, 865, 865, 64, "token", True),
    ("bf16", 1, 1, 1, 1, 64, "head", False), ("bf16", 1, 2, 61, 61, 64, "token", False), ("bf16", 1, 2, 127, 128, 64, "head", False),
    ("bf16", 1, 2, 128, 129, 64, "token", False), ("bf16", 2, 3, 129, 127, 64, "head", False), ("bf16", 3, 5, 257, 385, 64, "token", True),
    ("bf16", 2, 2, 300, 1, 64, "token", False), ("bf16", 2, 2, 1, 1000, 64, "head", False), ("bf16", 1, 12, 865, 865, 64, "token", False),
    ("bf16", 6, 3, 200, 200, 64, "head", True), ("bf16", 40, 12, 140, 140, 64, "token", True), ("bf16", 1, 1, 3457, 3457, 64, "head", False),
    ("bf16", 17, 11, 100, 130, 64, "token", False), ("bf16", 15, 11, 300, 70, 64, "head", False), ("bf16", 16, 10, 257, 257, 64, "head", False),
    # few queries, with their keys split and not
    ("f32", 3, 5, 4, 1000, 64, "token", True), ("f32", 2, 40, 2, 333, 32, "head", False), ("bf16", 4, 30, 3, 500, 16, "head", True),
    ("f32", 6, 100, 4, 70, 64, "token", True), ("bf16", 2, 3, 1, 129, 8, "token", False), ("f32", 5, 130, 3, 31, 16, "head", True),
    ("f32", 4, 3, 15, 700, 64, "token", True), ("f32", 30, 6, 16, 90, 32, "head", True), ("f32", 1, 2, 9, 2000, 64, "head", False),
    # more sequences than are put in order, and more items than a launch takes; the latter alone
    ("bf16", 140, 20, 900, 870, 64, "token", True), ("bf16", 127, 24, 900, 300, 64, "head", True), ("bf16", 128, 1, 300, 500, 64, "token", True),
    ("bf16", 2, 3, 70, 90, 32, "head", True), ("bf16", 1, 2, 33, 40, 16, "token", False), ("bf16", 1, 2, 33, 40, 8, "head", False),
]


def forward_reference(q, k, v, ql, kl, scale):
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bound_out, lse = out.clone(), torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    bound_lse = torch.zeros_like(lse)
    for b in range(q.shape[0]):
        n, m = ql[b], kl[b]
        if n == 0 or m == 0:
            continue
        qq, kk, vv = q[b, :, :n].double(), k[b, :, :m].double(), v[b, :, :m].double()
        s = torch.einsum("hnd,hmd->hnm", qq, kk) * scale
        p = torch.softmax(s, -1)
        e = score_error(qq, kk, scale)
        lse[b, :, :n] = torch.logsumexp(s, -1)
        # the sum of exponentials is off by e and its m additions, the logarithm and the sum with the maximum round
        bound_lse[b, :, :n] = e + m * U32 + 4 * U32 * lse[b, :, :n].abs() + 4 * U32
        out[b, :, :n] = torch.einsum("hnm,hmd->hnd", p, vv)
        # each probability: e twice (its own and the sum's), its rounding to the operator's type; the sum of m; the store
        mag = torch.einsum("hnm,hmd->hnd", p, vv.abs())
        bound_out[b, :, :n] = (2 * e + HALF[q.dtype] + 2 * m * U32) * mag + HALF[q.dtype] * 1.01 * out[b, :, :n].abs()
    return out, bound_out, lse, bound_lse


def run_forward(vk, q, k, v, ql, kl, scale=None):
    out = torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:3], 7.0, device="cuda")
    vk.attention_forward(q, k, v, out, lse, scale=scale, q_lens=ql, kv_lens=kl)
    return out, lse


@pytest.mark.parametrize("dtype,b,h,nq,nk,d,layout,ragged", ATTENTION)
def test_attention_forward(vk, dtype, b, h, nq, nk, d, layout, ragged):
    q, k, v, ql, kl, qt, kt = attention_case(TYPES[dtype], b, h, nq, nk, d, layout, ragged, 1)
    scale = d ** -0.5
    want, bound, lse_want, lse_bound = forward_reference(q, k, v, ql, kl, scale)
    out, lse = run_forward(vk, q, k, v, qt, kt)
    within(out, want, bound, "out")
    empty = lse_want == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    within(lse[~empty], lse_want[~empty], lse_bound[~empty], "lse")


def backward_reference(q, k, v, out, lse, g, ql, kl, scale):
    dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (q, k, v))
    bq, bk, bv = dq.clone(), dk.clone(), dv.clone()
    half = HALF[q.dtype]
    for b in range(q.shape[0]):
        n, m = ql[b], kl[b]
        if n == 0 or m == 0:
            continue
        qq, kk, vv, gg, oo = (x[b, :, :y].double() for x, y in ((q, n), (k, m), (v, m), (g, n), (out, n)))
        d = qq.shape[-1]
        e = score_error(qq, kk, scale) + 2 * U32 * float(lse[b, :, :n].abs().max())
        p = torch.exp(torch.einsum("hnd,hmd->hnm", qq, kk) * scale - lse[b, :, :n, None].double())
        dp = torch.einsum("hnd,hmd->hnm", gg, vv)
        delta = (gg * oo).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        # dp and delta: d products each and their difference; ds: its probability, the product, its rounding
        off = (d + 2) * U32 * (torch.einsum("hnd,hmd->hnm", gg.abs(), vv.abs()) + (gg * oo).abs().sum(-1, keepdim=True))
        ds_err = ds.abs() * (e + 2 * U32 + half) + p * off * 1.01
        dv[b, :, :m] = torch.einsum("hnm,hnd->hmd", p, gg)
        bv[b, :, :m] = (e + half + n * U32) * torch.einsum("hnm,hnd->hmd", p, gg.abs()) + half * 1.01 * dv[b, :, :m].abs()
        dq[b, :, :n] = scale * torch.einsum("hnm,hmd->hnd", ds, kk)
        bq[b, :, :n] = scale * torch.einsum("hnm,hmd->hnd", ds_err + m * U32 * ds.abs(), kk.abs()) + half * 1.01 * dq[b, :, :n].abs()
        dk[b, :, :m] = scale * torch.einsum("hnm,hnd->hmd", ds, qq)
        bk[b, :, :m] = scale * torch.einsum("hnm,hnd->hmd", ds_err + n * U32 * ds.abs(), qq.abs()) + half * 1.01 * dk[b, :, :m].abs()
    tiny = 1e-30
    return (dq, bq + tiny), (dk, bk + tiny), (dv, bv + tiny)


def run_backward(vk, q, k, v, out, lse, g, ql, kl):
    dq, dk, dv = torch.full_like(q, 7.0), torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    vk.attention_backward(q, k, v, out, lse, g, dq, dk, dv, q_lens=ql, kv_lens=kl)
    return dq, dk, dv


@pytest.mark.parametrize("dtype,b,h,nq,nk,d,layout,ragged", ATTENTION)
def test_attention_backward(vk, dtype, b, h, nq, nk, d, layout, ragged):
    q, k, v, ql, kl, qt, kt = attention_case(TYPES[dtype], b, h, nq, nk, d, layout, ragged, 2)
    scale = d ** -0.5
    out64, _, lse64, _ = forward_reference(q, k, v, ql, kl, scale)
    out = torch.empty_like(q).copy_(out64)
    lse = lse64.float()
    g = make((b, h, nq, d), TYPES[dtype], gen(3), layout)
    if ragged:
        for i in range(b):
            g[i, :, ql[i]:] = math.nan
            out[i, :, ql[i]:] = math.nan
            lse[i, :, ql[i]:] = math.nan
    want = backward_reference(q, k, v, out, lse, g, ql, kl, scale)
    for name, x, (w, bound) in zip(("dq", "dk", "dv"), run_backward(vk, q, k, v, out, lse, g, qt, kt), want):
        within(x, w, bound, name)


def test_attention_without_queries_or_keys(vk):
    for dtype in (torch.float32, torch.bfloat16):
        g = gen(4)
        q, none = make((2, 3, 70, 64), dtype, g), torch.empty(2, 3, 0, 64, dtype=dtype, device="cuda")
        out, lse = run_forward(vk, q, none, none, None, None)
        assert (out == 0).all() and (lse == -math.inf).all()
        dq, dk, dv = run_backward(vk, q, none, none, out, lse, q, None, None)
        assert (dq == 0).all() and dk.numel() == 0
        out, lse = run_forward(vk, none, q, q, None, None)
        assert out.numel() == 0
        dq, dk, dv = run_backward(vk, none, q, q, out, lse, none, None, None)
        assert (dk == 0).all() and (dv == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("side", ["q", "kv"])
def test_attention_lengths_of_one_side(vk, dtype, side):
    """Lengths of the queries or of the keys alone, out of range ones among them: as if the others were full."""
    t = TYPES[dtype]
    b, h, nq, nk = 5, 3, 260, 300
    q, k, v, _, _, _, _ = attention_case(t, b, h, nq, nk, 64, "token", False, 70)
    g = make((b, h, nq, 64), t, gen(71))
    n = nq if side == "q" else nk
    some, full = lens([n, -3, 0, 131, n + 9]), lens([nk if side == "q" else nq] * b)
    ql, kl = (some, None) if side == "q" else (None, some)
    qf, kf = (some, full) if side == "q" else (full, some)
    out, lse = run_forward(vk, q, k, v, ql, kl)
    want, want_lse = run_forward(vk, q, k, v, qf, kf)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    clamped = [n, 0, 0, 131, n]
    plain, bound, _, _ = forward_reference(q, k, v, clamped if side == "q" else [nq] * b, clamped if side == "kv" else [nk] * b, 0.125)
    within(out, plain, bound, "out")
    got, all_of_it = run_backward(vk, q, k, v, out, lse, g, ql, kl), run_backward(vk, q, k, v, out, lse, g, qf, kf)
    assert all(torch.equal(x, y) for x, y in zip(got, all_of_it))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_empty_sequences_only(vk, dtype):
    t = TYPES[dtype]
    q, k, v, _, _, _, _ = attention_case(t, 3, 2, 200, 150, 64, "head", False, 72)
    none = lens([0, 0, 0])
    for ql, kl in ((none, none), (None, none), (none, None)):
        out, lse = run_forward(vk, q, k, v, ql, kl)
        assert (out == 0).all() and (lse == -math.inf).all()
        assert all((x == 0).all() for x in run_backward(vk, q, k, v, out, lse, q, ql, kl))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 3])
def test_attention_of_few_queries_captured(vk, dtype, n):
    """A graph of the forms without tiles, replayed with other queries and lengths; keys past the lengths get zeros."""
    t = TYPES[dtype]
    q, k, v, _, _, _, _ = attention_case(t, 3, 4, n, 700, 64, "head", False, 75)
    g, kl = make(q.shape, t, gen(76)), lens([700, 1, 300])

    def both():
        out, lse = run_forward(vk, q, k, v, None, kl)
        return (out, lse, *run_backward(vk, q, k, v, out, lse, g, None, kl))

    both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    q.copy_(make(q.shape, t, gen(77)))
    kl.copy_(lens([0, 650, 2]))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, both()))
    assert (held[3][0] == 0).all() and (held[4][2, :, 2:] == 0).all() and (held[1][0] == -math.inf).all()
    want, bound, _, _ = forward_reference(q, k, v, [n] * 3, [0, 650, 2], 0.125)
    within(held[0], want, bound, "out")


def test_attention_of_a_sequence_by_itself(vk):
    """A sequence of a padded batch has the same bits whatever the others' lengths are."""
    q, k, v, _, _, _, _ = attention_case(torch.bfloat16, 6, 4, 700, 700, 64, "token", False, 73)
    g = make((6, 4, 700, 64), torch.bfloat16, gen(74))
    results = []
    for others in ([700, 300, 1, 0, 513], [0, 0, 650, 700, 129], [400] * 5):
        n = lens([450] + others)
        out, lse = run_forward(vk, q, k, v, n, n)
        results.append([x[0] for x in (out, lse, *run_backward(vk, q, k, v, out, lse, g, n, n))])
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(results[0], r))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_scores_that_grow(vk, dtype):
    """Scores of very different size along the keys (each block outgrows the last by far), and a scale of its own."""
    d, n, m = 64, 150, 700
    q, k, v, ql, kl, _, _ = attention_case(TYPES[dtype], 1, 2, n, m, d, "head", False, 5)
    steps = torch.tensor([0.0, 1.0, 6.0, 20.0, 0.5, 40.0], device="cuda").repeat_interleave(128)[:m]
    k = (k * steps[None, None, :, None]).to(k.dtype)
    scale = 0.3
    want, bound, lse_want, lse_bound = forward_reference(q, k, v, ql, kl, scale)
    out, lse = run_forward(vk, q, k, v, None, None, scale=scale)
    within(out, want, bound, "out")
    within(lse, lse_want, lse_bound, "lse")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ragged", [False, True])
def test_attention_scores_far_below_zero(vk, dtype, ragged):
    """Every score near -100: the columns past the sequence's end (a score of 0 there) must not count."""
    t = TYPES[dtype]
    q, k, v, _, _, _, _ = attention_case(t, 2, 2, 140, 300, 64, "head", False, 60)
    q, k = (q.abs() + 3).to(t), (-k.abs() - 3).to(t)
    ql, kl = ([140, 100], [201, 90]) if ragged else ([140, 140], [300, 300])
    qt, kt = (lens(ql), lens(kl)) if ragged else (None, None)
    want, bound, lse_want, lse_bound = forward_reference(q, k, v, ql, kl, 0.125)
    out, lse = run_forward(vk, q, k, v, qt, kt)
    within(out, want, bound, "out")
    live = lse_want != -math.inf
    assert lse_want[live].max() < -80
    within(lse[live], lse_want[live], lse_bound[live], "lse")
    g = make((2, 2, 140, 64), t, gen(61))
    grads = run_backward(vk, q, k, v, out, lse, g, qt, kt)
    for name, x, (w, b) in zip(("dq", "dk", "dv"), grads, backward_reference(q, k, v, out, lse, g, ql, kl, 0.125)):
        within(x, w, b, name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_scores_of_minus_infinity(vk, dtype):
    """Keys that score -inf have no weight; NaN stays in its own batch entry and head."""
    q, k, v, ql, kl, _, _ = attention_case(TYPES[dtype], 2, 2, 140, 300, 64, "head", False, 6)
    q, k = q.abs() + 0.1, k
    k[0, :, :130] = -math.inf  # all of q is positive: -inf, the first block of keys whole
    v[1, 1, 5, 3] = math.nan
    out, lse = run_forward(vk, q, k, v, None, None)
    want, bound, _, _ = forward_reference(q[:1], k[:1, :, 130:], v[:1, :, 130:], ql[:1], [170], 0.125)
    within(out[:1], want, bound, "out")
    assert torch.isfinite(out[1, 0]).all() and torch.isnan(out[1, 1, :, 3]).all() and torch.isfinite(lse).all()


def test_attention_gradient_by_differences(vk):
    """d/dt of sum(out * g) along a direction, by central differences in 64 bits."""
    q, k, v, ql, kl, _, _ = attention_case(torch.float32, 1, 2, 40, 50, 32, "head", False, 7)
    g = make((1, 2, 40, 32), torch.float32, gen(8))
    out, lse = run_forward(vk, q, k, v, None, None)
    grads = run_backward(vk, q, k, v, out, lse, g, None, None)

    def loss(q, k, v):
        return (torch.softmax(q @ k.transpose(-1, -2) * 32 ** -0.5, -1) @ v * g.double()).sum()

    base = [x.double() for x in (q, k, v)]
    for i in range(3):
        direction = torch.randn(base[i].shape, dtype=torch.float64, device="cuda", generator=gen(9 + i))
        t = 1e-5
        plus, minus = list(base), list(base)
        plus[i], minus[i] = base[i] + t * direction, base[i] - t * direction
        slope = (loss(*plus) - loss(*minus)) / (2 * t)
        along = (grads[i].double() * direction).sum()
        # the differences are good to t^2; the f32 gradient to about 2^-20 of the sum of its terms' sizes
        assert abs(along - slope) <= 2.0 ** -18 * (grads[i].double() * direction).abs().sum()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_repeats_captures_and_streams(vk, dtype):
    """The same bits on every call, from a replayed graph with new inputs, and on another stream."""
    t = TYPES[dtype]
    q, k, v, _, _, _, _ = attention_case(t, 2, 3, 200, 333, 64, "token", False, 10)
    g = make((2, 3, 200, 64), t, gen(11))
    ql, kl = lens([200, 77]), lens([333, 140])

    def both():
        out, lse = run_forward(vk, q, k, v, ql, kl)
        return (out, lse, *run_backward(vk, q, k, v, out, lse, g, ql, kl))

    first, again = both(), both()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        held2 = both()
    q.copy_(make(q.shape, t, gen(12)))
    kl.copy_(lens([50, 333]))
    graph.replay()
    second.replay()
    graph.replay()
    torch.cuda.synchronize()
    fresh = both()
    assert all(torch.equal(a, b) for a, b in zip(held, fresh))
    assert all(torch.equal(a, b) for a, b in zip(held2, fresh))
    assert not torch.equal(fresh[0], first[0])


def test_attention_on_a_context_of_its_own(vk):
    """With a ctx the call runs on the context's stream, and delta is the caller's."""
    q, k, v, ql, kl, _, _ = attention_case(torch.bfloat16, 1, 2, 100, 100, 64, "head", False, 13)
    want = run_forward(vk, q, k, v, None, None)
    ctx = vk.Context(0)
    out, lse = torch.empty_like(q), torch.empty(1, 2, 100, device="cuda")
    torch.cuda.synchronize()
    vk.attention_forward(q, k, v, out, lse, ctx=ctx)
    ctx.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    grads = [torch.empty_like(q) for _ in range(3)]
    with pytest.raises(ValueError):
        vk.attention_backward(q, k, v, out, lse, q, *grads, ctx=ctx)
    delta = torch.empty(1, 2, 100, device="cuda")
    torch.cuda.synchronize()
    vk.attention_backward(q, k, v, out, lse, q, *grads, delta=delta, ctx=ctx)
    ctx.synchronize()
    assert torch.equal(grads[0], run_backward(vk, q, k, v, out, lse, q, None, None)[0])
    # d products and the store, in f32
    bound = 65 * U32 * (q.double() * out.double()).abs().sum(-1)
    within(delta, (q.double() * out.double()).sum(-1), bound, "delta")


def test_attention_past_32_bit_offsets(vk):
    """A batch entry that starts past 2^31 elements: queries, keys, outputs and gradients."""
    n, h, d = 70, 2, 64
    step = 2 ** 31 + 512
    big = torch.empty(step + h * n * d, dtype=torch.bfloat16, device="cuda")
    far = big.as_strided((2, h, n, d), (step, n * d, d, 1))
    q = make((2, h, n, d), torch.bfloat16, gen(14))
    want, want_lse = run_forward(vk, q, q, q, None, None)
    far.copy_(q)
    out, lse = run_forward(vk, far, far, far, None, None)
    assert torch.equal(out, want)
    grads = run_backward(vk, q, q, q, want, want_lse, q, None, None)
    far.fill_(5.0)
    dk, dv = torch.empty_like(q), torch.empty_like(q)
    vk.attention_backward(q, q, q, want, want_lse, q, far, dk, dv)
    assert torch.equal(far, grads[0])
    far.fill_(5.0)
    dq = torch.empty_like(q)
    vk.attention_backward(q, q, q, want, want_lse, q, dq, far, dv)
    assert torch.equal(far, grads[1]) and torch.equal(dv, grads[2])


def test_attention_refusals(vk):
    q, k, v, _, _, _, _ = attention_case(torch.bfloat16, 2, 2, 30, 40, 64, "head", False, 15)
    out, lse = torch.empty_like(q), torch.empty(2, 2, 30, device="cuda")

    def refused(error, *a, **kw):
        before = out.clone()
        with pytest.raises(error):
            vk.attention_forward(*a, **kw)
        assert torch.equal(out, before)

    out.fill_(3.0)
    refused(TypeError, q.cpu(), k, v, out, lse)
    refused(TypeError, q.half(), k.half(), v.half(), out.half(), lse)
    refused(TypeError, q, k.float(), v, out, lse)
    refused(TypeError, q, k, v, out, lse.double())
    refused(ValueError, q, k, v[:, :, :39], out, lse)
    refused(ValueError, q, k, v, out, lse[:, :, :29])
    refused(ValueError, q[0], k, v, out, lse)
    refused(ValueError, q[..., ::2], k[..., ::2], v[..., ::2], out[..., ::2], lse)
    refused(ValueError, q, k, v, out, lse, q_lens=lens([1, 2, 3]))
    refused(TypeError, q, k, v, out, lse, kv_lens=lens([1, 2]).long())
    refused(vk.VestraError, q, k, v, out, lse, scale=0.0)
    refused(vk.VestraError, q, k, v, out, lse, scale=math.nan)
    refused(vk.VestraError, q, k, v, q, lse)
    refused(vk.VestraError, q, k[:1].expand(2, 2, 40, 64), v, out, lse)  # one place for two batch entries
    odd = torch.empty(2 * 2 * 40 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 2, 40, 64)
    refused(vk.VestraError, q, odd, v, out, lse)
    wide = torch.empty(2, 2, 40, 68, dtype=torch.bfloat16, device="cuda")[..., :64]  # rows of 136 bytes
    refused(vk.VestraError, q, wide, v, out, lse)
    with pytest.raises(vk.VestraError) as e:
        x = torch.empty(1, 1, 4, 24, device="cuda")
        vk.attention_forward(x, x, x, torch.empty_like(x), torch.empty(1, 1, 4, device="cuda"))
    assert e.value.status == vk.VK_UNSUPPORTED_SHAPE
    d = torch.empty_like(q)
    dk, dv = torch.empty_like(k), torch.empty_like(v)
    for bad in ((q, dk, dv), (d, k, dv), (d, dk, dk), (dk, d, dv)):
        with pytest.raises((vk.VestraError, ValueError)):
            vk.attention_backward(q, k, v, out, lse, out, *bad)


# ------------------------------------------------------------------ rotary positions
def rope_reference(x, pos, sections, freq, inverse):
    y, at = x.double().clone(), 0
    p = pos if pos.dim() == 3 else pos[None]
    for a, w in enumerate(sections):
        i = torch.arange(w // 2, dtype=torch.float64, device="cuda")
        angle = p[..., a, None].double() * float(freq) ** (-2.0 * i / w) if w else p[..., a, None].double()[..., :0]
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        if inverse:
            s = -s
        lo, hi = x[..., at:at + w // 2].double(), x[..., at + w // 2:at + w].double()
        y[..., at:at + w // 2], y[..., at + w // 2:at + w] = lo * c - hi * s, hi * c + lo * s
        at += w
    return y


def rope_bound(x, y, far):
    """sin and cos of the reduced angle: its rounding to f32 (2^-24 pi), 2 ulp of the functions, `far` for the double
    products of distant positions; two products and a sum; the store."""
    size = x.double().abs().amax(-1, keepdim=True)
    return (math.pi * U32 + 4 * U32 + far + 4 * U32) * 2 * size + HALF[x.dtype] * 1.01 * y.abs()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("b,h,n,d,sections,layout,own,inverse", [
    (1, 12, 865, 64, (32, 32), "head", False, False), (2, 3, 37, 64, (16, 24, 24), "token", True, True),
    (1, 1, 1, 8, (2, 2, 4), "head", False, False), (3, 2, 5, 100, (6, 18, 10, 2), "token", True, False),
    (2, 2, 9, 64, (64,), "head", False, True), (1, 2, 7, 66, (0, 20), "token", False, False), (1, 1, 3, 256, (128, 128), "head", False, False),
    (1, 5, 6, 7, (2, 4), "head", True, False),
])
def test_rope_axes(vk, dtype, b, h, n, d, sections, layout, own, inverse):
    t, g = TYPES[dtype], gen(20)
    q, k = make((b, h, n, d), t, g, layout), make((b, h, n, d), t, g, layout)
    shape = (b, n, len(sections)) if own else (n, len(sections))
    pos = torch.randint(-50, 5000, shape, device="cuda", generator=g)
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    vk.rope_axes(q, k, pos, sections, 100.0, qo, ko, inverse=inverse)
    for x, y in ((q, qo), (k, ko)):
        want = rope_reference(x, pos, sections, 100.0, inverse)
        within(y, want, rope_bound(x, want, 5000 * 2.0 ** -51), "rotated")
        rest = sum(sections)
        assert torch.equal(y[..., rest:], x[..., rest:])
    alone = torch.empty_like(q)
    vk.rope_axes(q, None, pos, sections, 100.0, alone, None, inverse=inverse)
    assert torch.equal(alone, qo)
    vk.rope_axes(q, k, pos, sections, 100.0, q, k, inverse=inverse)  # in place
    assert torch.equal(q, qo) and torch.equal(k, ko)


def test_rope_axes_far_positions_and_back(vk):
    g = gen(21)
    q = make((1, 4, 50, 64), torch.float32, g)
    pos = torch.randint(-2 ** 40, 2 ** 40, (50, 3), device="cuda", generator=g)
    y, z = torch.empty_like(q), torch.empty_like(q)
    vk.rope_axes(q, None, pos, (16, 24, 24), 100.0, y, None)
    # a product of two doubles, one of them rounded itself: 2^-52 of an angle below 2^40
    within(y, rope_reference(q, pos, (16, 24, 24), 100.0, False), rope_bound(q, y.double(), 2.0 ** -11), "far")
    vk.rope_axes(y, None, pos, (16, 24, 24), 100.0, z, None, inverse=True)
    # forwards and back: twice the bound, the angles being the same
    within(z, q.double(), 2 * rope_bound(q, q.double(), 0.0), "back")


def test_rope_axes_is_rope2d_for_two_halves(vk):
    """(y, x) sections of half a head each are the reference's rule (its tables are f32: positions below 64 here)."""
    g = gen(22)
    q = make((1, 3, 60, 64), torch.float32, g)
    pos = torch.randint(0, 64, (60, 2), device="cuda", generator=g)
    y, x = torch.empty_like(q), q.clone().view(-1)
    vk.rope_axes(q, None, pos, (32, 32), 100.0, y, None)
    vk.rope2d(x, 3, 60, 64, pos.view(-1), 100.0)
    # the reference's angle is an f32 product of an f32 power: 64 (1 + 1 + 1) 2^-24 off at most, powf within 2 ulp
    within(x.view_as(y), y.double(), rope_bound(q, y.double(), 64 * 6 * U32), "rope2d")


def test_rope_axes_gradient_by_differences(vk):
    """The inverse is the gradient: <R x, g> = <x, R^-1 g>."""
    gx = gen(23)
    x, g = make((1, 2, 30, 64), torch.float32, gx), make((1, 2, 30, 64), torch.float32, gx)
    pos = torch.randint(0, 500, (30, 3), device="cuda", generator=gx)
    y, back = torch.empty_like(x), torch.empty_like(x)
    vk.rope_axes(x, None, pos, (16, 24, 24), 100.0, y, None)
    vk.rope_axes(g, None, pos, (16, 24, 24), 100.0, back, None, inverse=True)
    left, right = (y.double() * g.double()).sum(), (x.double() * back.double()).sum()
    assert abs(left - right) <= 24 * U32 * (x.abs().double().sum() * g.abs().max().double()).item()


def test_rope_axes_capture_and_refusals(vk):
    q = make((2, 3, 20, 64), torch.bfloat16, gen(24))
    pos = torch.randint(0, 99, (20, 2), device="cuda", generator=gen(25))
    out, graph = torch.empty_like(q), torch.cuda.CUDAGraph()
    vk.rope_axes(q, None, pos, (32, 32), 100.0, out, None)
    with torch.cuda.graph(graph):
        vk.rope_axes(q, None, pos, (32, 32), 100.0, out, None)
    pos.add_(3)
    graph.replay()
    held = out.clone()
    vk.rope_axes(q, None, pos, (32, 32), 100.0, out, None)
    assert torch.equal(held, out)
    for sections, error in (((33, 31), vk.VestraError), ((32, 34), vk.VestraError), ((), ValueError), ((4,) * 5, ValueError)):
        with pytest.raises(error):
            vk.rope_axes(q, None, pos if len(sections) == 2 else pos[:, :1].expand(20, max(1, len(sections))).contiguous(), sections,
                         100.0, out, None)
    for freq in (0.0, -1.0, math.inf):
        with pytest.raises(vk.VestraError):
            vk.rope_axes(q, None, pos, (32, 32), freq, out, None)
    with pytest.raises(ValueError):
        vk.rope_axes(q, q, pos, (32, 32), 100.0, out, None)
    with pytest.raises(vk.VestraError):
        vk.rope_axes(q, q.clone(), pos, (32, 32), 100.0, out, out)
    with pytest.raises(vk.VestraError):
        k = q.clone()
        vk.rope_axes(q, k, pos, (32, 32), 100.0, k, out)
    with pytest.raises(TypeError):
        vk.rope_axes(q, None, pos.int(), (32, 32), 100.0, out, None)
    with pytest.raises(vk.VestraError):
        x = torch.empty(1, 1, 2, 258, device="cuda")
        vk.rope_axes(x, None, pos[:2], (2, 2), 100.0, torch.empty_like(x), None)
    empty = torch.empty(2, 3, 0, 64, device="cuda")
    vk.rope_axes(empty, None, pos[:0], (32, 32), 100.0, empty, None)


# ------------------------------------------------------------------ residual step between two norms
NORMS = [  # stream, branch, groups, rows, cols, scale, gate, post, d_h
    ("f32", "bf16", 1, 1, 768, True, False, False, True), ("f32", "bf16", 3, 37, 768, True, True, True, True),
    ("bf16", "bf16", 2, 50, 384, True, True, False, True), ("f32", "f32", 2, 19, 1024, False, True, True, True),
    ("f32", "f32", 1, 130, 33, True, True, True, True), ("bf16", "bf16", 5, 7, 1001, False, False, True, False),
    ("f32", "bf16", 1, 600, 256, True, False, False, True), ("f32", "f32", 4, 3, 1, True, True, False, True),
    ("bf16", "bf16", 1, 21, 2048, True, True, True, True), ("f32", "bf16", 2, 5, 4104, True, False, True, True),
    ("f32", "f32", 1, 9, 8192, True, True, True, True), ("f32", "f32", 1, 6, 8191, True, True, True, False),
    ("f32", "bf16", 2, 433, 768, True, True, True, False), ("f32", "bf16", 70, 2, 128, True, True, False, True),
    ("f32", "bf16", 1, 11, 512, True, False, True, True), ("bf16", "bf16", 1, 11, 100, False, False, False, True),
    # more rows than blocks have at once, of one warp and of four, with pieces of eight and of one
    ("f32", "bf16", 4, 3501, 72, True, True, True, True), ("bf16", "bf16", 2, 1701, 1104, True, True, False, True),
    ("f32", "f32", 3, 1100, 201, True, False, True, True),
]


def norm_inputs(stream, branch, groups, rows, cols, scale, gate, post, seed):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    s = {"x": r(groups, rows, cols).mul_(2).to(TYPES[stream]), "branch": r(groups, rows, cols).add_(0.3).to(TYPES[branch]),
         "gamma": r(cols) * 0.3 + 1, "beta": r(cols), "scale": r(cols) if scale else None,
         "gate": r(groups, cols) if gate else None, "post_gamma": r(cols) * 0.3 + 1 if post else None,
         "post_beta": r(cols) if post else None}
    return s


EPS = 1e-6


def standard64(x):
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + EPS)
    return (x - mean) * rstd, mean, rstd


def hat_error(x, mean, rstd, dx):
    """Bound of the error of (x - mean) rstd in f32, x itself off by dx: the mean (a sum of c values, in a tree or a
    chain of at most c / 32 + 8), the difference, the variance (the same sum of squares, halved by the root)."""
    c = x.shape[-1]
    chain = (c / 32 + 10) * U32
    d_mean = chain * x.abs().mean(-1, keepdim=True) + dx.mean(-1, keepdim=True)
    dev = (x - mean).abs()
    d_dev = dx + d_mean + U32 * dev
    rel_var = (chain + 4 * U32) + 2 * (dev * d_dev).mean(-1, keepdim=True) * rstd ** 2
    return d_dev * rstd * 1.01 + dev * rstd * (rel_var + 4 * U32), d_mean, rstd * (rel_var + 4 * U32)


def run_norm(vk, s):
    h, y = torch.full_like(s["x"], 7.0), torch.full_like(s["branch"], 7.0)
    stats = torch.full((*h.shape[:2], 2), 7.0, device="cuda")
    post = torch.full((*h.shape[:2], 2), 7.0, device="cuda") if s["post_gamma"] is not None else None
    vk.residual_norm_forward(s["x"], s["branch"], s["gamma"], s["beta"], EPS, h, y, stats, scale=s["scale"], gate=s["gate"],
                             post_gamma=s["post_gamma"], post_beta=s["post_beta"], post_stats=post)
    return h, y, stats, post


@pytest.mark.parametrize("stream,branch,groups,rows,cols,scale,gate,post,dh", NORMS)
def test_residual_norm_forward(vk, stream, branch, groups, rows, cols, scale, gate, post, dh):
    s = norm_inputs(stream, branch, groups, rows, cols, scale, gate, post, 30)
    h, y, stats, post_stats = run_norm(vk, s)
    n = s["branch"].double()
    n_err = torch.zeros_like(n)
    if post:
        hat, mean, rstd = standard64(n)
        e, e_mean, e_rstd = hat_error(n, mean, rstd, n_err)
        within(post_stats[..., :1], mean, e_mean, "post mean")
        within(post_stats[..., 1:], rstd, e_rstd, "post rstd")
        n = hat * s["post_gamma"].double() + s["post_beta"].double()
        n_err = e * s["post_gamma"].double().abs() + 2 * U32 * (n.abs() + (hat * s["post_gamma"].double()).abs())
    f = torch.ones_like(n)
    if scale:
        f = f * s["scale"].double()
    if gate:
        f = f * s["gate"].double()[:, None]
    want_h = s["x"].double() + f * n
    h_err = f.abs() * (n_err + 2 * U32 * n.abs()) * 1.01 + U32 * want_h.abs()
    within(h, want_h, h_err + HALF[TYPES[stream]] * 1.01 * want_h.abs(), "h")
    hat, mean, rstd = standard64(want_h)
    e, e_mean, e_rstd = hat_error(want_h, mean, rstd, h_err)
    within(stats[..., :1], mean, e_mean + 1e-12, "mean")
    within(stats[..., 1:], rstd, e_rstd, "rstd")
    want_y = hat * s["gamma"].double() + s["beta"].double()
    y_err = e * s["gamma"].double().abs() + 2 * U32 * (want_y.abs() + (hat * s["gamma"].double()).abs())
    within(y, want_y, y_err + HALF[TYPES[branch]] * 1.01 * want_y.abs(), "y")
    # in place on the stream: the same bits
    x = s["x"].clone()
    y2, st2 = torch.empty_like(y), torch.empty_like(stats)
    vk.residual_norm_forward(x, s["branch"], s["gamma"], s["beta"], EPS, x, y2, st2, scale=s["scale"], gate=s["gate"],
                             post_gamma=s["post_gamma"], post_beta=s["post_beta"], post_stats=post_stats)
    assert torch.equal(x, h) and torch.equal(y2, y)


def run_norm_backward(vk, s, h, stats, post_stats, d_h, d_y, **kw):
    grads = {"d_x": torch.full_like(h, 7.0), "d_branch": torch.full_like(s["branch"], 7.0)}
    for name in ("gamma", "beta", "scale", "gate", "post_gamma", "post_beta"):
        if s[name] is not None:
            grads["d_" + name] = torch.full_like(s[name], 7.0)
    grads.update(kw)
    vk.residual_norm_backward(d_h, d_y, h, s["branch"], stats, s["gamma"], scale=s["scale"], gate=s["gate"],
                              post_gamma=s["post_gamma"], post_beta=s["post_beta"], post_stats=post_stats, **grads)
    return grads


def norm_backward_reference(s, h, stats, post_stats, d_h, d_y):
    """Gradients in 64 bits and their bounds: products and sums of a row (a chain of at most c / 32 + 10), then column
    sums of r rows (a chain of at most r), in f32, and the stores."""
    c, r = h.shape[-1], h.shape[0] * h.shape[1]
    row, column = (c / 32 + 16) * U32, (r + 16) * U32
    mean, rstd = stats.double().unbind(-1)
    mean, rstd = mean[..., None], rstd[..., None]

    def through(t, t_err, hat, hat_err, rstd):
        m0, m1 = t.mean(-1, keepdim=True), (t * hat).mean(-1, keepdim=True)
        size = t.abs() + t.abs().mean(-1, keepdim=True) + hat.abs() * (t * hat).abs().mean(-1, keepdim=True)
        e = t_err + t_err.mean(-1, keepdim=True) + hat.abs() * (t_err * hat.abs() + t.abs() * hat_err).mean(-1, keepdim=True)
        e = e + hat_err * m1.abs() + (row + 6 * U32) * size
        return rstd * (t - m0 - hat * m1), rstd * e * 1.01

    def standard(x, mean, rstd):
        hat = (x - mean) * rstd
        return hat, 2 * U32 * (x - mean).abs() * rstd + U32 * hat.abs()

    want, bound = {}, {}

    def sums(name, terms, errs, dims):
        want[name] = terms.sum(dims)
        bound[name] = errs.sum(dims) * 1.01 + column * terms.abs().sum(dims) + 1e-30

    hat, hat_err = standard(h.double(), mean, rstd)
    g = d_y.double()
    sums("d_gamma", g * hat, g.abs() * (hat_err + U32 * hat.abs()), (0, 1))
    sums("d_beta", g, 0 * g, (0, 1))
    t = g * s["gamma"].double()
    dh, dh_err = through(t, U32 * t.abs(), hat, hat_err, rstd)
    if d_h is not None:
        dh = dh + d_h.double()
    dh_err = dh_err + 2 * U32 * dh.abs()
    want["d_x"], bound["d_x"] = dh, dh_err + HALF[h.dtype] * 1.01 * dh.abs()
    n = s["branch"].double()
    n_err = 0 * n
    if s["post_gamma"] is not None:
        pm, pr = post_stats.double().unbind(-1)
        b_hat, b_err = standard(n, pm[..., None], pr[..., None])
        n = b_hat * s["post_gamma"].double() + s["post_beta"].double()
        n_err = b_err * s["post_gamma"].double().abs() + 2 * U32 * (n.abs() + (b_hat * s["post_gamma"].double()).abs())
    one = torch.ones_like(n[:, :1])
    scale = one if s["scale"] is None else one * s["scale"].double()
    gate = one if s["gate"] is None else s["gate"].double()[:, None]
    terms, errs = dh * n, dh_err * n.abs() + dh.abs() * n_err + U32 * (dh * n).abs()
    if s["scale"] is not None:
        sums("d_scale", terms * gate, (errs + 2 * U32 * terms.abs()) * gate.abs(), (0, 1))
    if s["gate"] is not None:
        sums("d_gate", terms * scale, (errs + 2 * U32 * terms.abs()) * scale.abs(), 1)
    dn = dh * scale * gate
    dn_err = (dh_err + 3 * U32 * dh.abs()) * (scale * gate).abs()
    if s["post_gamma"] is not None:
        sums("d_post_gamma", dn * b_hat, dn_err * b_hat.abs() + dn.abs() * (b_err + U32 * b_hat.abs()), (0, 1))
        sums("d_post_beta", dn, dn_err, (0, 1))
        u = dn * s["post_gamma"].double()
        u_err = dn_err * s["post_gamma"].double().abs() + U32 * u.abs()
        dn, dn_err = through(u, u_err, b_hat, b_err, pr[..., None])
        dn_err = dn_err + 2 * U32 * dn.abs()
    want["d_branch"], bound["d_branch"] = dn, dn_err + HALF[s["branch"].dtype] * 1.01 * dn.abs()
    return want, bound


@pytest.mark.parametrize("stream,branch,groups,rows,cols,scale,gate,post,dh", NORMS)
def test_residual_norm_backward(vk, stream, branch, groups, rows, cols, scale, gate, post, dh):
    s = norm_inputs(stream, branch, groups, rows, cols, scale, gate, post, 31)
    h, y, stats, post_stats = run_norm(vk, s)
    g = gen(32)
    d_y = torch.randn(y.shape, device="cuda", generator=g).to(y.dtype)
    d_h = torch.randn(h.shape, device="cuda", generator=g).to(h.dtype) if dh else None
    grads = run_norm_backward(vk, s, h, stats, post_stats, d_h, d_y)
    want, bound = norm_backward_reference(s, h, stats, post_stats, d_h, d_y)
    assert set(grads) == set(want)
    for name in want:
        within(grads[name], want[name], bound[name] + 1e-30, name)
    again = run_norm_backward(vk, s, h, stats, post_stats, d_h, d_y)
    assert all(torch.equal(grads[x], again[x]) for x in grads)
    # in place on the gradients: the same bits
    dy2, dh2 = d_y.clone(), d_h.clone() if dh else torch.empty_like(h)
    placed = run_norm_backward(vk, s, h, stats, post_stats, dh2 if dh else None, dy2, d_x=dh2, d_branch=dy2)
    assert all(torch.equal(grads[x], placed[x]) for x in grads)


def test_residual_norm_gradient_by_differences(vk):
    s = norm_inputs("f32", "f32", 2, 5, 40, True, True, True, 33)
    g = gen(34)
    w_h, w_y = (torch.randn(2, 5, 40, device="cuda", generator=g) for _ in range(2))
    h, y, stats, post_stats = run_norm(vk, s)
    grads = run_norm_backward(vk, s, h, stats, post_stats, w_h, w_y)

    def loss(s):
        n = standard64(s["branch"])[0] * s["post_gamma"] + s["post_beta"]
        h = s["x"] + s["scale"] * s["gate"][:, None] * n
        return (h * w_h.double()).sum() + ((standard64(h)[0] * s["gamma"] + s["beta"]) * w_y.double()).sum()

    base = {k: v.double() for k, v in s.items()}
    for name in base:
        direction = torch.randn(base[name].shape, dtype=torch.float64, device="cuda", generator=g)
        t = 1e-5
        slope = (loss({**base, name: base[name] + t * direction}) - loss({**base, name: base[name] - t * direction})) / (2 * t)
        terms = grads["d_" + name].double() * direction
        assert abs(terms.sum() - slope) <= 2.0 ** -17 * terms.abs().sum() + 1e-7, name


def test_residual_norm_empty_capture_and_refusals(vk):
    s = norm_inputs("f32", "bf16", 2, 40, 256, True, True, True, 35)
    h, y, stats, post_stats = run_norm(vk, s)
    d_y = torch.randn(y.shape, device="cuda", generator=gen(36)).to(y.dtype)
    want = run_norm_backward(vk, s, h, stats, post_stats, None, d_y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run_norm_backward(vk, s, h, stats, post_stats, None, d_y)
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        run_norm_backward(vk, s, h, stats, post_stats, None, d_y)
    other.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(want[x], held[x]) for x in want)
    none = {**norm_inputs("f32", "bf16", 2, 0, 256, True, True, True, 37)}
    h0, y0, st0, ps0 = run_norm(vk, none)
    zero = run_norm_backward(vk, none, h0, st0, ps0, None, y0)
    assert all((zero[x] == 0).all() for x in zero)

    def refused(error, **kw):
        a = dict(x=s["x"], branch=s["branch"], gamma=s["gamma"], beta=s["beta"], eps=EPS, h=h, y=y, stats=stats, scale=s["scale"],
                 gate=s["gate"], post_gamma=s["post_gamma"], post_beta=s["post_beta"], post_stats=post_stats)
        a.update(kw)
        with pytest.raises(error):
            vk.residual_norm_forward(**a)

    refused(ValueError, gamma=s["gamma"][:-1])
    refused(TypeError, beta=s["beta"].bfloat16())
    refused(ValueError, gate=s["gate"][:1])
    refused(vk.VestraError, post_beta=None)
    refused(vk.VestraError, post_stats=None)
    refused(vk.VestraError, eps=math.nan)
    refused(vk.VestraError, eps=-1.0)
    refused(ValueError, x=s["x"].transpose(0, 1), h=h.transpose(0, 1), branch=s["branch"].transpose(0, 1), y=y.transpose(0, 1))
    refused(vk.VestraError, x=s["x"].bfloat16(), h=h.bfloat16(), branch=s["branch"].float(), y=y.float())
    refused(vk.VestraError, y=s["branch"])
    refused(TypeError, x=s["x"].half(), h=h.half())
    with pytest.raises(vk.VestraError) as e:
        wide = norm_inputs("f32", "f32", 1, 2, 8200, False, False, False, 38)
        run_norm(vk, wide)
    assert e.value.status == vk.VK_UNSUPPORTED_SHAPE
    with pytest.raises(vk.VestraError):
        run_norm_backward(vk, s, h, stats, post_stats, None, d_y, d_scale=None)
    with pytest.raises(vk.VestraError):
        run_norm_backward(vk, s, h, stats, post_stats, None, d_y, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        run_norm_backward(vk, s, h, stats, post_stats, None, d_y, ctx=vk.Context(0))


def test_residual_norm_in_place_and_at_odd_addresses(vk):
    """h written over x and the gradients over d_h and d_y, with more rows than blocks have at once: the same bits.
    Matrices that start 4 or 2 bytes off take another path; it sums in another order, within a few roundings."""
    s = norm_inputs("f32", "bf16", 3, 4001, 136, True, True, True, 50)
    h, y, stats, post_stats = run_norm(vk, s)
    g = gen(51)
    d_h, d_y = torch.randn(h.shape, device="cuda", generator=g), torch.randn(y.shape, device="cuda", generator=g).bfloat16()
    want = run_norm_backward(vk, s, h, stats, post_stats, d_h, d_y)
    x, y2 = s["x"].clone(), torch.empty_like(y)
    vk.residual_norm_forward(x, s["branch"], s["gamma"], s["beta"], EPS, x, y2, torch.empty_like(stats), scale=s["scale"],
                             gate=s["gate"], post_gamma=s["post_gamma"], post_beta=s["post_beta"],
                             post_stats=torch.empty_like(post_stats))
    assert torch.equal(x, h) and torch.equal(y2, y)
    dh2, dy2 = d_h.clone(), d_y.clone()
    got = run_norm_backward(vk, s, h, stats, post_stats, dh2, dy2, d_x=dh2, d_branch=dy2)
    assert all(torch.equal(got[n], want[n]) for n in want)

    def off(t):  # the same values, one element further
        return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

    moved = {n: (v if v is None else off(v)) for n, v in s.items()}
    h3, y3, stats3, post3 = run_norm(vk, moved)
    # h: a norm whose two sums of 136 and few products round differently, then three products and a sum
    within(h3, h, 2.0 ** -24 * (2 * 136 + 16) * (1 + h.abs() + s["x"].abs()).double() * 4, "h")
    got = run_norm_backward(vk, moved, off(h), stats, post_stats, off(d_h), off(d_y))
    # the same formulas on the same values: sums of 136 in another order, of terms no larger than the largest
    most = want["d_x"].abs().amax().double()
    within(got["d_x"], want["d_x"], 2.0 ** -24 * 4 * 136 * most, "d_x")


def test_residual_norm_refuses_shared_vectors(vk):
    s = norm_inputs("f32", "bf16", 2, 40, 256, True, True, True, 52)
    h, y, stats, post_stats = run_norm(vk, s)
    with pytest.raises(vk.VestraError):
        vk.residual_norm_forward(s["x"], s["branch"], s["gamma"], s["beta"], EPS, h, y, stats, post_gamma=s["post_gamma"],
                                 post_beta=s["post_beta"], post_stats=stats)
    for name in ("scale", "gate", "post_gamma"):
        with pytest.raises(vk.VestraError):
            run_norm_backward(vk, s, h, stats, post_stats, None, y, **{"d_" + name: s[name]})


def test_two_threads_on_streams_of_their_own(vk):
    """Calls without a ctx from two threads at once: each goes to its thread's stream, and none reports an error."""
    import threading

    inputs = [attention_case(torch.bfloat16, 2, 4, 300, 300, 64, "head", False, 60 + i)[:3] for i in range(2)]
    want = [run_forward(vk, *x, None, None) for x in inputs]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(50):
                    got[i] = run_forward(vk, *inputs[i], None, None)
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    vk.synchronize()
    for (out, lse), (w, wl) in zip(got, want):
        assert torch.equal(out, w) and torch.equal(lse, wl)


# ------------------------------------------------------------------ a run of them together
@pytest.mark.parametrize("dtype,tol", [("f32", 2e-5), ("bf16", 3e-2)])
def test_block_forward_and_backward(vk, dtype, tol):
    """A ViT block's attention half on two padded clips -- QKV product, rotary positions over (time, y, x), attention,
    out-projection, residual step with LayerScale and gate into the next norm -- and all its gradients, against
    64-bit automatic differentiation.  The tolerance is of the 2-norm: bf16 rounds about eight tensors on the longest
    path (each 2^-8 at most, 2^-9.2 as a root mean square, amplified by the products with gradients of their own
    rounding); f32 the same path at 2^-24 with sums of at most 256 terms."""
    t, g = TYPES[dtype], gen(40)
    b, h, n, d = 2, 4, 75, 64
    e = h * d
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, res = r(b, n, e).to(t), r(b, n, e).to(t)
    w_qkv, w_out = (r(e, 3 * e) / e ** 0.5).to(t), (r(e, e) / e ** 0.5).to(t)
    gamma, beta, ls, gate = r(e) * 0.1 + 1, r(e) * 0.1, r(e) * 0.1 + 0.5, r(b, e) * 0.1 + 1
    w_h, w_y = (r(b, n, e) * 0.1).to(t), (r(b, n, e) * 0.1).to(t)
    length = lens([n, 50])
    valid = (torch.arange(n, device="cuda") < length[:, None])
    pos = torch.stack([torch.arange(n, device="cuda") // 25, torch.arange(n, device="cuda") % 25 // 5,
                       torch.arange(n, device="cuda") % 5], 1).contiguous()
    sections = (16, 24, 24)
    # forward
    qkv = (x @ w_qkv).view(b, n, 3, h, d)
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    vk.rope_axes(q, k, pos, sections, 100.0, q, k)  # in place, in the QKV product
    att = torch.empty(b, n, h, d, device="cuda", dtype=t)
    lse = torch.empty(b, h, n, device="cuda")
    vk.attention_forward(q, k, v, att.transpose(1, 2), lse, q_lens=length, kv_lens=length)
    branch = att.view(b, n, e) @ w_out
    hid, y, stats = torch.empty_like(res), torch.empty_like(branch), torch.empty(b, n, 2, device="cuda")
    vk.residual_norm_forward(res, branch, gamma, beta, EPS, hid, y, stats, scale=ls, gate=gate)
    # backward
    d_res, d_branch = torch.empty_like(res), torch.empty_like(branch)
    sums = {"d_gamma": torch.empty_like(gamma), "d_beta": torch.empty_like(beta), "d_scale": torch.empty_like(ls),
            "d_gate": torch.empty_like(gate)}
    vk.residual_norm_backward(w_h, w_y, hid, branch, stats, gamma, d_res, d_branch, scale=ls, gate=gate, **sums)
    d_att = (d_branch @ w_out.t()).view(b, n, h, d)
    d_w_out = att.view(b * n, e).t() @ d_branch.view(b * n, e)
    d_qkv = torch.empty_like(qkv)
    dq, dk, dv = (d_qkv[:, :, i].transpose(1, 2) for i in range(3))
    vk.attention_backward(q, k, v, att.transpose(1, 2), lse, d_att.transpose(1, 2), dq, dk, dv, q_lens=length, kv_lens=length)
    vk.rope_axes(dq, dk, pos, sections, 100.0, dq, dk, inverse=True)
    d_x = d_qkv.view(b, n, 3 * e) @ w_qkv.t()
    d_w_qkv = x.view(b * n, e).t() @ d_qkv.view(b * n, 3 * e)
    # the same in 64 bits
    leaves = {"x": x, "res": res, "w_qkv": w_qkv, "w_out": w_out, "gamma": gamma, "beta": beta, "scale": ls, "gate": gate}
    leaf = {a: p.double().requires_grad_() for a, p in leaves.items()}

    def turn(z):
        out, at = [], 0
        for a, w in enumerate(sections):
            angle = pos[:, a, None].double() * 100.0 ** (-2.0 * torch.arange(w // 2, device="cuda", dtype=torch.float64) / w)
            lo, hi = z[..., at:at + w // 2], z[..., at + w // 2:at + w]
            out += [lo * angle.cos() - hi * angle.sin(), hi * angle.cos() + lo * angle.sin()]
            at += w
        return torch.cat(out, -1)

    q64, k64, v64 = (leaf["x"] @ leaf["w_qkv"]).view(b, n, 3, h, d).permute(2, 0, 3, 1, 4)
    score = (turn(q64) @ turn(k64).transpose(-1, -2) * d ** -0.5).masked_fill(~valid[:, None, None], -math.inf)
    a64 = (torch.softmax(score, -1) @ v64) * valid[:, None, :, None]
    branch64 = a64.transpose(1, 2).reshape(b, n, e) @ leaf["w_out"]
    h64 = leaf["res"] + leaf["scale"] * leaf["gate"][:, None] * branch64
    y64 = standard64(h64)[0] * leaf["gamma"] + leaf["beta"]
    ((h64 * w_h.double()).sum() + (y64 * w_y.double()).sum()).backward()
    got = {"x": d_x, "res": d_res, "w_qkv": d_w_qkv, "w_out": d_w_out, "gamma": sums["d_gamma"], "beta": sums["d_beta"],
           "scale": sums["d_scale"], "gate": sums["d_gate"]}
    assert (y.double() - y64).norm() <= tol * y64.norm()
    for name, value in got.items():
        want = leaf[name].grad
        assert (value.double() - want).norm() <= tol * want.norm(), name
