"""The trainable pieces of a ViT block, as measured cases: attention with its
row statistics and its backward pass, rotary positions over several axes, and
the residual step (LayerScale, gate, residual, the norms either side) with its
backward pass.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU,
``run`` makes one pass (plain torch operations, or the framework's operators
where ``own`` is true) and ``exact`` gives the same outputs in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _vk():
    path = os.path.join(os.getcwd(), "vestra-kernels_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import vestra_kernels

    return vestra_kernels


# ------------------------------------------------------------------ the cases
def _attention(op, dtype, batch, heads, q_tokens, kv_tokens, dim=64, layout="token", ragged=False):
    return {"op": op, "dtype": dtype, "batch": batch, "heads": heads, "q_tokens": q_tokens, "kv_tokens": kv_tokens,
            "dim": dim, "layout": layout, "ragged": ragged}


def _rope(dtype, batch, heads, tokens, dim, sections, layout="token", inverse=False, own_positions=False):
    return {"op": "rope", "dtype": dtype, "batch": batch, "heads": heads, "tokens": tokens, "dim": dim,
            "sections": sections, "layout": layout, "inverse": inverse, "own_positions": own_positions}


def _norm(op, stream, branch, groups, tokens, cols, post=False, gate=False):
    return {"op": op, "stream_type": stream, "branch_type": branch, "groups": groups, "tokens": tokens, "cols": cols,
            "post": post, "gate": gate}


def listed():
    return [
        # a few tokens of a thumbnail-sized view: the call's latency
        {"name": "attention, one small view", **_attention("attention", "bf16", 1, 6, 61, 61)},
        # the encoder's headline batch: 64 images of 504x336 (865 tokens), 12 heads, q/k/v slices of one QKV product
        {"name": "attention, 64 images", **_attention("attention", "bf16", 64, 12, 865, 865)},
        # full precision over a padded batch of views of several sizes, head-major
        {"name": "attention, padded f32", **_attention("attention", "f32", 5, 12, 865, 865, layout="head", ragged=True)},
        # a handful of small views in full precision, as a gradient check or a small head would train
        {"name": "attention backward, small f32", **_attention("attention_backward", "f32", 3, 6, 197, 197, layout="head", ragged=True)},
        # the headline batch, trained
        {"name": "attention backward, 64 images", **_attention("attention_backward", "bf16", 64, 12, 865, 865)},
        # cross-view layers: sequences of up to 3457 tokens, padded
        {"name": "attention backward, long views", **_attention("attention_backward", "bf16", 4, 12, 3457, 3457, ragged=True)},
        # one image's queries and keys, (y, x)
        {"name": "rope, one image", **_rope("f32", 1, 12, 865, 64, "32,32", layout="head")},
        # the gradient of a batch of clips, (time, y, x) with every clip's own positions
        {"name": "rope gradient, clips", **_rope("bf16", 16, 12, 3457, 64, "16,24,24", inverse=True, own_positions=True)},
        # one image between two blocks
        {"name": "residual norm, one image", **_norm("norm", "f32", "bf16", 1, 865, 768)},
        # the headline batch between two blocks, with a norm of the branch and a gate per image
        {"name": "residual norm, 64 images", **_norm("norm", "f32", "bf16", 64, 865, 768, post=True, gate=True)},
        # the gradients of a small bf16 batch
        {"name": "residual norm backward, small", **_norm("norm_backward", "bf16", "bf16", 2, 433, 768, gate=True)},
        # the gradients of the headline batch
        {"name": "residual norm backward, 64 images", **_norm("norm_backward", "f32", "bf16", 64, 865, 768, post=True)},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention_backward", "attention_backward", "rope", "norm", "norm_backward"])
    if op.startswith("attention"):
        dtype = rng.choice(["bf16", "bf16", "f32"])
        while True:
            batch, heads, q_tokens = _log(rng, 1, 64), _log(rng, 1, 24), _log(rng, 1, 3500)
            kv_tokens = q_tokens if rng.random() < 0.7 else _log(rng, 1, 3500)
            most = 64 * 12 * 865 * 865 if dtype == "bf16" else 4 * 12 * 865 * 865
            if batch * heads * q_tokens * kv_tokens <= most:
                break
        dim = 64 if dtype == "bf16" else rng.choice([32, 64])
        return _attention(op, dtype, batch, heads, q_tokens, kv_tokens, dim, rng.choice(["token", "head"]), rng.random() < 0.5)
    if op == "rope":
        while True:
            batch, heads, tokens = _log(rng, 1, 64), _log(rng, 1, 24), _log(rng, 1, 8000)
            if batch * heads * tokens <= 16 * 12 * 3457:
                break
        sections = rng.choice(["32,32", "16,24,24", "8,28,28", "16,16,16", "64", "20,20,20", "6,18,10"])
        return _rope(rng.choice(["f32", "bf16"]), batch, heads, tokens, 64, sections, rng.choice(["token", "head"]),
                     rng.random() < 0.5, rng.random() < 0.5)
    while True:
        groups, tokens, cols = _log(rng, 1, 64), _log(rng, 1, 3500), rng.choice([384, 768, 1024, 1536, _log(rng, 33, 2000)])
        if groups * tokens * cols <= 64 * 865 * 768:
            break
    stream, branch = rng.choice([("f32", "bf16"), ("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32")])
    return _norm(op, stream, branch, groups, tokens, cols, rng.random() < 0.5, rng.random() < 0.5)


def _lengths(case):
    """The valid tokens of each sequence of a padded batch: full ones, short ones, now and then an empty one."""
    r = random.Random("%(batch)d %(q_tokens)d %(kv_tokens)d" % case)
    q, k = [], []
    for b in range(case["batch"]):
        share = 1.0 if b == 0 else 0.0 if r.random() < 0.05 else r.uniform(0.2, 1.0)
        q.append(int(round(share * case["q_tokens"])))
        k.append(int(round(share * case["kv_tokens"])))
    return q, k


def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


EPS = 1e-6
FREQ = 100.0


# ------------------------------------------------------------------ inputs
def _heads(case, count, tokens, kind, gen, spread=1.0):
    """`count` tensors [batch, heads, tokens, dim], slices of one product's output (token-major) or apart (head-major)."""
    b, h, d = case["batch"], case["heads"], case["dim"]
    if case["layout"] == "token":
        x = torch.randn(b, tokens, count, h, d, generator=gen, device="cuda").mul_(spread).to(kind)
        return [x[:, :, i].transpose(1, 2) for i in range(count)]
    return [torch.randn(b, h, tokens, d, generator=gen, device="cuda").mul_(spread).to(kind) for _ in range(count)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    s = dict(case)
    op = case["op"]
    if op.startswith("attention"):
        kind = TYPES[case["dtype"]]
        if case["q_tokens"] == case["kv_tokens"]:
            s["q"], s["k"], s["v"] = _heads(case, 3, case["q_tokens"], kind, gen)
        else:
            (s["q"],) = _heads(case, 1, case["q_tokens"], kind, gen)
            s["k"], s["v"] = _heads(case, 2, case["kv_tokens"], kind, gen)
        s["q_lens"] = s["kv_lens"] = None
        if case["ragged"]:
            q, k = _lengths(case)
            s["q_lens"] = torch.tensor(q, dtype=torch.int32, device="cuda")
            s["kv_lens"] = torch.tensor(k, dtype=torch.int32, device="cuda")
        if op == "attention_backward":
            s["out"], s["lse"] = _attention_plain(s)
            (s["d_out"],) = _heads(case, 1, case["q_tokens"], kind, gen, 0.1)
    elif op == "rope":
        kind = TYPES[case["dtype"]]
        s["q"], s["k"] = _heads(case, 2, case["tokens"], kind, gen)
        axes = len(_sections(case))
        # a grid of patches from 1 on, its first axis the frame where there are three
        t = torch.arange(case["tokens"], device="cuda")
        by_axis = [t // 864, t % 864 // 36 + 1, t % 36 + 1] if axes == 3 else [t // 36 + 1, t % 36 + 1] if axes == 2 else [t]
        pos = torch.stack(by_axis, 1)
        if case["own_positions"]:
            pos = pos + torch.randint(0, 50, (case["batch"], 1, axes), generator=gen, device="cuda")
        s["positions"] = pos.to(torch.int64).contiguous()
        s["low"], s["high"] = _pairs(s)
    else:
        g, t, c = case["groups"], case["tokens"], case["cols"]
        stream, branch = TYPES[case["stream_type"]], TYPES[case["branch_type"]]
        s["x"] = normal(g, t, c).mul_(2.0).to(stream)
        s["branch"] = normal(g, t, c).add_(0.1).to(branch)
        s["gamma"], s["beta"] = normal(c).mul_(0.1).add_(1.0), normal(c).mul_(0.1)
        s["scale"] = normal(c).mul_(0.1).add_(0.5)
        s["gate"] = normal(g, c).mul_(0.2).add_(1.0) if case["gate"] else None
        s["post_gamma"] = normal(c).mul_(0.1).add_(1.0) if case["post"] else None
        s["post_beta"] = normal(c).mul_(0.1) if case["post"] else None
        if op == "norm_backward":
            s["h"], _, s["stats"], s["post_stats"] = _norm_plain(s)
            del s["x"]
            s["d_h"] = normal(g, t, c).mul_(0.1).to(stream)
            s["d_y"] = normal(g, t, c).mul_(0.1).to(branch)
    return s


# ------------------------------------------------------------------ plain forms
def _masked(s):
    """(probabilities, lse): rows past the lengths have no probabilities and lse -inf."""
    scores = torch.matmul(s["q"].float(), s["k"].float().transpose(-1, -2)) * (1.0 / math.sqrt(s["dim"]))
    if s["kv_lens"] is not None:
        scores = scores.masked_fill(~_valid(s, "kv")[:, None, None, :], -math.inf)
        scores = scores.masked_fill(~_valid(s, "q")[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total), (top + torch.log(total)).squeeze(-1)


def _valid(s, side):
    return torch.arange(s[side + "_tokens"], device="cuda") < s[side + "_lens"][:, None]


def _like(s, x):
    """x [batch, heads, tokens, dim] in the operator's type, in the layout of its inputs."""
    x = x.to(TYPES[s["dtype"]])
    return x.transpose(1, 2).contiguous().transpose(1, 2) if s["layout"] == "token" else x.contiguous()


def _attention_plain(s):
    p, lse = _masked(s)
    return _like(s, torch.matmul(p, s["v"].float())), lse


def _attention_backward_plain(s):
    scale = 1.0 / math.sqrt(s["dim"])
    scores = torch.matmul(s["q"].float(), s["k"].float().transpose(-1, -2)) * scale
    lse = s["lse"][..., None]
    p = torch.exp(scores - torch.where(lse == -math.inf, torch.zeros_like(lse), lse))
    d_out = s["d_out"].float()
    if s["kv_lens"] is not None:
        ok = _valid(s, "kv")[:, None, None, :] & _valid(s, "q")[:, None, :, None]
        p = p.masked_fill(~ok, 0.0)
    del scores
    dv = torch.matmul(p.transpose(-1, -2), d_out)
    delta = (d_out * s["out"].float()).sum(-1, keepdim=True)
    ds = p * (torch.matmul(d_out, s["v"].float().transpose(-1, -2)) - delta)
    del p
    dq = torch.matmul(ds, s["k"].float()) * scale
    dk = torch.matmul(ds.transpose(-1, -2), s["q"].float()) * scale
    return _like(s, dq), _like(s, dk), _like(s, dv)


def _angles(s):
    """[tokens] or [batch, tokens] angles of each axis' pairs, side by side, in 64 bits."""
    parts = []
    for axis, width in enumerate(_sections(s)):
        inv = FREQ ** (-2.0 * torch.arange(width // 2, device="cuda", dtype=torch.float64) / width)
        parts.append(s["positions"][..., axis, None].double() * inv)
    return torch.cat(parts, -1)


def _pairs(s):
    low, high, at = [], [], 0
    for width in _sections(s):
        low += range(at, at + width // 2)
        high += range(at + width // 2, at + width)
        at += width
    return torch.tensor(low, device="cuda"), torch.tensor(high, device="cuda")


def _rope_plain(s):
    angle = _angles(s)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if s["inverse"]:
        sin = -sin
    if cos.dim() == 3:
        cos, sin = cos[:, None], sin[:, None]
    low, high = s["low"], s["high"]
    outs = []
    for x in (s["q"], s["k"]):
        a, b = x[..., low].float(), x[..., high].float()
        y = x.clone()
        y[..., low] = (a * cos - b * sin).to(x.dtype)
        y[..., high] = (b * cos + a * sin).to(x.dtype)
        outs.append(y)
    return tuple(outs)


def _standard(x):
    mean = x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + EPS)
    return (x - mean) * rstd, torch.cat([mean, rstd], -1)


def _norm_plain(s):
    n, post_stats = s["branch"].float(), None
    if s["post"]:
        n, post_stats = _standard(n)
        n = n * s["post_gamma"] + s["post_beta"]
    n = n * s["scale"]
    if s["gate"] is not None:
        n = n * s["gate"][:, None]
    h = s["x"].float() + n
    y, stats = _standard(h)
    y = y * s["gamma"] + s["beta"]
    return h.to(TYPES[s["stream_type"]]), y.to(TYPES[s["branch_type"]]), stats, post_stats


def _norm_backward_plain(s):
    rows = (0, 1)
    h_hat = (s["h"].float() - s["stats"][..., :1]) * s["stats"][..., 1:]
    d_y = s["d_y"].float()
    out = {"d_gamma": (d_y * h_hat).sum(rows), "d_beta": d_y.sum(rows)}
    t = d_y * s["gamma"]
    d_h = s["d_h"].float() + s["stats"][..., 1:] * (t - t.mean(-1, keepdim=True) - h_hat * (t * h_hat).mean(-1, keepdim=True))
    n = b_hat = s["branch"].float()
    if s["post"]:
        b_hat = (b_hat - s["post_stats"][..., :1]) * s["post_stats"][..., 1:]
        n = b_hat * s["post_gamma"] + s["post_beta"]
    by_group = (d_h * n).sum(1)
    out["d_scale"] = (by_group if s["gate"] is None else by_group * s["gate"]).sum(0)
    d_n = d_h * s["scale"]
    if s["gate"] is not None:
        out["d_gate"] = by_group * s["scale"]
        d_n = d_n * s["gate"][:, None]
    if s["post"]:
        out["d_post_gamma"], out["d_post_beta"] = (d_n * b_hat).sum(rows), d_n.sum(rows)
        u = d_n * s["post_gamma"]
        d_n = s["post_stats"][..., 1:] * (u - u.mean(-1, keepdim=True) - b_hat * (u * b_hat).mean(-1, keepdim=True))
    out["d_x"], out["d_branch"] = d_h.to(TYPES[s["stream_type"]]), d_n.to(TYPES[s["branch_type"]])
    return out


# ------------------------------------------------------------------ one pass
def run(state):
    s, op = state, state["op"]
    if not own:
        plain = {"attention": _attention_plain, "attention_backward": _attention_backward_plain, "rope": _rope_plain,
                 "norm": _norm_plain, "norm_backward": _norm_backward_plain}
        return plain[op](s)
    vk = _vk()
    if op == "attention":
        out = torch.empty_like(s["q"])
        lse = torch.empty(s["q"].shape[:3], device="cuda")
        vk.attention_forward(s["q"], s["k"], s["v"], out, lse, q_lens=s["q_lens"], kv_lens=s["kv_lens"])
        return out, lse
    if op == "attention_backward":
        dq, dk, dv = torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])
        vk.attention_backward(s["q"], s["k"], s["v"], s["out"], s["lse"], s["d_out"], dq, dk, dv, q_lens=s["q_lens"],
                              kv_lens=s["kv_lens"])
        return dq, dk, dv
    if op == "rope":
        q, k = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        vk.rope_axes(s["q"], s["k"], s["positions"], _sections(s), FREQ, q, k, inverse=s["inverse"])
        return q, k
    row = s["branch"].shape[:2]
    if op == "norm":
        h, y = torch.empty_like(s["x"]), torch.empty_like(s["branch"])
        stats = torch.empty(*row, 2, device="cuda")
        post_stats = torch.empty(*row, 2, device="cuda") if s["post"] else None
        vk.residual_norm_forward(s["x"], s["branch"], s["gamma"], s["beta"], EPS, h, y, stats, scale=s["scale"], gate=s["gate"],
                                 post_gamma=s["post_gamma"], post_beta=s["post_beta"], post_stats=post_stats)
        return h, y, stats, post_stats
    vector = lambda x: None if x is None else torch.empty_like(x)  # noqa: E731
    out = {"d_x": torch.empty_like(s["h"]), "d_branch": torch.empty_like(s["branch"]), "d_gamma": vector(s["gamma"]),
           "d_beta": vector(s["beta"]), "d_scale": vector(s["scale"])}
    if s["gate"] is not None:
        out["d_gate"] = vector(s["gate"])
    if s["post"]:
        out["d_post_gamma"], out["d_post_beta"] = vector(s["post_gamma"]), vector(s["post_beta"])
    vk.residual_norm_backward(s["d_h"], s["d_y"], s["h"], s["branch"], s["stats"], s["gamma"], scale=s["scale"], gate=s["gate"],
                              post_gamma=s["post_gamma"], post_beta=s["post_beta"], post_stats=s["post_stats"], **out)
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op.startswith("attention"):
        size, h, d = (4 if case["dtype"] == "f32" else 2), case["heads"], case["dim"]
        q, k = _lengths(case) if case["ragged"] else ([case["q_tokens"]] * case["batch"], [case["kv_tokens"]] * case["batch"])
        pairs = h * sum(x * y for x, y in zip(q, k))
        read_q, read_k = h * sum(q) * d * size, h * sum(k) * d * size
        all_q, all_k = case["batch"] * h * case["q_tokens"] * d * size, case["batch"] * h * case["kv_tokens"] * d * size
        stats = case["batch"] * h * case["q_tokens"] * 4
        if op == "attention":  # q, k, v in; out and lse out
            return {"bytes": read_q + 2 * read_k + all_q + stats, "flops": 4 * pairs * d}
        # q, out, d_out, k, v and lse in; dq, dk, dv out
        return {"bytes": 3 * read_q + 2 * read_k + stats + all_q + 2 * all_k, "flops": 10 * pairs * d}
    if op == "rope":
        size = 4 if case["dtype"] == "f32" else 2
        values = 2 * case["batch"] * case["heads"] * case["tokens"] * case["dim"]
        places = (case["batch"] if case["own_positions"] else 1) * case["tokens"] * len(_sections(case)) * 8
        return {"bytes": 2 * values * size + places, "flops": 3 * values}
    rows, c = case["groups"] * case["tokens"], case["cols"]
    stream, branch = (4 if case["stream_type"] == "f32" else 2), (4 if case["branch_type"] == "f32" else 2)
    stats = rows * 8 * (2 if case["post"] else 1)
    if op == "norm":  # x and branch in; h, y and the statistics out
        return {"bytes": rows * c * 2 * (stream + branch) + stats, "flops": rows * c * (22 if case["post"] else 12)}
    # d_h, d_y, h and branch in; d_x and d_branch out
    return {"bytes": rows * c * (3 * stream + 3 * branch) + stats, "flops": rows * c * (40 if case["post"] else 24)}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_attention(s, backward):
    scale = s["dim"] ** -0.5
    q_len = s["q_lens"].tolist() if s["q_lens"] is not None else [s["q_tokens"]] * s["batch"]
    k_len = s["kv_lens"].tolist() if s["kv_lens"] is not None else [s["kv_tokens"]] * s["batch"]
    zeros = lambda like: torch.zeros(like.shape, dtype=torch.float64, device="cuda")  # noqa: E731
    out, lse = zeros(s["q"]), torch.full(s["q"].shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    dq, dk, dv = zeros(s["q"]), zeros(s["k"]), zeros(s["v"])
    for b in range(s["batch"]):
        n, m = q_len[b], k_len[b]
        if n == 0 or m == 0:
            continue
        q, k, v = s["q"][b, :, :n].double(), s["k"][b, :, :m].double(), s["v"][b, :, :m].double()
        scores = torch.einsum("hnd,hmd->hnm", q, k) * scale
        if not backward:
            lse[b, :, :n] = torch.logsumexp(scores, -1)
            out[b, :, :n] = torch.einsum("hnm,hmd->hnd", torch.softmax(scores, -1), v)
            continue
        p = torch.exp(scores - s["lse"][b, :, :n, None].double())
        g = s["d_out"][b, :, :n].double()
        dv[b, :, :m] = torch.einsum("hnm,hnd->hmd", p, g)
        along = torch.einsum("hnd,hnd->hn", g, s["out"][b, :, :n].double())
        p *= torch.einsum("hnd,hmd->hnm", g, v) - along[..., None]
        dq[b, :, :n] = scale * torch.einsum("hnm,hmd->hnd", p, k)
        dk[b, :, :m] = scale * torch.einsum("hnm,hnd->hmd", p, q)
    return (dq, dk, dv) if backward else (out, lse)


def _exact_rope(s):
    outs = []
    for x in (s["q"].double(), s["k"].double()):
        y, at = x.clone(), 0
        for axis, width in enumerate(_sections(s)):
            half = width // 2
            pos = s["positions"][..., axis].double()
            pos = pos[:, None, :, None] if pos.dim() == 2 else pos[None, None, :, None]
            i = torch.arange(half, dtype=torch.float64, device="cuda")
            turn = torch.polar(torch.ones_like(pos * i), pos * torch.exp(-2.0 * i / width * math.log(FREQ)))
            z = torch.complex(x[..., at:at + half], x[..., at + half:at + width])
            z = z * (turn.conj() if s["inverse"] else turn)
            y[..., at:at + half], y[..., at + half:at + width] = z.real, z.imag
            at += width
        outs.append(y)
    return tuple(outs)


def _exact_norm(s):
    c = s["cols"]

    def layer_norm(x, g, b):
        mean = x.sum(-1) / c
        var = ((x - mean[..., None]) ** 2).sum(-1) / c
        rstd = 1.0 / torch.sqrt(var + EPS)
        return (x - mean[..., None]) * rstd[..., None] * g.double() + b.double(), torch.stack([mean, rstd], -1)

    n, post_stats = s["branch"].double(), None
    if s["post"]:
        n, post_stats = layer_norm(n, s["post_gamma"], s["post_beta"])
    factor = s["scale"].double() if s["gate"] is None else s["scale"].double() * s["gate"].double()[:, None]
    h = s["x"].double() + factor * n
    y, stats = layer_norm(h, s["gamma"], s["beta"])
    return h, y, stats, post_stats


def _exact_norm_backward(s):
    c, d = s["cols"], lambda x: x.double()  # noqa: E731

    def through(grad, hat, rstd):
        """The gradient of a standardised row hat = (x - mean) rstd, given the gradient of hat."""
        return rstd * (grad - grad.sum(-1, keepdim=True) / c - hat * (grad * hat).sum(-1, keepdim=True) / c)

    mean, rstd = d(s["stats"]).unbind(-1)
    hat = (d(s["h"]) - mean[..., None]) * rstd[..., None]
    out = {"d_gamma": torch.einsum("gtc,gtc->c", d(s["d_y"]), hat), "d_beta": d(s["d_y"]).sum((0, 1))}
    d_h = d(s["d_h"]) + through(d(s["d_y"]) * d(s["gamma"]), hat, rstd[..., None])
    gate = torch.ones(s["groups"], c, dtype=torch.float64, device="cuda") if s["gate"] is None else d(s["gate"])
    n = d(s["branch"])
    if s["post"]:
        post_mean, post_rstd = d(s["post_stats"]).unbind(-1)
        b_hat = (n - post_mean[..., None]) * post_rstd[..., None]
        n = b_hat * d(s["post_gamma"]) + d(s["post_beta"])
    out["d_scale"] = torch.einsum("gtc,gtc,gc->c", d_h, n, gate)
    if s["gate"] is not None:
        out["d_gate"] = torch.einsum("gtc,gtc,c->gc", d_h, n, d(s["scale"]))
    d_n = d_h * (d(s["scale"]) * gate)[:, None]
    if s["post"]:
        out["d_post_gamma"], out["d_post_beta"] = torch.einsum("gtc,gtc->c", d_n, b_hat), d_n.sum((0, 1))
        d_n = through(d_n * d(s["post_gamma"]), b_hat, post_rstd[..., None])
    out["d_x"], out["d_branch"] = d_h, d_n
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op.startswith("attention"):
        return _exact_attention(s, op == "attention_backward")
    return {"rope": _exact_rope, "norm": _exact_norm, "norm_backward": _exact_norm_backward}[op](s)
