"""The attention-input and sparse-attention operators, measured through the calls a
program makes of them, beside their plain forms in elementary torch operations.

    rope_axes      rotation of a head's dimension pairs by positions on several axes
    qk_norm_rope   RMS norm of every query and key head, then that rotation
    block_means, block_means_update, block_select
                   mean key of every block of keys, and the blocks whose mean has the
                   largest product with a query
    attn_blocks    softmax attention of a query over its own blocks only

`own` chooses between the two: False runs the plain forms (nothing of this package is
imported), True the framework's operators. `exact` restates every case in float64.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_ES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6


def _ops():
    """The framework's operators (only where `own` is true)."""

    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hexo-bot_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from shrimp import ops

    return ops


# ---- cases ---------------------------------------------------------------------------


def listed():
    return [
        # rotation of one board's summary-token and cell queries: one position of a search
        dict(name="rope_board_b1", kind="rope", batch=1, length=264, heads=8, dim=16, axes=2,
             pairs="4+4", far=24, interleaved=False, dtype="bf16", train=False),
        # a clip of frames, time and two image axes, forward and backward of a training step
        dict(name="rope_clip_train", kind="rope", batch=2, length=12000, heads=16, dim=128, axes=3,
             pairs="16+24+24", far=4096, interleaved=True, dtype="f16", train=True),
        # one new token of each of 48 sequences in serving, few key heads, far positions
        dict(name="norm_rope_token_b48", kind="norm", batch=48, length=1, heads=16, kv_heads=4,
             dim=128, axes=1, pairs="64", far=400000, interleaved=False, dtype="bf16",
             train=False),
        # the benchmark's batch of boards: queries and keys as views of a fused projection
        dict(name="norm_rope_boards_b512", kind="norm", batch=512, length=264, heads=8, kv_heads=8,
             dim=16, axes=2, pairs="4+4", far=24, interleaved=False, dtype="bf16", train=False),
        # a training step on the main network's large boards in fp32
        dict(name="norm_rope_boards_train", kind="norm", batch=111, length=584, heads=3, kv_heads=3,
             dim=64, axes=2, pairs="16+16", far=40, interleaved=False, dtype="f32", train=True),
        # a training step on long sequences with shared key heads
        dict(name="norm_rope_long_train", kind="norm", batch=2, length=8190, heads=32, kv_heads=8,
             dim=128, axes=1, pairs="64", far=131072, interleaved=True, dtype="bf16", train=True),
        # choosing key blocks on one evaluator group of large boards
        dict(name="select_boards_b111", kind="select", batch=111, q_len=584, k_len=584, heads=3,
             kv_heads=3, dim=64, block=16, topk=8, ragged=0.8, dtype="bf16"),
        # choosing key blocks for every query of long sequences, heads in groups of four
        dict(name="select_long_b2", kind="select", batch=2, q_len=8000, k_len=8000, heads=16,
             kv_heads=4, dim=128, block=64, topk=16, ragged=1.0, dtype="f16"),
        # serving: one new token over a long cache whose block means are kept beside it
        dict(name="attn_token_b32", kind="attn", batch=32, q_len=1, k_len=32000, heads=16,
             kv_heads=4, dim=128, block=64, topk=16, ragged=0.5, dtype="bf16", train=False),
        # the main network's heads over one evaluator group of large boards
        dict(name="attn_boards_b111", kind="attn", batch=111, q_len=584, k_len=584, heads=3,
             kv_heads=3, dim=64, block=16, topk=8, ragged=0.8, dtype="bf16", train=False),
        # long sequences of eight heads, fp16, a ragged end
        dict(name="attn_long_b1", kind="attn", batch=1, q_len=8100, k_len=8100, heads=8,
             kv_heads=8, dim=64, block=64, topk=16, ragged=1.0, dtype="f16", train=False),
        # a training step: the choice, forward and backward, heads in pairs
        dict(name="attn_train_b2", kind="attn", batch=2, q_len=4096, k_len=4096, heads=8,
             kv_heads=4, dim=64, block=64, topk=8, ragged=0.7, dtype="bf16", train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    """What keeps a drawn case at or under the largest listed one of its kind: the dense
    scores that the plain form makes for select and attn, elements for the others."""

    if c["kind"] == "attn":
        dense = c["batch"] * c["heads"] * c["q_len"] * c["k_len"] * c["dim"]
        return dense * (3 if c["train"] else 1)
    if c["kind"] == "select":
        return c["batch"] * c["heads"] * (c["q_len"] + c["k_len"]) * c["dim"]
    return (c["batch"] * c["length"] * (c["heads"] + c.get("kv_heads", 0)) * c["dim"]
            * _ES[c["dtype"]] * (3 if c["train"] else 1))


def draw(rng):
    kind = rng.choice(("rope", "norm", "norm", "select", "attn", "attn"))
    most = {"bytes": 0, "cost": 0}
    for c in listed():
        if c["kind"] == kind:
            most = {"bytes": max(most["bytes"], work(c)["bytes"]), "cost": max(most["cost"], _cost(c))}
    while True:
        c = dict(kind=kind, batch=_log_int(rng, 1, 512), dtype=rng.choice(("bf16", "bf16", "f16", "f32")))
        kv = rng.choice((1, 2, 3, 4, 8))
        group = rng.choice((1, 1, 2, 4, 8))
        if kind in ("rope", "norm"):
            dim = rng.choice((16, 24, 32, 64, 64, 96, 128, 128))
            axes = rng.choice((1, 2, 2, 3))
            half = dim // 2 if rng.random() < 0.7 else max(axes, dim // 4)  # or half the head rotates
            cut = sorted(rng.sample(range(1, half), axes - 1)) + [half]
            pairs = [b - a for a, b in zip([0] + cut[:-1], cut)]
            c.update(length=_log_int(rng, 1, 12000), heads=kv * group, dim=dim, axes=axes,
                     pairs="+".join(map(str, pairs)), far=_log_int(rng, 8, 400000),
                     interleaved=rng.random() < 0.4, train=rng.random() < 0.5)
            if kind == "norm":
                c.update(kv_heads=kv)
        else:
            token = rng.random() < 0.25
            k_len = _log_int(rng, 20, 32000 if token else 8100)
            block = rng.choice((16, 16, 32, 64, 64, 128) if k_len < 2000 else (64, 64, 128))
            c.update(q_len=1 if token else k_len, k_len=k_len, heads=kv * group, kv_heads=kv,
                     dim=rng.choice((16, 24, 32, 64, 64, 128)), block=block,
                     topk=rng.choice((1, 3, 4, 8, 8, 16)), ragged=rng.choice((1.0, 0.9, 0.7, 0.4)),
                     dtype=rng.choice(("bf16", "bf16", "f16")))
            if kind == "attn":
                c.update(train=not token and rng.random() < 0.4)
        if work(c)["bytes"] <= most["bytes"] and _cost(c) <= most["cost"]:
            return c


# ---- inputs --------------------------------------------------------------------------


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _positions(case, g):
    """(B, S, axes) int32 positions: hex cells, frames and pixels, or places in a text,
    up to `far`; every axis on its own scale."""

    u = torch.rand(case["batch"], case["length"], case["axes"], generator=g, device=DEV)
    if case["axes"] == 2:  # axial coordinates lie on both sides of the origin
        u = 2 * u - 1
    scale = torch.tensor([1.0, 0.5, 0.5, 0.25][: case["axes"]], device=DEV)
    return (u * scale * case["far"]).round().to(torch.int32)


def _inputs(case, seed):
    """Everything of a case that is made from the seed (what `exact` also reads)."""

    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = _DT[case["dtype"]]
    b, h, d = case["batch"], case["heads"], case["dim"]
    if case["kind"] in ("rope", "norm"):
        n = case["length"]
        s = dict(pos=_positions(case, g), sections=[int(p) for p in case["pairs"].split("+")],
                 interleaved=case["interleaved"])
        # each axis has its own geometric range of frequencies, from 1 down to 1 / 10000
        s["freqs"] = torch.cat([10000.0 ** (-torch.arange(p, device=DEV, dtype=torch.float32) / p)
                                for p in s["sections"]])
        if case["kind"] == "rope":
            s["x"] = _randn(g, b, n, h, d).to(dt).transpose(1, 2)
            if case["train"]:
                s["gx"] = _randn(g, b, h, n, d).to(dt)
            return s
        hk = case["kv_heads"]
        qkv = _randn(g, b, n, h + 2 * hk, d).to(dt)  # a fused projection's rows
        s["q"] = qkv[:, :, :h].transpose(1, 2)
        s["k"] = qkv[:, :, h : h + hk].transpose(1, 2)
        s["q_weight"] = (1 + 0.2 * _randn(g, d)).to(dt)
        s["k_weight"] = (1 + 0.2 * _randn(g, d)).to(dt)
        if case["train"]:
            s["gq"] = _randn(g, b, h, n, d).to(dt)
            s["gk"] = _randn(g, b, hk, n, d).to(dt)
        return s
    hk, nq, nk = case["kv_heads"], case["q_len"], case["k_len"]
    # neighbouring keys are alike: runs of keys share a drift, as pieces of a board or text do
    runs = _randn(g, b, hk, nk // 24 + 1, d).repeat_interleave(24, 2)[:, :, :nk]
    s = dict(block=case["block"], topk=case["topk"], q=_randn(g, b, h, nq, d).to(dt),
             k=(_randn(g, b, hk, nk, d) + 0.7 * runs).to(dt))
    low = max(1, int(nk * case["ragged"]))
    s["k_lens"] = torch.randint(low, nk + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
    s["q_lens"] = s["k_lens"].clone() if nq == nk else torch.full_like(s["k_lens"], nq)
    if case["kind"] == "attn":
        s["v"] = _randn(g, b, hk, nk, d).to(dt)
        if case["train"]:
            s["g"] = _randn(g, b, h, nq, d).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    if case["kind"] == "attn" and case["q_len"] == 1:
        # a serving program keeps the means of the blocks before the one its last key is in
        s["means"] = _means(s["k"], s["k_lens"], s["block"])
        last = ((s["k_lens"] - 1) // s["block"]).long()
        s["means"][torch.arange(case["batch"], device=DEV), :, last] = 0
    if own:
        _ops()
        for key in ("x", "q", "k", "v", "q_weight", "k_weight"):
            if case.get("train") and key in s:
                s[key].requires_grad_()
    return s


# ---- plain forms: 32 bits, 64 for angles, block means and the scores that choose ------------


def _cos_sin(pos, freqs, sections):
    axis = torch.repeat_interleave(torch.arange(len(sections), device=DEV),
                                   torch.tensor(sections, device=DEV), output_size=sum(sections))
    angle = pos[:, :, axis].double() * freqs.double()  # far positions times frequencies
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def _rotate(x, cos, sin, interleaved, inverse=False):
    """x (B, H, S, D) float, its first 2 P dimensions rotated in pairs."""

    p = cos.shape[-1]
    a, b = (x[..., 0 : 2 * p : 2], x[..., 1 : 2 * p : 2]) if interleaved else (x[..., :p], x[..., p : 2 * p])
    if inverse:
        sin = -sin
    y = x.clone()
    if interleaved:
        y[..., 0 : 2 * p : 2] = a * cos - b * sin
        y[..., 1 : 2 * p : 2] = b * cos + a * sin
    else:
        y[..., :p] = a * cos - b * sin
        y[..., p : 2 * p] = b * cos + a * sin
    return y


def _norm_rotate(x, w, cos, sin, interleaved):
    x = x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return _rotate(x * r * w.float(), cos, sin, interleaved)


def _norm_rotate_back(x, w, g, cos, sin, interleaved):
    x, w = x.float(), w.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    g = _rotate(g.float(), cos, sin, interleaved, inverse=True)
    dw = (g * x * r).double().sum((0, 1, 2))  # a long sum
    g = g * w
    return r * g - x * (r * r * r * (g * x).mean(-1, keepdim=True)), dw


def _blocks(n, block):
    return -(-n // block)


def _means(k, k_lens, block):
    """(B, Hk, NB, D) fp32 mean of each block's live keys (zero for a block without one)."""

    b, hk, n, d = k.shape
    nb = _blocks(n, block)
    live = torch.arange(n, device=DEV) < k_lens[:, None]
    x = torch.where(live[:, None, :, None], k, torch.zeros_like(k)).double()
    x = torch.cat([x, x.new_zeros(b, hk, nb * block - n, d)], 2).view(b, hk, nb, block, d).sum(3)
    start = torch.arange(nb, device=DEV) * block
    count = (k_lens[:, None] - start).clamp(0, block).clamp(min=1)
    return (x / count[:, None, :, None]).float()


def _means_update(means, k, k_lens, block):
    """The mean of the block that holds each sequence's last key, in place."""

    b, hk, n, d = k.shape
    last = (k_lens - 1).clamp(min=0) // block
    idx = last[:, None] * block + torch.arange(block, device=DEV)
    live = idx < k_lens[:, None]
    rows = k[torch.arange(b, device=DEV)[:, None], :, idx.clamp(max=n - 1)]  # (B, block, Hk, D)
    x = torch.where(live[:, :, None, None], rows, torch.zeros_like(rows)).double().sum(1)
    means[torch.arange(b, device=DEV), :, last.long()] = (x / live.sum(1).clamp(min=1)[:, None, None]).float()


def _select(q, means, q_lens, k_lens, block, topk):
    """(B, Hk, Sq, topk) int32: ascending indices of the live blocks whose mean has the
    largest product with the sum of the group's queries (ties to the lower index), then -1."""

    b, h, nq, d = q.shape
    hk, nb = means.shape[1], means.shape[2]
    qs = q.view(b, hk, h // hk, nq, d).double().sum(2)
    live = torch.arange(nb, device=DEV) * block < k_lens[:, None]
    rows = torch.arange(nq, device=DEV) < q_lens[:, None]
    out = torch.full((b, hk, nq, topk), -1, device=DEV, dtype=torch.int32)
    k = min(topk, nb)
    for i in _slices(b, hk * nq * nb):
        sc = qs[i] @ means[i].double().transpose(2, 3)
        sc = sc.masked_fill(~live[i, None, None], float("-inf"))
        order = sc.sort(dim=-1, descending=True, stable=True)[1][..., :k]
        ok = live[i, None, None].expand_as(sc).gather(-1, order) & rows[i, None, :, None]
        pick = torch.where(ok, order, nb).sort(-1)[0]
        out[i, ..., :k] = torch.where(pick < nb, pick, -1).to(torch.int32)
    return out


def _slices(n, each):
    """Slices of n items of `each` elements, 2^28 elements or one item at a time."""

    step = max(1, 2**28 // each)
    return [slice(i, i + step) for i in range(0, n, step)]


def _chosen(sel, nb):
    """(..., NB) truth of a choice (..., topk)."""

    m = torch.zeros((*sel.shape[:-1], nb + 1), dtype=torch.bool, device=DEV)
    m.scatter_(-1, torch.where(sel >= 0, sel, nb).long(), True)
    return m[..., :nb]


def _attend_gathered(q, k, v, sel, k_lens, block):
    """Few queries: their blocks' keys gathered."""

    b, h, nq, d = q.shape
    hk, n = k.shape[1], k.shape[2]
    idx = (sel.long()[..., None] * block + torch.arange(block, device=DEV)).flatten(3)
    live = (idx >= 0) & (idx < k_lens[:, None, None, None])
    at = idx.clamp(0, n - 1).flatten(2)[..., None].expand(-1, -1, -1, d)
    kk = k.gather(2, at).view(b, hk, nq, -1, d).float()
    vv = v.gather(2, at).view(b, hk, nq, -1, d).float()
    qq = q.view(b, hk, h // hk, nq, d).transpose(2, 3).float()
    s = (qq @ kk.transpose(3, 4)) / math.sqrt(d)
    s = s.masked_fill(~live[:, :, :, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    o = (p @ vv) / torch.where(z > 0, z, torch.ones_like(z))
    lse = (m + torch.log(z))[..., 0]
    return (o.transpose(2, 3).reshape(b, h, nq, d).to(q.dtype), lse.transpose(2, 3).reshape(b, h, nq))


def _attend(q, k, v, sel, k_lens, block, g=None):
    """All keys under the choice's mask, some sequences at a time; with g also the
    gradients."""

    b, h, nq, d = q.shape
    hk, n = k.shape[1], k.shape[2]
    if nq * sel.shape[-1] <= 64 and g is None:
        return _attend_gathered(q, k, v, sel, k_lens, block)
    grp, nb, scale = h // hk, _blocks(n, block), 1 / math.sqrt(d)
    out = torch.empty(b, h, nq, d, dtype=q.dtype, device=DEV)
    lse = torch.empty(b, h, nq, device=DEV)
    grads = [torch.empty(t.shape, dtype=t.dtype, device=DEV) for t in (q, k, v)] if g is not None else []
    live = torch.arange(n, device=DEV) < k_lens[:, None]
    for i in _slices(b, h * nq * n):
        mask = _chosen(sel[i], nb).repeat_interleave(block, -1)[..., :n] & live[i, None, None]
        qq = q[i].float().view(-1, hk, grp, nq, d)
        kk = k[i].float()[:, :, None]
        vv = torch.where(live[i, None, :, None], v[i], torch.zeros_like(v[i])).float()[:, :, None]
        s = (qq @ kk.transpose(-1, -2) * scale).masked_fill(~mask[:, :, None], float("-inf"))
        m = s.amax(-1, keepdim=True)
        m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
        p = torch.exp(s - m)
        z = p.sum(-1, keepdim=True)
        lse[i] = (m + torch.log(z)).view(-1, h, nq)
        p = p / torch.where(z > 0, z, torch.ones_like(z))
        o = p @ vv
        out[i] = o.view(-1, h, nq, d).to(q.dtype)
        if g is not None:
            gg = g[i].float().view(-1, hk, grp, nq, d)
            dp = gg @ vv.transpose(-1, -2)
            ds = p * (dp - (gg * o).sum(-1, keepdim=True)) * scale
            grads[0][i] = (ds @ kk).view(-1, h, nq, d).to(q.dtype)
            grads[1][i] = (ds.flatten(2, 3).transpose(-1, -2) @ qq.flatten(2, 3)).to(q.dtype)
            grads[2][i] = (p.flatten(2, 3).transpose(-1, -2) @ gg.flatten(2, 3)).to(q.dtype)
    return (out, lse, *grads)


def _run_plain(s):
    c = s["case"]
    if c["kind"] in ("rope", "norm"):
        cos, sin = _cos_sin(s["pos"], s["freqs"], s["sections"])
        il = s["interleaved"]
        if c["kind"] == "rope":
            y = _rotate(s["x"].float(), cos, sin, il).to(s["x"].dtype)
            if not c["train"]:
                return y
            return y, _rotate(s["gx"].float(), cos, sin, il, inverse=True).to(s["x"].dtype)
        out = [_norm_rotate(s[t], s[t + "_weight"], cos, sin, il).to(s[t].dtype) for t in "qk"]
        if c["train"]:
            for t in "qk":
                w = s[t + "_weight"]
                dx, dw = _norm_rotate_back(s[t], w, s["g" + t], cos, sin, il)
                out += [dx.to(s[t].dtype), dw.to(w.dtype)]
        return out
    if "means" in s:
        means = s["means"]
        _means_update(means, s["k"], s["k_lens"], s["block"])
    else:
        means = _means(s["k"], s["k_lens"], s["block"])
    sel = _select(s["q"], means, s["q_lens"], s["k_lens"], s["block"], s["topk"])
    if c["kind"] == "select":
        return means, sel
    return (means, sel, *_attend(s["q"], s["k"], s["v"], sel, s["k_lens"], s["block"], s.get("g")))


# ---- the framework's operators ------------------------------------------------------------


def _run_own(s):
    ops = _ops()
    c = s["case"]
    if c["kind"] == "rope":
        y = ops.rope_axes(s["x"], s["pos"], s["freqs"], s["sections"], s["interleaved"])
        if not c["train"]:
            return y
        return y.detach(), *torch.autograd.grad(y, s["x"], s["gx"])
    if c["kind"] == "norm":
        q, k = ops.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["pos"], s["freqs"],
                                s["sections"], EPS, s["interleaved"])
        if not c["train"]:
            return [q, k]
        leaves = [s["q"], s["q_weight"], s["k"], s["k_weight"]]
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), leaves, (s["gq"], s["gk"]))]
    if "means" in s:
        means = s["means"]
        ops.block_means_update(means, s["k"], s["k_lens"], s["block"])
    else:
        means = ops.block_means(s["k"].detach(), s["k_lens"], s["block"])
    sel = ops.block_select(s["q"].detach(), means, s["q_lens"], s["k_lens"], s["block"], s["topk"])
    if c["kind"] == "select":
        return means, sel
    out, lse = ops.attn_blocks(s["q"], s["k"], s["v"], sel, s["q_lens"], s["k_lens"], s["block"])
    if not c["train"]:
        return means, sel, out, lse
    grads = torch.autograd.grad(out, [s["q"], s["k"], s["v"]], s["g"])
    return means, sel, out.detach(), lse.detach(), *grads


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- work ----------------------------------------------------------------------------


def work(case):
    """Inputs read once, outputs written once, and the operations of the formulas; of a
    cache that is longer than its query's choice only the chosen blocks and the means."""

    es, b, h, d = _ES[case["dtype"]], case["batch"], case["heads"], case["dim"]
    if case["kind"] in ("rope", "norm"):
        n, hk = case["length"], case.get("kv_heads", 0)
        elems = b * n * (h + hk) * d
        # forward: read, write; backward: read the gradient (and the input again), write
        passes = 2 + (0 if not case["train"] else 2 if case["kind"] == "rope" else 3)
        per = (3 if case["kind"] == "rope" else 7) * (1 if not case["train"] else 3)
        return {"bytes": elems * es * passes + b * n * case["axes"] * 4, "flops": elems * per}
    hk, nq, nk, topk = case["kv_heads"], case["q_len"], case["k_len"], case["topk"]
    nb = _blocks(nk, case["block"])
    live = (1 + case["ragged"]) / 2  # mean part of the longest sequence
    rows = int(b * h * nq * (live if nq == nk else 1))
    blocks = max(1, int(nb * live))
    keys = b * hk * nk * d * es * live
    means = b * hk * nb * d * 4
    sel = b * hk * nq * topk * 4
    q = b * h * nq * d * es
    if case["kind"] == "select":
        return {"bytes": int(q + keys + means + sel),
                "flops": int(rows // (h // hk) * blocks * d * 2 + keys // es)}
    seen = min(topk, blocks) * case["block"]
    few = nq * topk < nb  # the cache is not read whole
    kv = 2 * b * hk * nq * seen * d * es if few else 2 * keys
    flops = rows // (h // hk) * blocks * d * 2 + rows * seen * d * 4
    total = q * 2 + kv + means + sel + b * h * nq * 4
    if case["train"]:
        flops += rows * seen * d * 10
        total += 3 * q + 2 * kv  # q, out's gradient and dq; k, v again; dk, dv
    return {"bytes": int(total), "flops": int(flops)}


# ---- float64 values from the definitions -----------------------------------------------------


def _exact_rotated(x, pos, freqs, sections, interleaved, sign):
    """Complex form: pair p of a head times exp(i sign pos freq)."""

    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    p = len(axis)
    turn = torch.stack([pos[..., a].double() * freqs[i].double() for i, a in enumerate(axis)], -1)
    turn = torch.polar(torch.ones_like(turn), sign * turn).unsqueeze(1)
    if interleaved:
        z = torch.view_as_complex(x[..., : 2 * p].unflatten(-1, (p, 2)).contiguous()) * turn
        head = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :p], x[..., p : 2 * p]) * turn
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, x[..., 2 * p :]], -1)


def _exact_rows(s, c):
    args = (s["pos"], s["freqs"], s["sections"], s["interleaved"])
    if c["kind"] == "rope":
        y = _exact_rotated(s["x"].double(), *args, 1.0)
        return (y, _exact_rotated(s["gx"].double(), *args, -1.0)) if c["train"] else y
    out, back = [], []
    for t in "qk":
        x, w = s[t].double(), s[t + "_weight"].double()
        n = x / (x.square().sum(-1, keepdim=True) / c["dim"] + EPS).sqrt()
        out.append(_exact_rotated(n * w, *args, 1.0))
        if c["train"]:
            u = _exact_rotated(s["g" + t].double(), *args, -1.0)
            dw = torch.einsum("bhsd,bhsd->d", u, n)
            u = u * w
            inner = (u * n).sum(-1, keepdim=True) / c["dim"]
            back += [(u - n * inner) / (x.square().mean(-1, keepdim=True) + EPS).sqrt(), dw]
    return out + back


def exact(case, seed):
    if case["kind"] in ("rope", "norm"):
        if case["batch"] * case["length"] * case["heads"] * case["dim"] > 1.5e8:
            return None
        return _exact_rows(_inputs(case, seed), case)
    s = _inputs(case, seed)
    b, h, nq, d = s["q"].shape
    hk, n = s["k"].shape[1:3]
    block, topk, train = s["block"], s["topk"], case.get("train", False)
    nb, grp = (n + block - 1) // block, h // hk
    means = torch.zeros(b, hk, nb, d, dtype=torch.float64, device=DEV)
    sel = torch.full((b, hk, nq, topk), -1, dtype=torch.int32, device=DEV)
    out = torch.zeros(b, h, nq, d, dtype=torch.float64, device=DEV)
    lse = torch.full((b, h, nq), float("-inf"), dtype=torch.float64, device=DEV)
    dq, dk, dv = (torch.zeros(t, dtype=torch.float64, device=DEV) for t in
                  ((b, h, nq, d), (b, hk, n, d), (b, hk, n, d))) if train else (None, None, None)
    lens, rows = s["k_lens"].tolist(), s["q_lens"].tolist()
    for i in range(b):
        length, live, nr = lens[i], -(-lens[i] // block), rows[i]
        if length == 0 or nr == 0:
            continue
        member = torch.arange(length, device=DEV) // block
        for j in range(hk):
            key = s["k"][i, j, :length].double()
            mean = torch.zeros(live, d, dtype=torch.float64, device=DEV).index_add_(0, member, key)
            mean = mean / torch.bincount(member, minlength=live)[:, None]
            means[i, j, :live] = mean
            mine = s["q"][i, j * grp : (j + 1) * grp, :nr].double()
            # the choice is made on the means that the program holds, in 32 bits
            rank = (mine.sum(0) @ mean.float().double().T).argsort(dim=-1, descending=True, stable=True)
            take = rank[:, : min(topk, live)].sort(-1).values
            sel[i, j, :nr, : take.shape[1]] = take.int()
            if case["kind"] == "select":
                continue
            seen = torch.zeros(nr, live, dtype=torch.bool, device=DEV)
            seen[torch.arange(nr, device=DEV)[:, None], take] = True
            seen = seen[:, member]
            val = s["v"][i, j, :length].double()
            for t in range(grp):
                hh = j * grp + t
                sc = torch.where(seen, mine[t] @ key.T / d**0.5, float("-inf"))
                lse[i, hh, :nr] = torch.logsumexp(sc, -1)
                p = torch.exp(sc - lse[i, hh, :nr, None])
                out[i, hh, :nr] = p @ val
                if train:
                    gr = s["g"][i, hh, :nr].double()
                    da = gr @ val.T
                    da = p * (da - (p * da).sum(-1, keepdim=True)) / d**0.5
                    dq[i, hh, :nr] = da @ key
                    dk[i, j, :length] += da.T @ mine[t]
                    dv[i, j, :length] += p.T @ gr
    if case["kind"] == "select":
        return means, sel
    return (means, sel, out, lse) + ((dq, dk, dv) if train else ())
