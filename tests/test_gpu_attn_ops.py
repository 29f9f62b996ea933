"""The rotary and block operators as a program meets them: their registration, compiled
programs, threads and streams at once, and what must be refused rather than answered."""

import threading

import pytest
import torch
from torch.autograd import forward_ad

from shrimp import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
B, H, HK, S, D, BLOCK, TOPK = 2, 4, 2, 100, 64, 16, 3


@pytest.fixture(scope="module")
def data():
    g = torch.Generator().manual_seed(51)
    rnd = lambda *n: torch.randn(*n, generator=g).bfloat16().to(DEV)
    q, k, v = rnd(B, H, S, D), rnd(B, HK, S, D), rnd(B, HK, S, D)
    w, fr = torch.rand(D, generator=g).to(DEV), torch.rand(D // 2, generator=g).to(DEV)
    lens = lambda *n: torch.tensor(n, dtype=torch.int32, device=DEV)
    pos = torch.arange(S, dtype=torch.int32, device=DEV).unsqueeze(1)
    return q, k, v, w, fr, pos, lens(100, 63), lens(100, 80)


def _layer(data):
    _, _, _, _, fr, pos, ql, kl = data

    def layer(q, k, v, w):
        qn, kn = ops.qk_norm_rope(q, k, w, w, pos, fr, [D // 2])
        means = ops.block_means(kn.detach(), kl, BLOCK)
        sel = ops.block_select(qn.detach(), means, ql, kl, BLOCK, TOPK)
        out, lse = ops.attn_blocks(ops.rope_axes(qn, pos, fr, [D // 2]), kn, v, sel, ql, kl, BLOCK)
        return out.float().square().sum() + lse.clamp(min=-9).sum()

    return layer


def _grads(f, data):
    leaves = [t.clone().requires_grad_() for t in data[:4]]
    return torch.autograd.grad(f(*leaves), leaves)


def test_registration(data):
    q, k, v, w, fr, pos, ql, kl = data
    leaf = lambda t: t.clone().requires_grad_()
    means = ops.block_means(k, kl, BLOCK)
    sel = ops.block_select(q, means, ql, kl, BLOCK, TOPK)
    out, lse = ops.attn_blocks(q, k, v, sel, ql, kl, BLOCK)
    o, half = torch.ops.shrimp, [D // 2]
    for op, args in (
        (o.rope_axes, (leaf(q), pos, fr, half, False, False)),
        (o.qk_norm_rope, (leaf(q), leaf(k), leaf(w), leaf(w), pos, fr, half, 1e-6, False)),
        (o.qk_norm_rope_backward, (q, k, q, k, w, w, pos, fr, half, 1e-6, False)),
        (o.block_means, (k, kl, BLOCK)),
        (o.block_means_update, (means.clone(), k, kl, BLOCK)),
        (o.block_select, (q, means, ql, kl, BLOCK, TOPK)),
        (o.attn_blocks, (leaf(q), leaf(k), leaf(v), sel, ql, kl, BLOCK)),
        (o.attn_blocks_backward, (q, None, q, k, v, sel, ql, kl, out, lse, BLOCK)),
    ):
        torch.library.opcheck(op.default, args)


def test_compiled(data):
    layer = _layer(data)
    want = _grads(layer, data)
    got = _grads(torch.compile(layer, backend="aot_eager", fullgraph=True), data)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_traced(data):
    """A traced program holds the operators, not the results of the traced call."""

    q, k, v, w, fr, pos, ql, kl = data

    def run(q, k, v):
        qn, kn = ops.qk_norm_rope(q, k, w, w, pos, fr, [D // 2])
        sel = ops.block_select(qn, ops.block_means(kn, kl, BLOCK), ql, kl, BLOCK, TOPK)
        return ops.attn_blocks(ops.rope_axes(qn, pos, fr, [D // 2]), kn, v, sel, ql, kl, BLOCK)

    with torch.no_grad():
        traced = torch.jit.trace(run, (q, k, v))
        for a, b in zip(traced(q.flip(2), k * 0.5, v.flip(2)), run(q.flip(2), k * 0.5, v.flip(2))):
            assert torch.equal(a, b)


def test_streams_and_threads_at_once(data):
    layer = _layer(data)
    want = _grads(layer, data)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 4]):
            got.append(_grads(layer, data))
    torch.cuda.synchronize()
    threaded = [None] * 4

    def work(i):
        with torch.cuda.stream(streams[i]):
            threaded[i] = _grads(layer, data)
            streams[i].synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g in got + threaded:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_layouts_give_the_same_bits(data):
    q, k, v, _, _, _, ql, kl = data
    sel = ops.block_select(q, ops.block_means(k, kl, BLOCK), ql, kl, BLOCK, TOPK)
    one = k[:1, :1].expand(B, HK, S, D)
    turned = lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)
    for args, same in (
        ((q, one, one, sel, ql, kl), (q, one.contiguous(), one.contiguous(), sel, ql, kl)),
        ((turned(q), turned(k), turned(v), turned(sel), torch.stack([ql, ql], 1)[:, 1], kl), (q, k, v, sel, ql, kl)),
    ):
        for a, b in zip(ops.attn_blocks(*args, BLOCK), ops.attn_blocks(*same, BLOCK)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("which", ("q", "sel", "q_lens", "out", "lse"))
def test_changed_in_place_is_refused(data, which):
    q, k, v, _, _, _, ql, kl = data
    sel = ops.block_select(q, ops.block_means(k, kl, BLOCK), ql, kl, BLOCK, TOPK)
    leaf = q.clone().requires_grad_()
    t = dict(q=leaf * 1, sel=sel, q_lens=ql.clone())
    t["out"], t["lse"] = ops.attn_blocks(t["q"], k, v, t["sel"], t["q_lens"], kl, BLOCK)
    t[which].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(t["out"].float().sum(), leaf)


def test_forward_mode_is_refused(data):
    q, k, v, w, fr, pos, ql, kl = data
    sel = ops.block_select(q, ops.block_means(k, kl, BLOCK), ql, kl, BLOCK, TOPK)
    plain = ops.attn_blocks(q, k, v, sel, ql, kl, BLOCK)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: ops.rope_axes(dual, pos, fr, [D // 2]),
                     lambda: ops.qk_norm_rope(dual, k, w, w, pos, fr, [D // 2]),
                     lambda: ops.attn_blocks(dual, k, v, sel, ql, kl, BLOCK)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
        for a, b in zip(ops.attn_blocks(q, k, v, sel, ql, kl, BLOCK), plain):
            assert torch.equal(a, b)
