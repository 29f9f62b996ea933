"""shrimp::block_means, block_select and attn_blocks against float64 restatements.

Tolerances are elementwise bounds. U = 2^-24 is fp32's half step, H = finfo.eps / 2
the type's. A score sums d exact products in fp32: within (d + 2) U of the sum of
their magnitudes, E. A weight exp(score - max) is then within 2 E + 8 U + 2 U |score|
(natural units, both scores) relative, is rounded to the type (H, below fp16's normal range
2^-25 absolute beside a largest weight of 1), and n weights are added and rescaled in fp32
(n + 64 further steps of U). So a result is within
  W = (sum p |v|) (H + 2 E + (n + 80 + 4 |score|) U) + n 2^-25 max |v|
before its own rounding. Choices are compared exactly."""

import math

import pytest
import torch

from shrimp import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-24
DTYPES = (torch.bfloat16, torch.float16)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _heads(g, b, h, s, d, dt, layout="bhsd"):
    if layout == "bhsd":
        return torch.randn(b, h, s, d, generator=g).to(dt).to(DEV)
    if layout == "bshd":
        return torch.randn(b, s, h, d, generator=g).to(dt).to(DEV).transpose(1, 2)
    assert layout == "odd"  # one element in, rows of d + 3
    return torch.randn(b, s, h, d + 3, generator=g).to(dt).to(DEV)[..., 1 : d + 1].transpose(1, 2)


def _lens(*n):
    return torch.tensor(n, dtype=torch.int32, device=DEV)


# ---- means and choice ----------------------------------------------------------------


def _means_want(k, lens, block):
    b, hk, n, d = k.shape
    nb = -(-n // block)
    m, mag = torch.zeros(b, hk, nb, d, dtype=torch.float64), torch.zeros(b, hk, nb, d, dtype=torch.float64)
    for i in range(b):
        for j in range(nb):
            rows = k[i, :, j * block : min((j + 1) * block, lens[i])]
            if rows.shape[1]:
                m[i, :, j], mag[i, :, j] = rows.mean(1), rows.abs().mean(1)
    return m, mag


@pytest.mark.parametrize("dt", (torch.bfloat16, torch.float16, torch.float32), ids=str)
@pytest.mark.parametrize("shape", [
    (3, 2, 70, 64, 16, "bhsd"), (3, 4, 129, 128, 64, "bshd"), (3, 1, 40, 24, 32, "bshd"),
    (3, 3, 33, 20, 7, "odd"), (3, 1, 5, 1, 16, "bhsd"), (3, 2, 300, 96, 128, "odd"),
], ids=str)
def test_means(shape, dt):
    b, hk, n, d, block, layout = shape
    k = _heads(_gen(1), b, hk, n, d, dt, layout)
    lens = [n, max(n - block, 1), n // 2]
    for i, x in enumerate(lens):
        k[i, :, x:] = float("nan")  # never read
    got = ops.block_means(k, _lens(*lens), block)
    want, mag = _means_want(k.cpu().double(), lens, block)
    assert ((got.cpu().double() - want).abs() <= U * want.abs() + 2.0**-50 * mag + 2.0**-149).all()
    # one key at a time: the means a serving program holds are the same bits
    held = torch.full_like(got, 7.0)
    grown = _lens(*lens)
    for j in range(max(lens)):
        ops.block_means_update(held, k, torch.minimum(grown, torch.full_like(grown, j + 1)), block)
    for i, x in enumerate(lens):
        live = -(-x // block)
        assert torch.equal(held[i, :, :live], got[i, :, :live])
        assert (held[i, :, live:] == 7.0).all() and (got[i, :, live:] == 0).all()


def _select_want(q, means, q_lens, k_lens, block, topk):
    b, h, nq, d = q.shape
    hk, nb = means.shape[1:3]
    out = torch.full((b, hk, nq, topk), -1, dtype=torch.int32)
    qs = q.view(b, hk, h // hk, nq, d).sum(2)
    for i in range(b):
        live = min(-(-k_lens[i] // block), nb)
        sc = qs[i, :, : q_lens[i]] @ means[i, :, :live].transpose(1, 2)
        order = sc.argsort(dim=-1, descending=True, stable=True)[..., :topk]
        out[i, :, : q_lens[i], : order.shape[-1]] = order.sort(-1).values.int()
    return out


@pytest.mark.parametrize("dt", (torch.bfloat16, torch.float16, torch.float32), ids=str)
@pytest.mark.parametrize("shape", [
    # H, Hk, Sq, Sk, D, block, topk, layout
    (4, 4, 50, 300, 64, 16, 8, "bhsd"),
    (8, 2, 33, 700, 128, 1, 5, "bshd"),      # 700 blocks: carried from chunk to chunk
    (3, 1, 17, 300, 24, 1, 64, "bshd"),      # the most that can be chosen
    (2, 2, 16, 40, 32, 16, 8, "odd"),        # more than there are
    (6, 3, 5, 129, 20, 1, 3, "odd"),
    (4, 2, 1, 1000, 128, 1, 16, "bshd"),     # one new token
    (5, 1, 2, 4096, 16, 1, 64, "bhsd"),      # the most blocks
    (1, 1, 2, 90, 7, 2, 1, "odd"),
    (2, 1, 45, 60, 64, 1, 7, "bhsd"),        # up to 64, 128 and 256 blocks
    (3, 3, 37, 120, 128, 1, 16, "bshd"),
    (8, 4, 21, 250, 32, 1, 30, "bhsd"),
    (2, 2, 19, 256, 7, 1, 64, "odd"),
    (1, 1, 18, 257, 64, 1, 9, "bhsd"),
], ids=str)
def test_select(shape, dt):
    h, hk, sq, sk, d, block, topk, layout = shape
    g = _gen(2)
    b = 4
    q, k = _heads(g, b, h, sq, d, dt, layout), _heads(g, b, hk, sk, d, dt, layout)
    kl, ql = [sk, sk // 2 + 1, 1, 0], [sq, max(sq - 3, 1), sq, sq]
    means = ops.block_means(k, _lens(*kl), block)
    got = ops.block_select(q, means, _lens(*ql), _lens(*kl), block, topk)
    want = _select_want(q.cpu().double(), means.cpu().double(), ql, kl, block, topk)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("sq", (1, 20))
def test_close_scores(sq):
    """Scores that differ in their last bits, or past fp32's: the order of float64."""
    gen = _gen(14)
    d = 32
    for nb in (60, 120, 200, 300):
        q = torch.zeros(3, 1, sq, d, device=DEV)
        q[..., 0], q[..., 1] = 1, 2.0**-30
        means = torch.zeros(3, 1, nb, d, device=DEV)
        means[..., 0] = 1 + torch.randint(0, 40, (3, 1, nb), generator=gen).to(DEV) * 2.0**-23
        means[..., 1] = torch.randint(0, 3, (3, 1, nb), generator=gen).to(DEV)
        means[2, ..., 0] *= 1e38  # past fp32 in the group's sum
        q[2] *= 100
        ql, kl = [sq] * 3, [nb, nb - 7, nb]
        for topk in (1, 5, 16):
            got = ops.block_select(q, means, _lens(*ql), _lens(*kl), 1, topk)
            assert torch.equal(got.cpu(), _select_want(q.cpu().double(), means.cpu().double(), ql, kl, 1, topk))


@pytest.mark.parametrize("nb", (200, 300))
@pytest.mark.parametrize("sq", (1, 20))
def test_equal_and_unordered_scores(sq, nb):
    """Ties go to the lower block, a NaN below all, infinities above and below."""
    d = 32
    q = torch.zeros(1, 1, sq, d, device=DEV)
    q[..., 0] = 1
    means = torch.zeros(1, 1, nb, d, device=DEV)
    lens = (_lens(sq), _lens(nb))
    pick = lambda topk: ops.block_select(q, means, *lens, 1, topk)[0, 0]
    assert (pick(5) == torch.arange(5, device=DEV)).all()
    means[0, 0, 150:, 0] = 2.0
    means[0, 0, 7, 0] = -0.0
    assert (pick(nb - 148).cpu() == torch.tensor([0, 1, *range(150, nb)])).all() if nb == 200 else True
    means[0, 0, 3, 0] = float("inf")
    means[0, 0, 160, 0] = float("nan")
    assert (pick(3).cpu() == torch.tensor([3, 150, 151])).all()
    means[0, 0, :, 0] = float("nan")
    means[0, 0, 100, 0] = float("-inf")
    assert (pick(3).cpu() == torch.tensor([0, 1, 100])).all()


# ---- attention ----------------------------------------------------------------------------


def _attend_want(q, k, v, sel, ql, kl, block, dt):
    """out, lse and their bounds (see above), float64 on the CPU."""
    b, h, nq, d = q.shape
    hk, n = k.shape[1:3]
    out, ob = torch.zeros(b, h, nq, d, dtype=torch.float64), torch.zeros(b, h, nq, d, dtype=torch.float64)
    lse = torch.full((b, h, nq), -math.inf, dtype=torch.float64)
    lb = torch.zeros_like(lse)
    half = torch.finfo(dt).eps / 2
    for i in range(b):
        m = min(max(kl[i], 0), n)
        for j in range(h):
            seen = torch.zeros(nq, m, dtype=torch.bool)
            for row in range(min(max(ql[i], 0), nq)):
                for blk in sel[i, j // (h // hk), row].tolist():
                    if 0 <= blk < -(-m // block):
                        seen[row, blk * block : (blk + 1) * block] = True
            kk, vv, qq = k[i, j // (h // hk), :m], v[i, j // (h // hk), :m], q[i, j]
            s = (qq @ kk.T / math.sqrt(d)).masked_fill(~seen, -math.inf)
            e = ((qq.abs() @ kk.T.abs()) / math.sqrt(d)).masked_fill(~seen, 0).amax(-1, keepdim=True) if m else 0
            rows = seen.any(1)
            if not rows.any():
                continue
            top = s.masked_fill(~seen, 0).abs().amax(-1, keepdim=True)
            lse[i, j] = torch.logsumexp(s, -1)
            p = torch.exp(s - lse[i, j][:, None]).masked_fill(~seen, 0)
            out[i, j] = torch.where(rows[:, None], p @ vv, 0.0)
            rel = half + 2 * (d + 2) * U * e + (seen.sum(1, keepdim=True) + 80 + 4 * top) * U
            ob[i, j] = (p @ vv.abs()) * rel + seen.sum(1, keepdim=True) * 2.0**-25 * (vv.abs().max() if m else 0)
            lb[i, j] = ((d + 2) * U * e + (seen.sum(1, keepdim=True) + 80 + 4 * top) * U)[:, 0]
    return out, ob, lse, lb


def _check_attend(q, k, v, sel, ql, kl, block):
    dt = q.dtype
    out, lse = ops.attn_blocks(q, k, v, sel, _lens(*ql), _lens(*kl), block)
    assert out.dtype == dt and out.is_contiguous() and lse.dtype == torch.float32
    want, ob, wl, lb = _attend_want(*(t.detach().cpu().double() for t in (q, k, v)), sel.cpu(), ql, kl,
                                    block, dt)
    empty = wl == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty)
    assert (out.cpu()[empty] == 0).all()
    got = out.detach().cpu().double()
    tol = ob + (want.abs() + ob) * torch.finfo(dt).eps / 2 + torch.finfo(dt).smallest_normal
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), ((got - want).abs() / tol).max().item())
    d = (lse.cpu().double() - wl)[~empty].abs()
    assert (d <= (lb + 4 * U * wl.abs())[~empty]).all()
    return out, lse


ATTN = [
    # B, H, Hk, Sq, Sk, D, block, topk, layout
    (2, 3, 3, 100, 100, 64, 16, 4, "bhsd"),
    (2, 4, 2, 70, 150, 128, 64, 2, "bshd"),
    (2, 8, 1, 30, 200, 32, 32, 3, "bhsd"),
    (2, 4, 4, 65, 90, 24, 16, 3, "bshd"),     # the default network's heads
    (2, 8, 8, 40, 264, 16, 16, 8, "bshd"),    # the benchmark's
    (1, 6, 2, 129, 300, 64, 48, 3, "odd"),    # groups of three, blocks of three tiles
    (1, 5, 1, 20, 70, 20, 16, 2, "odd"),      # a head dim of no vector
    (1, 48, 1, 10, 64, 64, 16, 2, "bhsd"),    # the largest group
    (1, 40, 1, 11, 64, 8, 16, 2, "bhsd"),
    (2, 2, 2, 20, 20, 64, 64, 3, "bhsd"),     # one block, shorter than itself
    (3, 4, 1, 1, 300, 128, 64, 3, "bshd"),    # one new token
    (2, 40, 2, 3, 200, 64, 32, 4, "bhsd"),    # two tiles of heads
    (1, 2, 2, 8, 1100, 32, 16, 64, "bhsd"),   # the most blocks a query can name
    (1, 1, 1, 70, 9000, 16, 16, 8, "bhsd"),   # more blocks than masks are held for
    (2, 2, 1, 33, 256, 128, 128, 1, "bshd"),
    (1, 2, 1, 300, 333, 32, 96, 2, "bhsd"),   # blocks of two stages of 48
    (1, 2, 2, 150, 700, 64, 112, 3, "bshd"),  # of seven of 16
    (1, 48, 1, 20, 200, 128, 64, 2, "bhsd"),
    (1, 3, 3, 270, 2300, 24, 32, 5, "bhsd"),  # two windows of masks
]


@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("shape", ATTN, ids=str)
def test_attend(shape, dt):
    b, h, hk, sq, sk, d, block, topk, layout = shape
    g = _gen(3)
    q, k, v = (_heads(g, b, n, s, d, dt, layout) for n, s in ((h, sq), (hk, sk), (hk, sk)))
    kl = [sk, max(sk - block - 3, 1), 1][:b]
    ql = [sq, max(sq - 2, 1), sq][:b]
    for i, x in enumerate(kl):
        k[i, :, x:], v[i, :, x:] = float("nan"), float("inf")  # past the sequence: never read
    means = ops.block_means(k, _lens(*kl), block)
    _check_attend(q, k, v, ops.block_select(q, means, _lens(*ql), _lens(*kl), block, topk), ql, kl, block)
    # a choice of any form: unordered, repeated, absent
    nb = -(-sk // block)
    sel = torch.randint(-2, nb + 2, (b, hk, sq, topk), generator=g, dtype=torch.int32)
    sel[:, :, ::5] = -1
    sel[..., topk // 2] = sel[..., 0]
    sel[:, :, 3::7, :] = 2**31 - 1
    _check_attend(q, k, v, sel.to(DEV), ql, kl, block)


@pytest.mark.parametrize("sq", (2, 40))
def test_lengths(sq):
    """No keys, no queries, lengths past the tensors, negative ones."""
    g = _gen(4)
    b, h, hk, sk, d, block = 5, 2, 1, 50, 64, 16
    q, k, v = (_heads(g, b, n, s, d, torch.bfloat16) for n, s in ((h, sq), (hk, sk), (hk, sk)))
    sel = torch.arange(3, dtype=torch.int32, device=DEV).expand(b, hk, sq, 3).contiguous()
    ql, kl = [sq, 0, sq + 9, -1, 1], [0, sk, sk + 100, sk, -7]
    out, lse = _check_attend(q, k, v, sel, ql, kl, block)
    assert (out[[0, 1, 3, 4]] == 0).all() and (out[2] != 0).any()
    e = ops.attn_blocks(q, k[:, :, :0], v[:, :, :0], sel, _lens(*ql), _lens(*kl), block)
    assert (e[0] == 0).all() and (e[1] == -math.inf).all()
    e = ops.attn_blocks(q[:0], k[:0], v[:0], sel[:0], _lens(), _lens(), block)
    assert e[0].shape == (0, h, sq, d)
    e = ops.attn_blocks(q[:, :, :0], k, v, sel[:, :, :0], _lens(*ql), _lens(*kl), block)
    assert e[0].shape == (b, h, 0, d)


@pytest.mark.parametrize("sq", (2, 40))
@pytest.mark.parametrize("dt", DTYPES, ids=str)
def test_large_scores(sq, dt):
    """Scores of several hundred: the running maximum keeps every weight in range, and
    rows whose first block is far below their last."""
    g = _gen(5)
    b, h, hk, sk, d, block = 1, 2, 2, 128, 64, 16
    q, k, v = (_heads(g, b, n, s, d, dt) for n, s in ((h, sq), (hk, sk), (hk, sk)))
    q, k = q * 8, k * (1 + torch.arange(sk, device=DEV)[:, None].to(dt) / 8)
    sel = torch.arange(8, dtype=torch.int32, device=DEV).expand(b, hk, sq, 8).contiguous()
    _check_attend(q, k, v, sel, [sq], [sk], block)
    _check_attend(q, k, v, sel.flip(-1), [sq], [sk], block)


@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("bad", ("nan", "inf", "lowest"))
def test_bad_keys_stay_with_their_rows(bad, dt):
    """Keys and values that are not finite, or the type's lowest number, reach the rows that
    chose their block and no other, nor their gradients."""
    gen = _gen(6)
    x = torch.finfo(dt).min if bad == "lowest" else float(bad)
    for sq, block in ((2, 16), (40, 16), (40, 32), (40, 64)):
        q, k, v, g = (_heads(gen, 1, 1, s, 64, dt) for s in (sq, 4 * block, 4 * block, sq))
        sel = torch.zeros(1, 1, sq, 1, dtype=torch.int32, device=DEV)
        sel[:, :, ::2] = 2
        lens = (_lens(sq), _lens(4 * block))
        run = lambda: ops.attn_blocks(q, k, v, sel, *lens, block)
        back = lambda: ops.attn_blocks_backward(g, None, q, k, v, sel, *lens, *run(), block)
        clean, cg = run()[0], back()
        k[0, 0, 2 * block + 3], v[0, 0, 2 * block + 5] = x, x
        (out, lse), grads = run(), back()
        if bad != "lowest":
            assert out[:, :, ::2].isnan().any(-1).all() or out[:, :, ::2].isinf().any(-1).all()
        assert torch.equal(out[:, :, 1::2], clean[:, :, 1::2])
        assert torch.equal(grads[0][:, :, 1::2], cg[0][:, :, 1::2])
        assert all(torch.equal(grads[i][:, :, :block], cg[i][:, :, :block]) for i in (1, 2))


def test_rows_do_not_depend_on_the_batch():
    g = _gen(7)
    b, h, hk, s, d, block, topk = 9, 4, 2, 200, 64, 16, 4
    q, k, v = (_heads(g, b, n, s, d, torch.bfloat16) for n in (h, hk, hk))
    lens = _lens(*[s - 7 * i for i in range(b)])
    run = lambda i: ops.attn_blocks(q[i], k[i], v[i], ops.block_select(
        q[i], ops.block_means(k[i], lens[i], block), lens[i], lens[i], block, topk), lens[i], lens[i], block)
    full = run(slice(0, b))
    for i in (0, 4, 8):
        one = run(slice(i, i + 1))
        assert all(torch.equal(a[i : i + 1], c) for a, c in zip(full, one))


# ---- gradients -----------------------------------------------------------------------------


def _grad_want(q, k, v, sel, ql, kl, block, g, g_lse, dt):
    """Float64 gradients and their bounds: p is off by rp relative (E for the score and for
    lse, see above) and by H where it is an operand; dp by (d + 2) U of its magnitudes;
    delta by g times the bound and the rounding of out; ds by these and H; sums by a step
    of U per term."""
    b, h, nq, d = q.shape
    hk, n = k.shape[1:3]
    half, scale = torch.finfo(dt).eps / 2, 1 / math.sqrt(d)
    out, ob, lse, _ = _attend_want(q, k, v, sel, ql, kl, block, dt)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    eq, ek, ev = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i in range(b):
        m = min(max(kl[i], 0), n)
        for j in range(h):
            c = j // (h // hk)
            seen = torch.zeros(nq, m, dtype=torch.bool)
            for row in range(min(max(ql[i], 0), nq)):
                for blk in sel[i, c, row].tolist():
                    if 0 <= blk < -(-m // block):
                        seen[row, blk * block : (blk + 1) * block] = True
            if not seen.any():
                continue
            qq, kk, vv, gg = q[i, j], k[i, c, :m], v[i, c, :m], g[i, j]
            s = (qq @ kk.T * scale).masked_fill(~seen, 0)
            p = torch.where(seen, torch.exp(s - lse[i, j][:, None]), 0.0)
            e = (qq.abs() @ kk.T.abs() * scale * (d + 2) * U).masked_fill(~seen, 0).amax(-1, keepdim=True)
            rp = 2 * e + (seen.sum(1, keepdim=True) + 90 + 8 * s.abs().amax(-1, keepdim=True)) * U
            tiny = 2.0**-25 if dt == torch.float16 else 0.0
            dp, edp = gg @ vv.T, (d + 2) * U * (gg.abs() @ vv.abs().T)
            delta = (gg * out[i, j]).sum(-1, keepdim=True) - g_lse[i, j][:, None]
            edelta = (gg.abs() * (ob[i, j] + half * out[i, j].abs())).sum(-1, keepdim=True) + (d + 4) * U * (
                (gg * out[i, j]).abs().sum(-1, keepdim=True) + g_lse[i, j].abs()[:, None])
            ds = p * scale * (dp - delta)
            eds = p * scale * ((dp.abs() + delta.abs()) * (rp + 6 * U) + edp + edelta) + half * ds.abs() + tiny * seen
            rows = seen.any(1, keepdim=True)
            dq[i, j] = torch.where(rows, ds @ kk, 0.0)
            eq[i, j] = torch.where(rows, eds @ kk.abs() + (m + 8) * U * (ds.abs() @ kk.abs()), 0.0)
            dk[i, c, :m] += ds.T @ qq
            ek[i, c, :m] += eds.T @ qq.abs() + (nq * (h // hk) + 8) * U * (ds.abs().T @ qq.abs())
            dv[i, c, :m] += p.T @ gg
            ev[i, c, :m] += (p * (rp + half) + tiny * seen).T @ gg.abs() + (nq * (h // hk) + 8) * U * (p.T @ gg.abs())
    return (dq, eq), (dk, ek), (dv, ev)


def _check_grads(q, k, v, sel, ql, kl, block, g, g_lse):
    dt = q.dtype
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out, lse = ops.attn_blocks(q, k, v, sel, _lens(*ql), _lens(*kl), block)
    if g_lse is None:
        grads = torch.autograd.grad(out, [q, k, v], g)
    else:
        grads = torch.autograd.grad([out, lse], [q, k, v], [g, g_lse])
    gl = torch.zeros(q.shape[:3], dtype=torch.float64) if g_lse is None else g_lse.cpu().double()
    clean = lambda t, lens: torch.stack([torch.where(torch.arange(t.shape[2])[:, None] < lens[i], t[i], 0.0)
                                         for i in range(t.shape[0])])
    want = _grad_want(q.detach().cpu().double(), clean(k.detach().cpu().double(), kl),
                      clean(v.detach().cpu().double(), kl), sel.cpu(), ql, kl, block, g.cpu().double(), gl, dt)
    for name, got, (x, err) in zip("qkv", grads, want):
        assert got.dtype == dt and got.shape == x.shape
        y = got.cpu().double()
        tol = err + (x.abs() + err) * torch.finfo(dt).eps / 2 + torch.finfo(dt).smallest_normal
        bad = ~((y - x).abs() <= tol)
        assert not bad.any(), (name, int(bad.sum()), ((y - x).abs() / tol).max().item())
    return grads


@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("shape", ATTN, ids=str)
def test_gradients(shape, dt):
    b, h, hk, sq, sk, d, block, topk, layout = shape
    gen = _gen(8)
    q, k, v = (_heads(gen, b, n, s, d, dt, layout) for n, s in ((h, sq), (hk, sk), (hk, sk)))
    kl = [sk, max(sk - block - 3, 1), 1][:b]
    ql = [sq, max(sq - 2, 1), sq][:b]
    for i, x in enumerate(kl):
        k[i, :, x:], v[i, :, x:] = float("nan"), float("inf")
    g = _heads(gen, b, h, sq, d, dt, layout)
    means = ops.block_means(k, _lens(*kl), block)
    sel = ops.block_select(q, means, _lens(*ql), _lens(*kl), block, topk)
    first = _check_grads(q, k, v, sel, ql, kl, block, g, None)
    again = _check_grads(q, k, v, sel, ql, kl, block, g, None)
    assert all(torch.equal(a, c) for a, c in zip(first, again))
    nb = -(-sk // block)
    sel = torch.randint(-2, nb + 2, (b, hk, sq, topk), generator=gen, dtype=torch.int32)
    sel[:, :, ::5] = -1
    sel[..., topk // 2] = sel[..., 0]
    _check_grads(q, k, v, sel.to(DEV), ql, kl, block, g, torch.randn(b, h, sq, generator=gen).to(DEV))


def test_gradients_of_empty_rows():
    """Nothing flows from rows without a key or past q_lens, whatever their gradient."""
    gen = _gen(9)
    b, h, hk, sq, sk, d, block = 3, 2, 1, 40, 50, 64, 16
    q, k, v = (_heads(gen, b, n, s, d, torch.bfloat16) for n, s in ((h, sq), (hk, sk), (hk, sk)))
    sel = torch.zeros(b, hk, sq, 2, dtype=torch.int32, device=DEV)
    sel[:, :, ::2] = -1
    g = _heads(gen, b, h, sq, d, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    lens = (_lens(sq, 10, 0), _lens(0, 20, sk))
    out, lse = ops.attn_blocks(*leaves, sel, *lens, block)
    clean = torch.autograd.grad(out, leaves, g, retain_graph=True)
    g[:, :, ::2], g[0], g[1, :, 10:], g[2] = (float("nan"),) * 4
    grads = torch.autograd.grad(out, leaves, g)
    assert all(torch.equal(a, c) for a, c in zip(clean, grads))
    assert all((t[0] == 0).all() and (t[2] == 0).all() for t in grads)
    assert (grads[0][1, :, 1:10:2] != 0).any() and (grads[1][1, :, 16:] == 0).all()
    # no queries: the keys' gradients are zeros; no keys: the queries'
    e = ops.attn_blocks_backward(g[:, :, :0], None, q[:, :, :0], k, v, sel[:, :, :0], *lens,
                                 out[:, :, :0], lse[:, :, :0], block)
    assert (e[1] == 0).all() and (e[2] == 0).all()
    e = ops.attn_blocks_backward(g, None, q, k[:, :, :0], v[:, :, :0], sel, *lens, out, lse, block)
    assert (e[0] == 0).all() and e[1].shape == (b, hk, 0, d)


def test_gradient_against_differences():
    """Directional derivatives of a weighted sum of out and lse against central differences
    of the float64 restatement at a fixed choice (fp16 operands: each gradient's own bounds,
    H and some roundings, stay below 1e-2 of the sum of magnitudes)."""
    gen = _gen(10)
    b, h, hk, s, d, block = 1, 4, 2, 60, 32, 16
    q, k, v = (_heads(gen, b, n, s, d, torch.float16).requires_grad_() for n in (h, hk, hk))
    sel = torch.randint(0, 4, (b, hk, s, 2), generator=gen, dtype=torch.int32)
    out, lse = ops.attn_blocks(q, k, v, sel.to(DEV), _lens(s), _lens(s), block)
    g = torch.randn(out.shape, generator=gen).half()
    gl = torch.randn(lse.shape, generator=gen)
    grads = torch.autograd.grad([out, lse], [q, k, v], [g.to(DEV), gl.to(DEV)])
    base = [t.detach().cpu().double() for t in (q, k, v)]
    for i in range(3):
        d_i = torch.randn(base[i].shape, generator=gen).double()

        def f(t):
            x = [c + t * d_i if j == i else c for j, c in enumerate(base)]
            o, _, ls, _ = _attend_want(*x, sel, [s], [s], block, torch.float16)
            return (o * g.double()).sum() + (ls * gl.double()).sum()

        want = ((f(1e-5) - f(-1e-5)) / 2e-5).item()
        part = grads[i].cpu().double() * d_i
        assert abs(part.sum().item() - want) <= 1e-2 * part.abs().sum().item()


# ---- together, captured, on other streams ----------------------------------------------------


def test_norm_choice_attention_together():
    """The four operators in a row, as an attention block uses them, forward and backward,
    against the same row in float64 from the kernels' own choice: gradients within 5 % of
    their norms (each stage rounds to bf16: some 2^-8 each, amplified by the norm)."""
    gen = _gen(11)
    b, h, hk, s, d, block, topk = 2, 4, 2, 150, 64, 16, 4
    x = torch.randn(b, s, h + 2 * hk, d, generator=gen).to(torch.bfloat16).to(DEV).requires_grad_()
    w = (1 + 0.2 * torch.randn(2, d, generator=gen)).to(DEV).requires_grad_()
    pos = torch.randint(-20, 20, (b, s, 2), generator=gen, dtype=torch.int32).to(DEV)
    freqs = 100.0 ** (-torch.arange(16, dtype=torch.float32, device=DEV) / 16)
    lens = _lens(s, s - 30)

    def block_of(x, w):
        q, k, v = x.split([h, hk, hk], 2)
        q, k = ops.qk_norm_rope(q.transpose(1, 2), k.transpose(1, 2), w[0], w[1], pos, freqs, [8, 8])
        means = ops.block_means(k.detach(), lens, block)
        sel = ops.block_select(q.detach(), means, lens, lens, block, topk)
        return ops.attn_blocks(q, k, v.transpose(1, 2), sel, lens, lens, block)[0], sel

    out, sel = block_of(x, w)
    g = torch.randn(out.shape, generator=gen).to(torch.bfloat16).to(DEV)
    gx, gw = torch.autograd.grad(out, [x, w], g)
    xc, wc = (t.detach().cpu().double().requires_grad_() for t in (x, w))
    q, k, v = (t.transpose(1, 2) for t in xc.split([h, hk, hk], 2))
    th = pos.cpu().double().repeat_interleave(8, -1)[:, None] * freqs.cpu().double()

    def turn(t, wt):
        t = t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * wt
        a, c = t[..., :16], t[..., 16:32]
        return torch.cat([a * th.cos() - c * th.sin(), c * th.cos() + a * th.sin(), t[..., 32:]], -1)

    q, k = turn(q, wc[0]), turn(k, wc[1])
    k, v = k.repeat_interleave(h // hk, 1), v.repeat_interleave(h // hk, 1)
    member = torch.arange(s) // block
    seen = (sel.cpu().repeat_interleave(h // hk, 1)[..., None] == member).any(-2)
    seen &= torch.arange(s) < lens.cpu()[:, None, None, None]
    rows = seen.any(-1, keepdim=True)
    p = torch.softmax((q @ k.transpose(-1, -2) / 8).masked_fill(~seen, -1e30), -1) * rows
    want = p @ v
    wx, ww = torch.autograd.grad(want, [xc, wc], g.cpu().double())
    for got, ref in ((out, want), (gx, wx), (gw, ww)):
        assert (got.detach().cpu().double() - ref).norm() <= 0.05 * ref.detach().norm()


def test_captured():
    """Means, choice, attention and gradients in a graph, replayed with new inputs and
    eager work between; two graphs beside each other."""
    gen = _gen(12)
    b, h, hk, s, d, block, topk = 2, 4, 2, 130, 64, 16, 4
    lens = _lens(s, s - 20)
    new = lambda n: torch.randn(b, n, s, d, generator=gen).to(torch.bfloat16).to(DEV)
    calls = []
    for _ in range(2):
        ins = [new(h), new(hk), new(hk), new(h)]

        def run(ins=ins):
            q, k, v, g = ins
            means = ops.block_means(k, lens, block)
            ops.block_means_update(means, k, lens, block)
            sel = ops.block_select(q, means, lens, lens, block, topk)
            out, lse = ops.attn_blocks(q, k, v, sel, lens, lens, block)
            one = ops.attn_blocks(q[:, :, :1], k, v, sel[:, :, :1], lens, lens, block)
            return (means, sel, out, lse, *one,
                    *ops.attn_blocks_backward(g, None, q, k, v, sel, lens, lens, out, lse, block))

        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        calls.append((graph, outs, run, ins))
    for _ in range(3):
        for *_, ins in calls:
            for t in ins:
                t.copy_(new(t.shape[1]))
        for graph, *_ in calls:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs, run, _ in calls:
            assert all(torch.equal(a, c) for a, c in zip(outs, run()))


def test_other_stream():
    gen = _gen(13)
    b, h, s, d, block = 2, 2, 100, 64, 16
    q, k, v = (_heads(gen, b, h, s, d, torch.bfloat16) for _ in range(3))
    lens = _lens(s, s)

    def run():
        sel = ops.block_select(q, ops.block_means(k, lens, block), lens, lens, block, 3)
        return ops.attn_blocks(q, k, v, sel, lens, lens, block)[0]

    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert torch.equal(got, want)


def test_refused_on_the_device():
    q = torch.zeros(1, 4, 5, 64, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(1, 2, 40, 64, dtype=torch.bfloat16, device=DEV)
    ql, kl = _lens(5), _lens(40)
    means = ops.block_means(k, kl, 16)
    sel = ops.block_select(q, means, ql, kl, 16, 2)
    good = dict(q=q, k=k, v=k, sel=sel, q_lens=ql, k_lens=kl, block=16)
    ops.attn_blocks(**good)
    wrong = (ValueError, TypeError, RuntimeError)
    for bad in (dict(block=8), dict(block=24), dict(block=0), dict(q=q.float(), k=k.float(), v=k.float()),
                dict(v=k.half()), dict(v=k[:, :1]), dict(k=k[..., :32]), dict(q=q[:, :3]), dict(sel=sel.long()),
                dict(sel=sel[:, :1]), dict(sel=sel[..., :0]), dict(sel=sel.repeat(1, 1, 1, 33)), dict(q_lens=kl[:0]),
                dict(k_lens=kl.float()), dict(k_lens=kl.cpu()), dict(sel=sel.cpu()), dict(k=k.cpu(), v=k.cpu()),
                dict(q=torch.zeros(1, 130, 5, 64, dtype=torch.bfloat16, device=DEV)),
                dict(q=torch.zeros(1, 4, 5, 136, dtype=torch.bfloat16, device=DEV))):
        with pytest.raises(wrong):
            ops.attn_blocks(**{**good, **bad})
    pick = dict(q=q, means=means, q_lens=ql, k_lens=kl, block=16, topk=2)
    for bad in (dict(topk=0), dict(topk=65), dict(block=0), dict(means=means.half()), dict(means=means[:, :, :, :32]),
                dict(q=q[:, :3]), dict(q=q[0]), dict(q_lens=ql.repeat(2)), dict(means=means.cpu()),
                dict(q=q.double()), dict(means=torch.zeros(1, 2, 4097, 64, device=DEV))):
        with pytest.raises(wrong):
            ops.block_select(**{**pick, **bad})
    for bad in (dict(block=0), dict(k=k.int()), dict(k=k[0]), dict(k_lens=kl.cpu()),
                dict(k=torch.zeros(1, 1, 4097, 64, device=DEV), block=1),
                dict(k=torch.zeros(1, 1, 4, 129, device=DEV))):
        with pytest.raises(wrong):
            ops.block_means(**{**dict(k=k, k_lens=kl, block=16), **bad})
    for bad in (means.half(), means[:, :, :2], means.transpose(2, 3).contiguous().transpose(2, 3), means.cpu()):
        with pytest.raises(wrong):
            ops.block_means_update(bad, k, kl, 16)
    out, lse = ops.attn_blocks(**good)
    for bad in (dict(g=out[:, :2]), dict(g=out.half()), dict(lse=lse.half()), dict(g_lse=lse[:, :2]),
                dict(out=out[..., :32])):
        with pytest.raises(wrong):
            ops.attn_blocks_backward(**{**dict(g=out, g_lse=None, out=out, lse=lse), **good, **bad})


def test_lengths_of_64_bits_and_means_off_a_boundary():
    g = _gen(41)
    q, k = _heads(g, 2, 4, 20, 64, torch.bfloat16), _heads(g, 2, 2, 700, 64, torch.bfloat16)
    ql, kl = _lens(20, 17), _lens(700, 333)
    means = ops.block_means(k, kl, 16)
    sel = ops.block_select(q, means, ql, kl, 16, 5)
    # 2^32 + 5 rows are all of them, not 5
    far = torch.tensor([2**32 + 5, 333], device=DEV)
    assert torch.equal(ops.block_means(k, far, 16), means)
    assert torch.equal(ops.block_select(q, means, ql.long() + torch.tensor([2**32, 0], device=DEV), far, 16, 5), sel)
    off = torch.empty(means.numel() + 1, device=DEV)[1:].view(means.shape).copy_(means)
    assert off.data_ptr() % 16 and torch.equal(ops.block_select(q, off, ql, kl, 16, 5), sel)


def test_update_counts_as_a_change():
    k, kl = _heads(_gen(42), 1, 1, 40, 16, torch.float32), _lens(40)
    means = ops.block_means(k, kl, 16)
    w = torch.ones_like(means, requires_grad=True)
    loss = (w * means).sum()
    ops.block_means_update(means, k, kl, 16)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with pytest.raises(RuntimeError, match="carry no gradient"):
        ops.block_means_update(means.requires_grad_(), k, kl, 16)
    with torch.inference_mode():
        held = torch.zeros(1, 1, 3, 16, device=DEV)
        ops.block_means_update(held, k, kl, 16)
    assert torch.equal(held[:, :, 2], means.detach()[:, :, 2])


def test_gradients_without_heads():
    k = _heads(_gen(43), 2, 2, 50, 64, torch.bfloat16)
    q, sel = k.new_empty(2, 0, 40, 64), torch.zeros(2, 2, 40, 1, dtype=torch.int32, device=DEV)
    args = q, k, k, sel, _lens(40, 40), _lens(50, 20)
    out, lse = ops.attn_blocks(*args, 16)
    dq, dk, dv = ops.attn_blocks_backward(out, None, *args, out, lse, 16)
    assert out.shape == dq.shape == q.shape
    for x in (dk, dv):
        assert x.shape == k.shape and not x.any()


@pytest.mark.parametrize("d", (64, 60))
def test_saved_tensors_that_come_back_elsewhere(d):
    """Checkpointing and saved-tensor hooks free or replace what the forward read."""
    from torch.utils.checkpoint import checkpoint

    g = _gen(44)
    b, h, hk, n, block, topk = 2, 4, 2, 100, 16, 3
    q0, k0 = _heads(g, b, h, n, d, torch.bfloat16), _heads(g, b, hk, n, d, torch.bfloat16)
    sel = torch.randint(0, 7, (b, hk, n, topk), generator=g, dtype=torch.int32).to(DEV)
    ql, kl = _lens(100, 63), _lens(100, 80)
    w = torch.rand(d, generator=g).to(DEV)
    pos = torch.arange(n, dtype=torch.int32, device=DEV).unsqueeze(1)
    freqs = torch.rand(d // 2, generator=g).to(DEV)

    def layer(q, k):
        qn, kn = ops.qk_norm_rope(q, k, w, w, pos, freqs, [d // 2])
        qn, kn = ops.rope_axes(qn, pos * 2, freqs * 1.0, [d // 2]), kn * 1.0
        out, lse = ops.attn_blocks(qn, kn, kn + 1, sel, ql, kl, block)
        return out * 2.0, lse.clamp(min=-30.0)

    def grads(run):
        q, k = q0.clone().requires_grad_(), k0.clone().requires_grad_()
        out, lse = run(q, k)
        junk = [torch.full_like(out, 5.0) for _ in range(8)]  # over what was freed
        got = torch.autograd.grad(out.float().square().sum() + lse.sum(), [q, k])
        del junk
        return got

    want = grads(layer)

    def moved(q, k):
        with torch.autograd.graph.save_on_cpu():
            return layer(q, k)

    for run in (moved, lambda q, k: checkpoint(layer, q, k, use_reentrant=False)):
        for a, e in zip(grads(run), want):
            assert torch.equal(a, e)


def test_sizes_that_would_wrap_are_refused():
    k, ql, kl = _heads(_gen(45), 1, 1, 100, 64, torch.bfloat16), _lens(100), _lens(100)
    means = ops.block_means(k, kl, 16)
    sel = ops.block_select(k, means, ql, kl, 16, 2)
    for block in (0, -16, 2**31, 2**32 + 16):
        for call in (lambda: ops.block_means(k, kl, block), lambda: ops.block_means_update(means, k, kl, block),
                     lambda: ops.block_select(k, means, ql, kl, block, 2),
                     lambda: ops.attn_blocks(k, k, k, sel, ql, kl, block)):
            with pytest.raises(ValueError, match="block"):
                call()
    with pytest.raises(ValueError, match="sizes below"):
        ops.block_means(k[:, :, :1, :1].expand(1, 2**31, 1, 1), kl, 16)
    with pytest.raises(ValueError, match="sizes below"):
        ops.rope_axes(k[:, :, :1, :2].expand(1, 2**31, 1, 2), torch.zeros(1, 1, device=DEV), torch.ones(1, device=DEV),
                      [1])
    with pytest.raises(ValueError, match="means"):
        ops.block_select(k[:, :0], means, ql, kl, 16, 2)


@pytest.mark.parametrize("block,d,dt", [(16, 64, torch.bfloat16), (32, 40, torch.float16), (48, 64, torch.bfloat16),
                                        (64, 64, torch.float16)], ids=str)
def test_many_workgroups(block, d, dt):
    """Enough rows for the workgroups that take more of them at a time."""

    b, h, sq, sk, topk = 50, 4, 257, 70, 2
    gen = _gen(46)
    q, k, v, g = (_heads(gen, b, h, n, d, dt) for n in (sq, sk, sk, sq))
    ql, kl = [sq - i % 3 for i in range(b)], [sk - i for i in range(b)]
    means = ops.block_means(k, _lens(*kl), block)
    sel = ops.block_select(q, means, _lens(*ql), _lens(*kl), block, topk)
    out, lse = _check_attend(q, k, v, sel, ql, kl, block)
    _check_grads(q, k, v, sel, ql, kl, block, g, None)
    # non-finite keys of one block stay with the rows that chose it; the others are within
    # the bound of the same exact result (their blocks may be taken one by one: other sums)
    want, ob, _, _ = _attend_want(*(t[:1, :1].cpu().double() for t in (q, k, v)), sel[:1, :1].cpu(), ql, kl, block, dt)
    k[0, 0, 17] = float("inf")
    again, _ = ops.attn_blocks(q, k, v, sel, _lens(*ql), _lens(*kl), block)
    chose = (sel[0, 0] == 17 // block).any(-1).cpu()
    assert torch.equal(again[1:], out[1:]) and torch.equal(again[0, 1:], out[0, 1:])
    tol = ob + (want.abs() + ob) * torch.finfo(dt).eps / 2 + torch.finfo(dt).smallest_normal
    assert ((again[0, 0].cpu().double() - want[0, 0]).abs() <= tol[0, 0])[~chose].all()


@pytest.mark.parametrize("dt", DTYPES, ids=str)
def test_gradients_over_many_keys(dt):
    """Weights and score gradients far below the type's smallest normal number. The results'
    rounding alone is within H of each element, so of the norm; its mean square is a third of
    that (eps / 2 over sqrt 3), and what the sums of two numbers add is far below the rest.
    Results below the smallest normal number are off by half of its step."""

    b, h, hk, sq, sk, d, block, topk = 1, 2, 1, 40, 4096, 64, 64, 64
    gen = _gen(47)
    q, k, v, g = (_heads(gen, b, n, s, d, dt) for n, s in ((h, sq), (hk, sk), (hk, sk), (h, sq)))
    g = g * 2.0**-6
    sel = torch.arange(64, dtype=torch.int32, device=DEV).expand(b, hk, sq, topk).contiguous()
    x = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out, _ = ops.attn_blocks(*x, sel, _lens(sq), _lens(sk), block)
    got = torch.autograd.grad(out, x, g)
    y = [t.detach().cpu().double().requires_grad_() for t in (q, k, v)]
    p = torch.softmax(y[0] @ y[1].transpose(2, 3) / math.sqrt(d), -1)
    # delta = g . out with out as it was rounded
    want_v = p.transpose(2, 3) @ g.cpu().double()
    ds = p * (g.cpu().double() @ y[2].transpose(2, 3) - (g.double() * out.detach().double()).sum(-1, keepdim=True).cpu()) / math.sqrt(d)
    want = ds @ y[1], (ds.transpose(2, 3) @ y[0]).sum(1, keepdim=True), want_v.sum(1, keepdim=True)
    for name, a, e in zip("qkv", got, want):
        tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2 * math.sqrt(e.numel())
        assert (a.cpu().double() - e).norm() <= torch.finfo(dt).eps / 2 * e.norm() + tiny, name
