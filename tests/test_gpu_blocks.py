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
def test_equal_and_unordered_scores(sq):
    """Ties go to the lower block, a NaN below all, infinities above and below."""
    d, nb = 32, 200
    q = torch.zeros(1, 1, sq, d, device=DEV)
    q[..., 0] = 1
    means = torch.zeros(1, 1, nb, d, device=DEV)
    lens = (_lens(sq), _lens(nb))
    pick = lambda topk: ops.block_select(q, means, *lens, 1, topk)[0, 0]
    assert (pick(5) == torch.arange(5, device=DEV)).all()
    means[0, 0, 150:, 0] = 2.0
    means[0, 0, 7, 0] = -0.0
    assert (pick(52).cpu() == torch.tensor([0, 1, *range(150, 200)])).all()
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
    (1, 64, 1, 10, 64, 64, 16, 2, "bhsd"),    # the largest group
    (1, 40, 1, 11, 64, 8, 16, 2, "bhsd"),
    (2, 2, 2, 20, 20, 64, 64, 3, "bhsd"),     # one block, shorter than itself
    (3, 4, 1, 1, 300, 128, 64, 3, "bshd"),    # one new token
    (2, 40, 2, 3, 200, 64, 32, 4, "bhsd"),    # two tiles of heads
    (1, 2, 2, 8, 1100, 32, 16, 64, "bhsd"),   # the most blocks a query can name
    (1, 1, 1, 70, 9000, 16, 16, 8, "bhsd"),   # more blocks than masks are held for
    (2, 2, 1, 33, 256, 128, 128, 1, "bshd"),
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


def test_infinities_stay_with_their_rows():
    """A key of infinities gives NaN to the rows that chose its block and to no other."""
    g = _gen(6)
    for sq in (2, 40):
        q, k, v = (_heads(g, 1, 1, s, 64, torch.bfloat16) for s in (sq, 64, 64))
        sel = torch.zeros(1, 1, sq, 1, dtype=torch.int32, device=DEV)
        sel[:, :, ::2] = 2
        clean, _ = ops.attn_blocks(q, k, v, sel, _lens(sq), _lens(64), 16)
        k[0, 0, 40], v[0, 0, 41] = float("nan"), float("inf")
        out, lse = ops.attn_blocks(q, k, v, sel, _lens(sq), _lens(64), 16)
        assert out[:, :, ::2].isnan().all() and lse[:, :, ::2].isnan().all()
        assert torch.equal(out[:, :, 1::2], clean[:, :, 1::2])


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
