"""Sparse attention over blocks of keys that a cheap score selects for each query.

A sequence's keys fall into blocks of ``block``. ``shrimp::block_means`` keeps
one mean key per block, ``shrimp::block_select`` gives every query the ``topk``
blocks whose mean has the largest product with it, and ``shrimp::attn_blocks``
attends to those blocks only: beside ``shrimp::attn_pair`` and
``hexfield_eq::ray_attn`` the form whose cost per query does not grow with the
support. Query heads may share key heads (H a multiple of Hk); the heads of a
group choose together. The choice carries no gradient; the attention does, in q,
k and v.

    means = block_means(k, k_lens, 64)
    sel = block_select(q, means, q_lens, k_lens, 64, 16)
    out, lse = attn_blocks(q, k, v, sel, q_lens, k_lens, 64)

A serving program holds the means beside its cache of keys and calls
``block_means_update`` when a key was added.

Inputs live on a ROCm device; there is no CPU path.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._oplib import below, check_sizes, copies, define, direct, hooked, places, wants_grad

MAX_HEAD_DIM = 128
MAX_TOPK = 64
MAX_BLOCKS = 4096
MAX_GROUP = 48
MAX_KEYS = 2**30
MAX_ATTN_BLOCK = 2**20

_DT = {
    torch.float32: _lib.DT_F32,
    torch.float16: _lib.DT_F16,
    torch.bfloat16: _lib.DT_BF16,
}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t (B, heads, S, D) with a head's dimensions beside each other."""

    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_heads(what: str, name: str, t: torch.Tensor, types=_DT) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what}: the shrimp MI355X build runs on a ROCm device only "
                           f"(got {name} on {t.device})")
    if t.dim() != 4:
        raise ValueError(f"{what}: {name} must be (B, heads, S, D), got {tuple(t.shape)}")
    if t.dtype not in types:
        raise TypeError(f"{what}: {name} is {t.dtype}, one of "
                        f"{', '.join(str(x) for x in types)} expected")
    check_sizes(what, name, t)
    if not 1 <= t.shape[3] <= MAX_HEAD_DIM:
        raise ValueError(f"{what}: head dim {t.shape[3]} outside [1, {MAX_HEAD_DIM}]")


def _lens(what: str, name: str, lens: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    if lens.dtype not in (torch.int32, torch.int64) or tuple(lens.shape) != (like.shape[0],):
        raise ValueError(f"{what}: {name} {lens.dtype} {tuple(lens.shape)}; int32 "
                         f"({like.shape[0]},) expected")
    if lens.device != like.device:
        raise ValueError(f"{what}: {name} on {lens.device}, queries or keys on {like.device}")
    if lens.dtype == torch.int64:
        lens = lens.clamp(-1, MAX_KEYS)  # (2^32 + 5 is not 5)
    return lens.to(torch.int32).contiguous()


def _blocks(what: str, keys: int, block: int) -> int:
    if not 1 <= block <= MAX_KEYS or keys > MAX_KEYS:
        raise ValueError(f"{what}: block of {block} keys of {keys}, 1 to {MAX_KEYS} expected")
    nb = -(-keys // block)
    if nb > MAX_BLOCKS:
        raise ValueError(f"{what}: {keys} keys in blocks of {block} are {nb} blocks, at most "
                         f"{MAX_BLOCKS}")
    return nb


# ---- block_means, block_means_update -----------------------------------------------------------


def _launch_means(what, k, k_lens, block, means, last_only):
    k = _rows(k)
    lens = _lens(what, "k_lens", k_lens, k)
    b, hk, n, d = k.shape
    _lib.launch(_lib.load().shrimp_block_means, k.device, what, k.data_ptr(), *k.stride()[:3],
                _DT[k.dtype], lens.data_ptr(), means.data_ptr(), b, hk, n, d, block, last_only)


def _means_kernel(k, k_lens, block):
    what = "shrimp::block_means"
    _check_heads(what, "k", k)
    nb = _blocks(what, k.shape[2], block)
    means = torch.empty((k.shape[0], k.shape[1], nb, k.shape[3]), dtype=torch.float32, device=k.device)
    _launch_means(what, k, k_lens, block, means, 0)
    return means


def _means_fake(k, k_lens, block):
    return k.new_empty((k.shape[0], k.shape[1], -(-k.shape[2] // block), k.shape[3]),
                       dtype=torch.float32)


_block_means = define("block_means(Tensor k, Tensor k_lens, int block) -> Tensor",
                      _means_kernel, _means_fake)


def block_means(k: torch.Tensor, k_lens: torch.Tensor, block: int) -> torch.Tensor:
    """(B, Hk, ceil(Sk / block), D) float32: the mean of every block's keys below k_lens[b],
    summed in float64; zero for a block without one. k (B, Hk, Sk, D) bfloat16, float16 or
    float32. Carries no gradient."""

    return (_means_kernel if direct(k, k_lens) else _block_means)(k, k_lens, block)


def _update_kernel(means, k, k_lens, block):
    what = "shrimp::block_means_update"
    _check_heads(what, "k", k)
    if means.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what}: means are written in place and carry no gradient")
    want = (k.shape[0], k.shape[1], _blocks(what, k.shape[2], block), k.shape[3])
    if (means.dtype != torch.float32 or tuple(means.shape) != want or not means.is_contiguous()
            or means.device != k.device):
        raise ValueError(f"{what}: means {means.dtype} {tuple(means.shape)} on {means.device}; "
                         f"contiguous float32 {want} on {k.device} expected")
    _launch_means(what, k, k_lens, block, means, 1)
    torch.autograd.graph.increment_version(means)


def _update_fake(means, k, k_lens, block):
    return None


_block_means_update = define(
    "block_means_update(Tensor(a!) means, Tensor k, Tensor k_lens, int block) -> ()",
    _update_kernel, _update_fake)


def block_means_update(means: torch.Tensor, k: torch.Tensor, k_lens: torch.Tensor, block: int) -> None:
    """Writes the mean of the block that holds each sequence's last key, k_lens[b] - 1, in
    place (block 0 for an empty sequence); the other blocks' means stay. The same bits as
    block_means."""

    (_update_kernel if direct(means, k, k_lens) else _block_means_update)(means, k, k_lens, block)


# ---- block_select ----------------------------------------------------------------------------


def _select_kernel(q, means, q_lens, k_lens, block, topk):
    what = "shrimp::block_select"
    _check_heads(what, "q", q)
    b, h, sq, d = q.shape
    if means.dtype != torch.float32 or means.dim() != 4 or means.device != q.device:
        raise ValueError(f"{what}: means {means.dtype} {tuple(means.shape)} on {means.device}; "
                         f"float32 (B, Hk, NB, D) on {q.device} expected")
    hk, nb = means.shape[1], means.shape[2]
    if means.shape[0] != b or means.shape[3] != d or hk < 1 or h < hk or h % hk:
        raise ValueError(f"{what}: means {tuple(means.shape)} for queries {tuple(q.shape)}")
    if not 1 <= block <= MAX_KEYS or nb > MAX_BLOCKS or (nb - 1) * block >= MAX_KEYS:
        raise ValueError(f"{what}: {nb} blocks of {block} keys, at most {MAX_BLOCKS} and "
                         f"{MAX_KEYS} keys")
    if not 1 <= topk <= MAX_TOPK:
        raise ValueError(f"{what}: topk {topk} outside [1, {MAX_TOPK}]")
    q, means = _rows(q), means.contiguous()
    if means.data_ptr() % 16:
        means = means.clone()
    ql, kl = _lens(what, "q_lens", q_lens, q), _lens(what, "k_lens", k_lens, q)
    sel = torch.empty((b, hk, sq, topk), dtype=torch.int32, device=q.device)
    # (of the keys only their number is known here: all blocks full)
    a = _lib.BlockSelectArgs(q.data_ptr(), *q.stride()[:3], means.data_ptr(), ql.data_ptr(),
                             kl.data_ptr(), sel.data_ptr(), b, h, hk, sq, min(nb * block, MAX_KEYS), d,
                             block, topk,
                             _DT[q.dtype])
    _lib.launch(_lib.load().shrimp_block_select, q.device, what, ctypes.byref(a))
    return sel


def _select_fake(q, means, q_lens, k_lens, block, topk):
    return q.new_empty((q.shape[0], means.shape[1], q.shape[2], topk), dtype=torch.int32)


_block_select = define(
    "block_select(Tensor q, Tensor means, Tensor q_lens, Tensor k_lens, int block, int topk) -> Tensor",
    _select_kernel, _select_fake)


def block_select(q: torch.Tensor, means: torch.Tensor, q_lens: torch.Tensor, k_lens: torch.Tensor,
                 block: int, topk: int) -> torch.Tensor:
    """(B, Hk, Sq, topk) int32: for every query row below q_lens[b] the topk blocks (of those
    with keys below k_lens[b]) whose mean has the largest product with the sum of the
    group's queries, ascending, then -1; -1 throughout for later rows. Scores are float64;
    equal ones go to the lower block, NaN ranks lowest. q (B, H, Sq, D); topk <= 64."""

    run = _select_kernel if direct(q, means, q_lens, k_lens) else _block_select
    return run(q, means, q_lens, k_lens, block, topk)


# ---- attn_blocks -----------------------------------------------------------------------------


def _aligned(t: torch.Tensor, d8: int) -> torch.Tensor:
    """t with rows on 16-byte boundaries and a head dim of d8 (zeros behind its own)."""

    if t.shape[3] != d8:
        return torch.nn.functional.pad(t, (0, d8 - t.shape[3]))
    ok = t.stride(3) == 1 and t.data_ptr() % 16 == 0 and not any(s % 8 for s in t.stride()[:3])
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _attn_args(what, q, k, v, sel, q_lens, k_lens, block):
    """(q, k, v, sel, lens checked and laid out; head dim padded to a multiple of 8)"""

    types = (torch.bfloat16, torch.float16)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_heads(what, name, t, types)
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{what}: q is {q.dtype} on {q.device}, {name} {t.dtype} on {t.device}")
    b, h, sq, d = q.shape
    hk = k.shape[1]
    if (k.shape[0], k.shape[3]) != (b, d) or v.shape != k.shape:
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if hk < 1 or h % hk or h // hk > MAX_GROUP:
        raise ValueError(f"{what}: {h} query heads for {hk} key heads (at most {MAX_GROUP} each)")
    if not 16 <= block <= MAX_ATTN_BLOCK or block % 16:
        raise ValueError(f"{what}: blocks of {block} keys, a multiple of 16 up to "
                         f"{MAX_ATTN_BLOCK} expected")
    if (sel.dtype != torch.int32 or sel.dim() != 4 or tuple(sel.shape[:3]) != (b, hk, sq)
            or not 1 <= sel.shape[3] <= MAX_TOPK):
        raise ValueError(f"{what}: sel {sel.dtype} {tuple(sel.shape)}; int32 ({b}, {hk}, {sq}, 1 to "
                         f"{MAX_TOPK}) expected")
    if sel.device != q.device:
        raise ValueError(f"{what}: sel on {sel.device}, q on {q.device}")
    d8 = -(-d // 8) * 8
    return (_aligned(q, d8), _aligned(k, d8), _aligned(v, d8), sel.contiguous(),
            _lens(what, "q_lens", q_lens, q), _lens(what, "k_lens", k_lens, q))


def _attn_struct(q, k, v, sel, ql, kl, out, lse, block, d):
    return _lib.AttnBlocksArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
        sel.data_ptr(), ql.data_ptr(), kl.data_ptr(), out.data_ptr(), lse.data_ptr(), q.shape[0],
        q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], block, sel.shape[3],
        _DT[q.dtype], 1.0 / math.sqrt(d))


def _attn_run(q, k, v, sel, q_lens, k_lens, block):
    """((out, lse), argument struct, tensors it points to)"""

    what = "shrimp::attn_blocks"
    d = q.shape[-1]
    q, k, v, sel, ql, kl = _attn_args(what, q, k, v, sel, q_lens, k_lens, block)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
    a = _attn_struct(q, k, v, sel, ql, kl, out, lse, block, d)
    _lib.launch(_lib.load().shrimp_attn_blocks, q.device, what, ctypes.byref(a))
    return (out if out.shape[3] == d else out[..., :d].contiguous(), lse), a, (q, k, v, sel, ql, kl, out)


def _attn_kernel(q, k, v, sel, q_lens, k_lens, block):
    return _attn_run(q, k, v, sel, q_lens, k_lens, block)[0]


def _attn_fake(q, k, v, sel, q_lens, k_lens, block):
    return q.new_empty(q.shape), q.new_empty(q.shape[:3], dtype=torch.float32)


class _AttnBlocks(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, sel, q_lens, k_lens, block):
        ctx.args = None
        if direct(q, k, v, sel, q_lens, k_lens) and not hooked():
            (out, lse), ctx.args, laid = _attn_run(q, k, v, sel, q_lens, k_lens, block)
            given = (q, k, v, sel, q_lens, k_lens, out)
            ctx.keep, ctx.places = copies(laid, given), places(given + (lse,))
        else:
            out, lse = below(_attn_blocks, q, k, v, sel, q_lens, k_lens, block)
        ctx.save_for_backward(q, k, v, sel, q_lens, k_lens, out, lse)
        ctx.block = block
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, g_lse):
        if g is None and g_lse is None:
            return (None,) * 7
        saved = ctx.saved_tensors
        if g is None:
            g = torch.zeros_like(saved[6])
        if ctx.args is None or not direct(g) or places(saved) != ctx.places:
            grads = _attn_blocks_backward(g, g_lse, *saved, ctx.block)
        else:
            grads = _attn_back_run(ctx.args, g, g_lse, *saved[:2])
        return (*grads, None, None, None, None)


_attn_blocks = define(
    "attn_blocks(Tensor q, Tensor k, Tensor v, Tensor sel, Tensor q_lens, Tensor k_lens, int block)"
    " -> (Tensor, Tensor)", _attn_kernel, _attn_fake, _AttnBlocks)


def attn_blocks(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sel: torch.Tensor,
                q_lens: torch.Tensor, k_lens: torch.Tensor, block: int
                ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out (B, H, Sq, D), lse (B, H, Sq) float32): softmax(q k^T / sqrt(D)) v over the keys
    below k_lens[b] of the blocks that sel (B, Hk, Sq, topk) names for the row, and the log
    of the softmax's sum. Entries of sel outside the sequence's blocks name none, repeated
    ones count once. Rows from q_lens[b] on, and rows without a key, are 0 and -inf. q, k
    and v bfloat16 or float16, H a multiple of Hk; block a multiple of 16. Strides of heads
    and rows are below 2^31 elements."""

    if direct(q, k, v, sel, q_lens, k_lens):
        run = _AttnBlocks.apply if wants_grad(q, k, v) else _attn_kernel
        return run(q, k, v, sel, q_lens, k_lens, block)
    return _attn_blocks(q, k, v, sel, q_lens, k_lens, block)


def _attn_back_run(a, g, g_lse, q, k):
    """Gradients like q and k from the forward's arguments (whose head dim may be padded)."""

    d = q.shape[3]
    g = _aligned(g, a.d)
    g_lse = None if g_lse is None else g_lse.contiguous()
    dq = torch.empty((*q.shape[:3], a.d), dtype=q.dtype, device=q.device)
    dk = torch.empty((*k.shape[:3], a.d), dtype=q.dtype, device=q.device)
    dv = torch.empty((*k.shape[:3], a.d), dtype=q.dtype, device=q.device)
    lib = _lib.load()
    ref = ctypes.byref(a)
    n = lib.shrimp_attn_blocks_workspace(ref)
    ws = torch.empty(max(n, 0), dtype=torch.uint8, device=q.device)
    sb, sh, sn, _ = g.stride()
    gr = _lib.AttnBlocksGrads(g.data_ptr(), sb, sh, sn, _lib.ptr(g_lse), dq.data_ptr(),
                              dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), n)
    _lib.launch(lib.shrimp_attn_blocks_backward, q.device, "shrimp::attn_blocks_backward", ref,
                ctypes.byref(gr))
    if a.d == d:
        return dq, dk, dv
    return tuple(t[..., :d].contiguous() for t in (dq, dk, dv))


def _attn_back_kernel(g, g_lse, q, k, v, sel, q_lens, k_lens, out, lse, block):
    what = "shrimp::attn_blocks_backward"
    d = q.shape[-1]
    for name, t, like in (("g", g, q), ("out", out, q)):
        if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
            raise ValueError(f"{what}: {name} {t.dtype} {tuple(t.shape)} on {t.device} for q "
                             f"{like.dtype} {tuple(like.shape)} on {like.device}")
    for name, t in (("lse", lse), ("g_lse", g_lse)):
        if t is not None and (t.dtype != torch.float32 or t.shape != q.shape[:3] or t.device != q.device):
            raise ValueError(f"{what}: {name} {t.dtype} {tuple(t.shape)} on {t.device}")
    laid = _attn_args(what, q, k, v, sel, q_lens, k_lens, block)
    out, lse = _aligned(out, laid[0].shape[3]).contiguous(), lse.contiguous()
    return _attn_back_run(_attn_struct(*laid, out, lse, block, d), g, g_lse, q, k)


def _attn_back_fake(g, g_lse, q, k, v, sel, q_lens, k_lens, out, lse, block):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


_attn_blocks_backward = define(
    "attn_blocks_backward(Tensor g, Tensor? g_lse, Tensor q, Tensor k, Tensor v, Tensor sel,"
    " Tensor q_lens, Tensor k_lens, Tensor out, Tensor lse, int block) -> (Tensor, Tensor, Tensor)",
    _attn_back_kernel, _attn_back_fake)


def attn_blocks_backward(g: torch.Tensor, g_lse: Optional[torch.Tensor], q: torch.Tensor,
                         k: torch.Tensor, v: torch.Tensor, sel: torch.Tensor, q_lens: torch.Tensor,
                         k_lens: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, block: int
                         ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of q, k and v from those of attn_blocks' results (that of lse may be None),
    its arguments and its results. Every sum has a fixed order: the same call gives the same
    bits. In float16 a score's gradient past 2000 makes those of q and k
    not finite."""

    return _attn_blocks_backward(g, g_lse, q, k, v, sel, q_lens, k_lens, out, lse, block)
