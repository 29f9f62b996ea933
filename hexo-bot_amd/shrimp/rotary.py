"""Rotary positions on several axes, and the norm of queries and keys before them.

``shrimp::rope_axes`` turns pairs of a head's dimensions by angles pos * freq,
each pair by one axis of the position (a board's two axial coordinates, a
clip's time, height and width); ``shrimp::qk_norm_rope`` first divides every
query and key head by its root mean square and multiplies a weight, in the same
pass. They stand in front of ``shrimp::attn_pair`` / ``shrimp::attn_blocks`` for
networks whose attention carries positions in its queries and keys in place of
the clamped table of relative offsets. Both are differentiable in their heads
and weights; positions and frequencies get no gradient.

Inputs live on a ROCm device (bfloat16, float16 or float32); results are
contiguous and of the input's type. There is no CPU path.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from ._oplib import below, check_sizes, copies, define, direct, hooked, places, wants_grad

MAX_AXES = 4
MAX_HEAD_DIM = 256

_DT = {
    torch.float32: _lib.DT_F32,
    torch.float16: _lib.DT_F16,
    torch.bfloat16: _lib.DT_BF16,
}
_POS_DT = {torch.int32: _lib.DT_I32, torch.int64: _lib.DT_I64, torch.float32: _lib.DT_F32}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t (B, heads, S, D) with a head's dimensions beside each other."""

    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_heads(what: str, q: torch.Tensor, k: Optional[torch.Tensor]) -> None:
    for name, t in (("q", q), ("k", k)):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{what}: the shrimp MI355X build runs on a ROCm device only "
                               f"(got {name} on {t.device})")
        if t.dim() != 4:
            raise ValueError(f"{what}: {name} must be (B, heads, S, D), got {tuple(t.shape)}")
        if t.dtype not in _DT:
            raise TypeError(f"{what}: {name} is {t.dtype}; bfloat16, float16 or float32 expected")
        check_sizes(what, name, t)
    if not 1 <= q.shape[3] <= MAX_HEAD_DIM:
        raise ValueError(f"{what}: head dim {q.shape[3]} outside [1, {MAX_HEAD_DIM}]")
    if k is not None:
        if k.dtype != q.dtype or k.device != q.device:
            raise ValueError(f"{what}: q is {q.dtype} on {q.device}, k {k.dtype} on {k.device}")
        if (k.shape[0], k.shape[2], k.shape[3]) != (q.shape[0], q.shape[2], q.shape[3]):
            raise ValueError(f"{what}: q {tuple(q.shape)} and k {tuple(k.shape)} differ in more "
                             "than their heads")


def _args(what, q, k, pos, freqs, sections, interleaved, inverse, eps=0.0, q_w=None, k_w=None,
          gq=None, gk=None):
    """(argument struct, outputs, tensors that the launch reads) of one call; with the
    gradients gq and gk these are checked, and no outputs made."""

    _check_heads(what, q, k)
    b, h, s, d = q.shape
    sections = [int(n) for n in sections]
    axes = len(sections)
    if not 1 <= axes <= MAX_AXES or min(sections) < 0 or 2 * sum(sections) > d:
        raise ValueError(f"{what}: sections {sections} for a head of {d} dimensions (1 to "
                         f"{MAX_AXES} axes, two dimensions per pair)")
    if pos.dtype not in _POS_DT:
        raise TypeError(f"{what}: positions are {pos.dtype}; int32, int64 or float32 expected")
    if pos.dim() == 2:
        pos = pos.unsqueeze(0)
    if (pos.dim() != 3 or pos.shape[0] not in (1, b) or tuple(pos.shape[1:]) != (s, axes)):
        raise ValueError(f"{what}: positions {tuple(pos.shape)} for {b} sequences of {s} rows and "
                         f"{axes} axes")
    pos = pos.expand(b, s, axes)
    if freqs.dtype not in (torch.float32, torch.float64) or tuple(freqs.shape) != (sum(sections),):
        raise ValueError(f"{what}: frequencies {freqs.dtype} {tuple(freqs.shape)}; float32 or "
                         f"float64 ({sum(sections)},) expected")
    freqs = freqs.contiguous()
    w_dt = _lib.DT_F32
    if q_w is not None:
        if q_w.dtype != k_w.dtype or q_w.dtype not in _DT:
            raise TypeError(f"{what}: weights {q_w.dtype} and {k_w.dtype}; one of bfloat16, "
                            "float16 and float32 expected")
        if tuple(q_w.shape) != (d,) or tuple(k_w.shape) != (d,):
            raise ValueError(f"{what}: weights {tuple(q_w.shape)} and {tuple(k_w.shape)}, "
                             f"({d},) expected")
        if not eps > 0:
            raise ValueError(f"{what}: eps must be positive")
        w_dt = _DT[q_w.dtype]
        q_w, k_w = q_w.contiguous(), k_w.contiguous()
    for name, t in (("positions", pos), ("frequencies", freqs), ("q_weight", q_w), ("k_weight", k_w)):
        if t is not None and t.device != q.device:
            raise ValueError(f"{what}: {name} on {t.device}, q on {q.device}")
    q = _rows(q)
    hk, k_st, q_out, k_out = 0, (0, 0, 0), None, None
    if k is not None:
        k = _rows(k)
        hk, k_st = k.shape[1], k.stride()
    if gq is not None:
        for name, g, t in (("gq", gq, q), ("gk", gk, k)):
            if g.shape != t.shape or g.dtype != t.dtype or g.device != t.device:
                raise ValueError(f"{what}: {name} {g.dtype} {tuple(g.shape)} on {g.device} for "
                                 f"{t.dtype} {tuple(t.shape)} on {t.device}")
        gq, gk = _rows(gq), _rows(gk)
    else:
        q_out = torch.empty((b, h, s, d), dtype=q.dtype, device=q.device)
        if k is not None:
            k_out = torch.empty((b, hk, s, d), dtype=q.dtype, device=q.device)
    a = _lib.RopeArgs(
        q.data_ptr(), _lib.ptr(k), *q.stride()[:3], *k_st[:3],
        pos.data_ptr(), *pos.stride(), freqs.data_ptr(), _lib.ptr(q_w), _lib.ptr(k_w),
        _lib.ptr(q_out), _lib.ptr(k_out), None, None, 0, 0, 0, 0, 0, 0,
        b, s, h, hk, d, axes, (ctypes.c_int32 * MAX_AXES)(*sections), _DT[q.dtype],
        _POS_DT[pos.dtype], int(freqs.dtype == torch.float64), w_dt, int(interleaved),
        int(inverse), eps,
    )
    return a, q_out, k_out, (q, k, pos, freqs, q_w, k_w, gq, gk)


# ---- rope_axes -----------------------------------------------------------------------------


def _rope_kernel(x, pos, freqs, sections, interleaved=False, inverse=False):
    a, out, _, keep = _args("shrimp::rope_axes", x, None, pos, freqs, sections, interleaved, inverse)
    _lib.launch(_lib.load().shrimp_rope, x.device, "shrimp::rope_axes", ctypes.byref(a))
    del keep
    return out


def _rope_fake(x, pos, freqs, sections, interleaved=False, inverse=False):
    return x.new_empty(x.shape)


class _RopeAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, freqs, sections, interleaved, inverse):
        ctx.save_for_backward(pos, freqs)
        ctx.turn = (sections, interleaved, not inverse)
        ctx.args = None
        if not direct(x, pos, freqs) or hooked():
            return below(_rope_axes, x, pos, freqs, sections, interleaved, inverse)
        ctx.args, out, _, laid = _args("shrimp::rope_axes", x, None, pos, freqs, sections,
                                       interleaved, inverse)
        _lib.launch(_lib.load().shrimp_rope, x.device, "shrimp::rope_axes", ctypes.byref(ctx.args))
        ctx.keep, ctx.places = copies(laid[2:4], (pos, freqs)), places((pos, freqs))
        return out

    @staticmethod
    def backward(ctx, g):
        pos, freqs = ctx.saved_tensors
        if (ctx.args is None or wants_grad(g) or not direct(g)
                or places((pos, freqs)) != ctx.places):
            return rope_axes(g, pos, freqs, *ctx.turn), None, None, None, None, None
        g = _rows(g)
        out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
        a = _lib.RopeArgs.from_buffer_copy(ctx.args)
        a.q, a.q_out, a.inverse = g.data_ptr(), out.data_ptr(), int(ctx.turn[2])
        a.q_sb, a.q_sh, a.q_sn, _ = g.stride()
        _lib.launch(_lib.load().shrimp_rope, g.device, "shrimp::rope_axes", ctypes.byref(a))
        return out, None, None, None, None, None


_rope_axes = define(
    "rope_axes(Tensor x, Tensor pos, Tensor freqs, int[] sections, bool interleaved, bool inverse)"
    " -> Tensor", _rope_kernel, _rope_fake, _RopeAxes)


def rope_axes(x: torch.Tensor, pos: torch.Tensor, freqs: torch.Tensor, sections: Sequence[int],
              interleaved: bool = False, inverse: bool = False) -> torch.Tensor:
    """x (B, H, S, D) with the first 2 P dimensions of every head turned in P = sum(sections)
    pairs: pair p by pos[b, s, axis] * freqs[p], the first sections[0] pairs by axis 0, and
    so on. A pair is dimensions (p, P + p), or (2 p, 2 p + 1) with ``interleaved``; further
    dimensions pass. pos (B, S, axes), or (S, axes) for all sequences, int32, int64 or
    float32; freqs (P,) float32 or float64. Angles are formed in float64. ``inverse`` turns
    back."""

    if direct(x, pos, freqs):
        run = _RopeAxes.apply if wants_grad(x) else _rope_kernel
        return run(x, pos, freqs, sections, interleaved, inverse)
    return _rope_axes(x, pos, freqs, sections, interleaved, inverse)


# ---- qk_norm_rope --------------------------------------------------------------------------


def _norm_kernel(q, k, q_weight, k_weight, pos, freqs, sections, eps, interleaved):
    what = "shrimp::qk_norm_rope"
    a, q_out, k_out, keep = _args(what, q, k, pos, freqs, sections, interleaved, False, eps,
                                  q_weight, k_weight)
    _lib.launch(_lib.load().shrimp_rope, q.device, what, ctypes.byref(a))
    del keep
    return q_out, k_out


def _norm_fake(q, k, q_weight, k_weight, pos, freqs, sections, eps, interleaved):
    return q.new_empty(q.shape), k.new_empty(k.shape)


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, pos, freqs, sections, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, pos, freqs)
        ctx.rest = (sections, eps, interleaved)
        ctx.args = None
        if not direct(q, k, q_weight, k_weight, pos, freqs) or hooked():
            return below(_qk_norm_rope, q, k, q_weight, k_weight, pos, freqs, sections, eps, interleaved)
        what = "shrimp::qk_norm_rope"
        ctx.args, q_out, k_out, laid = _args(what, q, k, pos, freqs, sections, interleaved, False, eps,
                                             q_weight, k_weight)
        _lib.launch(_lib.load().shrimp_rope, q.device, what, ctypes.byref(ctx.args))
        given = (q, k, pos, freqs, q_weight, k_weight)
        ctx.keep = copies(laid, given)
        ctx.places = places((q, k, q_weight, k_weight, pos, freqs))
        return q_out, k_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        saved = ctx.saved_tensors
        if ctx.args is None or not direct(gq, gk) or places(saved) != ctx.places:
            grads = _qk_norm_rope_backward(gq, gk, *saved, *ctx.rest)
        else:
            a = _lib.RopeArgs.from_buffer_copy(ctx.args)
            grads = _launch_norm_back(a, _rows(gq), _rows(gk), *saved[:4])
        return (*grads, None, None, None, None, None)


_qk_norm_rope = define(
    "qk_norm_rope(Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor pos, Tensor freqs,"
    " int[] sections, float eps, bool interleaved) -> (Tensor, Tensor)",
    _norm_kernel, _norm_fake, _QkNormRope)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                 pos: torch.Tensor, freqs: torch.Tensor, sections: Sequence[int], eps: float = 1e-6,
                 interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """x / sqrt(mean(x^2) + eps) * weight over the dimensions of every head of q (B, H, S, D)
    and k (B, Hk, S, D), then rope_axes, in one launch with fp32 statistics. Weights (D,) of
    one type (bfloat16, float16 or float32)."""

    if direct(q, k, q_weight, k_weight, pos, freqs):
        run = _QkNormRope.apply if wants_grad(q, k, q_weight, k_weight) else _norm_kernel
        return run(q, k, q_weight, k_weight, pos, freqs, sections, eps, interleaved)
    return _qk_norm_rope(q, k, q_weight, k_weight, pos, freqs, sections, eps, interleaved)


def _launch_norm_back(a, gq, gk, q, k, q_weight, k_weight):
    """Gradients from the forward's arguments ``a`` (changed) and those of its results."""

    a.gq, a.gk = gq.data_ptr(), gk.data_ptr()
    a.gq_sb, a.gq_sh, a.gq_sn, _ = gq.stride()
    a.gk_sb, a.gk_sh, a.gk_sn, _ = gk.stride()
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=q.dtype, device=q.device)
    a.q_out, a.k_out = dq.data_ptr(), dk.data_ptr()
    lib = _lib.load()
    ref = ctypes.byref(a)
    n = lib.shrimp_qk_norm_rope_workspace(ref)
    ws = torch.empty(max(n, 0), dtype=torch.uint8, device=q.device)
    dqw = torch.empty(q_weight.shape, dtype=q_weight.dtype, device=q.device)
    dkw = torch.empty(k_weight.shape, dtype=q_weight.dtype, device=q.device)
    _lib.launch(lib.shrimp_qk_norm_rope_backward, q.device, "shrimp::qk_norm_rope_backward", ref,
                dqw.data_ptr(), dkw.data_ptr(), ws.data_ptr(), n)
    return dq, dk, dqw, dkw


def _norm_back_kernel(gq, gk, q, k, q_weight, k_weight, pos, freqs, sections, eps, interleaved):
    what = "shrimp::qk_norm_rope_backward"
    a, _, _, keep = _args(what, q, k, pos, freqs, sections, interleaved, False, eps, q_weight,
                          k_weight, gq, gk)
    grads = _launch_norm_back(a, keep[6], keep[7], q, k, q_weight, k_weight)
    del keep
    return grads


def _norm_back_fake(gq, gk, q, k, q_weight, k_weight, pos, freqs, sections, eps, interleaved):
    return (q.new_empty(q.shape), k.new_empty(k.shape), q_weight.new_empty(q_weight.shape),
            k_weight.new_empty(k_weight.shape))


_qk_norm_rope_backward = define(
    "qk_norm_rope_backward(Tensor gq, Tensor gk, Tensor q, Tensor k, Tensor q_weight,"
    " Tensor k_weight, Tensor pos, Tensor freqs, int[] sections, float eps, bool interleaved)"
    " -> (Tensor, Tensor, Tensor, Tensor)", _norm_back_kernel, _norm_back_fake)


def qk_norm_rope_backward(
    gq: torch.Tensor, gk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor,
    k_weight: torch.Tensor, pos: torch.Tensor, freqs: torch.Tensor, sections: Sequence[int],
    eps: float = 1e-6, interleaved: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of q, k, q_weight and k_weight from those of qk_norm_rope's results. The
    weights' sums have a fixed order, so the same call gives the same bits."""

    return _qk_norm_rope_backward(gq, gk, q, k, q_weight, k_weight, pos, freqs, sections, eps,
                                  interleaved)
