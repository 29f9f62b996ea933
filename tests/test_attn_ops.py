"""The rotary and block-attention operators without a GPU: struct layouts, refusals of the
C entries (each before any launch, with its message), refusals of the Python calls on host
tensors, and the shapes they promise to a tracer."""

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from shrimp import _lib, ops

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_struct_layouts_match_c(tmp_path):
    exe = tmp_path / "abi_layout_ops"
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(ROOT / "tests" / "abi_layout_ops.c"),
                    "-o", str(exe)], check=True)
    mirrors = {
        "shrimp_rope_args": _lib.RopeArgs,
        "shrimp_block_select_args": _lib.BlockSelectArgs,
        "shrimp_attn_blocks_args": _lib.AttnBlocksArgs,
        "shrimp_attn_blocks_grads": _lib.AttnBlocksGrads,
    }
    seen = 0
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n"):
        if not line:
            continue
        key, val = line.split()
        name, field = key.split(".")
        if field == "__size__":
            assert ctypes.sizeof(mirrors[name]) == int(val), name
        else:
            assert getattr(mirrors[name], field).offset == int(val), key
        seen += 1
    assert seen == len(mirrors) + sum(len(c._fields_) for c in mirrors.values())


def _refused(lib, rc, text):
    assert rc == -1
    assert text in lib.shrimp_last_error(), lib.shrimp_last_error()


def _rope(**kw):
    a = dict(q=64, k=64, q_sb=64, q_sh=16, q_sn=16, k_sb=64, k_sh=16, k_sn=16, pos=64, freqs=64, q_w=64,
             k_w=64, q_out=64, k_out=64, gq=64, gk=64, B=1, S=4, H=2, Hk=1, D=16, axes=1,
             sections=(ctypes.c_int32 * 4)(8), dt=_lib.DT_BF16, pos_dt=_lib.DT_I32, w_dt=_lib.DT_F32, eps=1e-6)
    return _lib.RopeArgs(**{**a, **kw})


def test_rope_refusals(lib):
    four = ctypes.c_int32 * 4
    for bad, text in (
        (dict(D=0), b"head dim"), (dict(D=257), b"head dim"), (dict(dt=_lib.DT_I32), b"element type"),
        (dict(axes=0), b"axes"), (dict(axes=5), b"axes"), (dict(sections=four(9)), b"pairs"),
        (dict(sections=four(-1)), b"pairs"), (dict(axes=2, sections=four(2**31 - 1, 2**31 - 1)), b"pairs"),
        (dict(q_w=None), b"weight is missing"), (dict(k_w=None), b"weight is missing"),
        (dict(w_dt=_lib.DT_I64), b"weight type"), (dict(eps=0.0), b"eps"), (dict(eps=float("nan")), b"eps"),
        (dict(pos_dt=_lib.DT_F16), b"position type"), (dict(pos=None), b"null positions"),
        (dict(freqs=None), b"null positions"), (dict(q=None), b"null q"), (dict(q_out=None), b"null q"),
        (dict(k=None), b"null k"), (dict(B=-1), b"negative"), (dict(H=1 << 20), b"H="),
        (dict(B=1 << 20, S=1 << 20), b"tokens"),
    ):
        a = _rope(**bad)
        _refused(lib, lib.shrimp_rope(ctypes.byref(a), None), text)
        assert lib.shrimp_qk_norm_rope_workspace(ctypes.byref(a)) == -1 or text in (b"null q", b"null k")
    _refused(lib, lib.shrimp_rope(None, None), b"null arguments")
    a = _rope()
    need = lib.shrimp_qk_norm_rope_workspace(ctypes.byref(a))
    assert need > 0
    back = lib.shrimp_qk_norm_rope_backward
    _refused(lib, back(ctypes.byref(a), None, 64, 64, need, None), b"null weight gradient")
    _refused(lib, back(ctypes.byref(a), 64, 64, 64, need - 1, None), b"workspace")
    _refused(lib, back(ctypes.byref(a), 64, 64, None, need, None), b"workspace")
    _refused(lib, back(ctypes.byref(_rope(gq=None)), 64, 64, 64, need, None), b"null q")
    _refused(lib, back(ctypes.byref(_rope(q_w=None, k_w=None)), 64, 64, 64, need, None), b"weights are required")
    for none in (dict(B=0), dict(S=0), dict(H=0, Hk=0)):  # nothing to do
        assert lib.shrimp_rope(ctypes.byref(_rope(**none, q=None, k=None, pos=None)), None) == 0


def test_block_refusals(lib):
    means = lambda **kw: lib.shrimp_block_means(*{**dict(
        k=64, sb=64, sh=64, sn=64, dt=_lib.DT_BF16, lens=64, means=64, B=1, Hk=1, Sk=100, D=64, block=16,
        last=0, st=None), **kw}.values())
    for bad, text in ((dict(D=129), b"head dim"), (dict(D=0), b"head dim"), (dict(block=0), b"block of"),
                      (dict(dt=9), b"element type"), (dict(Sk=5000, block=1), b"blocks"), (dict(B=-1), b"negative"),
                      (dict(k=None), b"null"), (dict(lens=None), b"null"), (dict(means=None), b"null"),
                      (dict(block=2**31 - 1), b"block of"), (dict(Sk=2**31 - 1, block=2**20), b"block of")):
        _refused(lib, means(**bad), text)
    assert means(B=0, k=None) == 0 and means(Sk=0, k=None) == 0

    def select(**kw):
        a = dict(q=64, q_sb=64, q_sh=64, q_sn=64, means=64, q_lens=64, k_lens=64, sel=64, B=1, H=2, Hk=1,
                 Sq=4, Sk=100, D=64, block=16, topk=4, dt=_lib.DT_BF16)
        return lib.shrimp_block_select(ctypes.byref(_lib.BlockSelectArgs(**{**a, **kw})), None)

    for bad, text in ((dict(D=129), b"head dim"), (dict(topk=0), b"topk"), (dict(topk=65), b"topk"),
                      (dict(Hk=0), b"query heads"), (dict(H=3, Hk=2), b"query heads"), (dict(block=0), b"block of"),
                      (dict(Sk=5000, block=1), b"blocks"), (dict(sel=None), b"null"), (dict(means=None), b"null"),
                      (dict(H=0), b"query heads"), (dict(means=72), b"16-byte"), (dict(block=2**31 - 1), b"block of"),
                      (dict(Sk=2**31 - 1, block=2**20), b"block of"), (dict(Sq=2**31 - 1), b"queries"),
                      (dict(B=2**31 - 1, H=2**31 - 1, Hk=2**31 - 1, Sq=2**30), b"queries"), (dict(dt=5), b"element type"), (dict(Sq=-1), b"negative")):
        _refused(lib, select(**bad), text)
    assert select(Sq=0, q=None) == 0


def _attn(**kw):
    a = dict(q=64, k=64, v=64, q_sb=64, q_sh=64, q_sn=64, k_sb=64, k_sh=64, k_sn=64, v_sb=64, v_sh=64, v_sn=64,
             sel=64, q_lens=64, k_lens=64, out=64, lse=64, B=1, H=2, Hk=1, Sq=40, Sk=100, d=64, block=16, topk=4,
             dt=_lib.DT_BF16, scale=0.125)
    return _lib.AttnBlocksArgs(**{**a, **kw})


def test_attn_blocks_refusals(lib):
    for bad, text in (
        (dict(d=12), b"head dim"), (dict(d=136), b"head dim"), (dict(d=0), b"head dim"),
        (dict(dt=_lib.DT_F32), b"element type"), (dict(block=8), b"multiple of 16"), (dict(block=40), b"multiple of 16"),
        (dict(topk=0), b"topk"), (dict(topk=65), b"topk"), (dict(H=49), b"query heads"), (dict(H=3, Hk=2), b"query heads"),
        (dict(Hk=0), b"query heads"), (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"),
        (dict(q=None), b"null"), (dict(sel=None), b"null"), (dict(k=None), b"null k"), (dict(lse=None), b"null"),
        (dict(q=72), b"16-byte"), (dict(k_sn=60), b"16-byte"), (dict(v_sh=1 << 31), b"16-byte"),
        (dict(q_sn=-64), b"16-byte"), (dict(out=72), b"16-byte"), (dict(Sk=(1 << 30) + 1), b"Sq="),
    ):
        a = _attn(**bad)
        _refused(lib, lib.shrimp_attn_blocks(ctypes.byref(a), None), text)
        assert lib.shrimp_attn_blocks_workspace(ctypes.byref(a)) == -1
    _refused(lib, lib.shrimp_attn_blocks(None, None), b"null arguments")
    assert lib.shrimp_attn_blocks(ctypes.byref(_attn(Sq=0, q=None, k=None)), None) == 0
    a = _attn()
    need = lib.shrimp_attn_blocks_workspace(ctypes.byref(a))
    assert need > 0
    grads = lambda **kw: _lib.AttnBlocksGrads(**{**dict(g=64, g_sb=64, g_sh=64, g_sn=64, dq=64, dk=64, dv=64,
                                                        workspace=64, workspace_bytes=need), **kw})
    for bad, text in ((dict(g=None), b"null gradient"), (dict(dq=None), b"null gradient"), (dict(dk=None), b"null gradient"),
                      (dict(dv=None), b"null gradient"), (dict(workspace=None), b"workspace"),
                      (dict(workspace_bytes=need - 1), b"workspace"), (dict(workspace=66), b"workspace"),
                      (dict(g_sn=4), b"16-byte"), (dict(dk=72), b"16-byte")):
        _refused(lib, lib.shrimp_attn_blocks_backward(ctypes.byref(a), ctypes.byref(grads(**bad)), None), text)
    _refused(lib, lib.shrimp_attn_blocks_backward(ctypes.byref(a), None, None), b"null gradients")
    # no queries: the keys' gradients are still written, so their pointers are needed
    none = _attn(Sq=0, k=None)
    _refused(lib, lib.shrimp_attn_blocks_backward(ctypes.byref(none), ctypes.byref(grads()), None), b"null k")
    for sq, text in ((3, b"queries"), (2**30, b"groups of queries")):
        huge = _attn(B=2**31 - 1, H=2**31 - 1, Hk=2**31 - 1, Sq=sq)
        _refused(lib, lib.shrimp_attn_blocks(ctypes.byref(huge), None), text)
    many = _attn(B=2**16, H=2**16, Hk=2**16, Sq=64)
    room = grads(workspace_bytes=2**62)
    _refused(lib, lib.shrimp_attn_blocks_backward(ctypes.byref(many), ctypes.byref(room), None), b"chunks of queries")
    _refused(lib, lib.shrimp_block_means(64, 64, 64, 64, _lib.DT_BF16, 64, 64, 2**31 - 1, 2**31 - 1, 100, 64, 1, 0, None),
             b"blocks of keys")
    big = _attn(B=2**31 - 1, H=2**20, Hk=2**20, Sq=2**30)
    assert lib.shrimp_attn_blocks_workspace(ctypes.byref(big)) > 2**62  # saturated, not wrapped


def test_host_tensors_are_refused():
    x = torch.zeros(1, 2, 3, 16)
    w, pos, freqs = torch.ones(16), torch.zeros(3, 1, dtype=torch.int32), torch.ones(8)
    lens = torch.tensor([3], dtype=torch.int32)
    sel = torch.zeros(1, 2, 3, 1, dtype=torch.int32)
    for call in (lambda: ops.rope_axes(x, pos, freqs, [8]),
                 lambda: ops.qk_norm_rope(x, x, w, w, pos, freqs, [8]),
                 lambda: ops.qk_norm_rope_backward(x, x, x, x, w, w, pos, freqs, [8]),
                 lambda: ops.block_means(x, lens, 16),
                 lambda: ops.block_means_update(torch.zeros(1, 2, 1, 16), x, lens, 16),
                 lambda: ops.block_select(x, torch.zeros(1, 2, 1, 16), lens, lens, 16, 1),
                 lambda: ops.attn_blocks(*[x.bfloat16()] * 3, sel, lens, lens, 16),
                 lambda: ops.attn_blocks_backward(x.bfloat16(), None, *[x.bfloat16()] * 3, sel, lens, lens,
                                                  x.bfloat16(), x[..., 0], 16)):
        with pytest.raises(RuntimeError, match="ROCm device only"):
            call()


def test_traced_shapes():
    """The operators under a fake-tensor mode: through the dispatcher, with the results' shapes
    and types. (Autograd's engine needs a device for fake device tensors, so the backward
    operators are called by name.)"""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(), torch.no_grad():
        dev = "cuda"
        bf = dict(dtype=torch.bfloat16, device=dev)
        q = torch.empty(2, 4, 50, 64, **bf)
        k = torch.empty(2, 2, 50, 64, **bf)
        w = torch.empty(64, device=dev)
        pos = torch.empty(50, 2, dtype=torch.int32, device=dev)
        freqs = torch.empty(32, device=dev)
        lens = torch.empty(2, dtype=torch.int32, device=dev)
        x = ops.rope_axes(q, pos, freqs, [16, 16])
        assert x.shape == q.shape and x.dtype == q.dtype
        qn, kn = ops.qk_norm_rope(q, k, w, w, pos, freqs, [16, 16])
        assert qn.shape == q.shape and kn.shape == k.shape
        grads = ops.qk_norm_rope_backward(qn, kn, q, k, w, w, pos, freqs, [16, 16])
        assert [g.shape for g in grads] == [q.shape, k.shape, w.shape, w.shape]
        means = ops.block_means(kn, lens, 16)
        assert means.shape == (2, 2, 4, 64) and means.dtype == torch.float32
        ops.block_means_update(means, kn, lens, 16)
        sel = ops.block_select(qn, means, lens, lens, 16, 3)
        assert sel.shape == (2, 2, 50, 3) and sel.dtype == torch.int32
        out, lse = ops.attn_blocks(qn, kn, kn, sel, lens, lens, 16)
        assert out.shape == q.shape and lse.shape == (2, 4, 50) and lse.dtype == torch.float32
        grads = ops.attn_blocks_backward(out, None, qn, kn, kn, sel, lens, lens, out, lse, 16)
        assert [g.shape for g in grads] == [q.shape, k.shape, k.shape]
