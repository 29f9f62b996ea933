"""shrimp::rope_axes and shrimp::qk_norm_rope against float64 restatements of their
formulas, forward and backward.

Tolerances are bounds, elementwise. U = 2^-24 is the half step of fp32. Sines and
cosines are within 4 U (reduction, polynomial and its roundings), so a rotated
element of (a, b) is within 8 U (|a| + |b|); an RMS over D terms is within
(D / 2 + 8) U relative (a sum of D terms, halved by the root); a sum of n terms
is within n U of the sum of their absolute values. Each result is rounded once to
its type: half a step, finfo.eps / 2, and an underflow step of the type."""

import pytest
import torch

from shrimp import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-24
DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _turn(x, pos, freqs, sections, interleaved, sign=1.0):
    """Rotation in float64 on the CPU, and |a| + |b| of every element's pair."""
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], dtype=torch.long)
    p = axis.numel()
    th = sign * pos.double()[..., axis] * freqs.double()
    c, s = th.cos()[:, None], th.sin()[:, None]
    y, mag = x.clone(), x.abs()
    ia = slice(0, 2 * p, 2) if interleaved else slice(0, p)
    ib = slice(1, 2 * p, 2) if interleaved else slice(p, 2 * p)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return y, mag


def _close(got, want, err, what):
    fi = torch.finfo(got.dtype)
    got = got.detach().cpu().double()
    tol = err + (want.abs() + err) * fi.eps / 2 + fi.smallest_normal * fi.eps
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), ((got - want).abs() / tol).max().item())


def _heads(g, b, h, s, d, dt, layout):
    """(B, H, S, D) on the device: contiguous, rows of a projection, or off its alignment."""
    if layout == "bhsd":
        return torch.randn(b, h, s, d, generator=g).to(dt).to(DEV)
    if layout == "bshd":
        return torch.randn(b, s, h, d, generator=g).to(dt).to(DEV).transpose(1, 2)
    if layout == "odd":  # one element in, rows of d + 3
        return torch.randn(b, s, h, d + 3, generator=g).to(dt).to(DEV)[..., 1 : d + 1].transpose(1, 2)
    assert layout == "dim"  # the head dimension is not the last in memory
    return torch.randn(b, h, d, s, generator=g).to(dt).to(DEV).transpose(2, 3)


def _pos(g, b, s, axes, far, dt=torch.int32):
    return ((2 * torch.rand(b, s, axes, generator=g) - 1) * far).round().to(dt).to(DEV)


def _freqs(sections, dt=torch.float32):
    return torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))
                      for n in sections]).to(dt).to(DEV)


# batch, q heads, k heads, rows, head dim, sections, layout, interleaved
SHAPES = [
    (3, 8, 8, 33, 16, [4, 4], "bshd", False),
    (2, 4, 4, 17, 24, [6, 6], "bshd", False),       # pairs in fours
    (2, 3, 1, 29, 64, [16, 16], "bhsd", False),
    (2, 8, 2, 13, 128, [16, 24, 24], "bshd", True),
    (1, 16, 4, 1, 128, [64], "bshd", False),        # one token
    (5, 2, 2, 1, 64, [8, 8, 8, 8], "bhsd", True),   # four axes
    (2, 3, 3, 11, 96, [11, 13], "odd", False),      # single elements, no power of two
    (2, 2, 1, 7, 21, [3, 5], "bhsd", True),         # an odd rest
    (1, 2, 2, 9, 256, [128], "odd", False),         # two units per lane
    (1, 1, 3, 5, 255, [100, 0, 20], "bhsd", False), # an axis without pairs
    (2, 5, 1, 6, 8, [2], "dim", False),
    (1, 70, 3, 4, 32, [8], "bshd", False),          # half the head passes
    (2, 2, 2, 5, 1, [0], "bhsd", False),            # nothing turns
]


@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rope_axes(shape, dt):
    b, h, _, s, d, sections, layout, il = shape
    g = _gen(1)
    x = _heads(g, b, h, s, d, dt, layout).requires_grad_()
    pos, freqs = _pos(g, b, s, len(sections), 40), _freqs(sections)
    y = ops.rope_axes(x, pos, freqs, sections, il)
    assert y.dtype == dt and y.is_contiguous()
    cpu = (pos.cpu(), freqs.cpu(), sections, il)
    want, mag = _turn(x.detach().cpu().double(), *cpu)
    _close(y, want, 8 * U * mag, "forward")
    gy = _heads(g, b, h, s, d, dt, layout)
    (gx,) = torch.autograd.grad(y, x, gy)
    want, mag = _turn(gy.cpu().double(), *cpu, sign=-1.0)
    _close(gx, want, 8 * U * mag, "backward")
    back = ops.rope_axes(gy, pos, freqs, sections, il, True)
    assert torch.equal(back, gx)


def _norm_want(x, w, pos, freqs, sections, il, eps):
    d = x.shape[-1]
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    y, mag = _turn(n * w, pos, freqs, sections, il)
    return y, (d / 2 + 18) * U * mag


def _norm_back_want(x, w, g, pos, freqs, sections, il, eps):
    d = x.shape[-1]
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    u, mag = _turn(g, pos, freqs, sections, il, sign=-1.0)
    eu = 8 * U * mag
    dot = (u * w * x).mean(-1, keepdim=True) * r**2
    mdot = (u.abs() * w.abs() * x.abs()).mean(-1, keepdim=True) * r**2
    edot = (eu * w.abs() * x.abs()).mean(-1, keepdim=True) * r**2
    dx = r * (u * w - x * dot)
    ex = r * (w.abs() * eu + (d / 2 + 12) * U * (u * w).abs() + x.abs() * (edot + (2.5 * d + 40) * U * mdot))
    rows = x.shape[0] * x.shape[1] * x.shape[2]
    dw = (u * x * r).sum((0, 1, 2))
    ew = (eu * (x * r).abs()).sum((0, 1, 2)) + (rows + d / 2 + 12) * U * (u * x * r).abs().sum((0, 1, 2))
    return dx, ex, dw, ew


@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_qk_norm_rope(shape, dt):
    b, h, hk, s, d, sections, layout, il = shape
    g = _gen(2)
    eps = 1e-5
    q = _heads(g, b, h, s, d, dt, layout).requires_grad_()
    k = _heads(g, b, hk, s, d, dt, layout).requires_grad_()
    wt = torch.float32 if d % 2 else dt  # weights of the model's type, or kept in fp32
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=g)).to(wt).to(DEV).requires_grad_() for _ in "qk")
    pos, freqs = _pos(g, b, s, len(sections), 300), _freqs(sections, torch.float64)
    out = ops.qk_norm_rope(q, k, qw, kw, pos, freqs, sections, eps, il)
    gs = [_heads(g, b, n, s, d, dt, layout) for n in (h, hk)]
    grads = torch.autograd.grad(out, [q, k, qw, kw], gs)
    cpu = (pos.cpu(), freqs.cpu(), sections, il, eps)
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        xc, wc, gc = x.detach().cpu().double(), w.detach().cpu().double(), gs[i].cpu().double()
        want, err = _norm_want(xc, wc, *cpu)
        assert out[i].is_contiguous() and out[i].dtype == dt
        _close(out[i], want, err, "forward " + "qk"[i])
        dx, ex, dw, ew = _norm_back_want(xc, wc, gc, *cpu)
        _close(grads[i], dx, ex, "gradient of " + "qk"[i])
        _close(grads[2 + i], dw, ew, "gradient of the weight of " + "qk"[i])


@pytest.mark.parametrize("pdt", (torch.int32, torch.int64, torch.float32), ids=str)
@pytest.mark.parametrize("fdt", (torch.float32, torch.float64), ids=str)
def test_far_positions(pdt, fdt):
    """Angles of far positions keep fp32's precision: formed and reduced in float64."""
    g = _gen(3)
    b, h, s, d, sections = 1, 2, 64, 64, [16, 16]
    x = _heads(g, b, h, s, d, torch.float32, "bhsd")
    pos, freqs = _pos(g, b, s, 2, 2**22, pdt), _freqs(sections, fdt)
    if pdt == torch.float32:
        pos = pos + 0.25
    want, mag = _turn(x.cpu().double(), pos.cpu(), freqs.cpu(), sections, False)
    _close(ops.rope_axes(x, pos, freqs, sections), want, 8 * U * mag, "far")


def test_broadcast_positions_and_gradients():
    """Positions shared by all sequences, strided positions, and an expanded gradient."""
    g = _gen(4)
    b, h, s, d, sections = 3, 2, 10, 32, [8, 8]
    x = _heads(g, b, h, s, d, torch.float32, "bshd").requires_grad_()
    pos, freqs = _pos(g, 1, s, 2, 20), _freqs(sections)
    full = ops.rope_axes(x, pos.expand(b, -1, -1).contiguous(), freqs, sections)
    assert torch.equal(ops.rope_axes(x, pos[0], freqs, sections), full)
    assert torch.equal(ops.rope_axes(x, pos, freqs, sections), full)
    wide = torch.zeros(b, s, 5, dtype=torch.int32, device=DEV)
    wide[..., 1::3] = pos
    assert torch.equal(ops.rope_axes(x, wide[..., 1::3], freqs, sections), full)
    (gx,) = torch.autograd.grad(full.sum(), x)
    want, mag = _turn(torch.ones(b, h, s, d, dtype=torch.float64), pos.cpu(), freqs.cpu(), sections,
                      False, sign=-1.0)
    _close(gx, want, 8 * U * mag, "expanded gradient")
    w = torch.ones(d, device=DEV, requires_grad=True)
    q, _ = ops.qk_norm_rope(x, x, w, w, pos, freqs, sections)
    gx, gw = torch.autograd.grad(q.sum(), [x, w])  # k's result unused, the weight shared
    dx, ex, dw, ew = _norm_back_want(x.detach().cpu().double(), torch.ones(d, dtype=torch.float64),
                                     torch.ones(b, h, s, d, dtype=torch.float64), pos.cpu(),
                                     freqs.cpu(), sections, False, 1e-6)
    _close(gx, dx, ex, "gradient of a shared input")
    _close(gw, dw, ew, "gradient of a shared weight")


def test_zero_rows_and_no_rows():
    x = torch.zeros(2, 3, 4, 16, dtype=torch.bfloat16, device=DEV)
    w = torch.ones(16, device=DEV, requires_grad=True)
    pos, freqs = torch.ones(4, 1, dtype=torch.int32, device=DEV), _freqs([8])
    q, k = ops.qk_norm_rope(x, x[:, :0], w, w, pos, freqs, [8])
    assert torch.equal(q, x) and k.shape == (2, 0, 4, 16)
    e = x[:, :, :0].clone().requires_grad_()
    q, k = ops.qk_norm_rope(e, e, w, w, pos[:0], freqs, [8])
    assert q.shape == e.shape
    ge, gw = torch.autograd.grad((q, k), [e, w], (q.detach(), k.detach()))
    assert ge.shape == e.shape and torch.equal(gw, torch.zeros_like(w))
    assert ops.rope_axes(x[:0], pos, freqs, [8]).shape == (0, 3, 4, 16)


def test_gradient_against_differences():
    """Directional derivative of a weighted sum against central differences of the float64
    restatement (step 1e-5: truncation and cancellation below 1e-8 of the sums); the
    gradients are fp32, within their own bounds, so 1e-4 of the sum of magnitudes."""
    g = _gen(5)
    b, h, s, d, sections = 2, 3, 5, 32, [8, 8]
    q, k = (_heads(g, b, h, s, d, torch.float32, "bshd").requires_grad_() for _ in "qk")
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=g)).to(DEV).requires_grad_() for _ in "qk")
    pos, freqs = _pos(g, b, s, 2, 30), _freqs(sections)
    out = ops.qk_norm_rope(q, k, qw, kw, pos, freqs, sections, 1e-5)
    gs = [torch.randn(o.shape, generator=g).to(DEV) for o in out]
    grads = torch.autograd.grad(out, [q, k, qw, kw], gs)
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        xc, wc, gc = x.detach().cpu().double(), w.detach().cpu().double(), gs[i].cpu().double()
        vx, vw = torch.randn(xc.shape, generator=g).double(), torch.randn(d, generator=g).double()
        f = lambda t: (_norm_want(xc + t * vx, wc + t * vw, pos.cpu(), freqs.cpu(), sections, False,
                                  1e-5)[0] * gc).sum()
        want = ((f(1e-5) - f(-1e-5)) / 2e-5).item()
        parts = torch.cat([(grads[i].cpu().double() * vx).flatten(), grads[2 + i].cpu().double() * vw])
        assert abs(parts.sum().item() - want) <= 1e-4 * parts.abs().sum().item()


def test_weight_gradient_repeats():
    g = _gen(6)
    x = _heads(g, 40, 8, 200, 16, torch.bfloat16, "bshd")
    w = torch.ones(16, device=DEV)
    pos, freqs = _pos(g, 40, 200, 2, 20), _freqs([4, 4])
    first = ops.qk_norm_rope_backward(x, x, x, x, w, w, pos, freqs, [4, 4])
    for _ in range(3):
        again = ops.qk_norm_rope_backward(x, x, x, x, w, w, pos, freqs, [4, 4])
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_captured_forward_and_backward():
    """Captured once, replayed with new inputs and eager work between; two graphs on one
    stream do not share their workspaces."""
    g = _gen(7)
    b, h, s, d, sections = 4, 4, 30, 64, [32]
    pos, freqs = _pos(g, b, s, 1, 1000), _freqs(sections)
    w = (1 + 0.3 * torch.randn(d, generator=g)).to(DEV)
    new = lambda: torch.randn(b, h, s, d, generator=g).to(torch.bfloat16).to(DEV)
    calls = []
    for _ in range(2):
        q, k, gq, gk = (new() for _ in range(4))
        run = lambda q=q, k=k, gq=gq, gk=gk: (
            *ops.qk_norm_rope(q, k, w, w, pos, freqs, sections),
            *ops.qk_norm_rope_backward(gq, gk, q, k, w, w, pos, freqs, sections),
            ops.rope_axes(q, pos, freqs, sections))
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        calls.append((graph, outs, run, (q, k, gq, gk)))
    for _ in range(3):
        for _, _, _, ins in calls:
            for t in ins:
                t.copy_(new())
        for graph, *_ in calls:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs, run, _ in calls:
            assert all(torch.equal(a, b) for a, b in zip(outs, run()))


def test_backward_in_a_captured_step():
    """autograd inside a capture (no eager graph of the leaves alive)."""
    g = _gen(8)
    q = _heads(g, 2, 4, 20, 64, torch.bfloat16, "bshd").requires_grad_()
    w = torch.ones(64, device=DEV, requires_grad=True)
    pos, freqs = _pos(g, 2, 20, 1, 100), _freqs([32])
    gy = torch.randn(2, 4, 20, 64, generator=g).to(torch.bfloat16).to(DEV)

    def step():
        out = ops.qk_norm_rope(q, q, w, w, pos, freqs, [32])
        return torch.autograd.grad(out, [q, w], (gy, gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    want = step()
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_refused_on_the_device():
    x = torch.zeros(1, 2, 3, 16, device=DEV)
    w = torch.ones(16, device=DEV)
    pos, freqs = torch.zeros(3, 1, dtype=torch.int32, device=DEV), _freqs([8])
    ok = dict(q=x, k=x, q_weight=w, k_weight=w, pos=pos, freqs=freqs, sections=[8])
    ops.qk_norm_rope(**ok)
    for bad in (dict(k=x.bfloat16()), dict(k=x[..., :8]), dict(q=x[0]), dict(q=x.double(), k=x.double()),
                dict(q_weight=w[:8]), dict(k_weight=w.half()), dict(pos=pos.to(torch.int16)),
                dict(pos=pos[:2]), dict(pos=pos.expand(2, 3, 1)), dict(freqs=freqs[:4]),
                dict(freqs=freqs.half()), dict(sections=[9]), dict(sections=[]), dict(sections=[-1, 9]),
                dict(sections=[2, 2, 2, 1, 1]), dict(eps=0.0), dict(eps=-1.0), dict(pos=pos.cpu()),
                dict(freqs=freqs.cpu()), dict(k=x.cpu()), dict(q=torch.zeros(1, 2, 3, 257, device=DEV))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.qk_norm_rope(**{**ok, **bad})
    with pytest.raises(ValueError):
        ops.qk_norm_rope_backward(x, x[:, :1], **ok)


def test_no_second_derivative_and_no_grad():
    x = torch.randn(1, 2, 3, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    pos, freqs = torch.ones(3, 1, dtype=torch.int32, device=DEV), _freqs([8])
    with torch.no_grad():
        q, k = ops.qk_norm_rope(x, x, w, w, pos, freqs, [8])
    assert not q.requires_grad and not k.requires_grad
    q, k = ops.qk_norm_rope(x, x, w, w, pos, freqs, [8])
    (gx,) = torch.autograd.grad(q.square().sum() + k.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):  # refused, not silently zero
        torch.autograd.grad(gx.sum(), x)
