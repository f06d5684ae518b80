"""Norm of the query and key heads with the rotation (qk_norm_rope) against its
definition in 64 bits, forward and backward.

Tolerance, per element: one rounding to the output's type (u = eps / 2 of the
value), and 64 roundings of 2^-24 in the fp32 chain relative to the
magnitudes that are added (a lane sums 16 squares, the team at most 5 more by
shuffles, then a reciprocal root of 2 ulp and a few products; the backward
adds a second such sum).  The weights' gradient sums a few rows per lane and
joins the lanes and warps: 128 roundings relative to the sum of magnitudes.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -24


def _tables(S, R, dtype, device, first=0, B=1):
    pos = torch.arange(first, first + S, dtype=torch.float64)[None, :, None] + 7 * torch.arange(B)[:, None, None]
    ang = pos * (1e4 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R))
    ang = torch.cat([ang, 0.9 * ang], -1)  # the two halves of a table need not be alike
    return ang.cos().to(dtype).to(device), ang.sin().to(dtype).to(device)


def _forward64(x, w, cos, sin, eps, offset):
    """(out, sum of the magnitudes that each output adds)"""
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    y = x * r * (w + offset)
    R = cos.shape[-1]
    h = R // 2
    c, s = cos[:, :, None], sin[:, :, None]
    a, b = y[..., :h], y[..., h:R]
    parts = [(a * c[..., :h], -b * s[..., :h]), (b * c[..., h:], a * s[..., h:])]
    out = torch.cat([p + q for p, q in parts] + [y[..., R:]], -1)
    return out, torch.cat([p.abs() + q.abs() for p, q in parts] + [y[..., R:].abs()], -1)


def _backward64(g, x, w, cos, sin, eps, offset):
    """(dx, its magnitudes, dw, its magnitudes)"""
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r
    R = cos.shape[-1]
    h = R // 2
    c, s = cos[:, :, None], sin[:, :, None]
    a, b = g[..., :h], g[..., h:R]
    parts = [(a * c[..., :h], b * s[..., h:]), (b * c[..., h:], -a * s[..., :h])]
    gy = torch.cat([p + q for p, q in parts] + [g[..., R:]], -1)
    gya = torch.cat([p.abs() + q.abs() for p, q in parts] + [g[..., R:].abs()], -1)
    gn, gna = gy * (w + offset), gya * (w + offset).abs()
    dx = r * (gn - n * (gn * n).mean(-1, keepdim=True))
    mag = r * (gna + n.abs() * (gna * n.abs()).mean(-1, keepdim=True))
    return dx, mag, (gy * n).sum((0, 1, 2)), (gya * n.abs()).sum((0, 1, 2))


def _close(got, want, mag, n):
    tiny = {torch.float16: 2.0 ** -25}.get(got.dtype, 0.0)  # half a step of the subnormals
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + n * ULP * mag * 1.01 + tiny
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, by up to {((got.double() - want).abs() / tol).max():.2f}x"


def _check(q, k, wq, wk, cos, sin, gq, gk, eps, offset):
    from voodoo_quant.fused_blocks import qk_norm_rope

    leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    qo, ko = qk_norm_rope(leaves[0], leaves[1], leaves[2], leaves[3], cos, sin, eps, weight_offset=offset)
    assert qo.shape == q.shape and qo.is_contiguous() and qo.dtype == q.dtype and ko.is_contiguous()
    grads = torch.autograd.grad((qo, ko), leaves, (gq, gk))
    c64, s64 = (t.double().expand(q.shape[0], -1, -1) if t.dim() == 3 else t.double()[None] for t in (cos, sin))
    for x, w, o, g, dx, dw in ((q, wq, qo, gq, grads[0], grads[2]), (k, wk, ko, gk, grads[1], grads[3])):
        x64, w64 = x.double(), w.double()
        want, mag = _forward64(x64, w64, c64, s64, eps, offset)
        _close(o, want, mag, 64)
        want, mag, wdw, wmag = _backward64(g.double(), x64, w64, c64, s64, eps, offset)
        assert dx.dtype == x.dtype and dw.dtype == w.dtype
        _close(dx, want, mag, 64)
        _close(dw, wdw, wmag, 128)


CASES = [
    # B, S, Hq, Hk, D, R, dtype, offset
    (1, 1, 16, 8, 128, 128, torch.bfloat16, 0.0),
    (1, 1, 1, 1, 16, 16, torch.float32, 0.0),
    (2, 33, 4, 2, 128, 128, torch.bfloat16, 0.0),
    (3, 7, 5, 1, 80, 32, torch.bfloat16, 0.0),
    (2, 13, 14, 2, 96, 96, torch.float16, 1.0),
    (1, 65, 3, 3, 64, 16, torch.float32, 0.0),
    (2, 9, 7, 2, 256, 64, torch.bfloat16, 1.0),
    (1, 5, 2, 1, 512, 512, torch.float16, 0.0),
    (1, 5, 3, 2, 272, 128, torch.float32, 0.0),
    (1, 300, 40, 8, 48, 48, torch.bfloat16, 0.0),
]


@pytest.mark.parametrize("B,S,Hq,Hk,D,R,dtype,offset", CASES)
def test_forward_and_backward_against_64_bits(cuda, B, S, Hq, Hk, D, R, dtype, offset):
    g = torch.Generator(device="cpu").manual_seed(S * 100 + D + Hq)

    def rnd(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype).to(cuda)

    cos, sin = _tables(S, R, dtype, cuda, first=12345)
    _check(rnd(B, S, Hq, D, scale=3.0), rnd(B, S, Hk, D), (1 - offset) + rnd(D, scale=0.2), (1 - offset) + rnd(D, scale=0.2),
           cos, sin, rnd(B, S, Hq, D), rnd(B, S, Hk, D), 1e-6, offset)


def test_strided_heads_and_gradients_and_wide_weights(cuda):
    """Column ranges of one projection, transposed gradients, float32 weights and tables beside bf16 heads, a table row
    per batch entry, a table without a batch dimension, and an unaligned view."""
    B, S, Hq, Hk, D = 2, 19, 6, 2, 64
    g = torch.Generator(device="cpu").manual_seed(3)
    qkv = torch.randn(B, S, (Hq + 2 * Hk) * D, generator=g).to(torch.bfloat16).to(cuda)
    q, k, _ = qkv.split([Hq * D, Hk * D, Hk * D], -1)
    q, k = q.view(B, S, Hq, D), k.view(B, S, Hk, D)
    gq = torch.randn(B, Hq, S, D, generator=g).to(torch.bfloat16).to(cuda).transpose(1, 2)
    gk = torch.randn(B, Hk, S, D, generator=g).to(torch.bfloat16).to(cuda).transpose(1, 2)
    wq, wk = (torch.rand(D, generator=g).to(cuda) + 0.5 for _ in range(2))
    cos, sin = _tables(S, D, torch.float32, cuda, B=B)
    _check(q, k, wq, wk, cos, sin, gq, gk, 1e-5, 0.0)
    cos, sin = _tables(S, D, torch.bfloat16, cuda)
    _check(q, k, wq.bfloat16(), wk, cos[0], sin[0], gq, gk, 1e-5, 0.0)
    flat = torch.randn(B * S * Hq * D + 1, generator=g).to(torch.bfloat16).to(cuda)
    _check(flat[1:].view(B, S, Hq, D), k, wq.bfloat16(), wk.bfloat16(), cos, sin, gq, gk, 1e-5, 0.0)
    # heads shared by expansion: read where they are
    _check(q[:, :, :1].expand(B, S, Hq, D), k, wq, wk, cos, sin, gq, gk, 1e-5, 0.0)


def test_gradient_against_differences(cuda):
    """Central differences of a weighted sum of the outputs, in float32 inputs moved along random directions: with a step
    h the difference quotient is off by h^2 / 6 of a third derivative of order one and by the outputs' rounding over
    2 h; h = 2^-7 keeps both below 2e-3 of the magnitudes."""
    from voodoo_quant.fused_blocks import qk_norm_rope

    B, S, Hq, Hk, D = 1, 6, 3, 2, 64
    g = torch.Generator(device="cpu").manual_seed(8)
    x = [torch.randn(*s, generator=g).to(cuda) for s in ((B, S, Hq, D), (B, S, Hk, D), (D,), (D,))]
    v = [torch.randn(*t.shape, generator=g).to(cuda) for t in x]
    gq, gk = (torch.randn(*t.shape, generator=g).to(cuda) for t in x[:2])
    cos, sin = _tables(S, D, torch.float32, cuda)

    def f(t):
        with torch.no_grad():
            qo, ko = qk_norm_rope(*[a + t * b for a, b in zip(x, v)], cos, sin, 1e-6)
        return float((qo.double() * gq.double()).sum() + (ko.double() * gk.double()).sum())

    h = 2.0 ** -7
    leaves = [t.clone().requires_grad_(True) for t in x]
    grads = torch.autograd.grad(qk_norm_rope(*leaves, cos, sin, 1e-6), leaves, (gq, gk))
    want = sum(float((a.double() * b.double()).sum()) for a, b in zip(grads, v))
    size = sum(float((a.double() * b.double()).abs().sum()) for a, b in zip(grads, v))
    assert abs((f(h) - f(-h)) / (2 * h) - want) < 2e-3 * size


def test_rows_that_hold_nothing_or_too_much(cuda):
    """A head of zeros is zeros (eps keeps the root finite) with gradient g * w / sqrt(eps); NaN and infinity stay in
    their own head."""
    from voodoo_quant.fused_blocks import qk_norm_rope

    S, H, D = 5, 4, 128
    g = torch.Generator(device="cpu").manual_seed(4)
    q = torch.randn(1, S, H, D, generator=g).to(torch.bfloat16).to(cuda)
    q[0, 1, 2] = 0
    clean = q.clone()
    q[0, 2, 1, 5] = float("nan")
    q[0, 3, 0, 100] = float("inf")
    k = q[:, :, :2].contiguous()
    w = torch.ones(D, dtype=torch.bfloat16, device=cuda)
    cos, sin = _tables(S, D, torch.bfloat16, cuda)
    qo, ko = qk_norm_rope(q, k, w, w, cos, sin, 1e-6)
    co, _ = qk_norm_rope(clean, k, w, w, cos, sin, 1e-6)
    assert torch.equal(qo[0, 1, 2], torch.zeros(D, dtype=torch.bfloat16, device=cuda))
    other = torch.ones(1, S, H, dtype=torch.bool, device=cuda)
    other[0, 2, 1] = other[0, 3, 0] = False
    assert torch.equal(qo[other], co[other]) and torch.isfinite(qo[other]).all()
    assert torch.isnan(qo[0, 2, 1]).all() and torch.isnan(qo[0, 3, 0]).any()


def test_empty_shapes_and_single_sided_calls(cuda):
    from voodoo_quant.fused_blocks import qk_norm_rope

    D = 64
    w = torch.ones(D, device=cuda, requires_grad=True)
    for B, S, Hq, Hk in ((0, 4, 2, 1), (2, 0, 2, 1), (1, 3, 0, 2), (1, 3, 2, 0)):
        q = torch.randn(B, S, Hq, D, device=cuda, requires_grad=True)
        k = torch.randn(B, S, Hk, D, device=cuda, requires_grad=True)
        cos, sin = _tables(S, D, torch.float32, cuda)
        qo, ko = qk_norm_rope(q, k, w, w, cos, sin)
        (qo.sum() + ko.sum()).backward()
        assert q.grad.shape == q.shape and torch.isfinite(w.grad).all()


def test_another_stream_a_captured_graph_and_repeats(cuda):
    """The same bits on a side stream, from a replayed graph with new inputs, and on every repeat."""
    from voodoo_quant import _C

    B, S, Hq, Hk, D = 2, 50, 8, 2, 128
    g = torch.Generator(device="cpu").manual_seed(5)
    sets = [[torch.randn(B, S, h, D, generator=g).to(torch.bfloat16).to(cuda) for h in (Hq, Hk, Hq, Hk)] for _ in range(2)]
    w = (torch.rand(D, generator=g) + 0.5).to(torch.bfloat16).to(cuda)
    cos, sin = _tables(S, D, torch.bfloat16, cuda)

    def call(q, k, gq, gk):
        qo, ko, operands, layout = _C.qk_norm_rope_fwd(q, k, w, w, cos, sin, 1e-6, saved=True)
        return (qo, ko, *_C.qk_norm_rope_bwd(gq, gk, operands, layout))

    want = [call(*s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(*sets[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    static = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(*static)
    for s, ref in zip(sets[::-1], want[::-1]):
        for a, b in zip(static, s):
            a.copy_(b)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_frozen_weights_and_unused_outputs(cuda):
    from voodoo_quant.fused_blocks import qk_norm_rope

    D = 64
    q = torch.randn(1, 4, 2, D, device=cuda, requires_grad=True)
    k = torch.randn(1, 4, 1, D, device=cuda)
    w = torch.ones(D, device=cuda)
    cos, sin = _tables(4, D, torch.float32, cuda)
    qo, _ = qk_norm_rope(q, k, w, w, cos, sin)
    qo.square().sum().backward()
    want = torch.autograd.functional.vjp(
        lambda x: _forward64(x, w.double(), cos.double(), sin.double(), 1e-6, 0.0)[0].square().sum(), q.detach().double())[1]
    # |q| is kept by norm and rotation up to eps: the gradient is the difference of near equals, each of order 2
    assert (q.grad.double() - want).abs().max() < 64 * ULP * 16


def test_offsets_past_32_bits(cuda):
    """Heads of more than 2^31 values, and a layout whose batch stride is past 2^31: the last positions come out as those
    of a call on them alone do."""
    from voodoo_quant import _C

    S, Hq, Hk, D = 440_000, 39, 1, 128
    g = torch.Generator(device=cuda).manual_seed(4)
    q = torch.zeros(1, S, Hq, D, dtype=torch.bfloat16, device=cuda)
    k = torch.zeros(1, S, Hk, D, dtype=torch.bfloat16, device=cuda)
    assert q.numel() > 2 ** 31
    n = 3
    for t in (q, k):
        t[:, -n:] = torch.randn(1, n, t.shape[2], D, device=cuda, generator=g)
    w = torch.ones(D, dtype=torch.bfloat16, device=cuda)
    cos, sin = (torch.randn(1, S, D, device=cuda, generator=g).bfloat16() for _ in range(2))

    def both(q, k, cos, sin):
        qo, ko, ops, layout = _C.qk_norm_rope_fwd(q, k, w, w, cos, sin, 1e-6, 0.0, saved=True)
        return qo, ko, *_C.qk_norm_rope_bwd(q, k, ops, layout, False)[:2]

    want = both(q[:, -n:], k[:, -n:], cos[:, -n:], sin[:, -n:])
    for got, exp in zip(both(q, k, cos, sin), want):
        assert torch.equal(got[:, -n:], exp) and not got[:, :-n].any()
    # two batch entries, 2^31 values and more apart
    flat = q.reshape(-1)
    far = flat.as_strided((2, n, Hq, D), (flat.numel() - n * Hq * D, Hq * D, D, 1))
    kk, cc, ss = k[:, -n:].expand(2, n, Hk, D), cos[:, -n:], sin[:, -n:]
    for got, exp in zip(both(far, kk, cc, ss), want):
        assert torch.equal(got[1:], exp)


def test_gradients_have_no_graph_of_their_own(cuda):
    """The gradients taken with create_graph are those taken without; a second derivative is refused, not zero."""
    from voodoo_quant.fused_blocks import qk_norm_rope

    g = torch.Generator(device=cuda).manual_seed(8)
    q, k, gq, gk = (torch.randn(1, 5, 2, 64, device=cuda, generator=g) for _ in range(4))
    w = torch.ones(64, device=cuda)
    cos, sin = (torch.randn(1, 5, 64, device=cuda, generator=g) for _ in range(2))
    leaves = [t.requires_grad_() for t in (q, k, w)]
    out = qk_norm_rope(q, k, w, w, cos, sin)
    plain = torch.autograd.grad(out, leaves, (gq, gk), retain_graph=True)
    gq.requires_grad_()
    graph = torch.autograd.grad(out, leaves, (gq, gk), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, graph))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        graph[0].sum().backward()
