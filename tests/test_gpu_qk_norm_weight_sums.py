"""The head norms' weight gradient where many terms meet in one lane, and where some of a step's
lanes hold no head."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -24


def test_long_sums_keep_their_bits(cuda):
    """2^20 positions of equal heads: every lane adds some thousand equal terms, whose rounding to the sum's own step is
    the same each time and so adds up.  Sums of at most 32 positions' and one position's heads in 32 bits, joined in 64,
    keep 36 roundings of 2^-24 here, the teams of a warp and the roundings of a block's sum and of the result 5 more; a
    normed value is off by the same factor everywhere, half of the 20 roundings of the mean square, a reciprocal root of
    4 and a product: 64 in all."""
    from voodoo_quant.fused_blocks import qk_norm_rope

    S, Hq, Hk, D, R = 1 << 20, 16, 1, 128, 16
    g = torch.Generator(device="cpu").manual_seed(3)
    x = (0.5 + torch.rand(2, D, generator=g)).to(torch.bfloat16).to(cuda)
    q, k = x[0].expand(1, S, Hq, D), x[1].expand(1, S, Hk, D)
    wq, wk = (torch.ones(D, device=cuda, requires_grad=True) for _ in range(2))
    cos, sin = (torch.full((1, 1, R), v, dtype=torch.bfloat16, device=cuda).expand(1, S, R) for v in (1.0, 0.0))
    one = torch.ones(1, dtype=torch.bfloat16, device=cuda)
    out = qk_norm_rope(q, k, wq, wk, cos, sin, 1e-6)
    dw = torch.autograd.grad(out, (wq, wk), (one.expand(1, S, Hq, D), one.expand(1, S, Hk, D)))
    del out
    for got, row, H in ((dw[0], x[0], Hq), (dw[1], x[1], Hk)):
        r = row.double()
        want = r * (r.square().mean() + 1e-6).rsqrt() * (S * H)
        off = ((got.double() - want).abs() / want).max()
        assert off <= 64 * ULP, f"{off / ULP:.0f} roundings of 2^-24"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_an_infinite_gradient_of_the_last_head(cuda, dtype):
    """5 heads of 128, four to a step: the lanes past the last head read it again and must add nothing of it, not even
    infinity times 0."""
    from voodoo_quant.fused_blocks import qk_norm_rope

    S, H, D, R = 3, 5, 128, 32
    g = torch.Generator(device="cpu").manual_seed(9)
    q, k, gq, gk = (torch.randn(1, S, H, D, generator=g).to(dtype).to(cuda) for _ in range(4))
    q[0, 1, H - 1, 100] = 0.5
    w = torch.ones(D, dtype=dtype, device=cuda, requires_grad=True)
    cos, sin = (torch.randn(1, S, R, generator=g).to(dtype).to(cuda) for _ in range(2))

    def grad(gq):
        return torch.autograd.grad(qk_norm_rope(q, k, w, w.detach(), cos, sin), w, (gq, gk))[0]

    clean = grad(gq)
    gq[0, 1, H - 1, 100] = math.inf
    bad = grad(gq)
    rest = torch.arange(D, device=cuda) != 100
    assert torch.isfinite(clean).all() and torch.equal(bad[rest], clean[rest])
    assert float(bad[100]) == math.inf
