"""Head norms where a warp walks several items -- over chunks of a position's heads, positions and batch entries -- and
sums weight gradients over all of them, against 64 bits; comparisons that a value which is no number fails."""

from __future__ import annotations

import pytest
import torch

import test_gpu_qk_norm_rope as base

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _close(got, want, mag, n):
    """As the other tests' (one rounding to the type, n of 2^-24 of the magnitudes), and false for NaN."""
    tiny = {F16: 2.0 ** -25}.get(got.dtype, 0.0)
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + n * base.ULP * mag * 1.01 + tiny
    ok = (got.double() - want).abs() <= tol
    assert ok.all(), f"{int((~ok).sum())} of {ok.numel()} off"


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    monkeypatch.setattr(base, "_close", _close)


@pytest.mark.parametrize("case", base.CASES)
def test_the_short_cases_hold_numbers(cuda, case):
    base.test_forward_and_backward_against_64_bits(cuda, *case)


def test_the_strided_cases_hold_numbers(cuda):
    base.test_strided_heads_and_gradients_and_wide_weights(cuda)


# B, S, Hq, Hk, D, R, heads, tables and weights.  With 148 SMs and 128 lanes a block: heads split in two chunks of five
# steps, some two items a warp; whole positions of four steps; teams of run-time size (float32 tables beside 16-bit
# heads, D of 16 and 512) and of each compile-time size; a sequence shorter than the stride over the items, so that one
# step of the walk passes several batch entries.
WALKS = [
    (3, 1021, 40, 8, 128, 128, BF16, BF16),
    (3, 1021, 40, 8, 128, 32, BF16, F32),
    (8, 2048, 16, 8, 128, 128, BF16, BF16),
    (3, 1021, 40, 8, 128, 128, F32, F32),
    (5, 1999, 14, 2, 96, 32, F16, F16),
    (2, 4099, 9, 3, 64, 64, F32, F32),
    (2, 3001, 6, 1, 256, 64, BF16, BF16),
    (701, 11, 33, 1, 16, 16, F16, F32),
    (2111, 5, 4, 2, 512, 256, BF16, BF16),
    (6000, 1, 8, 8, 80, 80, BF16, BF16),
]


@pytest.mark.parametrize("B,S,Hq,Hk,D,R,dtype,side", WALKS)
@pytest.mark.parametrize("offset", [0.0, 1.0])
def test_walks_against_64_bits(cuda, B, S, Hq, Hk, D, R, dtype, side, offset):
    g = torch.Generator(device=cuda).manual_seed(B * 31 + S + D)

    def rnd(*shape, dt=dtype, scale=1.0):
        return (torch.randn(*shape, generator=g, device=cuda) * scale).to(dt)

    cos, sin = base._tables(S, R, side, cuda, first=99, B=B if B < 10 else 1)
    base._check(rnd(B, S, Hq, D, scale=3.0), rnd(B, S, Hk, D), (1 - offset) + rnd(D, dt=side, scale=0.2),
                (1 - offset) + rnd(D, dt=side, scale=0.2), cos, sin, rnd(B, S, Hq, D), rnd(B, S, Hk, D), 1e-6, offset)


def test_repeats_of_a_walk_give_the_same_bits(cuda):
    from voodoo_quant import _C

    g = torch.Generator(device=cuda).manual_seed(2)
    q, gq = (torch.randn(3, 1021, 40, 128, generator=g, device=cuda).to(BF16) for _ in range(2))
    k, gk = (torch.randn(3, 1021, 8, 128, generator=g, device=cuda).to(BF16) for _ in range(2))
    w = torch.rand(128, generator=g, device=cuda)
    cos, sin = base._tables(1021, 128, BF16, cuda)
    runs = []
    for _ in range(3):
        qo, ko, ops, layout = _C.qk_norm_rope_fwd(q, k, w, w, cos, sin, 1e-6, saved=True)
        runs.append((qo, ko, *_C.qk_norm_rope_bwd(gq, gk, ops, layout)))
    frozen = _C.qk_norm_rope_bwd(gq, gk, ops, layout, False)
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))
    # without the weights' gradients another kernel: the same dx
    assert torch.equal(frozen[0], runs[0][2]) and torch.equal(frozen[1], runs[0][3]) and frozen[2] is None


def test_gradients_of_heads_that_hold_nothing_or_too_much(cuda):
    """A head of zeros passes g * w / sqrt(eps) on; NaN and infinity stay in their own head's dx."""
    from voodoo_quant.fused_blocks import qk_norm_rope

    S, H, D, eps = 5, 4, 128, 1e-6
    g = torch.Generator(device="cpu").manual_seed(4)
    q, gq = (torch.randn(1, S, H, D, generator=g).to(BF16).to(cuda) for _ in range(2))
    q[0, 1, 2] = 0
    clean = q.clone()
    q[0, 2, 1, 5] = float("nan")
    q[0, 3, 0, 100] = float("inf")
    w = (torch.rand(D, generator=g) + 0.5).to(BF16).to(cuda)
    cos, sin = base._tables(S, D, BF16, cuda)

    def dx(x):
        x = x.detach().requires_grad_()
        out = qk_norm_rope(x, x.detach()[:, :, :2], w, w, cos, sin, eps)
        return torch.autograd.grad(out[0], x, gq)[0]

    got, ref = dx(q), dx(clean)
    other = torch.ones(1, S, H, dtype=torch.bool, device=cuda)
    other[0, 2, 1] = other[0, 3, 0] = False
    assert torch.isfinite(ref).all() and torch.equal(got[other], ref[other])
    assert torch.isnan(got[0, 2, 1]).all() and torch.isnan(got[0, 3, 0]).any()
    want, mag, _, _ = base._backward64(gq.double(), clean.double(), w.double(), cos.double(), sin.double(), eps, 0.0)
    _close(ref, want, mag, 64)
    c, s, gz = cos[0, 1].double(), sin[0, 1].double(), gq[0, 1, 2].double()
    a, b = gz[:64], gz[64:]
    zero = torch.cat([a * c[:64] + b * s[64:], b * c[64:] - a * s[:64]]) * w.double() / eps ** 0.5
    assert ((ref[0, 1, 2].double() - zero).abs() <= 2.0 ** -8 * zero.abs() + 64 * base.ULP * mag[0, 1, 2]).all()
