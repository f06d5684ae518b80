"""Global norm and clipping of many gradients against 64 bits.

Tolerances: the squares of a vector of eight are summed in fp32 (8 roundings
of 2^-24 at most) and joined in 64 bits, so the norm is within 4 * 2^-24 and
its own rounding to float32; the factor adds three more, and each value is
rounded once to its type.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -24


def _params(shapes, dtypes, cuda, seed, scale=1.0, offset=0):
    """Parameters whose gradients are neighbouring pieces of one buffer per type, so most start at odd addresses."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    flat = {dt: torch.randn(offset + sum(math.prod(s) for s, d in zip(shapes, dtypes) if d == dt), generator=g)
            .mul_(scale).to(dt).to(cuda) for dt in set(dtypes)}
    at = {dt: offset for dt in flat}
    params = []
    for s, dt in zip(shapes, dtypes):
        n = math.prod(s)
        p = torch.zeros(s, dtype=dt, device=cuda, requires_grad=True)
        p.grad = flat[dt][at[dt]:at[dt] + n].view(s)
        at[dt] += n
        params.append(p)
    return params, flat


def _check(params, flat, max_norm, norm_type=2.0, offset=0):
    from voodoo_quant.training.grad_clip import clip_grad_norm_

    before = {dt: f.clone() for dt, f in flat.items()}
    all64 = torch.cat([f[offset:].double() for f in flat.values()])
    want = float(all64.norm() if norm_type == 2.0 else all64.abs().max())
    norm = clip_grad_norm_(params, max_norm, norm_type)
    assert norm.shape == () and norm.dtype == torch.float32 and norm.is_cuda
    assert abs(float(norm) - want) <= 6 * ULP * want
    scale = min(1.0, max_norm / (want + 1e-6))
    for dt, f in flat.items():
        b = before[dt].double()
        tiny = {torch.float16: 2.0 ** -25}.get(dt, 0.0)
        tol = (torch.finfo(dt).eps / 2 + 10 * ULP) * b.abs() * scale + tiny
        if scale == 1.0:
            assert torch.equal(f, before[dt])
        else:
            assert ((f.double() - b * scale)[offset:].abs() <= tol[offset:]).all()
        assert torch.equal(f[:offset], before[dt][:offset])
    return norm


F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CASES = [
    ([(6,)] * 226, [F32]),
    ([(1,)], [BF16]),
    ([(3,), (0,), (5, 7), ()], [F16]),
    ([(16384,)], [F32]),
    ([(4096,)], [F32]),
    ([(4097,)], [F32]),
    ([(255,), (256,), (257,), (1,), (2000,), (512,), (513,)], [BF16, F32, F16]),
    ([(16385,)], [F32]),
    ([(257, 129), (8191,), (8192,), (8193,), (1,), (100003,)], [BF16]),
    ([(n,) for n in range(1, 60)], [F32, BF16, F16]),
    ([(1000,)] * 700, [BF16, F32]),
    ([(11,)] * 241, [F32]),
    ([(40,)] * 3300, [F16, F32]),
    ([(3_000_001,), (5,), (1 << 20,)], [BF16, F16, F32]),
]


@pytest.mark.parametrize("shapes,kinds", CASES)
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_clip_against_64_bits(cuda, shapes, kinds, max_norm, norm_type):
    dtypes = [kinds[i % len(kinds)] for i in range(len(shapes))]
    for offset in (0, 1):
        params, flat = _params(shapes, dtypes, cuda, len(shapes), offset=offset)
        _check(params, flat, max_norm, norm_type, offset)


def test_neighbours_are_left_alone(cuda):
    """Values before, between and behind the clipped tensors stay as they are."""
    from voodoo_quant.training.grad_clip import clip_grad_norm_

    for dt in (F32, BF16, F16):
        flat = torch.ones(200001, dtype=dt, device=cuda)
        cuts = [(1, 5), (9, 10), (33, 20000), (20003, 20003), (20005, 199998)]
        params, mask = [], torch.zeros(200001, dtype=torch.bool, device=cuda)
        for a, b in cuts:
            p = torch.zeros(b - a, dtype=dt, device=cuda, requires_grad=True)
            p.grad = flat[a:b]
            mask[a:b] = True
            params.append(p)
        clip_grad_norm_(params, 0.25)
        assert (flat[~mask] == 1).all() and (flat[mask] < 0.01).all()


def test_strided_gradients(cuda):
    """A transposed gradient is scaled where it lies; one with gaps leaves the gaps."""
    from voodoo_quant.training.grad_clip import clip_grad_norm_

    g = torch.Generator(device="cpu").manual_seed(1)
    base = torch.randn(40, 64, generator=g).to(cuda)
    wide = torch.randn(30, 50, generator=g).to(cuda)
    p1 = torch.zeros(64, 40, device=cuda, requires_grad=True)
    p2 = torch.zeros(30, 20, device=cuda, requires_grad=True)
    p1.grad, p2.grad = base.t(), wide[:, 10:30]
    b0, w0 = base.clone(), wide.clone()
    want = float(torch.cat([b0.flatten(), w0[:, 10:30].flatten()]).double().norm())
    norm = clip_grad_norm_([p1, p2], 1.0)
    assert abs(float(norm) - want) <= 6 * ULP * want
    s = 1.0 / (want + 1e-6)
    assert torch.allclose(base.double(), b0.double() * s, rtol=1e-6, atol=0)
    w0[:, 10:30] = (w0[:, 10:30].double() * s).float()
    assert torch.equal(wide[:, :10], w0[:, :10]) and torch.equal(wide[:, 30:], w0[:, 30:])
    assert torch.allclose(wide, w0, rtol=1e-6, atol=0)


def test_values_whose_squares_leave_float32(cuda):
    from voodoo_quant.training.grad_clip import clip_grad_norm_

    for dt in (F32, BF16):
        for v in (1e30, 1e-30, 3e-38):
            for n in (100, 100000):
                p = torch.zeros(n, dtype=dt, device=cuda, requires_grad=True)
                p.grad = torch.full((n,), v, dtype=dt, device=cuda)
                val = float(p.grad[0])
                want = val * math.sqrt(n)
                assert abs(float(clip_grad_norm_([p], math.inf)) - want) <= 6 * ULP * want


@pytest.mark.parametrize("n", [10, 50000])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_what_is_not_finite(cuda, n, norm_type):
    """As torch's clipping: NaN makes every value NaN, infinity makes finite values zero; error_if_nonfinite raises with
    the gradients as they were."""
    from voodoo_quant.training.grad_clip import clip_grad_norm_, grad_norm

    for bad in (math.nan, math.inf):
        def fresh():
            p = torch.zeros(n, device=cuda, requires_grad=True)
            p.grad = torch.ones(n, device=cuda)
            p.grad[n // 2] = bad
            return p

        p = fresh()
        with pytest.raises(RuntimeError, match="non-finite"):
            clip_grad_norm_([p], 1.0, norm_type, error_if_nonfinite=True)
        assert float(p.grad[0]) == 1.0
        norm = clip_grad_norm_([p], 1.0, norm_type)
        ref = fresh()
        rn = torch.nn.utils.clip_grad_norm_([ref], 1.0, norm_type)
        assert torch.equal(torch.isnan(norm), torch.isnan(rn)) and float(norm) == float(rn) or math.isnan(float(rn))
        assert torch.equal(torch.isnan(p.grad), torch.isnan(ref.grad))
        ok = ~torch.isnan(ref.grad)
        assert torch.equal(p.grad[ok], ref.grad[ok])
        assert not math.isfinite(float(grad_norm([fresh().grad], norm_type)))
        p = fresh()
        clip_grad_norm_([p], math.inf, norm_type)
        assert float(p.grad[0]) == 1.0


def test_zeros_and_a_bound_of_zero(cuda):
    from voodoo_quant.training.grad_clip import clip_grad_norm_

    for n in (7, 100000):
        p = torch.zeros(n, device=cuda, requires_grad=True)
        p.grad = torch.zeros(n, device=cuda)
        assert float(clip_grad_norm_([p], 1.0)) == 0.0 and not p.grad.any()
        p.grad = torch.ones(n, device=cuda)
        clip_grad_norm_([p], 0.0)
        assert not p.grad.any()
    assert float(clip_grad_norm_([], 1.0)) == 0.0
    q = torch.zeros(3, device=cuda, requires_grad=True)
    assert float(clip_grad_norm_([q], 1.0)) == 0.0  # no gradient yet


def test_shared_memory_is_refused(cuda):
    from voodoo_quant.training.grad_clip import clip_grad_norm_

    g = torch.ones(100, device=cuda)
    ps = [torch.zeros(50, device=cuda, requires_grad=True) for _ in range(3)]
    ps[0].grad, ps[1].grad, ps[2].grad = g[:50], g[50:], g[49:99]
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_(ps, 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_([ps[0], ps[0]], 1.0)
    e = torch.zeros(4, 5, device=cuda, requires_grad=True)
    e.grad = torch.ones(4, 1, device=cuda).expand(4, 5)
    with pytest.raises(ValueError, match="expanded"):
        clip_grad_norm_([e], 1.0)
    assert (g == 1).all()


@pytest.mark.parametrize("n", [6, 30000])
def test_a_graph_that_saved_a_gradient_notices(cuda, n):
    """As after any other change in place: the backward of what was computed from the gradients before they were scaled
    raises; taking the norm alone changes nothing."""
    from voodoo_quant.training.grad_clip import clip_grad_norm_, grad_norm

    p = torch.nn.Parameter(torch.ones(n, device=cuda))
    (p.grad,) = torch.autograd.grad((p ** 3).sum(), p, create_graph=True)
    penalty = (p.grad ** 2).sum()
    grad_norm([p.grad])
    (g,) = torch.autograd.grad(penalty, p, retain_graph=True)
    assert torch.equal(g, torch.full_like(g, 36.0))  # d(3 p^2)^2 / dp = 36 p^3
    clip_grad_norm_([p], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(penalty, p)


@pytest.mark.parametrize("n", [6, 30000])
def test_streams_graphs_and_repeats(cuda, n):
    from voodoo_quant.training.grad_clip import clip_grad_norm_

    params, flat = _params([(n,)] * 20, [F32], cuda, 3)
    f = flat[F32]
    start = f.clone()
    want_norm = clip_grad_norm_(params, 1.0).clone()
    want = f.clone()
    side = torch.cuda.Stream()
    f.copy_(start)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm = clip_grad_norm_(params, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(norm, want_norm) and torch.equal(f, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(params, 1.0)
    for k in (1.0, 3.0):
        f.copy_(start * k)
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(norm) - k * float(want_norm)) <= 4 * ULP * k * float(want_norm)
        assert torch.allclose(f, want, rtol=1e-6, atol=0)


def test_trainer_clips_its_gates(cuda):
    """The trainer's update against torch's clipping of the same gradients."""
    from voodoo_quant.training.trainer import StepArgs, build_distill

    trainer, shape = build_distill("tiny", cuda, seed=0, args=StepArgs(max_steps=4))
    g = torch.Generator(device="cpu").manual_seed(2)
    want = []
    for p in trainer.trainable:
        p.grad = torch.randn(p.shape, generator=g).to(cuda)
        want.append(p.grad.clone())
    ref = [torch.zeros_like(p, requires_grad=True) for p in trainer.trainable]
    for p, w in zip(ref, want):
        p.grad = w
    torch.nn.utils.clip_grad_norm_(ref, 1.0)
    trainer.apply_update()
    for p, r in zip(trainer.trainable, ref):
        # the norms differ by a few roundings, and each value by its own
        assert torch.allclose(p.grad, r.grad, rtol=16 * ULP, atol=0)


def test_a_tensor_of_more_than_2_to_the_31_values(cuda):
    """Powers of two, so that the norm is known: n values of 1 / 2 have the norm sqrt(n) / 2."""
    from voodoo_quant.training.grad_clip import clip_grad_norm_

    n = 2 ** 31 + 2 ** 20 + 5
    p = torch.nn.Parameter(torch.empty(0, dtype=torch.bfloat16, device=cuda))
    p.data = torch.empty(1, dtype=torch.bfloat16, device=cuda).expand(n)
    p.grad = torch.full((n,), 0.5, dtype=torch.bfloat16, device=cuda)
    norm = clip_grad_norm_([p], math.sqrt(n) / 4)
    assert abs(float(norm) - math.sqrt(n) / 2) <= 6 * ULP * float(norm)
    # the factor is 1/2 within a few roundings of 2^-24: 0.25 is the nearest bf16 value by far
    assert (p.grad[0], p.grad[-1]) == (0.25, 0.25) and int((p.grad == 0.25).sum()) == n
