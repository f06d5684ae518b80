"""Which gradients clip_grad_norm_ takes to share memory: strided ones decided before any of them is copied.  The
kernel is replaced by torch on the CPU; the GPU test runs the same cases through it."""

from __future__ import annotations

import random

import pytest
import torch


def _param(g):
    p = torch.nn.Parameter(torch.empty(0, device=g.device))
    p.data = torch.zeros(1, device=g.device).expand(g.shape)
    p.grad = g
    return p


def _views(base, *geometry):
    return [base.as_strided(size, stride, at) for size, stride, at in geometry]


SHARED = [
    # the same strided gradient twice, overlapping column ranges, rows and columns that cross
    [((30, 20), (50, 1), 10), ((30, 20), (50, 1), 10)],
    [((30, 20), (50, 1), 0), ((30, 20), (50, 1), 19)],
    [((30, 20), (50, 1), 10), ((1, 50), (50, 1), 0)],
    # a strided view beside the contiguous gradient that it lies in, in either order
    [((30, 20), (50, 1), 10), ((30, 50), (50, 1), 0)],
    [((30, 50), (50, 1), 0), ((30, 20), (50, 1), 10)],
    # a transposed view over the same columns, every third value over every second
    [((20, 30), (1, 50), 10), ((30, 5), (50, 1), 12)],
    [((100,), (3,), 0), ((100,), (2,), 3)],
    # strides that make a tensor meet itself, none of them 0
    [((4, 4), (2, 3), 0)],
    [((5, 3), (2, 1), 0)],
    [((3, 3), (7, 7), 0)],
]
APART = [
    [((30, 20), (50, 1), 10), ((30, 10), (50, 1), 0), ((30, 20), (50, 1), 30)],
    [((20, 30), (1, 50), 10), ((30, 10), (50, 1), 0)],
    [((100,), (2,), 0), ((100,), (2,), 1)],
    [((2, 3), (3, 2), 0)],  # 0 2 4 3 5 7: no stride spans the other's reach, and yet no value twice
    [((10, 4), (50, 1), 0), ((40,), (1,), 500), ((3, 4), (5, 1), 4)],
    [((7, 3, 5), (1, 40, 8), 0), ((7, 3), (1, 40), 1000), ((2, 2), (400, 7), 161)],
]


def _stand_in(tensors, max_norm=float("inf"), norm_inf=False):
    """What the kernel does, for float32 on the CPU, with its own refusals."""
    from voodoo_quant import _C

    if not all(t.is_contiguous() for t in tensors):
        raise _C.NotContiguous("contiguous tensors expected")
    spans = sorted((t.data_ptr(), t.data_ptr() + t.nbytes) for t in tensors if t.numel())
    if any(b < e for (_, e), (b, _) in zip(spans, spans[1:])):
        raise ValueError("two of the tensors share memory: each value is scaled once")
    flat = torch.cat([t.reshape(-1).double() for t in tensors])
    norm = flat.abs().max() if norm_inf else flat.norm()
    if max_norm != float("inf"):
        for t in tensors:
            t.mul_(min(1.0, max_norm / (float(norm) + 1e-6)))
    return norm.float()


def _run(device):
    from voodoo_quant.training.grad_clip import clip_grad_norm_, grad_norm

    for geometry in SHARED:
        base = torch.ones(2000, device=device)
        grads = _views(base, *geometry)
        with pytest.raises(ValueError, match="share memory|shares memory"):
            clip_grad_norm_([_param(g) for g in grads], 0.5)
        with pytest.raises(ValueError, match="share memory|shares memory"):
            grad_norm(grads)
        assert torch.equal(base, torch.ones_like(base))
    for geometry in APART:
        base = torch.ones(2000, device=device)
        grads = _views(base, *geometry)
        n = sum(g.numel() for g in grads)
        norm = clip_grad_norm_([_param(g) for g in grads], 0.5)
        assert abs(float(norm) - n ** 0.5) <= 1e-6 * n ** 0.5
        assert abs(float(base.double().square().sum()) - (0.25 + 2000 - n)) <= 1e-4
        assert int((base != 1).sum()) == n


def test_strided_gradients_that_share_memory(monkeypatch):
    from voodoo_quant import _C

    monkeypatch.setattr(_C, "clip_grad_norm", _stand_in)
    _run("cpu")


@pytest.mark.gpu
def test_strided_gradients_that_share_memory_on_the_gpu(cuda):
    _run(cuda)


def test_against_the_sets_of_their_bytes():
    """Random small geometries of two types in one buffer against the sets of bytes that they touch."""
    from voodoo_quant.training.grad_clip import _meets_itself, _share

    rng = random.Random(5)
    raw = torch.zeros(4096, dtype=torch.uint8)

    def touched(t):
        at, es = t.data_ptr() - raw.data_ptr(), t.element_size()
        offsets = [at]
        for n, st in zip(t.shape, t.stride()):
            offsets = [o + i * st * es for o in offsets for i in range(n)]
        return [o + k for o in offsets for k in range(es)]

    kinds = {True: 0, False: 0}
    selves = {True: 0, False: 0}
    for _ in range(3000):
        pair = []
        for _ in range(2):
            buf = raw.view(rng.choice([torch.float32, torch.bfloat16]))
            dims = rng.randint(1, 3)
            size = [rng.randint(1, 5) for _ in range(dims)]
            stride = [rng.randint(0, 24) for _ in range(dims)]
            pair.append(buf.as_strided(size, stride, rng.randint(0, 60)))
        a, b = (touched(t) for t in pair)
        want = bool(set(a) & set(b))
        assert _share(*pair) == want and _share(*pair[::-1]) == want
        kinds[want] += 1
        want = len(set(a)) < len(a)
        assert _meets_itself(pair[0]) == want
        selves[want] += 1
    assert min(kinds.values()) > 300 and min(selves.values()) > 300


def test_large_column_ranges_are_decided_quickly():
    """Disjoint and touching column ranges of a buffer of 2^34 values (no memory behind it)."""
    from voodoo_quant.training.grad_clip import _refuse_sharing

    base = torch.empty(2 ** 17, 2 ** 17, device="meta")

    class At:  # a meta tensor with an address
        def __init__(self, t):
            self.t = t

        def __getattr__(self, name):
            return getattr(self.t, name)

        def data_ptr(self):
            return 4096 + 4 * self.t.storage_offset()

    cols = [At(base[:, 1000 * i:1000 * i + 1000]) for i in range(60)]
    _refuse_sharing(cols)
    with pytest.raises(ValueError, match="share memory"):
        _refuse_sharing(cols + [At(base[5:, 500:600])])
