"""Global gradient norm over many tensors, and clipping, on the B200 kernels.

The reference's step clips its gates' gradients with
``torch.nn.utils.clip_grad_norm_`` (voodoo_quant/training/trainer.py:2607-2616):
a norm per tensor, a norm of the norms and a product per tensor.  Here two
launches (one for a few thousand values) take the norm of all tensors and
scale them in place (``vq_clip_grad_norm``); nothing is read on the host.
"""

from __future__ import annotations

import math

import torch

from voodoo_quant import _C


def _norm_is_inf(norm_type: float) -> bool:
    if float(norm_type) not in (2.0, math.inf):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    return math.isinf(norm_type)


def _dense(g: torch.Tensor) -> torch.Tensor | None:
    """A contiguous view of all of g's memory, or None where g has gaps or overlaps."""
    if g.layout is not torch.strided:
        raise ValueError(f"clip_grad_norm_: dense gradients expected, got {g.layout}")
    if g.is_contiguous():
        return g
    order = sorted(range(g.dim()), key=lambda d: (g.stride(d), g.shape[d]), reverse=True)
    v = g.permute(order)
    return v if v.is_contiguous() else None


def _solvable(terms, target: int, budget: int = 1 << 16) -> bool:
    """Whether sum d_i c_i = target for whole d_i from lo_i to hi_i; terms: (c_i > 0, lo_i, hi_i).  Taken from the
    largest c_i down, each d_i only as far as the terms behind it can make up for; where that still leaves more than
    ``budget`` ways to try, the answer is yes."""
    terms = sorted(terms, reverse=True)
    low, high = [0], [0]
    for c, lo, hi in reversed(terms):
        low.append(low[-1] + c * lo)
        high.append(high[-1] + c * hi)
    low.reverse(), high.reverse()
    todo = [(0, target)]
    while todo:
        i, t = todo.pop()
        if i == len(terms):
            return True  # what is left is 0: the bounds below leave no other
        c, lo, hi = terms[i]
        first, last = max(lo, -((high[i + 1] - t) // c)), min(hi, (t - low[i + 1]) // c)
        budget -= max(last - first + 1, 1)
        if budget < 0:
            return True
        todo.extend((i + 1, t - c * d) for d in range(first, last + 1))
    return False


def _steps(t: torch.Tensor, es: int):
    return [(s * es, n - 1) for s, n in zip(t.stride(), t.shape) if n > 1]


def _meets_itself(t: torch.Tensor) -> bool:
    """Whether two places of t are one in memory."""
    steps = sorted(_steps(t, 1), reverse=True)
    if any(s == 0 for s, _ in steps):
        return True
    # two places that differ by d_i along each dimension, d of the largest stride that differs positive
    return any(_solvable([(s, 1, n)] + [(u, -m, m) for u, m in steps[i + 1:]], 0) for i, (s, n) in enumerate(steps))


def _share(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether a byte of a is one of b."""
    ea, eb = a.element_size(), b.element_size()
    terms = {1: (-(eb - 1), ea - 1)}  # a byte of each of the two values
    for steps, sign in ((_steps(a, ea), 1), (_steps(b, eb), -1)):
        for s, n in steps:
            if s:
                lo, hi = terms.get(s, (0, 0))
                terms[s] = (lo - n, hi) if sign < 0 else (lo, hi + n)
    return _solvable([(c, lo, hi) for c, (lo, hi) in terms.items()], b.data_ptr() - a.data_ptr())


def _refuse_sharing(grads) -> None:
    """Refuses gradients with gaps that meet themselves or another gradient: scaled as copies, the copies' addresses
    would not tell.  (Two without gaps are the library's to compare.)"""
    spans = []
    for g in grads:
        if g.numel() == 0:
            continue
        gaps = _dense(g) is None
        if gaps and _meets_itself(g):
            if any(st == 0 and n > 1 for st, n in zip(g.stride(), g.shape)):
                raise ValueError("clip_grad_norm_: an expanded gradient shares memory with itself")
            raise ValueError("clip_grad_norm_: a gradient whose strides overlap shares memory with itself")
        es, at = g.element_size(), g.data_ptr()
        spans.append((at, at + es + sum(s * n for s, n in _steps(g, es)), gaps, g))
    spans.sort(key=lambda s: s[0])
    open_ = []  # of those before, what reaches past this one's first byte
    for span in spans:
        open_ = [o for o in open_ if o[1] > span[0]]
        if any((o[2] or span[2]) and _share(o[3], span[3]) for o in open_):
            raise ValueError("clip_grad_norm_: two of the gradients share memory: each value is scaled once")
        open_.append(span)


def _run(grads, max_norm: float, norm_type: float) -> torch.Tensor:
    norm_inf = _norm_is_inf(norm_type)
    try:
        return _C.clip_grad_norm(grads, max_norm, norm_inf)  # checks that they are contiguous
    except _C.NotContiguous:
        pass
    _refuse_sharing(grads)
    flat, copies = [], []
    for g in grads:
        v = _dense(g)
        if v is None:  # scaled as a copy
            v = g.contiguous()
            copies.append((g, v))
        flat.append(v)
    norm = _C.clip_grad_norm(flat, max_norm, norm_inf)
    if not math.isinf(max_norm):
        for g, v in copies:
            g.copy_(v)
    return norm


def grad_norm(grads, norm_type: float = 2.0) -> torch.Tensor:
    """Global norm of ``grads`` (CUDA tensors in float32, bfloat16 or float16, mixed freely, on one device) as a
    float32 scalar on that device; ``norm_type`` 2 or inf."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if not grads:
        return torch.tensor(0.0)
    with torch.no_grad():
        return _run(grads, math.inf, norm_type)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale the gradients of ``parameters`` in place so that their global norm is at most ``max_norm`` and return the
    norm they had (a float32 scalar on their device), as ``torch.nn.utils.clip_grad_norm_`` does: every value times
    min(1, max_norm / (norm + 1e-6)), a norm that is not finite included (NaN gives NaN, inf gives zeros and NaN).
    An infinite ``max_norm`` leaves the gradients as they are.  ``error_if_nonfinite`` reads the norm on the host and
    raises RuntimeError before anything is scaled.  Parameters without a gradient are skipped; ``norm_type`` 2 or inf;
    gradients that share memory (with one another or with themselves, whatever their strides), or carry forward-mode
    tangents, are refused."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [g for g in [p.grad for p in params] if g is not None]
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative or NaN, got {max_norm}")
    if not grads:
        _norm_is_inf(norm_type)
        return torch.tensor(0.0)
    with torch.no_grad():
        if error_if_nonfinite:
            norm = _run(grads, math.inf, norm_type)
            if not bool(torch.isfinite(norm)):
                raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` is "
                                   "non-finite, so it cannot be clipped")
        return _run(grads, max_norm, norm_type)
