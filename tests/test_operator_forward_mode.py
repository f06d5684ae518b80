"""Forward-mode tangents (``torch.autograd.forward_ad``) through the head norms, the gated embedding and the clipping:
the kernels know nothing of them, so every call that meets one raises; none returns or scales values whose tangent is
lost.  The launches are replaced, no GPU needed."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw


def _dual(t):
    return fw.make_dual(t, torch.ones_like(t))


@pytest.fixture
def launches(monkeypatch):
    """Stand-ins of the raw calls: outputs of the right shapes, and a list of those that were reached."""
    from voodoo_quant import _C

    seen = []

    def qk_fwd(q, k, wq, wk, cos, sin, *rest, saved=False):
        seen.append("qk")
        out = q.detach().clone(), k.detach().clone()
        return (*out, (q, k, wq, wk, cos, sin), None) if saved else out

    def qk_bwd(gq, gk, operands, layout, want=True):
        seen.append("qk backward")
        return tuple(torch.zeros_like(t) for t in operands[:4])

    class Table:
        def __init__(self, types, blocks, rows, padded, cols):
            self.rows, self.cols = rows, cols

    def mix(ids, table, probs, *rest):
        seen.append("mix")
        return torch.zeros(*ids.shape, table.cols, dtype=torch.bfloat16)

    def gategrad(dy, table, plan, scale=1.0):
        seen.append("gategrad")
        return torch.zeros(1)

    for name, f in (("qk_norm_rope_fwd", qk_fwd), ("qk_norm_rope_bwd", qk_bwd), ("EmbedTable", Table),
                    ("embed_plan", lambda *a: torch.zeros(1)), ("embed_mix", mix), ("embed_gategrad", gategrad)):
        monkeypatch.setattr(_C, name, f)
    return seen


@pytest.mark.parametrize("grad_enabled", [False, True])
@pytest.mark.parametrize("which", range(6))
def test_head_norms_refuse_tangents(launches, which, grad_enabled):
    from voodoo_quant.fused_blocks import qk_norm_rope

    x = [torch.randn(1, 2, 2, 16), torch.randn(1, 2, 1, 16), torch.ones(16), torch.ones(16), torch.ones(1, 2, 16),
         torch.ones(1, 2, 16)]
    with torch.set_grad_enabled(grad_enabled), fw.dual_level():
        x[which] = _dual(x[which])
        with pytest.raises(NotImplementedError, match="forward-mode"):
            qk_norm_rope(*x)
        assert not launches
        x[which] = fw.unpack_dual(x[which]).primal
        qk_norm_rope(*x)  # a level without tangents
    assert launches == ["qk"]


def test_functional_jvp_is_refused(launches):
    from voodoo_quant.fused_blocks import qk_norm_rope

    q, w, c = torch.randn(1, 2, 2, 16), torch.ones(16), torch.ones(1, 2, 16)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: qk_norm_rope(t, q, w, w, c, c)[0], (q,), (q,))
    assert not launches


@pytest.mark.parametrize("requires_grad", [False, True])
def test_gated_embedding_refuses_tangents(launches, requires_grad):
    from voodoo_quant.layers import gated_embedding

    ids, p = torch.zeros(3, dtype=torch.long), torch.ones(1, requires_grad=requires_grad)
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            gated_embedding(ids, _dual(p), ["Q8_0"], [None], 1, 256)
        assert not launches
        gated_embedding(ids, p, ["Q8_0"], [None], 1, 256)
    assert launches == ["mix"]


def test_backwards_refuse_tangents_of_the_gradients(launches):
    """Forward mode over the backward: the gradients of the outputs carry the tangents."""
    from voodoo_quant.fused_blocks import qk_norm_rope
    from voodoo_quant.layers import gated_embedding

    q = torch.randn(1, 2, 2, 16, requires_grad=True)
    w, c = torch.ones(16), torch.ones(1, 2, 16)
    out = qk_norm_rope(q, q.detach(), w, w, c, c)[0]
    p = torch.ones(1, requires_grad=True)
    rows = gated_embedding(torch.zeros(3, dtype=torch.long), p, ["Q8_0"], [None], 1, 256)
    with fw.dual_level():
        for y, leaf, name in ((out, q, "qk backward"), (rows, p, "gategrad")):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, leaf, _dual(torch.ones_like(y)), retain_graph=True)
            assert name not in launches
            torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)
            assert name in launches


def test_clipping_refuses_tangents():
    from voodoo_quant.training.grad_clip import clip_grad_norm_, grad_norm

    p, plain = torch.zeros(4, 3, requires_grad=True), torch.zeros(2, requires_grad=True)
    plain.grad = torch.ones(2)
    for g in (torch.ones(4, 3), torch.ones(4, 6)[:, ::2]):
        with fw.dual_level():
            p.grad = None
            d = _dual(g)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                grad_norm([plain.grad, d])
            p.grad = d
            with pytest.raises(NotImplementedError, match="forward-mode"):
                clip_grad_norm_([plain, p], 0.5)
            p.grad = None
        assert torch.equal(g, torch.ones(4, 3)) and torch.equal(plain.grad, torch.ones(2))
