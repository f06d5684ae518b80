"""The embedding module of a vocabulary shard on the GPU: the shards' outputs add up to the whole table's, rows and gate
gradients."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu


def _module(weight, cuda, spec=None, scale=None):
    from voodoo_quant.layers import replace_embedding_with_mixed_quant
    from voodoo_quant.parallel import VocabParallelEmbedding
    from voodoo_quant.training.synthetic import rtn_candidate_provider

    m = nn.Module()
    if spec is None:
        m.emb = nn.Embedding(*weight.shape, device=cuda, dtype=weight.dtype)
        m.emb.weight.data.copy_(weight)
    else:
        m.emb = VocabParallelEmbedding(spec.slice_weight(weight), spec, weight)
    if scale is not None:
        m.emb.embed_scale = scale
    replace_embedding_with_mixed_quant(m, ["Q4_K", "Q6_K", "Q8_0"], candidate_provider=rtn_candidate_provider)
    return m.emb


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [None, 16.0])
def test_shards_add_up_to_the_whole_table(cuda, dtype, scale):
    from voodoo_quant import _C
    from voodoo_quant.parallel import ShardSpec

    V, D, cut = 300, 512, 130
    g = torch.Generator(device=cuda).manual_seed(3)
    weight = (torch.randn(V, D, generator=g, device=cuda) * 0.02).to(dtype)
    specs = [ShardSpec(full_out=V, full_in=D, row_offset=a, row_len=b - a, vocab_start=a) for a, b in ((0, cut), (cut, V))]
    whole, *parts = [_module(weight, cuda, s, scale) for s in (None, *specs)]
    assert [p.tp_vocab_start for p in parts] == [0, cut] and parts[0].num_embeddings == cut
    gates = torch.randn(3, generator=g, device=cuda)
    ids = torch.randint(0, V, (4, 700), generator=g, device=cuda)
    ids[:, ::3] = cut  # the first row of the second shard, many times
    ids[0, 0], ids[0, 1] = cut - 1, V - 1
    dy = torch.randn(4, 700, D, generator=g, device=cuda).to(dtype)
    out, grads = [], []
    for m in (whole, *parts):
        with torch.no_grad():
            m.gates.copy_(gates)
            plain = m(ids)
        e = m(ids)
        assert e.dtype == dtype and e.shape == (4, 700, D) and torch.equal(e, plain)
        e.backward(dy)
        out.append(e.detach())
        grads.append(m.gates.grad.double())
    here = ids < cut
    # every row is one shard's, the other's is zeros: no rounding in the sum
    assert torch.equal(out[0], out[1] + out[2])
    assert not out[1][~here].any() and not out[2][here].any()
    # the gradient's sums differ in their cut: each side is within 64 roundings of 2^-24 of its terms' magnitudes (at most
    # |dy| times three times a row's largest weight; as a gate's twice a probability's) and 6 of the softmax's backward
    mag = 6 * (scale or 1.0) * float((dy.double().abs().sum(-1) * weight.double().abs().amax(1)[ids]).sum())
    assert ((grads[0] - grads[1] - grads[2]).abs() <= 140 * 2.0 ** -24 * mag).all() and grads[0].any()
    assert _C.device_error() == 0


def test_a_shards_rows_are_summed_in_place(cuda, monkeypatch):
    """With the all-reduce replaced by the addition of the other shard's rows: the in-place sum is taken, and the backward
    runs behind it."""
    from voodoo_quant import parallel

    V, D, cut = 300, 512, 130
    g = torch.Generator(device=cuda).manual_seed(5)
    weight = (torch.randn(V, D, generator=g, device=cuda) * 0.02).bfloat16()
    specs = [parallel.ShardSpec(full_out=V, full_in=D, row_offset=a, row_len=b - a, vocab_start=a)
             for a, b in ((0, cut), (cut, V))]
    whole, first, second = [_module(weight, cuda, s) for s in (None, *specs)]
    ids = torch.randint(0, V, (2, 300), generator=g, device=cuda)
    dy = torch.randn(2, 300, D, generator=g, device=cuda).bfloat16()
    with torch.no_grad():
        other, want = second(ids), whole(ids)
    alone = first(ids)
    alone.backward(dy)
    grad, first.gates.grad = first.gates.grad.clone(), None
    summed = []

    def all_reduce(t, *args, **kw):
        summed.append(t.data_ptr())
        t.add_(other)

    monkeypatch.setattr(parallel.TP, "enabled", True)
    monkeypatch.setattr(parallel.dist, "all_reduce", all_reduce)
    monkeypatch.setattr(parallel, "_fwd_group", lambda: None)
    e = first(ids)
    assert summed == [e.data_ptr()] and torch.equal(e, want)
    e.backward(dy)
    assert torch.equal(first.gates.grad, grad)
    with torch.no_grad():
        assert torch.equal(first(ids), want)
