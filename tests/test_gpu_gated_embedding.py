"""Gated embedding lookup and its gradient over the sorted tokens against the
definition in 64 bits (blocks decoded by the oracle).

Tolerances.  Lookup: for scale 1 the rows are vq_mix's bit for bit; for others
one bf16 rounding (2^-8) of the value plus the fp32 chain -- K candidates,
each a product and a sum, of magnitudes below three times the row's largest
weight (code times scale and the block's offset are each within twice the
largest), so below 2e-5 of it for K <= 8.  Gradient: chains of at most 64
roundings of 2^-24 (a piece's 8 rows of dy, then a sub-block of 32 weights)
relative to the sum of |dy| times three times the row's largest weight; the
runs are joined in 64 bits.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import ggml_blocks

pytestmark = pytest.mark.gpu

ALL = ["Q2_K", "Q3_K", "Q4_K", "Q5_K", "Q6_K", "Q8_0", "IQ4_XS"]


def _table(V, D, types, seed, cuda):
    """Packed candidates of a random table of V rows and D columns (rows padded to 256), and them decoded in 64 bits."""
    from voodoo_quant.quants import rtn

    g = torch.Generator(device="cpu").manual_seed(seed)
    P = (D + 255) // 256 * 256
    w = torch.zeros(V, P)
    w[:, :D] = torch.randn(V, D, generator=g) * 0.02
    blocks = {q: rtn.quantize(w, q) for q in types}
    dec = [torch.from_numpy(ggml_blocks.dequantize(blocks[q].numpy().reshape(-1), q, V, P).astype(np.float64))[:, :D]
           for q in types]
    p = torch.softmax(torch.randn(len(types), generator=g), 0)
    return w[:, :D].contiguous(), blocks, [blocks[q].to(cuda).contiguous() for q in types], dec, p


def _ids(T, V, seed, low=0):
    """Random ids of which a third are one token and some name no row."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    ids = torch.randint(low, V, (T,), generator=g)
    ids[torch.rand(T, generator=g) < 0.33] = V // 2
    return ids


def _check_lookup(out, ids, dec, p, scale, start, rows):
    local = ids - start
    here = (local >= 0) & (local < rows)
    row = local.clamp(0, max(rows - 1, 0))
    want = sum(float(pk) * d[row] for pk, d in zip(p, dec)) * scale * here[:, None]
    top = sum(float(pk) * d.abs().amax(1)[row] for pk, d in zip(p, dec)) * scale
    tol = 2.0 ** -8 * want.abs() + 2e-5 * top[:, None]
    assert ((out.double().cpu() - want).abs() <= tol).all()
    assert not out.cpu()[~here].any()


def _check_grad(grad, dy, ids, dec, scale, start, rows):
    local = ids - start
    here = (local >= 0) & (local < rows)
    row, d = local[here], dy.double().cpu()[here]
    for k, w in enumerate(dec):
        want = float((d * w[row]).sum()) * scale
        mag = float((d.abs().sum(1) * w.abs().amax(1)[row]).sum()) * 3 * scale
        assert abs(float(grad[k]) - want) <= 64 * 2.0 ** -24 * mag + 2.0 ** -24 * abs(want), (k, float(grad[k]), want)


CASES = [
    # T, V, D, types, scale, start, rows of the shard
    (1, 50, 256, ["Q8_0"], 1.0, 0, 50),
    (7, 300, 512, ALL, 1.0, 0, 300),
    (300, 97, 1000, ["Q4_K", "IQ4_XS", "Q8_0"], 31.5, 0, 97),
    (1025, 800, 264, ["Q6_K", "Q3_K"], 1.0, 200, 300),
    (2500, 700, 1280, ALL[:6], 0.25, 350, 350),
    (9000, 1500, 256, ["Q2_K", "Q5_K"], 1.0, 0, 1500),
    (70, 40, 5120, ["Q3_K", "Q6_K", "Q2_K"], 1.0, 0, 40),
    (33, 60, 13, ["Q4_K", "Q8_0"], 2.0, 10, 17),
]


@pytest.mark.parametrize("T,V,D,types,scale,start,rows", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
def test_lookup_and_gradient_against_64_bits(cuda, T, V, D, types, scale, start, rows, dtype):
    from voodoo_quant import _C
    from voodoo_quant.layers import gated_embedding

    _, _, blocks, dec, p = _table(V, D, types, T + D, cuda)
    P = (D + 255) // 256 * 256
    dec = [d[start:start + rows] for d in dec]
    shard = [b.view(V, -1)[start:start + rows].reshape(-1).contiguous() for b in blocks]
    ids = _ids(T, V, T)
    probs = p.to(cuda).requires_grad_(True)
    ids_d = ids.to(cuda).to(torch.int32 if T % 2 else torch.int64)
    out = gated_embedding(ids_d, probs, types, shard, rows, D, scale=scale, vocab_start=start, dtype=dtype)
    assert out.shape == (T, D) and out.dtype == dtype
    _check_lookup(out.detach(), ids, dec, p, scale, start, rows)
    with torch.no_grad():  # without a plan of the tokens
        assert torch.equal(out, gated_embedding(ids_d, probs, types, shard, rows, D, scale=scale, vocab_start=start,
                                                dtype=dtype))
    if scale == 1.0:
        here = (ids >= start) & (ids < start + rows)
        sub = [b.view(rows, -1)[(ids[here] - start).to(cuda)].reshape(-1).contiguous() for b in shard]
        same = _C.mix(types, sub, p.to(cuda), int(here.sum()), P, D)[:, :D]
        assert torch.equal(out.detach()[here.to(cuda)], same.to(dtype))
    g = torch.Generator(device="cpu").manual_seed(T + 1)
    dy = torch.randn(T, D, generator=g).to(dtype)
    (grad,) = torch.autograd.grad(out, probs, dy.to(cuda))
    _check_grad(grad, dy, ids, dec, scale, start, rows)
    assert _C.device_error() == 0


@pytest.mark.parametrize("T,rows", [(1, 1), (5, 3), (1024, 511), (1025, 512), (4097, 70000), (16384, 151936), (20000, 200),
                                    (70001, 151936)])
def test_plan_is_a_stable_sort_in_pieces(cuda, T, rows):
    _check_plan(cuda, T, rows)


@pytest.mark.parametrize("T", [1, 1000, 1025, 4500])
@pytest.mark.parametrize("rows", [(1 << 27) - 1, 1 << 27, 1 << 30])
def test_plan_of_the_most_rows(cuda, T, rows):
    """The last sizes of three digits of nine bits, and four digits."""
    _check_plan(cuda, T, rows)


def _check_plan(cuda, T, rows):
    from voodoo_quant import _C

    g = torch.Generator(device="cpu").manual_seed(T)
    ids = torch.randint(-2, rows + 9, (T,), generator=g)
    start = 3
    local = ids - start
    keys = torch.where((local >= 0) & (local < rows), local, torch.full_like(local, rows))
    want, order = torch.sort(keys, stable=True)
    head = torch.ones(T, dtype=torch.bool)
    head[1:] = want[1:] != want[:-1]
    head |= torch.arange(T) % 1024 == 0
    begin = torch.where(head, torch.arange(T), torch.zeros(T, dtype=torch.long)).cummax(0).values
    at = ((torch.arange(T) - begin) % 8 == 0).nonzero()[:, 0]
    step = (4 * T + 255) // 256 * 64
    for dt in (torch.int64, torch.int32):
        plan = _C.embed_plan(ids.to(dt).to(cuda), rows, start).view(torch.int32).cpu().long()
        P = int(plan[0])
        second = 64 + step
        third = second + (4 * (T + 1) + 255) // 256 * 64
        assert P == at.numel() and plan[1] == T and plan[2] == rows
        assert torch.equal(plan[64:64 + T], order)
        assert torch.equal(plan[second:second + P], at) and plan[second + P] == T
        assert torch.equal(plan[third:third + P], want[at])


def test_one_token_for_all_and_one_shard_without_any(cuda):
    """Every position names the same row: its decode is shared and the sums of dy are long; a shard that no token falls
    into gives zeros."""
    from voodoo_quant import _C

    types = ["Q4_K", "Q8_0"]
    V, D, T = 30, 512, 5000
    _, _, blocks, dec, p = _table(V, D, types, 2, cuda)
    ids = torch.full((T,), 7)
    g = torch.Generator(device="cpu").manual_seed(1)
    dy = torch.randn(T, D, generator=g).to(torch.bfloat16)
    table = _C.EmbedTable(types, blocks, V, D, D)
    grad = _C.embed_gategrad(dy.to(cuda), table, _C.embed_plan(ids.to(cuda), V))
    _check_grad(grad, dy, ids, dec, 1.0, 0, V)
    plan = _C.embed_plan(ids.to(cuda), V, 100)
    none = _C.embed_gategrad(dy.to(cuda), table, plan)
    assert torch.equal(none, torch.zeros_like(none))
    for q in (plan, None):
        assert not _C.embed_mix(ids.to(cuda), table, p.to(cuda), vocab_start=100, plan=q).any()
    assert _C.device_error() == 0


def test_ids_outside_the_table(cuda):
    """Without a shard an id that is no row gives zeros, adds nothing and is reported; its neighbours are right."""
    from voodoo_quant import _C

    types = ["Q6_K", "Q8_0"]
    V, D = 20, 256
    _, _, blocks, dec, p = _table(V, D, types, 3, cuda)
    ids = torch.tensor([3, -1, 19, 20, 2 ** 40, -2 ** 62, 0])
    good = (ids >= 0) & (ids < V)
    assert _C.device_error() == 0
    table = _C.EmbedTable(types, blocks, V, D, D)
    plan = _C.embed_plan(ids.to(cuda), V)
    for q in (plan, None):
        out = _C.embed_mix(ids.to(cuda), table, p.to(cuda), plan=q)
        assert _C.device_error() == (4 << 16 | 30) and _C.device_error() == 0
        _check_lookup(out[good.to(cuda)], ids[good], dec, p, 1.0, 0, V)
        assert not out[~good.to(cuda)].any()
    dy = torch.ones(7, D, dtype=torch.bfloat16)
    dy[1] = float("nan")  # of an id that is not in the table
    grad = _C.embed_gategrad(dy.to(cuda), table, plan)
    _check_grad(grad, dy, ids, dec, 1.0, 0, V)


def test_a_plan_of_other_tokens_or_rows_is_reported(cuda):
    """Plans whose size alone does not tell them apart: nothing is read or written by them."""
    from voodoo_quant import _C

    types = ["Q5_K", "Q3_K"]
    V, D = 40, 256
    _, _, blocks, _, p = _table(V, D, types, 4, cuda)
    table = _C.EmbedTable(types, blocks, V, D, D)
    ids = torch.arange(20).to(cuda)
    dy = torch.ones(20, D, dtype=torch.bfloat16, device=cuda)
    assert _C.device_error() == 0
    for plan in (_C.embed_plan(torch.arange(25).to(cuda), V), _C.embed_plan(torch.arange(19).to(cuda), V),
                 _C.embed_plan(ids, V + 100)):
        _C.embed_mix(ids, table, p.to(cuda), plan=plan)
        assert _C.device_error() == (5 << 16 | 31)
        assert not _C.embed_gategrad(dy, table, plan).any()
        assert _C.device_error() == (5 << 16 | 31) and _C.device_error() == 0


def test_strided_gradients_and_multidimensional_ids(cuda):
    from voodoo_quant.layers import gated_embedding

    types = ["Q5_K", "IQ4_XS"]
    V, D = 90, 520
    _, _, blocks, dec, p = _table(V, D, types, 4, cuda)
    ids = _ids(60, V, 5).view(3, 4, 5)
    g = torch.Generator(device="cpu").manual_seed(6)
    wide = torch.randn(3, 4, 5, D + 3, generator=g)
    probs = p.to(cuda).requires_grad_(True)
    for dy in (wide[..., 1:D + 1], wide[..., :D].transpose(0, 2).contiguous().transpose(0, 2),
               wide[:1, :1, :1, :D].expand(3, 4, 5, D), wide[..., :1].expand(3, 4, 5, D)):
        out = gated_embedding(ids.to(cuda), probs, types, blocks, V, D, dtype=torch.float32)
        assert out.shape == (3, 4, 5, D)
        dev = wide.to(cuda).as_strided(dy.size(), dy.stride(), dy.storage_offset()) if dy.data_ptr() >= wide.data_ptr() \
            and dy.untyped_storage().data_ptr() == wide.untyped_storage().data_ptr() else dy.to(cuda)
        (grad,) = torch.autograd.grad(out, probs, dev)
        _check_grad(grad, dy.reshape(-1, D), ids.reshape(-1), dec, 1.0, 0, V)
    out = gated_embedding(torch.empty(0, 4, dtype=torch.long, device=cuda), probs, types, blocks, V, D)
    assert out.shape == (0, 4, D)
    (grad,) = torch.autograd.grad(out, probs, torch.empty_like(out))
    assert torch.equal(grad, torch.zeros_like(grad))


def test_unaligned_blocks(cuda):
    """Candidate blocks need 2-byte alignment only."""
    from voodoo_quant import _C

    V, D, T = 40, 512, 100
    for qt in ALL:
        _, _, blocks, dec, p = _table(V, D, [qt], 6, cuda)
        ids = _ids(T, V, 7)
        one = torch.ones(1, device=cuda)
        table = _C.EmbedTable([qt], blocks, V, D, D)
        want = _C.embed_mix(ids.to(cuda), table, one)
        plan = _C.embed_plan(ids.to(cuda), V)
        dy = torch.randn(T, D, generator=torch.Generator().manual_seed(5)).to(cuda)
        grad = _C.embed_gategrad(dy, table, plan)
        for off in (2, 6, 14):
            buf = torch.empty(blocks[0].numel() + 16, dtype=torch.uint8, device=cuda)
            b = buf[off:off + blocks[0].numel()]
            b.copy_(blocks[0].reshape(-1))
            table = _C.EmbedTable([qt], [b], V, D, D)
            assert torch.equal(_C.embed_mix(ids.to(cuda), table, one), want)
            assert torch.equal(_C.embed_mix(ids.to(cuda), table, one, plan=plan), want)
            assert torch.equal(_C.embed_gategrad(dy, table, plan), grad)


@pytest.mark.parametrize("T", [3000, 5000])  # a plan by one block, and by a cluster
def test_streams_graphs_and_repeats(cuda, T):
    """Two captured graphs, replayed one after the other and on two streams at once, give the eager calls' bits."""
    from voodoo_quant import _C

    types = ["Q3_K", "Q4_K", "Q8_0"]
    V, D = 500, 768
    _, _, blocks, dec, p = _table(V, D, types, 8, cuda)
    sets = [(_ids(T, V, s).to(cuda), torch.randn(T, D, generator=torch.Generator().manual_seed(s)).to(torch.bfloat16).to(cuda))
            for s in (1, 2)]
    pd = p.to(cuda)
    table = _C.EmbedTable(types, blocks, V, D, D)

    def call(ids, dy):
        plan = _C.embed_plan(ids, V)
        return (_C.embed_mix(ids, table, pd), _C.embed_mix(ids, table, pd, plan=plan), _C.embed_gategrad(dy, table, plan))

    want = [call(*s) for s in sets]
    again = [call(*s) for s in sets]
    assert all(torch.equal(a, b) for x, y in zip(want, again) for a, b in zip(x, y))
    assert all(torch.equal(x[0], x[1]) for x in want)  # the same rows with a plan and without
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(*s))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(outs, want) for a, b in zip(x, y))


def test_module_uses_the_fused_lookup(cuda):
    """MixedQuantEmbedding and Q8Embedding against their rows gathered and mixed one by one; a scaled embedding module
    keeps its factor when it is replaced."""
    import torch.nn as nn

    from voodoo_quant import _C
    from voodoo_quant.layers import replace_embedding_with_mixed_quant
    from voodoo_quant.training.q8_teacher import wrap_q8_teacher
    from voodoo_quant.training.synthetic import q8_quantizer, rtn_candidate_provider

    class Scaled(nn.Embedding):
        def __init__(self, *a, **kw):
            super().__init__(*a, **kw)
            self.embed_scale = torch.tensor(22.6)

    types = ["Q4_K", "Q8_0"]
    V, D = 64, 512
    m = nn.Module()
    m.emb = Scaled(V, D, device=cuda, dtype=torch.bfloat16)
    teacher = nn.Module()
    teacher.emb = Scaled(V, D, device=cuda, dtype=torch.bfloat16)
    teacher.emb.weight.data.copy_(m.emb.weight.data)
    weight = m.emb.weight.data.clone()
    replace_embedding_with_mixed_quant(m, types, candidate_provider=rtn_candidate_provider)
    wrap_q8_teacher(teacher, q8_quantizer)
    scale = float(torch.tensor(22.6).bfloat16())
    assert m.emb.scale == scale and teacher.emb.scale == scale
    ids = _ids(37, V, 9).to(cuda)
    out = m.emb(ids)
    out.float().sum().backward()
    assert m.emb.gates.grad.shape == (2,)
    dec = [_C.dequant(b, q, V, D).double().cpu() for q, b in zip(types, m.emb._candidate_blocks())]
    _check_lookup(out.detach(), ids.cpu(), dec, torch.tensor([0.5, 0.5]), scale, 0, V)
    q8 = _C.dequant(teacher.emb.qweight, "Q8_0", V, D).double().cpu()
    _check_lookup(teacher.emb(ids), ids.cpu(), [q8], torch.ones(1), scale, 0, V)
    assert (q8 - weight.double().cpu()).abs().max() < 0.02 * float(weight.abs().max())


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.float16])
def test_module_returns_its_sources_type(cuda, dtype):
    """The values are the mixture's in bfloat16, whatever the source's type."""
    import torch.nn as nn

    from voodoo_quant import _C
    from voodoo_quant.layers import replace_embedding_with_mixed_quant
    from voodoo_quant.training.synthetic import rtn_candidate_provider

    types = ["Q4_K", "Q8_0"]
    V, D = 40, 256
    m = nn.Module()
    m.emb = nn.Embedding(V, D, device=cuda, dtype=dtype)
    replace_embedding_with_mixed_quant(m, types, candidate_provider=rtn_candidate_provider)
    ids = _ids(21, V, 3).to(cuda)
    out = m.emb(ids)
    assert out.dtype == dtype
    dec = [_C.dequant(b, q, V, D).double().cpu() for q, b in zip(types, m.emb._candidate_blocks())]
    _check_lookup(out.detach(), ids.cpu(), dec, torch.tensor([0.5, 0.5]), 1.0, 0, V)
    out.sum().backward()
    assert m.emb.gates.grad.shape == (2,) and m.emb.gates.grad.any()


def test_offsets_past_32_bits(cuda):
    """A table of more than 2^32 bytes and rows of more than 2^31 values: the last ones are read and written as those of
    a small call are."""
    from voodoo_quant import _C

    D, rows, T = 16384, 260_000, 140_000
    _, _, small, _, _ = _table(3, D, ["Q8_0"], 12, cuda)
    bytes_row = small[0].numel() // 3
    big = torch.zeros(rows * bytes_row, dtype=torch.uint8, device=cuda)
    assert big.numel() > 2 ** 32 and T * D > 2 ** 31
    big[-3 * bytes_row:] = small[0].reshape(-1)
    one = torch.ones(1, device=cuda)
    table, few = _C.EmbedTable(["Q8_0"], [big], rows, D, D), _C.EmbedTable(["Q8_0"], small, 3, D, D)
    ids = torch.zeros(T, dtype=torch.int64, device=cuda)
    last = torch.tensor([2, 0, 1, 2], device=cuda)
    ids[-4:] = last + (rows - 3)
    want = _C.embed_mix(last, few, one)
    plan = _C.embed_plan(ids, rows)
    for q in (plan, None):
        out = _C.embed_mix(ids, table, one, plan=q)
        assert torch.equal(out[-4:], want) and not out[:-4].any()
        del out
    dy = torch.zeros(T, D, dtype=torch.bfloat16, device=cuda)
    dy[-4:] = torch.randn(4, D, generator=torch.Generator().manual_seed(2)).to(cuda)
    exact = float((dy[-4:].double() * want.double()).sum())
    mag = float((dy[-4:].double() * want.double()).abs().sum())
    grad = float(_C.embed_gategrad(dy, table, plan))
    # the rows in bf16 against the decoded ones: 2^-8 of each product; the sums as elsewhere
    assert abs(grad - exact) <= (2.0 ** -8 + 64 * 2.0 ** -24) * mag
    assert _C.device_error() == 0


def test_gradient_has_no_graph_of_its_own(cuda):
    """The gradient taken with create_graph, and a second time, is the first one; a second derivative is refused."""
    from voodoo_quant.layers import gated_embedding

    types = ["Q4_K", "Q6_K"]
    V, D = 30, 512
    _, _, blocks, _, p = _table(V, D, types, 14, cuda)
    for probs in (p.to(cuda).requires_grad_(), p.to(cuda).double().view(2, 1).requires_grad_()):
        out = gated_embedding(_ids(50, V, 2).to(cuda), probs, types, blocks, V, D)
        dy = torch.randn(50, D, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).bfloat16()
        (first,) = torch.autograd.grad(out, probs, dy, retain_graph=True)
        assert first.shape == probs.shape and first.dtype == probs.dtype
        dy.requires_grad_()
        (again,) = torch.autograd.grad(out, probs, dy, create_graph=True)
        assert torch.equal(first, again)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            again.sum().backward()


def test_a_plan_of_another_size_is_refused(cuda):
    from voodoo_quant import _C

    types = ["Q8_0"]
    _, _, blocks, _, p = _table(9, 256, types, 1, cuda)
    table = _C.EmbedTable(types, blocks, 9, 256, 256)
    plan = _C.embed_plan(torch.zeros(100, dtype=torch.int64, device=cuda), 9)
    with pytest.raises(ValueError, match="plan of"):
        _C.embed_gategrad(torch.zeros(500, 256, dtype=torch.bfloat16, device=cuda), table, plan)
    with pytest.raises(ValueError, match="plan of"):
        _C.embed_mix(torch.zeros(10, dtype=torch.int64, device=cuda), table, torch.ones(1, device=cuda), plan=plan)
