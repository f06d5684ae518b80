"""A lookup that meets the plan of other tokens or rows leaves zeros, not what the memory held before."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [256, 251, 13])
@pytest.mark.parametrize("T", [20, 3000])
def test_rows_of_a_bad_plan_are_zeros(cuda, T, cols):
    from voodoo_quant import _C

    V = 40
    g = torch.Generator(device=cuda).manual_seed(1)
    blocks = torch.randint(1, 100, (V * 272,), generator=g, device=cuda, dtype=torch.uint8)
    table = _C.EmbedTable(["Q8_0"], [blocks], V, 256, cols)
    ids = torch.arange(T, device=cuda) % V
    one = torch.ones(1, device=cuda)
    assert _C.device_error() == 0
    bad = [_C.embed_plan(ids, V + 100)]
    if T == 20:  # as many bytes as a plan of 20
        bad.append(_C.embed_plan(torch.arange(25, device=cuda), V))
    for plan in bad:
        dirty = torch.ones(T, cols, dtype=torch.bfloat16, device=cuda)
        at = dirty.data_ptr()
        del dirty
        out = _C.embed_mix(ids, table, one, plan=plan)
        assert out.data_ptr() == at  # the memory that held ones
        assert not out.any()
        assert _C.device_error() == (5 << 16 | 31)
    good = _C.embed_mix(ids, table, one, plan=_C.embed_plan(ids, V))
    assert torch.equal(good, _C.embed_mix(ids, table, one)) and good.any()
    assert _C.device_error() == 0
