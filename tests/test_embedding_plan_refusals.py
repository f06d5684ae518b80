"""What the Python calls of the gated embedding refuse of a plan and a factor, before anything is launched;
the library is replaced, no GPU needed."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch


class _Never:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


@pytest.fixture
def table(monkeypatch):
    """A table that takes CPU tensors for tensors of its device, and keeps those that it was asked about."""
    from voodoo_quant import _C

    t = _C.EmbedTable.__new__(_C.EmbedTable)
    t.blocks, t.rows, t.padded_cols, t.cols, t.device, t.K, t.types, t.ptrs = (), 4, 256, 256, -1, 1, None, None
    seen = []
    monkeypatch.setattr(_C.EmbedTable, "check", lambda self, *ts: seen.extend(ts))
    monkeypatch.setattr(_C, "_lib", _Never())
    return t, seen


BAD = [torch.zeros(1024, dtype=torch.int32), torch.zeros(2048, dtype=torch.uint8)[::2], torch.zeros(1024).bool(),
       torch.zeros(1, dtype=torch.uint8).expand(1024)]


@pytest.mark.parametrize("plan", BAD)
def test_lookup_refuses_what_is_no_plan(table, plan):
    from voodoo_quant import _C

    with pytest.raises(ValueError, match="plan"):
        _C.embed_mix(torch.zeros(3, dtype=torch.long), table[0], torch.ones(1), plan=plan)


@pytest.mark.parametrize("plan", BAD)
def test_gradient_refuses_what_is_no_plan(table, plan):
    from voodoo_quant import _C

    with pytest.raises(ValueError, match="plan"):
        _C.embed_gategrad(torch.zeros(3, 256), table[0], plan)


def test_the_plans_device_is_checked(table):
    """A plan on the host or another GPU is found out before its address is passed on."""
    from voodoo_quant import _C

    t, seen = table
    plan = torch.zeros(1024, dtype=torch.uint8)
    for call in (lambda: _C.embed_mix(torch.zeros(3, dtype=torch.long), t, torch.ones(1), plan=plan),
                 lambda: _C.embed_gategrad(torch.zeros(3, 256), t, plan)):
        seen.clear()
        with pytest.raises(AssertionError, match="was reached"):
            call()
        assert any(s is plan for s in seen)


@pytest.mark.parametrize("scale", [math.inf, -math.inf, math.nan, 1e39])
def test_a_scale_that_is_not_finite(scale):
    """Rows of other shards' tokens and of no token are zeros, which such a factor would turn into NaN."""
    from voodoo_quant import _C

    lib = _C.load_library()
    types, blocks = (ctypes.c_int * 1)(8), (ctypes.c_void_p * 1)(1 << 20)
    one = 1 << 20  # stands for an aligned address that the checks never read
    need = lib.vq_embed_gategrad_workspace_bytes(1)
    for rc in (lib.vq_embed_mix(1, types, blocks, one, one, 0, 4, None, 0, 0, 10, 256, 256, scale, 1, one, 256, None),
               lib.vq_embed_gategrad(1, types, blocks, one, lib.vq_embed_plan_bytes(4), 4, 10, 256, 256, scale, one, 256, 1,
                                     one, need - 1, one, None)):
        assert rc == -1 and "scale" in lib.vq_last_error().decode()
