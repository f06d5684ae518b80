"""What the head-norm, gated-embedding and clipping entry points refuse, by the C ABI's checks (which come before any
CUDA call) and the Python layer's; no GPU needed."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

ONE = 1 << 20  # stands for an aligned device address that the checks never read


def _lib():
    from voodoo_quant import _C

    return _C.load_library()


def _refused(rc, text):
    lib = _lib()
    assert rc == -1, rc
    assert text in lib.vq_last_error().decode(), lib.vq_last_error()


def _qk(**kw):
    a = dict(q=ONE, qs=(1024, 512, 128), Hq=4, k=ONE, ks=(1024, 256, 128), Hk=2, wq=ONE, wk=ONE, wf=0, cos=ONE, sin=ONE,
             cs=(0, 128), cf=0, B=1, S=2, D=128, R=128, eps=1e-6, off=0.0, dtype=1, qo=ONE, ko=ONE)
    a.update(kw)
    i3 = ctypes.c_int64 * 3
    i2 = ctypes.c_int64 * 2
    return _lib().vq_qk_norm_rope_fwd(a["q"], i3(*a["qs"]), a["Hq"], a["k"], i3(*a["ks"]), a["Hk"], a["wq"], a["wk"],
                                      a["wf"], a["cos"], a["sin"], i2(*a["cs"]), a["cf"], a["B"], a["S"], a["D"], a["R"],
                                      a["eps"], a["off"], a["dtype"], a["qo"], a["ko"], None)


@pytest.mark.parametrize("kw,text", [
    (dict(D=120), "head dimension"), (dict(D=0), "head dimension"), (dict(D=528), "head dimension"),
    (dict(R=8), "rotary dimension"), (dict(R=144), "rotary dimension"), (dict(R=0), "rotary dimension"),
    (dict(B=-1), "negative shape"), (dict(Hq=-1), "negative shape"), (dict(dtype=3), "dtype"),
    (dict(q=ONE + 2), "q: null pointer or not 16-byte aligned"), (dict(k=None), "k: null pointer"),
    (dict(qs=(1024, 516, 128)), "q: strides"), (dict(ks=(1024, 256, -128)), "k: strides"),
    (dict(wq=None), "weights"), (dict(wk=ONE + 4), "weights"), (dict(cos=None), "cos/sin"),
    (dict(cs=(0, 4)), "cos/sin strides"), (dict(qo=None), "outputs"), (dict(S=1 << 33), "too large"),
    (dict(B=1 << 20, S=1 << 20), "too large"),
])
def test_qk_norm_rope_refuses(kw, text):
    _refused(_qk(**kw), text)


def test_qk_norm_rope_of_nothing_is_fine():
    assert _qk(B=0) == 0 and _qk(S=0) == 0 and _qk(Hq=0, Hk=0) == 0


def test_qk_norm_rope_backward_needs_its_workspace():
    lib = _lib()
    i3, i2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2
    st, cs = i3(1024, 512, 128), i2(0, 128)
    need = lib.vq_qk_norm_rope_workspace_bytes(128)
    assert need > 0 and lib.vq_qk_norm_rope_workspace_bytes(0) == 0

    def call(ws, nbytes):
        return lib.vq_qk_norm_rope_bwd(ONE, st, ONE, st, ONE, st, 4, ONE, st, 4, ONE, ONE, 0, ONE, ONE, cs, 0, 1, 2, 128,
                                       128, 1e-6, 0.0, 1, ONE, ONE, ONE, ONE, ws, nbytes, None)

    _refused(call(None, need), "workspace")
    _refused(call(ONE, need - 1), "workspace")
    _refused(call(ONE + 4, need), "workspace")


def _table(types, ptrs):
    n = len(types)
    return n, (ctypes.c_int * n)(*types), (ctypes.c_void_p * n)(*ptrs)


def test_gated_embedding_refuses():
    lib = _lib()

    def mix(types=(8,), ptrs=(ONE,), probs=ONE, ids=ONE, i32=0, T=4, start=0, rows=10, padded=256, cols=256, out=ONE,
            ldo=256, plan=None, nplan=0):
        K, t, p = _table(types, ptrs)
        return lib.vq_embed_mix(K, t, p, probs, ids, i32, T, plan, nplan, start, rows, padded, cols, 1.0, 1, out, ldo, None)

    for kw, text in ((dict(padded=250), "multiple of 256"), (dict(cols=300, ldo=300), "multiple of 256"),
                     (dict(T=-1), "negative"), (dict(rows=-1), "negative"), (dict(start=-1), "negative"),
                     (dict(ldo=255), "leading dimension"), (dict(ptrs=(None,)), "null block pointer"),
                     (dict(ptrs=(ONE + 1,)), "2-byte aligned"), (dict(types=(8,) * 9, ptrs=(ONE,) * 9), "number of candidates"),
                     (dict(probs=None), "null pointer"), (dict(ids=ONE + 4), "misaligned"), (dict(T=1 << 31), "too large"),
                     (dict(ids=None), "null token ids"), (dict(plan=ONE, nplan=100), "plan of"),
                     (dict(plan=ONE + 8, nplan=1 << 20), "plan of")):
        _refused(mix(**kw), text)
    K, t, p = _table((99,), (ONE,))
    assert lib.vq_embed_mix(K, t, p, ONE, ONE, 0, 4, None, 0, 0, 10, 256, 256, 1.0, 1, ONE, 256, None) == -3
    assert mix(T=0) == 0 and mix(cols=0, ldo=0) == 0

    def grad(T=4, cols=256, lddy=256, code=1, dy=ONE, ws=ONE, nbytes=None, out=ONE, plan=ONE, nplan=None):
        K, t, p = _table((8,), (ONE,))
        need = lib.vq_embed_gategrad_workspace_bytes(1) if nbytes is None else nbytes
        pb = lib.vq_embed_plan_bytes(T) if nplan is None else nplan
        return lib.vq_embed_gategrad(K, t, p, plan, pb, T, 10, 256, cols, 1.0, dy, lddy, code, ws, need, out, None)

    for kw, text in ((dict(code=5), "dtype"), (dict(lddy=100), "leading dimension"), (dict(dy=None), "null pointer"),
                     (dict(ws=None), "workspace"), (dict(nbytes=16), "workspace"), (dict(ws=ONE + 8), "workspace"),
                     (dict(out=None), "null pointer"), (dict(plan=None), "plan of"), (dict(nplan=256), "plan of")):
        _refused(grad(**kw), text)
    assert lib.vq_embed_gategrad_workspace_bytes(9) == 0 and lib.vq_embed_gategrad_workspace_bytes(0) == 0
    assert lib.vq_embed_plan_bytes(-1) == 0 and lib.vq_embed_plan_bytes(1 << 31) == 0
    big = 1 << 20
    _refused(lib.vq_embed_plan(None, 0, 4, 0, 10, ONE, big, None), "null token ids")
    _refused(lib.vq_embed_plan(ONE, 0, -4, 0, 10, ONE, big, None), "negative")
    _refused(lib.vq_embed_plan(ONE, 0, 4, 0, 1 << 31, ONE, big, None), "too large")
    _refused(lib.vq_embed_plan(ONE, 0, 4, 0, 10, ONE, 100, None), "plan of")
    assert lib.vq_embed_plan(None, 0, 0, 0, 10, None, 0, None) == 0


def test_clip_refuses():
    lib = _lib()

    def clip(ptrs, nbytes_of, codes, max_norm=1.0, ws=ONE, nbytes=1 << 20, norm=ONE):
        n = len(ptrs)
        return lib.vq_clip_grad_norm(n, (ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*nbytes_of),
                                     (ctypes.c_int * n)(*codes), max_norm, 0, ws, nbytes, norm, None)

    for args, kw, text in (
            (([ONE], [4], [0]), dict(max_norm=-1.0), "max_norm"), (([ONE], [4], [0]), dict(max_norm=math.nan), "max_norm"),
            (([ONE], [-4], [0]), {}, "bad size"), (([ONE], [3], [1]), {}, "bad size"), (([ONE], [4], [3]), {}, "dtype"), (([None], [4], [0]), {}, "null"),
            (([ONE + 2], [4], [0]), {}, "misaligned"), (([ONE + 1], [4], [1]), {}, "misaligned"),
            (([ONE, ONE], [4, 4], [0, 0]), {}, "share memory"), (([ONE + 16, ONE], [8, 18], [1, 1]), {}, "share memory"),
            (([ONE], [4], [0]), dict(nbytes=8), "workspace"), (([ONE], [4], [0]), dict(ws=None), "workspace"),
            (([ONE], [4], [0]), dict(norm=None), "null")):
        _refused(clip(*args, **kw), text)


def test_python_checks_come_first():
    """CPU tensors have no fallback; bounds and types are refused before anything is launched."""
    from voodoo_quant import _C
    from voodoo_quant.fused_blocks import qk_norm_rope
    from voodoo_quant.layers import gated_embedding
    from voodoo_quant.training.grad_clip import clip_grad_norm_, grad_norm

    q = torch.zeros(1, 2, 4, 64)
    w, c = torch.ones(64), torch.ones(1, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        qk_norm_rope(q, q, w, w, c, c)
    with pytest.raises(ValueError, match="constants"):
        qk_norm_rope(q, q, w, w, c.clone().requires_grad_(True), c)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        gated_embedding(torch.zeros(3, dtype=torch.long), torch.ones(1), ["Q8_0"], [torch.zeros(34 * 8, dtype=torch.uint8)],
                        1, 256)
    with pytest.raises(ValueError, match="rows, got"):
        gated_embedding(torch.zeros(3, dtype=torch.long), torch.ones(1), ["Q8_0"], [], 1, 256, dtype=torch.int8)
    with pytest.raises(ValueError, match="negative"):
        gated_embedding(torch.zeros(3, dtype=torch.long), torch.ones(1), ["Q8_0"], [], 1, 256, vocab_start=-5)
    p = torch.zeros(4, requires_grad=True)
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        clip_grad_norm_([p], 1.0)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([p], bad)
    with pytest.raises(ValueError, match="norm_type"):
        clip_grad_norm_([p], 1.0, norm_type=1.0)
    with pytest.raises(ValueError, match="no tensors"):
        _C.clip_grad_norm([])
    assert float(grad_norm([])) == 0.0 and float(clip_grad_norm_([], 1.0)) == 0.0
    assert float(p.grad.sum()) == 4.0


def test_scaled_embeddings_keep_their_factor_on_cpu_paths():
    """The rows a vocabulary shard or a stand-in lookup returns carry the module's factor."""
    from voodoo_quant.layers import embed_scale

    e = torch.nn.Embedding(4, 8, dtype=torch.bfloat16)
    assert embed_scale(e) == 1.0
    e.embed_scale = 31.62
    assert embed_scale(e) == float(torch.tensor(31.62).bfloat16())


def test_head_norm_models_build_and_fuse_on_cpu():
    """The synthetic decoder with head norms is built from Qwen3 blocks; patched blocks run their own forward off the
    fused path."""
    pytest.importorskip("transformers")
    from voodoo_quant.fused_blocks import fuse_llama_blocks, fuse_qwen3_blocks
    from voodoo_quant.training import synthetic as S

    shape = S.SHAPES["tiny-qk"]
    a, b = (S.build_llama(shape, "cpu", seed=2) for _ in range(2))
    assert fuse_llama_blocks(b) == 0
    assert fuse_qwen3_blocks(b, causal_batches=True) == 2 * 7 + 1 + 1
    x = torch.randint(0, shape.vocab, (1, 16))
    with torch.no_grad():
        assert torch.equal(a(input_ids=x, use_cache=False).logits, b(input_ids=x, use_cache=False).logits)


def _windowed_decoder(window):
    from transformers import Qwen3Config, Qwen3ForCausalLM

    cfg = Qwen3Config(vocab_size=64, hidden_size=32, intermediate_size=48, num_hidden_layers=2, num_attention_heads=2,
                      num_key_value_heads=1, head_dim=16, use_sliding_window=True, sliding_window=window,
                      max_window_layers=1, max_position_embeddings=64)
    cfg._attn_implementation = "sdpa"
    assert ("sliding_attention" in cfg.layer_types) == (window is not None)
    torch.manual_seed(3)
    return Qwen3ForCausalLM(cfg)


def test_attention_windows_are_not_dropped(monkeypatch):
    """The paths that pass no mask to the layers refuse a window shorter than the batch, or are not taken."""
    pytest.importorskip("transformers")
    from types import SimpleNamespace

    from voodoo_quant import fused_blocks, parallel
    from voodoo_quant.training.trainer import GatedDistillTrainer, StepArgs

    model = _windowed_decoder(8)
    assert fused_blocks.windowed(model.model.layers, 9) and not fused_blocks.windowed(model.model.layers, 8)
    assert fused_blocks.windowed(model.model.layers)
    fused_blocks.use_sequence_parallel(model)
    x = torch.randint(0, 64, (1, 12))
    with torch.no_grad():
        want = _windowed_decoder(8)(input_ids=x, use_cache=False).logits
        assert torch.equal(model(input_ids=x, use_cache=False).logits, want)  # off: the model's own forward
        monkeypatch.setattr(parallel, "sp_enabled", lambda: True)
        with pytest.raises(ValueError, match="no window"):
            model.model(input_ids=x)
    monkeypatch.setattr(parallel, "sp_enabled", lambda: False)
    plain = _windowed_decoder(None)

    def joint(student, teacher):
        t = SimpleNamespace(args=StepArgs(joint_teacher=True), tp=True, _tsplit=(0, 0, 0, 1), student=student,
                            teacher=teacher)
        return GatedDistillTrainer._joint_ok(t)

    assert joint(plain, plain)
    assert not joint(model, plain) and not joint(plain, model)
