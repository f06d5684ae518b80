"""A decoder with head norms (Qwen3 blocks) on the fused path: the patched
model against the unpatched one, the calls that keep their own attention, and
a whole distillation step -- gated embedding, head norms with rotation, gate
gradients, clipping, update -- against a float32 torch restatement.

Tolerances.  Model against model: normed heads give attention scores of order
one, which carry every rounding of a query or key on, so two bf16 models are
not compared with one another but each with the same model in float32: the
fused blocks round to bf16 at a subset of the stock blocks' places (a head once
instead of after its norm, its weight, each product of the rotation and their
sum), each rounding an independent error of the same size, so their error is
the smaller but for the sampling of the two norms -- below a tenth over the
tens of thousands of values of logits, embedding and projection, below a half
over the 128 of a head's weights.  The step: as the Llama step
(test_gpu_trainer.py).
"""

from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

from conftest import cosine, rel_err

pytestmark = pytest.mark.gpu


def _rel(a, b):
    return rel_err(a.detach().float().cpu().numpy(), b.detach().float().cpu().numpy())


def _pair(cuda, fuse=True, causal=False, **kw):
    from voodoo_quant.fused_blocks import fuse_qwen3_blocks
    from voodoo_quant.training import synthetic as S

    shape = S.ModelShape(2, 512, 4, 2, 1536, 2048, False, head_dim=128, batch=2, seq=64, qk_norm=True)
    models = []
    for _ in range(2):
        m = S.build_llama(shape, cuda, seed=4)
        g = torch.Generator(device="cpu").manual_seed(1)
        with torch.no_grad():
            for layer in m.model.layers:
                for n in (layer.self_attn.q_norm, layer.self_attn.k_norm):
                    n.weight.copy_(1 + 0.3 * torch.randn(128, generator=g))
        models.append(m)
    # per layer: two norms, two head norms, attention, MLP and the decoder layer; plus the final norm
    if fuse:
        assert fuse_qwen3_blocks(models[1], causal) == 2 * 7 + 1 + int(causal)
        assert fuse_qwen3_blocks(models[1], causal) == 0
    x, _ = S.random_tokens(shape, cuda, seed=5)
    return models[0], models[1], x, shape


@pytest.mark.parametrize("causal", [False, True])
def test_fused_blocks_match_unpatched_model(cuda, causal):
    from voodoo_quant import _C

    ref, fused, x, shape = _pair(cuda, causal=causal)
    calls = []
    inner = _C.qk_norm_rope_fwd
    _C.qk_norm_rope_fwd = lambda *a, **k: (calls.append(1), inner(*a, **k))[1]
    gy = torch.randn(shape.batch, shape.seq, shape.vocab, generator=torch.Generator(device=cuda).manual_seed(6), device=cuda)
    try:
        out = []
        for m in (ref, fused):
            for p in m.parameters():
                p.requires_grad = True
            logits = m(input_ids=x, use_cache=False).logits
            logits.backward(gy.to(logits.dtype))
            a = m.model.layers[0].self_attn
            out.append([t.detach().clone() for t in (logits, m.model.embed_tokens.weight.grad, a.q_norm.weight.grad,
                                                     a.k_norm.weight.grad, a.q_proj.weight.grad)])
    finally:
        _C.qk_norm_rope_fwd = inner
    assert len(calls) == shape.layers
    exact = ref.float()
    exact.zero_grad(set_to_none=True)
    logits = exact(input_ids=x, use_cache=False).logits
    logits.backward(gy.to(torch.bfloat16).float())
    a = exact.model.layers[0].self_attn
    want = (logits.detach(), exact.model.embed_tokens.weight.grad, a.q_norm.weight.grad, a.k_norm.weight.grad,
            a.q_proj.weight.grad)
    for stock, fused_, w in zip(*out, want):
        assert _rel(fused_, w) <= _rel(stock, w) * (1.1 if w.numel() > 128 else 1.5)
        assert cosine(fused_.double().flatten().cpu().numpy(), w.double().flatten().cpu().numpy()) > 0.999


def test_masks_caches_windows_and_dropout_keep_their_own_attention(cuda):
    ref, fused, x, shape = _pair(cuda)
    mask = torch.ones_like(x)
    mask[0, :11] = 0

    def near(a, b, want):  # each against the float32 model
        assert _rel(b, want) <= 1.1 * _rel(a, want)

    def cached(m):  # a prompt, then a single token with its cache
        p = m(input_ids=x[:, :40], use_cache=True)
        return torch.cat([p.logits, m(input_ids=x[:, 40:41], past_key_values=p.past_key_values, use_cache=True).logits], 1)

    with torch.no_grad():
        exact = copy.deepcopy(ref).float()
        a, b, w = (m(input_ids=x, attention_mask=mask, use_cache=False).logits[mask.bool()] for m in (ref, fused, exact))
        near(a, b, w)
        near(*(cached(m) for m in (ref, fused, exact)))
    # a window shorter than the batch, with the causal batches' shortcuts on
    from transformers import Qwen3Config, Qwen3ForCausalLM

    from voodoo_quant.fused_blocks import fuse_qwen3_blocks

    cfg = Qwen3Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64, use_sliding_window=True, sliding_window=16, max_window_layers=1,
                      max_position_embeddings=256)
    cfg._attn_implementation = "sdpa"
    assert "sliding_attention" in cfg.layer_types
    torch.manual_seed(0)
    a = Qwen3ForCausalLM(cfg).to(cuda, torch.bfloat16)
    b = Qwen3ForCausalLM(cfg).to(cuda, torch.bfloat16)
    b.load_state_dict(a.state_dict())
    fuse_qwen3_blocks(b, causal_batches=True)
    y = torch.randint(0, 512, (2, 100), device=cuda)
    with torch.no_grad():
        la, lb = (m(input_ids=y, use_cache=False).logits for m in (a, b))
        near(la, lb, a.float()(input_ids=y, use_cache=False).logits)


def test_distill_step_matches_torch_restatement(cuda):
    from test_gpu_trainer import _set, _TorchGated

    from voodoo_quant import _C
    from voodoo_quant.layers import MixedQuantEmbedding
    from voodoo_quant.training import synthetic as S
    from voodoo_quant.training.trainer import StepArgs, build_distill

    args = StepArgs()
    trainer, shape = build_distill("tiny-qk", cuda, seed=3, args=args)
    assert type(trainer.student).__name__ == "Qwen3ForCausalLM"
    g = torch.Generator(device="cpu").manual_seed(5)
    with torch.no_grad():
        for layer in trainer.replaced.values():
            layer.gates.copy_(torch.randn(layer.num_candidates, generator=g).to(cuda))
    trainer.step_idx = 7
    x, y = S.random_tokens(shape, cuda, seed=11)
    x[:, 40:80] = x[0, 3]  # a token that fills a good part of the batch
    with torch.no_grad():
        t_logits = trainer.teacher(input_ids=x).logits.float()
    ref = S.build_llama(shape, cuda, seed=3).float()
    mods = {}
    for name, layer in trainer.replaced.items():
        mods[name] = _TorchGated(layer, isinstance(layer, MixedQuantEmbedding))
        _set(ref, name, mods[name])
    out = trainer.forward_backward(x, y)
    for p in ref.parameters():
        p.requires_grad = False
    for m in mods.values():
        m.tau = max(out["tau"], 1e-6)
        m.gates.requires_grad = True
    logits = ref(input_ids=x).logits.float()
    V = logits.shape[-1]
    lm = F.cross_entropy(logits.view(-1, V), y.view(-1))
    kl = F.kl_div(F.log_softmax(logits, -1).view(-1, V), F.softmax(t_logits, -1).view(-1, V), reduction="none").sum(-1).mean()
    cur = sum(m.eff_bytes() for m in mods.values()) + trainer.non_targeted_bytes
    size = torch.relu(torch.abs(cur / trainer.target_bytes - 1.0) - args.size_tolerance) ** 2
    loss = lm + args.distill_weight * kl + args.size_weight * size
    loss.backward()
    assert abs(out["loss"].item() - loss.item()) <= 1e-2 * abs(loss.item())
    a = torch.cat([trainer.replaced[n].gates.grad.double() for n in mods])
    b = torch.cat([mods[n].gates.grad.double() for n in mods])
    assert (a - b).norm() < 3e-2 * b.norm() and torch.dot(a, b) > 0.999 * a.norm() * b.norm()
    for n in mods:
        u, v = trainer.replaced[n].gates.grad.double(), mods[n].gates.grad.double()
        assert float(torch.dot(u, v) / (u.norm() * v.norm())) >= 0.999, n
    # the update clips these gradients to norm one
    before = {n: l.gates.detach().clone() for n, l in trainer.replaced.items()}
    trainer.apply_update()
    total = torch.cat([p.grad.double() for p in trainer.trainable]).norm()
    assert abs(float(total) - min(1.0, float(a.norm()))) < 1e-5
    assert all(not torch.equal(before[n], l.gates) for n, l in trainer.replaced.items())
    assert _C.device_error() == 0


def test_captured_step_replays(cuda):
    """The step as one CUDA graph (embedding plan and lookup, head norms, their backward inside it): replays on two
    batches give the eager losses and, within the run-to-run order of the attention's own backward, gradients."""
    from voodoo_quant.layers import set_static_shapes
    from voodoo_quant.training import synthetic as S
    from voodoo_quant.training.trainer import StepArgs, build_distill

    try:
        trainer, shape = build_distill("tiny-qk", cuda, seed=3,
                                       args=StepArgs(max_steps=9, ce_reduction="tokens", static_shapes=True))
        batches = [S.random_tokens(shape, cuda, seed=s) for s in (1, 2)]
        want = []
        for x, y in batches:
            out = trainer.forward_backward(x, y)
            want.append((float(out["loss"]), [p.grad.clone() for p in trainer.trainable]))
        del out
        trainer.capture(*batches[0])
        for (x, y), (loss, grads) in zip(batches[::-1], want[::-1]):
            trainer._gx.copy_(x), trainer._gy.copy_(y)
            trainer._graph.replay()
            torch.cuda.synchronize()
            assert abs(float(trainer._gout["loss"]) - loss) <= 1e-5 * abs(loss)
            got = torch.cat([p.grad for p in trainer.trainable]).double()
            ref = torch.cat(grads).double()
            assert (got - ref).norm() <= 1e-2 * ref.norm()
        out = trainer.replay_step(*batches[0])
        assert torch.isfinite(out["loss"])
        trainer.release_graph()
    finally:
        set_static_shapes(False)
