"""A distillation step on token ids that name no row of the embedding does not go on in silence."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _trainer(cuda, **kw):
    from voodoo_quant.training.synthetic import random_tokens
    from voodoo_quant.training.trainer import StepArgs, build_distill

    trainer, shape = build_distill("tiny", cuda, seed=0, args=StepArgs(max_steps=9, **kw))
    x, y = random_tokens(shape, cuda, seed=1)
    bad = x.clone()
    bad[0, 5] = shape.vocab
    return trainer, x, y, bad


def test_a_wrong_token_stops_the_training(cuda):
    """At the next step's update, or before the assignments are read; steps that follow on right tokens run."""
    trainer, x, y, bad = _trainer(cuda)
    trainer.step(x, y)
    trainer.step(x, y)
    trainer.check_device()
    trainer.step(bad, y)
    with pytest.raises(RuntimeError, match="token id outside the embedding table"):
        trainer.step(x, y)
    trainer.step(x, y)
    assert trainer.assignments()
    bad[0, 5] = -1
    trainer.step(bad, y)
    with pytest.raises(RuntimeError, match="token id outside the embedding table"):
        trainer.assignments()
    trainer.step(x, y)
    trainer.check_device()


def test_a_wrong_token_in_a_captured_step(cuda):
    from voodoo_quant.layers import set_static_shapes

    try:
        trainer, x, y, bad = _trainer(cuda, ce_reduction="tokens", static_shapes=True)
        trainer.capture(x, y)
        trainer.replay_step(x, y)
        trainer.replay_step(bad, y)
        with pytest.raises(RuntimeError, match="token id outside the embedding table"):
            trainer.replay_step(x, y)
        trainer.replay_step(x, y)
        trainer.check_device()
        trainer.release_graph()
    finally:
        set_static_shapes(False)


def test_the_words_copy_does_not_clear_it(cuda):
    from voodoo_quant import _C

    word = torch.full((1,), 7, dtype=torch.int32, device=cuda)
    stream = torch.cuda.current_stream().cuda_stream
    assert _C.load_library().vq_device_error_async(word.data_ptr(), stream) == 0 and int(word) == 0
    table = _C.EmbedTable(["Q8_0"], [torch.zeros(272, dtype=torch.uint8, device=cuda)], 1, 256, 256)
    _C.embed_mix(torch.tensor([3], device=cuda), table, torch.ones(1, device=cuda))
    for _ in range(2):
        assert _C.load_library().vq_device_error_async(word.data_ptr(), stream) == 0 and int(word) == 4 << 16 | 30
    assert _C.device_error() == 4 << 16 | 30
