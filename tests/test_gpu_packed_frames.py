"""Scaled rotary positions (HybridConfig.rope_scaling) are the model's, for its fixed frame as for packed batches."""
import math

import pytest
import torch

from r97training_b200.model import PackedBatch
from tests.gpu_util import assert_close_bf16, to_np
from tests.test_gpu_packed_step import TWO_RUNS, _fresh, _grad, _ids

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 4.0}, {"type": "yarn", "factor": 8.0, "original": 64}],
                         ids=lambda s: s["type"])
def test_whole_frames_with_scaled_positions(cuda, scaling):
    """theta 100 turns every pair many times over a sequence, so that unscaled positions are another function: the frame's
    gradient is far from the unscaled model's, and within two bf16 runs of the packed batch's."""
    cfg, model, ad, step = _fresh(cuda, rope_scaling=scaling, rope_theta=100.0)
    _, plain_model, plain_ad, plain_step = _fresh(cuda, rope_theta=100.0)
    assert torch.equal(ad.w, plain_ad.w)
    ids = _ids(cuda, 2 * cfg.seq, cfg.vocab, 3)
    frame = _grad(step, ad, ids)
    packed = _grad(step, ad, ids, batch=PackedBatch(model, [0, cfg.seq, 2 * cfg.seq]))
    assert math.isfinite(frame[0]) and abs(packed[0] - frame[0]) <= 1e-2 * frame[0]
    assert_close_bf16(to_np(packed[1]), to_np(frame[1]), **TWO_RUNS, what="packed against frame")
    other = _grad(plain_step, plain_ad, ids)[1].double()
    apart = float((frame[1].double() - other).norm() / other.norm())
    assert apart > 2 * TWO_RUNS["rel"], apart
