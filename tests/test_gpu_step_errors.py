"""A training step that refuses its call."""
import pytest
import torch

from r97training_b200._lib import R97bError, lib
from tests.test_gpu_packed_step import _fresh, _ids

pytestmark = pytest.mark.gpu


def test_a_refused_call_launches_nothing(cuda):
    cfg, model, ad, step = _fresh(cuda, rope_interleaved=True)
    torch.cuda.synchronize()
    before = lib().r97b_launch_count()
    with pytest.raises(R97bError, match="interleaved"):  # the fixed frame's pairs are neighbouring halves
        step.run(_ids(cuda, cfg.tokens, cfg.vocab, 1))
    assert lib().r97b_launch_count() == before
