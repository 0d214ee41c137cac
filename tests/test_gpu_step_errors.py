"""A training step that refuses its call, or fails inside it, leaves nothing in flight behind it: weights are decoded ahead
on a side stream, into buffers that go when the step does."""
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


def test_a_failed_run_waits_for_its_side_stream(cuda):
    """What follows on the caller's stream (the next owner of the step's buffers) comes after the decodes ahead."""
    cfg, model, ad, step = _fresh(cuda)
    ids = _ids(cuda, cfg.tokens, cfg.vocab, 1)
    step.run(ids)
    torch.cuda.synchronize()

    def fail(*a):
        with torch.cuda.stream(step.side):
            torch.cuda._sleep(200_000_000)  # some 100 ms of decoding still to come
        raise MemoryError("no room for the layer's tensors")

    step._attn_fwd = fail
    with pytest.raises(MemoryError):
        step.run(ids)
    mark = torch.cuda.Event()
    mark.record()
    mark.synchronize()
    assert step.side.query()
    del step._attn_fwd
    ad.g.zero_()
    loss = step.run(ids)
    torch.cuda.synchronize()
    assert torch.isfinite(loss) and torch.isfinite(ad.g).all()
