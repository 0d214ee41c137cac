"""Refusals of the packed-sequence calls that need no device."""
import pytest
import torch

from r97training_b200 import _lib as L
from r97training_b200 import ops


@pytest.mark.parametrize("device", ["cpu", torch.device("cpu"), "meta"])
def test_rope_tables_of_another_kind_of_device(device):
    """Not tables on the current GPU in place of those asked for."""
    with pytest.raises(L.R97bError):
        ops.rope_tables(8, 64, 1e4, device=device)


def _model(**kw):
    from r97training_b200.model import HybridConfig, HybridModel
    return HybridModel(HybridConfig(**{**dict(hidden=128, layers=2, gdn_per_attn=1, gdn_heads=2, gdn_qk_heads=1, attn_heads=1,
                                              attn_kv_heads=1, attn_head_dim=128, rotary_dim=32, ffn=128, vocab=128, rank=8,
                                              seq=128, micro_batch=1), **kw}), torch.device("cpu"))


@pytest.mark.parametrize("other", [dict(gdn_heads=4), dict(gdn_heads=4, gdn_qk_heads=2), dict(seq=256)])
def test_a_batch_of_another_model(other):
    """More GDN heads than the batch's tables count, or a longer rotary table than the step's: refused before anything
    runs (the step's kernels take their geometry from the batch)."""
    from r97training_b200.model import PackedBatch, TrainStep
    mine, theirs = _model(), _model(**other)
    batch = PackedBatch(theirs, [0, 100, 100 + theirs.cfg.seq])
    step = TrainStep.__new__(TrainStep)  # (an adapter's mirrors would need a device)
    step.model, step.cfg, step.packed = mine, mine.cfg, None
    ids = torch.zeros(batch.T, dtype=torch.int32)
    with pytest.raises(L.R97bError):
        step.run(ids, batch=batch)
    batch.check(theirs)
    PackedBatch(mine, [0, 100, 228]).check(_model(seq=256))
