"""The C++ step over a model with scaled rotary positions against the Python step's fixed frame: the same tables."""
import pytest
import torch

from tests.gpu_util import assert_close_bf16, to_np

pytestmark = pytest.mark.gpu


def test_cpp_step_takes_scaled_positions(cuda):
    from r97training_b200.cstep import CStep
    from tests.test_gpu_packed_step import TWO_RUNS, _fresh, _grad, _ids
    cfg, model, ad, step = _fresh(cuda, rope_theta=100.0, rope_scaling={"type": "yarn", "factor": 8.0, "original": 64})
    ids = _ids(cuda, 2 * cfg.seq, cfg.vocab, 3)
    loss, grad = _grad(step, ad, ids)
    tgt = torch.full((2, cfg.seq), -1, dtype=torch.int32, device=cuda)
    tgt[:, :-1] = ids.view(2, cfg.seq)[:, 1:]
    n, g = 2 * (cfg.seq - 1), torch.zeros_like(ad.g)
    cs = CStep(model, head_chunk=128)
    got = cs.run(ids, tgt.reshape(-1), n, ad.w, g)
    torch.cuda.synchronize()
    assert abs(got / n - loss) <= 1e-2 * loss
    assert_close_bf16(to_np(g), to_np(grad), **TWO_RUNS, what="adapter gradient")
    cs.close()
