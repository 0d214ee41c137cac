"""One split-K workspace under calls of different shapes (R97B_EPI_SPLIT_BF16, csrc/gemm_tc.cu): a call's tile counters
lie where an earlier, smaller call left partial sums. And a training step whose packed batches differ in length, which
shares one so."""
import numpy as np
import pytest
import torch

from r97training_b200 import ops
from r97training_b200.model import PackedBatch
from tests.gpu_util import assert_close_bf16, to_np
from tests.test_gpu_packed_step import TWO_RUNS, _fresh, _grad, _ids

pytestmark = pytest.mark.gpu


def _call(cuda, ws, M, N, bn, splits, seed, K=512):
    g = torch.Generator(device=cuda).manual_seed(seed)
    a = torch.randn(M, K, generator=g, device=cuda).bfloat16()
    b = (torch.randn(N, K, generator=g, device=cuda) * 0.1).bfloat16()
    out = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device=cuda)
    ops.gemm(a, b, out, mode=ops.EPI_SPLIT_BF16, splits=splits, bn=bn, ws=ws.buf)
    return out, a.double() @ b.double().T


@pytest.mark.parametrize("shapes", [
    [(300, 64, 64, 2), (70 * 128, 64, 64, 2)],                       # 3 tiles, then 70
    [(8192, 64, 64, 2), (8200, 64, 64, 2), (100, 64, 64, 2)],        # 64, 65, 1
    [(64, 256, 256, 4), (4096, 384, 128, 2), (12600, 64, 64, 2)],    # 1, 96, 99 of other widths
    [(128, 64, 64, 2), (128 * 900, 64, 64, 2), (128, 128, 128, 3), (128 * 300, 64, 64, 2)],
], ids=["3-70", "64-65-1", "widths", "900"])
def test_calls_of_different_shapes_share_a_workspace(cuda, shapes):
    shared = ops.SplitWorkspace(cuda, 96 << 20)
    for i, (M, N, bn, splits) in enumerate(shapes):
        got, want = _call(cuda, shared, M, N, bn, splits, i)
        alone, _ = _call(cuda, ops.SplitWorkspace(cuda, 96 << 20), M, N, bn, splits, i)
        torch.cuda.synchronize()
        assert torch.equal(got, alone), (i, M, N)
        assert_close_bf16(to_np(got), to_np(want), rel=4e-3, what=f"call {i}")  # one rounding to bf16: 2^-8
    assert int(shared.buf[:4096].abs().max()) == 0


def test_packed_batches_of_different_lengths_share_a_step(cuda):
    """A short batch, then one of 8200 tokens (65 tiles of rows): the gradient of a step that only saw the long one."""
    cfg, model, ad, step = _fresh(cuda)
    _, model2, ad2, step2 = _fresh(cuda)
    cu = np.minimum(np.arange(0, 8200 + 256, 256), 8200)
    ids = _ids(cuda, 8200, cfg.vocab, 7)
    _grad(step, ad, _ids(cuda, 300, cfg.vocab, 6), batch=PackedBatch(model, [0, 200, 300]))
    loss, grad = _grad(step, ad, ids, batch=PackedBatch(model, cu))
    want_loss, want = _grad(step2, ad2, ids, batch=PackedBatch(model2, cu))
    assert abs(loss - want_loss) <= 1e-3 * want_loss
    assert_close_bf16(to_np(grad), to_np(want), **TWO_RUNS, what="adapter gradient")
