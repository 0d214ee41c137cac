"""The blocks that begin in a batch's last 127 tokens, which the packed attention copies without the tensor maps: every mix of
them with blocks before, in views of wider rows, with what lies beside and behind them not finite."""
import math

import pytest
import torch

from r97training_b200 import ops
from r97training_b200.packed import PackedPlan
from tests.packed_ref import assert_within
from tests import packed_ref as ref
from tests.test_gpu_packed import _cu, _inputs

pytestmark = pytest.mark.gpu

LENS = [[1], [2, 1], [127], [128], [129], [255], [1] * 100, [3] * 43, [130, 1, 2, 30], [256, 100], [5, 250, 3, 3, 3],
        [300, 0, 64, 63], [127, 127], [1, 128, 126], [640, 1]]


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x)) if len(x) < 9 else f"{len(x)}x{x[0]}")
def test_tail_blocks(cuda, lens, D):
    Hq, Hkv, T = 4, 2, sum(lens)
    scale = 1 / math.sqrt(D)
    plan = PackedPlan(_cu(lens), cuda)
    q, k, v, do = _inputs(cuda, lens, Hq, Hkv, D, T + D)

    def wide(t, extra):
        """t inside rows of its heads and `extra` more columns, all else NaN, with three rows behind."""
        buf = torch.full((T + 3, t.shape[1] * D + extra), float("nan"), dtype=torch.bfloat16, device=cuda)
        view = buf[:, extra // 2:extra // 2 + t.shape[1] * D].view(T + 3, t.shape[1], D)
        view[:T] = t
        return view

    qw, kw, vw, dow = wide(q, 16), wide(k, 512), wide(v, 48), wide(do, 0)
    o, lse = ops.attn_packed_fwd(qw, kw, vw, plan, scale)
    dq, dk, dv = ops.attn_packed_bwd(qw, kw, vw, o, dow, lse, plan, scale)
    torch.cuda.synchronize()
    got = dict(o=o[:T], lse=lse[:, :T], dq=dq[:T], dk=dk[:T], dv=dv[:T])
    want = ref.attention(q, k, v, lens, scale, do, o_in=got["o"], lse_in=got["lse"])
    for n, t in got.items():
        assert_within(t, want[n], n)
    # the same bits with rows behind that the maps may claim: the last tokens' blocks then go through them
    far = [torch.cat([t, torch.full((200, *t.shape[1:]), float("nan"), dtype=t.dtype, device=cuda)]) for t in (q, k, v, do)]
    padded = PackedPlan(_cu(lens + [200]), cuda)
    o2, lse2 = ops.attn_packed_fwd(*far[:3], padded, scale)
    dq2 = ops.attn_packed_bwd(*far[:3], o2, far[3], lse2, padded, scale)[0]
    assert torch.equal(o2[:T], got["o"]) and torch.equal(lse2[:, :T], got["lse"]) and torch.equal(dq2[:T], got["dq"])


def test_smallest_steps(cuda):
    """A whole step of one token, of three sequences of one (nothing to predict: no loss, no gradient) and of two tokens."""
    from r97training_b200.model import PackedBatch
    from tests.test_gpu_packed_step import _fresh, _grad, _ids
    cfg, model, ad, step = _fresh(cuda)
    for cu in ([0, 1], [0, 1, 2, 3]):
        loss, grad = _grad(step, ad, _ids(cuda, cu[-1], cfg.vocab, 5), batch=PackedBatch(model, cu))
        assert loss == 0.0 and (grad == 0).all()
    loss, grad = _grad(step, ad, _ids(cuda, 2, cfg.vocab, 5), batch=PackedBatch(model, [0, 2]))
    assert 0 < loss < 4 * math.log(cfg.vocab) and torch.isfinite(grad).all() and (grad != 0).any()
