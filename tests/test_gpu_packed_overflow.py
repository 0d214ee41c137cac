"""Packed attention rows whose first key tiles hold no score above f32's lowest: q . k overflows to -inf there, the
definition gives those keys a probability of 0, and the row is what its other keys make it, however low their scores."""
import pytest
import torch

from r97training_b200 import ops
from r97training_b200.packed import PackedPlan
from tests import packed_ref as ref
from tests.packed_ref import assert_within

pytestmark = pytest.mark.gpu

SCALE = 0.0625


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("low", [128, 256, 384])
def test_first_tiles_below_f32(cuda, D, low):
    """Rows from `low` on see the keys before it at -2^200 and the others at about -256, 2^-369: a reference of 0 would
    flush them all. The rows before see ordinary scores. Head 1 is left ordinary throughout."""
    n, Hq, Hkv = 700, 4, 2
    g = torch.Generator(device=cuda).manual_seed(D + low)
    r = lambda h, s=1.0: (torch.randn(n, h, D, generator=g, device=cuda) * s).bfloat16()  # noqa: E731
    q, k, v, do = r(Hq), r(Hkv), r(Hkv), r(Hq, 0.1)
    q[low:, :2, 0], q[:low, :2, 0] = 2.0 ** 100, 0.0
    k[low:, 0, 0], k[:low, 0, 0] = -(2.0 ** -88), -(2.0 ** 100)
    do[:low] = 0.0
    plan = PackedPlan([0, n], cuda)
    o, lse = ops.attn_packed_fwd(q, k, v, plan, SCALE)
    dq, dk, dv = ops.attn_packed_bwd(q, k, v, o, do, lse, plan, SCALE)
    torch.cuda.synchronize()
    got = dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv)
    # the forward of the group that overflows: the first rows as a sequence of their own, the others as one without them
    part = lambda t, rows, h: t[rows, :h]  # noqa: E731
    for rows in (slice(0, low), slice(low, n)):
        want = ref.attention(part(q, rows, 2), part(k, rows, 1), part(v, rows, 1), [rows.stop - rows.start], SCALE)
        assert_within(o[rows, :2], want["o"], f"o {rows}")
        assert_within(lse[:2, rows], want["lse"], f"lse {rows}")
    # all of it, the overflowing scores replaced by -1536, whose probability is 0 in 64 bits too
    near = k.clone()
    near[:low, 0, 0] = -1.5 * 2.0 ** -86
    whole = ref.attention(q, near, v, [n], SCALE, do, o_in=o, lse_in=lse)
    for name, t in got.items():
        assert_within(t, whole[name], name)


@pytest.mark.parametrize("D", [128, 256])
def test_rows_of_nothing(cuda, D):
    """Rows all of whose scores overflow to -inf: lse -inf and NaN, and no other row's affair."""
    lens = [200, 90]
    g = torch.Generator(device=cuda).manual_seed(D)
    r = lambda h: torch.randn(290, h, D, generator=g, device=cuda).bfloat16()  # noqa: E731
    q, k, v = r(2), r(1), r(1)
    plan = PackedPlan([0, 200, 290], cuda)
    want_o, want_lse = ops.attn_packed_fwd(q, k, v, plan, SCALE)
    k[:200, :, 0] = -(2.0 ** 100)
    q[:200, :, 0] = 2.0 ** 100
    o, lse = ops.attn_packed_fwd(q, k, v, plan, SCALE)
    torch.cuda.synchronize()
    assert (lse[:, :200] == -float("inf")).all() and torch.isnan(o[:200].float()).all()
    assert torch.equal(o[200:], want_o[200:]) and torch.equal(lse[:, 200:], want_lse[:, 200:])
    assert sum(lens) == 290
