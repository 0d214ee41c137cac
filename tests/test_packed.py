"""The packed-sequence operators on the host: the block tables, the refusals of every entry point before any device
work, and the 64-bit forms the GPU tests compare against, checked by central differences."""
import ctypes
import math

import numpy as np
import pytest
import torch

from r97training_b200 import _lib as L
from r97training_b200 import ops
from r97training_b200.packed import PackedPlan
from tests import packed_ref as ref

FAKE = 1 << 20  # aligned addresses that no refused call dereferences: operands here, outputs at multiples of OUT
OUT = 1 << 22


def _blocks(cu):
    cu = np.asarray(cu, np.int32)
    n = L.lib().r97b_packed_blocks(cu.ctypes.data, len(cu) - 1, None, None)
    if n < 0:
        return n
    q, k = np.full((n, 4), -7, np.int32), np.full((n, 4), -7, np.int32)
    assert L.lib().r97b_packed_blocks(cu.ctypes.data, len(cu) - 1, q.ctypes.data, k.ctypes.data) == n
    return q, k


@pytest.mark.parametrize("lens", [[1], [128], [129], [0, 5, 0, 0, 300, 128], [700, 3, 257], [0]])
def test_block_tables(lens):
    cu = np.cumsum([0] + lens)
    q, k = _blocks(cu)
    want = {(int(cu[s]), n, i, 0) for s, n in enumerate(lens) for i in range(-(-n // 128))}
    assert {tuple(r) for r in q.tolist()} == want and {tuple(r) for r in k.tolist()} == want
    assert len(q) == len(want)
    assert (np.diff(q[:, 2]) <= 0).all()  # the most keys to visit first
    left = -(-k[:, 1] // 128) - k[:, 2]
    assert (np.diff(left) <= 0).all()     # the most queries to visit first


@pytest.mark.parametrize("cu", [[1, 4], [0, 5, 3], [0, -1]])
def test_bad_cu_seqlens(cu):
    assert _blocks(cu) == -1
    with pytest.raises(L.R97bError):
        PackedPlan(cu, "cpu")


def test_plan_positions_and_limits():
    p = PackedPlan([0, 3, 3, 4, 204], "cpu")
    assert p.pos.tolist() == [0, 1, 2, 0] + list(range(200)) and (p.T, p.n_seq, p.max_len) == (204, 4, 200)
    assert PackedPlan([0], "cpu").T == 0 and PackedPlan([0, 0, 0], "cpu").n_blocks == 0
    with pytest.raises(L.R97bError):
        PackedPlan([], "cpu")
    with pytest.raises(L.R97bError):
        PackedPlan([0, 2 ** 31], "cpu")
    assert L.lib().r97b_packed_blocks(None, 1, None, None) == -1


HOST = np.array([[0, 300, 0, 0], [0, 300, 1, 0], [0, 300, 2, 0]], np.int32)  # 300 tokens, longest first


def _plan():
    return L.R97bPacked(1, 3, 300, FAKE, FAKE, HOST.ctypes.data)


def _rows(ptr=FAKE, tok=2048, head=256):
    return L.R97bHeadRows(ptr, tok, head)


def _fwd_args(**kw):
    a = L.R97bAttnPackedFwd(8, 2, 256, 0.0625, _rows(), _rows(), _rows(), _rows(OUT), FAKE, 300)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def _bwd_args(**kw):
    a = L.R97bAttnPackedBwd(8, 2, 256, 0.0625, _rows(), _rows(), _rows(), _rows(), _rows(), FAKE, 300, _rows(OUT),
                            _rows(2 * OUT), _rows(3 * OUT), 4 * OUT, 1 << 40)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


BAD_COMMON = [dict(Hq=0), dict(Hkv=0), dict(Hq=7), dict(D=192), dict(D=64), dict(lse=None), dict(ld_lse=299),
              dict(q=_rows(None)), dict(k=_rows(FAKE + 2)), dict(v=_rows(head=248)), dict(o=_rows(head=252)),
              dict(q=_rows(tok=2040)), dict(o=_rows(tok=0)), dict(k=_rows(tok=-2048)), dict(v=_rows(tok=2052)),
              dict(lse=FAKE + 1)]


@pytest.mark.parametrize("bad", BAD_COMMON + [dict(p=dict(T=-1)), dict(p=dict(n_blocks=2)), dict(p=dict(q_blocks=None)),
                                              dict(p=dict(k_blocks=FAKE + 4)), dict(p=dict(T=0)),
                                              dict(p=dict(n_blocks=301)), dict(p=dict(k_blocks_host=None))])
def test_attention_refusals(bad):
    h = L.lib()
    bad = dict(bad)
    plan = _plan()
    for n, v in bad.pop("p", {}).items():
        setattr(plan, n, v)
    assert h.r97b_attn_packed_fwd(ctypes.byref(plan), ctypes.byref(_fwd_args(**bad)), None) == 1
    assert h.r97b_attn_packed_bwd(ctypes.byref(plan), ctypes.byref(_bwd_args(**bad)), None) == 1


def test_attention_refusals_of_one_direction():
    h = L.lib()
    plan = _plan()
    ref_ = ctypes.byref(plan)
    assert h.r97b_attn_packed_fwd(None, ctypes.byref(_fwd_args()), None) == 1
    assert h.r97b_attn_packed_fwd(ref_, None, None) == 1
    assert h.r97b_attn_packed_bwd(ref_, None, None) == 1
    need = h.r97b_attn_packed_bwd_workspace_bytes(ref_, 8, 2, 256)
    assert need >= 0
    assert h.r97b_attn_packed_fwd(ref_, ctypes.byref(_fwd_args(o=_rows())), None) == 1  # over an operand
    for bad in (dict(dout=_rows(None)), dict(dq=_rows(OUT, head=8)), dict(dk=_rows(OUT + 8)), dict(dv=_rows(OUT, tok=256)),
                dict(dq=_rows()), dict(dk=_rows()), dict(dv=_rows()), dict(dk=_rows(OUT)), dict(dv=_rows(2 * OUT)),
                dict(ws=OUT), dict(ws=FAKE)):
        assert h.r97b_attn_packed_bwd(ref_, ctypes.byref(_bwd_args(**bad)), None) == 1
    assert h.r97b_attn_packed_bwd(ref_, ctypes.byref(_bwd_args(ws=FAKE + 16)), None) == 1
    if need:
        assert h.r97b_attn_packed_bwd(ref_, ctypes.byref(_bwd_args(ws_bytes=need - 1)), None) == 1
        assert h.r97b_attn_packed_bwd(ref_, ctypes.byref(_bwd_args(ws=None)), None) == 1
    for Hq, Hkv, D in ((8, 3, 256), (0, 1, 128), (8, 2, 96)):
        assert h.r97b_attn_packed_bwd_workspace_bytes(ref_, Hq, Hkv, D) == -1


def test_nothing_to_do_is_ok():
    """A batch of empty sequences launches nothing."""
    h = L.lib()
    plan = L.R97bPacked(2, 0, 0, None, None, None)
    assert h.r97b_attn_packed_fwd(ctypes.byref(plan), ctypes.byref(_fwd_args()), None) == 0
    assert h.r97b_attn_packed_bwd(ctypes.byref(plan), ctypes.byref(_bwd_args()), None) == 0
    assert h.r97b_qk_rope_fwd(ctypes.byref(_rope_args(T=0)), None) == 0


def _rope_args(**kw):
    a = L.R97bRope()
    a.D, a.rot, a.n_parts, a.T, a.n_pos, a.eps = 256, 64, 2, 300, 300, 1e-6
    a.cos_tab = a.sin_tab = a.pos = FAKE
    for i in range(2):
        p = a.part[i]
        p.heads, p.w, p.x, p.y, p.dx = 4, FAKE, _rows(), _rows(), _rows()
    part = kw.pop("part", {})
    for n, v in kw.items():
        setattr(a, n, v)
    for n, v in part.items():
        setattr(a.part[1], n, v)
    return a


@pytest.mark.parametrize("bad", [dict(D=192), dict(rot=0), dict(rot=24), dict(rot=272), dict(n_parts=0),
                                 dict(n_parts=3), dict(T=-1), dict(n_pos=0), dict(cos_tab=None),
                                 dict(sin_tab=FAKE + 4), dict(pos=None), dict(part=dict(heads=0)),
                                 dict(part=dict(w=FAKE + 4)), dict(part=dict(x=_rows(None))),
                                 dict(part=dict(y=_rows(tok=1016))), dict(part=dict(y=_rows(FAKE + 8)))])
def test_rope_refusals(bad):
    h = L.lib()
    assert h.r97b_qk_rope_fwd(ctypes.byref(_rope_args(**bad)), None) == 1
    assert h.r97b_qk_rope_bwd(ctypes.byref(_rope_args(**bad)), None) == 1
    assert h.r97b_qk_rope_fwd(None, None) == 1
    assert h.r97b_qk_rope_bwd(ctypes.byref(_rope_args(part=dict(dx=_rows(None)))), None) == 1


@pytest.mark.parametrize("bad", [dict(n_pos=0), dict(rot=0), dict(rot=7), dict(theta=1.0), dict(theta=math.nan),
                                 dict(theta=math.inf), dict(scaling=3), dict(scaling=1, factor=0.5),
                                 dict(scaling=1, factor=math.nan), dict(scaling=2, original=0.0),
                                 dict(scaling=2, beta_slow=32.0), dict(scaling=2, beta_slow=0.0), dict(cos=None)])
def test_rope_table_refusals(bad):
    a = dict(cos=FAKE, sin=FAKE, n_pos=16, rot=64, theta=1e4, scaling=0, factor=4.0, original=4096.0, beta_fast=32.0,
             beta_slow=1.0)
    a.update(bad)
    assert L.lib().r97b_rope_tables(*a.values(), None) == 1


def test_wrappers_refuse_host_tensors_and_unknown_scalings():
    plan = PackedPlan([0, 4], "cpu")
    q = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(L.R97bError):
        ops.attn_packed_fwd(q, q, q, plan, 1.0)
    with pytest.raises(L.R97bError):
        ops.attn_packed_bwd(q, q, q, q, q, torch.zeros(2, 4), plan, 1.0)
    with pytest.raises(L.R97bError):
        ops.qk_rope_fwd([(q, None)], torch.zeros(4, 32), torch.zeros(4, 32), plan.pos)
    for sc in ({"type": "cubic"}, {"type": "linear"}, {"type": "yarn", "factor": 2.0},
               {"type": "linear", "factor": 2.0, "original": 4096}):
        with pytest.raises(L.R97bError):
            ops.rope_tables(8, 64, 1e4, scaling=sc)


# ------------------------------------------------------------------------------------------ the 64-bit forms

def _central(fn, x, step=1e-5):
    g = torch.zeros_like(x)
    flat, gf = x.view(-1), g.view(-1)
    for i in range(flat.numel()):
        keep = float(flat[i])
        flat[i] = keep + step
        hi = fn()
        flat[i] = keep - step
        lo = fn()
        flat[i] = keep
        gf[i] = (hi - lo) / (2 * step)
    return g


def test_attention_form_against_differences():
    """Central differences with step h of a smooth function are off by O(h^2) ~ 1e-10 and rounding / h ~ 1e-11."""
    gen = torch.Generator().manual_seed(3)
    lens, T = [1, 0, 5, 3], 9
    q, k, v, do = (torch.randn(T, h, 8, generator=gen, dtype=torch.float64) for h in (4, 2, 2, 4))
    out = ref.attention(q, k, v, lens, 0.4, do)
    loss = lambda: float((ref.attention(q, k, v, lens, 0.4)["o"][0] * do).sum())  # noqa: E731
    for t, n in ((q, "dq"), (k, "dk"), (v, "dv")):
        assert torch.allclose(out[n][0], _central(loss, t), rtol=0, atol=1e-8)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_rope_form_against_differences(interleaved, norm):
    gen = torch.Generator().manual_seed(4)
    x, do = (torch.randn(3, 2, 16, generator=gen, dtype=torch.float64) for _ in range(2))
    w = torch.randn(16, generator=gen, dtype=torch.float64) if norm else None
    ang = torch.randn(3, 4, generator=gen, dtype=torch.float64)
    cos, sin = 1.1 * torch.cos(ang), 1.1 * torch.sin(ang)
    loss = lambda: float((ref.rope_fwd(x, w, cos, sin, interleaved, 1e-6) * do).sum())  # noqa: E731
    got = ref.rope_bwd(x, w, do, cos, sin, interleaved, 1e-6)
    assert torch.allclose(got, _central(loss, x), rtol=0, atol=1e-8)


# ------------------------------------------------------------------------------------------ batches

def test_step_packed_lays_sequences_end_to_end():
    from r97training_b200.data import TokenSeq, step_packed, step_rows
    batch = [TokenSeq([5, 6, 7], [0, 1, 0]), TokenSeq([], []), TokenSeq([9], [1]), TokenSeq([1, 2, 3, 4], [0, 0, 1, 1])]
    ids, tgt, cu, scored = step_packed(batch)
    assert ids.tolist() == [5, 6, 7, 9, 1, 2, 3, 4] and cu.tolist() == [0, 3, 3, 4, 8]
    assert tgt.tolist() == [6, -1, -1, -1, -1, 3, 4, -1] and scored == 3
    _, frame, n = step_rows(batch, 4, 4)
    assert n == scored and frame.reshape(4, 4)[3].tolist() == tgt[4:].tolist()
    ids, tgt, cu, scored = step_packed([])
    assert len(ids) == len(tgt) == scored == 0 and cu.tolist() == [0]
    with pytest.raises(ValueError):
        step_packed([TokenSeq([1, 2], [1])])
