"""GPU parity of the packed-sequence operators, through the C ABI: causal grouped-query attention over ragged
sequences (r97b_attn_packed_fwd / _bwd, csrc/attn_packed.cu) and rotary positions with the q/k norm (r97b_qk_rope_fwd /
_bwd, r97b_rope_tables, csrc/rope.cu), against the 64-bit forms of tests/packed_ref.py with their elementwise bounds."""
import math

import pytest
import torch

from r97training_b200 import ops
from r97training_b200._lib import R97bError
from r97training_b200.packed import PackedPlan
from tests import packed_ref as ref
from tests.packed_ref import assert_within

pytestmark = pytest.mark.gpu


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _inputs(dev, lens, Hq, Hkv, D, seed, qstd=1.0, extra=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    T = sum(lens) + extra
    r = lambda h, s=1.0: (torch.randn(T, h, D, generator=g, device=dev) * s).bfloat16()  # noqa: E731
    return r(Hq, qstd), r(Hkv), r(Hkv), r(Hq, 0.1)


def _check(q, k, v, do, lens, scale, plan=None):
    """One forward and backward against the 64-bit forms: the backward on the forward's own o and lse, then end to
    end; and the same bits from a second call."""
    T = sum(lens)
    plan = plan or PackedPlan(_cu(lens), q.device)
    o, lse = ops.attn_packed_fwd(q, k, v, plan, scale)
    dq, dk, dv = ops.attn_packed_bwd(q, k, v, o, do, lse, plan, scale)
    o2, lse2 = ops.attn_packed_fwd(q, k, v, plan, scale)
    again = ops.attn_packed_bwd(q, k, v, o, do, lse, plan, scale)
    torch.cuda.synchronize()
    s = slice(0, T)
    assert torch.equal(o[s], o2[s]) and torch.equal(lse[:, s], lse2[:, s])
    got = dict(o=o[s], lse=lse[:, s], dq=dq[s], dk=dk[s], dv=dv[s])
    for n, t in zip(("dq", "dk", "dv"), again):
        assert torch.equal(got[n], t[s]), n
    own = ref.attention(q[s], k[s], v[s], lens, scale, do[s], o_in=o[s], lse_in=lse[:, s])
    for n in ("o", "lse", "dq", "dk", "dv"):
        assert_within(got[n], own[n], n)
    whole = ref.attention(q[s], k[s], v[s], lens, scale, do[s])
    for n in ("dq", "dk", "dv"):
        assert_within(got[n], whole[n], n + " end to end")
    return got


LENS = [[1], [1, 1, 2], [127], [128], [129], [256, 1], [5, 0, 133, 64, 0], [384], [511, 3, 250], [700]]


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x)))
def test_attention_lengths(cuda, lens, D):
    _check(*_inputs(cuda, lens, 4, 2, D, sum(lens) + D), lens, 1 / math.sqrt(D))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (4, 1), (6, 2), (7, 1), (16, 4)])
def test_attention_heads(cuda, Hq, Hkv, D):
    lens = [200, 77]
    _check(*_inputs(cuda, lens, Hq, Hkv, D, Hq * 10 + D), lens, 1 / math.sqrt(D))


@pytest.mark.parametrize("D", [128, 256])
def test_attention_many_units(cuda, D):
    """More (block, head) units than SMs, with long and short sequences mixed."""
    lens = [1500, 3, 40, 900, 128, 1, 640, 333]
    _check(*_inputs(cuda, lens, 8, 2, D, 5 + D), lens, 1 / math.sqrt(D))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("qstd", [0.0, 8.0, 40.0])
def test_attention_score_ranges(cuda, D, qstd):
    """Equal scores; sharp ones; scores of hundreds, where a row is one-hot and its maximum moves from tile to tile."""
    lens = [600, 130]
    _check(*_inputs(cuda, lens, 4, 2, D, 9 + D, qstd=qstd), lens, 1 / math.sqrt(D))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("rising", [True, False])
def test_attention_moving_maximum(cuda, D, rising):
    """Keys whose scores rise (or fall) by 20 a tile: each tile replaces the running maximum, or none does."""
    lens = [900]
    q, k, v, do = _inputs(cuda, lens, 4, 2, D, 21 + D)
    step = torch.arange(900, device=cuda).float() / 128
    ramp = (step if rising else step.flip(0)) * 20
    q[:, :, 0] = math.sqrt(D)
    k[:, :, 0] = ramp[:, None].bfloat16()
    _check(q, k, v, do, lens, 1 / math.sqrt(D))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("scale", [0.0, -0.05, 1.0])
def test_attention_scales(cuda, D, scale):
    lens = [300, 20]
    _check(*_inputs(cuda, lens, 2, 1, D, 31 + D), lens, scale)


@pytest.mark.parametrize("D", [128, 256])
def test_attention_strided_views(cuda, D):
    """Every operand and result a view inside wider rows; what lies between is left as it was."""
    lens, Hq, Hkv = [150, 0, 301], 4, 2
    T, rows = sum(lens), sum(lens) + 9
    q, k, v, do = _inputs(cuda, lens, Hq, Hkv, D, 41 + D)
    plan = PackedPlan(_cu(lens), cuda)

    def wide(t, heads, pitch, fill):
        buf = torch.full((rows, heads * pitch + 24), fill, dtype=torch.bfloat16, device=cuda)
        view = buf[:, 8:8 + heads * pitch].view(rows, heads, pitch)[:, :, 8:8 + D]
        if t is not None:
            view[:T] = t
        return buf, view

    nan = float("nan")
    (_, qw), (_, kw), (_, vw), (_, dow) = (wide(t, h, D + 16, nan) for t, h in ((q, Hq), (k, Hkv), (v, Hkv), (do, Hq)))
    outs = {n: wide(None, h, p, 7.0) for n, h, p in (("o", Hq, D + 24), ("dq", Hq, D + 16), ("dk", Hkv, 2 * D),
                                                     ("dv", Hkv, D + 8))}
    lse = torch.full((Hq, rows + 3), 7.0, device=cuda)
    scale = 1 / math.sqrt(D)
    ops.attn_packed_fwd(qw, kw, vw, plan, scale, o=outs["o"][1], lse=lse)
    ops.attn_packed_bwd(qw, kw, vw, outs["o"][1], dow, lse, plan, scale, dq=outs["dq"][1], dk=outs["dk"][1],
                        dv=outs["dv"][1])
    want = _check(q, k, v, do, lens, scale, plan)
    assert torch.equal(lse[:, :T], want["lse"]) and (lse[:, T:] == 7).all()
    for n, (buf, view) in outs.items():
        assert torch.equal(view[:T], want[n]), n
        view[:T] = 7.0
        assert (buf == 7).all(), f"{n}: written outside its rows"


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_sequences_do_not_mix(cuda, D, bad):
    """Non-finite rows of one sequence, and of the padding behind the last, reach no other sequence."""
    lens = [100, 37, 165, 90]
    T = sum(lens)
    q, k, v, do = _inputs(cuda, lens, 4, 2, D, 51 + D, extra=60)
    plan = PackedPlan(_cu(lens), cuda)
    scale = 1 / math.sqrt(D)
    o, lse = ops.attn_packed_fwd(q, k, v, plan, scale)
    want = (o, lse.T, *ops.attn_packed_bwd(q, k, v, o, do, lse, plan, scale))
    for t in (q, k, v, do):
        t[100:137] = bad
        t[T:] = bad
    o2, lse2 = ops.attn_packed_fwd(q, k, v, plan, scale)
    got = (o2, lse2.T, *ops.attn_packed_bwd(q, k, v, o2, do, lse2, plan, scale))
    torch.cuda.synchronize()
    for n, a, b in zip(("o", "lse", "dq", "dk", "dv"), got, want):
        for r in (slice(0, 100), slice(137, T)):
            assert torch.equal(a[r], b[r]), n
        assert not torch.isfinite(a[100:137].float()).all(), n


@pytest.mark.parametrize("D", [128, 256])
def test_attention_prefix_sums_as_one_sequence(cuda, D):
    """A sequence's results do not depend on what it is packed with."""
    lens = [190, 333]
    q, k, v, do = _inputs(cuda, lens, 4, 2, D, 61 + D)
    scale = 1 / math.sqrt(D)
    both = _check(q, k, v, do, lens, scale)
    alone = _check(q[190:].clone(), k[190:].clone(), v[190:].clone(), do[190:].clone(), [333], scale)
    assert torch.equal(both["o"][190:], alone["o"]) and torch.equal(both["lse"][:, 190:], alone["lse"])
    assert torch.equal(both["dq"][190:], alone["dq"])
    for n in ("dk", "dv"):  # (their split over query heads may differ with the batch: each within its bound above)
        assert (both[n][190:].float() - alone[n].float()).abs().max() <= 4 * ref.U * alone[n].float().abs().max()


def test_attention_long(cuda):
    """A long sequence of an odd length; the forward and dq at its last rows and dk, dv at its first."""
    D, Hq, Hkv, n = 128, 2, 1, 20011
    q, k, v, do = _inputs(cuda, [n], Hq, Hkv, D, 71)
    plan = PackedPlan([0, n], cuda)
    scale = 1 / math.sqrt(D)
    o, lse = ops.attn_packed_fwd(q, k, v, plan, scale)
    dq, dk, dv = ops.attn_packed_bwd(q, k, v, o, do, lse, plan, scale)
    x = torch.einsum("thd,sd->hts", q.double(), k[:, 0].double()) * scale
    x = x.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=cuda).tril(), -math.inf)
    p = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
    del x
    want_o = torch.einsum("hts,sd->thd", p, v[:, 0].double())
    A = torch.einsum("hts,sd->thd", p, v[:, 0].double().abs())
    assert_within(o, (want_o, ref.U * (A + want_o.abs()) + 4e-5 * A), "o")
    want_dv = torch.einsum("hts,thd->sd", p, do.double())
    A = torch.einsum("hts,thd->sd", p, do.double().abs())
    # 4e-5: the scores' f32 error, D 2^-24 of magnitudes of about 7, in the row's sum; 1e-3: n = 20011 terms of 2^-24
    assert_within(dv[:, 0], (want_dv, ref.U * (A + want_dv.abs()) + 1e-3 * A), "dv")


@pytest.mark.parametrize("D", [128, 256])
def test_attention_streams_and_graph(cuda, D):
    """A side stream, and two captured graphs with a workspace each, replayed on new inputs, give the eager bits."""
    lens = [300, 45, 128]
    plan = PackedPlan(_cu(lens), cuda)
    scale = 1 / math.sqrt(D)
    a, b = _inputs(cuda, lens, 4, 2, D, 81), _inputs(cuda, lens, 4, 2, D, 82)

    def step(t, ws=None, stream=None):
        o, lse = ops.attn_packed_fwd(*t[:3], plan, scale, stream=stream)
        return (o, lse, *ops.attn_packed_bwd(*t[:3], o, t[3], lse, plan, scale, ws, stream=stream))

    want_a, want_b = step(a), step(b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(a)
    side.synchronize()
    given = step(a, stream=side)  # the stream as an argument
    side.synchronize()
    for x, y, z in zip(got, want_a, given):
        assert torch.equal(x, y) and torch.equal(x, z)
    held = [tuple(t.clone() for t in a) for _ in range(2)]
    graphs, outs = [], []
    for t in held:
        ws = ops.attn_packed_bwd_workspace(plan, 4, 2, D)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((step(t, ws), ws))
        graphs.append(g)
    for dst, src in zip(held[1], b):
        dst.copy_(src)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
    torch.cuda.synchronize()
    for (got, _), want in zip(outs, (want_a, want_b)):
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_given_stream_owns_what_a_call_allocates(cuda):
    """A call on a stream that is busy: its workspace and results are not handed to the current stream's next
    allocations while it waits there."""
    lens = [260, 77]
    plan = PackedPlan(_cu(lens), cuda)
    q, k, v, do = _inputs(cuda, lens, 4, 2, 128, 83)
    cos, sin = ops.rope_tables(300, 64, 1e4)
    side = torch.cuda.Stream()

    def chain(stream):
        (qr,) = ops.qk_rope_fwd([(q, None)], cos, sin, plan.pos, stream=stream)
        o, lse = ops.attn_packed_fwd(qr, k, v, plan, 0.1, stream=stream)
        return ops.attn_packed_bwd(qr, k, v, o, do, lse, plan, 0.1, stream=stream)

    want = chain(None)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(40_000_000)  # some 20 ms ahead of the calls
    got = chain(side)
    sizes = [t.numel() * t.element_size() for t in (q, k)] + [ops.attn_packed_bwd_workspace(plan, 4, 2, 128).numel()]
    over = [torch.full((n,), 255, dtype=torch.uint8, device=cuda) for n in sizes for _ in range(4)]
    torch.cuda.synchronize()
    assert all(int(t[0]) == 255 for t in over)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_attention_far_offsets(cuda):
    """Rows whose element offsets pass 2^31."""
    lens, D = [200, 40], 128
    q, k, v, do = _inputs(cuda, lens, 2, 1, D, 91)
    tok = 1 << 24
    rows = sum(lens)
    buf = torch.empty(rows * tok, dtype=torch.bfloat16, device=cuda)
    at = lambda off, h: buf.as_strided((rows, h, D), (tok, D, 1), off)  # noqa: E731
    far = [at(i * 1024, t.shape[1]).copy_(t) for i, t in enumerate((q, k, v, do))]
    outs = [at((4 + i) * 1024, h) for i, h in enumerate((2, 2, 1, 1))]
    plan, scale = PackedPlan(_cu(lens), cuda), 1 / math.sqrt(D)
    o, lse = ops.attn_packed_fwd(*far[:3], plan, scale, o=outs[0])
    ops.attn_packed_bwd(*far[:3], o, far[3], lse, plan, scale, dq=outs[1], dk=outs[2], dv=outs[3])
    o2, lse2 = ops.attn_packed_fwd(q, k, v, plan, scale)
    want = (o2, *ops.attn_packed_bwd(q, k, v, o2, do, lse2, plan, scale))
    torch.cuda.synchronize()
    assert torch.equal(lse, lse2)
    for x, y in zip(outs, want):
        assert torch.equal(x, y)


def test_attention_wrapper_refusals(cuda):
    lens = [64, 10]
    q, k, v, do = _inputs(cuda, lens, 4, 2, 128, 1)
    plan = PackedPlan(_cu(lens), cuda)
    ok = lambda **kw: ops.attn_packed_fwd(**{**dict(q=q, k=k, v=v, plan=plan, scale=1.0), **kw})  # noqa: E731
    o, lse = ok()
    for bad in (dict(q=q.float()), dict(q=q[:40]), dict(k=k[:, :1]), dict(v=v[:, :, :64]), dict(q=q[:, :3]),
                dict(k=k[:, :1].expand(-1, 2, -1)), dict(q=q[:1].expand(74, -1, -1)), dict(q=q[0]),
                dict(v=v.transpose(0, 1).contiguous().transpose(0, 1)), dict(lse=lse[:, :40]), dict(lse=lse.double()),
                dict(plan=PackedPlan([0, 75], cuda)), dict(plan=PackedPlan(_cu(lens), "cpu")), dict(o=o[:, :, ::2])):
        with pytest.raises(R97bError):
            ok(**bad)
    with pytest.raises(R97bError):
        ops.attn_packed_bwd(q, k, v, o, do[:, :2], lse, plan, 1.0)
    with pytest.raises(R97bError):
        ops.attn_packed_bwd(q, k, v, o, do, lse[:2], plan, 1.0)
    with pytest.raises(R97bError):
        ok(o=q)  # over an operand
    dq = torch.empty_like(q)
    for bad in (dict(dq=q), dict(dk=k), dict(dv=do[:, :2]), dict(dq=dq, dk=dq[:, :2])):
        with pytest.raises(R97bError):
            ops.attn_packed_bwd(q, k, v, o, do, lse, plan, 1.0, **bad)
    empty = PackedPlan([0, 0], cuda)
    o0, l0 = ops.attn_packed_fwd(q[:0], k[:0], v[:0], empty, 1.0)
    assert o0.shape == (0, 4, 128) and l0.shape == (4, 0)
    assert ops.attn_packed_bwd(q[:0], k[:0], v[:0], o0, do[:0], l0, empty, 1.0)[1].shape == (0, 2, 128)


# ------------------------------------------------------------------------------------------------ rotary positions

def _tables(dev, n_pos, rot, theta, scaling):
    inv, amp = ref.rope_frequencies(rot, theta, scaling)
    ang = torch.arange(n_pos, dtype=torch.float64, device=dev)[:, None] * torch.tensor(inv, dtype=torch.float64,
                                                                                       device=dev)
    return amp * torch.cos(ang), amp * torch.sin(ang)


YARN = {"type": "yarn", "factor": 8.0, "original": 4096}


@pytest.mark.parametrize("rot,theta,scaling", [(64, 1e7, None), (128, 1e4, {"type": "linear", "factor": 4.0}),
                                               (128, 1e6, YARN), (16, 1e4, {**YARN, "original": 64, "beta_fast": 4.0}),
                                               (2, 1e4, YARN)])
def test_rope_tables(cuda, rot, theta, scaling):
    """To one f32 rounding of the value, plus the f64 angle's own error at the last position."""
    n = 70001
    cos, sin = ops.rope_tables(n, rot, theta, scaling=scaling, device=cuda)
    wc, ws = _tables(cuda, n, rot, theta, scaling)
    assert cos.shape == (n, rot // 2) and cos.dtype == torch.float32
    slack = n * 2.0 ** -50  # a few f64 roundings of the frequency times the position
    for got, want in ((cos, wc), (sin, ws)):
        assert_within(got, (want, ref.E32 * want.abs() + slack), "table")


ROPES = [(256, 64, False, True), (128, 64, False, True), (128, 128, True, True), (64, 16, True, True),
         (64, 64, False, False), (256, 256, False, True), (128, 48, False, True), (256, 96, True, False)]


@pytest.mark.parametrize("D,rot,interleaved,norm", ROPES)
@pytest.mark.parametrize("lens,heads", [([1], (1, 1)), ([5, 0, 70, 1], (8, 2)), ([33], (9, 5))])
def test_rope_both_directions(cuda, D, rot, interleaved, norm, lens, heads):
    """Queries beside their gates and keys, in the projection's rows. Two roundings of products and one of the norm
    in f32 (8 E32 of the magnitudes), one to bf16."""
    plan = PackedPlan(_cu(lens), cuda)
    T, pad = plan.T, 3
    g = torch.Generator(device=cuda).manual_seed(D + rot + T)
    y = torch.randn(T + pad, (2 * heads[0] + heads[1]) * D, generator=g, device=cuda).bfloat16()
    xs = [y[:, :2 * heads[0] * D].view(-1, heads[0], 2 * D)[:, :, :D], y[:, 2 * heads[0] * D:].view(-1, heads[1], D)]
    ws = [1 + 0.2 * torch.randn(D, generator=g, device=cuda) if norm else None for _ in heads]
    cos, sin = ops.rope_tables(max(lens), rot, 1e4, scaling={"type": "linear", "factor": 2.0}, device=cuda)
    outs = [torch.full((T + pad, h, D), 7.0, dtype=torch.bfloat16, device=cuda) for h in heads]
    ops.qk_rope_fwd(list(zip(xs, ws)), cos, sin, plan.pos, interleaved=interleaved, outs=outs)
    douts = [(0.1 * torch.randn(T + pad, h, D, generator=g, device=cuda)).bfloat16() for h in heads]
    dy = torch.full_like(y, 7.0)
    dxs = [dy[:, :2 * heads[0] * D].view(-1, heads[0], 2 * D)[:, :, :D], dy[:, 2 * heads[0] * D:].view(-1, heads[1], D)]
    ops.qk_rope_bwd([(x, w, d, dx) for x, w, d, dx in zip(xs, ws, douts, dxs)], cos, sin, plan.pos,
                    interleaved=interleaved)
    torch.cuda.synchronize()
    at = plan.pos.long()
    c, s = cos[at].double(), sin[at].double()
    for x, w, o, d, dx in zip(xs, ws, outs, douts, dxs):
        want = ref.rope_fwd(x[:T], w, c, s, interleaved, 1e-6)
        slack = (16 + D / 4) * ref.E32 * want.abs().amax(-1, keepdim=True)
        assert_within(o[:T], (want, ref.U * want.abs() + slack), "y")
        want = ref.rope_bwd(x[:T], w, d[:T], c, s, interleaved, 1e-6)
        slack = (32 + D) * ref.E32 * (want.abs().amax(-1, keepdim=True) + d[:T].double().abs().amax(-1, keepdim=True) * 4)
        assert_within(dx[:T], (want, ref.U * want.abs() + slack), "dx")
        assert (o[T:] == 7).all() and (dx[T:] == 7).all()
    assert (dy[:, :2 * heads[0] * D].view(-1, heads[0], 2 * D)[:, :, D:] == 7).all()  # the gates' columns


def test_rope_in_place_and_one_tensor(cuda):
    """The output may be the input; a single tensor; positions in any order and repeated."""
    x = torch.randn(50, 4, 128, device=cuda).bfloat16()
    pos = torch.randint(0, 900, (50,), dtype=torch.int32, device=cuda)
    cos, sin = ops.rope_tables(900, 128, 1e4, device=cuda)
    (want,) = ops.qk_rope_fwd([(x, None)], cos, sin, pos)
    ops.qk_rope_fwd([(x, None)], cos, sin, pos, outs=[x])
    torch.cuda.synchronize()
    assert torch.equal(x, want)


def test_rope_positions_outside_the_table(cuda):
    """Their rows are zero, the others as they would be, and the device error word says so."""
    import ctypes

    from r97training_b200._lib import lib
    bits = ctypes.c_uint(0)
    lib().r97b_device_error(ctypes.byref(bits))
    x = torch.randn(6, 3, 128, device=cuda).bfloat16()
    w = torch.ones(128, device=cuda)
    cos, sin = ops.rope_tables(4, 64, 1e4, device=cuda)
    good = torch.tensor([0, 3, 1, 2, 3, 0], dtype=torch.int32, device=cuda)
    bad = torch.tensor([0, 4, 1, -1, 3, 2 ** 31 - 1], dtype=torch.int32, device=cuda)
    (want,) = ops.qk_rope_fwd([(x, w)], cos, sin, good)
    lib().r97b_device_error(ctypes.byref(bits))
    assert bits.value == 0
    (got,) = ops.qk_rope_fwd([(x, w)], cos, sin, bad)
    dx = torch.full_like(x, 7.0)
    ops.qk_rope_bwd([(x, w, x, dx)], cos, sin, bad)
    lib().r97b_device_error(ctypes.byref(bits))
    assert bits.value & 2
    for r in range(6):
        if r in (1, 3, 5):
            assert (got[r] == 0).all() and (dx[r] == 0).all()
        else:
            assert torch.equal(got[r], want[r])


def test_rope_wrapper_refusals(cuda):
    x = torch.zeros(8, 2, 128, dtype=torch.bfloat16, device=cuda)
    pos = torch.zeros(8, dtype=torch.int32, device=cuda)
    w = torch.ones(128, device=cuda)
    cos, sin = ops.rope_tables(8, 64, 1e4, device=cuda)
    go = lambda **kw: ops.qk_rope_fwd(kw.pop("parts", [(x, w)]), kw.pop("cos", cos), kw.pop("sin", sin),  # noqa: E731
                                      kw.pop("pos", pos), **kw)
    go()
    for bad in (dict(parts=[]), dict(parts=[(x, w)] * 3), dict(parts=[(x, w[:64])]), dict(parts=[(x, w.double())]),
                dict(parts=[(x[:4], w)]), dict(parts=[(x, w)], outs=[]), dict(parts=[(x[:, :, ::2], None)]),
                dict(cos=cos[:, :31]), dict(sin=sin.double()), dict(sin=sin[:4]), dict(pos=pos.long()),
                dict(pos=pos[::2]), dict(pos=pos.view(2, 4)), dict(pos=pos.cpu())):
        with pytest.raises(R97bError):
            go(**bad)
    with pytest.raises(R97bError):
        ops.qk_rope_bwd([(None, w, x, x)], cos, sin, pos)
    assert go(pos=pos[:0])[0].shape == x.shape
