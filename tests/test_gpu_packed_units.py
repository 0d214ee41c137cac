"""How the packed attention's key passes divide their work (csrc/attn_packed.cu, split_of and Walk): key blocks left
whole, split over some or all of their query heads, and whole blocks launched before the split ones, each against the
64-bit form, with the division that the lengths are meant to reach asserted first. And sequences of a length at which
every tile loop, reference and offset is far into its range."""
import math

import numpy as np
import pytest
import torch

from r97training_b200 import ops
from r97training_b200.packed import PackedPlan
from tests.packed_ref import E32, U, assert_within
from tests.test_gpu_packed import _check, _cu, _inputs

pytestmark = pytest.mark.gpu


def _division(plan, Hq, Hkv, D):
    """(split blocks, parts a block, whole blocks before them): the rule restated, and held to what the workspace has
    room for."""
    sms = torch.cuda.get_device_properties(plan.device).multi_processor_count
    grp = Hq // Hkv
    host = plan._k_host.reshape(-1, 4).astype(np.int64)
    queries = -(-host[:, 1] // 128) - host[:, 2]
    limit = 1.15 * int(queries.sum()) * Hq / sms
    split, parts, first = 0, 1, 0
    if grp > 1 and queries[0] * grp > limit:
        fits = [d for d in range(2, grp) if grp % d == 0 and queries[0] * grp / d <= limit]
        parts = min(fits, default=grp)
        split = int((queries * grp > limit).sum())
        while split + first < len(queries) and queries[split + first] * parts > queries[0]:
            first += 1
    ws = ops.attn_packed_bwd_workspace(plan, Hq, Hkv, D).numel()
    sums = 4 * 2 * split * parts * Hkv * 128 * D
    assert ws == max(4 * Hq * (-(-plan.T // 64) * 64) + sums, 256), "the division's rule has changed: see these lengths"
    return split, parts, first


DIVISIONS = [
    ([1024] * 8, 16, 4, "whole"),
    ([1300, 1100, 900, 700, 500, 300, 200, 100], 16, 4, "some heads a part"),
    ([1500, 1000, 1000, 800, 800, 600, 600, 300, 77], 16, 4, "some heads a part, whole blocks first"),
    ([1700, 1700, 1700, 400, 400, 400, 400, 400], 16, 4, "some heads a part, whole blocks first"),
    ([1500, 1200, 900, 900, 900, 600, 600, 300, 77], 12, 2, "some heads a part"),
    ([1500] + [200] * 20, 16, 4, "a part a head, whole blocks first"),
    ([900, 130], 6, 1, "a part a head"),
]


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("lens,Hq,Hkv,kind", DIVISIONS, ids=lambda x: "-".join(map(str, x)) if isinstance(x, list) else None)
def test_divisions(cuda, lens, Hq, Hkv, kind, D):
    plan = PackedPlan(_cu(lens), cuda)
    split, parts, first = _division(plan, Hq, Hkv, D)
    if torch.cuda.get_device_properties(cuda).multi_processor_count == 148:
        names = "whole" if not split else ("a part a head" if parts == Hq // Hkv else "some heads a part")
        assert kind == names + (", whole blocks first" if first else ""), (split, parts, first)
    _check(*_inputs(cuda, lens, Hq, Hkv, D, sum(lens) + D), lens, 1 / math.sqrt(D), plan)


@pytest.mark.parametrize("D", [128, 256])
def test_many_short_sequences(cuda, D):
    """Hundreds of sequences of 0 to 5 tokens: a unit each, more than the SMs take at once."""
    lens = [(7 * i * i + 3 * i) % 6 for i in range(150)]
    _check(*_inputs(cuda, lens, 4, 2, D, 7 + D), lens, 1 / math.sqrt(D))


@pytest.mark.parametrize("D", [128, 256])
def test_long_sequence_slices(cuda, D):
    """One sequence of 20011 tokens, its key blocks split and whole ones before them: o, lse and dq at its last rows and
    at two of its middle, dk and dv at its first keys, at its last and at two of its middle, in 64 bits. The bounds are
    packed_ref.attention's, on the rows and keys compared."""
    n, Hq, Hkv = 20011, 2, 1
    scale = 1 / math.sqrt(D)
    q, k, v, do = _inputs(cuda, [n], Hq, Hkv, D, 71 + D)
    plan = PackedPlan([0, n], cuda)
    split, parts, first = _division(plan, Hq, Hkv, D)
    assert split > 0 and parts == 2 and first > 0
    o, lse = ops.attn_packed_fwd(q, k, v, plan, scale)
    dq, dk, dv = ops.attn_packed_bwd(q, k, v, o, do, lse, plan, scale)
    torch.cuda.synchronize()
    f = lambda t: t.double()  # noqa: E731
    kf, vf = f(k[:, 0]), f(v[:, 0])

    def tile(rows, keys, h):
        """Scores, their bound, dP, its magnitudes' sum, and the mask of `rows` against `keys`."""
        seen = torch.arange(n, device=cuda)[rows][:, None] >= torch.arange(n, device=cuda)[keys][None, :]
        qh, dh = f(q[rows, h]), f(do[rows, h])
        x = qh @ kf[keys].T * scale
        # the score's own share of packed_ref's bound; the caller adds the lse's
        es = (D + 4) * E32 * (qh.abs() @ kf[keys].abs().T) * scale + 8 * E32 * x.abs() + 8 * E32
        return seen, x, es, dh @ vf[keys].T, dh.abs() @ vf[keys].abs().T

    def grads(rows, keys, h):
        """P, dS and their bounds from the forward's own lse and o."""
        seen, x, es, dp, mag = tile(rows, keys, h)
        lse_h, ob, dh = f(lse[h, rows])[:, None], f(o[rows, h]), f(do[rows, h])
        es = es + 8 * E32 * lse_h.abs()
        p = torch.exp(x - lse_h) * seen
        delta = (dh * ob).sum(1, keepdim=True)
        d_err = D * E32 * (dh * ob).abs().sum(1, keepdim=True)
        # rows of the sequence's first 128 tokens: delta is the row's sum of P o dP, over keys that are all here
        at = torch.arange(n, device=cuda)[rows]
        if int(at.min()) < 128:
            s2, x2, e2, dp2, mag2 = tile(rows, slice(0, 128), h)
            p2 = torch.exp(x2 - lse_h) * s2
            own = (p2 * dp2).sum(1, keepdim=True)
            own_err = (p2 * ((e2 + 8 * E32 * lse_h.abs()) * dp2.abs() + (D + 128) * E32 * mag2)).sum(1, keepdim=True)
            head = (at < 128)[:, None]
            delta, d_err = torch.where(head, own, delta), torch.where(head, own_err, d_err)
        ds = p * (dp - delta)
        err = U * ds.abs() + es * p * (dp.abs() + delta.abs()) + p * (
            d_err + (D + 2) * E32 * mag + 2 * E32 * delta.abs()) + n * Hq * E32 * ds.abs()
        return p, p * (U + es + n * Hq * E32), ds, err

    for rows in (slice(n - 200, n), slice(9984 - 40, 9984 + 40), slice(13000, 13064)):
        for h in range(Hq):
            seen, x, es, _, _ = tile(rows, slice(0, n), h)
            x = x.masked_fill(~seen, -math.inf)
            want_lse = torch.logsumexp(x, 1)
            p = torch.exp(x - want_lse[:, None])
            A, want_o = p @ vf.abs(), p @ vf
            es = (es + 8 * E32 * want_lse.abs()[:, None]).masked_fill(~seen, 0)
            rel = es.amax(1, keepdim=True) * 2 + n * E32
            assert_within(o[rows, h], (want_o, U * A + U * want_o.abs() + rel * A * 2), f"o {rows}")
            assert_within(lse[h, rows], (want_lse, rel[:, 0] + 8 * E32 * want_lse.abs()), f"lse {rows}")
            _, _, ds, err = grads(rows, slice(0, n), h)
            want = ds @ kf * scale
            assert_within(dq[rows, h], (want, (err @ kf.abs()) * scale + U * want.abs() + 1e-30), f"dq {rows}")
    for keys in (slice(0, 200), slice(9984 - 40, 9984 + 40), slice(13000, 13064), slice(n - 60, n)):
        out = {"dk": [0.0, 0.0], "dv": [0.0, 0.0]}
        for h in range(Hq):
            for a in range(0, n, 4096):
                rows = slice(a, min(n, a + 4096))
                p, p_err, ds, ds_err = grads(rows, keys, h)
                qh, dh = f(q[rows, h]), f(do[rows, h])
                for name, m, e, t in (("dk", ds * scale, ds_err * scale, qh), ("dv", p, p_err, dh)):
                    out[name][0] = out[name][0] + m.T @ t
                    out[name][1] = out[name][1] + e.T @ t.abs()
        for name, got in (("dk", dk), ("dv", dv)):
            want, err = out[name]
            assert_within(got[keys, 0], (want, err + U * want.abs() + 1e-30), f"{name} {keys}")
