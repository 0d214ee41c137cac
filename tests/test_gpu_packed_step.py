"""The training step over packed batches (TrainStep.run with a PackedBatch): rotary positions, the attention core and
its backward together with the rest of the step, from the chat batcher's sub-batches to the adapter gradient.
Gradients are held to this repository's bf16 bar (relative L2 <= 1e-2, cosine >= 0.999), as the fixed frame's are."""
import math

import numpy as np
import pytest
import torch

from r97training_b200 import data as D
from r97training_b200 import iqr as IQ
from r97training_b200._lib import R97bError
from r97training_b200.model import Adapter, HybridConfig, HybridModel, PackedBatch, TrainStep
from tests import packed_ref as ref
from tests.gpu_util import assert_close_bf16, to_np

pytestmark = pytest.mark.gpu

# Two bf16 runs of one function, each inside the bar of the exact gradient g: |a - b| <= |a - g| + |b - g| <= 2e-2 |g|, and
# with each within the angle t of g, cos(a, b) >= cos 2t = 2 cos^2 t - 1 = 2 x 0.999^2 - 1.
TWO_RUNS = dict(rel=2e-2, cos=2 * 0.999 ** 2 - 1)

BASE = dict(hidden=512, layers=4, gdn_heads=4, gdn_qk_heads=2, attn_heads=4, attn_kv_heads=2, ffn=512, vocab=1024, rank=8,
            alpha=16, seq=256, micro_batch=2, attn_head_dim=128, rotary_dim=64)


def _fresh(dev, **kw):
    cfg = HybridConfig(**{**BASE, **kw})
    model = HybridModel(cfg, dev)
    ad = Adapter(model, dev, b_std=0.05)
    return cfg, model, ad, TrainStep(model, ad, head_chunk=128)


def _ids(dev, n, vocab, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randint(0, vocab, (n,), generator=g, device=dev, dtype=torch.int32)


def _grad(step, ad, *a, **kw):
    ad.g.zero_()
    loss = step.run(*a, **kw)
    torch.cuda.synchronize()
    return float(loss), ad.g.clone()


@pytest.mark.parametrize("Dh", [128, 256])
def test_whole_frames_match_the_fixed_frame(cuda, Dh):
    cfg, model, ad, step = _fresh(cuda, attn_head_dim=Dh)
    ids = _ids(cuda, 2 * cfg.seq, cfg.vocab, 3)
    want = _grad(step, ad, ids)
    got = _grad(step, ad, ids, batch=PackedBatch(model, [0, cfg.seq, 2 * cfg.seq]))
    again = _grad(step, ad, ids)  # the frame's own run after a packed one
    assert math.isfinite(got[0]) and abs(got[0] - want[0]) <= 1e-2 * want[0]
    assert_close_bf16(to_np(got[1]), to_np(want[1]), **TWO_RUNS, what="adapter gradient")
    assert again[0] == want[0]
    assert_close_bf16(to_np(again[1]), to_np(want[1]), rel=5e-4, cos=0.9999, what="the frame again")


def test_a_packed_batch_is_the_mean_of_its_sequences(cuda):
    """Odd lengths, one token, an empty sequence: the gradient is the scored-token mean of each sequence's own."""
    cfg, model, ad, step = _fresh(cuda)
    lens = [37, 1, 200, 0, 130, 2]
    cu = np.cumsum([0] + lens)
    ids = _ids(cuda, int(cu[-1]), cfg.vocab, 5)
    loss, grad = _grad(step, ad, ids, batch=PackedBatch(model, cu))
    sum_l, sum_g, scored = 0.0, torch.zeros_like(grad), 0
    for a, n in zip(cu, lens):
        if n < 2:
            continue
        li, gi = _grad(step, ad, ids[a:a + n], batch=PackedBatch(model, [0, n]))
        sum_l, sum_g, scored = sum_l + li * (n - 1), sum_g + gi * (n - 1), scored + n - 1
    assert abs(loss - sum_l / scored) <= 2e-3 * abs(loss)  # the rows' CE, each from bf16 logits (2^-8), averaged
    assert_close_bf16(to_np(grad), to_np(sum_g / scored), **TWO_RUNS, what="adapter gradient")


def test_chat_batches_match_their_padded_frame(cuda):
    """The batcher's sub-batch laid end to end and laid into the padded frame: the same loss and gradient."""
    cfg, model, ad, step = _fresh(cuda, vocab=512, micro_batch=4, seq=256)
    chat = D.ChatData()
    lines = "\n".join('{"messages": [{"role": "user", "content": "%s"}, {"role": "assistant", "content": "%s"}]}'
                      % ("q" * (3 + 17 * i), "answer " * (2 + 3 * i)) for i in range(6))
    seqs = chat.read(lines, 256)
    batcher = D.Batcher(seqs, D.BatcherConfig(token_budget=420, devices=1, seed=2))
    sub = batcher.next()[0]
    assert 1 < len(sub) <= 4
    ids, tgt, cu, scored = D.step_packed(sub)
    fids, ftgt, fscored = D.step_rows(sub, 4, 256)
    assert scored == fscored > 0
    dev = lambda a: torch.from_numpy(a).to(cuda)  # noqa: E731
    want = _grad(step, ad, dev(fids), dev(ftgt), n_scored=scored)
    got = _grad(step, ad, dev(ids), dev(tgt), n_scored=scored, batch=PackedBatch(model, cu))
    assert abs(got[0] - want[0]) <= 2e-3 * abs(want[0])
    assert_close_bf16(to_np(got[1]), to_np(want[1]), **TWO_RUNS, what="adapter gradient")


@pytest.mark.parametrize("Dh,rot,interleaved,scaling", [(256, 64, False, None),
                                                        (128, 128, True, {"type": "yarn", "factor": 4.0, "original": 64}),
                                                        (128, 32, False, {"type": "linear", "factor": 2.0})])
def test_attention_sublayer_vs_fp32(cuda, Dh, rot, interleaved, scaling):
    """The gated-attention sublayer over ragged sequences against fp32 autograd on the same decoded weights."""
    cfg, model, ad, step = _fresh(cuda, attn_head_dim=Dh, rotary_dim=rot, rope_interleaved=interleaved,
                                  rope_scaling=scaling, max_pos=300)
    lens = [150, 1, 0, 290, 64]
    batch = PackedBatch(model, np.cumsum([0] + lens))
    li, T, d = 3, sum(lens), cfg.hidden
    blk = model.blocks[li]
    g = torch.Generator(device=cuda).manual_seed(11)
    x = torch.randn(T, d, device=cuda, generator=g).bfloat16()
    dh1 = (torch.randn(T, d, device=cuda, generator=g) * 0.1).bfloat16()
    step.T, step.packed = T, batch
    sv = {}
    h1 = step._attn_fwd(li, blk, x, sv)
    ad.g.zero_()
    dx = step._attn_bwd(li, blk, x, sv, dh1)
    torch.cuda.synchronize()
    Hq, Hkv, r, s = cfg.attn_heads, cfg.attn_kv_heads, cfg.rank, cfg.lora_scale
    inv, amp = ref.rope_frequencies(rot, cfg.rope_theta, scaling)
    ang = batch.plan.pos.double()[:, None] * torch.tensor(inv, dtype=torch.float64, device=cuda)
    cos, sin = (amp * torch.cos(ang)).float(), (amp * torch.sin(ang)).float()
    leaves = []

    def lin(xin, grp):
        W = torch.cat([IQ.dequant_bf16(w).float() for w in grp.iqr], 0)
        A = ad.a_view(ad.w, grp).detach().clone().requires_grad_(True)
        Bs = [ad.b_view(ad.w, grp, i).detach().clone().requires_grad_(True) for i in range(len(grp.projs))]
        leaves.append((grp, A, Bs))
        t = xin @ A.t()
        return xin @ W.t() + s * torch.cat([t[:, i * r:(i + 1) * r] @ B.t() for i, B in enumerate(Bs)], 1)

    def rms(v, w):
        return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + cfg.eps) * w

    xf = x.float().requires_grad_(True)
    y = lin(rms(xf, blk["w_in"]), blk["groups"][0])
    q, k, v = step._qkv_views(y)
    gate = y[:, :2 * Hq * Dh].view(T, Hq, 2 * Dh)[:, :, Dh:]
    q = ref.rotate(rms(q, blk["q_norm"]), cos, sin, interleaved)
    k = ref.rotate(rms(k, blk["k_norm"]), cos, sin, interleaved)
    outs = []
    for a, b in ref.spans(lens):
        n = b - a
        sc = torch.einsum("thd,shd->hts", q[a:b], k[a:b].repeat_interleave(Hq // Hkv, 1)) / math.sqrt(Dh)
        sc = sc.masked_fill(torch.ones(n, n, dtype=torch.bool, device=cuda).triu(1), -math.inf)
        outs.append(torch.einsum("hts,shd->thd", torch.softmax(sc, -1), v[a:b].repeat_interleave(Hq // Hkv, 1)))
    ga = (torch.cat(outs) * torch.sigmoid(gate)).reshape(T, Hq * Dh)
    want = xf + lin(ga, blk["groups"][1])
    want.backward(dh1.float())
    assert_close_bf16(to_np(h1), to_np(want), what="h1")
    assert_close_bf16(to_np(dx), to_np(xf.grad), what="dx")
    for grp, A, Bs in leaves:
        assert_close_bf16(to_np(ad.a_view(ad.g, grp)), to_np(A.grad), what=f"dA {grp.name}")
        for i, B in enumerate(Bs):
            assert_close_bf16(to_np(ad.b_view(ad.g, grp, i)), to_np(B.grad), what=f"dB {grp.name}.{i}")


def test_packed_refusals(cuda):
    cfg, model, ad, step = _fresh(cuda)
    with pytest.raises(R97bError):
        PackedBatch(model, [0, cfg.seq + 1])   # beyond the rotary table
    with pytest.raises(R97bError):
        PackedBatch(model, [0, 0])
    with pytest.raises(R97bError):
        PackedBatch(model, [0, 5, 3])
    batch = PackedBatch(model, [0, 5, 9])
    with pytest.raises(R97bError):
        step.run(_ids(cuda, 8, cfg.vocab, 1), batch=batch)
    with pytest.raises(R97bError):
        step.run(_ids(cuda, 9, cfg.vocab, 1), _ids(cuda, 8, cfg.vocab, 1), batch=batch)
    assert step.packed is None and step.T == cfg.tokens
    cfg, model, ad, step = _fresh(cuda, rope_interleaved=True)
    with pytest.raises(R97bError):  # the fixed frame's rotation takes neighbouring halves
        step.run(_ids(cuda, cfg.tokens, cfg.vocab, 1))
