"""Timed cases of the packed-sequence training operators: rotary positions (with the q/k RMS norm) and causal
grouped-query attention over ragged sequences laid end to end, each forward and backward.

`run` makes the framework's calls when `own` is true and computes the same results in elementary torch operations
otherwise; `exact` restates the operators in 64 bits.
"""
import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
THETA = 1e7


# ------------------------------------------------------------------------------------------------ cases

def listed():
    """Shapes: the 9B-class step's attention layers (16 query heads over 4 key/value heads of 256, 64 rotated), the small
    hybrid's (8 over 2 of 128, 64 rotated), and a fully rotated interleaved 128 head for long contexts."""
    big = dict(hq=16, hkv=4, d=256, rot=64, layout="half", scaling="none")
    small = dict(hq=8, hkv=2, d=128, rot=64, layout="half", scaling="none")
    long = dict(hq=16, hkv=4, d=128, rot=128, layout="interleaved", scaling="yarn")
    return [
        # a handful of short turns: launch latency
        dict(name="rope_turns", op="rope", back=False, lens="1,9,30", **small),
        # one step's tokens of the 9B-class model, forward and adjoint
        dict(name="rope_step", op="rope", back=False, lens="4096,4096", **big),
        dict(name="rope_step_back", op="rope", back=True, lens="4096,4096", **big),
        # one long document with scaled positions, adjoint
        dict(name="rope_long_back", op="rope", back=True, lens="32749", **long),
        # evaluation of a handful of short turns: launch latency
        dict(name="attn_turns", op="attn", back=False, lens="1,9,30", **small),
        # a token-budget batch of chat conversations, small hybrid
        dict(name="attn_chat", op="attn", back=False, lens=_chat(8192, 5), **small),
        # one attention layer of the 9B-class step
        dict(name="attn_step", op="attn", back=False, lens="4096,4096", **big),
        # training on a handful of short turns
        dict(name="train_turns", op="attn", back=True, lens="1,9,130", **big),
        # training on a token-budget batch of chat conversations, both models' heads
        dict(name="train_chat_128", op="attn", back=True, lens=_chat(16384, 6), **small),
        dict(name="train_chat_256", op="attn", back=True, lens=_chat(8192, 7), **big),
        # one attention layer of the 9B-class step, forward and backward
        dict(name="train_step", op="attn", back=True, lens="4096,4096", **big),
        # one long document of an odd length
        dict(name="train_long", op="attn", back=True, lens="12301", **long),
    ]


def _chat(budget, seed):
    """Lengths of one token-budget batch of conversations: log-uniform between 16 and 2048 tokens, filled to `budget`."""
    import random
    rng = random.Random(seed)
    lens, left = [], budget
    while left > 0:
        n = min(left, int(round(math.exp(rng.uniform(math.log(16), math.log(2048))))))
        lens.append(n)
        left -= n
    return ",".join(str(n) for n in lens)


def draw(rng):
    hkv = rng.choice([1, 2, 4])
    d = rng.choice([128, 256])
    case = dict(op=rng.choice(["rope", "attn", "attn"]), back=rng.random() < 0.6, hq=hkv * rng.choice([1, 2, 3, 4]),
                hkv=hkv, d=d, rot=rng.choice([16, 32, 64, 128]), layout=rng.choice(["half", "interleaved"]),
                scaling=rng.choice(["none", "linear", "yarn"]))
    total = int(round(math.exp(rng.uniform(math.log(8), math.log(9000)))))
    if rng.random() < 0.3:
        lens = [total]
    else:  # a few cuts at any token; cuts that meet leave an empty sequence, which a batch may hold
        cuts = sorted(rng.randrange(total + 1) for _ in range(rng.randrange(1, 12)))
        lens = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    case["lens"] = ",".join(str(n) for n in lens)
    return case


def _lens(case):
    return [int(n) for n in case["lens"].split(",")]


def _pairs(case):
    return sum(n * (n + 1) // 2 for n in _lens(case))


def work(case):
    tokens, d, hq, hkv, rot = sum(_lens(case)), case["d"], case["hq"], case["hkv"], case["rot"]
    heads = hq + hkv
    if case["op"] == "rope":
        row = 2 * d * tokens * heads
        table = 2 * 4 * (rot // 2) * max(_lens(case)) + 2 * 4 * d + 4 * tokens
        flops = tokens * heads * (4 * d + 3 * rot) * (2 if case["back"] else 1)
        return {"bytes": row * (3 if case["back"] else 2) + table, "flops": flops}
    q, kv, lse = 2 * d * hq * tokens, 2 * d * hkv * tokens, 4 * hq * tokens
    if not case["back"]:
        return {"bytes": 2 * q + 2 * kv + lse, "flops": 4 * d * hq * _pairs(case)}
    # forward, then S again, dP, dV, dK and dQ
    return {"bytes": 4 * q + 4 * kv + lse, "flops": 14 * d * hq * _pairs(case)}


# ------------------------------------------------------------------------------------------------ inputs

def _scaling(case):
    if case["scaling"] == "linear":
        return {"type": "linear", "factor": 4.0}
    if case["scaling"] == "yarn":
        return {"type": "yarn", "factor": 8.0, "original": 4096, "beta_fast": 32.0, "beta_slow": 1.0}
    return None


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed * 1000003 + 17)
    lens, d, hq, hkv = _lens(case), case["d"], case["hq"], case["hkv"]
    T = sum(lens)

    def rand(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=DEVICE) * std).to(torch.bfloat16)

    s = {}
    if case["op"] == "rope":
        # the fused projection's rows: each query head beside its output gate, then the keys, then the values
        s["y"] = rand(T, 2 * hq * d + 2 * hkv * d)
        s["wq"] = 1.0 + 0.1 * torch.randn(d, generator=g, device=DEVICE)
        s["wk"] = 1.0 + 0.1 * torch.randn(d, generator=g, device=DEVICE)
        if case["back"]:
            s["dq"], s["dk"] = rand(T, hq, d, std=0.1), rand(T, hkv, d, std=0.1)
    else:
        # queries and keys as the norm leaves them: rows of length sqrt(d)
        s["q"], s["k"] = rand(T, hq, d), rand(T, hkv, d)
        s["y"] = rand(T, 2 * hkv * d)  # the values are read inside the projection's wider rows
        if case["back"]:
            s["do"] = rand(T, hq, d, std=0.1)
    return s


def _qk_views(y, case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    q = y[:, :2 * hq * d].view(-1, hq, 2 * d)[:, :, :d]
    k = y[:, 2 * hq * d:2 * hq * d + hkv * d].view(-1, hkv, d)
    return q, k


def _v_view(y, case):
    hkv, d = case["hkv"], case["d"]
    return y[:, hkv * d:].view(-1, hkv, d)


def prepare(case, seed):
    st = dict(case=case, **_inputs(case, seed))
    lens = _lens(case)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    st["cu"] = cu
    if case["op"] == "rope":
        st["q"], st["k"] = _qk_views(st["y"], case)
        if case["back"]:  # the projection's cotangent, whose other columns other operators fill
            st["dy"] = torch.zeros_like(st["y"])
            st["dyq"], st["dyk"] = _qk_views(st["dy"], case)
    else:
        st["v"] = _v_view(st["y"], case)
    if own:
        from r97training_b200 import ops
        from r97training_b200.packed import PackedPlan
        st["ops"] = ops
        st["plan"] = PackedPlan(cu, DEVICE)
        if case["op"] == "rope":
            st["cos"], st["sin"] = ops.rope_tables(max(lens), case["rot"], THETA, scaling=_scaling(case), device=DEVICE)
        elif case["back"]:
            st["ws"] = ops.attn_packed_bwd_workspace(st["plan"], case["hq"], case["hkv"], case["d"])
    elif case["op"] == "rope":
        st["cos"], st["sin"] = _tables(case, max(lens))
        st["pos"] = torch.cat([torch.arange(n, device=DEVICE) for n in lens])
    return st


# ------------------------------------------------------------------------------------------------ plain form

def _tables(case, n_pos):
    """cos and sin of pos * inv_i, angles in 64 bits."""
    rot, half = case["rot"], case["rot"] // 2
    i = torch.arange(half, dtype=torch.float64, device=DEVICE)
    inv = THETA ** (-2.0 * i / rot)
    sc, mult = _scaling(case), 1.0
    if sc and sc["type"] == "linear":
        inv = inv / sc["factor"]
    elif sc:
        def turns_dim(turns):
            return rot * math.log(sc["original"] / (turns * 2.0 * math.pi)) / (2.0 * math.log(THETA))
        low = max(math.floor(turns_dim(sc["beta_fast"])), 0)
        high = min(math.ceil(turns_dim(sc["beta_slow"])), half - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        inv = inv * (1.0 - ramp) + inv / sc["factor"] * ramp
        mult = 0.1 * math.log(sc["factor"]) + 1.0
    ang = torch.arange(n_pos, dtype=torch.float64, device=DEVICE)[:, None] * inv[None, :]
    return (torch.cos(ang) * mult).float(), (torch.sin(ang) * mult).float()


def _rotate(x, cos, sin, rot, layout, sign=1.0):
    half = rot // 2
    if layout == "half":
        a, b = x[..., :half], x[..., half:rot]
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    c, s = cos[:, None, :], sin[:, None, :] * sign
    ra, rb = a * c - b * s, b * c + a * s
    out = x.clone()
    if layout == "half":
        out[..., :half], out[..., half:rot] = ra, rb
    else:
        out[..., 0:rot:2], out[..., 1:rot:2] = ra, rb
    return out


def _plain_rope(st):
    case = st["case"]
    cos, sin = st["cos"][st["pos"]], st["sin"][st["pos"]]
    outs = []
    for name, w in (("q", st["wq"]), ("k", st["wk"])):
        x = st[name].float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        if not case["back"]:
            outs.append(_rotate(x * r * w, cos, sin, case["rot"], case["layout"]).to(torch.bfloat16))
            continue
        d = _rotate(st["d" + name].float(), cos, sin, case["rot"], case["layout"], -1.0) * w
        dx = r * d - x * r * r * r * (d * x).mean(-1, keepdim=True)
        st["dy" + name].copy_(dx)
        outs.append(st["dy" + name])
    return outs


def _plain_attn(st):
    case = st["case"]
    hq, hkv, d, back = case["hq"], case["hkv"], case["d"], case["back"]
    grp, scale = hq // hkv, 1.0 / math.sqrt(d)
    q, k, v = st["q"], st["k"], st["v"]
    T = q.shape[0]
    o = torch.empty((T, hq, d), dtype=torch.bfloat16, device=q.device)
    lse = torch.empty((hq, T), dtype=torch.float32, device=q.device)
    if back:
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(k)
    for b0, b1 in zip(st["cu"], st["cu"][1:]):
        n = b1 - b0
        if n == 0:
            continue
        later = torch.ones((n, n), dtype=torch.bool, device=q.device).triu(1)
        for g in range(hkv):
            h = slice(g * grp, (g + 1) * grp)
            qf = q[b0:b1, h].float().transpose(0, 1)                       # [grp, n, d]
            kf, vf = k[b0:b1, g].float(), v[b0:b1, g].float()              # [n, d]
            s = (torch.matmul(qf, kf.t()) * scale).masked_fill(later, float("-inf"))
            m = s.max(-1, keepdim=True).values
            p = torch.exp(s - m)
            del s
            l = p.sum(-1, keepdim=True)
            p = p / l
            of = torch.matmul(p, vf)
            o[b0:b1, h] = of.transpose(0, 1).to(torch.bfloat16)
            lse[h, b0:b1] = (m + torch.log(l)).squeeze(-1)
            if back:
                do = st["do"][b0:b1, h].float().transpose(0, 1)
                dv[b0:b1, g] = torch.matmul(p.transpose(1, 2), do).sum(0).to(torch.bfloat16)
                delta = (do * of).sum(-1, keepdim=True)
                ds = p * (torch.matmul(do, vf.t()) - delta) * scale
                dq[b0:b1, h] = torch.matmul(ds, kf).transpose(0, 1).to(torch.bfloat16)
                dk[b0:b1, g] = torch.matmul(ds.transpose(1, 2), qf).sum(0).to(torch.bfloat16)
                del ds
            del p
    return [o, lse, dq, dk, dv] if back else [o, lse]


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    if not own:
        return _plain_rope(state) if case["op"] == "rope" else _plain_attn(state)
    ops, plan = state["ops"], state["plan"]
    if case["op"] == "rope":
        inter = case["layout"] == "interleaved"
        if case["back"]:
            ops.qk_rope_bwd([(state["q"], state["wq"], state["dq"], state["dyq"]),
                             (state["k"], state["wk"], state["dk"], state["dyk"])],
                            state["cos"], state["sin"], plan.pos, interleaved=inter, eps=EPS)
            return [state["dyq"], state["dyk"]]
        return list(ops.qk_rope_fwd([(state["q"], state["wq"]), (state["k"], state["wk"])], state["cos"], state["sin"],
                                    plan.pos, interleaved=inter, eps=EPS))
    scale = 1.0 / math.sqrt(case["d"])
    q, k, v = state["q"], state["k"], state["v"]
    o, lse = ops.attn_packed_fwd(q, k, v, plan, scale)
    if not case["back"]:
        return [o, lse]
    dq, dk, dv = ops.attn_packed_bwd(q, k, v, o, state["do"], lse, plan, scale, state["ws"])
    return [o, lse, dq, dk, dv]


# ------------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_rope(case, s) if case["op"] == "rope" else _exact_attn(case, s)


def _exact_rope(case, s):
    rot, d = case["rot"], case["d"]
    half = rot // 2
    sc = _scaling(case)
    # the angle of pair i at position p: p / (theta^(2 i / rot)), and its scaled forms
    freq = [math.pow(THETA, -2.0 * i / rot) for i in range(half)]
    amp = 1.0
    if sc is not None and sc["type"] == "linear":
        freq = [f / sc["factor"] for f in freq]
    elif sc is not None:
        def at(turns):  # the (real) pair whose wavelength turns `turns` times over the original length
            return rot * math.log(sc["original"] / (2.0 * math.pi * turns)) / (2.0 * math.log(THETA))
        lo, hi = max(math.floor(at(sc["beta_fast"])), 0), min(math.ceil(at(sc["beta_slow"])), half - 1)
        keep = [1.0 - min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for i in range(half)]
        freq = [f * w + f / sc["factor"] * (1.0 - w) for f, w in zip(freq, keep)]
        amp = 1.0 + 0.1 * math.log(sc["factor"])
    pos = torch.tensor([p for n in _lens(case) for p in range(n)], dtype=torch.float64, device=DEVICE)
    ang = pos[:, None] * torch.tensor(freq, dtype=torch.float64, device=DEVICE)
    rotor = torch.polar(torch.full_like(ang, amp), ang)[:, None, :]
    first = list(range(half)) if case["layout"] == "half" else list(range(0, rot, 2))
    second = [i + half for i in first] if case["layout"] == "half" else [i + 1 for i in first]

    def turn(x, z):
        c = torch.complex(x[..., first], x[..., second]) * z
        y = x.clone()
        y[..., first], y[..., second] = c.real, c.imag
        return y

    out = []
    for x, w, dy in zip(_qk_views(s["y"], case), (s["wq"], s["wk"]), (s.get("dq"), s.get("dk"))):
        x, w = x.double(), w.double()
        rms = torch.sqrt(x.pow(2).sum(-1, keepdim=True) / d + EPS)
        if dy is None:
            out.append(turn(x / rms * w, rotor))
        else:
            g = turn(dy.double(), rotor.conj()) * w
            out.append((g - x * (g * x).sum(-1, keepdim=True) / (d * rms * rms)) / rms)
    return out


def _exact_attn(case, s):
    hq, hkv, d, back = case["hq"], case["hkv"], case["d"], case["back"]
    lens = _lens(case)
    if _pairs(case) * hq * d > 16e11:  # the score matrices would take too long in 64 bits
        return None
    T = sum(lens)
    v_all = _v_view(s["y"], case)
    z = dict(dtype=torch.float64, device=DEVICE)
    o, lse, dq = torch.zeros(T, hq, d, **z), torch.zeros(hq, T, **z), torch.zeros(T, hq, d, **z)
    dk, dv = torch.zeros(T, hkv, d, **z), torch.zeros(T, hkv, d, **z)
    start = 0
    for n in lens:
        rows = slice(start, start + n)
        start += n
        if n == 0:
            continue
        seen = torch.ones(n, n, dtype=torch.bool, device=DEVICE).tril()
        for h in range(hq):
            g = h // (hq // hkv)
            qh, kh, vh = s["q"][rows, h].double(), s["k"][rows, g].double(), v_all[rows, g].double()
            a = torch.where(seen, qh @ kh.T / math.sqrt(d), torch.full((), -math.inf, **z))
            norm = torch.logsumexp(a, 1)
            a = torch.exp(a - norm[:, None])
            lse[h, rows] = norm
            o[rows, h] = a @ vh
            if back:
                doh = s["do"][rows, h].double()
                dv[rows, g] += a.T @ doh
                a = a * (doh @ vh.T - (doh * o[rows, h]).sum(1, keepdim=True)) / math.sqrt(d)
                dq[rows, h] = a @ kh
                dk[rows, g] += a.T @ qh
    return [o, lse, dq, dk, dv] if back else [o, lse]
