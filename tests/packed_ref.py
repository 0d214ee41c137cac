"""Plain 64-bit forms of the packed-sequence operators (rotary positions, causal GQA attention and its backward), with
elementwise bounds on what a bf16 kernel with f32 sums may be off by.

u = 2^-8 is half a bf16 step relative to the value: what one rounding to bf16 costs. The kernels round the probabilities
and dS to bf16 before the second products, and each output once."""
import math

import torch

U = 2.0 ** -8    # one rounding to bf16
E32 = 2.0 ** -24  # one rounding to f32


def spans(lens):
    out, t = [], 0
    for n in lens:
        out.append((t, t + n))
        t += n
    return out


def attention(q, k, v, lens, scale, dout=None, o_in=None, lse_in=None):
    """f64 (o, lse) and, with dout, (dq, dk, dv), each with its bound: a dict name -> (value, bound). The backward
    follows the operator's definition on the given o and lse (o_in, lse_in), or the forward's own in 64 bits, with
    the bound widened by what a bf16 o costs its row sums."""
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    grp = Hq // Hkv
    z = dict(dtype=torch.float64, device=q.device)
    f = lambda t: t.double()  # noqa: E731
    val = {n: torch.zeros(s, **z) for n, s in (("o", (T, Hq, D)), ("lse", (Hq, T)), ("dq", (T, Hq, D)),
                                               ("dk", (T, Hkv, D)), ("dv", (T, Hkv, D)))}
    err = {n: torch.zeros_like(t) for n, t in val.items()}
    for b0, b1 in spans(lens):
        n = b1 - b0
        if n == 0:
            continue
        seen = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        for h in range(Hq):
            g = h // grp
            qh, kh, vh = f(q[b0:b1, h]), f(k[b0:b1, g]), f(v[b0:b1, g])
            x = (qh @ kh.T * scale).masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(x, 1)
            # the scores: D products summed in f32 in any order, scaled and moved to base 2 (a few more roundings of
            # the score and of the row's maximum or lse), then exp2 to 2 f32 steps
            mag = (qh.abs() @ kh.abs().T) * abs(scale)
            es = (D + 4) * E32 * mag + 8 * E32 * (x.masked_fill(~seen, 0).abs() + lse.abs()[:, None]) + 8 * E32
            es = es.masked_fill(~seen, 0)
            p = torch.exp(x - lse[:, None])
            A = p @ vh.abs()
            o = p @ vh
            # a sum of n f32 terms is off by at most n roundings of their magnitudes' sum; the row's own sum divides
            rel = es.amax(1, keepdim=True) * 2 + n * E32
            o_err = U * A + U * o.abs() + rel * A * 2
            val["o"][b0:b1, h], err["o"][b0:b1, h] = o, o_err
            val["lse"][h, b0:b1], err["lse"][h, b0:b1] = lse, rel[:, 0] + 8 * E32 * lse.abs()
            if dout is None:
                continue
            do = f(dout[b0:b1, h])
            if o_in is None:
                delta, d_err = (do * o).sum(1, keepdim=True), (do.abs() * o_err).sum(1, keepdim=True)
            else:
                ob = f(o_in[b0:b1, h])
                delta, d_err = (do * ob).sum(1, keepdim=True), D * E32 * (do * ob).abs().sum(1, keepdim=True)
            if lse_in is not None:
                p = torch.exp(x - f(lse_in[h, b0:b1])[:, None])
            dv = p.T @ do
            val["dv"][b0:b1, g] += dv
            err["dv"][b0:b1, g] += (p * (U + es + n * grp * E32)).T @ do.abs()
            dp = do @ vh.T
            # a sequence's first 128 rows take the row sum of p dp, its equal, from products summed in f32
            first = (p * dp).sum(1, keepdim=True)
            f_err = (p * (es * dp.abs() + (D + n) * E32 * (do.abs() @ vh.abs().T))).sum(1, keepdim=True)
            head = (torch.arange(n, device=q.device) < 128)[:, None]
            delta, d_err = torch.where(head, first, delta), torch.where(head, f_err, d_err)
            ds = p * (dp - delta)
            ds_err = U * ds.abs() + es * p * (dp.abs() + delta.abs()) + p * (
                d_err + (D + 2) * E32 * (do.abs() @ vh.abs().T) + 2 * E32 * delta.abs())
            ds_err = ds_err + n * grp * E32 * ds.abs()
            val["dq"][b0:b1, h] = ds @ kh * scale
            err["dq"][b0:b1, h] = (ds_err @ kh.abs()) * abs(scale)
            val["dk"][b0:b1, g] += ds.T @ qh * scale
            err["dk"][b0:b1, g] += (ds_err.T @ qh.abs()) * abs(scale)
    for n in ("dq", "dk", "dv"):
        err[n] += U * val[n].abs()
    # a bf16 result in its subnormal range, or an f32 one flushed to zero, is off by less than this
    return {n: (val[n], err[n] + 1e-30) for n in val if dout is not None or n in ("o", "lse")}


def assert_within(got, want, what):
    value, bound = want
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - value).abs() - bound
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0, (f"{what}: off by {float((got - value).abs().flatten()[over.argmax()]):.3e} where "
                        f"{float(bound.flatten()[over.argmax()]):.3e} is allowed")


def rope_frequencies(rot, theta, scaling=None):
    """(pair frequencies, amplitude) in f64 Python arithmetic."""
    half = rot // 2
    inv, amp = [theta ** (-2.0 * i / rot) for i in range(half)], 1.0
    if scaling and scaling["type"] == "linear":
        inv = [f / scaling["factor"] for f in inv]
    elif scaling:
        def pair(turns):
            return rot * math.log(scaling["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low = max(math.floor(pair(scaling.get("beta_fast", 32.0))), 0)
        high = min(math.ceil(pair(scaling.get("beta_slow", 1.0))), half - 1)
        ramp = [min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(half)]
        inv = [f * (1 - r) + f / scaling["factor"] * r for f, r in zip(inv, ramp)]
        amp = 0.1 * math.log(scaling["factor"]) + 1.0
    return inv, amp


def rotate(x, cos, sin, interleaved, inverse=False):
    """x [T, heads, D] f64, cos and sin [T, rot / 2]: the first rot dims rotated in pairs."""
    half = cos.shape[1]
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    c, s = cos[:, None], -sin[:, None] if inverse else sin[:, None]
    y = x.clone()
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    return y


def rope_fwd(x, w, cos, sin, interleaved, eps):
    x = x.double()
    n = x if w is None else x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    return rotate(n, cos.double(), sin.double(), interleaved)


def rope_bwd(x, w, dout, cos, sin, interleaved, eps):
    d = rotate(dout.double(), cos.double(), sin.double(), interleaved, inverse=True)
    if w is None:
        return d
    x, d = x.double(), d * w.double()
    r = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    return r * d - x * r ** 3 * (d * x).mean(-1, keepdim=True)
