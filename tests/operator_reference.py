"""The added operators written from their definitions in float64, and bounds on how far a kernel's rounding may take it.

HALF is half a step of bf16 relative to the value (2^-8): what one rounding to bf16 may be off by.
"""
import math

import torch

HALF = torch.finfo(torch.bfloat16).eps / 2


def within(got, ref, slack, what):
    """|got - ref| <= HALF |ref| (the output's one rounding) + slack, element by element; NaN nowhere."""
    got, ref = got.double().cpu(), ref.double().cpu()
    slack = slack.double().cpu() if torch.is_tensor(slack) else slack
    # from 2^128 (1 - 2^-9) on a value rounds to infinity
    beyond = torch.isinf(got) & (got.sign() == ref.sign()) & (ref.abs() + slack >= 2.0 ** 128 * (1 - 2.0 ** -9))
    off = torch.where(beyond, 0.0, (got - ref).abs() - (HALF * ref.abs() + slack))
    # the smallest bf16 step, for values that round to subnormals
    bad = ~(off <= 2.0 ** -133)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, by up to {off.max().item():.3e} more than the bound"


# ---- q/k norm with rotation ----------------------------------------------------------------------------------------
def rotate(x, pos, theta, sign=1):
    """x [T][H][hd] turned by sign * pos * theta^(-2i / hd) in interleaved pairs."""
    hd = x.shape[-1]
    a = pos.double()[:, None] * theta ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=x.device) / hd)
    c, s = torch.cos(a)[:, None], sign * torch.sin(a)[:, None]
    e, o = x[..., 0::2], x[..., 1::2]
    return torch.stack([c * e - s * o, c * o + s * e], -1).flatten(-2)


def norm_rope(x, w, pos, theta, eps, hd):
    x = x.double().view(x.shape[0], -1, hd)
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    return rotate(n if w is None else n * w.double(), pos, theta).flatten(1), n


def norm_rope_bwd(x, w, dy, pos, theta, eps, hd):
    x = x.double().view(x.shape[0], -1, hd)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x * r
    g = rotate(dy.double().view(x.shape), pos, theta, -1)
    a = g if w is None else g * w.double()
    c = (a * n).mean(-1, keepdim=True)
    dx = r * (a - n * c)
    size = (r * (a.abs().amax(-1, keepdim=True) + n.abs().amax(-1, keepdim=True) * (a * n).abs().mean(-1, keepdim=True))).expand_as(x)
    return dx.flatten(1), (g * n).sum((0, 1)), (g * n).abs().sum((0, 1)), size.flatten(1)


# ---- attention with a window and sinks -------------------------------------------------------------------------------
def window_mask(n, t, window, sinks, device):
    p = torch.arange(t - n, t, device=device)[:, None]
    j = torch.arange(t, device=device)[None, :]
    return (j <= p) & ((p - j < window) | (j < sinks))


def window_attention(q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q, k, v, window, sinks, do=None, o_given=None):
    """dict of o, lse and their slack (what the rounding of probabilities to bf16 may add), with `do` also dq, dk, dv and theirs.
    o_given: the output the backward forms delta from. Masked keys are never multiplied: they may hold anything."""
    z = lambda x: torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    r = {"o": z(q), "o_slack": z(q), "lse": torch.zeros((hq, q.shape[0]), dtype=torch.float64, device=q.device)}
    if do is not None:
        for name, x in (("dq", q), ("dk", k), ("dv", v)):
            r[name], r[name + "_slack"] = z(x), z(x)
    for qo, n, ko, t in zip(q_offs, q_lens, k_offs, k_lens):
        if n == 0 or t == 0:
            continue
        see = window_mask(n, t, window, sinks, q.device)
        used = see.any(0)  # keys that some query sees
        for h in range(hq):
            c, g = slice(h * hd, (h + 1) * hd), h // (hq // hkv)
            ck = slice(g * hd, (g + 1) * hd)
            Q = q[qo:qo + n, c].double()
            K = torch.where(used[:, None], k[ko:ko + t, ck].double(), 0.0)
            V = torch.where(used[:, None], v[ko:ko + t, ck].double(), 0.0)
            s = torch.where(see, Q @ K.T / math.sqrt(hd), -math.inf)
            lse = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[:, None])
            o = p @ V
            r["o"][qo:qo + n, c], r["lse"][h, qo:qo + n] = o, lse
            r["o_slack"][qo:qo + n, c] = 1.02 * HALF * (p @ V.abs())
            if do is None:
                continue
            dO = do[qo:qo + n, c].double()
            delta = (dO * (o if o_given is None else o_given[qo:qo + n, c].double())).sum(1, keepdim=True)
            dp = dO @ V.T
            ds = p * (dp - delta) / math.sqrt(hd)
            # dS is rounded once to bf16; its fp32 error: 2^-14 of the terms that are subtracted
            err = HALF * ds.abs() + 2.0 ** -14 * p * (dO.abs() @ V.abs().T + (dO.abs() * o.abs()).sum(1, keepdim=True)) / math.sqrt(hd)
            r["dq"][qo:qo + n, c] = ds @ K
            r["dq_slack"][qo:qo + n, c] = 1.02 * (err @ K.abs())
            r["dk"][ko:ko + t, ck] += ds.T @ Q
            r["dk_slack"][ko:ko + t, ck] += 1.02 * (err.T @ Q.abs())
            r["dv"][ko:ko + t, ck] += p.T @ dO
            # probabilities below 2^-126 are formed as 0 (the exponential's results are never subnormal)
            r["dv_slack"][ko:ko + t, ck] += 1.02 * HALF * (p.T @ dO.abs()) + 2.0 ** -126 * dO.abs().sum(0)
    return r


# ---- 8-bit values ------------------------------------------------------------------------------------------------------
def held8(x):
    """What x stands for after e4m3 rounding with a power of two per 32 columns; infinities and NaN become NaN."""
    x = x.double()
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], 32):
        b = x[:, c:c + 32]
        fine = torch.where(torch.isfinite(b), b.abs(), 0.0).amax(1, keepdim=True)
        m, e = torch.frexp(fine.clamp(min=1e-300) / 448)  # a power of two itself has m = 1/2
        unit = torch.exp2(torch.where(m > 0.5, e, e - 1).clamp(min=-124).double())
        v = torch.where(unit == 2.0 ** 120, (b / unit).clamp(-240, 240), b / unit)  # 256 * 2^120 is no bf16 number
        step = torch.exp2(torch.frexp(v.abs().clamp(min=2.0 ** -6))[1].double() - 4)
        out[:, c:c + 32] = torch.where(torch.isfinite(b), torch.round(v / step) * step * unit, math.nan)
    return out


def swiglu(a, b):
    return a / (1 + torch.exp(-a)) * b


def swiglu_bwd(a, b, dh):
    g = 1 / (1 + torch.exp(-a))
    return dh * b * g * (1 + a * (1 - g)), dh * a * g
