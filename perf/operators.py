"""The operators around a decoder block's attention and feed-forward that this library adds to the block's other ops, as
cases that can be timed and checked: per-head RMSNorm of queries and keys with the position rotation, attention with a
sliding window and sink tokens, and SwiGLU activations held in 8 bits between the forward and the backward. Every
operator is written here in plain torch (`own` false) and as the call a user makes of the library (`own` true); `exact`
evaluates the same definitions in float64.

Sizes: 16 query / 4 key-value heads of 128, theta 500000 and 8192 tokens are the decoder configuration of bench.py;
1408 columns and 65536 routed rows (8192 tokens, top-8) its MoE layer; the others are generic.
"""
import math

import numpy as np
import torch

own = False

BF = torch.bfloat16
EPS = 1e-5
THETA = 500000


def listed():
    return [
        # queries and keys of one step of 24 sequences that are being continued far into a long text
        {"name": "qk_decode_far", "op": "qk", "tokens": 24, "hq": 16, "hkv": 4, "hd": 128, "far": True, "weighted": True, "train": False},
        # a ragged batch with small heads, forward only (evaluation), no norm weights (config.txt's "QK Norm Weight Type: none")
        {"name": "qk_eval_hd64", "op": "qk", "tokens": 4097, "hq": 24, "hkv": 8, "hd": 64, "far": False, "weighted": False, "train": False},
        # the decoder configuration's training step, one layer, forward and backward
        {"name": "qk_train", "op": "qk", "tokens": 8192, "hq": 16, "hkv": 4, "hd": 128, "far": False, "weighted": True, "train": True},
        # one new token of one sequence: latency
        {"name": "window_one_token", "op": "window", "q": "1", "k": "2500", "hq": 16, "hkv": 4, "hd": 128, "window": 1024, "sinks": 4, "train": False},
        # one new token (or two) of each of 32 sequences of very different lengths
        {"name": "window_tokens_of_32", "op": "window", "q": "1,1,1,2,1,1,1,1,1,1,1,1,1,1,2,1,1,1,1,1,1,1,1,1,1,1,1,1,1,1,1,1",
         "k": "9000,4097,1,2,15000,800,64,12345,7000,5100,4096,333,16000,8192,127,2048,6001,11000,95,4500,9999,1500,3500,14001,10,5000,7777,250,13000,6400,4099,700",
         "hq": 16, "hkv": 4, "hd": 128, "window": 4096, "sinks": 4, "train": False},
        # evaluation of long prompts in chunks: the queries are the last tokens of their sequences
        {"name": "window_chunked_prompt", "op": "window", "q": "2048,777,130", "k": "9300,777,1154", "hq": 16, "hkv": 4, "hd": 128, "window": 2048, "sinks": 4, "train": False},
        # the decoder configuration's training step, one layer
        {"name": "window_train", "op": "window", "q": "8192", "k": "8192", "hq": 16, "hkv": 4, "hd": 128, "window": 1024, "sinks": 4, "train": True},
        # packed documents of ragged lengths, heads of 64 without sharing, a short window
        {"name": "window_train_ragged_hd64", "op": "window", "q": "2900,1,1717,40,129,513", "k": "2900,1,1717,40,129,513", "hq": 8, "hkv": 8, "hd": 64, "window": 500, "sinks": 17, "train": True},
        # few routed rows: latency
        {"name": "act8_few_rows", "op": "act8", "rows": 96, "cols": 1408, "use": "restore"},
        # an odd number of rows, columns that end inside a scale block
        {"name": "act8_restore_odd", "op": "act8", "rows": 10007, "cols": 1000, "use": "restore"},
        # the MoE layer's x1 and x3: kept by the forward, read by the backward
        {"name": "act8_layer_backward", "op": "act8", "rows": 65536, "cols": 1408, "use": "backward"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qk", "window", "window", "window", "act8"])
    if op == "qk":
        hq, hkv = rng.choice([(16, 4), (24, 8), (8, 8), (6, 2), (5, 1), (32, 4)])
        hd = rng.choice([64, 128, 128, 256, 32])
        most = 8192 * 20 * 128 // ((hq + hkv) * hd)
        return {"op": "qk", "tokens": _log(rng, 1, most), "hq": hq, "hkv": hkv, "hd": hd, "far": rng.random() < 0.4,
                "weighted": rng.random() < 0.7, "train": rng.random() < 0.6}
    if op == "act8":
        cols = 8 * _log(rng, 4, 512)
        return {"op": "act8", "rows": _log(rng, 1, 65536 * 1408 // cols), "cols": cols, "use": rng.choice(["restore", "backward"])}
    hq, hkv = rng.choice([(16, 4), (16, 16), (8, 1), (12, 4), (10, 2), (4, 4), (14, 7)])
    hd = rng.choice([64, 128, 128])
    case = {"op": "window", "hq": hq, "hkv": hkv, "hd": hd, "sinks": rng.choice([0, 1, 4, 4, 16, 33, 130])}
    if rng.random() < 0.35:  # a few new tokens of sequences of any length
        n = _log(rng, 1, 48)
        q = [rng.choice([1, 1, 1, 1, 2, 3]) for _ in range(n)]
        k = [max(a, _log(rng, 1, 15000)) for a in q]
        case |= {"window": _log(rng, 16, min(8192, 32 * 4096 // n)), "train": False}
    else:
        n, left = _log(rng, 1, 12), _log(rng, 64, 6144)
        cut = sorted(rng.randrange(1, left) for _ in range(n - 1))
        q = [b - a for a, b in zip([0] + cut, cut + [left])]
        q = [v for v in q if v]
        case["train"] = rng.random() < 0.65
        k = [v if case["train"] and rng.random() < 0.8 else v + _log(rng, 1, 2000) for v in q]
        case["window"] = _log(rng, 1, min(4096, 8192 * 1024 // left))
    return case | {"q": ",".join(map(str, q)), "k": ",".join(map(str, k))}


def _lens(text):
    return [int(v) for v in text.split(",")]


def _offs(lens):
    return [0] + np.cumsum(lens)[:-1].tolist()


# ---------------------------------------------------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    bf = lambda *shape: randn(*shape).to(BF)
    s = dict(case)
    if case["op"] == "qk":
        T, hq, hkv, hd = case["tokens"], case["hq"], case["hkv"], case["hd"]
        # projections have other scales from head to head and from token to token
        s["q"] = (randn(T, hq, hd) * (0.3 + 3 * torch.rand((T, hq, 1), generator=g, device="cuda"))).to(BF).view(T, hq * hd)
        s["k"] = (randn(T, hkv, hd) * (0.3 + 3 * torch.rand((T, hkv, 1), generator=g, device="cuda"))).to(BF).view(T, hkv * hd)
        s["wq"] = (1 + 0.2 * randn(hd)).to(BF) if case["weighted"] else None
        s["wk"] = (1 + 0.2 * randn(hd)).to(BF) if case["weighted"] else None
        if case["far"]:
            s["pos"] = torch.randint(0, 1 << 20, (T,), generator=g, device="cuda", dtype=torch.int32)
        else:  # packed sequences that start anew
            s["pos"] = (torch.arange(T, device="cuda") % max(1, T // 3 + 1)).to(torch.int32)
        s["oq"], s["ok"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        if case["train"]:
            s["doq"], s["dok"] = bf(T, hq * hd), bf(T, hkv * hd)
            s["dq"], s["dk"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
            s["dwq"] = torch.empty(hd, dtype=BF, device="cuda") if case["weighted"] else None
            s["dwk"] = torch.empty(hd, dtype=BF, device="cuda") if case["weighted"] else None
    elif case["op"] == "window":
        q, k, hq, hkv, hd = _lens(case["q"]), _lens(case["k"]), case["hq"], case["hkv"], case["hd"]
        s["q_lens"], s["k_lens"], s["q_offs"], s["k_offs"] = q, k, _offs(q), _offs(k)
        s["xq"], s["xk"], s["xv"] = bf(sum(q), hq * hd), bf(sum(k), hkv * hd), bf(sum(k), hkv * hd)
        s["o"] = torch.empty_like(s["xq"])
        s["lse"] = torch.empty((hq, sum(q)), dtype=torch.float32, device="cuda")
        # of every packed row its sequence and its position there
        on = lambda a, dt: torch.from_numpy(np.asarray(a, dt)).cuda()
        s["q_seq"] = on(np.repeat(np.arange(len(q)), q), np.int32)
        s["k_seq"] = on(np.repeat(np.arange(len(k)), k), np.int32)
        s["q_pos"] = on(np.concatenate([np.arange(b - a, b) for a, b in zip(q, k)]), np.int32)
        s["k_pos"] = on(np.concatenate([np.arange(b) for b in k]), np.int32)
        if case["train"]:
            s["do"] = bf(sum(q), hq * hd)
            s["dq"], s["dk"], s["dv"] = torch.empty_like(s["xq"]), torch.empty_like(s["xk"]), torch.empty_like(s["xv"])
    else:
        R, f = case["rows"], case["cols"]
        # rows of different experts have different scales; some values stand far out
        scale = 0.2 + 2 * torch.rand((R, 1), generator=g, device="cuda")
        far = 1 + 7 * (torch.rand((1, f), generator=g, device="cuda") < 0.01)
        s["x1"], s["x3"] = (randn(R, f) * scale * far).to(BF), (randn(R, f) * scale).to(BF)
        s["h"], s["h2"] = torch.empty_like(s["x1"]), torch.empty_like(s["x1"])
        nb = (f + 31) // 32
        u8 = lambda *shape: torch.empty(shape, dtype=torch.uint8, device="cuda")
        s["c1"], s["e1"], s["c3"], s["e3"] = u8(R, f), u8(R, nb), u8(R, f), u8(R, nb)
        s["a"], s["b"] = torch.empty_like(s["x1"]), torch.empty_like(s["x1"])
        if case["use"] == "backward":
            s["dh"] = bf(R, f)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if s["op"] == "qk":
        return _qk_own(s) if own else _qk_plain(s)
    if s["op"] == "window":
        return _window_own(s) if own else _window_plain(s)
    return _act8_own(s) if own else _act8_plain(s)


def _workspace(n):
    return torch.empty(max(16, n), dtype=torch.uint8, device="cuda")


def _qk_own(s):
    from ml_dataflow_b200 import ops

    T, hq, hkv, hd = s["tokens"], s["hq"], s["hkv"], s["hd"]
    ops.qk_norm_rope(T, hq, hkv, hd, EPS, THETA, s["pos"], s["wq"], s["wk"], s["q"], s["k"], s["oq"], s["ok"])
    if not s["train"]:
        return s["oq"], s["ok"]
    if "ws" not in s:  # a program sizes its workspace once
        s["ws"] = _workspace(ops.qk_norm_rope_bwd_workspace_bytes(T, hq, hkv, hd))
    ops.qk_norm_rope_bwd(T, hq, hkv, hd, EPS, THETA, s["pos"], s["wq"], s["wk"], s["q"], s["k"], s["doq"], s["dok"], s["dq"],
                         s["dk"], s["dwq"], s["dwk"], False, s["ws"])
    return s["oq"], s["ok"], s["dq"], s["dk"], s["dwq"], s["dwk"]


def _window_own(s):
    from ml_dataflow_b200 import ops

    args = (s["q_offs"], s["q_lens"], s["k_offs"], s["k_lens"], s["hq"], s["hkv"], s["hd"], s["xq"], s["xk"], s["xv"], s["o"], s["lse"])
    ops.attention_window_fwd(*args, s["window"], s["sinks"])
    if not s["train"]:
        return s["o"], s["lse"]
    if "ws" not in s:
        s["ws"] = _workspace(ops.attention_window_workspace_bytes(len(s["q_lens"]), s["hq"], s["hkv"], s["hd"], s["xq"].shape[0], s["sinks"]))
    ops.attention_window_bwd(*args, s["do"], s["dq"], s["dk"], s["dv"], s["window"], s["sinks"], s["ws"])
    return s["o"], s["lse"], s["dq"], s["dk"], s["dv"]


def _act8_own(s):
    from ml_dataflow_b200 import ops

    R, f = s["rows"], s["cols"]
    ops.swiglu_act8(R, f, s["x1"], s["x3"], s["h"], s["c1"], s["e1"], s["c3"], s["e3"])
    if s["use"] == "restore":
        ops.swiglu_recompute_act8(R, f, s["c1"], s["e1"], s["c3"], s["e3"], s["a"], s["b"], s["h2"])
    else:
        ops.swiglu_bwd_x_act8(R, f, s["c1"], s["e1"], s["c3"], s["e3"], s["dh"], s["a"], s["b"], s["h2"])
    return s["h"], s["a"], s["b"], s["h2"]


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _angles(pos, hd):
    """cos and sin of position * theta^(-2i / hd), the angles in 64 bits: they reach a million radians."""
    i = torch.arange(0, hd, 2, device=pos.device, dtype=torch.float64)
    a = pos.double()[:, None] * torch.exp(i * (-math.log(THETA) / hd))[None, :]
    return torch.cos(a).float()[:, None, :], torch.sin(a).float()[:, None, :]


def _rotate(x, cos, sin):
    e, o = x[..., 0::2], x[..., 1::2]
    return torch.stack([cos * e - sin * o, cos * o + sin * e], dim=-1).flatten(-2)


def _qk_plain(s):
    T, hd = s["tokens"], s["hd"]
    cos, sin = _angles(s["pos"], hd)

    def forward(x, w):
        x = x.float().view(T, -1, hd)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * r
        return _rotate(n if w is None else n * w.float(), cos, sin).reshape(T, -1).to(BF)

    def backward(x, w, dy):
        x = x.float().view(T, -1, hd)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * r
        gy = _rotate(dy.float().view(T, -1, hd), cos, -sin)  # the rotation's transpose
        gn = gy if w is None else gy * w.float()
        dx = r * (gn - n * (gn * n).mean(-1, keepdim=True))
        dw = None if w is None else (gy * n).sum((0, 1), dtype=torch.float64).to(BF)
        return dx.reshape(T, -1).to(BF), dw

    oq, ok = forward(s["q"], s["wq"]), forward(s["k"], s["wk"])
    if not s["train"]:
        return oq, ok
    (dq, dwq), (dk, dwk) = backward(s["q"], s["wq"], s["doq"]), backward(s["k"], s["wk"], s["dok"])
    return oq, ok, dq, dk, dwq, dwk


def _window_plain(s):
    hq, hkv, hd = s["hq"], s["hkv"], s["hd"]
    group, Tq, Tk = hq // hkv, s["xq"].shape[0], s["xk"].shape[0]
    heads_q = lambda x: x.float().view(Tq, hkv, group, hd).permute(1, 2, 0, 3).reshape(hkv, group * Tq, hd)
    heads_k = lambda x: x.float().view(Tk, hkv, hd).transpose(0, 1)
    tokens_q = lambda x: x.view(hkv, group, Tq, hd).permute(2, 0, 1, 3).reshape(Tq, hq * hd).to(BF)
    tokens_k = lambda x: x.transpose(0, 1).reshape(Tk, hkv * hd).to(BF)
    d = s["q_pos"][:, None] - s["k_pos"][None, :]
    seen = (s["q_seq"][:, None] == s["k_seq"][None, :]) & (d >= 0) & ((d < s["window"]) | (s["k_pos"] < s["sinks"])[None, :])
    q, k, v = heads_q(s["xq"]), heads_k(s["xk"]), heads_k(s["xv"])
    scale = 1 / math.sqrt(hd)
    a = torch.matmul(q, k.transpose(1, 2)).mul_(scale).view(hkv, group, Tq, Tk)
    a.masked_fill_(~seen, -math.inf)
    m = a.amax(-1, keepdim=True)
    p = a.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    p = p.div_(l).view(hkv, group * Tq, Tk)
    o = torch.matmul(p, v)
    lse = (m + l.log()).view(hq, Tq)
    if not s["train"]:
        return tokens_q(o), lse
    do = heads_q(s["do"])
    dv = torch.matmul(p.transpose(1, 2), do)
    ds = torch.matmul(do, v.transpose(1, 2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(1, 2), q)
    return tokens_q(o), lse, tokens_q(dq), tokens_k(dk), tokens_k(dv)


def _keep8(x):
    """Values as e4m3 times a power of two for each 32 columns of a row (the smallest that keeps all of them within
    e4m3's range of 448): what they stand for, in 32 bits."""
    R, f = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -f % 32)).view(R, -1, 32)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))  # m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp_(min=-124)
    kept = torch.ldexp(torch.ldexp(b, -e).to(torch.float8_e4m3fn).float(), e)
    return kept.view(R, -1)[:, :f]


def _act8_plain(s):
    x1, x3 = s["x1"].float(), s["x3"].float()
    h = (x1 * torch.sigmoid(x1) * x3).to(BF)
    a, b = _keep8(s["x1"]), _keep8(s["x3"])
    g = torch.sigmoid(a)
    h2 = (a * g * b).to(BF)
    if s["use"] == "restore":
        return h, a.to(BF), b.to(BF), h2
    dh = s["dh"].float()
    return h, (dh * b * g * (1 + a * (1 - g))).to(BF), (dh * a * g).to(BF), h2


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "qk":
        rows, hd = case["tokens"] * (case["hq"] + case["hkv"]), case["hd"]
        n = rows * hd
        w = 4 * hd if case["weighted"] else 0
        fwd = {"bytes": 4 * n + 4 * case["tokens"] + w, "flops": 7 * n}
        return {"bytes": fwd["bytes"] + 4 * n + w, "flops": fwd["flops"] + 14 * n} if case["train"] else fwd
    if case["op"] == "window":
        W, S, hq, hkv, hd = case["window"], case["sinks"], case["hq"], case["hkv"], case["hd"]
        pairs = keys = 0
        for a, b in zip(_lens(case["q"]), _lens(case["k"])):
            p = np.arange(b - a, b, dtype=np.int64)
            pairs += int((np.minimum(W, p + 1) + np.minimum(S, np.maximum(0, p + 1 - W))).sum())
            first = max(0, b - a - W + 1)
            keys += b - first + min(S, first)
        tq, tk = sum(_lens(case["q"])), sum(_lens(case["k"]))
        n = {"bytes": 4 * tq * hq * hd + 4 * keys * hkv * hd + 4 * tq * hq, "flops": 4 * pairs * hq * hd}
        if case["train"]:
            n = {"bytes": n["bytes"] + 4 * tq * hq * hd + 4 * tk * hkv * hd, "flops": n["flops"] + 10 * pairs * hq * hd}
        return n
    n = case["rows"] * case["cols"]
    if case["use"] == "restore":
        return {"bytes": 12 * n, "flops": 20 * n}
    return {"bytes": 14 * n, "flops": 25 * n}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"qk": _qk_exact, "window": _window_exact, "act8": _act8_exact}[case["op"]](s)


def _leaf(x):
    return None if x is None else x.detach().double().requires_grad_(True)


def _qk_exact(s):
    T, hd = s["tokens"], s["hd"]
    freq = torch.tensor([THETA ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones(T, 1, hd // 2, dtype=torch.float64, device="cuda"), (s["pos"].double()[:, None] * freq)[:, None, :])

    def f(x, w):
        x = x.view(T, -1, hd)
        y = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / hd + EPS)
        if w is not None:
            y = y * w
        return torch.view_as_real(torch.view_as_complex(y.reshape(T, -1, hd // 2, 2)) * turn).reshape(T, -1)

    q, k, wq, wk = _leaf(s["q"]), _leaf(s["k"]), _leaf(s["wq"]), _leaf(s["wk"])
    oq, ok = f(q, wq), f(k, wk)
    if not s["train"]:
        return oq.detach(), ok.detach()
    torch.autograd.backward([oq, ok], [s["doq"].double(), s["dok"].double()])
    return oq.detach(), ok.detach(), q.grad, k.grad, None if wq is None else wq.grad, None if wk is None else wk.grad


def _window_exact(s):
    """Sequence by sequence and head by head; the gradients by automatic differentiation."""
    hq, hkv, hd, W, S = s["hq"], s["hkv"], s["hd"], s["window"], s["sinks"]
    o, lse = torch.zeros_like(s["xq"], dtype=torch.float64), torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros_like(x, dtype=torch.float64) for x in (s["xq"], s["xk"], s["xv"]))
    for qo, n, ko, t in zip(s["q_offs"], s["q_lens"], s["k_offs"], s["k_lens"]):
        i = torch.arange(t - n, t, device="cuda").view(n, 1)
        j = torch.arange(t, device="cuda").view(1, t)
        hidden = (j > i) | ((j <= i - W) & (j >= S))
        for h in range(hq):
            c, ck = slice(h * hd, (h + 1) * hd), slice(h // (hq // hkv) * hd, (h // (hq // hkv) + 1) * hd)
            q, k, v = _leaf(s["xq"][qo:qo + n, c]), _leaf(s["xk"][ko:ko + t, ck]), _leaf(s["xv"][ko:ko + t, ck])
            with torch.set_grad_enabled(s["train"]):
                a = (q @ k.T / hd ** 0.5).masked_fill(hidden, -math.inf)
                z = torch.logsumexp(a, 1)
                y = torch.exp(a - z[:, None]) @ v
            o[qo:qo + n, c], lse[h, qo:qo + n] = y.detach(), z.detach()
            if s["train"]:
                y.backward(s["do"][qo:qo + n, c].double())
                dq[qo:qo + n, c] = q.grad
                dk[ko:ko + t, ck] += k.grad
                dv[ko:ko + t, ck] += v.grad
    return (o, lse, dq, dk, dv) if s["train"] else (o, lse)


def _act8_exact(s):
    def kept(x):  # nearest number with four significant bits (ties to even), spaced 2^-9 at least, in units of the block's scale
        x = x.double()
        R, f = x.shape
        out = torch.zeros_like(x)
        for c in range(0, f, 32):
            b = x[:, c:c + 32]
            top = b.abs().amax(1, keepdim=True)
            m, e = torch.frexp(top.clamp(min=1e-300) / 448)  # a power of two itself has m = 1/2
            unit = torch.exp2(torch.where(m > 0.5, e, e - 1).clamp(min=-124).double())
            v = b / unit
            step = torch.exp2(torch.frexp(v.abs().clamp(min=2.0 ** -6))[1].double() - 4)
            out[:, c:c + 32] = torch.round(v / step) * step * unit
        return out

    x1, x3 = s["x1"].double(), s["x3"].double()
    h = x1 / (1 + torch.exp(-x1)) * x3
    del x1, x3
    a, b = kept(s["x1"]).requires_grad_(True), kept(s["x3"]).requires_grad_(True)
    h2 = a / (1 + torch.exp(-a)) * b
    if s["use"] == "restore":
        return h, a.detach(), b.detach(), h2.detach()
    h2.backward(s["dh"].double())
    return h, a.grad, b.grad, h2.detach()
