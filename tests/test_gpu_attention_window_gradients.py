"""GPU: dq, dk and dv of b200_attention_window_bwd, element by element, against the gradient of the defined function: the float64 reference
forms delta from its own output, where the kernels form it from the output as it is stored, in bf16. And all gradients at large scores."""
import math

import pytest

pytestmark = pytest.mark.gpu

CASES = [
    # q_lens, k_lens, hq, hkv, hd, window, sinks: few keys to a query, where delta weighs most; ragged batches; every form of the kernels
    ([200], [200], 4, 2, 128, 1, 0),
    ([200], [200], 4, 2, 128, 2, 0),
    ([300, 1, 70], [300, 40, 190], 8, 2, 64, 3, 1),
    ([130, 45], [130, 700], 4, 4, 128, 16, 4),
    ([700], [700], 5, 1, 128, 200, 4),
    ([1, 2, 33], [50, 2, 90], 8, 1, 128, 5, 2),
    ([2600], [2600], 8, 4, 64, 300, 4),
    ([90, 60], [90, 200], 4, 2, 32, 4, 1),
    ([60], [60], 2, 1, 200, 9, 0),
]


def _inputs(q_lens, k_lens, hq, hkv, hd, seed):
    import torch

    from gpu_util import require_b200

    require_b200()
    offs = lambda lens: [sum(lens[:i]) for i in range(len(lens))]
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda n, c: torch.randn((n, c), generator=g, device="cuda").to(torch.bfloat16)
    tq, tk = sum(q_lens), sum(k_lens)
    return (offs(q_lens), q_lens, offs(k_lens), k_lens, hq, hkv, hd), rand(tq, hq * hd), rand(tk, hkv * hd), rand(tk, hkv * hd), rand(tq, hq * hd)


def _run(lay, q, k, v, do, window, sinks):
    import torch

    from ml_dataflow_b200 import ops

    n, hq, hkv, hd = len(lay[1]), *lay[4:]
    o, lse = torch.empty_like(q), torch.empty((hq, q.shape[0]), device="cuda")
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ws = torch.empty(ops.attention_window_workspace_bytes(n, hq, hkv, hd, q.shape[0], sinks), dtype=torch.uint8, device="cuda")
    ops.attention_window_fwd(*lay, q, k, v, o, lse, window, sinks)
    ops.attention_window_bwd(*lay, q, k, v, o, lse, do, dq, dk, dv, window, sinks, ws)
    torch.cuda.synchronize()
    assert ops.attention_status() == 0
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _delta_slack(lay, q, k, v, do, window, sinks, ref):
    """What a delta of the stored output may move dq and dk by: the output is off by its own rounding, HALF of it, and by what the rounding of
    the probabilities made of it (o_slack), and dS by P times the sum of that over |dO|."""
    import torch

    from operator_reference import HALF, window_mask

    q_offs, q_lens, k_offs, k_lens, hq, hkv, hd = lay
    dq, dk = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (q, k))
    for qo, n, ko, t in zip(q_offs, q_lens, k_offs, k_lens):
        see = window_mask(n, t, window, sinks, "cuda")
        for h in range(hq):
            c, ck = slice(h * hd, (h + 1) * hd), slice(h // (hq // hkv) * hd, (h // (hq // hkv) + 1) * hd)
            Q, K = q[qo:qo + n, c].double(), k[ko:ko + t, ck].double()
            p = torch.softmax(torch.where(see, Q @ K.T / math.sqrt(hd), -math.inf), 1)
            off = HALF * ref["o"][qo:qo + n, c].abs() + 1.02 * ref["o_slack"][qo:qo + n, c]
            err = p * (do[qo:qo + n, c].double().abs() * off).sum(1, keepdim=True) / math.sqrt(hd)
            dq[qo:qo + n, c] = 1.02 * (err @ K.abs())
            dk[ko:ko + t, ck] += 1.02 * (err.T @ Q.abs())
    return dq, dk


@pytest.mark.parametrize("q_lens,k_lens,hq,hkv,hd,window,sinks", CASES)
def test_against_the_gradient_of_the_function(q_lens, k_lens, hq, hkv, hd, window, sinks):
    from operator_reference import window_attention, within

    lay, q, k, v, do = _inputs(q_lens, k_lens, hq, hkv, hd, sum(k_lens) + window)
    got = _run(lay, q, k, v, do, window, sinks)
    ref = window_attention(*lay, q, k, v, window, sinks, do)
    dq, dk = _delta_slack(lay, q, k, v, do, window, sinks, ref)
    within(got["o"], ref["o"], ref["o_slack"], "o")
    within(got["dq"], ref["dq"], ref["dq_slack"] + dq, "dq")
    within(got["dk"], ref["dk"], ref["dk_slack"] + dk, "dk")
    within(got["dv"], ref["dv"], ref["dv_slack"], "dv")


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_scores(sign, hd):
    """Scores of several hundred, rising or falling along the keys."""
    import torch

    from operator_reference import window_attention, within

    window, sinks = 400, 3
    lay, q, k, v, do = _inputs([600], [600], 2, 1, hd, 11)
    ramp = torch.linspace(-1, 1, 600, device="cuda")[:, None]
    q = (q.float() * 0.1 + 6).to(torch.bfloat16)
    k = (k.float() * 0.1 + sign * ramp * 6 * math.sqrt(128 / hd)).to(torch.bfloat16)
    got = _run(lay, q, k, v, do, window, sinks)
    ref = window_attention(*lay, q, k, v, window, sinks, do, got["o"])
    # Scores reach 6 * 6 * 128 / sqrt(128) = 407. They are summed in fp32 in steps of 16 products, eight at most, each off by up to 2^-23 of the
    # sum: 2^-20 of a score, and as much again of the log-sum-exp: a probability moves by 407 * 2^-19 of itself, a fifth of its rounding to bf16
    assert 300 < ref["lse"].abs().max().item() < 420
    assert (got["lse"].double() - ref["lse"]).abs().max().item() <= 407 * 2.0 ** -19
    within(got["o"], ref["o"], 1.25 * ref["o_slack"], "o")
    for name in ("dq", "dk", "dv"):
        # probabilities below 2^-126 are formed as 0: |dS| of at most 2^-126 * 1000, times 600 rows or keys of up to 10
        within(got[name], ref[name], 1.25 * ref[name + "_slack"] + 2.0 ** -100, name)
