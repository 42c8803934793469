"""GPU: b200_attention_window_fwd / _bwd against the definition in float64, element by element: one query to thousands, ragged packed
sequences, windows from one key to more than the sequence, no sinks to more sinks than a tile, every head layout, masked places that
hold NaN, gaps between sequences, more sequences than one launch takes."""
import math

import pytest

pytestmark = pytest.mark.gpu

CASES = [
    # q_lens, k_lens, hq, hkv, hd, window, sinks
    ([1], [1], 1, 1, 128, 1, 0),
    ([1], [2500], 16, 4, 128, 1024, 4),
    ([129], [129], 4, 4, 64, 1, 0),
    ([300, 77, 1], [300, 77, 1], 16, 4, 128, 128, 4),
    ([257], [700], 4, 2, 128, 100, 0),
    ([64, 0, 40], [200, 31, 640], 8, 2, 128, 129, 1),
    ([513], [513], 2, 1, 128, 127, 130),
    ([900], [900], 6, 2, 64, 256, 17),
    ([640], [1700], 3, 1, 64, 300, 33),
    ([385, 130], [900, 130], 8, 2, 128, 5000, 7),
    ([1100], [1100], 2, 2, 128, 64, 300),
    ([700], [700], 5, 1, 128, 200, 4),
    ([33, 200], [333, 200], 4, 2, 32, 50, 3),
    ([70], [90], 3, 3, 96, 40, 2),
    ([45], [300], 2, 1, 256, 64, 5),
    ([20], [20], 2, 2, 8, 7, 1),
    ([1, 2, 1, 3], [900, 4097, 1, 64], 16, 4, 128, 512, 4),
    ([1, 1, 5, 1], [33, 3000, 2000, 7], 8, 1, 64, 1000, 40),
    (list(range(1, 61)), [n + (n % 3) * 50 for n in range(1, 61)], 4, 2, 128, 24, 2),
    ([1] * 70, [3 * n + 1 for n in range(70)], 4, 1, 64, 40, 4),
    # enough blocks of keys to fill the GPU: heads of a group on one unit, the sinks' far tiles on others
    ([2600], [2600], 8, 4, 128, 300, 4),
    ([4000], [4500], 8, 4, 64, 128, 130),
    ([2000, 0, 700], [2100, 300, 700], 12, 4, 128, 200, 17),
    ([1700, 900], [1700, 900], 8, 8, 64, 1, 1),
    ([3000], [3000], 6, 6, 128, 2000, 1100),            # more sinks than are split off
    ([1, 1, 2], [700, 3, 260], 24, 1, 128, 300, 5),     # few queries: more rows than one 16-row tile of a group; 48 rows go to the tiles
    ([1, 2], [500, 900], 40, 1, 64, 1000, 0),           # a group of 40 heads
    ([1, 3, 1], [2000, 130, 77], 21, 3, 128, 90, 2),    # an odd group
    # few queries' tiles on many keys: shared by 2, 4 or 8 CTAs, some of which see nothing of a short sequence or of a tile of a pair
    ([600], [5200], 16, 2, 128, 4000, 4),
    ([300], [2100], 8, 4, 128, 1500, 17),
    ([129, 20, 9], [2500, 20, 400], 4, 1, 64, 2300, 0),
    ([257, 40], [1700, 300], 3, 3, 128, 1400, 130),
    ([500], [3000], 5, 5, 64, 2600, 3),
    ([2] * 200, [2 + 5 * n for n in range(200)], 2, 1, 64, 64, 3),  # more sequences than one launch of the few-query form takes
]


def _offs(lens, gap):
    at, out = gap, []
    for n in lens:
        out.append(at)
        at += n + gap
    return out, at


def _setup(q_lens, k_lens, hq, hkv, hd, window, sinks, seed, gap=0, fill=0.0):
    import torch

    from gpu_util import require_b200

    require_b200()
    q_offs, tq = _offs(q_lens, gap)
    k_offs, tk = _offs(k_lens, gap)
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rows(total, cols, offs, lens):
        x = torch.full((total, cols), fill, dtype=torch.bfloat16, device="cuda")
        for o, n in zip(offs, lens):
            x[o:o + n] = torch.randn((n, cols), generator=g, device="cuda").to(torch.bfloat16)
        return x

    q, do = rows(tq, hq * hd, q_offs, q_lens), rows(tq, hq * hd, q_offs, q_lens)
    k, v = rows(tk, hkv * hd, k_offs, k_lens), rows(tk, hkv * hd, k_offs, k_lens)
    return q_offs, k_offs, q, k, v, do


def _run(q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q, k, v, do, window, sinks, mark=7.0, backward=True):
    import torch

    from ml_dataflow_b200 import ops

    o, lse = torch.full_like(q, mark), torch.full((hq, q.shape[0]), mark, dtype=torch.float32, device="cuda")
    ops.attention_window_fwd(q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q, k, v, o, lse, window, sinks)
    out = {"o": o, "lse": lse}
    if backward:
        n = ops.attention_window_workspace_bytes(len(q_lens), hq, hkv, hd, q.shape[0], sinks)
        ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
        dq, dk, dv = torch.full_like(q, mark), torch.full_like(k, mark), torch.full_like(v, mark)
        ops.attention_window_bwd(q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q, k, v, o, lse, do, dq, dk, dv, window, sinks, ws)
        out |= {"dq": dq, "dk": dk, "dv": dv}
    torch.cuda.synchronize()
    assert ops.attention_status() == 0
    return out


def _compare(got, ref):
    import torch

    from operator_reference import within

    within(got["o"], ref["o"], ref["o_slack"], "o")
    # fp32 scores of |s| up to ~10: 2^-20 of them, the exponentials' 2^-22 and the sum's additions
    assert (got["lse"].double() - ref["lse"]).abs().max().item() <= 2e-5
    for name in ("dq", "dk", "dv"):
        if name in got:
            within(got[name], ref[name], ref[name + "_slack"], name)


@pytest.mark.parametrize("q_lens,k_lens,hq,hkv,hd,window,sinks", CASES)
def test_forward_and_backward(q_lens, k_lens, hq, hkv, hd, window, sinks):
    from operator_reference import window_attention

    q_offs, k_offs, q, k, v, do = _setup(q_lens, k_lens, hq, hkv, hd, window, sinks, 3 * sum(q_lens) + hd)
    args = (q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q, k, v)
    got = _run(*args, do, window, sinks)
    _compare(got, window_attention(*args, window, sinks, do, got["o"]))


@pytest.mark.parametrize("hd", [128, 64, 32])
def test_only_visible_rows_matter_and_rows_outside_stay(hd):
    """NaN between the sequences and in keys that no query sees; marks in the outputs outside the sequences."""
    import torch

    from operator_reference import window_attention

    q_lens, k_lens, hq, hkv, window, sinks = [140, 1, 30, 260], [700, 900, 1300, 260], 4, 2, 150, 5
    q_offs, k_offs, q, k, v, do = _setup(q_lens, k_lens, hq, hkv, hd, window, sinks, 8, gap=3, fill=math.nan)
    for o, n, t in zip(k_offs, q_lens, k_lens):
        dead = slice(o + sinks, o + max(sinks, t - n - window + 1))
        k[dead], v[dead] = math.nan, math.inf
    args = (q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q, k, v)
    got = _run(*args, do, window, sinks)
    inside_q, inside_k = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda"), torch.zeros(k.shape[0], dtype=torch.bool, device="cuda")
    for o, n in zip(q_offs, q_lens):
        inside_q[o:o + n] = True
    for o, n in zip(k_offs, k_lens):
        inside_k[o:o + n] = True
    for name, inside in (("o", inside_q), ("dq", inside_q), ("dk", inside_k), ("dv", inside_k)):
        assert torch.all(got[name][~inside] == 7.0), name
        got[name][~inside] = 0
    assert torch.all(got["lse"][:, ~inside_q] == 7.0)
    got["lse"][:, ~inside_q] = 0
    _compare(got, window_attention(*args, window, sinks, do, got["o"]))


@pytest.mark.parametrize("hd", [128, 64, 96])
def test_a_window_of_everything_is_causal_attention(hd):
    """window >= the sequence, with or without sinks: the same bits, and close to b200_attention_fwd."""
    import torch

    from ml_dataflow_b200 import ops

    q_lens, k_lens, hq, hkv = [400, 90], [520, 90], 4, 2
    q_offs, k_offs, q, k, v, do = _setup(q_lens, k_lens, hq, hkv, hd, 0, 0, 5)
    got = [_run(q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q, k, v, do, w, s) for w, s in ((520, 0), (2 ** 31 - 1, 0))]
    for name in got[0]:
        assert torch.equal(got[0][name], got[1][name]), name
    ws = torch.empty(ops.attention_workspace_bytes(False, hq, hkv, hd, q.shape[0], 400, 520) + 16, dtype=torch.uint8, device="cuda")
    o, lse = torch.empty_like(q), torch.empty_like(got[0]["lse"])
    ops.attention_fwd(q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q, k, v, o, lse, True, ws)
    # both within two roundings (probabilities, output) of the exact result, whose size is at most that of v (|v| < 6)
    assert (o.float() - got[0]["o"].float()).abs().max().item() <= 4 * 6 * 2.0 ** -8
    assert (lse - got[0]["lse"]).abs().max().item() <= 4e-5


@pytest.mark.parametrize("hd", [128, 64, 40])
def test_two_runs_give_the_same_bits(hd):
    import torch

    q_lens, k_lens, hq, hkv, window, sinks = [700, 1, 300], [700, 800, 900], 6, 2, 130, 6
    q_offs, k_offs, q, k, v, do = _setup(q_lens, k_lens, hq, hkv, hd, window, sinks, 6)
    a, b = (_run(q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q, k, v, do, window, sinks) for _ in range(2))
    for name in a:
        assert torch.equal(a[name], b[name]), name


def test_large_scores_and_one_dominant_key():
    """Scores of several hundred, rising along the keys (the running maximum moves at every step) and falling."""
    import torch

    from operator_reference import window_attention

    q_lens = k_lens = [600]
    hq, hkv, hd, window, sinks = 2, 1, 128, 400, 3
    q_offs, k_offs, q, k, v, do = _setup(q_lens, k_lens, hq, hkv, hd, window, sinks, 2)
    ramp = torch.linspace(-1, 1, 600, device="cuda")[:, None]
    for sign in (1, -1):
        k2 = (k.float() * 0.1 + sign * ramp * 4).to(torch.bfloat16)
        q2 = (q.float() * 0.1 + 4).to(torch.bfloat16)
        args = (q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q2, k2, v)
        got = _run(*args, do, window, sinks)
        ref = window_attention(*args, window, sinks, do, got["o"])
        # scores reach 4 * 4 * 128 / sqrt(128) = 181, and 2^-21 of them (a product and a sum of fp32) moves a probability by 2^-13 of itself
        assert (got["lse"].double() - ref["lse"]).abs().max().item() <= 181 * 2.0 ** -20
        from operator_reference import within

        within(got["o"], ref["o"], 1.1 * ref["o_slack"], "o")
        within(got["dv"], ref["dv"], 1.1 * ref["dv_slack"], "dv")


def test_captured_and_replayed():
    import torch

    from ml_dataflow_b200 import ops

    q_lens, k_lens, hq, hkv, hd, window, sinks = [300, 1], [300, 900], 4, 2, 128, 100, 4
    q_offs, k_offs, q, k, v, do = _setup(q_lens, k_lens, hq, hkv, hd, window, sinks, 6)
    o, lse, dq, dk, dv = (torch.empty_like(t) for t in (q, torch.empty((hq, q.shape[0]), device="cuda"), q, k, v))
    ws = torch.empty(ops.attention_window_workspace_bytes(2, hq, hkv, hd, q.shape[0], sinks), dtype=torch.uint8, device="cuda")

    def step():
        args = (q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q, k, v, o, lse)
        ops.attention_window_fwd(*args, window, sinks)
        ops.attention_window_bwd(*args, do, dq, dk, dv, window, sinks, ws)

    step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    v.mul_(2)
    for t in (o, dq, dk, dv):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    replayed = [t.clone() for t in (o, lse, dq, dk, dv)]
    step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(replayed, (o, lse, dq, dk, dv)))


def test_gradient_against_differences():
    import torch

    from operator_reference import HALF, window_attention

    q_lens, k_lens, hq, hkv, hd, window, sinks = [90, 40], [90, 140], 2, 1, 64, 30, 3
    q_offs, k_offs, q, k, v, do = _setup(q_lens, k_lens, hq, hkv, hd, window, sinks, 21)
    lay = (q_offs, q_lens, k_offs, k_lens, hq, hkv, hd)
    got = _run(*lay, q, k, v, do, window, sinks)
    g = torch.Generator(device="cuda").manual_seed(1)
    u = [torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64) for t in (q, k, v)]
    f = lambda s: (window_attention(*lay, *(t.double() + s * d for t, d in zip((q, k, v), u)), window, sinks)["o"] * do.double()).sum()
    h = 2.0 ** -12
    want = ((f(h) - f(-h)) / (2 * h)).item()
    terms = torch.cat([(got[n].double() * d).flatten() for n, d in zip(("dq", "dk", "dv"), u)])
    # a gradient carries its own rounding and those of the probabilities, dS and the output that delta is formed from: three more of
    # like size; independent signs, six standard deviations
    assert abs(terms.sum().item() - want) <= 6 * 2 * HALF * terms.norm().item()


@pytest.mark.parametrize("hd", [128, 64, 40])
def test_more_window_or_sinks_than_there_are_keys(hd):
    """The largest numbers that the arguments take: every key before a query is seen, as with a window of the whole sequence."""
    import torch

    from operator_reference import window_attention

    q_lens, k_lens, hq, hkv = [400, 2, 90], [520, 300, 90], 4, 2
    q_offs, k_offs, q, k, v, do = _setup(q_lens, k_lens, hq, hkv, hd, 0, 0, 5)
    run = lambda w, s: _run(q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q, k, v, do, w, s)
    want = run(520, 0)
    for w, s in ((2 ** 31 - 1, 2 ** 31 - 1), (520, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 100)):
        got = run(w, s)
        assert all(torch.equal(got[n], want[n]) for n in want), (w, s)
    got, args = run(1, 2 ** 31 - 1), (q_offs, q_lens, k_offs, k_lens, hq, hkv, hd, q, k, v)  # sinks only
    _compare(got, window_attention(*args, 1, 2 ** 31 - 1, do, got["o"]))


@pytest.mark.parametrize("hd", [128, 32])
def test_sequences_without_queries(hd):
    """No query at all: nothing is written forward, keys and values get zeros."""
    import torch

    hq, hkv = 4, 2
    for q_lens, k_lens, pad in (([0, 0], [130, 7], 0), ([0, 0], [130, 7], 5)):
        k_offs, tk = _offs(k_lens, 2)
        q = torch.full((pad, hq * hd), math.nan, dtype=torch.bfloat16, device="cuda")
        k = torch.randn((tk, hkv * hd), device="cuda").to(torch.bfloat16)
        got = _run([0, 0], q_lens, k_offs, k_lens, hq, hkv, hd, q, k, k.clone(), q.clone(), 9, 3)
        inside = torch.zeros(tk, dtype=torch.bool, device="cuda")
        for o, n in zip(k_offs, k_lens):
            inside[o:o + n] = True
        assert torch.all(got["o"] == 7.0) and torch.all(got["lse"] == 7.0) and torch.all(got["dq"] == 7.0)
        for n in ("dk", "dv"):
            assert torch.all(got[n][inside] == 0) and torch.all(got[n][~inside] == 7.0), n
