"""GPU: windowed attention in batches of more work units than the GPU has SMs, so that a CTA walks several: one unit's loads begin under
the last one's products. One sequence (units in rounds), several (dealt out by the host, or in rounds where there are too many), halves of
pairs behind whole ones, pairs of heads and of neighbouring tiles; alone against float64, and on three streams at once bit for bit."""
import pytest

pytestmark = pytest.mark.gpu

CASES = [
    # q_lens, k_lens, hq, hkv, hd, window, sinks
    ([2600], [2600], 16, 4, 128, 300, 4),                       # one sequence: rounds, halves in the last
    ([2600], [2600], 16, 4, 64, 5000, 0),                       # units from one block to all: no halves
    ([3500], [3600], 12, 12, 64, 500, 130),                     # no sharing: pairs of neighbouring tiles
    ([1024] * 6, [1024] * 6, 16, 4, 128, 512, 4),               # several sequences: dealt out
    ([700, 1300, 90, 2000, 513], [700, 1300, 90, 2000, 600], 16, 4, 64, 700, 17),
    ([900, 1500, 700], [900, 1500, 1000], 15, 5, 128, 200, 0),  # an odd group, dealt out
    ([1500, 700, 300], [5000, 700, 900], 16, 4, 128, 900, 4),   # chunks of prompts
    ([130 + 7 * i for i in range(60)], [130 + 9 * i for i in range(60)], 8, 2, 128, 100, 2),  # more sequences than one launch takes
    ([50 + 37 * i for i in range(40)], [50 + 37 * i for i in range(40)], 8, 2, 64, 1024, 1),  # too many kinds of units to deal out: rounds
    ([1, 900, 2, 1200], [500, 900, 700, 1300], 24, 4, 128, 333, 5),  # two forms in one call
]


def _pairs(q_lens, hq, hkv):
    """Pairs of tiles of sequences that the form for few queries does not take."""
    tiles = [(n + 127) // 128 for n in q_lens if n * (hq // hkv) > 32]
    return sum(t * (hq // 2) if hq // hkv % 2 == 0 else (t + 1) // 2 * hq for t in tiles)


class Call:
    def __init__(self, q_lens, k_lens, hq, hkv, hd, window, sinks, seed, backward=True):
        import torch

        from ml_dataflow_b200 import ops

        offs = lambda lens: [sum(lens[:i]) for i in range(len(lens))]
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda n, c: torch.randn((n, c), generator=g, device="cuda").to(torch.bfloat16)
        tq, tk = sum(q_lens), sum(k_lens)
        self.lay, self.mask, self.backward = (offs(q_lens), q_lens, offs(k_lens), k_lens, hq, hkv, hd), (window, sinks), backward
        self.q, self.k, self.v, self.do = rand(tq, hq * hd), rand(tk, hkv * hd), rand(tk, hkv * hd), rand(tq, hq * hd)
        self.out = {"o": torch.zeros_like(self.q), "lse": torch.zeros((hq, tq), device="cuda")}
        if backward:
            self.out |= {"dq": torch.zeros_like(self.q), "dk": torch.zeros_like(self.k), "dv": torch.zeros_like(self.v)}
            self.ws = torch.empty(ops.attention_window_workspace_bytes(len(q_lens), hq, hkv, hd, tq, sinks), dtype=torch.uint8, device="cuda")

    def run(self):
        from ml_dataflow_b200 import ops

        o = self.out
        args = (*self.lay, self.q, self.k, self.v, o["o"], o["lse"])
        ops.attention_window_fwd(*args, *self.mask)
        if self.backward:
            ops.attention_window_bwd(*args, self.do, o["dq"], o["dk"], o["dv"], *self.mask, self.ws)

    def take(self):
        got = {n: t.clone() for n, t in self.out.items()}
        for t in self.out.values():
            t.zero_()
        return got


@pytest.mark.parametrize("q_lens,k_lens,hq,hkv,hd,window,sinks", CASES)
def test_forward_and_backward(q_lens, k_lens, hq, hkv, hd, window, sinks):
    import torch

    from gpu_util import require_b200
    from operator_reference import window_attention, within

    require_b200()
    from ml_dataflow_b200 import ops

    assert _pairs(q_lens, hq, hkv) > ops.device_info()[0]
    call = Call(q_lens, k_lens, hq, hkv, hd, window, sinks, 5 * sum(q_lens) + hd)
    call.run()
    got = call.take()
    torch.cuda.synchronize()
    assert ops.attention_status() == 0
    ref = window_attention(*call.lay, call.q, call.k, call.v, window, sinks, call.do, got["o"])
    within(got["o"], ref["o"], ref["o_slack"], "o")
    # fp32 scores of |s| up to ~10: 2^-20 of them, the exponentials' 2^-22 and the sum's additions
    assert (got["lse"].double() - ref["lse"]).abs().max().item() <= 2e-5
    for name in ("dq", "dk", "dv"):
        within(got[name], ref[name], ref[name + "_slack"], name)


@pytest.mark.parametrize("hd", [128, 64])
def test_three_streams_at_once(hd):
    """Dealt units, units in rounds, and units shared by clusters: late and unordered arrivals in every walk."""
    import torch

    from gpu_util import require_b200

    require_b200()
    from ml_dataflow_b200 import ops

    calls = [Call([1024] * 5, [1024] * 5, 8, 2, hd, 300, 4, 1, backward=False), Call([2600], [2600], 16, 4, hd, 400, 0, 2, backward=False),
             Call([300], [2600], 8, 4, hd, 2000, 17, 3, backward=False)]
    assert all(_pairs(c.lay[1], *c.lay[4:6]) > ops.device_info()[0] for c in calls[:2])
    want = []
    for c in calls:
        c.run()
        want.append(c.take())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(300):
        for _ in range(3):
            for c, s in zip(calls, streams):
                with torch.cuda.stream(s):
                    c.run()
        torch.cuda.synchronize()
        for c, ref in zip(calls, want):
            got = c.take()
            assert all(torch.equal(got[n], ref[n]) for n in ref)
        torch.cuda.synchronize()
    assert ops.attention_status() == 0


def test_captured_and_replayed():
    import torch

    from gpu_util import require_b200

    require_b200()
    call = Call([1024] * 4 + [3], [1024] * 4 + [700], 16, 4, 128, 400, 4, 9)
    call.run()
    want = call.take()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call.run()
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    got = call.take()
    assert all(torch.equal(got[n], want[n]) for n in want)
