"""GPU: the q/k norm with rotation, the windowed attention and the 8-bit activations on several streams at once and in graphs that share
a workspace: the same bits as one call after the other."""
import pytest

pytestmark = pytest.mark.gpu

HQ, HKV, WINDOW, SINKS = 8, 2, 150, 4


class Work:
    """Norm and rotation, attention, both backwards, and a SwiGLU held in 8 bits: inputs, outputs and what the calls need."""

    def __init__(self, seed, q_lens, HD=128, workspace=None):
        import torch

        from ml_dataflow_b200 import ops

        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
        self.lens, T = q_lens, sum(q_lens)
        self.offs = [sum(q_lens[:i]) for i in range(len(q_lens))]
        self.T, self.f, self.HD = T, 200, HD
        self.q, self.k, self.v, self.do = rand(T, HQ * HD), rand(T, HKV * HD), rand(T, HKV * HD), rand(T, HQ * HD)
        self.wq, self.wk = rand(HD), rand(HD)
        self.pos = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in q_lens])
        self.x1, self.x3, self.dh = rand(T, self.f), rand(T, self.f), rand(T, self.f)
        like = torch.empty_like
        u8 = lambda *s: torch.empty(s, dtype=torch.uint8, device="cuda")
        self.out = dict(yq=like(self.q), yk=like(self.k), o=like(self.q), lse=torch.empty((HQ, T), device="cuda"), dyq=like(self.q), dyk=like(self.k),
                        dv=like(self.v), dq=like(self.q), dk=like(self.k), dwq=like(self.wq), dwk=like(self.wk), h=like(self.x1), c1=u8(T, self.f),
                        s1=u8(T, 7), c3=u8(T, self.f), s3=u8(T, 7), dx1=like(self.x1), dx3=like(self.x1))
        self.ws_bytes = max(ops.attention_window_workspace_bytes(len(q_lens), HQ, HKV, HD, T, SINKS),
                            ops.qk_norm_rope_bwd_workspace_bytes(T, HQ, HKV, HD))
        self.ws = u8(self.ws_bytes) if workspace is None else workspace

    def run(self):
        from ml_dataflow_b200 import ops

        o, T, HD = self.out, self.T, self.HD
        ops.qk_norm_rope(T, HQ, HKV, HD, 1e-5, 10000, self.pos, self.wq, self.wk, self.q, self.k, o["yq"], o["yk"])
        args = (self.offs, self.lens, self.offs, self.lens, HQ, HKV, HD, o["yq"], o["yk"], self.v, o["o"], o["lse"])
        ops.attention_window_fwd(*args, WINDOW, SINKS)
        held = o["c1"], o["s1"], o["c3"], o["s3"]
        ops.swiglu_act8(T, self.f, self.x1, self.x3, o["h"], *held)
        ops.swiglu_bwd_x_act8(T, self.f, *held, self.dh, o["dx1"], o["dx3"])
        ops.attention_window_bwd(*args, self.do, o["dyq"], o["dyk"], o["dv"], WINDOW, SINKS, self.ws)
        ops.qk_norm_rope_bwd(T, HQ, HKV, HD, 1e-5, 10000, self.pos, self.wq, self.wk, self.q, self.k, o["dyq"], o["dyk"], o["dq"], o["dk"], o["dwq"],
                             o["dwk"], False, self.ws)

    def take(self):
        got = {n: t.clone() for n, t in self.out.items()}
        for t in self.out.values():
            t.zero_()
        return got


def _same(a, b):
    import torch

    for n in a:
        assert torch.equal(a[n], b[n]), n


@pytest.mark.parametrize("hd", [128, 64])
def test_three_streams_at_once(hd):
    import torch

    from gpu_util import require_b200

    require_b200()
    from ml_dataflow_b200 import ops

    works = [Work(1, [700, 33, 400], hd), Work(2, [1, 1, 3, 1], hd), Work(3, [1500], hd)]
    want = []
    for w in works:
        w.run()
        want.append(w.take())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in works]  # none of them is the one the tensors were made on
    for _ in range(300):  # loads that arrive late and out of order are rare
        for _ in range(3):
            for w, s in zip(works, streams):
                with torch.cuda.stream(s):
                    w.run()
        torch.cuda.synchronize()
        for w, ref in zip(works, want):
            _same(w.take(), ref)
        torch.cuda.synchronize()
    assert ops.attention_status() == 0


def test_graphs_that_share_a_workspace():
    import torch

    from gpu_util import require_b200

    require_b200()
    big = Work(4, [900, 200])
    small = Work(5, [70, 1], workspace=big.ws)
    assert small.ws_bytes <= big.ws_bytes
    want = []
    for w in (big, small):
        w.run()
        want.append(w.take())
    torch.cuda.synchronize()
    graphs = []
    for w in (big, small):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            w.run()
        graphs.append(graph)
    for order in ((0, 1, 1, 0), (1, 0, 0, 1)):
        big.ws.fill_(255)
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        _same(big.take(), want[0])
        _same(small.take(), want[1])
        torch.cuda.synchronize()
