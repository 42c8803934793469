"""GPU: the q/k norm with rotation, the windowed attention and the 8-bit activations behind an event of another stream that writes their inputs
late. Their kernels are set up while the stream's kernel before them drains; what a waited-for event stands for must still be done first, in a
captured graph of two branches too."""
import pytest

pytestmark = pytest.mark.gpu


def _ops():
    """name -> (call, inputs, outputs)"""
    import torch

    from ml_dataflow_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(4)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
    like, u8 = torch.empty_like, lambda *s: torch.empty(s, dtype=torch.uint8, device="cuda")
    T, hq, hkv, hd, f = 700, 4, 2, 64, 200
    pos, w, lens, offs = torch.arange(T, device="cuda", dtype=torch.int32), rand(hd), [500, 200], [0, 500]
    q, k, v, do = rand(T, hq * hd), rand(T, hkv * hd), rand(T, hkv * hd), rand(T, hq * hd)
    oq, ok, dw, dw2, ws = like(q), like(k), like(w), like(w), u8(ops.qk_norm_rope_bwd_workspace_bytes(T, hq, hkv, hd))
    head = (T, hq, hkv, hd, 1e-5, 10000, pos, w, w, q, k)
    o, lse, dq, dk, dv = like(q), torch.empty((hq, T), device="cuda"), like(q), like(k), like(v)
    ws2 = u8(ops.attention_window_workspace_bytes(2, hq, hkv, hd, T, 4))
    attn = (offs, lens, offs, lens, hq, hkv, hd, q, k, v, o, lse)
    q1, o1, lse1 = rand(2, hq * hd), torch.empty((2, hq * hd), dtype=torch.bfloat16, device="cuda"), torch.empty((hq, 2), device="cuda")
    few = ([0, 1], [1, 1], offs, lens, hq, hkv, hd, q1, k, v, o1, lse1)
    x, y, h, dx, dy = rand(T, f), rand(T, f), rand(T, f), rand(T, f), rand(T, f)
    held = u8(T, f), u8(T, 7), u8(T, f), u8(T, 7)
    ops.attention_window_fwd(*attn, 90, 4)
    ops.swiglu_act8(T, f, x, y, h, *held)
    return {
        "qk_norm_rope": (lambda: ops.qk_norm_rope(*head, oq, ok), (q, k), (oq, ok)),
        "qk_norm_rope_bwd": (lambda: ops.qk_norm_rope_bwd(*head, do, v, oq, ok, dw, dw2, False, ws), (q, k, do, v), (oq, ok, dw, dw2)),
        "attention_window_fwd": (lambda: ops.attention_window_fwd(*attn, 90, 4), (q, k, v), (o, lse)),
        "attention_window_fwd, few queries": (lambda: ops.attention_window_fwd(*few, 90, 4), (q1, k, v), (o1, lse1)),
        "attention_window_bwd": (lambda: ops.attention_window_bwd(*attn, do, dq, dk, dv, 90, 4, ws2), (q, k, v, o, lse, do), (dq, dk, dv)),
        "swiglu_act8": (lambda: ops.swiglu_act8(T, f, x, y, h, *held), (x, y), (h, *held)),
        "swiglu_recompute_act8": (lambda: ops.swiglu_recompute_act8(T, f, *held, dx, dy, h), held, (dx, dy, h)),
        "swiglu_bwd_x_act8": (lambda: ops.swiglu_bwd_x_act8(T, f, *held, x, dx, dy), (*held, x), (dx, dy)),
    }


@pytest.mark.parametrize("captured", [False, True])
def test_inputs_written_late_on_another_stream(captured):
    import torch

    from gpu_util import require_b200

    require_b200()
    ops = _ops()
    before, _, _ = _ops()["qk_norm_rope"]  # on tensors of its own
    side = torch.cuda.Stream()
    for name, (call, inputs, outputs) in ops.items():
        kept = [t.clone() for t in inputs]
        call()
        want = [t.clone() for t in outputs]
        torch.cuda.synchronize()

        def late():
            main = torch.cuda.current_stream()
            for t in inputs:
                t.zero_()
            side.wait_stream(main)
            with torch.cuda.stream(side):
                torch.cuda._sleep(2_000_000)  # about a millisecond
                for t, c in zip(inputs, kept):
                    t.copy_(c)
            before()  # the kernel that this stream's next one overlaps with
            main.wait_stream(side)
            call()

        graph = torch.cuda.CUDAGraph()
        if captured:
            with torch.cuda.graph(graph):
                late()
        for _ in range(3):
            for t in outputs:
                t.zero_()
            graph.replay() if captured else late()
            torch.cuda.synchronize()
            assert all(torch.equal(t, c) for t, c in zip(outputs, want)), name
