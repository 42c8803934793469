"""GPU: ops.LAUNCHES after calls of the q/k norm with rotation, the windowed attention and the 8-bit activations: the kernels that a captured
graph of the same calls holds. How many there are follows from the sizes: sequences of a launch, queries few enough for the split form, joins."""
import pytest

pytestmark = pytest.mark.gpu


def _counted(call):
    """(what the counter says, the kernels of a graph)."""
    import torch
    from cuda.bindings import runtime as rt

    from ml_dataflow_b200 import ops

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        before = ops.LAUNCHES
        call()
        said = ops.LAUNCHES - before
    raw = rt.cudaGraph_t(graph.raw_cuda_graph())
    err, _, n = rt.cudaGraphGetNodes(raw)
    assert err == rt.cudaError_t.cudaSuccess
    err, nodes, n = rt.cudaGraphGetNodes(raw, n)
    assert err == rt.cudaError_t.cudaSuccess
    kernels = 0
    for node in nodes[:n]:
        err, kind = rt.cudaGraphNodeGetType(node)
        assert err == rt.cudaError_t.cudaSuccess
        kernels += kind == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel
    return said, kernels


WINDOW = [
    # q_lens, k_lens, hq, hkv, hd, window, sinks
    ([1], [300], 4, 2, 128, 100, 4),                  # the split form alone
    ([1] * 70, [200] * 70, 4, 2, 64, 100, 4),         # more sequences than the tiles take in one launch, one of the split form
    ([1] * 200, [30] * 200, 4, 2, 64, 100, 0),        # two of the split form
    ([400, 1], [400, 90], 4, 2, 128, 100, 4),         # both forms
    ([40] * 60, [40] * 60, 8, 2, 128, 30, 0),         # two launches of tiles
    ([300], [300], 8, 1, 128, 100, 4),                # the backward's heads are split and joined
    ([2600], [2600], 8, 4, 128, 300, 4),              # sinks' shares are joined
    ([3000], [3000], 8, 8, 64, 300, 0),               # nothing to join
    ([50, 20], [50, 90], 2, 2, 32, 16, 2),            # another head size
    ([0, 0], [40, 9], 4, 2, 64, 9, 3),                # no query
]


@pytest.mark.parametrize("q_lens,k_lens,hq,hkv,hd,window,sinks", WINDOW)
def test_windowed_attention(q_lens, k_lens, hq, hkv, hd, window, sinks):
    import torch

    from gpu_util import require_b200

    require_b200()
    from ml_dataflow_b200 import ops

    offs = lambda lens: [sum(lens[:i]) for i in range(len(lens))]
    tq, tk = sum(q_lens) + 1, sum(k_lens)
    rand = lambda n, c: torch.randn((n, c), device="cuda").to(torch.bfloat16)
    q, k, v, do = rand(tq, hq * hd), rand(tk, hkv * hd), rand(tk, hkv * hd), rand(tq, hq * hd)
    o, dq, dk, dv, lse = torch.zeros_like(q), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.zeros((hq, tq), device="cuda")
    ws = torch.empty(ops.attention_window_workspace_bytes(len(q_lens), hq, hkv, hd, tq, sinks), dtype=torch.uint8, device="cuda")
    args = (offs(q_lens), q_lens, offs(k_lens), k_lens, hq, hkv, hd, q, k, v, o, lse)
    said, kernels = _counted(lambda: ops.attention_window_fwd(*args, window, sinks))
    assert said == kernels and (kernels > 0) == any(q_lens)
    said, kernels = _counted(lambda: ops.attention_window_bwd(*args, do, dq, dk, dv, window, sinks, ws))
    assert said == kernels > 0


@pytest.mark.parametrize("rows", [0, 5, 3000])
def test_norm_with_rotation_and_8_bit_activations(rows):
    import torch

    from gpu_util import require_b200

    require_b200()
    from ml_dataflow_b200 import ops

    hq, hkv, hd, f = 4, 2, 64, 72
    rand = lambda *s: torch.randn(s, device="cuda").to(torch.bfloat16)
    u8 = lambda *s: torch.empty(s, dtype=torch.uint8, device="cuda")
    q, k, w = rand(rows, hq * hd), rand(rows, hkv * hd), rand(hd)
    dw, dw2, oq, ok = torch.zeros_like(w), torch.zeros_like(w), torch.empty_like(q), torch.empty_like(k)
    pos, ws = torch.zeros(rows, dtype=torch.int32, device="cuda"), u8(max(16, ops.qk_norm_rope_bwd_workspace_bytes(rows, hq, hkv, hd)))
    x, y, h = rand(rows, f), rand(rows, f), rand(rows, f)
    held = u8(rows, f), u8(rows, 3), u8(rows, f), u8(rows, 3)
    head = (rows, hq, hkv, hd, 1e-5, 10000, pos, w, w, q, k)
    for call in (lambda: ops.qk_norm_rope(*head, oq, ok), lambda: ops.qk_norm_rope_bwd(*head, oq, ok, oq, ok),
                 lambda: ops.qk_norm_rope_bwd(*head, oq, ok, oq, ok, dw, dw2, True, ws), lambda: ops.swiglu_act8(rows, f, x, y, h, *held),
                 lambda: ops.swiglu_recompute_act8(rows, f, *held, x, y, h), lambda: ops.swiglu_bwd_x_act8(rows, f, *held, h, x, y)):
        said, kernels = _counted(call)
        assert said == kernels and (kernels > 0) == (rows > 0)
