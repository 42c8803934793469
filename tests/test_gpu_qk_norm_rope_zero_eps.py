"""GPU: b200_qk_norm_rope / _bwd with eps = 0 on rows that are not zero. The number of heads is not always a multiple of those a warp takes
at once: the places behind the last head hold zeros, whose 1 / 0 must not reach the weight gradients of the others."""
import pytest

pytestmark = pytest.mark.gpu

THETA = 10000


@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("T", [1, 33, 700])  # 700: a warp runs over several tokens
@pytest.mark.parametrize("hq,hkv,hd", [(5, 1, 128), (6, 2, 64), (3, 3, 96), (7, 1, 24), (2, 0, 8), (16, 4, 128), (3, 1, 256)])
def test_forward_and_backward(hq, hkv, hd, T, weighted):
    import torch

    from gpu_util import require_b200
    from operator_reference import norm_rope, norm_rope_bwd, within

    require_b200()
    from ml_dataflow_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(100 * hd + T)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
    q, k, dyq, dyk = rand(T, hq * hd), rand(T, hkv * hd), rand(T, hq * hd), rand(T, hkv * hd)
    wq, wk = ((1 + 0.3 * rand(hd)).to(torch.bfloat16) if weighted else None for _ in range(2))
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    oq, ok, dq, dk = (torch.full_like(t, 7.0) for t in (q, k, q, k))
    gq, gk = (torch.full((hd,), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ws = torch.empty(ops.qk_norm_rope_bwd_workspace_bytes(T, hq, hkv, hd), dtype=torch.uint8, device="cuda")
    ops.qk_norm_rope(T, hq, hkv, hd, 0.0, THETA, pos, wq, wk, q, k, oq, ok)
    ops.qk_norm_rope_bwd(T, hq, hkv, hd, 0.0, THETA, pos, wq, wk, q, k, dyq, dyk, dq, dk, gq, gk, False, ws)
    torch.cuda.synchronize()
    for x, w, dy, y, dx, dw in ((q, wq, dyq, oq, dq, gq), (k, wk, dyk, ok, dk, gk)):
        if x.shape[1] == 0:
            assert torch.all(dw == 0)
            continue
        ref = norm_rope(x, w, pos, THETA, 0.0, hd)[0]
        rdx, rdw, terms, size = norm_rope_bwd(x, w, dy, pos, THETA, 0.0, hd)
        # fp32 arithmetic of a pair: a few 2^-24 of its larger member, and 2^-22 of it for the angle
        pair = (2.0 ** -19 * ref.abs().view(T, -1, hd).amax(-1, keepdim=True).expand(-1, -1, hd)).flatten(1)
        within(y, ref, pair, "y")
        within(dx, rdx, 2.0 ** -18 * size, "dx")
        # at most 256 additions follow one another in fp32 (a lane's heads, warps, blocks): 2^-16 of the terms' sum
        within(dw, rdw, 2.0 ** -16 * terms, "dw")
