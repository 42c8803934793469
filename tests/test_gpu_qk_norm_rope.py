"""GPU: b200_qk_norm_rope / _bwd against the definition in float64: head sizes from 8 to 256 (also ones that are no power of
two), one token to thousands, positions of millions, missing weights, in place, zero rows, accumulating and overwritten weight
gradients, a captured graph, and differences of the forward."""
import pytest

pytestmark = pytest.mark.gpu

THETA, EPS = 500000, 1e-5
SHAPES = [  # tokens, query heads, key heads, head_dim
    (1, 16, 4, 128), (24, 16, 4, 128), (333, 5, 1, 64), (2367, 3, 3, 128), (2368, 2, 1, 128), (2500, 16, 4, 128), (7, 2, 2, 8), (65, 4, 2, 24),
    (50, 3, 1, 96), (129, 6, 2, 256), (40, 7, 0, 16), (3, 70, 10, 32), (11, 1, 1, 200),
]


def _inputs(T, hq, hkv, hd, seed, far=False):
    import torch

    from gpu_util import require_b200

    require_b200()
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
    q, k = 2 * r(T, hq * hd), r(T, hkv * hd)
    pos = torch.randint(0, 1 << 21 if far else 9000, (T,), generator=g, device="cuda", dtype=torch.int32)
    return q, k, pos, (1 + 0.3 * r(hd)).to(torch.bfloat16), (1 + 0.3 * r(hd)).to(torch.bfloat16), r(T, hq * hd), r(T, hkv * hd)


def _tol(ref, hd):
    """fp32 arithmetic of a pair: a few 2^-24 of its larger member, and 2^-22 of it for the angle."""
    return (2.0 ** -19 * ref.abs().view(ref.shape[0], -1, hd).amax(-1, keepdim=True).expand(-1, -1, hd)).flatten(1)


@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("T,hq,hkv,hd", SHAPES)
def test_forward_and_backward(T, hq, hkv, hd, weighted):
    import torch

    from ml_dataflow_b200 import ops
    from operator_reference import norm_rope, norm_rope_bwd, within

    q, k, pos, wq, wk, dyq, dyk = _inputs(T, hq, hkv, hd, T + hd, far=weighted)
    if T > 2:
        q[1] = 0  # a row of zeros: r = 1 / sqrt(eps)
    if not weighted:
        wq = wk = None
    oq, ok = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    ops.qk_norm_rope(T, hq, hkv, hd, EPS, THETA, pos, wq, wk, q, k, oq, ok)
    n = ops.qk_norm_rope_bwd_workspace_bytes(T, hq, hkv, hd)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    dq, dk = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    gq, gk = (torch.full((hd,), v, dtype=torch.bfloat16, device="cuda") for v in (0.5, -2.0))
    ops.qk_norm_rope_bwd(T, hq, hkv, hd, EPS, THETA, pos, wq, wk, q, k, dyq, dyk, dq, dk, gq, gk, True, ws)
    gq2, gk2 = torch.full_like(gq, 9.0), torch.full_like(gk, 9.0)
    ops.qk_norm_rope_bwd(T, hq, hkv, hd, EPS, THETA, pos, wq, wk, q, k, dyq, dyk, dq, dk, gq2, gk2, False, ws)
    torch.cuda.synchronize()
    for x, w, dy, y, dx, acc, start, over in ((q, wq, dyq, oq, dq, gq, 0.5, gq2), (k, wk, dyk, ok, dk, gk, -2.0, gk2)):
        if x.shape[1] == 0:
            assert torch.all(over == 0) and torch.all(acc == start)
            continue
        ref, _ = norm_rope(x, w, pos, THETA, EPS, hd)
        within(y, ref, _tol(ref, hd), "y")
        rdx, rdw, terms, size = norm_rope_bwd(x, w, dy, pos, THETA, EPS, hd)
        within(dx, rdx, 2.0 ** -18 * size, "dx")
        # at most 256 additions follow one another in fp32 (a lane's heads, warps, blocks): 2^-16 of the terms' sum
        within(over, rdw, 2.0 ** -16 * terms, "dw written")
        within(acc, rdw + start, 2.0 ** -16 * terms, "dw added")


def test_in_place_and_reruns_give_the_same_bits():
    import torch

    from ml_dataflow_b200 import ops

    T, hq, hkv, hd = 777, 16, 4, 128
    q, k, pos, wq, wk, dyq, dyk = _inputs(T, hq, hkv, hd, 3)
    oq, ok = torch.empty_like(q), torch.empty_like(k)
    ops.qk_norm_rope(T, hq, hkv, hd, EPS, THETA, pos, wq, wk, q, k, oq, ok)
    q2, k2 = q.clone(), k.clone()
    ops.qk_norm_rope(T, hq, hkv, hd, EPS, THETA, pos, wq, wk, q2, k2, q2, k2)
    assert torch.equal(oq, q2) and torch.equal(ok, k2)
    ws = torch.empty(ops.qk_norm_rope_bwd_workspace_bytes(T, hq, hkv, hd), dtype=torch.uint8, device="cuda")
    got = []
    for _ in range(2):
        a, b = dyq.clone(), dyk.clone()
        gq, gk = torch.empty_like(wq), torch.empty_like(wk)
        ops.qk_norm_rope_bwd(T, hq, hkv, hd, EPS, THETA, pos, wq, wk, q, k, a, b, a, b, gq, gk, False, ws)
        got.append((a, b, gq, gk))
    assert all(torch.equal(x, y) for x, y in zip(*got))
    # without weight gradients no workspace is asked for
    a, b = torch.empty_like(dyq), torch.empty_like(dyk)
    ops.qk_norm_rope_bwd(T, hq, hkv, hd, EPS, THETA, pos, wq, wk, q, k, dyq, dyk, a, b)
    assert torch.equal(a, got[0][0]) and torch.equal(b, got[0][1])


def test_workspace_of_the_largest_batch_serves_every_smaller_one():
    from gpu_util import require_b200

    require_b200()
    from ml_dataflow_b200 import ops

    for hd in (8, 64, 128, 256):
        sizes = [ops.qk_norm_rope_bwd_workspace_bytes(T, 16, 4, hd) for T in (1, 100, 1000, 2367, 2368, 2369, 5000, 100000)]
        assert sizes == sorted(sizes)


def test_captured_and_replayed_on_another_stream():
    import torch

    from ml_dataflow_b200 import ops

    T, hq, hkv, hd = 96, 16, 4, 128
    q, k, pos, wq, wk, dyq, dyk = _inputs(T, hq, hkv, hd, 5)
    out = [torch.empty_like(t) for t in (q, k, q, k, wq, wk)]
    ws = torch.empty(ops.qk_norm_rope_bwd_workspace_bytes(T, hq, hkv, hd), dtype=torch.uint8, device="cuda")

    def step():
        ops.qk_norm_rope(T, hq, hkv, hd, EPS, THETA, pos, wq, wk, q, k, out[0], out[1])
        ops.qk_norm_rope_bwd(T, hq, hkv, hd, EPS, THETA, pos, wq, wk, q, k, dyq, dyk, out[2], out[3], out[4], out[5], False, ws)

    step()
    torch.cuda.synchronize()
    ref = [t.clone() for t in out]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    q.mul_(2)  # new values under the captured graph
    for t in out:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    again = [t.clone() for t in out]
    step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, out)) and not torch.equal(again[2], ref[2])


def test_gradient_against_differences():
    """The derivative of a weighted sum of the outputs along a direction, from the kernel's gradients and from central differences
    of the definition in float64 (step 2^-12: the cubic term is below 2^-20 of the derivative's scale)."""
    import torch

    from ml_dataflow_b200 import ops
    from operator_reference import HALF, norm_rope

    T, hq, hkv, hd = 40, 3, 1, 64
    q, k, pos, wq, wk, dyq, dyk = _inputs(T, hq, hkv, hd, 9)
    dq, dk, gq, gk = (torch.empty_like(t) for t in (q, k, wq, wk))
    ws = torch.empty(ops.qk_norm_rope_bwd_workspace_bytes(T, hq, hkv, hd), dtype=torch.uint8, device="cuda")
    ops.qk_norm_rope_bwd(T, hq, hkv, hd, EPS, THETA, pos, wq, wk, q, k, dyq, dyk, dq, dk, gq, gk, False, ws)
    g = torch.Generator(device="cuda").manual_seed(1)
    for x, w, dy, dx, dw in ((q, wq, dyq, dq, gq), (k, wk, dyk, dk, gk)):
        ux, uw = (torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64) for t in (x, w))
        f = lambda s: (norm_rope(x.double() + s * ux, w.double() + s * uw, pos, THETA, EPS, hd)[0] * dy.double()).sum()
        h = 2.0 ** -12
        want = ((f(h) - f(-h)) / (2 * h)).item()
        terms = torch.cat([(dx.double() * ux).flatten(), (dw.double() * uw).flatten()])
        # every gradient is rounded once; the signs of the roundings are independent (six times their standard deviation)
        assert abs(terms.sum().item() - want) <= 6 * HALF * terms.norm().item() + 1e-5 * terms.abs().sum().item()
