"""GPU: SwiGLU activations held in 8 bits against the definition in float64. The codes are one rounding of exact numbers, so
what they stand for has to be equal to the bit; h and the gradients are held to their one rounding to bf16."""
import math

import pytest

pytestmark = pytest.mark.gpu

SHAPES = [(1, 8), (3, 32), (5, 40), (7, 1000), (96, 1408), (1, 4096), (513, 56), (2100, 1408), (33, 8192), (4099, 24)]


def _inputs(R, f, seed):
    import torch

    from gpu_util import require_b200

    require_b200()
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    scale = torch.exp2(torch.randint(-20, 12, (R, 1), generator=g, device="cuda").float())
    x1, x3 = (r(R, f) * scale).to(torch.bfloat16), (r(R, f) * 3).to(torch.bfloat16)
    return x1, x3, r(R, f).to(torch.bfloat16)


def _codes(R, f):
    import torch

    u8 = lambda *s: torch.empty(s, dtype=torch.uint8, device="cuda")
    nb = (f + 31) // 32
    return u8(R, f), u8(R, nb), u8(R, f), u8(R, nb)


def _check(x1, x3, dh):
    import torch

    from ml_dataflow_b200 import ops
    from operator_reference import held8, swiglu, swiglu_bwd, within

    R, f = x1.shape
    c = _codes(R, f)
    assert ops.act8_scales_bytes(R, f) == c[1].numel()
    h, a, b, h2 = (torch.full_like(x1, 7.0) for _ in range(4))
    ops.swiglu_act8(R, f, x1, x3, h, *c)
    ops.swiglu_recompute_act8(R, f, *c, a, b, h2)
    d1, d3, h3 = (torch.full_like(x1, 7.0) for _ in range(3))
    ops.swiglu_bwd_x_act8(R, f, *c, dh, d1, d3, h3)
    torch.cuda.synchronize()
    ra, rb = held8(x1), held8(x3)
    assert torch.equal(a.double().nan_to_num(nan=1e300), ra.nan_to_num(nan=1e300))
    assert torch.equal(b.double().nan_to_num(nan=1e300), rb.nan_to_num(nan=1e300))
    fine = torch.isfinite(ra) & torch.isfinite(rb)
    z = lambda t: torch.where(fine, t.double(), 0.0)
    # the sigmoid's exponential carries up to |x1| * 2^-23 relative, the rest a few 2^-24. exp(-x1) passes fp32's range at
    # x1 = -88.7, where the sigmoid is 2^-128: it is then 0, off by less than 2^-126, and the SwiGLU by that times |x1 x3|
    rel = (ra.abs().nan_to_num(nan=0.0).clamp(max=90) + 8) * 2.0 ** -22
    ref = swiglu(ra, rb)
    tiny = 2.0 ** -126 * (1 + ra.abs().nan_to_num(nan=0.0)) * (1 + rb.abs().nan_to_num(nan=0.0))
    within(z(h2), z(ref), z(rel * ref.abs() + tiny), "h of the held values")
    assert torch.equal(z(h3), z(h2))
    r1, r3 = swiglu_bwd(ra, rb, dh.double())
    g = 1 / (1 + torch.exp(-ra))
    size = (dh.double() * rb).abs() * g * (1 + ra.abs() * (1 - g))
    within(z(d1), z(r1), z(rel * size + tiny * dh.abs().double()), "dx1")
    within(z(d3), z(r3), z(rel * r3.abs() + tiny * dh.abs().double()), "dx3")
    return c, h, a, b, h2, d1, d3


@pytest.mark.parametrize("R,f", SHAPES)
def test_keep_restore_backward(R, f):
    import torch

    from ml_dataflow_b200 import ops
    from operator_reference import swiglu, within

    x1, x3, dh = _inputs(R, f, R + f)
    c, h, a, b, h2, d1, d3 = _check(x1, x3, dh)
    ref = swiglu(x1.double(), x3.double())
    within(h, ref, (x1.double().abs().clamp(max=90) + 8) * 2.0 ** -22 * ref.abs()
           + 2.0 ** -126 * (1 + x1.double().abs()) * (1 + x3.double().abs()), "h")
    # without h the codes are the same; the backward's outputs may lie over the upstream gradient
    c2 = _codes(R, f)
    ops.swiglu_act8(R, f, x1, x3, None, *c2)
    assert all(torch.equal(s, t) for s, t in zip(c, c2))
    for which in (0, 1):  # h over either input
        ins = [x1.clone(), x3.clone()]
        c3 = _codes(R, f)
        ops.swiglu_act8(R, f, *ins, ins[which], *c3)
        assert torch.equal(ins[which], h) and all(torch.equal(s, t) for s, t in zip(c, c3))
    for which in (0, 1):
        up, other = dh.clone(), torch.empty_like(dh)
        out = (up, other) if which == 0 else (other, up)
        ops.swiglu_bwd_x_act8(R, f, *c, up, *out)
        assert torch.equal(out[0], d1) and torch.equal(out[1], d3)
    only = torch.empty_like(h2)
    ops.swiglu_recompute_act8(R, f, *c, out=only)
    assert torch.equal(only, h2)


def test_values_at_the_borders_of_the_format():
    """Block maxima at and next to 448 times a power of two, ties, the smallest steps, zeros of both signs, subnormal bf16 and the
    largest bf16 numbers."""
    import torch

    from gpu_util import require_b200

    require_b200()
    rows = []
    for top in (448.0, 450.0, 446.0, 449.0, 1.75, 1.7578125, 1.0, 3.3e38, 2.0 ** -126, 2.0 ** -133, 2.0 ** -100, 0.0):
        for m in (1.0, -1.0):
            row = torch.zeros(64, dtype=torch.float64)
            row[0] = m * top
            steps = torch.arange(1, 32, dtype=torch.float64)
            row[1:32] = top * (steps / 32) * 1.03125
            row[32:63] = top * torch.exp2(-steps / 2)
            row[63] = -0.0
            rows.append(row)
    # every tie between two neighbouring codes: odd multiples of half a step
    ties = torch.tensor([(16 + 2 * m + 1) / 32 * 2.0 ** e for e in range(-8, 10) for m in range(8)], dtype=torch.float64)
    ties = ties[ties <= 448][:128].view(2, 64)
    rows += [ties[0], ties[1]]
    x = torch.stack(rows).float().to(torch.bfloat16).cuda()
    _check(x, x.flip(0).contiguous(), torch.ones_like(x))


def test_infinities_and_nan_keep_to_themselves():
    import torch

    x1, x3, dh = _inputs(40, 96, 4)
    x1 = torch.randn_like(x1.float()).to(torch.bfloat16)
    plain = x1.clone()
    x1[3, 5], x1[4, 40], x1[5, 95], x1[6, 32:64] = math.inf, -math.inf, math.nan, math.nan
    c, h, a, *_ = _check(x1, x3, dh)
    hit = torch.isnan(a)
    assert int(hit.sum()) == 35 and not torch.isfinite(x1[hit]).any()
    # the others of the block are as if the odd one had been zero
    plain[3, 5] = plain[4, 40] = plain[5, 95] = 0
    plain[6, 32:64] = 0
    a2 = _check(plain, x3, dh)[2]
    assert torch.equal(a[~hit], a2[~hit])


def test_gradient_against_differences():
    """<gradient, direction> from the kernel and from central differences of silu(x1) x3 at the held values, in float64."""
    import torch

    from ml_dataflow_b200 import ops
    from operator_reference import HALF, swiglu

    R, f = 64, 96
    x1, x3, dh = _inputs(R, f, 12)
    x1 = torch.randn_like(x1.float()).to(torch.bfloat16)
    c = _codes(R, f)
    a, b, d1, d3 = (torch.empty_like(x1) for _ in range(4))
    ops.swiglu_act8(R, f, x1, x3, None, *c)
    ops.swiglu_recompute_act8(R, f, *c, a, b)
    ops.swiglu_bwd_x_act8(R, f, *c, dh, d1, d3)
    g = torch.Generator(device="cuda").manual_seed(1)
    u, v = (torch.randn((R, f), generator=g, device="cuda", dtype=torch.float64) for _ in range(2))
    fn = lambda s: (swiglu(a.double() + s * u, b.double() + s * v) * dh.double()).sum()
    step = 2.0 ** -12
    want = ((fn(step) - fn(-step)) / (2 * step)).item()
    terms = torch.cat([(d1.double() * u).flatten(), (d3.double() * v).flatten()])
    assert abs(terms.sum().item() - want) <= 6 * HALF * terms.norm().item() + 1e-5 * terms.abs().sum().item()


def test_more_than_2_to_31_values():
    """Offsets past 32 bits: the last rows of a tensor of 2^31 + 2^21 values."""
    import torch

    from gpu_util import require_b200

    require_b200()
    from ml_dataflow_b200 import ops
    from operator_reference import held8

    f = 1 << 14
    R = (1 << 17) + 128
    x = torch.zeros((R, f), dtype=torch.bfloat16, device="cuda")
    x[-2:] = torch.randn((2, f), device="cuda").to(torch.bfloat16)
    c = _codes(R, f)
    ops.swiglu_act8(R, f, x, x, None, *c)
    a = torch.empty_like(x)
    ops.swiglu_recompute_act8(R, f, *c, x_w1=a)
    torch.cuda.synchronize()
    assert torch.equal(a[-2:].double(), held8(x[-2:])) and not a[:-2].any()
