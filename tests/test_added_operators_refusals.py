"""CPU: what the q/k norm with rotation, the windowed attention and the 8-bit activations refuse, before any CUDA call: the C entry
points return -1, the Python front end raises. Sizing functions answer on the host."""
import ctypes

import pytest


def _lib():
    from ml_dataflow_b200 import _lib

    return _lib.load()


def _ints(*v):
    return (ctypes.c_int * len(v))(*v)


BF, F32 = 5, 3
P = ctypes.c_void_p(1 << 20)  # an aligned address that is never read: the refusal comes first
ODD = ctypes.c_void_p((1 << 20) + 4)


def test_qk_norm_rope_refusals():
    lib = _lib()
    fwd = lambda dt=BF, T=4, hq=2, hkv=1, hd=64, eps=1e-5, theta=10000, pos=P, w=None, q=P, k=P, oq=P, ok=P: lib.b200_qk_norm_rope(
        dt, T, hq, hkv, hd, eps, theta, pos, w, w, q, k, oq, ok, None)
    for bad in (dict(dt=F32), dict(T=-1), dict(hq=0), dict(hkv=-1), dict(hd=12), dict(hd=0), dict(hd=264), dict(eps=-1.0), dict(theta=0),
                dict(pos=None), dict(q=None), dict(k=None), dict(oq=None), dict(ok=None), dict(q=ODD), dict(ok=ODD), dict(w=ODD)):
        assert fwd(**bad) == -1, bad
    assert fwd(T=0) == 0
    ws = lib.b200_qk_norm_rope_bwd_workspace_bytes
    assert ws(0, 2, 1, 64) == ws(5, 0, 1, 64) == ws(5, 2, 1, 12) == 0 and ws(5, 2, 1, 64) >= 2 * 64 * 4

    def bwd(dt=BF, bdt=BF, T=4, dyq=P, dyk=P, dxq=P, dwq=P, nbytes=1 << 30, work=P):
        return lib.b200_qk_norm_rope_bwd(dt, bdt, T, 2, 1, 64, 1e-5, 10000, P, None, None, P, P, dyq, dyk, dxq, P, dwq, None, 1, nbytes, work,
                                         None)

    for bad in (dict(dt=F32), dict(bdt=F32), dict(dyq=None), dict(dyk=None), dict(dxq=None), dict(dyq=ODD), dict(nbytes=16), dict(work=None),
                dict(work=ODD)):
        assert bwd(**bad) == -1, bad


def test_attention_window_refusals():
    lib = _lib()

    def fwd(dt=BF, n=1, tq=8, tk=8, qo=(0,), ql=(8,), ko=(0,), kl=(8,), hq=2, hkv=1, hd=128, q=P, k=P, v=P, o=P, lse=P, w=4, s=0):
        return lib.b200_attention_window_fwd(dt, n, tq, tk, _ints(*qo), _ints(*ql), _ints(*ko), _ints(*kl), hq, hkv, hd, q, k, v, o, lse, w, s,
                                             None)

    bad = [dict(dt=F32), dict(n=-1), dict(tq=-1), dict(tk=7), dict(tq=7), dict(qo=(-1,)), dict(ko=(1,)), dict(ql=(9,)), dict(kl=(7,)), dict(ql=(-1,)),
           dict(hq=3, hkv=2), dict(hq=0), dict(hkv=0), dict(hd=100), dict(hd=264), dict(hd=0), dict(w=0), dict(w=-5), dict(s=-1), dict(q=None),
           dict(k=None), dict(v=None), dict(o=None), dict(lse=None), dict(q=ODD), dict(o=ODD),
           dict(qo=(2 ** 31 - 4,), ql=(8,)),  # an end past 32 bits
           dict(n=2, tq=12, tk=20, qo=(0, 6), ql=(8, 4), ko=(0, 10), kl=(10, 10)),  # overlapping queries
           dict(n=3, tq=12, tk=30, qo=(8, 0, 9), ql=(2, 8, 2), ko=(0, 10, 20), kl=(10, 10, 10))]
    for b in bad:
        assert fwd(**b) == -1, b
    assert fwd(n=0, tq=0, tk=0) == 0

    def bwd(ko=(0, 10), qo=(0, 6), dq=P, nbytes=1 << 40, work=P, dt=BF, w=4):
        return lib.b200_attention_window_bwd(dt, 2, 12, 20, _ints(*qo), _ints(6, 6), _ints(*ko), _ints(10, 10), 2, 1, 128, P, P, P, P, P, P, dq, P,
                                             P, w, 0, nbytes, work, None)

    for b in (dict(ko=(0, 9)), dict(ko=(5, 0)), dict(qo=(0, 5)), dict(dq=None), dict(dq=ODD), dict(nbytes=8), dict(work=None), dict(work=ODD), dict(dt=F32),
              dict(w=0)):
        assert bwd(**b) == -1, b


def test_overlapping_outputs_are_refused(capfd):
    """Outputs over inputs or one another; weight gradients in one array."""
    lib = _lib()
    at = lambda i: ctypes.c_void_p((i + 1) << 20)  # 1 MB apart, more than any of these tensors
    error = lambda: capfd.readouterr().err
    one, n8 = _ints(0), _ints(8)

    def fwd(**same):
        a = {n: at(i) for i, n in enumerate(("q", "k", "v", "o", "lse"))}
        a |= {n: a[m] for n, m in same.items()}
        return lib.b200_attention_window_fwd(BF, 1, 8, 8, one, n8, one, n8, 2, 1, 128, a["q"], a["k"], a["v"], a["o"], a["lse"], 4, 0, None)

    def bwd(**same):
        a = {n: at(i) for i, n in enumerate(("q", "k", "v", "o", "lse", "do", "dq", "dk", "dv", "ws"))}
        a |= {n: a[m] for n, m in same.items()}
        return lib.b200_attention_window_bwd(BF, 1, 8, 8, one, n8, one, n8, 2, 1, 128, a["q"], a["k"], a["v"], a["o"], a["lse"], a["do"], a["dq"],
                                             a["dk"], a["dv"], 4, 0, 1 << 40, a["ws"], None)

    for call, pairs in ((fwd, (("o", "q"), ("o", "v"), ("lse", "o"), ("lse", "k"))),
                        (bwd, (("dq", "q"), ("dq", "do"), ("dk", "k"), ("dv", "dk"), ("dk", "dq"), ("ws", "dv"), ("ws", "lse"), ("dv", "o")))):
        for a, b in pairs:
            assert call(**{a: b}) == -1 and "overlaps" in error(), (a, b)
    assert lib.b200_qk_norm_rope_bwd(BF, BF, 4, 2, 1, 64, 1e-5, 10000, at(0), None, None, at(1), at(2), at(3), at(4), at(5), at(6), at(7),
                                     ctypes.c_void_p((8 << 20) + 64), 1, 1 << 30, at(9), None) == -1
    assert "overlap" in error()


def test_attention_window_workspace_covers_smaller_batches():
    ws = _lib().b200_attention_window_workspace_bytes
    assert ws(0, 4, 2, 128, 10, 0) == ws(1, 0, 2, 128, 10, 0) == ws(1, 4, 2, 128, 0, 0) == ws(1, 4, 2, 128, 5, -1) == 0
    for hd in (32, 64, 128):
        for grow in ([(1, 100), (1, 1000), (4, 1000), (4, 9000), (90, 9000)],):
            for sinks in (0, 4, 300):
                sizes = [ws(n, 16, 4, hd, t, sinks) for n, t in grow]
                assert sizes == sorted(sizes) and sizes[0] >= 100 * 16 * 4
            assert ws(3, 16, 4, hd, 5000, 0) <= ws(3, 16, 4, hd, 5000, 4) <= ws(3, 16, 4, hd, 5000, 200)


def test_act8_refusals():
    lib = _lib()
    for call, n_in in ((lib.b200_swiglu_act8, 7), (lib.b200_swiglu_recompute_act8, 7), (lib.b200_swiglu_bwd_x_act8, 8)):
        ptrs = [P] * n_in
        assert call(F32, 4, 64, *ptrs, None) == -1
        assert call(BF, -1, 64, *ptrs, None) == -1
        assert call(BF, 4, 60, *ptrs, None) == -1
        assert call(BF, 4, 0, *ptrs, None) == -1
        assert call(BF, 0, 64, *[None] * n_in, None) == 0
        assert call(BF, 4, 64, *[None] * n_in, None) == -1
        assert call(BF, 4, 64, *[ODD] * n_in, None) == -1
    # codes missing; no output asked for; a gradient missing
    assert lib.b200_swiglu_act8(BF, 4, 64, P, P, P, P, None, P, P, None) == -1
    assert lib.b200_swiglu_recompute_act8(BF, 4, 64, P, P, P, P, None, None, None, None) == -1
    assert lib.b200_swiglu_bwd_x_act8(BF, 4, 64, P, P, P, P, P, None, P, None, None) == -1
    n = lib.b200_act8_scales_bytes
    assert (n(3, 64), n(3, 65), n(3, 8), n(0, 8), n(-1, 8)) == (6, 9, 3, 0, 0)
    assert n(1 << 20, 1 << 17) == 1 << 32


def test_the_front_end_refuses_tensors_that_are_not_on_the_current_device():
    torch = pytest.importorskip("torch")
    from ml_dataflow_b200 import ops

    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    u8 = torch.zeros((4, 64), dtype=torch.uint8)
    with pytest.raises(ValueError):
        ops.swiglu_act8(4, 64, x, x, x, u8, u8, u8, u8)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(4, 1, 1, 64, 1e-5, 10000, torch.zeros(4, dtype=torch.int32), None, None, x, x, x, x)
    with pytest.raises(ValueError):
        ops.attention_window_fwd([0], [4], [0], [4], 1, 1, 64, x, x, x, x, torch.zeros(1, 4), 4, 0)
    with pytest.raises(ValueError):
        ops.attention_window_fwd([0], [4, 1], [0], [4], 1, 1, 64, x, x, x, x, torch.zeros(1, 4), 4, 0)
    with pytest.raises(ValueError):
        ops.attention_window_fwd([0], [4], [0], [4], 1, 1, 64, x, x, x, x, torch.zeros(1, 4), 1 << 32, 0)


def test_block_options_mirror_and_refusals():
    """The structure as ctypes sees it; inconsistent options are refused before any CUDA call; unknown levels have no size."""
    import test_abi_exports as abi

    from ml_dataflow_b200 import _lib

    assert abi._struct_fields("B200TransformerBlockOptions") == [f[0] for f in _lib.TransformerBlockOptions._fields_]
    lib = _lib.load()
    assert lib.b200_transformer_block_fwd_options(None, None, None, None, None) == -1
    blk = _lib.TransformerBlock()  # all zeros: bad dimensions
    assert lib.b200_transformer_block_bwd_options(ctypes.byref(blk), None, None, None, None, None, None) == -1
    p = P.value
    m = _lib.MoeBlock(8, 64, 4, 2, 32, *[p] * 4, 2048, 2048, 2048, *[p] * 5, None, *[p] * 8, 1 << 20, p, 1 << 20, *[p] * 7)
    one = _ints(0)
    seqs = ctypes.cast(one, ctypes.c_void_p)
    blk = _lib.TransformerBlock(8, 64, 2, 1, 32, 10000, 1e-5, 1, 8, seqs, seqs, *[p] * 7, *[p] * 11, 1 << 20, m)
    for bad in (dict(qk_norm=1, q_raw=p), dict(qk_norm=1, q_raw=p, k_raw=p, qk_eps=-1.0), dict(window=-1), dict(num_sinks=3), dict(window=4, num_sinks=-1),
                dict(codes_w1=p), dict(codes_w1=p, scales_w1=p, codes_w3=p)):
        o = _lib.TransformerBlockOptions(**bad)
        assert lib.b200_transformer_block_fwd_options(ctypes.byref(blk), ctypes.byref(o), P, ctypes.c_void_p(p + 4096), None) == -1, bad


def test_saved_set_in_8_bits_is_the_stated_layout():
    lib = _lib()
    for T, E, k, f in ((300, 16, 4, 192), (8192, 64, 8, 1408), (1, 2, 1, 8), (5, 4, 2, 40)):
        R, at = T * k, 0
        for s in [4 * T * E, 2 * R, 4 * R, 4 * (E + 1), 4 * E, 4 * R, 4 * R, R * f, R * ((f + 31) // 32), R * f, R * ((f + 31) // 32)]:
            at = (at + 255) // 256 * 256 + s
        assert lib.b200_moe_saved_activations_bytes(T, E, k, f, 4) == at
        assert lib.b200_moe_saved_activations_bytes(T, E, k, f, 5) == 0
