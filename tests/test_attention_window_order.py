"""CPU: the windowed attention's check that sequences do not share rows, for offsets in any order: what it refuses, and that many sequences
do not make it slow. No kernel is launched: the tensors are missing, which is refused next."""
import ctypes
import random
import time

BF = 5


def _fwd(capfd, offs, lens, total):
    """What the forward's refusal says."""
    from ml_dataflow_b200 import _lib

    ints = lambda v: (ctypes.c_int * len(v))(*v)
    ko = [0] * len(offs)  # the forward only reads keys: these may be shared
    capfd.readouterr()
    rc = _lib.load().b200_attention_window_fwd(BF, len(offs), total, max(lens), ints(offs), ints(lens), ints(ko), ints(lens), 2, 1, 64, None, None,
                                               None, None, None, 4, 0, None)
    assert rc == -1
    return capfd.readouterr().err


def test_overlaps_are_found_in_any_order(capfd):
    rng = random.Random(5)
    seen = set()
    for _ in range(400):
        n = rng.randint(2, 9)
        offs, lens = [rng.randrange(0, 60) for _ in range(n)], [rng.choice([0, 1, 2, 3, 8]) for _ in range(n)]
        if not any(lens):
            continue
        shared = any(lens[a] and lens[b] and offs[a] < offs[b] + lens[b] and offs[b] < offs[a] + lens[a] for a in range(n) for b in range(a))
        err = _fwd(capfd, offs, lens, 80)
        assert ("overlap" in err) == shared and ("null tensor" in err) != shared, (offs, lens, err)
        seen.add(shared)
    assert seen == {True, False}


def test_many_sequences_in_descending_order_are_checked_quickly(capfd):
    """A comparison of every pair would be 4.5e10 of them here."""
    n = 300000
    start = time.perf_counter()
    err = _fwd(capfd, list(range(n - 1, -1, -1)), [1] * n, n)
    assert "null tensor" in err
    assert time.perf_counter() - start < 5.0
    assert "overlap" in _fwd(capfd, list(range(n - 1, 0, -1)) + [7], [1] * n, n)
