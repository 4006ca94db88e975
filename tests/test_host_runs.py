"""Runs and token indexes that be42.Lib.rope_append and kv_accept take from the host:
integers that 32 bits hold, refused before anything is planned otherwise."""
import types

import numpy as np
import pytest
import torch

import be42


class Calls(be42.Lib):
    """The library's checks without its calls: what would be given to the entry point."""

    def __init__(self):
        self.torch, self.got = torch, []

    def _on(self, dev, name, *args):
        self.got.append((name, args))


POOL = types.SimpleNamespace(device=0, handle=None, head_dim=64, n_kv=2)
BAD = [[(0, 1, 0.5, 3)], [(0, 1, 0.0, 3)], np.ones((1, 4), bool), [(0, 1, 0, 1 << 31)], [(0, 1, 0, 1 << 70)],
       np.full((1, 4), 1 << 63, np.uint64), np.full((1, 4), -(1 << 31) - 1), [(0, 1, "0", 3)], [0, 1, 0, 3]]


@pytest.mark.parametrize("runs", BAD)
def test_runs_that_are_no_integers(runs):
    c = Calls()
    with pytest.raises(be42.Be42Error, match="be42_kv_accept: runs"):
        c.kv_accept(POOL, runs, [0, 1, 2])
    k = torch.empty(3, 2, 64)
    with pytest.raises(be42.Be42Error, match="be42_rope_append: runs"):
        c.rope_append(POOL, [r[1:] for r in runs] if isinstance(runs[0], tuple) else runs, k, k)
    assert not c.got


@pytest.mark.parametrize("index", [[0.0, 1.0], np.ones(2, bool), [0, 1 << 31], np.array([0, 1 << 63], np.uint64), [[0, 1]]])
def test_indexes_that_are_no_integers(index):
    c = Calls()
    with pytest.raises(be42.Be42Error, match="be42_kv_accept: index"):
        c.kv_accept(POOL, [(0, 1, 0, 2)], index)
    assert not c.got


@pytest.mark.parametrize("kind", [list, tuple, np.int64, np.int32, np.uint8, np.uint64, torch.tensor, "strided"])
def test_integers_of_every_kind(kind):
    rows, index = [(4, 1, 20, 2), (4, 0, 7, 1)], [3, 5, 9]
    if kind == "strided":
        a, b = np.array(rows, np.int32).repeat(2, 1)[:, ::2], np.array(index, np.int32).repeat(2)[::2]
    else:
        make = kind if kind in (list, tuple, torch.tensor) else lambda x: np.array(x, kind)  # noqa: E731
        a, b = make(rows), make(index)
    seen = []

    class Reads(Calls):
        def _on(self, dev, name, pool, runs, n, at, m, *more):
            import ctypes as C
            seen.append(((C.c_int * (4 * n)).from_address(runs)[:], (C.c_int * m).from_address(at)[:], more))

    Reads().kv_accept(POOL, a, b, layers=3, from_step=1, to_step=2)
    assert seen == [([4, 1, 20, 2, 4, 0, 7, 1], index, (3, 1, 2))]


def test_no_runs():
    c = Calls()
    c.kv_accept(POOL, [], [])
    c.kv_accept(POOL, np.zeros((0, 4), np.int32), np.zeros(0))
    assert [a[2] for _, a in c.got] == [0, 0]
