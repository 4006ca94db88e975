"""What an append leaves of its slots' counts (pages in use, pages with a hash, tokens
of a page) where a launch holds a run in several pieces: pages that follow one another
by the first, the others listed."""
import numpy as np
import pytest
import torch

from test_gpu_rope_append import PAGE, held_rows, make, rows_of, same, state

pytestmark = pytest.mark.gpu


def append_both(be, rng, pool, by_hand, runs):
    """The same tokens by one call, and by be42_kv_append of each run."""
    n, kvh, hd = sum(r[2] for r in runs), pool.n_kv, pool.head_dim
    k, v = (rows_of(rng, n, kvh, hd, False).cuda() for _ in range(2))
    be.rope_append(pool, runs, k, v)
    at = 0
    for slot, p0, c in runs:
        by_hand.append(slot, k[at:at + c].reshape(c, -1), v[at:at + c].reshape(c, -1), p0)
        at += c


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("hd", [64, 40])
@pytest.mark.parametrize("first,then", [(5, 16 * 40), (500, 3000), (17, 16 * 16 + 3), (31, 1 + 16 * 20)])
def test_runs_that_go_on_from_inside_a_page(be, kind, hd, first, then):
    """An old page and 16 or more new ones: everything that the pool holds is what
    be42_kv_append leaves."""
    rng = np.random.default_rng(first)
    pool, by_hand = (make(be, kind, 6, 2, hd, -(-(first + then) // PAGE)) for _ in range(2))
    append_both(be, rng, pool, by_hand, [(s, 0, first) for s in range(6)])
    same(state(pool), state(by_hand))
    append_both(be, rng, pool, by_hand, [(s, first, then) for s in (3, 0, 5, 1)])
    a = state(pool)
    assert list(a["n_logical"]) == list(a["length"])
    assert list(a["n_indexed"]) == [(first + then) // PAGE if s in (3, 0, 5, 1) else first // PAGE for s in range(6)]
    same(a, state(by_hand))


def apart(be, kind, hd, per, stretch):
    """A pool of which the pages that it gives out next lie in such stretches (slot 0
    had them), the ones between held by slot 1."""
    pool = make(be, kind, 4, 1, hd, per)
    row = torch.zeros(2 * per * PAGE, 1, hd, device="cuda")
    at = 0
    for n in stretch:
        c = min(n, per - at) * PAGE
        if c:
            be.rope_append(pool, [(0, at * PAGE, c), (1, at * PAGE, c)], row[:2 * c], row[:2 * c])
            at += c // PAGE
    pool.reset(0)
    return pool, at


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("stretch", [[1] * 560, [3, 40, 1], [1, 2, 15, 16, 17, 40, 1, 1, 300, 3, 1, 20, 16], [20, 1, 1, 30, 1, 16, 2, 16]])
@pytest.mark.parametrize("first", [0, 5])
def test_pages_of_all_orders(be, kind, stretch, first):
    """Runs from a page's begin and from inside one, over pages apart (more than a
    launch lists) and in a row."""
    rng = np.random.default_rng(len(stretch) + first)
    hd, per = 64, sum(stretch) + 8
    pool, pages = apart(be, kind, hd, per, stretch)
    n = pages * PAGE - 11
    other = make(be, kind, 4, 1, hd, per)
    if first:
        append_both(be, rng, pool, other, [(0, 0, first), (2, 0, 3)])
    append_both(be, rng, pool, other, [(2, 3 if first else 0, 30), (0, first, n - first)])
    a, b = state(pool), state(other)
    assert (a["page_table"] == a["host_table"]).all()
    lens = [n, pages * PAGE, 33 if first else 30, 0]
    assert list(a["n_logical"]) == list(a["length"]) == [-(-m // PAGE) for m in lens]
    assert list(a["n_indexed"]) == [m // PAGE for m in lens]
    for slot in (0, 2):
        m, at, bt = lens[slot], pool.layer_pages(slot), other.layer_pages(slot)
        assert (a["ntok"][at] == b["ntok"][bt]).all()
        assert (a["page_hash"].reshape(4, per)[slot][:m // PAGE] == b["page_hash"].reshape(4, per)[slot][:m // PAGE]).all()
        assert (a["centroid"][at[:m // PAGE]] == b["centroid"][bt[:m // PAGE]]).all()
        x, y = held_rows(pool, slot, m), held_rows(other, slot, m)
        for name in x:
            assert (x[name] == y[name]).all(), name


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("later", [3, 12, 20, 60])
def test_a_replay_leaves_what_the_call_leaves(be, kind, later):
    """Behind later appends: pages past the captured positions stay, the page of the last
    captured token ends with it, in a replay as in a call."""
    rng = np.random.default_rng(later)
    k, more = (rows_of(rng, n, 1, 64, False).cuda() for n in (40, later))
    pools = [make(be, kind, 4, 1, 64, 8) for _ in range(2)]
    for pool in pools:
        be.rope_append(pool, [(0, 0, 20), (1, 0, 10)], k[:30], k[:30])

    def step(pool):
        be.rope_append(pool, [(2, 0, 20), (0, 20, 5)], k[:25], k[:25])
        be.kv_accept(pool, [(0, 1, 10, 10)], range(10))

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(pools[0])
    for i in range(3):
        if i == 1:
            for pool in pools:
                for slot, n in ((0, 25), (1, 20), (2, 20)):
                    be.rope_append(pool, [(slot, n, later)], more, more)
        k.copy_(rows_of(rng, 40, 1, 64, False))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        step(pools[1])
        a = state(pools[0])
        same(a, state(pools[1]))
        for slot, n in ((0, 25), (1, 20), (2, 20)):
            table, held = a["page_table"].reshape(4, 8)[slot], n + (later if i else 0)
            ntok = [a["ntok"][p] for p in table[:-(-held // PAGE)]]
            want = [min(PAGE, held - PAGE * j) for j in range(len(ntok))]
            want[(n - 1) // PAGE] = (n - 1) % PAGE + 1
            assert ntok == want and a["n_logical"][slot] == len(want) and a["n_indexed"][slot] == held // PAGE


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("counts", [[248], [249], [265], [240, 8], [240, 9, 30], [3] * 64, [4] * 65, [100, 200, 300]])
@pytest.mark.parametrize("first", [15, 16])
def test_accepts_past_what_a_launch_takes(be, kind, counts, first):
    """248 tokens or 64 runs: rows, counts and seals of every slot."""
    rng = np.random.default_rng(len(counts) + first)
    n, batch = sum(counts), len(counts)
    pages = -(-(max(n, max(counts) + first)) // PAGE)
    pool = make(be, kind, batch + 1, 1, 64, pages)
    k = rows_of(rng, n + batch * first, 1, 64, False).cuda()
    be.rope_append(pool, [(s, 0, first) for s in range(batch)] + [(batch, 0, n)], k, k)
    index = rng.permutation(n)
    src = held_rows(pool, batch, n)
    be.kv_accept(pool, [(batch, s, first, c) for s, c in enumerate(counts)], index)
    a, at = state(pool), 0
    for s, c in enumerate(counts):
        got = held_rows(pool, s, first + c)
        for name in got:
            assert (got[name][first:] == src[name][torch.from_numpy(index[at:at + c]).cuda()]).all(), (s, name)
        at += c
        assert a["n_logical"][s] == a["length"][s] == -(-(first + c) // PAGE) and a["n_indexed"][s] == (first + c) // PAGE
        table = a["page_table"].reshape(-1, pages)[s]
        assert [a["ntok"][p] for p in table[:a["length"][s]]] == [min(PAGE, first + c - PAGE * j) for j in range(a["length"][s])]
        rows = got["k"].double() * (got["k_scale"].double()[..., None] if kind == "int8" else 1.0)
        for j in range((first + c) // PAGE):
            x = rows[PAGE * j:PAGE * j + PAGE, 0].cpu().numpy()
            # sixteen products and fifteen sums, each half a step of at most the sum of sizes
            assert (np.abs(a["centroid"][table[j]] - x.mean(0)) <= 31 * 2.0 ** -24 * np.abs(x).mean(0)).all()


def test_more_pages_than_a_grid_holds(be):
    """2^24 - 1 pages in a row, and three more, which go into another launch."""
    most = (1 << 24) - 1
    n, hd = most * PAGE, 8
    pool = make(be, "int8", 2, 1, hd, most)
    t = pool.tensors()
    k = torch.zeros(n + 40, 1, hd, dtype=torch.bfloat16, device="cuda")
    for i in (0, 5, n - 1, n, n + 39):
        k[i] = 1.0 + i % 7
    be.rope_append(pool, [(0, 0, n), (1, 0, 40)], k, k)
    assert list(pool.fetch("n_logical", 2, np.int32)) == [most, 3] and list(pool.fetch("n_indexed", 2, np.int32)) == [most, 2]
    pages = [pool.layer_pages(s) for s in range(2)]
    for i in (0, 5, 6, n - 1, n, n + 1, n + 39):
        page, off = pages[int(i >= n)][i % n // PAGE], i % n % PAGE
        want = k[i, 0].float()
        assert (t["k"][page, 0, off] == (127 if float(want[0]) else 0)).all()
        assert float(t["k_scale"][page, 0, off]) == (np.float32(want[0].item()) / np.float32(127) if float(want[0]) else 1.0)
