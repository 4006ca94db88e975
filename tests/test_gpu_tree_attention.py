"""Attention of trees of drafts (be42_tree_attention) against float64 over the
pages' own values; tolerances as for the attention behind a prefix: a score's
error d is hd * 2^-22 * scale * max_t sum_i |q_i k_ti| / sqrt(hd) + 2^-22 of the
score, the output's 2 d max|v| + 2^-20 max|v|; bf16 queries add the rounding of
the weights to 16 bits, 2^-16 of the sum of sizes, and of the output, 2^-8 of
itself."""
import math

import numpy as np
import pytest
import torch

from test_gpu_prefix_attention import PAGE, make_pool, pool_of, whole_numbers

pytestmark = pytest.mark.gpu


def trees_of(rng, sizes, kind="bushy"):
    """Parents of every draft, within its tree."""
    out = []
    for n in sizes:
        if kind == "chain":
            out.append(np.arange(n) - 1)
        elif kind == "roots":
            out.append(np.full(n, -1))
        else:
            out.append(np.array([rng.integers(max(-1, i - 6), i) for i in range(n)], np.int64))
    return np.concatenate(out + [np.zeros(0, np.int64)]).astype(np.int32)


def path(parents, i):
    seen = []
    while i >= 0:
        seen.append(i)
        i = parents[i] if parents[i] < i else -1
    return seen


def reference(q, k, v, H, scale, starts, parents, draft, slots, lens, max_len):
    """Output, tolerance of fp32 queries, sum of weighted sizes; NaN where no tree
    has the row."""
    n, _, hd = q.shape
    out, tol, size = np.full((n, H, hd), np.nan), np.zeros((n, H)), np.zeros((n, H, hd))
    for b in range(len(starts) - 1):
        lo, hi = starts[b], starts[b + 1]
        ctx = min(lens[b], max_len)
        ctx = max(min(ctx, len(k[slots[b]])), 0) if 0 <= slots[b] < len(k) else 0
        for i in range(lo, hi):
            at = [lo + j for j in path(parents[lo:hi], i - lo) if lo + j < len(k[draft])]
            kk = np.concatenate([k[slots[b]][:ctx] if ctx else k[draft][:0], k[draft][at]])
            vv = np.concatenate([v[slots[b]][:ctx] if ctx else v[draft][:0], v[draft][at]])
            if not len(kk):
                out[i] = 0
                continue
            g = H // kk.shape[1]
            for kvh in range(kk.shape[1]):
                K, V, h = kk[:, kvh], vv[:, kvh], slice(kvh * g, (kvh + 1) * g)
                s = q[i, h] @ K.T * scale
                w = np.exp(s - s.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                out[i, h], size[i, h] = w @ V, w @ np.abs(V)
                d = hd * 2.0 ** -22 * abs(scale) * (np.abs(q[i, h]) @ np.abs(K).T).max(1) / math.sqrt(hd) + 2.0 ** -22 * np.abs(s).max(1)
                tol[i, h] = (2 * d + 2.0 ** -20) * np.abs(V).max()
    return out, tol, size


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def check(got, q, k, v, H, scale, starts, parents, draft, slots, lens, max_len):
    want, tol, size = reference(q.double().numpy(), k, v, H, scale, starts, parents, draft, slots, lens, max_len)
    tol = np.broadcast_to(tol[..., None], want.shape)
    if q.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * np.abs(want) + 2.0 ** -16 * size
    rows = ~np.isnan(want[:, 0, 0])
    off = np.abs(got.cpu().double().numpy() - want)[rows]
    assert np.isfinite(off).all() and (off <= tol[rows]).all(), (off / np.maximum(tol[rows], 1e-300)).max()


def run(be, pool, k, v, q, H, starts, parents, draft, slots, lens, max_len, max_tree=None, give=("parents", "slots", "lens"), **kw):
    scale = kw.pop("scale", 1.0 / math.sqrt(q.shape[2]))
    sizes = np.diff(starts)
    got = be.tree_attention(pool, q.cuda(), ints(starts), ints(parents) if "parents" in give else None, draft, scale,
                            max_tree or max(1, int(sizes.max())), slots=ints(slots) if "slots" in give else None,
                            lens=ints(lens) if "lens" in give else None, max_len=max_len, **kw)
    assert got.dtype == q.dtype and got.shape == q.shape
    check(got, q, k, v, H, scale, starts, parents, draft, slots, lens, max_len)
    return got


def queries(seed, n, H, hd, bf16):
    q = torch.randn(n, H, hd, generator=torch.Generator().manual_seed(seed))
    return q.bfloat16() if bf16 else q


def starts_of(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kvh,hd", [(8, 8, 64), (6, 2, 128), (4, 1, 64), (20, 1, 128), (3, 3, 128), (72, 2, 64)])
@pytest.mark.parametrize("far", [0, 3000])
def test_heads(be, kind, bf16, heads, kvh, hd, far):
    """In one launch, and in parts."""
    sizes, lens = [3, 9, 1, 17], [0, 5, 40, 333 + far]
    pool, k, v = make_pool(be, kind, 5, kvh, hd, lens + [30], 1)
    parents = trees_of(np.random.default_rng(2), sizes)
    whole = be.lib.be42_tree_attention_workspace_bytes(30, 4, heads, kvh, hd, 17, 333 + far) == 16
    assert whole == (far == 0)
    run(be, pool, k, v, queries(2, 30, heads, hd, bf16), heads, starts_of(sizes), parents, 4, [0, 1, 2, 3], lens, 333 + far)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 500, 511, 513, 1000, 2049, 5003])
def test_context_lengths(be, kind, ctx):
    sizes, lens = [5, 2, 11], [ctx, max(ctx - 1, 0), ctx // 2]
    pool, k, v = make_pool(be, kind, 4, 2, 128, [max(n, 1) for n in lens] + [18], 3 + ctx)
    run(be, pool, k, v, queries(4, 18, 8, 128, False), 8, starts_of(sizes), trees_of(np.random.default_rng(5), sizes), 3, [0, 1, 2], lens, ctx)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("shape", ["bushy", "chain", "roots"])
@pytest.mark.parametrize("sizes,ctx", [([1], 20), ([16, 16], 20), ([15, 17, 1], 900), ([64, 3], 100), ([33, 0, 64, 0], 1500), ([256], 700),
                                       ([200, 256, 130], 40), ([1] * 40, 60), ([1] * 70 + [9], 1300)])
def test_tree_sizes(be, kind, bf16, shape, sizes, ctx):
    """Trees that begin and end anywhere in a page, empty ones, the largest; tiles of
    16, 64 and 128 rows."""
    rng = np.random.default_rng(sum(sizes))
    lens = rng.integers(0, ctx + 1, len(sizes))
    lens[0] = ctx
    n = sum(sizes)
    pool, k, v = make_pool(be, kind, len(sizes) + 1, 2, 64, list(lens) + [n], 6)
    q = queries(7, n, 6, 64, bf16)
    parents = trees_of(rng, sizes, shape)
    run(be, pool, k, v, q, 6, starts_of(sizes), parents, len(sizes), range(len(sizes)), lens, ctx,
        give=("slots", "lens") if shape == "chain" else ("parents", "slots", "lens"))


@pytest.mark.parametrize("far", [0, 2000])
def test_slots_of_all_kinds(be, far):
    """One context for several trees, slots outside the pool, lengths past what a slot
    holds and past max_len, none given; a drafts' slot that holds fewer than there are."""
    held = [40, 100 + far, 7, 25]
    pool, k, v = make_pool(be, "bf16", 4, 2, 64, held, 8)
    sizes = [4, 7, 3, 5, 6, 8]
    starts, parents = starts_of(sizes), trees_of(np.random.default_rng(9), sizes)
    q = queries(10, 33, 4, 64, False)
    run(be, pool, k, v, q, 4, starts, parents, 3, [1, 1, -1, 4, 0, 2 ** 31 - 1], [100 + far, 50, 30, 30, 1 << 30, 5], 90 + far)
    run(be, pool, k, v, q, 4, starts, parents, 3, [0, 1, 2, 2, 1, 0], [-5, 3, 0, 7, 0, 0], 100 + far)
    few = starts_of([4, 7, 3])
    run(be, pool, k, v, q[:14], 4, few, parents[:14], 3, range(3), [1 << 30] * 3, 100 + far, give=("parents",))
    full = pool.max_logical * PAGE
    got = be.tree_attention(pool, q[:14].cuda(), ints(few), ints(parents[:14]), 3, 0.125, 7)
    check(got, q[:14], k, v, 4, 0.125, few, parents[:14], 3, range(3), [full] * 3, full)


@pytest.mark.parametrize("ctx", [100, 3000])
def test_rows_of_no_tree_stay(be, ctx):
    """Drafts before the first tree, behind the last, and past max_tree."""
    pool, k, v = make_pool(be, "bf16", 3, 2, 64, [ctx, 50, 60], 11)
    q = queries(12, 60, 4, 64, False)
    starts = [5, 25, 48]
    parents = trees_of(np.random.default_rng(13), [5, 20, 23, 12])
    for max_tree in (23, 9):
        out = torch.full((60, 4, 64), 7.0, device="cuda")
        be.tree_attention(pool, q.cuda(), ints(starts), ints(parents), 2, 0.125, max_tree, slots=ints([0, 1]), lens=ints([ctx, 50]),
                          max_len=ctx, out=out)
        have = np.zeros(60, bool)
        for a, b in zip(starts, starts[1:]):
            have[a:min(b, a + max_tree)] = True
        assert (out[torch.from_numpy(~have).cuda()] == 7).all()
        want, tol, _ = reference(q.double().numpy(), k, v, 4, 0.125, starts, parents, 2, [0, 1], [ctx, 50], ctx)
        off = np.abs(out.cpu().double().numpy() - want)[have]
        assert (off <= tol[have][..., None]).all()


def test_parents_that_are_no_earlier_draft(be):
    """End the path, whatever they hold."""
    pool, k, v = make_pool(be, "bf16", 2, 1, 64, [20, 12], 14)
    bad = np.array([-1, 0, 2, 7, -9, 2 ** 31 - 1, -2 ** 31, 6, 8, 8, 3, 10], np.int64)
    run(be, pool, k, v, queries(15, 12, 2, 64, False), 2, [0, 12], bad.astype(np.int32), 1, [0], [20], 20)


def test_starts_outside(be):
    """Bounds of trees that no call should give: reads and writes stay inside."""
    pool, k, v = make_pool(be, "bf16", 2, 1, 64, [20, 30], 16)
    q = queries(17, 30, 2, 64, False).cuda()
    parents = ints(trees_of(np.random.default_rng(1), [30]))
    for starts in ([-5, 40], [2 ** 31 - 1, -2 ** 31], [30, 31], [10, 2 ** 31 - 1], [-2 ** 31, 5]):
        out = torch.full((30, 2, 64), 7.0, device="cuda")
        be.tree_attention(pool, q, ints(starts), parents, 1, 0.125, 30, lens=ints([20]), max_len=20, out=out)
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("ctx", [50, 1600])
def test_bad_drafts_reach_who_sees_them(be, kind, bf16, bad, where, ctx):
    """Not their siblings, not another tree's, not the drafts above them."""
    sizes = [13, 40, 6]
    rng = np.random.default_rng(18)
    n, kvh, hd, H = sum(sizes), 2, 64, 4
    pool, k, v = make_pool(be, kind, 4, kvh, hd, [ctx, 30, 9, n], 19)
    starts, parents = starts_of(sizes), trees_of(rng, sizes)
    q = queries(20, n, H, hd, bf16)
    args = (ints(starts), ints(parents), 3, 0.125, 40)
    kw = dict(slots=ints([0, 1, 2]), lens=ints([ctx, 30, 9]), max_len=ctx)
    clean = be.tree_attention(pool, q.cuda(), *args, **kw)
    t = pool.tensors()
    hit = [4, 13 + 7, 13 + 30]
    for i in hit:
        page, off = int(pool.layer_pages(3)[i // PAGE]), i % PAGE
        if kind == "int8":
            t[where + "_scale"][page, :, off] = bad
        elif where == "k":
            t["k"][page, :, off, 5] = bad
        else:
            t["v"][page, :, 5, off] = bad
    got = be.tree_attention(pool, q.cuda(), *args, **kw)
    for b in range(3):
        lo, hi = starts[b], starts[b + 1]
        for i in range(lo, hi):
            sees = [lo + j in hit for j in path(parents[lo:hi], i - lo)]
            if any(sees):
                if math.isnan(bad) or where == "v":
                    assert not torch.isfinite(got[i].float()).all(), i
            elif kind == "int8":
                assert (got[i] == clean[i]).all(), i
            else:
                # its values' products are formed one token at a time: other sums
                assert (got[i].double() - clean[i].double()).abs().max() <= (2.0 ** -7 if bf16 else 2.0 ** -19) * 5, i


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("H,ctx", [(4, 50), (4, 1603), (32, 1603), (60, 1603)])
def test_what_lies_behind_the_lengths(be, kind, bf16, where, H, ctx):
    """NaN in tokens of a slot from its length on, and in drafts behind the last tree."""
    sizes, kvh, hd = [9, 8], 2, 128
    pool, k, v = make_pool(be, kind, 3, kvh, hd, [ctx + 40, 45, 30], 28)
    t, lens = pool.tensors(), [ctx, 13]
    for slot, at, held in ((0, ctx, ctx + 40), (1, 13, 45), (2, 17, 30)):
        for i in range(at, held):
            page, off = int(pool.layer_pages(slot)[i // PAGE]), i % PAGE
            if kind == "int8":
                t[where + "_scale"][page, :, off] = math.nan
            elif where == "k":
                t["k"][page, :, off] = math.nan
            else:
                t["v"][page, :, :, off] = math.nan
    run(be, pool, k, v, queries(29, 17, H, hd, bf16), H, starts_of(sizes), trees_of(np.random.default_rng(3), sizes), 2, [0, 1], lens, ctx)


@pytest.mark.parametrize("n", [256, 255, 129, 33])
@pytest.mark.parametrize("shape", ["chain", "one"])
def test_the_deepest_and_the_widest(be, n, shape):
    """A chain of all drafts behind drafts of another tree, and one root with all others below it."""
    parents = np.concatenate([trees_of(None, [21], "chain"), np.arange(n) - 1 if shape == "chain" else np.minimum(np.arange(n), 1) - 1])
    pool, k, v = make_pool(be, "bf16", 3, 1, 64, [700, 5, 21 + n], 30)
    run(be, pool, k, v, queries(31, 21 + n, 3, 64, False), 3, [0, 21, 21 + n], parents, 2, [0, 1], [700, 5], 700, max_tree=256)


def test_infinite_values_give_infinities(be):
    """Of a token that weighs something: with its sign."""
    pool, k, v = make_pool(be, "bf16", 2, 1, 64, [20, 6], 21)
    t = pool.tensors()
    t["v"][int(pool.layer_pages(1)[0]), 0, 3, 2] = -math.inf
    parents = [-1, 0, 0, 2, 1, 3]
    got = be.tree_attention(pool, queries(22, 6, 1, 64, False).cuda(), ints([0, 6]), ints(parents), 1, 0.125, 6, lens=ints([20]),
                            slots=ints([0]), max_len=20)
    for i in range(6):
        if i in (2, 3, 5):
            assert got[i, 0, 3] == -math.inf and torch.isfinite(got[i, 0, :3]).all() and torch.isfinite(got[i, 0, 4:]).all()
        else:
            assert torch.isfinite(got[i]).all()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("ctx", [40, 1700])
@pytest.mark.parametrize("scale", [0.01, 1.0, 1e9, -1e9, 1e30])
def test_scores_of_any_size(be, kind, bf16, ctx, scale):
    """Scores of whole numbers, exact; V of whole numbers below 128: weights are off by
    2^-22 of themselves, sums by 2^-20."""
    kvh, hd, H, sizes = 2, 128, 8, [30, 20]
    rng = np.random.default_rng(ctx)
    held = [ctx, ctx // 2, 50]
    k = [whole_numbers(rng, n, kvh, hd, 4) for n in held]
    v = [whole_numbers(rng, n, kvh, hd, 100) for n in held]
    k[2][3] = k[0][ctx // 2] = k[2][0]
    pool = pool_of(be, kind, k, v)
    q = torch.from_numpy(rng.integers(-3, 4, (50, H, hd)).astype(np.float32))
    q = q.bfloat16() if bf16 else q
    starts, parents = starts_of(sizes), trees_of(rng, sizes)
    got = be.tree_attention(pool, q.cuda(), ints(starts), ints(parents), 2, scale, 30, slots=ints([0, 1]), lens=ints(held[:2]), max_len=ctx)
    k, v = ([a.astype(np.float64) for a in x] for x in (k, v))
    want = reference(q.double().numpy(), k, v, H, float(np.float32(scale)), starts, parents, 2, [0, 1], held[:2], ctx)[0]
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= 127 * 2.0 ** -19 + (2.0 ** -7 * 127 if bf16 else 0.0)).all(), off.max()


@pytest.mark.parametrize("ctx", [60, 2500])
def test_strided_queries_streams_and_replays(be, ctx):
    """Queries as a view; on a stream of the caller's; captured with a workspace and
    replayed with other trees, slots and lengths."""
    sizes = [20, 31, 13]
    n, H, kvh, hd = 64, 8, 2, 128
    pool, k, v = make_pool(be, "bf16", 4, kvh, hd, [ctx, ctx - 7, 40, n], 23)
    wide = torch.randn(n, H + 3, hd, device="cuda")
    q = wide[:, 1:H + 1]
    starts, lens, slots = ints(starts_of(sizes)), ints([ctx, ctx - 7, 40]), ints([0, 1, 2])
    parents = ints(trees_of(np.random.default_rng(24), sizes))
    need = be.lib.be42_tree_attention_workspace_bytes(n, 3, H, kvh, hd, 40, ctx)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = torch.empty(n, H, hd, device="cuda")

    def call():
        return be.tree_attention(pool, q, starts, parents, 3, 0.09, 40, slots=slots, lens=lens, max_len=ctx, out=out, workspace=ws)

    def right():
        check(out, q.cpu(), k, v, H, 0.09, starts.cpu().numpy(), parents.cpu().numpy(), 3, slots.cpu().numpy(), lens.cpu().numpy(), ctx)

    call()
    right()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out.zero_()
        call()
    s.synchronize()
    right()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    rng = np.random.default_rng(25)
    for more in ([20, 31, 13], [40, 4, 20], [1, 0, 30], [22, 40, 2]):
        starts.copy_(ints(starts_of(more)))
        parents.copy_(ints(np.concatenate([trees_of(rng, more), np.zeros(n - sum(more), np.int32)])))
        lens.copy_(ints(rng.integers(0, ctx, 3)))
        slots.copy_(ints(rng.permutation(3)))
        wide.copy_(torch.randn(n, H + 3, hd, device="cuda"))
        out.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        right()
        assert (out[sum(more):] == 7).all()
        first = out.clone()
        g.replay()
        torch.cuda.synchronize()
        assert (out == first).all()


def test_captured_without_a_workspace_is_refused(be):
    import be42
    pool, k, v = make_pool(be, "bf16", 2, 1, 64, [20, 6], 26)
    q, st = torch.zeros(6, 1, 64, device="cuda"), ints([0, 6])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            x = q + 1
            a = (pool.handle, x.data_ptr(), 0, 64, 6, 1, st.data_ptr(), 1, 6, None, 1, None, None, 20, 0.1, x.data_ptr(), None, 0, s.cuda_stream)
            assert be.lib.be42_tree_attention(*a) == -1 and "workspace" in be.last_error()
    assert be42


def test_python_refusals(be):
    import be42
    pool, k, v = make_pool(be, "bf16", 2, 2, 64, [20, 6], 27)
    q, st, par = torch.zeros(6, 4, 64, device="cuda"), ints([0, 6]), ints([-1] * 6)
    ok = dict(q=q, starts=st, parents=par, draft_slot=1, scale=0.1, max_tree=6, slots=ints([0]), lens=ints([20]), max_len=20)
    be.tree_attention(pool, **ok)
    for bad in (dict(q=q.double()), dict(q=q[..., :32]), dict(q=q.cpu()), dict(q=q.transpose(0, 1)), dict(starts=st.long()),
                dict(starts=st[:0]), dict(parents=par[:5]), dict(slots=ints([0, 1])), dict(lens=ints([[1]])), dict(max_tree=1 << 32),
                dict(draft_slot=-1), dict(max_len=1 << 31), dict(out=q.bfloat16()), dict(out=q[:5]), dict(scale=math.nan),
                dict(workspace=torch.empty(4, dtype=torch.uint8, device="cuda")), dict(q=q[:, :3])):
        with pytest.raises(be42.Be42Error):
            be.tree_attention(pool, **dict(ok, **bad))
    assert be.tree_attention(pool, **dict(ok, q=q[:0], parents=par[:0])).shape == (0, 4, 64)
