"""Norms + rotation + append (be42_rope_append) and accepted drafts
(be42_kv_accept).

Queries against the formula in 64 bits.  Tolerance: a normalised element is
rounded to fp32 once (2^-24 of itself); of the rotation's two products one is
rounded, and their sum: 2^-24 of |x0 c|, |x1 s| each for the elements, of |x1 s|
for its product and of the sum, at most 4 * 2^-24 * (|x0 c| + |x1 s|) in all; bf16
outputs add half a step, 2^-8 of themselves.  The slack of 1 + 2^-20 is for what
64 bits lose and products of these bounds.  Pages are what be42_kv_append stores of
the rotated rows, to the bit."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE, EPS = 16, 1e-5


def make(be, kind, slots, kvh, hd, pages, seed=0):
    import be42
    hp = np.random.default_rng(seed).standard_normal((hd, 16)).astype(np.float32)
    return be.kv_pool(be42.KV_BF16 if kind == "bf16" else be42.KV_INT8, slots, kvh, hd, pages, hp)


def state(pool):
    """Everything that a pool holds, on the device and beside it."""
    cap, n = pool.s.capacity, pool.n_layers * pool.max_logical
    t = {k: v.view(torch.int16).cpu().numpy() if v.dtype == torch.bfloat16 else v.cpu().numpy() for k, v in pool.tensors().items()}
    for name, count, dt in (("ntok", cap, np.int32), ("page_table", n, np.int32), ("n_logical", pool.n_layers, np.int32),
                            ("page_hash", n, np.uint16), ("n_indexed", pool.n_layers, np.int32)):
        t[name] = pool.fetch(name, count, dt)
    pt, free, top, length = pool.export()
    return dict(t, host_table=pt, free=free[:top + 1], length=length)


def same(a, b, but=()):
    for k in a:
        if k not in but:
            assert a[k].shape == b[k].shape and (a[k].view(np.uint8) == b[k].view(np.uint8)).all(), k


def tables(n, half, seed=1):
    a = np.random.default_rng(seed).uniform(-math.pi, math.pi, (n, half))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def rotated(x, w, cos, sin, pos, dim, interleaved):
    """64 bits: [n][heads][hd] and the tolerance of each element."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(EPS))) * w.astype(np.float64)
    y, tol, half = x.copy(), np.abs(x) * 2.0 ** -24, dim // 2
    if half:
        i0, i1 = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, half), slice(half, dim))
        for t, p in enumerate(pos):
            if not 0 <= p < len(cos):
                continue
            c, s = cos[p].astype(np.float64), sin[p].astype(np.float64)
            a, b = x[t][:, i0], x[t][:, i1]
            y[t][:, i0], y[t][:, i1] = a * c - b * s, a * s + b * c
            tol[t][:, i0] = 4 * 2.0 ** -24 * (np.abs(a * c) + np.abs(b * s))
            tol[t][:, i1] = 4 * 2.0 ** -24 * (np.abs(a * s) + np.abs(b * c))
    return y, tol * (1 + 2.0 ** -20) + 1e-45


def rows_of(rng, n, heads, hd, bf16):
    x = torch.from_numpy((rng.standard_normal((n, heads, hd)) * np.exp(rng.standard_normal((n, heads, 1)))).astype(np.float32))
    return x.bfloat16() if bf16 else x


def weight(rng, hd):
    return torch.from_numpy((1 + 0.3 * rng.standard_normal(hd)).astype(np.float32)).bfloat16()


def check_rows(got, x, w, cos, sin, pos, dim, interleaved):
    want, tol = rotated(x.double().numpy(), None if w is None else w.double().numpy(), cos, sin, pos, dim, interleaved)
    if got.dtype == torch.bfloat16:
        tol = tol * 1.01 + 2.0 ** -8 * np.abs(want)
    off = np.abs(got.cpu().double().numpy() - want)
    assert (off <= tol).all(), (off / tol).max()


def dev(x):
    return None if x is None else x.cuda()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads,kvh,hd,dim,inter", [
    (8, 8, 64, 64, False), (8, 2, 128, 128, False), (24, 8, 128, 128, True), (6, 2, 128, 64, False), (6, 2, 64, 32, True),
    (4, 1, 256, 256, False), (4, 2, 256, 64, True), (5, 1, 8, 8, False), (3, 3, 40, 40, False), (2, 1, 72, 20, True),
    (4, 4, 136, 136, False), (36, 1, 64, 64, False), (4, 2, 64, 0, False), (4, 2, 64, 2, False)])
def test_values_and_pages(be, kind, bf16, norm, heads, kvh, hd, dim, inter):
    """Queries by the formula; pages as be42_kv_append stores the rotated keys, which
    are those that the same call gives for them as queries."""
    import be42
    rng = np.random.default_rng(heads + hd + dim)
    runs = [(2, 0, 37), (0, 0, 1), (1, 0, 16)]
    n = 54
    pos = np.concatenate([a + np.arange(c) for _, a, c in runs])
    cos, sin = tables(30, dim // 2)                   # positions from 30 on are not rotated
    q, k, v = (rows_of(rng, n, h, hd, bf16) for h in (heads, kvh, kvh))
    qw, kw = (weight(rng, hd), weight(rng, hd)) if norm else (None, None)
    rope = be42.Rope(torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda(), interleaved=inter)
    pool, by_hand = (make(be, kind, 3, kvh, hd, 4) for _ in range(2))
    args = dict(rope=rope, q_norm=dev(qw), k_norm=dev(kw), eps=EPS)
    got = be.rope_append(pool, runs, k.cuda(), v.cuda(), q=q.cuda(), **args)
    assert got.dtype == q.dtype
    check_rows(got, q, qw, cos, sin, pos, dim, inter)
    # fp32 rows of the same values, so that the rotated keys are not rounded
    scratch = make(be, kind, 3, kvh, hd, 4)
    keys = be.rope_append(scratch, runs, k.float().cuda(), v.float().cuda(), q=k.float().cuda(), rope=rope, q_norm=dev(kw),
                          k_norm=dev(kw), eps=EPS)
    check_rows(keys, k.float(), kw, cos, sin, pos, dim, inter)
    at = 0
    for slot, p0, c in runs:
        by_hand.append(slot, keys[at:at + c].reshape(c, -1), v[at:at + c].float().cuda().reshape(c, -1), p0)
        at += c
    same(state(pool), state(by_hand))
    same(state(scratch), state(by_hand))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_rotation_as_the_decode_step(be, kind):
    """Without norms: y0 = fma(x0, c, -(x1 s)), y1 = fma(x0, s, x1 c), each product of
    the second element rounded first."""
    import be42
    rng = np.random.default_rng(3)
    n, heads, hd = 40, 6, 128
    cos, sin = tables(64, hd // 2)
    q, k, v = (rows_of(rng, n, h, hd, False) for h in (heads, 2, 2))
    pool = make(be, kind, 1, 2, hd, 4)
    got = be.rope_append(pool, [(0, 0, n)], k.cuda(), v.cuda(), q=q.cuda(),
                         rope=be42.Rope(torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda())).cpu().numpy()
    x0, x1 = q.numpy()[..., :64], q.numpy()[..., 64:]
    c, s = cos[:n, None], sin[:n, None]
    a = (x0.astype(np.float64) * c - (x1 * s)).astype(np.float32)
    b = (x0.astype(np.float64) * s + (x1 * c)).astype(np.float32)
    assert (got == np.concatenate([a, b], -1)).all()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_appends_that_go_on(be, kind):
    """Runs that begin inside pages, fill them, and take positions again: as
    be42_kv_append of the same rows; a page that is written to its end again gets the
    centroid and hash of what it now holds."""
    rng = np.random.default_rng(5)
    kvh, hd = 2, 64
    pool, by_hand = (make(be, kind, 5, kvh, hd, 8) for _ in range(2))
    for runs in ([(0, 0, 5), (3, 0, 20), (1, 0, 0)], [(3, 20, 1), (0, 5, 11)], [(4, 0, 128), (0, 16, 1)], [(0, 17, 40), (1, 0, 15)],
                 [(1, 15, 1), (2, 0, 33), (3, 21, 11)]):
        n = sum(r[2] for r in runs)
        k, v = (rows_of(rng, n, kvh, hd, False).cuda() for _ in range(2))
        assert be.rope_append(pool, runs, k, v) is None
        at = 0
        for slot, p0, c in runs:
            if c:
                by_hand.append(slot, k[at:at + c].reshape(c, -1), v[at:at + c].reshape(c, -1), p0)
            at += c
        same(state(pool), state(by_hand))
    # positions 3 .. 40 of slot 0 again: its first two pages are sealed once more
    k, v = (rows_of(rng, 38, kvh, hd, False).cuda() for _ in range(2))
    be.rope_append(pool, [(0, 3, 38)], k, v)
    by_hand.append(0, k.reshape(38, -1), v.reshape(38, -1), 3)
    a, b = state(pool), state(by_hand)
    same(a, b, ("centroid", "page_hash"))
    fresh = make(be, kind, 1, kvh, hd, 8)
    t = pool.tensors()
    pages = torch.from_numpy(pool.layer_pages(0)).cuda().long()
    kk = t["k"][pages].float() if kind == "bf16" else t["k"][pages].float() * t["k_scale"][pages][..., None]
    kk = kk.transpose(1, 2).reshape(-1, kvh * hd)[:32].contiguous()
    fresh.append(0, kk, kk, 0)
    if kind == "bf16":                                # (codes of decoded codes may be others)
        for j in range(2):
            assert (t["centroid"][pages[j]] == fresh.tensors()["centroid"][int(fresh.layer_pages(0)[j])]).all()
        assert (a["page_hash"][:2] == state(fresh)["page_hash"][:2]).all()
    c = t["centroid"][pages[:2]].double().cpu()
    want = kk.view(2, 16, kvh, hd)[:, :, 0].double().mean(1).cpu()
    # sixteen terms: fifteen sums, each half a step of at most the sum of sizes
    assert ((c - want).abs() <= 15 * 2.0 ** -24 * kk.view(2, 16, kvh, hd)[:, :, 0].double().abs().mean(1).cpu()).all()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("lens", [[11] * 150, [700] * 17, [10245], [10239, 3, 40], [1] * 64, [1] * 65, [0, 16, 0, 17]])
def test_many_runs_and_pages(be, kind, lens):
    """Past what one launch takes: 64 runs, 640 pages."""
    rng = np.random.default_rng(len(lens))
    kvh, hd = 1, 64
    pool, by_hand = (make(be, kind, len(lens), kvh, hd, -(-max(lens) // PAGE)) for _ in range(2))
    n = sum(lens)
    k, v = (rows_of(rng, n, kvh, hd, False).cuda() for _ in range(2))
    be.rope_append(pool, [(s, 0, c) for s, c in enumerate(lens)], k, v)
    at = 0
    for s, c in enumerate(lens):
        if c:
            by_hand.append(s, k[at:at + c].reshape(c, -1), v[at:at + c].reshape(c, -1), 0)
        at += c
    same(state(pool), state(by_hand))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("mix", [False, True])
def test_pages_apart_and_in_a_row(be, kind, mix):
    """600 pages of which no two follow one another, past what one launch lists; or
    stretches of such and of others, up and down."""
    rng = np.random.default_rng(9)
    kvh, hd, per = 1, 64, 600
    pool = make(be, kind, 4, kvh, hd, per)
    row = torch.zeros(2 * per * PAGE, kvh, hd, device="cuda")
    stretch = [1] * per if not mix else [1, 2, 15, 16, 17, 40, 1, 1, 300, 3, 1, 20, 16]
    at = 0
    for n in stretch:
        c = min(n, per - at) * PAGE
        if c:
            be.rope_append(pool, [(0, at * PAGE, c), (1, at * PAGE, c)], row[:2 * c], row[:2 * c])
            at += c // PAGE
    pool.reset(0)
    n = at * PAGE - 5
    k, v = (rows_of(rng, n + 30, kvh, hd, False).cuda() for _ in range(2))
    be.rope_append(pool, [(2, 0, 30), (0, 0, n)], k, v)
    steps = np.diff(pool.layer_pages(0))
    assert ((np.abs(steps) == 1).sum() > 4) == mix
    other = make(be, kind, 2, kvh, hd, per)
    other.append(0, k[30:].reshape(n, -1), v[30:].reshape(n, -1), 0)
    other.append(1, k[:30].reshape(30, -1), v[:30].reshape(30, -1), 0)
    for a, b, m in ((0, 0, n), (2, 1, 30)):
        x, y = held_rows(pool, a, m), held_rows(other, b, m)
        for name in x:
            assert (x[name] == y[name]).all(), name
    x, y = state(pool), state(other)
    assert (x["page_table"].reshape(4, per) == x["host_table"].reshape(4, per)).all()
    assert (x["page_hash"].reshape(4, per)[0][:n // PAGE] == y["page_hash"].reshape(2, per)[0][:n // PAGE]).all()
    assert (x["ntok"][pool.layer_pages(0)] == y["ntok"][other.layer_pages(0)]).all()


def test_views_positions_and_in_place(be):
    """q, k and v as views of one product, queries in place and into another view, and
    angles that are not the places', far and negative ones (no rotation) among them."""
    import be42
    rng = np.random.default_rng(9)
    n, H, kvh, hd = 29, 6, 2, 128
    cos, sin = tables(50, hd // 2)
    rope = be42.Rope(torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda())
    pos = rng.integers(0, 50, n).astype(np.int32)
    pos[[3, 7, 8]] = [50, -1, 2 ** 31 - 1]
    at = torch.from_numpy(pos).cuda()
    for bf16 in (False, True):
        x = rows_of(rng, n, H + 2 * kvh + 1, hd, bf16).cuda()
        q, k, v = x[:, 1:H + 1], x[:, H + 1:H + 1 + kvh], x[:, H + 1 + kvh:]
        before = x.clone()
        pool, other, third = (make(be, "bf16", 1, kvh, hd, 2) for _ in range(3))
        got = be.rope_append(pool, [(0, 0, n)], k, v, q=q, rope=rope, positions=at)
        check_rows(got, q.cpu(), None, cos, sin, pos, hd, False)
        assert (x == before).all()
        wide = torch.full((n, 2 * H, hd), 7.0, dtype=x.dtype, device="cuda")
        assert be.rope_append(third, [(0, 0, n)], k, v, q=q, rope=rope, positions=at, out=wide[:, H:]).data_ptr() == wide[:, H:].data_ptr()
        assert (wide[:, H:] == got).all() and (wide[:, :H] == 7).all()
        be.rope_append(other, [(0, 0, n)], k, v, q=q, rope=rope, positions=at, out=q)
        assert (q == got).all() and (x[:, H + 1:] == before[:, H + 1:]).all() and (x[:, 0] == before[:, 0]).all()
        same(state(pool), state(other))
        same(state(pool), state(third))


def test_unaligned_rows(be):
    """Rows that lie on no 16-byte word give what aligned ones give."""
    import be42
    rng = np.random.default_rng(10)
    n, H, kvh, hd = 20, 4, 2, 64
    rope = be42.Rope(*(torch.from_numpy(a).cuda() for a in tables(50, hd // 2)))
    w = weight(rng, hd)
    odd = torch.empty(hd + 1, dtype=torch.bfloat16, device="cuda")[1:].copy_(w)
    for bf16 in (False, True):
        x = rows_of(rng, n, 1, (H + 2 * kvh) * hd, bf16).cuda()[:, 0]
        far = torch.empty(n, x.shape[1] + 3, dtype=x.dtype, device="cuda")[:, 1:-2].copy_(x)
        pools, got = [make(be, "int8", 1, kvh, hd, 2) for _ in range(2)], []
        for pool, y, ww in zip(pools, (x, far), (w.cuda(), odd)):
            q, k, v = (a.unflatten(1, (-1, hd)) for a in y.split([H * hd, kvh * hd, kvh * hd], 1))
            got.append(be.rope_append(pool, [(0, 0, n)], k, v, q=q, rope=rope, q_norm=ww, k_norm=ww))
        assert (got[0] == got[1]).all()
        same(state(pools[0]), state(pools[1]))


def test_a_bad_row_stays_alone(be):
    """Infinities and NaN in one token's rows reach no other row's."""
    import be42
    rng = np.random.default_rng(11)
    n, H, kvh, hd = 35, 4, 2, 64
    rope = be42.Rope(*(torch.from_numpy(a).cuda() for a in tables(50, hd // 2)))
    for kind in ("bf16", "int8"):
        q, k, v = (rows_of(rng, n, h, hd, False).cuda() for h in (H, kvh, kvh))
        w = weight(rng, hd).cuda()
        pools, got = [make(be, kind, 1, kvh, hd, 4) for _ in range(2)], []
        for pool, bad in zip(pools, (False, True)):
            a, b, c = q.clone(), k.clone(), v.clone()
            if bad:
                a[5, 1, 3], b[5, 0, 7], c[5, 1, 0] = math.nan, math.inf, -math.inf
            got.append(be.rope_append(pool, [(0, 0, n)], b, c, q=a, rope=rope, q_norm=w, k_norm=w))
        keep = [t for t in range(n) if t != 5]
        assert (got[0][keep] == got[1][keep]).all()
        for name in ("k", "v") if kind == "bf16" else ("k", "v", "k_scale", "v_scale"):
            for t in keep:
                page = int(pools[0].layer_pages(0)[t // PAGE])
                a, b = (p.tensors()[name][page] for p in pools)
                i = (slice(None), slice(None), t % PAGE) if kind == "bf16" and name == "v" else (slice(None), t % PAGE)
                assert (a[i] == b[i]).all(), (name, t)


def test_refusals_change_nothing(be):
    import be42
    pool = make(be, "bf16", 4, 2, 64, 4)
    k = torch.randn(40, 2, 64, device="cuda")
    be.rope_append(pool, [(0, 0, 20), (1, 0, 20)], k, k)
    before = state(pool)
    for runs, word in ([[(4, 0, 40)], "out of range"], [[(-1, 0, 40)], "out of range"], [[(0, 20, 20), (0, 40, 20)], "twice"],
                       [[(2, 0, 20), (2, 20, 20)], "twice"], [[(0, 40, 40)], "positions"], [[(0, 25, 40)], "positions"],
                       [[(2, 0, 30), (1, 49, 10)], "skips"], [[(0, -1, 40)], "positions"]):
        with pytest.raises(be42.Be42Error, match=word):
            be.rope_append(pool, runs, k, k)
        same(state(pool), before)
    taken = [pool.page_alloc() for _ in range(int(pool.export()[2]))]        # one is left
    held = state(pool)
    with pytest.raises(be42.Be42Error, match="exhausted"):
        be.rope_append(pool, [(0, 20, 5), (2, 0, 17), (1, 20, 18)], k, k)
    same(state(pool), held)
    for p in reversed(taken):
        pool.page_free(p)
    for bad in (dict(runs=[(2, 0, 39)]), dict(runs=[(2, 0, 41), (3, 0, -1)]), dict(v=k[:39]), dict(v=k.bfloat16()), dict(k=k.double()),
                dict(q=torch.randn(40, 3, 64, device="cuda")), dict(q=torch.randn(39, 4, 64, device="cuda")), dict(out=k),
                dict(positions=torch.zeros(40, dtype=torch.int64, device="cuda")), dict(k=k.transpose(0, 1)), dict(k=k[:, :1], v=k[:, :1]),
                dict(k_norm=torch.ones(64, device="cuda")), dict(q_norm=torch.ones(32, device="cuda", dtype=torch.bfloat16)),
                dict(k=k.cpu(), v=k.cpu())):
        a = dict(dict(runs=[(2, 0, 40)], k=k, v=k), **bad)
        with pytest.raises(be42.Be42Error):
            be.rope_append(pool, a.pop("runs"), a.pop("k"), a.pop("v"), **a)
    assert be.rope_append(pool, [], k[:0], k[:0]) is None
    assert be.rope_append(pool, [(2, 0, 0)], k[:0], k[:0], q=k[:0]).shape == (0, 2, 64)
    same(state(pool), before, ("free",))
    with pytest.raises(be42.Be42Error):
        be42.Rope(torch.zeros(4, 8, device="cuda"), torch.zeros(4, 7, device="cuda"))


def test_tensors_outlive_their_pool_object(be):
    pool = make(be, "bf16", 1, 1, 64, 2)
    k = torch.randn(20, 1, 64, device="cuda")
    be.rope_append(pool, [(0, 0, 20)], k, k)
    page = int(pool.layer_pages(0)[0])
    t = pool.tensors()
    del pool
    assert (t["k"][page, 0] == k[:16, 0].bfloat16()).all() and (t["v"][page, 0].t() == k[:16, 0].bfloat16()).all()


def filled(be, kind, kvh, hd, slots, pages, held, seed):
    pool = make(be, kind, slots, kvh, hd, pages, seed)
    rng = np.random.default_rng(seed)
    for s, n in enumerate(held):
        if n:
            pool.append(s, *(rows_of(rng, n, kvh, hd, False).cuda().reshape(n, -1) for _ in range(2)), 0)
    return pool


def held_rows(pool, slot, n):
    """K and V (codes and scales) of a slot's first n tokens."""
    t, pages = pool.tensors(), torch.from_numpy(pool.layer_pages(slot)).cuda().long()
    out = {}
    for name, x in t.items():
        if name == "centroid":
            continue
        y = x[pages]
        y = y.movedim(-1, 1) if name == "v" and "k_scale" not in t else y.transpose(1, 2)
        out[name] = y.flatten(0, 1)[:n].clone()
    return out


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("kvh,hd,batch,layers,drafts", [(2, 64, 3, 2, 20), (8, 128, 24, 28, 24), (1, 40, 70, 3, 7), (3, 256, 1, 1, 300),
                                                       (1, 64, 5, 40, 64)])
def test_accepted_drafts(be, kind, kvh, hd, batch, layers, drafts):
    """Rows, bit for bit; the tokens around them, tables, counts and seals as if they
    had been appended."""
    rng = np.random.default_rng(batch + layers)
    ctx = rng.integers(1, 60, batch)
    count = np.minimum(rng.integers(0, 9, batch), drafts) if drafts < 300 else np.array([290])
    count[0] = max(count[0], 1)
    if batch > 2:
        ctx[1], count[1], ctx[2], count[2] = 10, 6, 16, min(7, drafts)    # to a page's end; from a page's first place
    held = list(np.tile(ctx, layers)) + [batch * drafts] * layers
    pages = max(-(-batch * drafts // PAGE), 6, -(-int((ctx + count).max()) // PAGE))
    pool = filled(be, kind, kvh, hd, layers * (batch + 1), pages, held, 7)
    paths = [b * drafts + rng.permutation(drafts)[:c] for b, c in enumerate(count)]
    before = {s: held_rows(pool, s, n) for s, n in enumerate(held)}
    pages_before = state(pool)
    runs = np.array([(layers * batch, b, ctx[b], count[b]) for b in range(batch)])
    be.kv_accept(pool, runs, np.concatenate(paths), layers=layers, from_step=1, to_step=batch)
    after = state(pool)
    for l in range(layers):
        for b in range(batch):
            s, n = l * batch + b, int(ctx[b] + count[b])
            got, src = held_rows(pool, s, n), before[layers * batch + l]
            at = torch.from_numpy(paths[b]).cuda().long()
            for name in got:
                assert (got[name][:ctx[b]] == before[s][name]).all() and (got[name][ctx[b]:] == src[name][at]).all(), (l, b, name)
            assert after["length"][s] == after["n_logical"][s] == -(-n // PAGE) and after["n_indexed"][s] == n // PAGE
            table = after["page_table"].reshape(-1, pages)[s]
            assert (table == after["host_table"].reshape(-1, pages)[s]).all()
            assert after["ntok"][table[-(-n // PAGE) - 1]] == n - (n - 1) // PAGE * PAGE
            # the seal of the last full page, by appending the page's keys elsewhere
        assert (after["n_logical"][layers * batch + l] == pages_before["n_logical"][layers * batch + l])
    if kind == "bf16":
        b = int(np.argmax((ctx + count) // PAGE > ctx // PAGE))
        j = int(ctx[b] + count[b]) // PAGE - 1
        if j >= ctx[b] // PAGE:
            rows = held_rows(pool, b, (j + 1) * PAGE)
            other = make(be, kind, 1, kvh, hd, j + 1, 7)
            other.append(0, rows["k"].float().reshape((j + 1) * PAGE, -1), rows["v"].float().reshape((j + 1) * PAGE, -1), 0)
            o = state(other)
            assert after["page_hash"].reshape(-1, pages)[b][j] == o["page_hash"][j]
            assert (after["centroid"][after["page_table"].reshape(-1, pages)[b][j]] == o["centroid"][o["page_table"][j]]).all()


def test_replays_among_other_appends(be):
    """A captured append and accept whose pages were new: replayed behind appends that
    went on, which stay."""
    pool = filled(be, "bf16", 1, 64, 4, 4, [20, 10, 0, 0], 5)
    k = torch.randn(40, 1, 64, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        be.rope_append(pool, [(2, 0, 20)], k[:20], k[:20])
        be.kv_accept(pool, [(0, 1, 10, 10)], range(10))
    for _ in range(3):
        g.replay()
    rows = held_rows(pool, 0, 10)["k"]
    for slot, n in ((1, 20), (2, 20)):
        be.rope_append(pool, [(slot, n, 20)], k[20:], k[20:])
    torch.cuda.synchronize()
    before = state(pool)
    assert list(before["n_logical"]) == [2, 3, 3, 0]
    k[:20] *= 2
    g.replay()
    torch.cuda.synchronize()
    after = state(pool)
    same(after, before, ("k", "v", "ntok", "centroid", "page_hash"))
    for slot, first in ((1, rows), (2, None)):
        got = held_rows(pool, slot, 40)["k"]
        assert (got[20:] == k[20:].bfloat16()).all()
        assert (got[10:20] == first).all() if slot == 1 else (got[:20] == k[:20].bfloat16()).all()


def test_a_replayed_accept_after_a_reset_writes_nothing(be):
    """The slot's page, an old one at the capture, is another's or nobody's by then."""
    pool = filled(be, "int8", 2, 64, 3, 4, [20, 10, 17], 6)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        be.kv_accept(pool, [(0, 1, 10, 6)], range(6))
    pool.reset(1)
    torch.cuda.synchronize()
    before = state(pool)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        same(state(pool), before)


def test_accept_refusals_change_nothing(be):
    import be42
    pool = filled(be, "int8", 1, 64, 4, 4, [20, 5, 40, 0], 3)
    before = state(pool)
    for runs, index, kw, word in (
            ([(2, 0, 20, 1)], [48], {}, "token 48"), ([(2, 0, 20, 1)], [-1], {}, "token -1"), ([(3, 0, 20, 1)], [0], {}, "token 0"),
            ([(2, 2, 40, 1)], [0], {}, "read and filled"), ([(2, 0, 20, 1), (0, 1, 5, 1)], [0, 0], {}, "read and filled"),
            ([(2, 0, 20, 1), (2, 0, 21, 1)], [0, 1], {}, "twice"), ([(2, 0, 50, 1)], [0], {}, "skips"), ([(2, 0, 63, 2)], [0, 1], {}, "positions"),
            ([(4, 0, 20, 1)], [0], {}, "out of range"), ([(2, -1, 20, 1)], [0], {}, "out of range"),
            ([(2, 0, 20, 1)], [0], dict(layers=2, from_step=2, to_step=1), "out of range"),
            ([(2, 0, 20, 1)], [0], dict(layers=2, from_step=0, to_step=2 ** 31 - 1), "out of range"),
            ([(2, 0, 20, 1)], [0, 1], {}, "2 tokens"), ([(2, 0, 20, 2), (2, 1, 5, -1)], [0], {}, "more")):
        with pytest.raises(be42.Be42Error, match=word):
            be.kv_accept(pool, runs, index, **kw)
        same(state(pool), before)
    be.kv_accept(pool, [], [])
    be.kv_accept(pool, [(2, 0, 20, 0)], [])
    be.kv_accept(pool, [(2, 0, 20, 1)], [1], layers=0)
    same(state(pool), before)


def test_other_stream(be):
    """On a stream of the caller's, behind work queued there."""
    import be42
    rng = np.random.default_rng(12)
    n, kvh, hd = 30, 2, 64
    k = rows_of(rng, n, kvh, hd, False).cuda()
    pools = [make(be, "int8", 2, kvh, hd, 4) for _ in range(2)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = []
    for pool, stream in zip(pools, (torch.cuda.current_stream(), s)):
        with torch.cuda.stream(stream):
            x = k * 2.0
            got.append(be.rope_append(pool, [(0, 0, n)], x, x, q=x))
            be.kv_accept(pool, [(0, 1, 0, 3)], [4, 29, 7])
        stream.synchronize()
    assert (got[0] == got[1]).all()
    same(state(pools[0]), state(pools[1]))
