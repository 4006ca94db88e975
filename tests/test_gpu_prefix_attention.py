"""Attention behind a shared prefix (be42_prefix_attention) against float64 over
the pages' own values.

Tolerance: a score is a sum of hd products of exact factors in fp32 (three
products of parts for an fp32 query), so its error d is at most
hd * 2^-22 * scale * max_t sum_i |q_i k_ti| / sqrt(hd) in norm terms (random
signs; 16 of those standard deviations), plus 2^-22 of the score itself in the
exponential's argument; weights then are off by d relatively, the output by
2 d max|v|, and by 2^-20 max|v| for the sums.  bf16 queries add the rounding
of the weights and of the output, 2^-8 max|v| each."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 16


def make_pool(be, kind, n_slots, kvh, hd, held, seed, order=None):
    """A pool whose slot s holds held[s] tokens; slots are filled a page at a
    time in turn, so that their pages interleave.  -> (pool, k, v): the values
    the pages hold, per slot [tokens][kvh][hd] float64."""
    import be42
    rng = np.random.default_rng(seed)
    pool = be.kv_pool(be42.KV_BF16 if kind == "bf16" else be42.KV_INT8, n_slots, kvh, hd, max(1, -(-max(held) // PAGE)) + 1)
    k = [rng.standard_normal((n, kvh, hd)).astype(np.float32) for n in held]
    v = [rng.standard_normal((n, kvh, hd)).astype(np.float32) for n in held]
    dk, dv = [torch.from_numpy(a).cuda() for a in k], [torch.from_numpy(a).cuda() for a in v]
    step = 3 * PAGE
    for at in range(0, max(held), step):
        for s, n in enumerate(held):
            if at < n:
                m = min(step, n - at)
                pool.append(s, dk[s][at:at + m].reshape(m, -1), dv[s][at:at + m].reshape(m, -1), at)

    def stored(a):
        if kind == "bf16":
            return torch.from_numpy(a).bfloat16().double().numpy()
        amax = np.abs(a).max(-1, keepdims=True)
        sc, inv = (amax / np.float32(127)).astype(np.float32), (np.float32(127) / amax).astype(np.float32)
        x = a * inv
        return np.trunc(x + np.copysign(np.float32(0.5), x)).clip(-127, 127).astype(np.float64) * sc

    return pool, [stored(a) for a in k], [stored(a) for a in v]


def reference(q, k, v, n_heads, scale, prefix_slot, prefix_len, slots, lens, max_len):
    """float64 out [B][H][hd] and the tolerance of each query and head."""
    B, H, hd = q.shape
    out, tol = np.zeros((B, H, hd)), np.zeros((B, H))
    for b in range(B):
        own = slots[b]
        n = min(lens[b], max_len)
        n = min(n, len(k[own])) if 0 <= own < len(k) else 0
        p = min(prefix_len, len(k[prefix_slot]))
        kk = np.concatenate([k[prefix_slot][:p]] + ([k[own][:n]] if n > 0 else []))
        vv = np.concatenate([v[prefix_slot][:p]] + ([v[own][:n]] if n > 0 else []))
        if not len(kk):
            continue
        g = H // kk.shape[1]
        for h in range(H):
            K, V = kk[:, h // g], vv[:, h // g]
            s = K @ q[b, h] * scale
            w = np.exp(s - s.max())
            out[b, h] = (w / w.sum()) @ V
            d = hd * 2.0 ** -22 * abs(scale) * (np.abs(K) @ np.abs(q[b, h])).max() / math.sqrt(hd) + 2.0 ** -22 * np.abs(s).max()
            tol[b, h] = (2 * d + 2.0 ** -20) * np.abs(V).max()
    return out, tol, [np.abs(np.concatenate([a.reshape(-1) for a in v] + [np.zeros(1)])).max()]


def run(be, pool, q, k, v, prefix_slot, prefix_len, slots, lens, max_len, scale=None, give_slots=True, give_lens=True,
        q_dev=None, **kw):
    B, H, hd = q.shape
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    bf16 = q.dtype == torch.bfloat16
    st = torch.tensor(list(slots), dtype=torch.int32, device="cuda") if give_slots else None
    lt = torch.tensor(list(lens), dtype=torch.int32, device="cuda") if give_lens else None
    got = be.prefix_attention(pool, q.cuda() if q_dev is None else q_dev, prefix_slot, prefix_len, scale, slots=st,
                              lens=lt, max_len=max_len, **kw)
    assert got.dtype == q.dtype and got.shape == q.shape
    want, tol, vmax = reference(q.double().numpy(), k, v, H, scale, prefix_slot, prefix_len, slots, lens, max_len)
    tol = tol + (2.0 ** -7 * vmax[0] if bf16 else 0.0)
    off = np.abs(got.cpu().double().numpy() - want).max(-1)
    assert np.isfinite(got.float().cpu().numpy()).all()
    assert (off <= tol).all(), (np.unravel_index((off - tol).argmax(), off.shape), off.max(), tol.min())
    return got


def queries(seed, B, H, hd, bf16):
    q = torch.randn(B, H, hd, generator=torch.Generator().manual_seed(seed))
    return q.bfloat16() if bf16 else q


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kvh,hd", [(8, 8, 64), (6, 2, 128), (4, 1, 64), (20, 1, 128), (3, 3, 128), (72, 2, 64)])
def test_heads(be, kind, bf16, heads, kvh, hd):
    held = [0, 5, 40, 100, 333]
    pool, k, v = make_pool(be, kind, 5, kvh, hd, held, 1)
    run(be, pool, queries(2, 4, heads, hd, bf16), k, v, 4, 333, [0, 1, 2, 3], [0, 5, 40, 100], 100)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 31, 32, 33, 47, 64, 100, 127, 128, 129, 500, 1000, 2049, 5003])
def test_prefix_lengths(be, kind, prefix):
    held = [17, 1, 0, max(prefix, 1)]
    pool, k, v = make_pool(be, kind, 4, 2, 128, held, 3 + prefix)
    run(be, pool, queries(4, 3, 8, 128, False), k, v, 3, prefix, [0, 1, 2], [17, 1, 0], 17)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("own", [0, 1, 15, 16, 17, 32, 33, 63, 64, 65, 130, 700, 1500])
def test_own_lengths(be, kind, own):
    """No prefix, a short one; a query that sees less than its slot holds."""
    held = [max(own, 1), 20, 50]
    pool, k, v = make_pool(be, kind, 3, 2, 64, held, 5 + own)
    for prefix in (0, 50):
        run(be, pool, queries(6, 3, 4, 64, False), k, v, 2, prefix, [0, 1, 0], [own, 0, max(own - 3, 0)], max(own, 1))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B", [1, 2, 9, 16, 17, 33, 70, 129])
def test_batches(be, kind, bf16, B):
    held = [(b * 7) % 50 for b in range(B)] + [1203]
    pool, k, v = make_pool(be, kind, B + 1, 2, 128, held, 7 + B)
    run(be, pool, queries(8, B, 8, 128, bf16), k, v, B, 1203, range(B), held[:B], 50)


def test_query_with_nothing_to_see_gets_zeros(be):
    pool, k, v = make_pool(be, "bf16", 3, 2, 64, [0, 30, 0], 9)
    q = queries(10, 2, 4, 64, False)
    got = run(be, pool, q, k, v, 2, 0, [0, 1], [0, 30], 30)
    assert not got[0].any() and got[1].any()
    assert not be.prefix_attention(pool, q.cuda(), 1, 0, 0.1, max_len=0).any()
    # a prefix of a slot that holds nothing
    assert not be.prefix_attention(pool, q.cuda(), 2, 40, 0.1, max_len=0).any()


def test_lengths_are_cut_at_what_the_slot_holds(be):
    pool, k, v = make_pool(be, "bf16", 4, 2, 64, [20, 7, 33, 100], 11)
    q = queries(12, 3, 4, 64, False)
    run(be, pool, q, k, v, 3, 112, [0, 1, 2], [112, 8, 40], 112)          # more than held
    run(be, pool, q, k, v, 3, 100, [0, 1, 2], [20, 7, 33], 10)            # more than max_len
    run(be, pool, q, k, v, 3, 100, [0, -1, 4], [20, 7, 33], 40)           # slots outside the pool hold nothing
    run(be, pool, q, k, v, 3, 100, [0, 1, 2], [-5, -2 ** 31, 2 ** 31 - 1], 40)
    run(be, pool, q, k, v, 3, 100, [0, 1, 2], [20, 7, 33], 40, give_slots=False, give_lens=False)
    # the same slot as prefix and as own tokens, and twice as own
    run(be, pool, q, k, v, 3, 60, [3, 3, 0], [100, 100, 3], 100)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_unwritten_token_slots_are_not_read(be, kind):
    """Page slots past a slot's tokens, and pages nobody holds, full of NaN
    patterns: the result does not move."""
    held = [5, 18, 0, 35]
    pool, k, v = make_pool(be, kind, 4, 2, 128, held, 13)
    q = queries(14, 3, 6, 128, False)
    want = run(be, pool, q, k, v, 3, 35, [0, 1, 2], [5, 18, 0], 18)
    used = {}
    for s, n in enumerate(held):
        for i, ph in enumerate(pool.layer_pages(s)):
            used[int(ph)] = min(PAGE, n - i * PAGE)
    cap, kvh, hd = pool.s.capacity, 2, 128
    if kind == "bf16":
        K, V = pool.fetch("k", cap * kvh * PAGE * hd, np.uint16), pool.fetch("v", cap * kvh * PAGE * hd, np.uint16)
        Kr, Vr = K.reshape(cap, kvh, PAGE, hd), V.reshape(cap, kvh, hd, PAGE)
        for ph in range(cap):
            Kr[ph, :, used.get(ph, 0):], Vr[ph, :, :, used.get(ph, 0):] = 0x7FC0, 0x7FC0
        put = (("k", K), ("v", V))
    else:
        put = []
        for f in ("k_scale", "v_scale"):
            S = pool.fetch(f, cap * kvh * PAGE, np.float32)
            for ph in range(cap):
                S.reshape(cap, kvh, PAGE)[ph, :, used.get(ph, 0):] = np.nan
            put.append((f, S))
    for f, a in put:
        be.check(be.lib.be42_memcpy_h2d(getattr(pool.s, f), a.ctypes.data, a.nbytes, None), "h2d")
    torch.cuda.synchronize()
    assert torch.equal(run(be, pool, q, k, v, 3, 35, [0, 1, 2], [5, 18, 0], 18), want)


def test_nan_of_one_query_stays_there(be):
    pool, k, v = make_pool(be, "bf16", 4, 2, 64, [5, 9, 3, 300], 15)
    q = queries(16, 3, 4, 64, False)
    want = run(be, pool, q, k, v, 3, 300, [0, 1, 2], [5, 9, 3], 9)
    q[1, 2, 7] = math.nan
    got = be.prefix_attention(pool, q.cuda(), 3, 300, 0.125, slots=torch.arange(3, dtype=torch.int32, device="cuda"),
                              lens=torch.tensor([5, 9, 3], dtype=torch.int32, device="cuda"), max_len=9)
    assert torch.isnan(got[1, 2]).all()
    got[1, 2] = want[1, 2]
    assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_large_scores_and_small_values(be, kind):
    """Scores hundreds apart (weights of zero), queries far from one."""
    pool, k, v = make_pool(be, kind, 3, 1, 64, [40, 3, 700], 17)
    for mul in (300.0, 1e-30, 0.0):
        q = queries(18, 2, 4, 64, False) * mul
        run(be, pool, q, k, v, 2, 700, [0, 1], [40, 3], 40)
    run(be, pool, queries(18, 2, 4, 64, False), k, v, 2, 700, [0, 1], [40, 3], 40, scale=-3.0)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
def test_continuations_of_several_tokens(be, kind, bf16):
    """Queries of one slot at consecutive positions, each as if alone."""
    held = [9, 30, 400]
    pool, k, v = make_pool(be, kind, 3, 2, 128, held, 19)
    slots, lens = [0] * 9 + [1] * 30, list(range(1, 10)) + list(range(1, 31))
    run(be, pool, queries(20, 39, 6, 128, bf16), k, v, 2, 400, slots, lens, 30)


@pytest.mark.parametrize("bf16", [False, True])
def test_strided_queries(be, bf16):
    """The q part of rows that hold q, k and v side by side, off 16 bytes."""
    pool, k, v = make_pool(be, "bf16", 4, 2, 64, [5, 9, 3, 100], 21)
    for pad, off in ((256, 0), (7, 1), (2, 2)):
        q = queries(22, 3, 4, 64, bf16)
        wide = torch.full((3, 256 + pad + off), math.nan, dtype=q.dtype, device="cuda")
        wide[:, off:off + 256] = q.reshape(3, 256).cuda()
        run(be, pool, q, k, v, 3, 100, [0, 1, 2], [5, 9, 3], 9, q_dev=wide[:, off:off + 256].unflatten(1, (4, 64)))


@pytest.mark.parametrize("B,heads,prefix,max_len", [(1, 4, 50, 9), (3, 8, 3000, 40), (70, 8, 900, 0), (5, 4, 0, 300)])
def test_workspace_of_the_caller(be, B, heads, prefix, max_len):
    """Exactly the bytes asked for, full of NaN patterns, nothing behind them touched."""
    held = [min(max_len, 3 + b) for b in range(B)] + [max(prefix, 1)]
    pool, k, v = make_pool(be, "bf16", B + 1, 2, 64, held, 23)
    size = be.lib.be42_prefix_attention_workspace_bytes(B, heads, 2, 64, prefix, max_len)
    ws = torch.full((size + 256,), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((B, heads, 64), math.nan, device="cuda")
    got = run(be, pool, queries(24, B, heads, 64, False), k, v, B, prefix, range(B), held[:B], max_len,
              workspace=ws[:size], out=out)
    assert got is out and (ws[size:] == 255).all()


def test_repeats_to_the_bit(be):
    pool, k, v = make_pool(be, "int8", 9, 2, 128, [50] * 8 + [4000], 25)
    q = queries(26, 8, 8, 128, False)
    a = run(be, pool, q, k, v, 8, 4000, range(8), [50] * 8, 50)
    for _ in range(3):
        assert torch.equal(run(be, pool, q, k, v, 8, 4000, range(8), [50] * 8, 50), a)


def test_refusals(be):
    import be42
    pool, k, v = make_pool(be, "bf16", 3, 2, 64, [5, 9, 30], 27)
    q = torch.zeros(2, 4, 64, device="cuda")
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    for kw in (dict(q=q.half()), dict(q=q[:, :, :32]), dict(q=q[0]), dict(q=q.cpu()), dict(q=q[:, :3]),
               dict(q=q.transpose(0, 1)), dict(prefix_slot=3), dict(prefix_len=1000), dict(slots=i.long()),
               dict(lens=i[:1]), dict(lens=i.cpu()), dict(out=q.bfloat16()), dict(out=q[:1]), dict(max_len=-1),
               dict(scale=math.nan), dict(workspace=q), dict(workspace=torch.zeros(1, dtype=torch.uint8, device="cuda"))):
        a = dict(q=q, prefix_slot=2, prefix_len=30, scale=0.1, slots=i, lens=i, max_len=9)
        a.update(kw)
        with pytest.raises(be42.Be42Error):
            be.prefix_attention(pool, **a)
    assert be.prefix_attention(pool, q[:0], 2, 30, 0.1).shape == (0, 4, 64)


def test_graph_decodes_on(be):
    """Captured once, replayed while slots grow and the batch's slots change
    places: each replay equals the eager call and float64."""
    B, kvh, hd = 3, 2, 64
    pool, k, v = make_pool(be, "bf16", 4, kvh, hd, [4, 1, 0, 200], 29)
    q = torch.zeros(B, 4, hd, device="cuda")
    slots = torch.arange(B, dtype=torch.int32, device="cuda")
    lens = torch.tensor([4, 1, 0], dtype=torch.int32, device="cuda")
    ws = torch.empty(be.lib.be42_prefix_attention_workspace_bytes(B, 4, kvh, hd, 200, 12), dtype=torch.uint8, device="cuda")
    call = lambda: be.prefix_attention(pool, q, 3, 200, 0.125, slots=slots, lens=lens, max_len=12, workspace=ws)  # noqa: E731
    call()
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        got = call()
    held = [4, 1, 0]
    rng = np.random.default_rng(30)
    for step in range(5):
        place = rng.permutation(B)
        for s in range(B):
            a, b = (rng.standard_normal((1, kvh, hd)).astype(np.float32) for _ in range(2))
            pool.append(s, torch.from_numpy(a).cuda().reshape(1, -1), torch.from_numpy(b).cuda().reshape(1, -1), held[s])
            k[s] = np.concatenate([k[s], torch.from_numpy(a).bfloat16().double().numpy()])
            v[s] = np.concatenate([v[s], torch.from_numpy(b).bfloat16().double().numpy()])
            held[s] += 1
        qc = queries(31 + step, B, 4, hd, False)
        q.copy_(qc)
        slots.copy_(torch.from_numpy(place.astype(np.int32)))
        lens.copy_(torch.tensor([held[p] for p in place], dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        again = run(be, pool, qc, k, v, 3, 200, [int(p) for p in place], [held[p] for p in place], 12, scale=0.125)
        assert torch.equal(again, got), step


def test_two_graphs_and_two_streams(be):
    """Calls without a workspace share none: two graphs replayed at once, a larger
    eager call and calls on two streams leave each other's results alone."""
    pool, _, _ = make_pool(be, "bf16", 9, 2, 64, [30] * 8 + [3000], 40)
    sizes = ((4, 3000), (8, 1700))
    qs = [queries(41 + i, b, 8, 64, False).cuda() for i, (b, _) in enumerate(sizes)]
    call = lambda i: be.prefix_attention(pool, qs[i], 8, sizes[i][1], 0.125, max_len=30)  # noqa: E731
    want = [call(0), call(1)]
    many = queries(43, 64, 8, 64, False).cuda()
    slots = torch.zeros(64, dtype=torch.int32, device="cuda")
    streams, graphs, got = [torch.cuda.Stream() for _ in qs], [torch.cuda.CUDAGraph() for _ in qs], []
    torch.cuda.synchronize()
    for i in range(2):
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            got.append(call(i))
    for _ in range(4):
        be.prefix_attention(pool, many, 8, 3000, 0.125, slots=slots, max_len=30)
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
            a.zero_()
        torch.cuda.synchronize()
    eager = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                eager[i].append(call(i))
    torch.cuda.synchronize()
    for runs, b in zip(eager, want):
        assert all(torch.equal(a, b) for a in runs)


def test_calls_that_would_use_anothers_memory_are_refused(be):
    import be42
    pool, _, _ = make_pool(be, "bf16", 3, 2, 64, [5, 9, 300], 44)
    q, out = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 4, 64, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=torch.cuda.Stream()):
        rc = be.lib.be42_prefix_attention(pool.handle, be.p(q), 0, 256, 2, 4, 2, 300, None, None, 9, 0.1, be.p(out), None, 0,
                                          be.stream())
        said = be.last_error()
        out.add_(1)
    assert rc == -1 and "captured" in said
    for kw in (dict(prefix_len=(1 << 32) + 30), dict(max_len=1 << 32), dict(prefix_slot=(1 << 32) + 2)):
        a = dict(prefix_slot=2, prefix_len=30, scale=0.1, max_len=9)
        a.update(kw)
        with pytest.raises(be42.Be42Error):
            be.prefix_attention(pool, q, **a)
    pool.device = 1                           # as if it lay on another GPU
    with pytest.raises(be42.Be42Error, match="pool on GPU 1"):
        be.prefix_attention(pool, q, 2, 30, 0.1, max_len=9)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B", [2, 20, 150])
def test_scale_of_zero_takes_the_mean(be, kind, bf16, B):
    pool, k, v = make_pool(be, kind, 3, 2, 64, [5, 40, 333], 45)
    run(be, pool, queries(46, B, 4, 64, bf16), k, v, 2, 333, [i % 2 for i in range(B)], [5 + i % 30 for i in range(B)], 40,
        scale=0.0)
    run(be, pool, queries(46, B, 4, 64, bf16), k, v, 2, 333, [i % 2 for i in range(B)], [5 + i % 30 for i in range(B)], 40,
        scale=1e-42)


def test_pages_past_32_bits(be):
    """A pool whose pages lie past 4 GiB of K and of V: a slot of 33 copies of the
    same tokens attends as one copy does, and a slot behind it as it should."""
    import be42
    kvh, hd, n, copies = 64, 128, 8192, 33
    pool = be.kv_pool(be42.KV_BF16, 2, kvh, hd, copies * n // PAGE + 32)
    gen = torch.Generator(device="cuda").manual_seed(47)
    k, v = (torch.randn(n, kvh * hd, generator=gen, device="cuda") for _ in range(2))
    for i in range(copies):
        pool.append(0, k, v, i * n)
    k1, v1 = (torch.randn(333, kvh * hd, generator=gen, device="cuda") for _ in range(2))
    pool.append(1, k1, v1, 0)
    assert copies * n * kvh * hd * 2 > 1 << 32
    for bf16 in (False, True):
        q = queries(48, 3, kvh, hd, bf16).cuda()
        one = be.prefix_attention(pool, q, 0, n, 0.09, max_len=0).double()
        all_ = be.prefix_attention(pool, q, 0, copies * n, 0.09, max_len=0).double()
        # either is off by the tolerance above: scores below 30, sums of up to 2^18 terms
        assert (one - all_).abs().max() <= (2.0 ** -7 if bf16 else 2 * (2 * 34 * 2.0 ** -22 + 2.0 ** -20)) * v.abs().max()
        kk, vv = (x.bfloat16().double().view(333, kvh, hd).cpu().numpy() for x in (k1, v1))
        got = be.prefix_attention(pool, q, 1, 333, 0.09, max_len=0)
        want, tol, vmax = reference(q.cpu().double().numpy(), [kk[:0], kk], [vv[:0], vv], kvh, 0.09, 1, 333, [0] * 3, [0] * 3, 0)
        off = np.abs(got.cpu().double().numpy() - want).max(-1)
        assert (off <= tol + (2.0 ** -7 * vmax[0] if bf16 else 0.0)).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kvh,prefix", [(8, 8, 100), (8, 2, 100), (8, 2, 3000)])
def test_nan_of_one_sequences_pages_stays_there(be, bad, bf16, heads, kvh, prefix):
    """Queries beside it (in one launch: of the same 16 rows) see numbers only."""
    held = [20, 33, 7, 40, 0, 12]
    pool, k, v = make_pool(be, "bf16", 7, kvh, 64, held + [prefix], 50)
    x = torch.full((1, kvh * 64), bad, device="cuda")
    pool.append(1, x, x, held[1])
    slots, lens = [0, 1, 2, 3, 4, 5, 1], [20, 34, 7, 40, 0, 12, 33]
    q = queries(51, 7, heads, 64, bf16)
    got = be.prefix_attention(pool, q.cuda(), 6, prefix, 0.125, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"),
                              lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), max_len=40).cpu().double().numpy()
    want, tol, vmax = reference(q.double().numpy(), k, v, heads, 0.125, 6, prefix, slots, lens, 40)
    for b in (0, 2, 3, 4, 5, 6):
        off = np.abs(got[b] - want[b]).max(-1)
        assert (off <= tol[b] + (2.0 ** -7 * vmax[0] if bf16 else 0.0)).all(), b
    assert not np.isfinite(got[1]).all()


def pool_of(be, kind, ks, vs):
    """A pool whose slot s holds the tokens ks[s], vs[s] ([n][kvh][hd] fp32)."""
    import be42
    _, kvh, hd = ks[0].shape
    pool = be.kv_pool(be42.KV_BF16 if kind == "bf16" else be42.KV_INT8, len(ks), kvh, hd, max(len(a) for a in ks) // PAGE + 1)
    for s, (a, b) in enumerate(zip(ks, vs)):
        if len(a):
            pool.append(s, torch.from_numpy(a).cuda().reshape(len(a), -1), torch.from_numpy(b).cuda().reshape(len(b), -1), 0)
    return pool


def whole_numbers(rng, n, kvh, hd, top):
    """Numbers of up to `top` with a largest of 127 in each row: INT8 pages (scale
    1) and bf16 pages hold them exactly."""
    a = rng.integers(-top, top + 1, (n, kvh, hd)).astype(np.float32)
    a[np.arange(n)[:, None], np.arange(kvh)[None], rng.integers(0, hd, (n, kvh))] = 127 * rng.choice([-1.0, 1.0], (n, kvh))
    return a


# calls of each form: one launch, tiles of 16, 64 and 128 rows (B, prefix)
FORMS = [(3, 200), (2, 3000), (20, 4100), (70, 1700)]


def check_form(be, B, heads, kvh, hd, prefix, max_len):
    """Whether a call of FORMS takes the launches that it is meant to."""
    parts = be.lib.be42_prefix_attention_workspace_bytes(B, heads, kvh, hd, prefix, max_len) > 16
    assert parts == (prefix > 1000), (B, prefix)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,prefix", FORMS)
@pytest.mark.parametrize("scale", [0.01, 1.0, 1e4, 1e9, -1e9, 1e20, 1e30])
def test_scores_of_any_size(be, kind, bf16, B, prefix, scale):
    """Scores that fp32 sums hold exactly, so that only their differences round:
    weights of tokens that count are off by 2^-22 of themselves at most (two
    roundings of an exponent below 24, the exponential's own), the sums by 2^-20
    as above.  V of whole numbers below 128 and of one element in 127: exact in
    either page.  At large scales one token, or equal ones in either slot or part,
    takes it all."""
    kvh, hd, heads = 2, 128, 8
    rng = np.random.default_rng(B + prefix)
    held = [(5 * b) % 23 for b in range(B)] + [prefix]
    k = [whole_numbers(rng, n, kvh, hd, 4) for n in held]
    v = [whole_numbers(rng, n, kvh, hd, 100) for n in held]
    for b in range(0, B, 3):                               # the same key in the slot and in the prefix, at places apart
        if held[b]:
            k[b][-1] = k[B][prefix // 2] = k[B][0] = k[B][prefix - 1]
    pool = pool_of(be, kind, k, v)
    check_form(be, B, heads, kvh, hd, prefix, 23)
    q = torch.from_numpy(rng.integers(-3, 4, (B, heads, hd)).astype(np.float32))
    q = q.bfloat16() if bf16 else q
    k, v = ([a.astype(np.float64) for a in x] for x in (k, v))
    lens = torch.tensor(held[:B], dtype=torch.int32, device="cuda")
    got = be.prefix_attention(pool, q.cuda(), B, prefix, scale, lens=lens, max_len=23).double().cpu().numpy()
    sc = float(np.float32(scale))
    want = reference(q.double().numpy(), k, v, heads, sc, B, prefix, range(B), held[:B], 23)[0]
    tol = 127 * 2.0 ** -19 + (2.0 ** -7 * 127 if bf16 else 0.0)
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all(), np.abs(got - want).max()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("B,prefix", FORMS)
def test_scores_of_minus_infinity(be, kind, B, prefix):
    """Scores that overflow downwards weigh nothing, also where they come first
    (the prefix's first steps, all own tokens of some queries); a query that has
    no others has seen tokens all the same: no zeros, 0 / 0."""
    kvh, hd, heads = 2, 64, 8
    rng = np.random.default_rng(B)
    held = [(5 * b) % 23 for b in range(B)] + [prefix]
    k, v = ([rng.standard_normal((n, kvh, hd)).astype(np.float32) * x for n in held] for x in (2.0 ** -100, 1.0))
    k = [np.abs(a) for a in k]
    for b in range(0, B, 2):
        k[b][:] = -(2.0 ** 60)
    k[B][:150] = -(2.0 ** 60)
    pool = pool_of(be, kind, k, v)
    q = torch.full((B, heads, hd), 2.0 ** 100, dtype=torch.bfloat16)
    lens = torch.tensor(held[:B], dtype=torch.int32, device="cuda")
    got = be.prefix_attention(pool, q.cuda(), B, prefix, 0.125, lens=lens, max_len=23).double().cpu().numpy()
    keep = [(a > -1).all((1, 2)) for a in k]
    stay = [a[i] for a, i in zip(k, keep)]
    pages = pool_of(be, kind, stay, [a[i] for a, i in zip(v, keep)])
    fewer = torch.tensor([len(a) for a in stay[:B]], dtype=torch.int32, device="cuda")
    want = be.prefix_attention(pages, q.cuda(), B, len(stay[B]), 0.125, lens=fewer, max_len=23).double().cpu().numpy()
    # the same tokens in other steps: two roundings to bf16, weights of 16 bits or of bf16, sums
    assert np.isfinite(got).all() and (np.abs(got - want) <= 2.0 ** -7 * np.abs(v[B]).max()).all()
    for max_len in (23, 3000):                             # one launch or two
        bad = be.prefix_attention(pool, q.cuda(), B, 150, 0.125, lens=lens, max_len=max_len).cpu()
        others = torch.tensor([b % 2 == 1 and held[b] > 0 for b in range(B)])
        assert torch.isnan(bad[~others]).all() and torch.isfinite(bad[others]).all()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("B,prefix", FORMS)
def test_weights_of_bf16_queries(be, kind, hd, B, prefix):
    """bf16 queries lose no more than the rounding of the output, 2^-8 of itself,
    whatever the batch: a weight enters the products as two bf16 parts, off by 2^-16
    of itself at most; scores and sums are off as for fp32 queries."""
    kvh, heads = 2, 8
    held = [(5 * b) % 23 for b in range(B)] + [prefix]
    pool, k, v = make_pool(be, kind, B + 1, kvh, hd, held, B)
    q = queries(B, B, heads, hd, True)
    lens = torch.tensor(held[:B], dtype=torch.int32, device="cuda")
    got = be.prefix_attention(pool, q.cuda(), B, prefix, 1 / math.sqrt(hd), lens=lens, max_len=23).double().cpu().numpy()
    qd = q.double().numpy()
    want, tol, _ = reference(qd, k, v, heads, 1 / math.sqrt(hd), B, prefix, range(B), held[:B], 23)
    sizes = reference(qd, k, [np.abs(a) for a in v], heads, 1 / math.sqrt(hd), B, prefix, range(B), held[:B], 23)[0]
    off = np.abs(got - want)
    bound = 2.0 ** -8 * np.abs(want) + 2.0 ** -16 * sizes + tol[..., None]
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("B,heads,kvh,prefix,max_len", [
    (65, 5, 1, 1537, 17), (65, 5, 1, 5003, 17), (129, 4, 2, 2049, 17), (129, 4, 2, 1800, 0), (257, 1, 1, 2048, 5),
    (14, 20, 1, 100, 17), (14, 20, 1, 100, 0), (8, 66, 2, 333, 40)])
def test_tiles_of_128_rows(be, kind, bf16, hd, B, heads, kvh, prefix, max_len):
    """More than 256 rows of a KV head, in tiles of 128 whose last is cut, over
    prefixes whose parts end inside a stage and a page; the tolerance of bf16
    queries as for their weights above."""
    G = heads // kvh
    assert B * G > 256
    whole = be.lib.be42_prefix_attention_workspace_bytes(B, heads, kvh, hd, prefix, max_len) == 16
    assert whole == (prefix == 100 and max_len == 0)       # (in one part; groups above 16 have no one-launch form)
    held = [(5 * b) % (max_len + 1) for b in range(B)] + [prefix]
    pool, k, v = make_pool(be, kind, B + 1, kvh, hd, held, B + prefix)
    q = queries(B, B, heads, hd, bf16)
    lens = torch.tensor(held[:B], dtype=torch.int32, device="cuda")
    args = heads, 1 / math.sqrt(hd), B, prefix, range(B), held[:B], max_len
    got = be.prefix_attention(pool, q.cuda(), B, prefix, args[1], lens=lens, max_len=max_len).double().cpu().numpy()
    qd = q.double().numpy()
    want, tol, _ = reference(qd, k, v, *args)
    bound = np.broadcast_to(tol[..., None], want.shape)
    if bf16:
        bound = bound + 2.0 ** -8 * np.abs(want) + 2.0 ** -16 * reference(qd, k, [np.abs(a) for a in v], *args)[0]
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()
