"""Log probabilities, entropy and top alternatives (be42_logprobs) against
float64.  Tolerances: a logit's z = (x - max) / T carries at most three fp32
roundings (2^-24 of |z| each, with T's inverse), its exponential and the sum's
additions at most 80 more (a lane adds its entries, up to 128 at these sizes, in
fp32, each off by 2^-24 of a sum that grows from nothing: half of 128; lanes and
runs are added in 64 bits), so log s is off by no more than e = 2^-24 * (3 * sum p |z| + 80) and
the stored results by half a step more.  The entropy's second sum has the same
terms weighted with z."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def reference(x, temp):
    """x: CPU float tensor [rows][n] -> (lp, entropy, lp tolerance without the
    token's own part, entropy tolerance) in 64 bits."""
    z = (x.double() - x.double().amax(1, keepdim=True)) / temp
    lp = torch.log_softmax(x.double() / temp, 1)
    p = lp.exp()
    zz = torch.where(p > 0, z, torch.zeros_like(z)).abs()
    H = -torch.special.xlogy(p, p).sum(1)
    m1, m2 = (p * zz).sum(1), (p * zz * zz).sum(1)
    e = U * (3 * m1 + 80)
    return lp, H, e, e * (1 + m1) + U * (3 * m2 + 80 * m1) + 2 * U * H.abs()


def ids_of(x, k):
    """Ids by value, equal ones by id; a NaN counts as -infinity."""
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    return torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32)


def check(be, x, tokens, temp=1.0, top_k=0, dev=None, **kw):
    """x: CPU float32 or bfloat16; dev: the same logits as the call sees them."""
    d = x.cuda() if dev is None else dev
    got = be.logprobs(d, tokens.cuda(), temp=temp, top_k=top_k, entropy=True, **kw)
    lp, H, e, eH = reference(x.float(), temp)
    t = float(np.float32(temp))
    want = lp.gather(1, tokens.long())
    off = (got["logprobs"].cpu().double() - want).abs()
    same = (got["logprobs"].cpu().double() == want)           # both -infinity
    assert (same | (off <= e[:, None] + 4 * U * (want.abs() + abs(t - temp) / t * want.abs() / U))).all(), off.max()
    assert ((got["entropy"].cpu().double() - H).abs() <= eH).all(), (got["entropy"].cpu().double() - H).abs().max()
    if top_k:
        ids = ids_of(x.float(), top_k)
        assert torch.equal(got["top_ids"].cpu(), ids)
        want = lp.gather(1, ids.long())
        g = got["top_logprobs"].cpu().double()
        assert ((g == want) | ((g - want).abs() <= e[:, None] + 4 * U * want.abs())).all()
    return got


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (5, 63), (4, 64), (2, 65), (3, 257), (2, 1000), (7, 4096), (3, 4099),
                                    (2, 8191), (5, 8193), (3, 16385), (2, 32003), (40, 5001), (1, 128256), (9, 128256),
                                    (2, 151936), (1, 300001)])
def test_matches_float64(be, bf16, rows, n):
    rng = np.random.default_rng(rows * 1000003 + n)
    x = torch.from_numpy((rng.standard_normal((rows, n)) * 2.5).astype(np.float32))
    x = x.bfloat16() if bf16 else x
    tokens = torch.from_numpy(rng.integers(0, n, (rows, 3)).astype(np.int32))
    for temp, k in ((1.0, min(n, 20)), (0.5, min(n, 1)), (2.0, min(n, 64)), (1.0, 0)):
        check(be, x, tokens, temp, k)


@pytest.mark.parametrize("bf16", [False, True])
def test_many_rows(be, bf16):
    """More rows than the chip has workgroups for, and a peaked distribution."""
    rng = np.random.default_rng(3)
    x = torch.from_numpy((rng.standard_normal((700, 20011)) * 6.0).astype(np.float32))
    x = x.bfloat16() if bf16 else x
    check(be, x, torch.from_numpy(rng.integers(0, 20011, (700, 1)).astype(np.int32)), 1.0, 7)


@pytest.mark.parametrize("n", [50, 4096, 40000, 128256])
def test_ties_and_zeros(be, n):
    """Equal logits everywhere, few distinct ones, and zeros of both signs."""
    rng = np.random.default_rng(4)
    x = torch.zeros(5, n)
    x[1] = torch.from_numpy(rng.integers(-2, 3, n).astype(np.float32))
    x[2, ::2] = -0.0
    x[3] = torch.arange(n, dtype=torch.float32)
    x[4] = -torch.arange(n, dtype=torch.float32)
    check(be, x, torch.zeros(5, 1, dtype=torch.int32), 1.0, min(n, 64))
    check(be, x.bfloat16(), torch.zeros(5, 1, dtype=torch.int32), 1.0, min(n, 64))


@pytest.mark.parametrize("n", [70, 5000, 128256])
def test_masked_rows(be, n):
    """-infinity for most of a row, the type's lowest value as a mask, one token
    left, fewer left than alternatives are asked for."""
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((5, n)).astype(np.float32))
    x[0][torch.from_numpy(rng.random(n) < 0.9)] = -math.inf
    x[1, :] = -math.inf
    x[1, n // 2] = 3.0
    x[2, torch.arange(n) % 3 != 0] = torch.finfo(torch.float32).min
    x[3, 5:] = -math.inf
    x[4, : n - 2] = -math.inf
    tokens = torch.tensor([[0, 1], [n // 2, 0], [0, 1], [4, 5], [n - 1, 0]], dtype=torch.int32)
    got = check(be, x, tokens, 1.0, 20)
    assert got["logprobs"][1, 0] == 0 and got["logprobs"][1, 1] == -math.inf and got["entropy"][1] == 0


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,n", [(6, 40), (6, 4099), (29, 34245), (6, 128256)])
@pytest.mark.parametrize("share", [0.02, 0.3, 0.7, 0.99])
def test_scattered_masks(be, bf16, rows, n, share):
    """-infinity here and there, in even and odd places alike."""
    rng = np.random.default_rng(n + int(100 * share))
    x = torch.from_numpy((rng.standard_normal((rows, n)) * 2.5).astype(np.float32))
    off = torch.from_numpy(rng.random((rows, n)) < share)
    off[0] = False
    off[1, ::2] = True
    off[2, 1::2] = True
    off[:, n // 3] = False
    x[off] = -math.inf
    x = x.bfloat16() if bf16 else x
    tokens = torch.from_numpy(rng.integers(0, n, (rows, 2)).astype(np.int32))
    for temp, k in ((1.0, 1), (1.5, 20), (1.0, 0)):
        check(be, x, tokens, temp, k)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [64, 4099, 128256])
def test_top_ids_beside_nan_and_infinity(be, bf16, n):
    """NaN of both kinds (the signalling one is what a maximum may pass on) and
    +infinity, beside which the other alternatives are still found."""
    rng = np.random.default_rng(n + 77)
    x = torch.from_numpy((rng.standard_normal((4, n)) * 2.5).astype(np.float32))
    x = x.bfloat16() if bf16 else x
    bits = x.view(torch.int16 if bf16 else torch.int32)
    at = torch.from_numpy(rng.permutation(n)[: max(n // 50, 3)])
    bits[0, at] = 0x7FA0 if bf16 else 0x7FA00000
    bits[1, at] = 0x7FC0 if bf16 else 0x7FC00000
    bits[2, at] = -0x0060 if bf16 else -0x00600000           # a signalling NaN with its sign set
    x[3, at] = math.inf
    got = be.logprobs(x.cuda(), top_k=20, entropy=True)
    assert torch.equal(got["top_ids"].cpu(), ids_of(x.float(), 20))
    assert torch.isnan(got["entropy"]).all() and torch.isnan(got["top_logprobs"]).all()


@pytest.mark.parametrize("n", [64, 5000, 128256])
def test_rows_without_a_distribution(be, n):
    rng = np.random.default_rng(6)
    x = torch.from_numpy(rng.standard_normal((5, n)).astype(np.float32))
    x[0, n - 1] = math.nan
    x[1, 7] = math.inf
    x[2] = -math.inf
    x[3] = math.nan
    tokens = torch.full((5, 1), 3, dtype=torch.int32)
    got = be.logprobs(x.cuda(), tokens.cuda(), top_k=9, entropy=True)
    for name in ("logprobs", "entropy", "top_logprobs"):
        bad = torch.isnan(got[name].cpu().reshape(5, -1))
        assert bad[:4].all() and not bad[4].any(), name
    assert torch.equal(got["top_ids"].cpu(), ids_of(x, 9))


def test_token_ids_outside_the_vocabulary(be):
    x = torch.randn(2, 300, generator=torch.Generator().manual_seed(1))
    tokens = torch.tensor([[-1, 300, 2 ** 31 - 1, -2 ** 31], [299, 0, 0, 299]], dtype=torch.int32)
    got = be.logprobs(x.cuda(), tokens.cuda())["logprobs"].cpu()
    assert (got[0] == -math.inf).all() and torch.isfinite(got[1]).all()
    assert got[1, 0] == got[1, 3] and got[1, 1] == got[1, 2]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [129, 4096, 33333])
def test_strides_and_alignment(be, bf16, n):
    rng = np.random.default_rng(7)
    for pad, off in ((0, 1), (1, 0), (8, 3), (64, 0), (7, 2)):
        x = torch.from_numpy((rng.standard_normal((3, n)) * 2).astype(np.float32))
        x = x.bfloat16() if bf16 else x
        wide = torch.full((3, n + pad + off), math.nan, dtype=x.dtype, device="cuda")
        wide[:, off:off + n] = x.cuda()
        tokens = torch.from_numpy(rng.integers(0, n, (3, 2)).astype(np.int32))
        check(be, x, tokens, 1.0, 10, dev=wide[:, off:off + n])


@pytest.mark.parametrize("rows,n,k", [(1, 100, 5), (3, 128256, 20), (300, 40000, 64), (2, 128256, 0)])
def test_workspace_of_the_caller(be, rows, n, k):
    """Exactly the bytes asked for, full of NaN patterns, nothing behind them touched."""
    x = torch.randn(rows, n, generator=torch.Generator().manual_seed(2))
    size = be.lib.be42_logprobs_workspace_bytes(n, rows, k)
    ws = torch.full((size + 256,), 255, dtype=torch.uint8, device="cuda")
    check(be, x, torch.zeros(rows, 1, dtype=torch.int32), 1.0, k, workspace=ws[:size])
    assert (ws[size:] == 255).all()


def test_parts_alone(be):
    """Each output by itself is what it is with the others."""
    x = torch.randn(4, 50000, generator=torch.Generator().manual_seed(3)).cuda()
    tokens = torch.arange(4, dtype=torch.int32, device="cuda")[:, None]
    full = be.logprobs(x, tokens, top_k=8, entropy=True)
    for kw in (dict(tokens=tokens), dict(entropy=True), dict(top_k=8)):
        for name, v in be.logprobs(x, **kw).items():
            assert torch.equal(v, full[name]), name
    empty = be.logprobs(x[:0], tokens[:0], top_k=8, entropy=True)
    assert empty["top_ids"].shape == (0, 8)


def test_refusals(be):
    import be42
    x, tokens = torch.zeros(4, 64, device="cuda"), torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    for kw in (dict(logits=x.half()), dict(logits=x.t()), dict(logits=x[0]), dict(tokens=tokens.long()),
               dict(tokens=tokens[:2]), dict(tokens=tokens.cpu()), dict(temp=0.0), dict(top_k=65), dict(logits=x.cpu()),
               dict(tokens=None), dict(workspace=x), dict(workspace=torch.zeros(1, dtype=torch.uint8, device="cuda"))):
        a = dict(logits=x, tokens=tokens)
        a.update(kw)
        with pytest.raises(be42.Be42Error):
            be.logprobs(**a)


def test_graph_and_other_stream(be):
    """Captured on a stream of its own with its own workspace, replayed on new
    logits, and eager calls of other sizes between."""
    n = 128256
    x = torch.randn(3, n, device="cuda")
    tokens = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    ws = torch.empty(be.lib.be42_logprobs_workspace_bytes(n, 3, 10), dtype=torch.uint8, device="cuda")
    be.logprobs(x, tokens, top_k=10, entropy=True, workspace=ws)
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        got = be.logprobs(x, tokens, top_k=10, entropy=True, workspace=ws)
    for k in range(4):
        x.copy_(torch.randn(3, n, generator=torch.Generator().manual_seed(40 + k)))
        tokens.fill_(k)
        g.replay()
        torch.cuda.synchronize()
        eager = be.logprobs(x, tokens, top_k=10, entropy=True)
        be.logprobs(torch.randn(70, 5000, device="cuda"), top_k=3)
        for name, v in eager.items():
            assert torch.equal(v, got[name]), (k, name)


def test_two_graphs_and_two_streams(be):
    """Calls without a workspace share none: two graphs replayed at once, a larger
    eager call and calls on two streams leave each other's results alone."""
    shapes = ((3, 128256), (5, 60000))
    xs = [torch.randn(s, generator=torch.Generator().manual_seed(50 + i)).cuda() for i, s in enumerate(shapes)]
    want = [be.logprobs(x, top_k=10, entropy=True) for x in xs]
    big = torch.randn(9, 500000, device="cuda")
    streams, graphs, got = [torch.cuda.Stream() for _ in xs], [torch.cuda.CUDAGraph() for _ in xs], []
    torch.cuda.synchronize()
    for x, s, g in zip(xs, streams, graphs):
        with torch.cuda.graph(g, stream=s):
            got.append(be.logprobs(x, top_k=10, entropy=True))
    for _ in range(4):
        be.logprobs(big, top_k=64, entropy=True)
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(a[n], b[n]) for n in b)
            for n in a:
                a[n].zero_()
        torch.cuda.synchronize()
    eager = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                eager[i].append(be.logprobs(xs[i], top_k=10, entropy=True))
    torch.cuda.synchronize()
    for runs, b in zip(eager, want):
        assert all(torch.equal(a[n], b[n]) for a in runs for n in b)


def test_capture_with_the_librarys_workspace_is_refused(be):
    x, ent = torch.randn(2, 128256, device="cuda"), torch.zeros(2, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=torch.cuda.Stream()):
        rc = be.lib.be42_logprobs(None, be.p(ent), None, None, be.p(x), 0, x.shape[1], x.shape[1], 2, 1.0, None, 0, 0, None, 0,
                                  be.stream())
        said = be.last_error()
        ent.add_(1)
    assert rc == -1 and "captured" in said


@pytest.mark.parametrize("bf16", [False, True])
def test_rows_past_32_bits(be, bf16):
    """Three rows 2^31 - 8 entries apart, the last past 2^32."""
    n, apart = 40000, (1 << 31) - 8
    x = torch.randn(3, n, generator=torch.Generator().manual_seed(60)) * 2.5
    x = x.bfloat16() if bf16 else x
    far = torch.empty(2 * apart + n, dtype=x.dtype, device="cuda").as_strided((3, n), (apart, 1))
    far.copy_(x)
    check(be, x, torch.tensor([[0, 7], [n - 1, 5], [n // 2, 1]], dtype=torch.int32), 1.0, 10, dev=far)


def low_rows(n, bf16, mask, seed):
    """Rows that a finite mask leaves one token, four, the first two thirds, the last token of."""
    rng = np.random.default_rng(seed)
    x = torch.from_numpy((rng.standard_normal((4, n)) * 2.5).astype(np.float32))
    lowest = torch.finfo(torch.bfloat16 if bf16 else torch.float32).min
    fill = lowest if mask == "lowest" else mask
    keep = torch.zeros(4, n, dtype=torch.bool)
    keep[0, n // 2] = True
    keep[1, torch.from_numpy(rng.integers(0, n, 4))] = True
    keep[2, : n - n // 3] = True
    keep[3, n - 1] = True
    x[~keep] = fill
    tokens = torch.tensor([[n // 2, n - 1]] * 4, dtype=torch.int32)
    return x.bfloat16() if bf16 else x, tokens


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [1, 5, 70, 3000, 4096, 5001, 32003, 128256])
@pytest.mark.parametrize("mask", ["lowest", -1e31])
def test_finite_masks(be, bf16, n, mask):
    """Whole words, lanes and chunks at the type's lowest value, or at another far
    below any logit, in rows that end inside a chunk.  (bf16 rounds -1e31 alike
    for the call and the reference.)"""
    x, tokens = low_rows(n, bf16, mask, n)
    for temp, k in ((1.0, min(n, 20)), (1.5, 0)):
        check(be, x, tokens, temp, k)
    for off in (1, 3):                                     # rows that begin off 16 bytes
        wide = torch.full((4, n + 5 + off), math.nan, dtype=x.dtype, device="cuda")
        wide[:, off:off + n] = x.cuda()
        check(be, x, tokens, 1.0, min(n, 5), dev=wide[:, off:off + n])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [1, 5, 70, 5001, 128256])
@pytest.mark.parametrize("temp", [1e27, 1e29, 1.4e30])
def test_high_temperatures(be, bf16, n, temp):
    """All but uniform: nothing but the row's own entries counts, and a mask of
    -1e30 is a token like others."""
    rng = np.random.default_rng(n)
    x = torch.from_numpy((rng.standard_normal((3, n)) * 2.5).astype(np.float32))
    x[1, ::3] = -1e30
    x = x.bfloat16() if bf16 else x
    check(be, x, torch.tensor([[0, n - 1]] * 3, dtype=torch.int32), float(np.float32(temp)), min(n, 7))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [1, 5, 3000, 32003, 128256])
def test_rows_far_from_zero(be, bf16, n):
    """Rows that hold one value only, however large, are uniform: log s is not lost
    beside the reference."""
    t = torch.bfloat16 if bf16 else torch.float32
    f = torch.finfo(t)
    x = torch.tensor([f.min, -1e30, -1e18, 1e18, f.max], dtype=t)[:, None].expand(5, n).contiguous()
    tokens = torch.tensor([[0, n - 1]] * 5, dtype=torch.int32)
    for temp, k in ((1.0, min(n, 5)), (0.25, 0)):
        got = check(be, x, tokens, temp, k)
        assert (got["logprobs"].cpu().double() + math.log(n)).abs().max() <= 81 * U * max(1.0, math.log(n))
