"""Residual + RMS norm + codes (be42_norm_quant_rows_int8 / _fp8): the sum, the
scales and every code equal those of the definition in 64 bits, y rounded once
to fp32 and coded by the oracle's codec, bit for bit.  (Sums in 64 bits of two
orders differ by ~1e-16 of the row's rms, which moves the fp32 rounding of one
value in ~1e8; the tests hold ~1e6 values.)"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-5


def inputs(rng, rows, cols, bf16):
    x = (rng.standard_normal((rows, cols)) * 0.7).astype(np.float32)
    r = (rng.standard_normal((rows, cols)) * 2.0).astype(np.float32)
    x[:, ::37] *= 9.0
    w = torch.from_numpy((1.0 + 0.1 * rng.standard_normal(cols)).astype(np.float32)).bfloat16()
    dt = torch.bfloat16 if bf16 else torch.float32
    return torch.from_numpy(x).to(dt), torch.from_numpy(r).to(dt), w


def defined(orc, x, r, w, eps, kind):
    """(codes, scales, h) of CPU tensors."""
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    d = h.double().numpy()
    y = (d / np.sqrt((d * d).mean(1, keepdims=True) + np.float64(np.float32(eps))) * w.double().numpy()).astype(np.float32)
    rows = [(orc.quant_int8 if kind == "int8" else orc.quant_fp8)(np.ascontiguousarray(v)) for v in y]
    return np.stack([c for c, _ in rows]), np.array([s for _, s in rows], np.float32), h


def check(got, want, sum_given=True):
    q, s, h = got
    wq, ws, wh = want
    np.testing.assert_array_equal(s.cpu().numpy().view(np.uint32), ws.view(np.uint32))
    np.testing.assert_array_equal(q.cpu().numpy(), wq)
    if sum_given:
        assert torch.equal(h.cpu(), wh)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 3), (1, 17), (3, 64), (5, 250), (4, 1000), (7, 1024), (9, 2064),
                                       (1, 4096), (33, 4096), (3, 4100), (2, 8192), (3, 14336), (2, 16384), (2, 16388),
                                       (2, 20001), (1, 70000), (130, 96)])
def test_matches_definition(be, orc, kind, bf16, rows, cols):
    x, r, w = inputs(np.random.default_rng(rows * 100003 + cols), rows, cols, bf16)
    for res in (r, None):
        got = be.norm_quant_rows(x.cuda(), w.cuda(), EPS, kind, residual=None if res is None else res.cuda())
        assert (got[2] is None) == (res is None)
        check(got, defined(orc, x, res, w, EPS, kind), res is not None)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("cols", [40, 4096, 20004])
def test_sum_replaces_its_input(be, orc, kind, bf16, cols):
    x, r, w = inputs(np.random.default_rng(5), 6, cols, bf16)
    want = defined(orc, x, r, w, EPS, kind)
    for which in ("x", "residual"):
        a, b = x.cuda(), r.cuda()
        check(be.norm_quant_rows(a, w.cuda(), EPS, kind, residual=b, sum=a if which == "x" else b), want)
        assert torch.equal(a.cpu(), want[2] if which == "x" else x)
        assert torch.equal(b.cpu(), want[2] if which != "x" else r)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("cols", [256, 4096, 16400])
def test_strides_and_alignment(be, orc, kind, bf16, cols):
    """Rows inside wider ones, and rows that begin off 16 bytes."""
    rng = np.random.default_rng(6)
    for pad, off in ((8, 0), (5, 0), (3, 1), (16, 2)):
        x, r, w = inputs(rng, 3, cols, bf16)
        xw, rw = (torch.full((3, cols + pad + off), float("nan"), dtype=x.dtype, device="cuda") for _ in range(2))
        xw[:, off:off + cols], rw[:, off:off + cols] = x.cuda(), r.cuda()
        wide = torch.cat([torch.zeros(off, dtype=w.dtype), w]).cuda()[off:]
        got = be.norm_quant_rows(xw[:, off:off + cols], wide, EPS, kind, residual=rw[:, off:off + cols])
        check(got, defined(orc, x, r, w, EPS, kind))
        # outputs off their words too
        q = torch.zeros(3 * cols + 8, dtype=torch.uint8, device="cuda")[1:]
        s = torch.zeros(3, device="cuda")
        h = torch.zeros(3 * cols + off, dtype=x.dtype, device="cuda")[off:]
        fn = be.lib.be42_norm_quant_rows_int8 if kind == "int8" else be.lib.be42_norm_quant_rows_fp8
        assert fn(be.p(q), be.p(s), be.p(h), be.p(xw[:, off:]), xw.stride(0), be.p(rw[:, off:]), rw.stride(0), int(bf16),
                  be.p(wide), 3, cols, EPS, be.stream()) == 0, be.last_error()
        codes = q[:3 * cols].view(3, cols)
        check((codes.view(torch.int8) if kind == "int8" else codes, s, h[:3 * cols].view(3, cols)),
              defined(orc, x, r, w, EPS, kind))
        assert not q[3 * cols:].any()


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_codes_are_those_of_the_row_codec(be, kind):
    """Composed from the library's own codec on the GPU: the same bits."""
    x, r, w = (t.cuda() for t in inputs(np.random.default_rng(7), 50, 2048, False))
    q, s, h = be.norm_quant_rows(x, w, EPS, kind, residual=r)
    d = h.double()
    y = (d / torch.sqrt((d * d).mean(1, keepdim=True) + float(np.float32(EPS))) * w.double()).float()
    q2, s2 = be.quant_rows_int8(y) if kind == "int8" else be.quant_rows_fp8(y)
    assert torch.equal(q, q2) and torch.equal(s, s2)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("cols", [64, 4096, 20000])
def test_zero_tiny_and_large_rows(be, orc, kind, cols):
    x = torch.zeros(5, cols)
    x[1, 3] = 1e-30
    x[2] = 1e18
    x[3, ::2], x[3, 1::2] = 3e38, -3e38       # squares beyond fp32
    x[4] = 1e-22
    w = torch.ones(cols, dtype=torch.bfloat16)
    check(be.norm_quant_rows(x.cuda(), w.cuda(), EPS, kind), defined(orc, x, None, w, EPS, kind), False)
    # without eps a row of zeros is 0 / 0
    got = be.norm_quant_rows(x[1:].cuda(), w.cuda(), 0.0, kind)
    check(got, defined(orc, x[1:], None, w, 0.0, kind), False)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_bad_rows_stay_alone(be, orc, kind):
    x, r, w = inputs(np.random.default_rng(8), 6, 1024, False)
    want = defined(orc, x, r, w, EPS, kind)
    x[1, 5], x[4, 1000] = float("nan"), float("inf")
    q, s, h = be.norm_quant_rows(x.cuda(), w.cuda(), EPS, kind, residual=r.cuda())
    keep = [0, 2, 3, 5]
    np.testing.assert_array_equal(q.cpu().numpy()[keep], want[0][keep])
    np.testing.assert_array_equal(s.cpu().numpy()[keep], want[1][keep])


def test_refusals(be):
    x, w = torch.zeros(4, 64, device="cuda"), torch.ones(64, dtype=torch.bfloat16, device="cuda")
    import be42
    bad = [dict(kind="int4"), dict(x=x.half()), dict(x=x.t()), dict(w=w.float()), dict(w=w[:32]), dict(x=x.cpu()),
           dict(residual=x.bfloat16()), dict(residual=x[:2]), dict(residual=x[:, :32]), dict(sum=x[:, ::2]),
           dict(sum=x[:2]), dict(eps=-1.0), dict(x=x[0])]
    for kw in bad:
        a = dict(x=x, w=w, eps=EPS, kind="int8")
        a.update(kw)
        with pytest.raises(be42.Be42Error):
            be.norm_quant_rows(**a)
    q, s, h = be.norm_quant_rows(x[:0], w, EPS, "int8", residual=x[:0])
    assert q.shape == (0, 64) and s.shape == (0,) and h.shape == (0, 64)


def test_graph_and_other_stream(be, orc):
    """Captured on a stream of its own, replayed on new inputs with the
    program's own work between."""
    x, r, w = (t.cuda() for t in inputs(np.random.default_rng(9), 20, 4096, False))
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    be.norm_quant_rows(x, w, EPS, "fp8", residual=r)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        got = be.norm_quant_rows(x, w, EPS, "fp8", residual=r)
    for k in range(4):
        a, b, _ = inputs(np.random.default_rng(20 + k), 20, 4096, False)
        x.copy_(a)
        r.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        check(got, defined(orc, a, b, w.cpu(), EPS, "fp8"))
        assert torch.equal(be.norm_quant_rows(x, w, EPS, "fp8", residual=r)[0], got[0])


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("cols", [8, 3])
def test_more_rows_than_one_launch_takes(be, orc, kind, cols):
    rows = (1 << 21) + 3
    gen = torch.Generator().manual_seed(13)
    x, r = (torch.randn(rows, cols, generator=gen).bfloat16() for _ in range(2))
    w = torch.randn(cols, generator=gen).bfloat16()
    q, s, h = be.norm_quant_rows(x.cuda(), w.cuda(), EPS, kind, residual=r.cuda())
    at = [0, 1, rows // 2, (1 << 21) - 1, 1 << 21, rows - 1]
    check((q[at], s[at], h[at]), defined(orc, x[at], r[at], w, EPS, kind))
    assert torch.equal(h.cpu(), x + r)


@pytest.mark.parametrize("cols", [4096, 1001])
def test_rows_past_32_bits(be, orc, cols):
    """Three rows 2^31 - 8 elements apart, the last past 2^32."""
    apart = (1 << 31) - 8
    x, r, w = inputs(np.random.default_rng(14), 3, cols, True)
    far = torch.empty(2 * apart + cols, dtype=x.dtype, device="cuda").as_strided((3, cols), (apart, 1))
    far.copy_(x)
    check(be.norm_quant_rows(far, w.cuda(), EPS, "int8", residual=r.cuda()), defined(orc, x, r, w, EPS, "int8"))
    far.copy_(r)
    check(be.norm_quant_rows(x.cuda(), w.cuda(), EPS, "fp8", residual=far), defined(orc, x, r, w, EPS, "fp8"))


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("cols", [8193, 16383, 16384, 18432, 28672, 32764, 32768, 32776, 40001])
def test_long_rows(be, orc, kind, bf16, cols):
    """About the lengths at which the form of a row changes."""
    x, r, w = inputs(np.random.default_rng(cols), 3, cols, bf16)
    for res in (r, None):
        got = be.norm_quant_rows(x.cuda(), w.cuda(), EPS, kind, residual=None if res is None else res.cuda())
        check(got, defined(orc, x, res, w, EPS, kind), res is not None)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_the_longest_row(be, orc, kind):
    """A row of 2^31 - 1: a thread's place in it passes 32 bits with a sign.  61
    distinct values whose squares add up without rounding."""
    cols, period = 2 ** 31 - 1, 61
    base = ((torch.arange(period) - 30) / 8.0).bfloat16()
    d = base.double()
    full, rest = divmod(cols, period)
    mean = (full * (d * d).sum() + (d[:rest] * d[:rest]).sum()) / cols
    y = (d / torch.sqrt(mean + float(np.float32(EPS)))).float().numpy()
    codes, scale = (orc.quant_int8 if kind == "int8" else orc.quant_fp8)(y)
    some = 1 << 15                                         # periods that are repeated at once

    def row(v):
        v = v.cuda().repeat(some)
        return v.repeat(-(-cols // v.numel()))[:cols]

    q, s, h = be.norm_quant_rows(row(base)[None], torch.ones(cols, dtype=torch.bfloat16, device="cuda"), EPS, kind)
    assert h is None and s.cpu().numpy()[0] == np.float32(scale)
    assert torch.equal(q[0], row(torch.from_numpy(codes)))
