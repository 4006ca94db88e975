"""Products with block scales (be42_quant_blocks_fp8, be42_gemm_fp8_block,
be42_linear_fp8_block).

Codes and scales are those of be42_quant_rows_fp8 of every group, to the bit.
Products against 64 bits over the codes.  Tolerance of fp32 outputs: products of
codes are exact in fp32; a block's sum of at most 128 terms, in any order and cut
instead of rounded, is off by 128 * 2^-23 of the sum of their sizes, the scale by
two roundings, the sum over blocks by one rounding a block.  bf16 outputs: a term
of a block's sum may be cut at 2^-17 of the largest of 64 (twice what is seen),
64 * 2^-17 <= 2^-11 of the sum of sizes, and half a step, 2^-8 of the output."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def values(q):
    return q.view(torch.float8_e4m3fn).double()


def spread(s, rows, cols, per_row):
    s = s.double()
    s = s if per_row else s.repeat_interleave(128, 0)[:rows]
    return s.repeat_interleave(128, 1)[:, :cols]


def operands(seed, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kb = -(-k // 128)

    def codes(rows):
        x = torch.randn(rows, k, generator=g, device="cuda") * torch.exp(2 * torch.randn(rows, 1, generator=g, device="cuda"))
        return (x * 20).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)

    sx = torch.exp(torch.randn(m, kb, generator=g, device="cuda"))
    sw = torch.exp(torch.randn(-(-n // 128), kb, generator=g, device="cuda"))
    return codes(m), sx, codes(n), sw


def check(y, xq, sx, wq, sw):
    (m, k), n = xq.shape, wq.shape[0]
    a, b = values(xq) * spread(sx, m, k, True), values(wq) * spread(sw, n, k, False)
    want, size = a @ b.T.contiguous(), a.abs() @ b.abs().T.contiguous()
    kb = sx.shape[1]
    if y.dtype == torch.bfloat16:
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + (kb + 2) * 2.0 ** -23) * size * 1.01
    else:
        tol = (128 + 2 + kb) * 2.0 ** -23 * size
    off = (y.double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol.clamp(min=1e-300)).max())


SHAPES = [(1, 4096, 4096), (1, 128, 128), (1, 1, 16), (2, 130, 48), (3, 127, 144), (16, 512, 2048), (15, 4096, 14336), (17, 256, 1024),
          (17, 129, 1040), (33, 64, 112), (64, 64, 128), (65, 200, 256), (100, 2064, 4112), (128, 128, 128), (129, 257, 400),
          (200, 1000, 2064), (256, 256, 4096), (300, 4096, 1024), (333, 2064, 528), (513, 640, 640), (1000, 1024, 2048),
          (2000, 2064, 1040), (1030, 4100, 512), (2, 14336, 4096), (8, 50000, 512), (40, 20000, 272), (70, 30000, 128)]


@pytest.mark.parametrize("yb", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products(be, m, n, k, yb):
    xq, sx, wq, sw = operands(m + n + k, m, n, k)
    y = be.gemm_fp8_block(xq, sx, wq, sw, dtype=torch.bfloat16 if yb else None)
    assert y.dtype == (torch.bfloat16 if yb else torch.float32) and y.shape == (m, n)
    check(y, xq, sx, wq, sw)


@pytest.mark.parametrize("yb", [False, True])
def test_every_code(be, yb):
    """All 254 numbers against one: exact."""
    codes = torch.tensor([c for c in range(256) if c & 127 != 127], dtype=torch.uint8, device="cuda")
    n = len(codes)
    for m in (1, 20, 300):
        wq = torch.zeros(n, 32, dtype=torch.uint8, device="cuda")
        wq[:, 17] = codes
        xq = torch.zeros(m, 32, dtype=torch.uint8, device="cuda")
        xq[:, 17] = 0x38
        one = torch.ones(m, 1, device="cuda")
        y = be.gemm_fp8_block(xq, one, wq, torch.ones(2, 1, device="cuda"), dtype=torch.bfloat16 if yb else None)
        assert (y.double() == values(codes)).all()


@pytest.mark.parametrize("yb", [False, True])
@pytest.mark.parametrize("m", [1, 7, 40, 200, 700])
def test_scales_that_are_no_numbers(be, yb, m):
    """Reach the outputs of their rows and features alone; a block of scale 0 or of
    zero codes adds nothing."""
    n, k = 300, 512
    xq, sx, wq, sw = operands(5, m, n, k)
    clean = be.gemm_fp8_block(xq, sx, wq, sw, dtype=torch.bfloat16 if yb else None)
    a, b = sx.clone(), sw.clone()
    a[m // 2, 1] = math.nan
    b[1, 3] = math.inf
    y = be.gemm_fp8_block(xq, a, wq, b, dtype=torch.bfloat16 if yb else None)
    rows = torch.arange(m, device="cuda") != m // 2
    cols = (torch.arange(n, device="cuda") // 128) != 1
    assert (y[rows][:, cols] == clean[rows][:, cols]).all()
    assert torch.isnan(y[m // 2]).all() and not torch.isfinite(y[:, ~cols].float()).any()
    a = sx.clone()
    a[:, 2] = 0
    z = xq.clone()
    z[:, 256:384] = 0
    p, q = (be.gemm_fp8_block(x, s, wq, sw, dtype=torch.bfloat16 if yb else None) for x, s in ((xq, a), (z, sx)))
    assert (p == q).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 127), (5, 129), (7, 4096), (1, 14336), (300, 1040), (2000, 272), (9, 130), (4, 250)])
def test_codes(be, bf16, rows, cols):
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(4 * torch.randn(rows, cols, generator=g, device="cuda"))
    x[rows // 2, : cols // 2] = 0
    x = x.bfloat16() if bf16 else x
    far = torch.empty(rows, cols + 3, dtype=x.dtype, device="cuda")[:, 1:cols + 1].copy_(x)
    pad = torch.nn.functional.pad(x.float(), (0, -cols % 128)).view(-1, 128).contiguous()
    q, s = be.quant_rows_fp8(pad)
    q = q.view(rows, -1)[:, :cols]
    for y in (x, far):
        got, sc = be.quant_blocks_fp8(y)
        assert (got == q).all() and (sc.view(-1) == s).all()


@pytest.mark.parametrize("yb", [False, True])
@pytest.mark.parametrize("xb", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_is_codes_and_product(be, m, n, k, xb, yb):
    _, _, wq, sw = operands(m * n + k, 1, n, k)
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn(m, k, generator=g, device="cuda") * torch.exp(torch.randn(m, k, generator=g, device="cuda"))
    x = x.bfloat16() if xb else x
    dt = torch.bfloat16 if yb else torch.float32
    far = torch.empty(m, k + 5, dtype=x.dtype, device="cuda")[:, 3:k + 3].copy_(x)
    xq, sx = be.quant_blocks_fp8(x)
    want = be.gemm_fp8_block(xq, sx, wq, sw, dtype=dt)
    for y in (x, far):
        got = be.linear_fp8_block(y, wq, sw, dtype=dt)
        assert got.dtype == dt
        check(got, xq, sx, wq, sw)
        # (up to four tokens' products are formed in the same launch, the same way)
        assert (got == want).all()


@pytest.mark.parametrize("m,n,k", [(4096, 14336, 2048), (4000, 14352, 2064), (3900, 14290, 2048)])
def test_more_tiles_than_whole_rounds(be, m, n, k):
    """Features that go in two launches of different tiles: the same bits as alone."""
    xq, sx, wq, sw = operands(m + n, m, n, k)
    y = torch.full((m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    be.gemm_fp8_block(xq, sx, wq, sw, out=y)
    for a in (0, 12160, n // 128 * 128 - 256):
        part = y[:, a:a + 1000 if a == 0 else n].contiguous()
        w = wq[a:a + part.shape[1]]
        check(part, xq, sx, w, sw[a // 128:a // 128 + -(-w.shape[0] // 128)])
        assert (be.gemm_fp8_block(xq, sx, w.contiguous(), sw[a // 128:a // 128 + -(-w.shape[0] // 128)].contiguous(), dtype=torch.bfloat16) == part).all()


def test_rows_do_not_change_with_the_batch_in_bits_that_count(be):
    """A row's output alone and among others: the same within its tolerance."""
    xq, sx, wq, sw = operands(1, 700, 384, 1040)
    for yb in (False, True):
        for m in (1, 5, 16, 17, 64, 65, 256, 700):
            y = be.gemm_fp8_block(xq[:m].contiguous(), sx[:m].contiguous(), wq, sw, dtype=torch.bfloat16 if yb else None)
            check(y, xq[:m], sx[:m], wq, sw)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (5, 300, 1040), (90, 500, 2048), (600, 2064, 1024)])
def test_streams_replays_and_outputs(be, m, n, k):
    import be42
    _, _, wq, sw = operands(3, 1, n, k)
    x = torch.randn(m, k, device="cuda")
    for dt in (torch.float32, torch.bfloat16):
        want = be.linear_fp8_block(x, wq, sw, dtype=dt)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = be.linear_fp8_block(x * 1.0, wq, sw, dtype=dt)
        s.synchronize()
        assert (got == want).all()
        ws = torch.empty(be.lib.be42_linear_fp8_block_workspace_bytes(m, n, k, int(dt == torch.bfloat16)), dtype=torch.uint8, device="cuda")
        out = torch.empty(m, n, dtype=dt, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            be.linear_fp8_block(x, wq, sw, out=out, workspace=ws)
        for i in range(4):
            x.copy_(torch.randn(m, k, device="cuda") * (i + 1))
            out.fill_(7)
            ws.fill_(255)
            g.replay()
            torch.cuda.synchronize()
            assert (out == be.linear_fp8_block(x, wq, sw, dtype=dt)).all()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = x + 1
            a = (y.data_ptr(), 0, y.data_ptr(), 0, k, wq.data_ptr(), sw.data_ptr(), m, n, k, None, 0, s.cuda_stream)
            assert be.lib.be42_linear_fp8_block(*a) == -1 and "workspace" in be.last_error()
    assert be42


def test_python_refusals(be):
    import be42
    xq, sx, wq, sw = operands(3, 4, 130, 144)
    x = torch.randn(4, 144, device="cuda")
    for bad in (dict(xq=xq[:, :128]), dict(xq=xq.to(torch.int8)), dict(sx=sx[:, :1]), dict(sx=sx.double()), dict(wq=wq[:, :128]),
                dict(wq=wq.to(torch.int8)), dict(sw=sw[:1]), dict(sw=sw.cpu()), dict(dtype=torch.float16), dict(out=torch.empty(4, 129, device="cuda")),
                dict(out=torch.empty(4, 130, device="cuda"), dtype=torch.bfloat16), dict(xq=xq[0])):
        with pytest.raises(be42.Be42Error):
            be.gemm_fp8_block(**dict(dict(xq=xq, sx=sx, wq=wq, sw=sw), **bad))
    for bad in (dict(x=x[:, :128]), dict(x=x.double()), dict(x=x.cpu()), dict(x=x.t()), dict(x=x[0]), dict(wq=wq.cpu()),
                dict(workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(be42.Be42Error):
            be.linear_fp8_block(**dict(dict(x=x, wq=wq, sw=sw), **bad))
    with pytest.raises(be42.Be42Error):
        be.linear_fp8_block(x[:, :136], wq[:, :136].contiguous(), sw)
    assert be.linear_fp8_block(x[:0], wq, sw).shape == (0, 130)
    assert be.gemm_fp8_block(xq[:0], sx[:0], wq, sw).shape == (0, 130)
