"""Bits of the products with block scales and of their codes, where they can be lost:
groups of the smallest magnitudes; sums of a block by the 8-bit matrix instructions,
which align the terms of eight elements (k = 8 i .. 8 i + 7) to the largest's exponent
and cut each below 2^-13 of it, and add these sums in fp32; rows of the largest k."""
import pytest
import torch

from test_gpu_block_product import operands, spread, values

pytestmark = pytest.mark.gpu


def tiny(rows, cols, seed):
    """Groups of 128 whose largest magnitudes lie around 224 * 2^-128, where 1 / scale
    becomes infinite, and down to the smallest of fp32; zeros of both signs among them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, -(-cols // 128), 128, generator=g, device="cuda")
    x[torch.rand(x.shape, generator=g, device="cuda") < 0.3] = 0.0
    x[torch.rand(x.shape, generator=g, device="cuda") < 0.1] = -0.0
    size = 2.0 ** torch.randint(-149, -110, x.shape[:2], generator=g, device="cuda").double()
    return (x.double() * size[..., None]).float().view(rows, -1)[:, :cols].contiguous()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 128), (300, 1040), (9, 130), (2, 4096)])
def test_codes_of_the_smallest_groups(be, bf16, rows, cols):
    """As be42_quant_rows_fp8 gives them for each group, to the bit."""
    x = tiny(rows, cols, rows + cols)
    x = x.bfloat16() if bf16 else x
    assert rows == 1 or float(x.double().abs().max()) > 224 * 2.0 ** -128 > float(x.double().abs()[x != 0].min())
    pad = torch.nn.functional.pad(x.float(), (0, -cols % 128)).view(-1, 128).contiguous()
    q, s = be.quant_rows_fp8(pad)
    far = torch.empty(rows, cols + 3, dtype=x.dtype, device="cuda")[:, 1:cols + 1].copy_(x)
    for y in (x, far):
        got, sc = be.quant_blocks_fp8(y)
        assert (got == q.view(rows, -1)[:, :cols]).all() and (sc.view(-1) == s).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("m", [1, 2, 3, 40])
def test_products_of_the_smallest_groups(be, bf16, m):
    """The product that forms the codes and the one of codes: the same bits."""
    n, k = 200, 1040
    _, _, wq, sw = operands(7, 1, n, k)
    sw = sw * 2.0 ** 100                               # (outputs that fp32 holds)
    x = tiny(m, k, m)
    x = x.bfloat16() if bf16 else x
    xq, sx = be.quant_blocks_fp8(x)
    want = be.gemm_fp8_block(xq, sx, wq, sw)
    assert torch.isfinite(want).all() and float(want.abs().max()) > 0
    assert (be.linear_fp8_block(x, wq, sw) == want).all()


def held(g, rows, k, low):
    """Codes of 1 .. 1.875 times 2^low .. 1, of either sign."""
    x = torch.randint(8, 16, (rows, k), generator=g, device="cuda").float() / 8
    x = x * 2.0 ** -torch.randint(0, 1 - low, (rows, k), generator=g, device="cuda").float()
    return torch.where(torch.rand(rows, k, generator=g, device="cuda") < 0.5, -x, x).to(torch.float8_e4m3fn).view(torch.uint8)


@pytest.mark.parametrize("yb", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 128, 128), (16, 300, 1040), (17, 129, 1040), (33, 64, 112), (100, 2064, 2048), (261, 516, 2048),
                                   (513, 640, 640), (1000, 1024, 2048), (2000, 2064, 1040), (4096, 14336, 2048), (3900, 14290, 1040)])
def test_sums_that_every_product_holds(be, yb, m, n, k):
    """Terms are multiples of 2^-11 and below 4, so that of any eight the last bit is at
    least 2^-11 of the largest's power of two; 2048 of them stay below 2^13, which fp32
    holds to 2^-11: sums are exact, powers of two as scales too, and bf16 outputs are
    rounded once."""
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    xq, wq = held(g, m, k, -3), held(g, n, k, -2)
    kb = -(-k // 128)
    sx = 2.0 ** torch.randint(-8, 9, (m, 1), generator=g, device="cuda").float().expand(m, kb).contiguous()
    sw = 2.0 ** torch.randint(-8, 9, (-(-n // 128), 1), generator=g, device="cuda").float().expand(-1, kb).contiguous()
    a, b = values(xq) * spread(sx, m, k, True), values(wq) * spread(sw, n, k, False)
    want = a @ b.T.contiguous()
    got = be.gemm_fp8_block(xq, sx, wq, sw, dtype=torch.bfloat16 if yb else None)
    assert (got == want.float().to(got.dtype)).all()


@pytest.mark.parametrize("m,n,k", [(17, 130, 1040), (40, 200, 272), (200, 256, 640)])
@pytest.mark.parametrize("shape", ["wide", "outliers", "cancelling"])
def test_what_8_bit_products_cut(be, m, n, k, shape):
    """bf16 outputs: seven terms of eight lose less than 2^-13 of the largest each; fp32
    sums of at most 16 groups a block, of their scaled sums and of the blocks lose at most
    2^-23 of the sizes each; the output's rounding is half a step."""
    g = torch.Generator(device="cuda").manual_seed(m * k)
    x = torch.randn(m, k, generator=g, device="cuda")
    if shape == "wide":
        x = x * torch.exp(2 * torch.randn(m, k, generator=g, device="cuda"))
    elif shape == "outliers":
        x = x / 16 * torch.where(torch.rand(k, generator=g, device="cuda") < 0.02, 4000.0, 1.0)
    else:
        x[:, 0::8] = 448.0
        x[:, 1::8] = -448.0
    w = torch.randn(n, k, generator=g, device="cuda") * 16
    if shape == "cancelling":
        w[:, 1::8] = w[:, 0::8]
    xq, wq = (t.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) for t in (x, w))
    kb = -(-k // 128)
    sx, sw = torch.rand(m, kb, generator=g, device="cuda") + 0.5, torch.rand(-(-n // 128), kb, generator=g, device="cuda") + 0.5
    a, b = values(xq) * spread(sx, m, k, True), values(wq) * spread(sw, n, k, False)
    want, size = a @ b.T.contiguous(), a.abs() @ b.abs().T.contiguous()
    most = torch.zeros_like(want)
    for i in range(0, k, 8):
        most += (a[:, None, i:i + 8] * b[None, :, i:i + 8]).abs().amax(-1)
    tol = 2.0 ** -8 * want.abs() + 1.01 * (7 * 2.0 ** -13 * most + (16 + 2 + kb) * 2.0 ** -23 * size)
    got = be.gemm_fp8_block(xq, sx, wq, sw, dtype=torch.bfloat16)
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    # exact sums in bf16: fp32 outputs, rounded by the caller
    tol = 2.0 ** -8 * want.abs() + 1.01 * (128 + 2 + kb) * 2.0 ** -23 * size
    off = (be.gemm_fp8_block(xq, sx, wq, sw).bfloat16().double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("yb", [False, True])
@pytest.mark.parametrize("m,n", [(2, 130), (16, 40), (20, 130), (300, 256)])
def test_the_largest_k(be, m, n, yb):
    """2^22 elements a row, some of them not zero: every sum is exact."""
    k = 1 << 22
    g = torch.Generator(device="cuda").manual_seed(m)
    at = torch.cat([torch.randint(0, k, (200,), generator=g, device="cuda"), k - 1 - torch.arange(20, device="cuda"), torch.arange(20, device="cuda")]).unique()
    xq = torch.zeros(m, k, dtype=torch.uint8, device="cuda")
    xq[:, at] = held(g, m, len(at), -3)
    wq = torch.full((n, k), 0x38, dtype=torch.uint8, device="cuda")
    wq[:, at] = held(g, n, len(at), -2)
    one, ones = torch.ones(m, k // 128, device="cuda"), torch.ones(-(-n // 128), k // 128, device="cuda")
    want = (values(xq[:, at]) @ values(wq[:, at]).T.contiguous()).float()
    dt = torch.bfloat16 if yb else torch.float32
    assert (be.gemm_fp8_block(xq, one, wq, ones, dtype=dt) == want.to(dt)).all()
    x = torch.zeros(m, k, device="cuda")
    x[:, at] = values(xq[:, at]).float()
    codes, scales = be.quant_blocks_fp8(x)
    assert (be.linear_fp8_block(x, wq, ones, dtype=dt) == be.gemm_fp8_block(codes, scales, wq, ones, dtype=dt)).all()
