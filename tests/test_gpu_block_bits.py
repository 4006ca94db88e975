"""Bits of the products with block scales and of their codes, where they can be lost:
groups of the smallest magnitudes."""
import numpy as np
import pytest
import torch

from test_gpu_block_product import operands

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
