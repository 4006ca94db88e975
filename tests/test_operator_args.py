"""Arguments that the norm + codes, prefix attention and log probability entry
points refuse, and their workspace sizes: checked before any device call, so
without a GPU.  The pointers are never followed."""
import ctypes as C

import pytest

import be42

PTR = 1 << 20          # an aligned address
INT_MAX = 2 ** 31 - 1


@pytest.fixture(scope="module")
def lib():
    return be42.Lib()


def refused(lib, rc, word):
    assert rc == -1, rc
    assert word in lib.last_error(), lib.last_error()


def norm(lib, fp8=False, **kw):
    a = dict(q=PTR, scales=PTR, sum=None, x=PTR, x_stride=64, residual=None, residual_stride=64, bf16=0, w=PTR, rows=4,
             cols=64, eps=1e-5)
    assert set(kw) <= set(a)
    a.update(kw)
    fn = lib.lib.be42_norm_quant_rows_fp8 if fp8 else lib.lib.be42_norm_quant_rows_int8
    return fn(*a.values(), None)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("kw,word", [
    (dict(q=None), "null"), (dict(scales=None), "null"), (dict(x=None), "null"), (dict(w=None), "null"),
    (dict(rows=-1), "shape"), (dict(cols=0), "shape"), (dict(x_stride=63), "stride"),
    (dict(residual=PTR, residual_stride=10), "stride"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(sum=PTR, x_stride=65), "contiguous"), (dict(sum=8 * PTR, residual=8 * PTR, residual_stride=80), "contiguous"),
    (dict(x=PTR + 2), "unaligned"), (dict(x=PTR + 1, bf16=1), "unaligned"), (dict(w=PTR + 1), "unaligned"),
    (dict(scales=PTR + 2), "unaligned"), (dict(sum=PTR + 2), "unaligned"), (dict(residual=PTR + 2), "unaligned"),
])
def test_norm_quant_refusals(lib, fp8, kw, word):
    refused(lib, norm(lib, fp8, **kw), word)


def test_norm_quant_no_rows(lib):
    assert norm(lib, rows=0) == 0
    assert norm(lib, True, rows=0) == 0


def score(lib, **kw):
    a = dict(logprobs=PTR, entropy=PTR, top_ids=PTR, top_logprobs=PTR, logits=PTR, bf16=0, row_stride=100, n=100, rows=3,
             temp=1.0, tokens=PTR, n_tokens=1, top_k=5, workspace=None, bytes=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.lib.be42_logprobs(*a.values(), None)


@pytest.mark.parametrize("kw,word", [
    (dict(rows=1 << 24, n=1, row_stride=1, top_k=1), "at most"),
    (dict(logits=None), "null"), (dict(n=0), "rows of"), (dict(rows=-1), "rows of"), (dict(row_stride=99), "stride"),
    (dict(n=(1 << 30) + 1, row_stride=INT_MAX), "rows of"),
    (dict(temp=0.0), "temperature"), (dict(temp=-1.0), "temperature"), (dict(temp=float("inf")), "temperature"),
    (dict(temp=float("nan")), "temperature"), (dict(temp=1e-40), "temperature"),
    (dict(n_tokens=-1), "tokens"), (dict(tokens=None), "tokens"), (dict(logprobs=None), "tokens"),
    (dict(top_k=-1), "top"), (dict(top_k=65), "top"), (dict(n=4, top_k=5), "top"),
    (dict(top_ids=None), "arrays"), (dict(top_logprobs=None), "arrays"),
    (dict(n_tokens=0, top_k=0, entropy=None), "nothing"), (dict(logits=PTR + 2), "unaligned"),
    (dict(logits=PTR + 1, bf16=1), "unaligned"), (dict(workspace=PTR, bytes=8), "workspace"),
    (dict(workspace=PTR + 8, bytes=1 << 30), "workspace"),
])
def test_logprobs_refusals(lib, kw, word):
    refused(lib, score(lib, **kw), word)


def test_logprobs_no_rows(lib):
    assert score(lib, rows=0) == 0


def test_logprobs_workspace(lib):
    f = lib.lib.be42_logprobs_workspace_bytes
    assert f(0, 1, 0) == 0 and f(10, 0, 0) == 0 and f(10, 1, 11) == 0 and f(100, 1, 65) == 0 and f(100, 1, -1) == 0
    assert f(1, 1, 0) == f(128256, 5000, 20) == 16                # in one launch
    assert 16 < f(128256, 1, 0) < f(128256, 1, 20) < f(128256, 40, 20)
    # sizes past 32 bits do not wrap
    assert f(INT_MAX, 1000, 64) > f(INT_MAX, 40, 64) >= f(128256, 40, 64)


def pool(**kw):
    a = dict(kind=be42.KV_BF16, n_layers=4, n_kv=2, head_dim=64, max_logical=8, capacity=32)
    a.update(kw)
    return be42.KVPoolStruct(**a)


def prefix(lib, p=None, **kw):
    p = p if p is not None else pool()
    a = dict(pool=C.addressof(p), q=PTR, q_bf16=0, q_stride=256, n_queries=3, n_heads=4,
             prefix_slot=3, prefix_len=20, slots=PTR, lens=PTR, max_len=16, scale=0.125, out=PTR, workspace=None, bytes=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.lib.be42_prefix_attention(*a.values(), None)


@pytest.mark.parametrize("kw,word", [
    (dict(pool=None), "null"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(n_heads=3), "heads"),
    (dict(n_heads=0), "heads"), (dict(n_queries=-1), "queries"), (dict(q_stride=255), "stride"),
    (dict(prefix_slot=4), "slot"), (dict(prefix_slot=-1), "slot"), (dict(prefix_len=129), "holds"),
    (dict(prefix_len=-1), "holds"), (dict(max_len=-1), "holds"),
    (dict(max_len=(1 << 30) + 1), "holds"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=-1e31), "scale"), (dict(q=PTR + 2), "unaligned"),
    (dict(out=PTR + 2), "unaligned"), (dict(q=PTR + 1, q_bf16=1), "unaligned"),
    (dict(n_queries=1 << 25, max_len=0), "queries of"), (dict(n_queries=1 << 24), "queries of"),
    (dict(slots=None, n_queries=5), "slots"), (dict(workspace=PTR + 8, bytes=1 << 30), "workspace"),
    (dict(workspace=PTR, bytes=8), "workspace"),
])
def test_prefix_attention_refusals(lib, kw, word):
    refused(lib, prefix(lib, **kw), word)


def test_prefix_attention_refuses_head_dims(lib):
    for hd in (8, 32, 96, 256):
        refused(lib, prefix(lib, pool(head_dim=hd), q_stride=4096), "head_dim")


def test_prefix_attention_no_queries(lib):
    assert prefix(lib, n_queries=0) == 0


def test_prefix_attention_workspace(lib):
    f = lib.lib.be42_prefix_attention_workspace_bytes
    assert f(0, 4, 2, 64, 10, 10) == 0 and f(1, 3, 2, 64, 10, 10) == 0 and f(1, 4, 2, 96, 10, 10) == 0
    assert f(1, 4, 2, 64, 1, INT_MAX) == 0 and f(1, 4, 2, 64, -1, 10) == 0 and f(1, 4, 2, 64, 10, -1) == 0
    assert f(1, 4, 2, 64, 0, 0) > 0 and f(128, 32, 8, 128, 32768, 1024) > 0
    # sizes past 32 bits do not wrap
    assert f(1 << 20, 64, 8, 128, 1 << 20, 1 << 20) >= f(1 << 10, 64, 8, 128, 1 << 20, 1 << 20) > 0


@pytest.mark.parametrize("shape,stride", [((2, 64), 1 << 31), ((2, 64), (1 << 32) + 64), ((1 << 31, 2), 2),
                                          ((1, (1 << 32) + 8), 1 << 33)])
def test_strides_and_shapes_past_32_bits(lib, shape, stride):
    """ctypes would pass them on cut to 32 bits."""
    import torch
    x = torch.empty(0, device="meta", dtype=torch.bfloat16).as_strided(shape, (stride, 1))
    with pytest.raises(be42.Be42Error, match="32 bits"):
        lib._rows("f", "x", x, (torch.bfloat16,))


@pytest.mark.parametrize("n_heads,hd", [(1 << 25, 64), (1 << 24, 128), (1 << 25, 128)])
def test_prefix_attention_heads_past_32_bits(lib, n_heads, hd):
    """The elements of a query's heads, counted in 32 bits, would be below any stride."""
    for n in (1, 2):
        refused(lib, prefix(lib, pool(head_dim=hd), n_heads=n_heads, n_queries=n, max_len=0), "stride")


@pytest.mark.parametrize("n_queries,n_heads", [(INT_MAX, 1 << 20), (1 << 29, 1 << 15), (INT_MAX, 1 << 24)])
def test_prefix_attention_rows_past_32_bits(lib, n_queries, n_heads):
    """Their tiles of 128, counted in 32 bits, would be none, or fewer than none."""
    assert lib.lib.be42_prefix_attention_workspace_bytes(n_queries, n_heads, 1, 64, 1000, 0) == 0
    assert lib.lib.be42_prefix_attention_workspace_bytes(n_queries, n_heads, 1, 64, 1000, 30) == 0
    p = pool(n_kv=1, max_logical=100)
    refused(lib, prefix(lib, p, n_queries=n_queries, n_heads=n_heads, q_stride=INT_MAX, prefix_len=1000, max_len=0), "queries of")


def test_logprobs_of_many_tokens(lib):
    """A wave's place among them is an int; ctypes would pass longer lists on cut to 32 bits."""
    for n_tokens in ((1 << 30) + 1, INT_MAX):
        refused(lib, score(lib, n_tokens=n_tokens), "tokens")
    import torch
    x = torch.empty(1, 64, device="meta")
    for kw, word in ((dict(tokens=torch.empty(1, (1 << 32) + 3, device="meta", dtype=torch.int32)), "32 bits"),
                     (dict(top_k=(1 << 32) + 3), "top"), (dict(top_k=-1), "top")):
        with pytest.raises(be42.Be42Error, match=word):
            lib.logprobs(x, **kw)
