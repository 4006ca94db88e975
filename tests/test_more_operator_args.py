"""Arguments that the append with norms and rotation, the accepted drafts, the
tree attention and the products with block scales refuse, and their workspace
sizes: checked before any device call, so without a GPU.  The pointers are never
followed."""
import ctypes as C

import numpy as np
import pytest

import be42
from test_operator_args import INT_MAX, PTR, lib, pool, refused  # noqa: F401


def block_gemm(lib, **kw):
    a = dict(y=PTR, y_bf16=0, xq=PTR, sx=PTR, wq=PTR, sw=PTR, m=3, n=100, k=144, workspace=None, bytes=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.lib.be42_gemm_fp8_block(*a.values(), None)


def linear(lib, **kw):
    a = dict(y=PTR, y_bf16=0, x=PTR, x_bf16=0, x_stride=144, wq=PTR, sw=PTR, m=3, n=100, k=144, workspace=None, bytes=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.lib.be42_linear_fp8_block(*a.values(), None)


SHAPES = [(dict(m=-1), "m -1"), (dict(n=0), "n 0"), (dict(k=0), "k 0"), (dict(k=136), "multiple"), (dict(k=(1 << 22) + 16), "at most"),
          (dict(m=INT_MAX, n=INT_MAX), "m 2147483647")]


@pytest.mark.parametrize("kw,word", SHAPES + [
    (dict(y=None), "null"), (dict(xq=None), "null"), (dict(sx=None), "null"), (dict(wq=None), "null"), (dict(sw=None), "null"),
    (dict(xq=PTR + 8), "unaligned"), (dict(wq=PTR + 8), "unaligned"), (dict(y=PTR + 4), "unaligned"), (dict(sx=PTR + 2), "unaligned"),
    (dict(sw=PTR + 2), "unaligned"), (dict(workspace=PTR + 8, bytes=1 << 30), "workspace"), (dict(workspace=PTR, bytes=8), "workspace")])
def test_block_gemm_refusals(lib, kw, word):  # noqa: F811
    refused(lib, block_gemm(lib, **kw), word)


@pytest.mark.parametrize("kw,word", SHAPES[:5] + [
    (dict(m=INT_MAX, n=INT_MAX), "m 2147483647"), (dict(y=None), "null"), (dict(x=None), "null"), (dict(wq=None), "null"),
    (dict(sw=None), "null"), (dict(x_stride=143), "stride"), (dict(x=PTR + 2), "unaligned"), (dict(x=PTR + 1, x_bf16=1), "unaligned"),
    (dict(wq=PTR + 8), "unaligned"), (dict(workspace=PTR + 8, bytes=1 << 30), "workspace"), (dict(workspace=PTR, bytes=8), "workspace")])
def test_linear_refusals(lib, kw, word):  # noqa: F811
    refused(lib, linear(lib, **kw), word)


def test_no_rows(lib):  # noqa: F811
    assert block_gemm(lib, m=0, xq=None, y=None) == 0
    assert linear(lib, m=0) == 0
    assert lib.lib.be42_quant_blocks_fp8(None, None, None, 0, 64, 0, 64, None) == 0


@pytest.mark.parametrize("kw,word", [
    (dict(q=None), "null"), (dict(scales=None), "null"), (dict(x=None), "null"), (dict(rows=-1), "shape"), (dict(cols=0), "shape"),
    (dict(x_stride=63), "stride"), (dict(x=PTR + 2), "unaligned"), (dict(x=PTR + 1, x_bf16=1), "unaligned"),
    (dict(scales=PTR + 1), "unaligned"), (dict(rows=INT_MAX), "rows of")])
def test_quant_blocks_refusals(lib, kw, word):  # noqa: F811
    a = dict(q=PTR, scales=PTR, x=PTR, x_bf16=0, x_stride=64, rows=4, cols=64)
    a.update(kw)
    refused(lib, lib.lib.be42_quant_blocks_fp8(*a.values(), None), word)


def test_product_workspaces(lib):  # noqa: F811
    for f in (lib.lib.be42_gemm_fp8_block_workspace_bytes, lib.lib.be42_linear_fp8_block_workspace_bytes):
        for bad in ((0, 1, 16), (1, 0, 16), (1, 1, 0), (1, 1, 24), (1, 1, (1 << 22) + 16)):
            assert f(*bad, 0) == f(*bad, 1) == 0
        assert f(1, 4096, 4096, 0) == f(2, 4096, 4096, 1) == 16          # in one launch
    f = lib.lib.be42_linear_fp8_block_workspace_bytes
    assert f(1 << 20, 64, 1 << 16, 0) > 1 << 36       # sizes past 32 bits do not wrap
    for m, n, k in ((5, 64, 4096), (40, 4096, 4096), (261, 2064, 14352), (4096, 14336, 4096)):
        for yb in (0, 1):
            assert f(m, n, k, yb) >= lib.lib.be42_gemm_fp8_block_workspace_bytes(m, n, k, yb) + m * k + m * (-(-k // 128)) * 4
    assert lib.lib.be42_gemm_fp8_block_workspace_bytes(261, 2064, 14352, 0) > 16       # few tiles: in parts


def tree(lib, p=None, **kw):  # noqa: F811
    p = p if p is not None else pool()
    a = dict(pool=C.addressof(p), q=PTR, q_bf16=0, q_stride=256, n_tokens=9, n_heads=4, starts=PTR, n_trees=3, max_tree=5,
             parents=PTR, draft_slot=3, slots=PTR, lens=PTR, max_len=100, scale=0.125, out=PTR, workspace=None, bytes=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.lib.be42_tree_attention(*a.values(), None)


@pytest.mark.parametrize("kw,word", [
    (dict(pool=None), "null"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(starts=None), "null"),
    (dict(n_heads=3), "heads"), (dict(n_heads=0), "heads"), (dict(n_tokens=-1), "drafts"), (dict(q_stride=255), "stride"),
    (dict(n_trees=-1), "trees"), (dict(max_tree=0), "trees"), (dict(max_tree=257), "trees"), (dict(draft_slot=4), "slot"),
    (dict(draft_slot=-1), "slot"), (dict(max_len=-1), "max_len"), (dict(max_len=(1 << 30) + 1), "max_len"),
    (dict(scale=float("nan")), "scale"), (dict(scale=2e30), "scale"), (dict(q=PTR + 2), "unaligned"), (dict(out=PTR + 2), "unaligned"),
    (dict(q=PTR + 1, q_bf16=1), "unaligned"), (dict(starts=PTR + 2), "unaligned"), (dict(parents=PTR + 1), "unaligned"),
    (dict(slots=None, n_trees=5), "slots"), (dict(n_tokens=1 << 25), "drafts of"), (dict(n_trees=1 << 25), "trees of"),
    (dict(workspace=PTR + 8, bytes=1 << 30), "workspace"), (dict(workspace=PTR, bytes=8), "workspace")])
def test_tree_attention_refusals(lib, kw, word):  # noqa: F811
    refused(lib, tree(lib, **kw), word)


def test_tree_attention_head_dims_and_no_drafts(lib):  # noqa: F811
    refused(lib, tree(lib, pool(head_dim=72)), "head_dim")
    assert tree(lib, n_tokens=0) == 0 and tree(lib, n_trees=0) == 0


def test_tree_attention_workspace(lib):  # noqa: F811
    f = lib.lib.be42_tree_attention_workspace_bytes
    assert f(0, 1, 8, 2, 64, 4, 100) == 0 and f(4, 0, 8, 2, 64, 4, 100) == 0 and f(4, 1, 8, 3, 64, 4, 100) == 0
    assert f(4, 1, 8, 2, 96, 4, 100) == 0 and f(4, 1, 8, 2, 64, 0, 100) == 0 and f(4, 1, 8, 2, 64, 257, 100) == 0
    assert f(4, 1, 8, 2, 64, 4, -1) == 0 and f(4, 1, 8, 2, 64, 4, (1 << 30) + 1) == 0
    assert f(4, 1, 8, 2, 64, 4, 100) == 16                        # in one launch
    assert 16 < f(64, 1, 8, 2, 64, 64, 10000) < f(64, 1, 32, 2, 128, 64, 100000)
    assert f(1 << 20, 1 << 12, 32, 8, 128, 256, 4096) > 1 << 33   # sizes past 32 bits do not wrap


def runs(*rows):
    return np.array(rows, np.int32).reshape(len(rows), -1)


def append(lib, p=None, r=None, rope=None, **kw):  # noqa: F811
    p = p if p is not None else pool()
    r = runs((0, 0, 3)) if r is None else r
    rope = rope or dict(cos=PTR, sin=PTR, len=100, dim=64, interleaved=0)
    st = be42.RopeStruct(**rope)
    a = dict(pool=C.addressof(p), runs=r.ctypes.data, n_runs=len(r), n_tokens=3, q=PTR, q_stride=256, n_heads=4, k=PTR, k_stride=128, v=PTR,
             v_stride=128, bf16=0, q_norm=PTR, k_norm=PTR, eps=1e-5, rope=C.addressof(st), positions=None, q_out=PTR, q_out_stride=256)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.lib.be42_rope_append(*a.values(), None)


@pytest.mark.parametrize("kw,word", [
    (dict(pool=None), "null"), (dict(runs=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(n_runs=-1), "runs"),
    (dict(n_heads=3), "heads"), (dict(n_heads=0), "heads"), (dict(q=None), "heads"), (dict(q_out=None), "q_out"),
    (dict(q_stride=255), "strides"), (dict(k_stride=127), "strides"), (dict(v_stride=127), "strides"),
    (dict(q_out=2 * PTR, q_out_stride=255), "strides"), (dict(q_stride=300), "in place"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(q=PTR + 2, q_out=2 * PTR), "unaligned"), (dict(k=PTR + 2), "unaligned"),
    (dict(k=PTR + 1, bf16=1), "unaligned"), (dict(q_norm=PTR + 1), "unaligned"), (dict(positions=PTR + 2), "unaligned"),
    (dict(rope=dict(cos=None, sin=PTR, len=100, dim=64)), "table"), (dict(rope=dict(cos=PTR, sin=PTR, len=100, dim=66)), "rope"),
    (dict(rope=dict(cos=PTR, sin=PTR, len=100, dim=7)), "rope"), (dict(rope=dict(cos=PTR, sin=PTR, len=-1, dim=8)), "rope"),
    (dict(rope=dict(cos=PTR, sin=PTR + 1, len=9, dim=8)), "unaligned"), (dict(r=runs((0, 0, INT_MAX), (1, 0, INT_MAX))), "tokens"), (dict(n_tokens=4), "tokens"),
    (dict(n_tokens=-1), "tokens"), (dict(r=runs((0, 0, 4), (1, 0, -1))), "tokens")])
def test_rope_append_refusals(lib, kw, word):  # noqa: F811
    refused(lib, append(lib, **kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(pool=None), "null"), (dict(runs=None), "null"), (dict(index=None), "null"), (dict(n_runs=-1), "runs"), (dict(n_index=-1), "runs"),
    (dict(n_runs=0), "without a run"), (dict(layers=-1), "layers"), (dict(layers=5), "slots"), (dict(layers=INT_MAX, n_runs=INT_MAX), "slots")])
def test_kv_accept_refusals(lib, kw, word):  # noqa: F811
    p, r, i = pool(), runs((3, 0, 0, 1)), np.zeros(1, np.int32)
    a = dict(pool=C.addressof(p), runs=r.ctypes.data, n_runs=1, index=i.ctypes.data, n_index=1, layers=1, from_step=0, to_step=0)
    a.update(kw)
    refused(lib, lib.lib.be42_kv_accept(*a.values(), None), word)


def test_launches_past_what_a_grid_holds_are_refused(lib):  # noqa: F811
    """Whose first launch would fit, or whose pages would have been planned."""
    refused(lib, block_gemm(lib, m=1, n=1 << 28), "n 268435456")
    refused(lib, linear(lib, m=1, n=1 << 28), "n 268435456")
    refused(lib, tree(lib, n_heads=2, q_stride=128, n_trees=200000, max_tree=256, max_len=36000), "trees of")
    refused(lib, append(lib, n_heads=1 << 17, q_stride=1 << 23, q_out_stride=1 << 23), "heads")
    p, r, i = pool(), runs((3, 0, 0, 1)), np.zeros(1, np.int32)
    p.n_kv = 65536
    refused(lib, lib.lib.be42_kv_accept(C.addressof(p), r.ctypes.data, 1, i.ctypes.data, 1, 1, 0, 0, None), "kv heads")


def test_rope_layout_matches_the_header():
    assert [n for n, _ in be42.RopeStruct._fields_] == ["cos", "sin", "len", "dim", "interleaved"]
    assert C.sizeof(be42.RopeStruct) == 32
