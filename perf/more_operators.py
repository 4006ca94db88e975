"""The operators of a layer that checks drafted tokens against a paged cache, as
cases that can be timed.

  append   norms of queries and keys, rotation, K and V into pages (Lib.rope_append)
  accept   the drafts that were right move behind their contexts (Lib.kv_accept)
  tree     attention of trees of drafts over contexts and drafts (Lib.tree_attention)
  product  activations in codes with a scale for 128 of them, times E4M3 weights
           with a scale for each block of 128 x 128 (Lib.linear_fp8_block)

Shapes are those of the benchmark's workloads (bench.py): 32 or 24 query heads
over 8 KV heads of 128, the tiny decoder's 8 heads of 64, 28 layers, 4096 and
14336 features, and odd ones between.

`own` selects the library's kernels; without it `run` is the same mathematics
in elementary torch operations.  `exact` restates it in 64 bits.  The codecs
(INT8 page rows: amax / 127, halves away from zero; E4M3: amax / 224, mantissas
rounded half up and capped at 7) are storage formats of the library, so their
fp32 steps are restated, as is the order in which the page pool gives out pages.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE, BLOCK = 16, 128
EPS = 1e-5
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


def listed():
    return [
        # one user's next token in one layer: latency
        dict(name="append_one", op="append", kv="bf16", heads=24, kv_heads=8, head_dim=128, runs=1, count=1, ctx=1000,
             bf16=False, norm=False, rot=128, pairs=False, placed=False),
        # a layer's drafts of 16 sequences, placed by their depth, INT8 pages
        dict(name="append_drafts", op="append", kv="int8", heads=32, kv_heads=8, head_dim=128, runs=1, count=261, ctx=0,
             bf16=False, norm=True, rot=128, pairs=False, placed=True),
        # prompts: bandwidth
        dict(name="append_prompts", op="append", kv="bf16", heads=32, kv_heads=8, head_dim=128, runs=4, count=4000, ctx=500,
             bf16=True, norm=True, rot=128, pairs=False, placed=False),
        # one sequence's accepted drafts, all layers of a small model: latency
        dict(name="accept_one", op="accept", kv="bf16", kv_heads=8, head_dim=128, layers=28, batch=1, drafts=16, count=5,
             ctx=90),
        # a serving batch's
        dict(name="accept_batch", op="accept", kv="int8", kv_heads=8, head_dim=128, layers=28, batch=24, drafts=24, count=7,
             ctx=60),
        # a few drafts of the tiny decoder behind short contexts: latency
        dict(name="tree_smallest", op="tree", kv="bf16", heads=8, kv_heads=8, head_dim=64, trees=2, drafts=5, ctx=300,
             bf16=False),
        # INT8 pages, larger trees of few sequences, heads that no tile divides
        dict(name="tree_int8", op="tree", kv="int8", heads=24, kv_heads=8, head_dim=128, trees=5, drafts=61, ctx=4001,
             bf16=False),
        # a serving batch with bf16 activations
        dict(name="tree_batch", op="tree", kv="bf16", heads=32, kv_heads=8, head_dim=128, trees=32, drafts=16, ctx=4096,
             bf16=True),
        # long contexts
        dict(name="tree_long", op="tree", kv="bf16", heads=32, kv_heads=8, head_dim=128, trees=16, drafts=64, ctx=32768,
             bf16=True),
        # one token's attention output: latency and the weights' bytes
        dict(name="product_one", op="product", m=1, n=4096, k=4096, x_bf16=False, y_bf16=False),
        # a few drafts' hidden rows, whose last block of features is short
        dict(name="product_drafts", op="product", m=261, n=2064, k=14352, x_bf16=False, y_bf16=False),
        # a prompt's gate or up product
        dict(name="product_prompt", op="product", m=4096, n=14336, k=4096, x_bf16=True, y_bf16=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (24, 8, 128), (8, 8, 64), (16, 2, 128), (12, 1, 64), (28, 4, 128)]


def draw(rng):
    op = rng.choice(["append", "accept", "tree", "tree", "product", "product"])
    heads, kv_heads, hd = rng.choice(HEADS)
    kv, bf16 = rng.choice(["bf16", "bf16", "int8"]), rng.random() < 0.5
    if op == "append":
        runs = _log(rng, 1, 64)
        return dict(op=op, kv=kv, heads=heads, kv_heads=kv_heads, head_dim=hd, runs=runs, count=_log(rng, 1, 12000 // runs),
                    ctx=rng.choice([0, _log(rng, 1, 800)]), bf16=bf16, norm=rng.random() < 0.6,
                    rot=rng.choice([hd, hd, hd // 2]), pairs=rng.random() < 0.3, placed=rng.random() < 0.3)
    if op == "accept":
        drafts = _log(rng, 2, 64)
        return dict(op=op, kv=kv, kv_heads=kv_heads, head_dim=hd, layers=_log(rng, 1, 28), batch=_log(rng, 1, 24),
                    drafts=drafts, count=min(drafts, _log(rng, 1, 8)), ctx=_log(rng, 1, 100))
    if op == "tree":
        trees, drafts = _log(rng, 1, 32), _log(rng, 1, 64)
        return dict(op=op, kv=kv, heads=heads, kv_heads=kv_heads, head_dim=hd, trees=trees, drafts=drafts,
                    ctx=_log(rng, 16, min(32768, 200000 // trees, 3000000 // (trees * drafts))), bf16=bf16)
    n, k = _log(rng, 128, 14336), _log(rng, 128, 14336)
    k = 16 * (k // 16)
    y_bf16 = rng.random() < 0.5
    most = 4096 * 14336 * 4096 // (1 if y_bf16 else 4)
    return dict(op=op, m=_log(rng, 1, max(2, min(4096, most // (n * k)))), n=n, k=k, x_bf16=bf16, y_bf16=y_bf16)


# ---- inputs ------------------------------------------------------------------


def _gen(seed, *more):
    g = torch.Generator(device="cuda")
    g.manual_seed(hash((int(seed),) + more) & 0x7FFFFFFFFFFF)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _cuda(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


def _plan(case, seed):
    """The slots of a pool: tokens that each holds beforehand; and a call's
    tokens, in order: their slot and position.  (Lengths are the case's, so that
    outputs have one shape; trees and paths are the seed's.)"""
    g, any_, op = np.random.default_rng(5), np.random.default_rng(seed), case["op"]
    if op == "append":
        held = g.integers(0, case["ctx"] + 1, case["runs"])
        count = g.integers(max(1, case["count"] // 2), case["count"] + 1, case["runs"])
        return dict(held=held, slot=np.arange(case["runs"]), pos0=held, count=count)
    if op == "accept":
        # slots: every layer's contexts, then every layer's drafts
        layers, batch, drafts = case["layers"], case["batch"], case["drafts"]
        ctx = g.integers(1, case["ctx"] + 1, batch)
        count = g.integers(1, case["count"] + 1, batch)
        # a path down a tree: later drafts, in order, of the sequence's own
        index = [b * drafts + np.sort(any_.choice(drafts, n, replace=False)) for b, n in enumerate(count)]
        return dict(held=np.concatenate([np.tile(ctx, layers), np.full(layers, batch * drafts)]),
                    slot=np.arange(layers * batch), src=layers * batch + np.repeat(np.arange(layers), batch),
                    pos0=np.tile(ctx, layers), count=np.tile(count, layers),
                    index=np.tile(np.concatenate(index), layers))
    lens = g.integers(0, case["ctx"] + 1, case["trees"])
    lens[0] = case["ctx"]
    size = g.integers(max(1, case["drafts"] // 2), case["drafts"] + 1, case["trees"])
    size[-1] = case["drafts"]
    starts = np.concatenate([[0], np.cumsum(size)])
    # a draft follows one of the eight before it, or the context
    parents = np.concatenate([np.arange(n) - 1 - np.minimum(any_.integers(0, 8, n), np.arange(n)) for n in size])
    return dict(held=np.concatenate([lens, [starts[-1]]]), lens=lens, starts=starts, parents=parents)


def _held(case, seed, slot, n):
    """K and V [n][kv_heads][head_dim] that a slot holds beforehand."""
    g, kvh, hd = _gen(seed, slot), case["kv_heads"], case["head_dim"]
    k, v = _randn(g, n, kvh, hd), _randn(g, n, kvh, hd)
    k[:: 97] *= 1.5
    return k, v


def _page_codes(x):
    """INT8 page rows: codes and scales [.., head_dim] -> [..]."""
    amax = x.abs().amax(-1)
    some, one = amax > 0, torch.ones_like(amax)
    full = torch.full_like(amax, 127.0)                  # a tensor: division by a number multiplies by its inverse
    scale = torch.where(some, amax / full, one)
    a = (x * torch.where(some, full / amax, one)[..., None]).abs()
    t = torch.trunc(a)
    c = (t + (a - t >= 0.5)).clamp(max=127.0)
    return torch.where(x < 0, -c, c).to(torch.int8), scale


def _table(case, p):
    """Physical page of every slot's pages, as the pool gives them out: from the
    last one down, to what each slot held, then to the call's tokens."""
    held = p["held"]
    end = held.copy()
    if "pos0" in p:
        end[p["slot"]] = p["pos0"] + p["count"]
    before, after = -(-held // PAGE), -(-end // PAGE)
    most = max(1, int(after.max()))
    cap = most * len(held)
    table, at = np.zeros((len(held), most), np.int64), 0
    for first, last in ((np.zeros_like(before), before), (before, after)):
        for s in range(len(held)):
            n = max(0, int(last[s] - first[s]))
            table[s, first[s]:first[s] + n] = cap - 1 - at - np.arange(n)
            at += n
    return table, most, cap


def _fill(case, seed, held, table, cap, dtype=None):
    """Pages as the pool lays them out, with what the slots hold."""
    kvh, hd, int8 = case["kv_heads"], case["head_dim"], case["kv"] == "int8"
    kind = dtype or (torch.int8 if int8 else BF16)
    t = dict(k=torch.zeros(cap, kvh, PAGE, hd, dtype=kind, device="cuda"),
             v=torch.zeros(cap, kvh, *((PAGE, hd) if int8 else (hd, PAGE)), dtype=kind, device="cuda"))
    if int8:
        t.update({x: torch.zeros(cap, kvh, PAGE, device="cuda", dtype=dtype or F32) for x in ("k_scale", "v_scale")})
    for slot, n in enumerate(held):
        if n:
            _store(t, *_held(case, seed, slot, int(n)), *_places(table, np.full(n, slot), np.arange(n)), int8)
    return t


def _places(table, slot, pos):
    return _cuda(table[slot, pos // PAGE], np.int64), _cuda(pos % PAGE, np.int64)


def _store(t, k, v, page, off, int8):
    """Rows of K and V to their places."""
    if int8:
        for x, rows in (("k", k), ("v", v)):
            codes, scale = _page_codes(rows)
            t[x][page, :, off] = codes
            t[x + "_scale"][page, :, off] = scale.to(t[x + "_scale"].dtype)
    else:
        t["k"][page, :, off] = k.to(t["k"].dtype)
        t["v"][page, :, :, off] = v.to(t["v"].dtype)


def _centroids(t, pages, out):
    """Mean key of head 0 of some pages."""
    k = t["k"][pages, 0].to(F32 if out.dtype == F32 else F64)
    if "k_scale" in t:
        k = k * t["k_scale"][pages, 0][..., None]
    out[pages] = k.sum(1) * (1.0 / PAGE)


def _sealed(table, held, slot, end, first):
    """Physical pages that are full, of each slot from its page `first` on."""
    return _cuda(np.concatenate([table[s, f:e // PAGE] for s, f, e in zip(slot, first, end)] or [[]]), np.int64)


def _qkv(case, seed, n):
    """The q/k/v product's rows of n tokens."""
    g, heads, kvh, hd = _gen(seed, -1), case["heads"], case["kv_heads"], case["head_dim"]
    x = _randn(g, n, (heads + 2 * kvh) * hd) * torch.where(torch.rand((heads + 2 * kvh) * hd, generator=g, device="cuda") < 0.02, 4.0, 1.0)
    x = x.to(BF16) if case["bf16"] else x
    w = [(1.0 + 0.1 * _randn(g, hd)).to(BF16) for _ in range(2)] if case["norm"] else [None, None]
    far = torch.randint(0, 8, (n,), generator=g, device="cuda", dtype=torch.int32)
    return x, w, far


def _angles(case, n):
    half = case["rot"] // 2
    a = np.arange(n)[:, None] * (10000.0 ** (-np.arange(half) / half))[None]
    return torch.from_numpy(np.cos(a).astype(np.float32)).cuda(), torch.from_numpy(np.sin(a).astype(np.float32)).cuda()


def _drafts(case, seed, n):
    q = _randn(_gen(seed, -1), n, case["heads"], case["head_dim"])
    return q.to(BF16) if case["bf16"] else q


def _weights(case, seed):
    """Activations with a few large features; E4M3 weights with a scale for each
    block, the largest of a block at the format's end."""
    g, m, n, k = _gen(seed), case["m"], case["n"], case["k"]
    x = _randn(g, m, k) * torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 8.0, 1.0)
    w = (_randn(g, n, k) * 100.0).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    sw = (0.5 + torch.rand(-(-n // BLOCK), -(-k // BLOCK), generator=g, device="cuda")) * 2e-4
    return x.to(BF16) if case["x_bf16"] else x, w.view(torch.uint8), sw


def prepare(case, seed):
    op = case["op"]
    s = dict(case)
    if own:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "42-berlin-engine_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import be42
        s["lib"] = be42.load()
        s["lib"].init()
    if op == "product":
        s["x"], s["w"], s["sw"] = _weights(case, seed)
        return s
    p = _plan(case, seed)
    kvh, hd = case["kv_heads"], case["head_dim"]
    table, most, cap = _table(case, p)
    if own:
        s["pool"] = s["lib"].kv_pool(be42.KV_BF16 if case["kv"] == "bf16" else be42.KV_INT8, len(p["held"]), kvh, hd, most)
        for slot, n in enumerate(p["held"]):
            if n:
                k, v = _held(case, seed, slot, int(n))
                s["pool"].append(slot, k.reshape(n, kvh * hd), v.reshape(n, kvh * hd), 0)
        s["pages"] = {x: t for x, t in s["pool"].tensors().items() if x in ("k", "v", "k_scale", "v_scale", "centroid")}
    else:
        s["pages"] = _fill(case, seed, p["held"], table, cap)
        if op != "tree":
            s["pages"]["centroid"] = torch.zeros(cap, hd, device="cuda")
            _centroids(s["pages"], _sealed(table, None, np.arange(len(p["held"])), p["held"], 0 * p["held"]), s["pages"]["centroid"])
    if op == "tree":
        n = int(p["starts"][-1])
        s["q"], s["scale"], s["total"] = _drafts(case, seed, n), 1.0 / math.sqrt(hd), n
        s["starts"], s["parents"], s["lens"] = _cuda(p["starts"]), _cuda(p["parents"]), _cuda(p["lens"])
        s["slots"] = torch.arange(case["trees"], dtype=torch.int32, device="cuda")
        s["table"] = _cuda(table, np.int64)
        return s
    if own:
        if op == "append":
            s["runs"] = np.stack([p["slot"], p["pos0"], p["count"]], 1).astype(np.int32)
        else:
            # of the first layer; the others' slots follow
            s["runs"] = np.stack([p["src"], p["slot"], p["pos0"], p["count"]], 1).astype(np.int32)[:case["batch"]]
            s["index"] = p["index"].astype(np.int32)[:len(p["index"]) // case["layers"]]
    else:
        slot = np.repeat(p["slot"], p["count"])
        pos = np.concatenate([a + np.arange(n) for a, n in zip(p["pos0"], p["count"])])
        s["page"], s["off"] = _places(table, slot, pos)
        s["full"] = _sealed(table, None, p["slot"], p["pos0"] + p["count"], p["pos0"] // PAGE)
        if op == "accept":
            s["from_page"], s["from_off"] = _places(table, np.repeat(p["src"], p["count"]), p["index"])
        else:
            s["pos"] = _cuda(pos)
    if op == "append":
        n, q = int(p["count"].sum()), case["heads"] * hd
        x, (s["q_norm"], s["k_norm"]), far = _qkv(case, seed, n)
        s["q"], s["k"], s["v"] = x[:, :q].unflatten(1, (-1, hd)), x[:, q:q + kvh * hd].unflatten(1, (-1, hd)), \
            x[:, q + kvh * hd:].unflatten(1, (-1, hd))
        s["cos"], s["sin"] = _angles(case, most * PAGE + 8)
        s["placed_at"] = None
        if case["placed"]:
            s["placed_at"] = far + _cuda(np.concatenate([a + np.arange(n) for a, n in zip(p["pos0"], p["count"])]))
        if own:
            s["rope"] = be42.Rope(s["cos"], s["sin"], interleaved=case["pairs"])
    return s


# ---- the operators -------------------------------------------------------------


def run(s):
    op = s["op"]
    if own:
        lib = s["lib"]
        if op == "append":
            q = lib.rope_append(s["pool"], s["runs"], s["k"], s["v"], q=s["q"], rope=s["rope"], positions=s["placed_at"],
                                q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
            return dict(s["pages"], q=q)
        if op == "accept":
            lib.kv_accept(s["pool"], s["runs"], s["index"], layers=s["layers"], from_step=1, to_step=s["batch"])
            return s["pages"]
        if op == "tree":
            return lib.tree_attention(s["pool"], s["q"], s["starts"], s["parents"], s["trees"], s["scale"], s["drafts"],
                                      slots=s["slots"], lens=s["lens"], max_len=s["ctx"])
        return lib.linear_fp8_block(s["x"], s["w"], s["sw"], dtype=BF16 if s["y_bf16"] else F32)
    return dict(append=_append, accept=_accept, tree=_tree, product=_product)[op](s)


def _normed(x, w):
    # in 64 bits, rounded once: codes lie on borders of the normalised value
    if w is None:
        return x.to(F32)
    d = x.to(F64)
    r = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + float(np.float32(EPS)))
    return (d * r * w.to(F64)).to(F32)


def _pairs(x, rot, pairs):
    if pairs:
        return x[..., 0:rot:2], x[..., 1:rot:2]
    return x[..., :rot // 2], x[..., rot // 2:rot]


def _unpair(a, b, pairs):
    return torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1)


def _rotated(x, c, s, rot, pairs):
    """One product of each is rounded to fp32, the other is not: their sum is
    rounded once."""
    a, b = _pairs(x, rot, pairs)
    a64, b64, c64, s64 = a.to(F64), b.to(F64), c.to(F64), s.to(F64)
    return torch.cat([_unpair((a64 * c64 - (b * s).to(F64)).to(F32), (a64 * s64 + (b * c).to(F64)).to(F32), pairs),
                      x[..., rot:]], -1)


def _append(s):
    at = (s["pos"] if s["placed_at"] is None else s["placed_at"]).long()
    c, sn = s["cos"][at][:, None], s["sin"][at][:, None]
    q = _rotated(_normed(s["q"], s["q_norm"]), c, sn, s["rot"], s["pairs"]).to(s["q"].dtype)
    k = _rotated(_normed(s["k"], s["k_norm"]), c, sn, s["rot"], s["pairs"])
    t = s["pages"]
    _store(t, k, s["v"].to(F32), s["page"], s["off"], s["kv"] == "int8")
    _centroids(t, s["full"], t["centroid"])
    return dict(t, q=q)


def _accept(s):
    t, a, b, c, d = s["pages"], s["from_page"], s["from_off"], s["page"], s["off"]
    t["k"][c, :, d] = t["k"][a, :, b]
    if s["kv"] == "int8":
        t["v"][c, :, d] = t["v"][a, :, b]
        t["k_scale"][c, :, d] = t["k_scale"][a, :, b]
        t["v_scale"][c, :, d] = t["v_scale"][a, :, b]
    else:
        t["v"][c, :, :, d] = t["v"][a, :, :, b]
    _centroids(t, s["full"], t["centroid"])
    return t


def _tree(s):
    kvh, hd, heads, trees = s["kv_heads"], s["head_dim"], s["heads"], s["trees"]
    grp, most, total, int8 = heads // kvh, s["drafts"], s["total"], s["kv"] == "int8"
    t = s["pages"]

    def rows(x, pages):
        """[..][pages] -> [..][kv heads][tokens][head_dim]"""
        y = t[x][pages].to(F32)
        if int8:
            y = y * t[x + "_scale"][pages][..., None]
        elif x == "v":
            y = y.transpose(-1, -2)
        return y.movedim(-3, -4).flatten(-3, -2)

    starts = s["starts"].long()
    j = torch.arange(most, device="cuda")
    at = starts[:-1, None] + j                           # [trees][most]: a tree's drafts
    real = at < starts[1:, None]
    at = at.clamp(max=total - 1)
    # what each draft sees of its tree: itself and what lies above it
    up = torch.eye(most, device="cuda", dtype=F64) + (s["parents"].long()[at][..., None] == j).to(F64)
    sees = (torch.linalg.matrix_power(up, most) > 0) & real[:, None, :]
    used = -(-s["ctx"] // PAGE)
    ctx = s["table"][:trees, :used]
    kc, vc = rows("k", ctx), rows("v", ctx)
    mine = s["table"][trees, :-(-total // PAGE)]
    kd, vd = (rows(x, mine)[:, at].transpose(0, 1) for x in "kv")      # [trees][kv heads][most][head_dim]
    q = s["q"].to(F32).view(total, kvh, grp, hd)[at].permute(0, 2, 1, 3, 4).reshape(trees, kvh, most * grp, hd)
    sc = torch.matmul(q, kc.transpose(2, 3)) * s["scale"]
    sd = torch.matmul(q, kd.transpose(2, 3)) * s["scale"]
    inside = torch.arange(used * PAGE, device="cuda") < s["lens"][:, None]
    sc = torch.where(inside[:, None, None, :], sc, -math.inf)
    sd = torch.where(sees.repeat_interleave(grp, 1)[:, None], sd, -math.inf)
    top = torch.maximum(sc.amax(-1), sd.amax(-1))[..., None]
    top = torch.where(top == -math.inf, 0.0, top)        # rows that are padding
    ec, ed = torch.exp(sc - top), torch.exp(sd - top)
    out = (torch.matmul(ec, vc) + torch.matmul(ed, vd)) / (ec.sum(-1) + ed.sum(-1))[..., None]
    out = out.view(trees, kvh, most, grp, hd).permute(0, 2, 1, 3, 4).reshape(trees, most, heads, hd)
    i = torch.arange(total, device="cuda")
    b = torch.searchsorted(starts[1:], i, right=True)
    return out[b, i - starts[b]].to(s["q"].dtype)


def _e4m3(y, scale):
    """E4M3 values of y / scale, as the library's codec rounds them."""
    v = y * (torch.ones_like(scale) / scale)
    a = v.abs().clamp(max=448.0)
    # floor of log2 rounded to fp32, as the codec's exponent is
    e = (torch.floor(torch.log2(a.to(F64)).to(F32)) + 7.0).clamp(0.0, 15.0)
    frac = torch.where(e == 0, a * 64.0, torch.ldexp(a, 7.0 - e) - 1.0)
    m = torch.trunc(frac * 8.0 + 0.5).clamp(max=7.0)
    c = torch.where(e == 0, m / 512.0, torch.ldexp(1.0 + m / 8.0, e - 7.0))
    return torch.where(a == 0, torch.zeros_like(c), torch.where(v < 0, -c, c))


def _blocks(k):
    return torch.arange(k, device="cuda") // BLOCK


def _product(s):
    m, k = s["x"].shape
    x = torch.nn.functional.pad(s["x"].to(F32), (0, -k % BLOCK)).view(m, -1, BLOCK)
    amax = x.abs().amax(-1)
    sx = torch.where(amax > 0, amax / torch.full_like(amax, 224.0), torch.ones_like(amax))[..., None]
    x = (_e4m3(x, sx) * sx).view(m, -1)[:, :k]
    w = s["w"].view(torch.float8_e4m3fn).to(F32) * s["sw"][_blocks(s["w"].shape[0])][:, _blocks(k)]
    return torch.matmul(x, w.t()).to(BF16 if s["y_bf16"] else F32)


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    op = case["op"]
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        blocks = -(-k // BLOCK)
        return dict(bytes=m * k * (2 if case["x_bf16"] else 4) + n * k + 4 * blocks * -(-n // BLOCK) +
                    m * n * (2 if case["y_bf16"] else 4), flops=2.0 * m * n * k)
    kvh, hd = case["kv_heads"], case["head_dim"]
    row = 2 * kvh * (hd * 2 if case["kv"] == "bf16" else hd + 4)
    p = _plan(case, 0)
    if op == "append":
        n, e = int(p["count"].sum()), 2 if case["bf16"] else 4
        return dict(bytes=n * ((2 * case["heads"] + 2 * kvh) * hd * e + row), flops=8.0 * n * (case["heads"] + 2 * kvh) * hd)
    if op == "accept":
        return dict(bytes=2 * row * int(p["count"].sum()), flops=0)
    n = int(p["starts"][-1])
    size = np.diff(p["starts"])
    depth = np.ones(n)
    for i in range(n):
        up = p["parents"][i]
        depth[i] += depth[p["starts"][np.searchsorted(p["starts"], i, side="right") - 1] + up] if up >= 0 else 0
    return dict(bytes=row * (int(p["lens"].sum()) + n) + 2 * n * case["heads"] * hd * (2 if case["bf16"] else 4),
                flops=4.0 * case["heads"] * hd * (float((size * p["lens"]).sum()) + float(depth.sum())))


# ---- the definition in 64 bits ---------------------------------------------------


def exact(case, seed):
    return dict(append=_exact_append, accept=lambda *_: None, tree=_exact_tree, product=_exact_product)[case["op"]](case, seed)


def _exact_append(case, seed):
    p = _plan(case, seed)
    kvh, hd, heads, half = case["kv_heads"], case["head_dim"], case["heads"], case["rot"] // 2
    table, most, cap = _table(case, p)
    int8 = case["kv"] == "int8"
    t = _fill(case, seed, p["held"], table, cap, None if int8 else F64)
    if not int8:
        # what was there is held in bf16
        t = {x: v.to(BF16).to(F64) for x, v in t.items()}
    pos = np.concatenate([a + np.arange(n) for a, n in zip(p["pos0"], p["count"])])
    x, w, far = _qkv(case, seed, len(pos))
    at = torch.from_numpy(pos).cuda() + (far if case["placed"] else 0)
    co, si = (a.double()[at][:, None] for a in _angles(case, most * PAGE + 8))
    x = x.double().view(len(pos), -1, hd)

    def turned(y, weight):
        if weight is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + float(np.float32(EPS))) * weight.double()
        z = torch.complex(y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if case["pairs"] else \
            torch.complex(y[..., :half], y[..., half:2 * half])
        z = z * torch.complex(co, si)
        out = y.clone()
        if case["pairs"]:
            out[..., 0:2 * half:2], out[..., 1:2 * half:2] = z.real, z.imag
        else:
            out[..., :half], out[..., half:2 * half] = z.real, z.imag
        return out

    q, k, v = turned(x[:, :heads], w[0]), turned(x[:, heads:heads + kvh], w[1]), x[:, heads + kvh:]
    page, off = _places(table, np.repeat(p["slot"], p["count"]), pos)
    out = dict(q=q)
    if int8:
        for name, rows in (("k", k), ("v", v)):
            amax = rows.abs().amax(-1)
            scale = t[name + "_scale"].double()
            scale[page, :, off] = torch.where(amax > 0, amax / 127.0, 1.0)
            out[name + "_scale"] = scale
        return dict(out, k=None, v=None, centroid=None)
    t["k"][page, :, off] = k
    t["v"][page, :, :, off] = v
    return dict(out, k=t["k"], v=t["v"], centroid=None)


def _exact_tree(case, seed):
    p = _plan(case, seed)
    kvh, hd, heads = case["kv_heads"], case["head_dim"], case["heads"]
    grp = heads // kvh

    def held(slot, n):
        """[kv heads][n][head_dim] as the pages hold them."""
        pair = _held(case, seed, slot, n)
        if case["kv"] == "bf16":
            return [t.to(BF16).to(F64).permute(1, 0, 2) for t in pair]
        coded = [_page_codes(t) for t in pair]
        return [(c.to(F64) * sc.to(F64)[..., None]).permute(1, 0, 2) for c, sc in coded]

    n = int(p["starts"][-1])
    q = _drafts(case, seed, n).to(F64).view(n, kvh, grp, hd)
    kd, vd = held(case["trees"], n)
    out = torch.empty(n, kvh, grp, hd, dtype=F64, device="cuda")
    for b in range(case["trees"]):
        lo, hi, ctx = int(p["starts"][b]), int(p["starts"][b + 1]), int(p["lens"][b])
        sees = np.zeros((hi - lo, hi - lo), bool)
        for i, up in enumerate(p["parents"][lo:hi]):     # a parent comes before its children
            if up >= 0:
                sees[i] = sees[up]
            sees[i, i] = True
        kc, vc = held(b, ctx)
        k, v = torch.cat([kc, kd[:, lo:hi]], 1), torch.cat([vc, vd[:, lo:hi]], 1)
        m = hi - lo
        z = torch.matmul(q[lo:hi].permute(1, 0, 2, 3).reshape(kvh, m * grp, hd), k.transpose(1, 2)) / math.sqrt(hd)
        hidden = torch.from_numpy(~sees).cuda().repeat_interleave(grp, 0)
        z[:, :, ctx:] = z[:, :, ctx:].masked_fill(hidden, -math.inf)
        out[lo:hi] = torch.matmul(torch.softmax(z, -1), v).view(kvh, m, grp, hd).permute(1, 0, 2, 3)
    return out.reshape(n, heads, hd)


def _exact_product(case, seed):
    x, w, sw = _weights(case, seed)
    x = x.cpu().float().numpy()
    m, k = x.shape
    pad = -(-k // BLOCK) * BLOCK - k
    x = np.pad(x, ((0, 0), (0, pad))).reshape(m, -1, BLOCK)
    amax = np.abs(x).max(-1)
    with np.errstate(divide="ignore", invalid="ignore"):
        scale = np.where(amax > 0, amax / np.float32(224.0), np.float32(1.0))
        mag = np.abs(x * (np.float32(1.0) / scale)[..., None])
        # binade of the magnitude; one that fp32's log2 rounds up to belongs to the next
        lg = np.log2(mag.astype(np.float64)).astype(np.float32)
    binade = np.clip(np.floor(np.maximum(lg, -100.0)).astype(np.int64), -7, 8)
    step = np.where(binade < -6, 2.0 ** -9, 2.0 ** (binade - 3.0))
    low = np.where(binade < -6, 0.0, 2.0 ** binade.astype(np.float64))
    # the codec adds its half in fp32
    code = np.trunc(((mag.astype(np.float64) - low) / step).astype(np.float32) + np.float32(0.5))
    val = np.sign(x) * (low + step * np.minimum(code, 7.0)) * scale.astype(np.float64)[..., None]
    val = torch.from_numpy(val.reshape(m, -1)[:, :k]).cuda()
    wide = w.view(torch.float8_e4m3fn).double()
    for b in range(sw.shape[1]):
        wide[:, b * BLOCK:(b + 1) * BLOCK] *= sw[:, b].double().repeat_interleave(BLOCK)[:w.shape[0], None]
    return torch.matmul(val, wide.t())
