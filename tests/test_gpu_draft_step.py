"""Steps that check drafted tokens, from the library's operators as they are used
together: in each layer the QKV product with block scales -> norms + rotation +
append to the drafts' slot -> attention of the draft trees -> output product; then
the accepted drafts of all layers go behind their sequences, and the next step
reads them there.  Each operator is compared with its definition in 64 bits over
the values that the one before it left; captured and replayed, the whole run
repeats to the bit.

Tolerances are those of the operators' own tests.  A key in the pages is off by
the rotation's tolerance and the page's rounding: half a step of bf16, 2^-8 of
itself, or of an INT8 row's codes, amax / 254, with its three fp32 roundings."""
import math

import numpy as np
import pytest
import torch

from test_gpu_block_product import check as check_product
from test_gpu_prefix_attention import make_pool
from test_gpu_rope_append import EPS, check_rows, held_rows, rotated, tables, weight
from test_gpu_tree_attention import check as check_attention, ints, path, starts_of, trees_of

pytestmark = pytest.mark.gpu

D, H, KVH, HD, LAYERS = 512, 8, 2, 64, 2
SCALE = 1.0 / math.sqrt(HD)
# four sequences; one has no context yet, one no drafts but the last token of its own
CTX = [37, 0, 203, 16]
SIZES = [7, 12, 1, 20]
MOST = 24
MAX_LEN = 256
B = len(CTX)
DRAFTS = LAYERS * B                                   # slots of the drafts, behind the sequences'
FEATURES = (H + 2 * KVH) * HD


def held(pool, slot, n):
    """K and V of a slot's first n tokens [n][kvh][hd], in 64 bits."""
    if n == 0:
        return np.zeros((0, KVH, HD)), np.zeros((0, KVH, HD))
    r = {k: x.double().cpu().numpy() for k, x in held_rows(pool, slot, n).items()}
    return tuple(r[w] * (r[w + "_scale"][..., None] if w + "_scale" in r else 1.0) for w in "kv")


class Steps:
    def __init__(self, be, kv, bf16, seed):
        import be42
        rng = np.random.default_rng(seed)
        self.be, self.kv, self.dt = be, kv, torch.bfloat16 if bf16 else torch.float32
        n = sum(SIZES)
        self.pool, _, _ = make_pool(be, kv, LAYERS * (B + 1), KVH, HD, CTX * LAYERS + [n] * LAYERS, seed)
        self.parents = trees_of(rng, SIZES)
        self.accepted = [path(self.parents[a:], i)[::-1] for a, i in zip(starts_of(SIZES), [6, 9, 0, 17])]
        depth = [len(path(self.parents[a:a + s], i)) - 1 for a, s in zip(starts_of(SIZES), SIZES) for i in range(s)]
        self.cos, self.sin = tables(MAX_LEN, HD // 2)
        self.rope = be42.Rope(torch.from_numpy(self.cos).cuda(), torch.from_numpy(self.sin).cuda())

        def product(rows, cols):
            w = rng.standard_normal((rows, cols)) / math.sqrt(cols)
            scale = np.abs(w.reshape(rows // 128, 128, cols // 128, 128)).max((1, 3)).astype(np.float32) / 448
            q = torch.from_numpy(w / scale.repeat(128, 0).repeat(128, 1)).float().to(torch.float8_e4m3fn)
            return q.view(torch.uint8).cuda(), torch.from_numpy(scale).cuda()

        self.qkv = [product(FEATURES, D) for _ in range(LAYERS)]
        self.proj = [product(D, H * HD) for _ in range(LAYERS)]
        self.qw, self.kw = [[weight(rng, HD) for _ in range(LAYERS)] for _ in range(2)]
        self.norms = [(a.cuda(), b.cuda()) for a, b in zip(self.qw, self.kw)]
        # the drafts, then one token behind each sequence's accepted ones
        self.x = [torch.from_numpy(rng.standard_normal((m, D)).astype(np.float32)).to(self.dt).cuda() for m in (n, B)]
        ctx = [CTX, [c + len(a) for c, a in zip(CTX, self.accepted)]]
        self.trees = [(SIZES, self.parents, ctx[0], np.repeat(ctx[0], SIZES) + depth), ([1] * B, np.full(B, -1), ctx[1], np.array(ctx[1]))]
        self.on_gpu = [(ints(starts_of(s)), ints(p), ints(c), ints(pos)) for s, p, c, pos in self.trees]
        self.slots = [ints(l * B + np.arange(B)) for l in range(LAYERS)]
        yb = int(bf16)
        self.ws = torch.empty(max([be.lib.be42_tree_attention_workspace_bytes(n, B, H, KVH, HD, MOST, MAX_LEN)] +
                                  [be.lib.be42_linear_fp8_block_workspace_bytes(m, o, i, yb) for m in (n, B)
                                   for o, i in ((FEATURES, D), (D, H * HD))]), dtype=torch.uint8, device="cuda")

    def step(self, i, look=None):
        """Step i; `look` is called when a layer's rows are in the pages and read."""
        be, x, r = self.be, self.x[i], []
        starts, parents, lens, pos = self.on_gpu[i]
        for l in range(LAYERS):
            y = be.linear_fp8_block(x, *self.qkv[l], dtype=self.dt, workspace=self.ws)
            q, k, v = y.view(-1, H + 2 * KVH, HD).split((H, KVH, KVH), 1)
            given = q.clone()
            q = be.rope_append(self.pool, [(DRAFTS + l, 0, len(x))], k, v, q=q, rope=self.rope, positions=pos,
                               q_norm=self.norms[l][0], k_norm=self.norms[l][1], eps=EPS, out=q)
            attn = be.tree_attention(self.pool, q, starts, parents, DRAFTS + l, SCALE, MOST, slots=self.slots[l], lens=lens,
                                     max_len=MAX_LEN, workspace=self.ws)
            out = be.linear_fp8_block(attn.view(-1, H * HD), *self.proj[l], dtype=self.dt, workspace=self.ws)
            r.append(dict(x=x, given=given, y=y, q=q, attn=attn, out=out))
            x = x + out
            if look:
                look(i, l, r[-1])
        return r

    def accept(self):
        starts = starts_of(SIZES)
        runs = [(DRAFTS, b, CTX[b], len(a)) for b, a in enumerate(self.accepted)]
        self.be.kv_accept(self.pool, runs, np.concatenate([starts[b] + a for b, a in enumerate(self.accepted)]),
                          layers=LAYERS, from_step=1, to_step=B)

    def run(self, look=None, accepted=None):
        r = self.step(0, look)
        self.accept()
        if accepted:
            accepted()
        return r + self.step(1, look)

    def check(self, i, l, r):
        sizes, parents, ctx, pos = self.trees[i]
        n, be = sum(sizes), self.be
        k, v = r["y"].view(n, -1, HD)[:, H:].split((KVH, KVH), 1)
        for x, y, w in ((r["x"], torch.cat([r["given"], k, v], 1).view(n, -1), self.qkv[l]),
                        (r["attn"].view(n, -1), r["out"], self.proj[l])):
            check_product(y, *be.quant_blocks_fp8(x), *w)
        check_rows(r["q"], r["given"].cpu(), self.qw[l], self.cos, self.sin, pos, HD, False)
        k, v = k.cpu().double().numpy(), v.cpu().double().numpy()
        k, tol = rotated(k, self.kw[l].double().numpy(), self.cos, self.sin, pos, HD, False)
        pages = [held(self.pool, s, c) for s, c in zip(range(l * B, l * B + B), ctx)] + [held(self.pool, DRAFTS + l, n)]
        for want, e, got in ((k, tol, pages[B][0]), (v, 0 * tol, pages[B][1])):
            if self.kv == "bf16":
                e = 1.01 * e + 2.0 ** -8 * np.abs(want)
            else:
                e = e + ((np.abs(want) + e).max(-1, keepdims=True)) / 127 * (0.5 + 127 * 3 * 2.0 ** -24)
            assert (np.abs(got - want) <= e).all()
        check_attention(r["attn"], r["q"].cpu(), [p[0] for p in pages], [p[1] for p in pages], H, SCALE, starts_of(sizes), parents,
                        B, list(range(B)), ctx, MAX_LEN)


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
def test_each_step_of_the_run(be, kv, bf16):
    s = Steps(be, kv, bf16, 5)
    assert [len(a) for a in s.accepted][2] == 1 and sum(len(a) for a in s.accepted) > B
    before = {}

    def look(i, l, r):
        s.check(i, l, r)
        if i == 0:
            before[l] = [held(s.pool, l * B + b, c) for b, c in enumerate(CTX)], held(s.pool, DRAFTS + l, sum(SIZES))

    def accepted():
        for l in range(LAYERS):
            for b, (c, a) in enumerate(zip(CTX, s.accepted)):
                got, (own, drafts) = held(s.pool, l * B + b, c + len(a)), before[l]
                for j in range(2):
                    assert (got[j][:c] == own[b][j]).all() and (got[j][c:] == drafts[j][starts_of(SIZES)[b] + a]).all()

    s.run(look, accepted)


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("bf16", [False, True])
def test_the_run_captured(be, kv, bf16):
    """One graph of both steps, replayed over new inputs, between eager runs."""
    s = Steps(be, kv, bf16, 6)
    s.run()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        got = s.run()
    gen = torch.Generator().manual_seed(7)
    for i in range(4):
        for x in s.x:
            x.copy_(torch.randn(x.shape, generator=gen))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        replayed = [{n: t.clone() for n, t in r.items()} for r in got]
        pages = {n: t.clone() for n, t in s.pool.tensors().items()}
        eager = s.run()
        torch.cuda.synchronize()
        for a, b in zip(replayed, eager):
            for n in a:
                assert torch.equal(a[n], b[n]), (i, n)
        for n, t in s.pool.tensors().items():
            assert torch.equal(pages[n].view(torch.uint8), t.view(torch.uint8)), (i, n)
