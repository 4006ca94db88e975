"""A layer of a serving step from the library's operators, as they are used
together: residual + norm + codes -> QKV product -> append to the pages ->
attention behind the shared prefix -> codes -> output product -> residual + norm
+ codes -> logits product -> log probabilities.  Codes jump where a value crosses
the middle of two of them, so each step is compared with its definition in 64
bits over the values that the step before it left; captured and replayed, the
whole run repeats to the bit.

Tolerances: the INT8 product's sum is exact and at most 127^2 * 512 < 2^24, so
three roundings of half a step are left; the E4M3 product adds up k terms in
fp32, off by no more than k * 2^-23 of the sum of their sizes.  The attention's and the
log probabilities' are those of their own tests."""
import math

import numpy as np
import pytest
import torch

from test_gpu_norm_quant import check as check_codes, defined
from test_gpu_prefix_attention import PAGE, make_pool, reference as attended
from test_gpu_score import U, ids_of, reference as scored

pytestmark = pytest.mark.gpu

D, H, KVH, HD, VOCAB, EPS = 512, 8, 2, 64, 5003, 1e-5
SCALE = 1.0 / math.sqrt(HD)
# five sequences behind 203 shared tokens; three tokens of the first are scored at
# once, the others decode one each
OWN = [9, 0, 31, 16, 40]
SLOTS = [0, 0, 0, 1, 2, 3, 4]
POS = [9, 10, 11, 0, 31, 16, 40]
PREFIX_SLOT, PREFIX = 5, 203
MAX_LEN = 64


def e4m3(codes):
    c = codes.astype(np.int64)
    e, m = c >> 3 & 15, c & 7
    return np.where(c & 128, -1.0, 1.0) * np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))


def weights(be, rng, kind, n, k):
    w = torch.from_numpy((rng.standard_normal((n, k)) / math.sqrt(k)).astype(np.float32)).cuda()
    return (be.quant_rows_int8 if kind == "int8" else be.quant_rows_fp8)(w)


def check_product(y, q, s, w, sw, kind):
    val = (lambda c: c.cpu().numpy().astype(np.float64)) if kind == "int8" else (lambda c: e4m3(c.cpu().numpy()))
    a, b = val(q), val(w)
    sc = s.cpu().numpy().astype(np.float64)[:, None] * sw.cpu().numpy().astype(np.float64)[None, :]
    want = a @ b.T * sc
    tol = 3 * U * np.abs(want) + (0.0 if kind == "int8" else a.shape[1] * 2.0 ** -23) * (np.abs(a) @ np.abs(b).T) * sc
    off = np.abs(y.cpu().numpy().astype(np.float64) - want)
    assert (off <= tol).all(), (off - tol).max()


def held_as(a, kind):
    """[..., hd] fp32 as the pages hold it, in 64 bits."""
    if kind == "bf16":
        return torch.from_numpy(a).bfloat16().double().numpy()
    amax = np.abs(a).max(-1, keepdims=True)
    sc, inv = (amax / np.float32(127)).astype(np.float32), (np.float32(127) / amax).astype(np.float32)
    x = a * inv
    return np.trunc(x + np.copysign(np.float32(0.5), x)).clip(-127, 127).astype(np.float64) * sc


class Step:
    def __init__(self, be, kind, kv, seed):
        rng = np.random.default_rng(seed)
        self.be, self.kind, self.kv = be, kind, kv
        self.pool, self.k, self.v = make_pool(be, kv, 6, KVH, HD, OWN + [PREFIX], seed)
        self.w1, self.w2 = (torch.from_numpy((1 + 0.1 * rng.standard_normal(D)).astype(np.float32)).bfloat16().cuda()
                            for _ in range(2))
        self.qkv = weights(be, rng, kind, (H + 2 * KVH) * HD, D)
        self.proj = weights(be, rng, kind, D, H * HD)
        self.head = weights(be, rng, kind, VOCAB, D)
        B = len(SLOTS)
        self.x = torch.from_numpy(rng.standard_normal((B, D)).astype(np.float32)).cuda()
        self.delta = torch.from_numpy((0.3 * rng.standard_normal((B, D))).astype(np.float32)).cuda()
        self.tokens = torch.from_numpy(rng.integers(0, VOCAB, (B, 2)).astype(np.int32)).cuda()
        self.slots = torch.tensor(SLOTS, dtype=torch.int32, device="cuda")
        self.lens = torch.tensor([p + 1 for p in POS], dtype=torch.int32, device="cuda")
        size = max(be.lib.be42_prefix_attention_workspace_bytes(B, H, KVH, HD, PREFIX, MAX_LEN),
                   be.lib.be42_logprobs_workspace_bytes(VOCAB, B, 5))
        self.ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def run(self):
        be, r = self.be, {}
        r["q1"], r["s1"], r["h1"] = be.norm_quant_rows(self.x, self.w1, EPS, self.kind, residual=self.delta)
        r["qkv"] = be.gemm(r["q1"], r["s1"], *self.qkv, self.kind)
        k, v = (r["qkv"][:, (H + i * KVH) * HD:(H + (i + 1) * KVH) * HD].contiguous() for i in range(2))
        at = 0
        while at < len(SLOTS):                                    # runs of tokens of one sequence
            n = SLOTS[at:].count(SLOTS[at])
            self.pool.append(SLOTS[at], k[at:at + n], v[at:at + n], POS[at])
            at += n
        queries = r["qkv"][:, :H * HD].unflatten(1, (H, HD))      # strided rows
        r["attn"] = be.prefix_attention(self.pool, queries, PREFIX_SLOT, PREFIX, SCALE, slots=self.slots, lens=self.lens,
                                        max_len=MAX_LEN, workspace=self.ws)
        r["qa"], r["sa"] = (be.quant_rows_int8 if self.kind == "int8" else be.quant_rows_fp8)(r["attn"].view(-1, H * HD))
        r["out"] = be.gemm(r["qa"], r["sa"], *self.proj, self.kind)
        r["h2"] = r["h1"].clone()
        r["q2"], r["s2"], _ = be.norm_quant_rows(r["out"], self.w2, EPS, self.kind, residual=r["h2"], sum=r["h2"])
        r["logits"] = be.gemm(r["q2"], r["s2"], *self.head, self.kind)
        r.update(be.logprobs(r["logits"], self.tokens, temp=0.75, top_k=5, entropy=True, workspace=self.ws))
        return r


def check(step, r, orc):
    kind = step.kind
    check_codes((r["q1"], r["s1"], r["h1"]), defined(orc, step.x.cpu(), step.delta.cpu(), step.w1.cpu(), EPS, kind))
    check_product(r["qkv"], r["q1"], r["s1"], *step.qkv, kind)
    qkv = r["qkv"].cpu().numpy().reshape(len(SLOTS), H + 2 * KVH, HD)
    k, v = [a.copy() for a in step.k], [a.copy() for a in step.v]
    for b, (s, p) in enumerate(zip(SLOTS, POS)):
        k[s] = np.concatenate([k[s][:p], held_as(qkv[b:b + 1, H:H + KVH], step.kv)])
        v[s] = np.concatenate([v[s][:p], held_as(qkv[b:b + 1, H + KVH:], step.kv)])
    want, tol, _ = attended(qkv[:, :H].astype(np.float64), k, v, H, SCALE, PREFIX_SLOT, PREFIX, SLOTS,
                            [p + 1 for p in POS], MAX_LEN)
    off = np.abs(r["attn"].cpu().double().numpy() - want).max(-1)
    assert (off <= tol).all(), (off - tol).max()
    check_product(r["out"], r["qa"], r["sa"], *step.proj, kind)
    check_codes((r["q2"], r["s2"], r["h2"]), defined(orc, r["out"].cpu(), r["h1"].cpu(), step.w2.cpu(), EPS, kind))
    check_product(r["logits"], r["q2"], r["s2"], *step.head, kind)
    x = r["logits"].cpu()
    lp, ent, e, e_ent = scored(x, 0.75)
    for got, ids in ((r["logprobs"], step.tokens.cpu()), (r["top_logprobs"], ids_of(x, 5))):
        want = lp.gather(1, ids.long())
        assert ((got.cpu().double() - want).abs() <= e[:, None] + 4 * U * want.abs()).all()
    assert torch.equal(r["top_ids"].cpu(), ids_of(x, 5))
    assert ((r["entropy"].cpu().double() - ent).abs() <= e_ent).all()


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_each_step_of_the_run(be, orc, kind, kv):
    step = Step(be, kind, kv, 11)
    assert POS[0] // PAGE == POS[2] // PAGE and POS[5] % PAGE == 0
    check(step, step.run(), orc)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_the_run_captured(be, orc, kind):
    """One graph of the run, replayed over new inputs, between eager runs."""
    step = Step(be, kind, "bf16", 12)
    step.run()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        held = step.run()
    gen = torch.Generator().manual_seed(3)
    for i in range(4):
        step.x.copy_(torch.randn(step.x.shape, generator=gen))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = {n: t.clone() for n, t in held.items()}
        check(step, got, orc)
        eager = step.run()
        for n in got:
            assert torch.equal(got[n], eager[n]), (i, n)
        torch.cuda.synchronize()
