"""The operators that score and answer a batch which shares one prompt, as
cases that can be timed.

  norm    residual addition + RMS norm + 8-bit codes with one scale a row, the
          input form of the prefill products (Lib.norm_quant_rows)
  prefix  attention of many queries over a shared prefix slot of the page pool
          and every query's own slot (Lib.prefix_attention)
  score   log probabilities of given tokens, entropy and the top alternatives
          of logits rows (Lib.logprobs)

Shapes are those of the benchmark's workloads (bench.py): 32 or 24 query heads
over 8 KV heads of 128, the tiny decoder's 8 heads of 64, 4096 and 14336
features, vocabularies of 128256 and 4096, and odd ones between.

`own` selects the library's kernels; without it `run` is the same mathematics
in elementary torch operations.  `exact` restates it in 64 bits.  The row
codecs (INT8: amax / 127, halves away from zero; E4M3: amax / 224, mantissas
rounded half up and capped at 7) are storage formats of the library, so their
fp32 steps are restated, as are those of the INT8 pages.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 16
EPS = 1e-5
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


def listed():
    return [
        # one user's token before the q/k/v products: latency
        dict(name="norm_one", op="norm", kind="int8", rows=1, cols=4096, bf16=False, res=True),
        # a few sequences' continuations, rows that no tile divides, a bf16 stream
        dict(name="norm_ragged", op="norm", kind="fp8", rows=777, cols=2064, bf16=True, res=True),
        # the norm of an FFN's hidden row before the down product, no residual
        dict(name="norm_wide", op="norm", kind="fp8", rows=300, cols=14336, bf16=False, res=False),
        # a long prompt: bandwidth
        dict(name="norm_prompt", op="norm", kind="int8", rows=8192, cols=4096, bf16=False, res=True),
        # two answers of the tiny decoder behind a short prompt: latency
        dict(name="prefix_smallest", op="prefix", kv="bf16", heads=8, kv_heads=8, head_dim=64, prefix=300, batch=2,
             per=1, own_max=40, bf16=False),
        # a serving batch behind a system prompt that ends inside a page
        dict(name="prefix_batch", op="prefix", kv="bf16", heads=32, kv_heads=8, head_dim=128, prefix=8190, batch=32,
             per=1, own_max=256, bf16=False),
        # multiple choice: four tokens of each of 14 continuations at once, INT8 pages
        dict(name="prefix_choices", op="prefix", kv="int8", heads=24, kv_heads=8, head_dim=128, prefix=4001, batch=14,
             per=4, own_max=61, bf16=False),
        # a large batch behind a long document
        dict(name="prefix_large", op="prefix", kv="bf16", heads=32, kv_heads=8, head_dim=128, prefix=32768, batch=128,
             per=1, own_max=1024, bf16=True),
        # the chosen token of one sequence with 20 alternatives: latency
        dict(name="score_one", op="score", rows=1, vocab=128256, tokens=1, top_k=20, temp=1.0, bf16=False, masked=False),
        # answers among four letters, a grammar's mask, an odd vocabulary
        dict(name="score_choices", op="score", rows=333, vocab=32003, tokens=4, top_k=0, temp=1.0, bf16=False, masked=True),
        # a decode batch, alternatives at a temperature
        dict(name="score_batch", op="score", rows=48, vocab=128256, tokens=1, top_k=5, temp=0.7, bf16=False, masked=False),
        # every token of a prompt: bandwidth
        dict(name="score_prompt", op="score", rows=2000, vocab=128256, tokens=1, top_k=5, temp=1.0, bf16=True, masked=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "prefix", "prefix", "score"])
    bf16 = rng.random() < 0.4
    if op == "norm":
        cols = _log(rng, 64, 14336)
        return dict(op=op, kind=rng.choice(["int8", "fp8"]), rows=_log(rng, 1, 8192 * 4096 // max(cols, 4096)),
                    cols=16 * (cols // 16) if rng.random() < 0.7 else cols, bf16=bf16, res=rng.random() < 0.7)
    if op == "prefix":
        heads, kv_heads, hd = rng.choice([(32, 8, 128), (24, 8, 128), (8, 8, 64), (16, 2, 128), (12, 1, 64), (28, 4, 128)])
        per = rng.choice([1, 1, 1, 2, 5])
        return dict(op=op, kv=rng.choice(["bf16", "bf16", "int8"]), heads=heads, kv_heads=kv_heads, head_dim=hd,
                    prefix=_log(rng, 16, 32768), batch=_log(rng, 1, 128 // per), per=per, own_max=_log(rng, per, 1024),
                    bf16=bf16)
    vocab = _log(rng, 4096, 128256)
    return dict(op=op, rows=_log(rng, 1, 1900 * 128256 // max(vocab, 32000) // (1 if bf16 else 2)), vocab=vocab,
                tokens=rng.choice([1, 1, 2, 4]), top_k=rng.choice([0, 1, 5, 20]), temp=rng.choice([1.0, 1.0, 0.7, 1.3]),
                bf16=bf16, masked=rng.random() < 0.3)


# ---- inputs ------------------------------------------------------------------


def _gen(seed, *more):
    g = torch.Generator(device="cuda")
    g.manual_seed(hash((int(seed),) + more) & 0x7FFFFFFFFFFF)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _norm_inputs(case, seed):
    """A residual stream with a few large features, the layer's output that is
    added to it, and a norm weight around one."""
    g, rows, cols = _gen(seed), case["rows"], case["cols"]
    spread = torch.where(torch.rand(cols, generator=g, device="cuda") < 0.01, 8.0, 1.0)
    t = BF16 if case["bf16"] else F32
    x = (0.7 * _randn(g, rows, cols) * (spread if not case["res"] else 1.0)).to(t)
    res = (2.0 * _randn(g, rows, cols) * spread).to(t) if case["res"] else None
    return x, res, (1.0 + 0.1 * _randn(g, cols)).to(BF16)


def _prefix_shape(case):
    """Pages of a slot, and the slots: every sequence's own, then the prefix."""
    return -(-max(case["prefix"], case["own_max"]) // PAGE), case["batch"] + 1


def _lens(case, seed):
    """Own tokens of every sequence (0 .. own_max, at least what its queries
    stand on), and what each query sees: query j of a sequence the tokens up
    to its own position."""
    g, per = np.random.default_rng(seed), case["per"]
    own_len = g.integers(per if per > 1 else 0, case["own_max"] + 1, case["batch"])
    sees = (own_len[:, None] - (per - 1) + np.arange(per)).reshape(-1)
    return own_len, sees


def _tokens_of(case, seed, slot, n):
    """K and V [n][kv_heads][head_dim] of a slot, N(0, 1); the prefix holds
    some keys that many queries look at."""
    g, kvh, hd = _gen(seed, slot), case["kv_heads"], case["head_dim"]
    k, v = _randn(g, n, kvh, hd), _randn(g, n, kvh, hd)
    if slot == case["batch"]:
        k[:: 97] *= 1.5
    return k, v


def _queries(case, seed):
    q = _randn(_gen(seed, -1), case["batch"] * case["per"], case["heads"], case["head_dim"])
    return q.to(BF16) if case["bf16"] else q


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


def _logits(case, seed):
    g, rows, n = _gen(seed), case["rows"], case["vocab"]
    x = 2.5 * _randn(g, rows, n)
    if case["masked"]:
        # a grammar allows a share of the vocabulary in every other row
        off = torch.rand(rows, n, generator=g, device="cuda") < 0.3
        off[::2] = False
        x = torch.where(off, -math.inf, x)
    tokens = torch.randint(0, n, (rows, case["tokens"]), generator=g, device="cuda", dtype=torch.int32)
    return x.to(BF16) if case["bf16"] else x, tokens


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
    if op == "norm":
        s["x"], s["residual"], s["w"] = _norm_inputs(case, seed)
    elif op == "score":
        s["logits"], s["given"] = _logits(case, seed)
    else:
        pages, slots = _prefix_shape(case)
        kvh, hd, batch, per = case["kv_heads"], case["head_dim"], case["batch"], case["per"]
        own_len, sees = _lens(case, seed)
        s["q"], s["scale"] = _queries(case, seed), 1.0 / math.sqrt(hd)
        s["slots"] = torch.arange(batch, dtype=torch.int32, device="cuda").repeat_interleave(per)
        s["lens"] = torch.from_numpy(sees.astype(np.int32)).cuda()
        filled = [int(n) for n in own_len] + [case["prefix"]]
        if own:
            s["pool"] = s["lib"].kv_pool(be42.KV_BF16 if case["kv"] == "bf16" else be42.KV_INT8, slots, kvh, hd, pages)
            for slot, n in enumerate(filled):
                if n:
                    k, v = _tokens_of(case, seed, slot, n)
                    s["pool"].append(slot, k.reshape(n, kvh * hd), v.reshape(n, kvh * hd), 0)
        else:
            # the same pages as plain tensors: [page][16][kv_heads][head_dim], a table of each slot's pages
            used = [-(-n // PAGE) for n in filled]
            table = np.zeros((slots, pages), np.int64)
            at = 0
            for slot, n in enumerate(used):
                table[slot, :n] = np.arange(at, at + n)
                at += n
            k, v = (torch.zeros(at, PAGE, kvh, hd, device="cuda") for _ in range(2))
            for slot, n in enumerate(filled):
                if n:
                    first = int(table[slot, 0]) * PAGE
                    k.view(-1, kvh, hd)[first:first + n], v.view(-1, kvh, hd)[first:first + n] = \
                        _tokens_of(case, seed, slot, n)
            s["table"] = torch.from_numpy(table).cuda()
            s["k"], s["v"] = ((x.to(BF16), None) if case["kv"] == "bf16" else _page_codes(x) for x in (k, v))
    return s


# ---- the operators -------------------------------------------------------------


def run(s):
    op = s["op"]
    if own:
        lib = s["lib"]
        if op == "norm":
            q, scale, h = lib.norm_quant_rows(s["x"], s["w"], EPS, s["kind"], residual=s["residual"])
            return _norm_outputs(s, q.view(torch.float8_e4m3fn) if s["kind"] == "fp8" else q, scale, h)
        if op == "prefix":
            return lib.prefix_attention(s["pool"], s["q"], s["batch"], s["prefix"], s["scale"], slots=s["slots"],
                                        lens=s["lens"], max_len=s["own_max"])
        return lib.logprobs(s["logits"], s["given"], temp=s["temp"], top_k=s["top_k"], entropy=True)
    return dict(norm=_norm, prefix=_prefix, score=_score)[op](s)


def _norm_outputs(s, codes, scale, h):
    """Codes as the numbers they are (whole ones, or E4M3 values), in units of
    their row's scale; the new residual stream where there is one."""
    return dict(codes=codes, scale=scale, sum=h) if s["res"] else dict(codes=codes, scale=scale)


def _norm(s):
    h = s["x"] if s["residual"] is None else (s["x"].to(F32) + s["residual"].to(F32)).to(s["x"].dtype)
    # in 64 bits: codes lie on borders of the normalised value
    d = h.to(F64)
    r = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + float(np.float32(EPS)))
    y = (d * r * s["w"].to(F64)).to(F32)
    amax = y.abs().amax(1)
    some = amax > 0
    one = torch.ones_like(amax)
    full = torch.full_like(amax, 127.0 if s["kind"] == "int8" else 224.0)
    scale = torch.where(some, amax / full, one)
    if s["kind"] == "int8":
        v = y * torch.where(some, full / amax, one)[:, None]
        a = v.abs()
        t = torch.trunc(a)
        c = (t + (a - t >= 0.5)).clamp(max=127.0)
        return _norm_outputs(s, torch.where(v < 0, -c, c).to(torch.int8), scale, h)
    v = y * torch.where(some, one / scale, one)[:, None]
    a = v.abs().clamp(max=448.0)
    # floor of log2 rounded to fp32, as the codec's exponent is
    e = (torch.floor(torch.log2(a.to(F64)).to(F32)) + 7.0).clamp(0.0, 15.0)
    frac = torch.where(e == 0, a * 64.0, torch.ldexp(a, 7.0 - e) - 1.0)
    m = torch.trunc(frac * 8.0 + 0.5).clamp(max=7.0)
    c = torch.where(e == 0, m / 512.0, torch.ldexp(1.0 + m / 8.0, e - 7.0))
    c = torch.where(a == 0, torch.zeros_like(c), torch.where(v < 0, -c, c))
    return _norm_outputs(s, c.to(torch.float8_e4m3fn), scale, h)


def _prefix(s):
    kvh, hd, n, heads = s["kv_heads"], s["head_dim"], s["q"].shape[0], s["heads"]
    grp = heads // kvh

    def rows(pages, at):
        x, scale = pages
        x = x[at].to(F32)                                # [.., pages][16][kv heads][head_dim]
        return x if scale is None else x * scale[at][..., None]

    used, mine = -(-s["prefix"] // PAGE), -(-s["own_max"] // PAGE)
    shared = s["table"][s["batch"], :used]
    ownt = s["table"][:s["batch"], :mine]
    kp, vp = (rows(s[x], shared).reshape(-1, kvh, hd)[:s["prefix"]].transpose(0, 1) for x in "kv")
    ko, vo = (rows(s[x], ownt).reshape(s["batch"], mine * PAGE, kvh, hd).transpose(1, 2) for x in "kv")
    q = s["q"].to(F32).view(n, kvh, grp, hd)
    sp = torch.matmul(q.transpose(0, 1).reshape(kvh, n * grp, hd), kp.transpose(1, 2))
    sp = sp.view(kvh, n, grp, -1).transpose(0, 1) * s["scale"]
    # queries of one sequence side by side: [batch][kv heads][per * grp][head_dim]
    qo = q.view(s["batch"], s["per"], kvh, grp, hd).transpose(1, 2).reshape(s["batch"], kvh, -1, hd)
    so = torch.matmul(qo, ko.transpose(2, 3)).view(s["batch"], kvh, s["per"], grp, -1).transpose(1, 2)
    so = so.reshape(n, kvh, grp, -1) * s["scale"]
    seen = torch.arange(mine * PAGE, device="cuda") < s["lens"][:, None]
    so = torch.where(seen[:, None, None, :], so, -math.inf)
    top = torch.maximum(sp.amax(-1), so.amax(-1))[..., None]
    ep, eo = torch.exp(sp - top), torch.exp(so - top)
    total = ep.sum(-1) + eo.sum(-1)
    out = torch.matmul(ep.transpose(0, 1).reshape(kvh, n * grp, -1), vp).view(kvh, n, grp, hd).transpose(0, 1)
    eo = eo.view(s["batch"], s["per"], kvh, grp, -1).transpose(1, 2).reshape(s["batch"], kvh, s["per"] * grp, -1)
    oo = torch.matmul(eo, vo).view(s["batch"], kvh, s["per"], grp, hd).transpose(1, 2).reshape(n, kvh, grp, hd)
    return ((out + oo) / total[..., None]).reshape(n, heads, hd).to(s["q"].dtype)


def _score(s):
    x = s["logits"].to(F32)
    z = (x - x.amax(1, keepdim=True)) / s["temp"]
    e = torch.exp(z)
    total = e.sum(1)
    lse = torch.log(total)
    ez = torch.where(e > 0, e * z, torch.zeros_like(z))
    out = dict(logprobs=torch.gather(z, 1, s["given"].long()) - lse[:, None], entropy=lse - ez.sum(1) / total)
    if s["top_k"]:
        # order by value, then by the lower id: one key for both
        bits = (x + 0.0).view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64) << 32
        key |= 0xFFFFFFFF - torch.arange(x.shape[1], device="cuda")
        ids = 0xFFFFFFFF - (torch.topk(key, s["top_k"], dim=1).values & 0xFFFFFFFF)
        out.update(top_ids=ids.to(torch.int32), top_logprobs=torch.gather(z, 1, ids) - lse[:, None])
    return out


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    if case["op"] == "norm":
        n, e = case["rows"] * case["cols"], 2 if case["bf16"] else 4
        return dict(bytes=n * (e * (3 if case["res"] else 1) + 1) + 2 * case["cols"] + 4 * case["rows"], flops=8.0 * n)
    if case["op"] == "prefix":
        kvh, hd, n = case["kv_heads"], case["head_dim"], case["batch"] * case["per"]
        own_len, sees = _lens(case, 0)
        row = 2 * (hd * 2 if case["kv"] == "bf16" else hd + 4)
        held = kvh * row * (case["prefix"] + int(own_len.sum()))
        return dict(bytes=held + 2 * n * case["heads"] * hd * (2 if case["bf16"] else 4),
                    flops=4.0 * case["heads"] * hd * (n * case["prefix"] + int(sees.sum())))
    n = case["rows"] * case["vocab"]
    return dict(bytes=n * (2 if case["bf16"] else 4) + case["rows"] * (8 * case["tokens"] + 4 + 8 * case["top_k"]),
                flops=5.0 * n)


# ---- the definition in 64 bits ---------------------------------------------------


def exact(case, seed):
    return dict(norm=_exact_norm, prefix=_exact_prefix, score=_exact_score)[case["op"]](case, seed)


def _half_up(a):
    """Whole numbers next to a >= 0, halves upwards, from fp32 values in 64 bits."""
    return np.floor(a.astype(np.float64) + 0.5)


def _exact_norm(case, seed):
    x, res, w = (None if t is None else t.cpu() for t in _norm_inputs(case, seed))
    wide = x.double().numpy()
    if res is not None:
        h = torch.from_numpy(wide + res.double().numpy()).to(F32).to(x.dtype)   # both sums are exact in 64 bits
        wide = h.double().numpy()
    rms = np.sqrt(np.einsum("rc,rc->r", wide, wide) / case["cols"] + np.float64(np.float32(EPS)))
    y = (wide / rms[:, None] * w.double().numpy()).astype(np.float32)
    amax = np.abs(y).max(1)
    full = np.float32(127.0 if case["kind"] == "int8" else 224.0)
    with np.errstate(divide="ignore"):
        scale = np.where(amax > 0, amax / full, np.float32(1.0))
        inv = full / amax if case["kind"] == "int8" else np.float32(1.0) / scale
    v = y * np.where(amax > 0, inv, np.float32(1.0))[:, None]
    mag = np.abs(v)
    if case["kind"] == "int8":
        codes = (np.sign(v) * np.minimum(_half_up(mag), 127.0)).astype(np.int8)
        out = dict(codes=torch.from_numpy(codes), scale=torch.from_numpy(scale.astype(np.float64)))
    else:
        # binade of the magnitude; one that fp32's log2 rounds up to belongs to the next
        with np.errstate(divide="ignore"):
            lg = np.log2(mag.astype(np.float64)).astype(np.float32)
        binade = np.clip(np.floor(np.maximum(lg, -100.0)).astype(np.int64), -7, 8)
        step = np.where(binade < -6, 2.0 ** -9, 2.0 ** (binade - 3.0))           # spacing of the codes
        low = np.where(binade < -6, 0.0, 2.0 ** binade.astype(np.float64))
        # the codec adds its half in fp32
        m = np.trunc(((mag.astype(np.float64) - low) / step).astype(np.float32) + np.float32(0.5))
        val = np.sign(v) * (low + step * np.minimum(m, 7.0))
        out = dict(codes=torch.from_numpy(val), scale=torch.from_numpy(scale.astype(np.float64)))
    if case["res"]:
        out["sum"] = torch.from_numpy(wide)
    return out


def _exact_prefix(case, seed):
    kvh, hd, batch, per, heads = (case[k] for k in ("kv_heads", "head_dim", "batch", "per", "heads"))
    grp = heads // kvh
    own_len, sees = _lens(case, seed)

    def held(slot, n):
        """[kv heads][n][head_dim] as the pages hold them."""
        pair = _tokens_of(case, seed, slot, n)
        if case["kv"] == "bf16":
            return [t.to(BF16).to(F64).permute(1, 0, 2) for t in pair]
        coded = [_page_codes(t) for t in pair]
        return [(c.to(F64) * sc.to(F64)[..., None]).permute(1, 0, 2) for c, sc in coded]

    q = _queries(case, seed).to(F64).view(batch, per, kvh, grp, hd)
    kp, vp = held(batch, case["prefix"])
    out = torch.empty(batch, per, kvh, grp, hd, dtype=F64, device="cuda")
    for b in range(batch):
        k, v = kp, vp
        n = int(own_len[b])
        if n:
            more = held(b, n)
            k, v = torch.cat([kp, more[0]], 1), torch.cat([vp, more[1]], 1)
        s = torch.matmul(q[b].permute(1, 0, 2, 3).reshape(kvh, per * grp, hd), k.transpose(1, 2)) / math.sqrt(hd)
        s = s.view(kvh, per, grp, -1)
        for j in range(per):
            s[:, j, :, case["prefix"] + int(sees[b * per + j]):] = -math.inf
        p = torch.softmax(s, -1).reshape(kvh, per * grp, -1)
        out[b] = torch.matmul(p, v).view(kvh, per, grp, hd).permute(1, 0, 2, 3)
    return out.reshape(batch * per, heads, hd)


def _exact_score(case, seed):
    x, tokens = _logits(case, seed)
    out = dict(logprobs=[], entropy=[], top_ids=[], top_logprobs=[])
    for part, given in zip(x.split(256), tokens.split(256)):
        lp = torch.log_softmax(part.to(F64) / case["temp"], 1)
        out["logprobs"].append(lp.gather(1, given.long()))
        out["entropy"].append(-torch.special.xlogy(lp.exp(), lp.exp()).sum(1))
        if case["top_k"]:
            # ties go to the lowest id: a stable order
            ids = torch.sort(part.to(F32), dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
            out["top_ids"].append(ids.to(torch.int32))
            out["top_logprobs"].append(lp.gather(1, ids))
    return {k: torch.cat(v) for k, v in out.items() if v}
