"""Cases of the serving operators around the expert layer: the paged 8-bit
key/value cache (plan, append, attend) and the token log probabilities.

Every case runs one pass through one operator.  ``own = False`` computes it in
plain torch operations in 32 bits; ``own = True`` calls ``exl3_b200``.

Shared terms: a page holds ``page`` consecutive tokens of one request; the
caches are [pages, kv_heads, page, dim] 8-bit codes with one power-of-two
scale per (page, kv head) of K and of V; ``block_table[b, i]`` is the page of
request b's tokens [i * page, (i + 1) * page).
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
MOST_ELEMS = 2048 * 131072          # logits of the largest log-probability case
MOST_CODES = 4 * 131072 * 8 * 128   # key codes of the largest decode case
MOST_PAIRS = 4096 * 16384 * 32      # (query head, key) pairs of the largest prompt case
EXP_LO, EXP_HI = -40, 40            # exponents a scale may take


def listed():
    return [
        # block tables and slot maps
        # one decode step of 64 running requests, a token each
        dict(name="plan_decode_64", op="plan", requests=64, new=1, context=4096, page=16),
        # a large mixed step: 512 requests, up to 61 new tokens each behind their own contexts
        dict(name="plan_ragged_512", op="plan", requests=512, new=61, context=9001, page=64),
        # cache writes
        # the same decode step: a token of each of 64 requests joins its page
        dict(name="append_decode_64", op="append", requests=64, new=1, context=4096, page=16, kv_heads=4, dim=128,
             x="bf16", code="e4m3"),
        # prompts of odd lengths, 8190 tokens in all
        dict(name="append_prompt_8190", op="append", requests=3, new=2730, context=3430, page=64, kv_heads=8, dim=128,
             x="f16", code="int8"),
        # attention over the cache
        # one user, one token, a short odd context: latency
        dict(name="attend_one_1021", op="attend", requests=1, new=1, context=1021, page=16, heads=32, kv_heads=4,
             dim=128, window=0, x="bf16", code="e4m3"),
        # 64 users decoding over ragged contexts up to 8192
        dict(name="attend_decode_64", op="attend", requests=64, new=1, context=8192, page=16, heads=32, kv_heads=4,
             dim=128, window=0, x="bf16", code="e4m3"),
        # few users, long contexts, 3 tokens each (drafted tokens being verified)
        dict(name="attend_long_128k", op="attend", requests=4, new=3, context=131072, page=64, heads=64, kv_heads=8,
             dim=128, window=0, x="f16", code="int8"),
        # odd prompts, narrow heads and a sliding window
        dict(name="attend_window_1777", op="attend", requests=5, new=1777, context=2500, page=32, heads=24, kv_heads=8,
             dim=64, window=1000, x="f16", code="int8"),
        # a prompt's last chunk of 4096 over a cached prefix, 16384 tokens in all
        dict(name="attend_prompt_4096", op="attend", requests=1, new=4096, context=16384, page=64, heads=32, kv_heads=4,
             dim=128, window=0, x="bf16", code="e4m3"),
        # log probabilities
        # one user's next token with its 20 best alternatives
        dict(name="logprobs_one", op="logprobs", rows=1, vocab=100277, x="f32", top=20),
        # 64 users' next tokens with 5 alternatives
        dict(name="logprobs_decode_64", op="logprobs", rows=64, vocab=131072, x="bf16", top=5),
        # scoring a 2048-token text (perplexity): no alternatives
        dict(name="logprobs_score_2048", op="logprobs", rows=2048, vocab=131072, x="bf16", top=0),
    ]


def _size(rng, lo, hi):
    """A size in [lo, hi], even over the logarithm; every other one odd; never the excluded 3 * 1024."""
    while True:
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        if rng.random() < 0.5:
            n |= 1
        n = min(hi, max(lo, n))
        if n != 3 * 1024:
            return n


def draw(rng):
    while True:
        case = _draw(rng)
        if 3 * 1024 not in (*case.values(), case.get("requests", 0) * case.get("new", 0)):
            return case


def _draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "logprobs"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        new = rng.choice([1, _size(rng, 1, 512)])
        return dict(op=op, requests=min(_size(rng, 1, 1024), max(1, 16384 // new)), new=new,
                    context=new + _size(rng, 1, 16384), page=page)
    heads = dict(kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]), x=rng.choice(["bf16", "f16"]),
                 code=rng.choice(["e4m3", "int8"]))
    if op == "append":
        new = rng.choice([1, _size(rng, 1, 4096)])
        return dict(op=op, requests=min(_size(rng, 1, 256), max(1, 8190 // new)), new=new,
                    context=new + _size(rng, 1, 1024), page=page, **heads)
    if op == "attend":
        group = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        while heads["kv_heads"] * group > 64:
            group //= 2
        if rng.random() < 0.55:  # a decode step: one to four tokens a request
            new, context = rng.choice([1, 1, 1, 2, 4]), _size(rng, 16, 65536)
            requests = min(_size(rng, 1, 128), max(1, MOST_CODES // (2 * context * heads["kv_heads"] * heads["dim"])))
        else:                    # prompts, whole or chunked
            new = _size(rng, 16, 4096)
            context = min(16384, new + rng.choice([0, _size(rng, 1, 12000)]))
            pairs = new * context * heads["kv_heads"] * group
            while pairs > MOST_PAIRS // 2:
                new, context = max(1, new // 2), max(1, context // 2)
                pairs = new * context * heads["kv_heads"] * group
            requests = min(_size(rng, 1, 16), max(1, MOST_PAIRS // (2 * pairs)))
        window = rng.choice([0, 0, 0, _size(rng, 64, 4096)])
        return dict(op=op, requests=requests, new=new, context=context, page=page, heads=heads["kv_heads"] * group,
                    window=window, **heads)
    rows = _size(rng, 1, 2048)
    vocab = _size(rng, 1000, min(262144, MOST_ELEMS // rows))
    x = rng.choice(["bf16", "f16", "f32"])
    if x == "f32":
        rows = max(1, rows // 2)
    return dict(op=op, rows=rows, vocab=vocab, x=x, top=rng.choice([0, 1, 5, 20]))


DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def _spread(n, lo, hi):
    """n lengths in [lo, hi], the first of them hi, the others spread evenly but in no order."""
    lo = min(lo, hi)
    return [hi if i == 0 else lo + int((hi - lo) * ((0.6180339887 * i) % 1.0)) for i in range(n)]


def _lengths(case):
    """(tokens already cached, new tokens) of every request; the first has the case's full sizes."""
    new = [max(1, v) for v in _spread(case["requests"], (case["new"] + 1) // 2, case["new"])]
    if case["op"] == "append" and case["new"] > 1:
        new = [case["new"]] * case["requests"]
    total = _spread(case["requests"], max(case["new"], case["context"] // 4), max(case["new"], case["context"]))
    return [t - n for t, n in zip(total, new)], new


def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZE[case["x"]] + case["rows"] * (8 + 12 + 12 * case["top"]), "flops": 5.0 * n}
    lens, new = _lengths(case)
    tokens, P = sum(new), case["page"]
    if case["op"] == "plan":
        taken = sum(-(-(a + n) // P) - -(-a // P) for a, n in zip(lens, new))
        return {"bytes": 8 * len(lens) + 8 * taken + 8 * len(lens) + 12 * tokens, "flops": 10.0 * tokens}
    row = case["kv_heads"] * case["dim"]
    if case["op"] == "append":
        return {"bytes": 2 * tokens * row * 3 + 8 * tokens, "flops": 4.0 * tokens * row}
    W = case["window"] or 1 << 60
    codes = sum(min(a + n, W + n - 1) for a, n in zip(lens, new))
    pairs = 0
    for a, n in zip(lens, new):
        full = max(0, min(n, W - a))  # queries whose window reaches position 0
        pairs += (2 * a + 1 + full) * full // 2 + (n - full) * W
    q = tokens * case["heads"] * case["dim"]
    return {"bytes": 2 * codes * row + 4 * q + 8 * (codes // P + 1) * case["kv_heads"],
            "flops": 4.0 * pairs * case["heads"] * case["dim"]}


# --- inputs -----------------------------------------------------------------

QMAX = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def _exponent(amax, code):
    """The smallest e with amax <= QMAX * 2^e, within [EXP_LO, EXP_HI]."""
    m, e = torch.frexp(amax.float())
    top, bits = (0.875, 9) if code == "e4m3" else (127 / 128, 7)
    e = torch.where(m <= top, e - bits, e - bits + 1)
    return torch.where(amax > 0, e, EXP_LO).clamp(EXP_LO, EXP_HI)


def _encode(x, e, code):
    """x / 2^e rounded to codes (to nearest, ties to even)."""
    y = torch.ldexp(x.float(), -e).clamp(-QMAX[code], QMAX[code])
    return y.to(torch.float8_e4m3fn) if code == "e4m3" else torch.nan_to_num(torch.round(y), 0.0).to(torch.int8)


def _cache(gen, pages, case):
    """A filled cache: normal values, a few loud channels in K."""
    out = []
    for loud in (True, False):
        codes = torch.empty(pages, case["kv_heads"], case["page"], case["dim"], dtype=CODE[case["code"]], device=DEV)
        scale = torch.empty(pages, case["kv_heads"], device=DEV)
        gain = torch.ones(case["kv_heads"], 1, case["dim"], device=DEV)
        if loud:
            gain = torch.exp(0.5 * torch.randn(gain.shape, generator=gen, device=DEV))
        step = max(1, (1 << 26) // (case["kv_heads"] * case["page"] * case["dim"]))
        for p in range(0, pages, step):
            x = torch.randn(codes[p:p + step].shape, generator=gen, device=DEV) * gain
            e = _exponent(x.abs().amax((2, 3)), case["code"])
            codes[p:p + step] = _encode(x, e[:, :, None, None], case["code"])
            scale[p:p + step] = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
        out.append((codes, scale))
    return out


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "logprobs":
        x = torch.empty(case["rows"], case["vocab"], dtype=DTYPES[case["x"]], device=DEV)
        for r in range(0, case["rows"], 256):
            x[r:r + 256] = torch.randn(x[r:r + 256].shape, generator=gen, device=DEV) * 2.5
        # most asked tokens are likely ones, some are not
        best = x.argmax(1)
        other = torch.randint(0, case["vocab"], (case["rows"],), generator=gen, device=DEV)
        loud = torch.rand(case["rows"], generator=gen, device=DEV) < 0.7
        return s | {"logits": x, "tokens": torch.where(loud, best, other)}
    lens, new = _lengths(case)
    P, B = case["page"], case["requests"]
    have = [-(-a // P) for a in lens]
    held = [-(-(a + n) // P) for a, n in zip(lens, new)]
    width = max(held) + 2
    before = case["op"] == "plan"  # the plan itself hands out the new pages
    owned = have if before else held
    spare = sum(held) - sum(have) if before else 0
    pages = sum(owned) + spare + 5
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    owned_t = torch.tensor(owned, device=DEV)
    first = torch.cumsum(owned_t, 0) - owned_t
    col = torch.arange(width, device=DEV)
    table = torch.where(col < owned_t[:, None], order[(first[:, None] + col).clamp(max=pages - 1)], 0).to(torch.int32)
    s |= {"lens": _i32(lens), "new": _i32(new), "table": table, "tokens": sum(new), "most": max(new)}
    if case["op"] == "plan":
        return s | {"free": order[sum(owned):].contiguous(), "cursor": torch.zeros(1, dtype=torch.int32, device=DEV)}
    (k, ks), (v, vs) = _cache(gen, pages, case)
    s |= {"k": k, "v": v, "ks": ks, "vs": vs}
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), torch.cumsum(s["new"], 0)])
    s["cu"], s["kv_lens"] = cu.to(torch.int32), s["lens"] + s["new"]
    kind = DTYPES[case["x"]]
    if case["op"] == "append":
        t = torch.arange(sum(new), device=DEV)
        b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
        pos = s["lens"][b] + t - cu[b]
        s["slots"] = table[b, pos // P].long() * P + pos % P
        # K and V as they leave a fused projection: slices of one row per token
        heads = case["kv_heads"]
        rows = torch.randn(sum(new), 3 * heads, case["dim"], generator=gen, device=DEV).to(kind)
        return s | {"knew": rows[:, heads:2 * heads], "vnew": rows[:, 2 * heads:]}
    q = torch.randn(sum(new), case["heads"], case["dim"], generator=gen, device=DEV)
    return s | {"q": (q * 1.2).to(kind)}


# --- plain forms ------------------------------------------------------------

def _plan(s):
    P, lens, new, table = s["case"]["page"], s["lens"].long(), s["new"].long(), s["table"]
    total = lens + new
    have = (lens + P - 1) // P
    need = (total + P - 1) // P - have
    start = s["cursor"].long() + torch.cumsum(need, 0) - need
    col = torch.arange(table.shape[1], device=DEV)
    fresh = (col >= have[:, None]) & (col < (have + need)[:, None])
    at = (start[:, None] + col - have[:, None]).clamp(0, s["free"].numel() - 1)
    table = torch.where(fresh, s["free"][at], table)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), torch.cumsum(new, 0)])
    t = torch.arange(s["tokens"], device=DEV)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    pos = lens[b] + t - cu[b]
    slots = table[b, pos // P].long() * P + pos % P
    return {"block_table": table, "kv_lens": total.int(), "cu_tokens": cu.int(), "positions": pos.int(),
            "slots": slots, "cursor": (s["cursor"] + need.sum()).int()}


def _append(s):
    case = s["case"]
    P, code = case["page"], case["code"]
    page, off = s["slots"] // P, s["slots"] % P
    pages, run = torch.unique_consecutive(page, return_inverse=True)  # a page's tokens follow one another
    begin = torch.full_like(pages, P).scatter_reduce_(0, run, off, "amin")
    kept = (torch.arange(P, device=DEV) < begin[:, None])[:, None, :, None]
    for x, cache, scale in ((s["knew"], s["k"], s["ks"]), (s["vnew"], s["v"], s["vs"])):
        x = x.float()
        amax = torch.zeros(pages.numel(), x.shape[1], device=DEV)
        amax.scatter_reduce_(0, run[:, None].expand(-1, x.shape[1]), x.abs().amax(2), "amax")
        e = _exponent(amax, code)
        old = torch.frexp(scale[pages])[1] - 1
        e = torch.where(begin[:, None] > 0, torch.maximum(e, old), e)
        tile = cache[pages].float()
        again = _encode(tile, (e - old)[:, :, None, None], code)
        both = torch.where(kept, again.float(), tile)
        both[run, :, off] = _encode(x, e[run][:, :, None], code).float()
        cache[pages] = both.to(cache.dtype)
        scale[pages] = torch.ldexp(torch.ones_like(amax), e)
    return {"k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}


def _attend(s):
    case = s["case"]
    P, B, Hk, D = case["page"], case["requests"], case["kv_heads"], case["dim"]
    G, Q = case["heads"] // Hk, s["most"]
    table, kv_lens, cu, new = s["table"].long(), s["kv_lens"].long(), s["cu"].long(), s["new"].long()
    L = table.shape[1] * P
    k = (s["k"].float() * s["ks"][:, :, None, None])[table].permute(0, 2, 1, 3, 4).reshape(B, Hk, L, D)
    v = (s["v"].float() * s["vs"][:, :, None, None])[table].permute(0, 2, 1, 3, 4).reshape(B, Hk, L, D)
    i = torch.arange(Q, device=DEV)
    row = (cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    live = i < new[:, None]
    q = s["q"].float()[row].view(B, Q, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Q, D)
    p = torch.matmul(q, k.transpose(2, 3)).view(B, Hk, G, Q, L)
    p *= 1.0 / math.sqrt(D)
    at, pos = torch.arange(L, device=DEV), (s["lens"].long()[:, None] + i)[:, :, None]
    hidden = (at > pos) | (at >= kv_lens[:, None, None])
    if case["window"]:
        hidden |= at <= pos - case["window"]
    p.masked_fill_(hidden[:, None, None], -math.inf)
    m = p.amax(-1, keepdim=True).clamp(min=-3e38)
    p.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, Hk, G * Q, L), v).view(B, Hk, G, Q, D) / total.clamp(min=1e-38)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, Q, Hk * G, D)
    return out[live].to(s["q"].dtype)


def _logprobs(s):
    case = s["case"]
    x = s["logits"].float()
    xt = x.gather(1, s["tokens"][:, None])
    at = torch.arange(case["vocab"], device=DEV)
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1)
    lse = torch.log(total)
    out = {"logprob": (xt - m)[:, 0] - lse, "entropy": lse - (e * (x - m)).sum(1) / total,
           "rank": (1 + (x > xt).sum(1) + ((x == xt) & (at < s["tokens"][:, None])).sum(1)).int()}
    if case["top"]:
        # one whole-number key per entry, so that equal logits go by index
        bits = x.view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) + ((1 << 20) - 1 - at)
        ids = (1 << 20) - 1 - (torch.topk(key, case["top"], 1).values & ((1 << 20) - 1))
        out |= {"top_ids": ids.int(), "top_logprobs": x.gather(1, ids) - m - lse[:, None]}
    return out


PLAIN = {"plan": _plan, "append": _append, "attend": _attend, "logprobs": _logprobs}


# --- the framework's operators ------------------------------------------------

_modules = []


def _framework():
    if not _modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "vllm-exl3_b200"))
        from exl3_b200 import kv_cache, logprobs
        _modules.extend((kv_cache, logprobs))
    return _modules


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return PLAIN[op](s)
    kv, lp = _framework()
    if op == "plan":
        p = kv.kv_plan(s["lens"], s["new"], s["table"], s["free"], s["cursor"], page_size=case["page"],
                       n_tokens=s["tokens"])
        return {"block_table": s["table"], "kv_lens": p.kv_lens, "cu_tokens": p.cu_tokens, "positions": p.positions,
                "slots": p.slots, "cursor": p.cursor}
    if op == "append":
        kv.kv_append(s["knew"], s["vnew"], s["slots"], s["k"], s["v"], s["ks"], s["vs"])
        return {"k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}
    if op == "attend":
        return kv.kv_attend(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["kv_lens"], cu_tokens=s["cu"],
                            max_new=s["most"], window=case["window"])
    r = lp.token_logprobs(s["logits"], s["tokens"], top=case["top"])
    out = {"logprob": r.logprob, "entropy": r.entropy, "rank": r.rank}
    if case["top"]:
        out |= {"top_ids": r.top_ids, "top_logprobs": r.top_logprobs}
    return out


# --- 64-bit values ------------------------------------------------------------

def _pow2_for(amax, code):
    """The scale of a page from its largest magnitude, by trying exponents upwards."""
    e = np.full(amax.shape, EXP_LO)
    for _ in range(EXP_HI - EXP_LO):
        e += amax > QMAX[code] * np.exp2(e)
    return e


def _round64(y, code):
    if code == "int8":
        return np.clip(np.rint(y), -127, 127)
    mag = np.abs(y)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(mag, 2.0 ** -20))), -6) - 3)  # spacing of e4m3 at |y|
    return np.sign(y) * np.minimum(np.rint(mag / step) * step, 448)


def _exact_append(s):
    case, out = s["case"], {}
    P, slots = case["page"], s["slots"].cpu().numpy()
    edges = np.flatnonzero(np.diff(slots // P)) + 1
    for name, new, cache, scale in (("k", s["knew"], s["k"], s["ks"]), ("v", s["vnew"], s["v"], s["vs"])):
        new, codes = new.double().cpu().numpy(), cache.double().cpu().numpy()
        scale = scale.double().cpu().numpy()
        for part in np.split(np.arange(len(slots)), edges):
            page, first = slots[part[0]] // P, slots[part[0]] % P
            rows = new[part].transpose(1, 0, 2)  # [heads, tokens, dim]
            e = _pow2_for(np.abs(rows).max((1, 2)), case["code"])
            if first:
                was = np.log2(scale[page]).astype(int)
                e = np.maximum(e, was)
                codes[page, :, :first] = _round64(codes[page, :, :first] * np.exp2(was - e)[:, None, None],
                                                  case["code"])
            codes[page, :, first:first + len(part)] = _round64(rows * np.exp2(-e)[:, None, None], case["code"])
            scale[page] = np.exp2(e)
        out[name], out[name + "_scale"] = codes, scale
    return out


def _exact_attend(s):
    case = s["case"]
    D, G, P = case["dim"], case["heads"] // case["kv_heads"], case["page"]
    lens, news, cu = s["lens"].tolist(), s["new"].tolist(), s["cu"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b in range(case["requests"]):
        total = lens[b] + news[b]
        page = s["table"][b, :-(-total // P)].long()
        rows = slice(cu[b], cu[b] + news[b])
        last = torch.arange(lens[b], total, device=DEV)[:, None]
        at = torch.arange(total, device=DEV)
        ok = (at <= last) & (at > last - case["window"]) if case["window"] else at <= last
        for h in range(case["kv_heads"]):
            k, v = ((c[page, h].double() * f[page, h].double()[:, None, None]).reshape(-1, D)[:total]
                    for c, f in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            for g in range(h * G, (h + 1) * G):
                score = (s["q"][rows, g].double() @ k.T / D ** 0.5).masked_fill(~ok, float("-inf"))
                out[rows, g] = torch.softmax(score, 1) @ v
    return out


def _exact_logprobs(s):
    case = s["case"]
    top, parts = case["top"], []
    for r in range(0, case["rows"], 64):
        x = s["logits"][r:r + 64].double()
        logp = torch.log_softmax(x, 1)
        entropy = -(logp.exp() * logp).sum(1)
        best = [torch.sort(logp, dim=1, descending=True, stable=True).values[:, :top]] if top else []
        parts.append([logp.gather(1, s["tokens"][r:r + 64, None])[:, 0], entropy] + best)
    got = [torch.cat(c) for c in zip(*parts)]
    out = {"logprob": got[0], "entropy": got[1], "rank": None}
    if top:
        out |= {"top_ids": None, "top_logprobs": got[2]}
    return out


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["op"]](s)
