"""The serving operators around a paged key / value cache, and rotary positions: what they are measured on.

Four operators, used one after the other in a layer of a model that serves: q and k get rotary positions, k and v of the new
tokens are written into the pages of a cache (as they are, or in 8 bits with a scale for each token and head), the new tokens
attend to all that their sequences hold there, and a cache is read back into contiguous rows (to hand a sequence on, or to
train on it).  Rotary positions have a backward pass too.

``run`` computes them in plain torch (32 bits, rounded once) unless ``own`` is set; then it makes the framework's calls.
Every case is a dict of plain values, ``draw`` gives further cases of the same ranges, ``exact`` the results in 64 bits."""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


# ---------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------

def _rotary(kind, dtype, B, S, H, Hkv, D, rotary_dim, interleaved=False, scaling="none", factor=1.0, far=0):
    """B sequences of S tokens, or with B = 0 one packed run of S tokens; Hkv = 0: no k.  ``far``: largest first position."""
    return {"kind": kind, "dtype": dtype, "B": B, "S": S, "H": H, "Hkv": Hkv, "D": D, "rotary_dim": rotary_dim, "interleaved": interleaved,
            "scaling": scaling, "factor": factor, "far": far}


def _cache(kind, dtype, cache, B, Hkv, D, page, context, new, packed, ragged, **more):
    """B sequences of up to ``context`` tokens, the last ``new`` (at most, where packed) of each of them new."""
    return {"kind": kind, "dtype": dtype, "cache": cache, "B": B, "Hkv": Hkv, "D": D, "page": page, "context": context, "new": new,
            "packed": packed, "ragged": ragged, **more}


def listed():
    return [
        # Training step of a causal language model with grouped heads: q and k rotated, and their gradients rotated back.
        dict(_rotary("rotary_step", "bf16", 4, 4096, 32, 8, 128, 128), name="rotary_step"),
        # A few tokens far into a long context: the positional 64 columns of 192-wide queries, interleaved, stretched frequencies.
        dict(_rotary("rotary", "fp16", 0, 77, 16, 1, 192, 64, True, "yarn", 16.0, 900000), name="rotary_part_far"),
        # The keys and values of prompts, rotated on their way into 16-bit pages.
        dict(_cache("append", "bf16", "16", 4, 8, 128, 64, 2048, 2048, False, False, rotary=True), name="append_prompts"),
        # Ragged prompts of a batch, one after the other, quantised on their way into the cache.
        dict(_cache("append", "fp16", "e4m3", 6, 8, 128, 32, 4096, 2100, True, True, rotary=True), name="append_ragged_8bit"),
        # One token of every sequence of a batch that generates, quantised: latency of a launch.
        dict(_cache("append", "bf16", "e4m3", 64, 8, 128, 16, 1000, 1, False, True, rotary=False), name="append_token_8bit"),
        # Sequences leave an 8-bit cache for another program: contiguous rows in 16 bits.
        dict(_cache("read", "bf16", "e4m3", 8, 8, 128, 64, 8192, 1, False, True), name="read_8bit"),
        # The same of a small 16-bit cache with narrow heads and odd lengths.
        dict(_cache("read", "fp16", "16", 3, 4, 64, 16, 999, 1, False, True), name="read_small"),
        # One token of one short sequence: all latency.
        dict(_cache("attend", "fp16", "16", 1, 4, 64, 16, 333, 1, False, False, H=16, window=0), name="attend_one"),
        # Batched generation with grouped heads over sequences of many lengths: the bytes of the cache.
        dict(_cache("attend", "bf16", "16", 64, 8, 128, 64, 8192, 1, False, True, H=32, window=0), name="attend_tokens"),
        # The same from an 8-bit cache, fewer and longer sequences.
        dict(_cache("attend", "bf16", "e4m3", 16, 8, 128, 64, 32768, 1, False, True, H=32, window=0), name="attend_tokens_8bit"),
        # A chunk of a long prompt against what the sequence already has: compute-bound.
        dict(_cache("attend", "bf16", "16", 2, 8, 128, 64, 16384, 1024, False, False, H=32, window=0), name="attend_chunk"),
        # A step of a server: prompts' chunks and single tokens in one packed batch, sliding window, small pages, narrow heads.
        dict(_cache("attend", "fp16", "16", 24, 4, 64, 16, 3000, 700, True, True, H=16, window=1024), name="attend_mixed_window"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["rotary", "rotary_step", "append", "append", "read", "attend", "attend", "attend", "attend"])
    if kind.startswith("rotary"):
        D, part = rng.choice([(64, 64), (128, 128), (128, 128), (128, 32), (192, 64), (80, 32), (256, 64)])
        H = rng.choice([8, 16, 32])
        scaling, factor = rng.choice([("none", 1.0), ("none", 1.0), ("linear", 4.0), ("ntk", 8.0), ("yarn", 16.0)])
        return _rotary(kind, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice([0, 1, 2, 4]), _log_int(rng, 1, 4096), H, rng.choice([0, 1, H // 4, H]),
                       D, part, rng.choice([False, False, True]), scaling, factor, rng.choice([0, 5000, 900000]))
    dtype, cache = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["16", "16", "e4m3"])
    Hkv, D, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 64, 128, 256])
    B, context, ragged, packed = _log_int(rng, 1, 64), _log_int(rng, 16, 32768), rng.choice([True, True, False]), rng.choice([True, False])
    new = _log_int(rng, 1, min(context, 2048)) if kind == "append" or rng.random() < 0.5 else 1
    if kind == "read":
        return _cache(kind, dtype, cache, B, Hkv, D, page, context, 1, False, ragged)
    if kind == "append":
        return _cache(kind, dtype, cache, B, Hkv, D, page, context, new, packed, ragged, rotary=rng.choice([True, False]))
    window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
    return _cache(kind, dtype, cache, B, Hkv, D, page, context, new, packed, ragged, H=Hkv * rng.choice([1, 3, 4, 8, 16]), window=window)


def draw(rng):
    top = [work(c) for c in listed()]
    most_flops, most_bytes = max(w["flops"] for w in top), max(w["bytes"] for w in top)
    while True:
        case = _draw_once(rng)
        w = work(case)
        pairs = case["B"] * case["context"] * case["H"] * case["new"] if case["kind"] == "attend" else 0
        pool = 2 * case["B"] * case["context"] * case["Hkv"] * case["D"] if "context" in case else 0
        # the plain form holds all pairs of a padded batch, and a cache of 32-bit values
        if w["flops"] <= most_flops and w["bytes"] <= most_bytes and pairs <= 1.1e9 and pool <= 1.1e9:
            return case


def _lengths(case):
    """(new tokens, tokens with them) of every sequence; of the case alone, so that the work of a pass is known."""
    rng = random.Random("%(B)d %(context)d %(new)d %(packed)s" % case)
    news, lens = [], []
    for b in range(case["B"]):
        n = case["new"]
        if case["packed"] and b > 0:   # mixed batches: about half of the sequences have one new token
            n = 1 if rng.random() < 0.5 else _log_int(rng, 1, n)
        least = max(n, case["context"] // 4)
        lens.append(case["context"] if b == 0 or not case["ragged"] else rng.randint(least, case["context"]))
        news.append(n)
    return news, lens


# ---------------------------------------------------------------------------------------------------------------
# what a user's program has in hand before the call
# ---------------------------------------------------------------------------------------------------------------

def _frequencies(dim, base=10000.0, scaling="none", factor=1.0, original=4096):
    """(angle of one position for each pair of columns, magnitude) as float64."""
    f = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "ntk":
        wider = base * factor ** (dim / (dim - 2.0))
        f = [wider ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == "yarn":   # columns that turn often keep their frequency, those that turn less than once are stretched
        at = [dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
        ramp = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(dim // 2)]
        f = [x / factor * r + x * (1.0 - r) for x, r in zip(f, ramp)]
        return f, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_rotary(c, gen, dtype):
    B, S, lead = c["B"], c["S"], ((c["B"], c["S"]) if c["B"] else (c["S"],))
    first = torch.randint(0, c["far"] + 1, (max(B, 1), 1), generator=gen, device="cuda")
    pos = first + torch.arange(S, device="cuda")
    st = {"q": _randn(gen, *lead, c["H"], c["D"], dtype=dtype), "positions": pos if B else pos[0]}
    st["k"] = _randn(gen, *lead, c["Hkv"], c["D"], dtype=dtype) if c["Hkv"] else None
    if c["kind"] == "rotary_step":
        st["grads"] = [_randn(gen, *t.shape, dtype=dtype) for t in (st["q"], st["k"]) if t is not None]
        if own:
            for t in (st["q"], st["k"]):
                if t is not None:
                    t.requires_grad_()
    f, st["magnitude"] = _frequencies(c["rotary_dim"], scaling=c["scaling"], factor=c["factor"])
    st["freq"] = torch.tensor(f, dtype=torch.float64, device="cuda")
    if own:
        from metaattention_b200 import RotaryEmbedding
        st["rope"] = RotaryEmbedding(c["rotary_dim"], interleaved=c["interleaved"], scaling=None if c["scaling"] == "none" else c["scaling"], factor=c["factor"])
    return st


def _pool(gen, pages, page, Hkv, D, dtype, cache):
    """Keys or values of a pool [pages, page, heads, D], kept page by page and head by head; N(0, 1), and in 8 bits with their scales."""
    if cache == "16":
        return _randn(gen, pages, Hkv, page, D, dtype=dtype).transpose(1, 2), None
    codes = (_randn(gen, pages, Hkv, page, D, dtype=torch.float16) * 100).clamp(-448, 448).to(E4M3).transpose(1, 2)
    scale = torch.randint(118, 122, (pages, Hkv, page), generator=gen, device="cuda", dtype=torch.uint8).view(E8M0).transpose(1, 2)
    return codes, scale


def _prepare_cache(c, gen, dtype):
    news, lens = _lengths(c)
    B, Hkv, D, page = c["B"], c["Hkv"], c["D"], c["page"]
    per_seq = -(-c["context"] // page)
    pages = B * per_seq + 3
    st = {"news": news, "lens": lens, "most": max(lens)}
    st["pool_k"], st["k_scale"] = _pool(gen, pages, page, Hkv, D, dtype, c["cache"])
    st["pool_v"], st["v_scale"] = _pool(gen, pages, page, Hkv, D, dtype, c["cache"])
    st["table"] = torch.randperm(pages, generator=gen, device="cuda")[:B * per_seq].view(B, per_seq).to(torch.int32)
    st["cache_seqlens"] = _int32(lens)
    st["cu_seqlens"] = _int32([sum(news[:i]) for i in range(B + 1)]) if c["packed"] else None
    lead = (sum(news),) if c["packed"] else (B, c["new"])
    if c["kind"] == "append":
        st["k"], st["v"] = _randn(gen, *lead, Hkv, D, dtype=dtype), _randn(gen, *lead, Hkv, D, dtype=dtype)
        st["freq"] = torch.tensor(_frequencies(D)[0], dtype=torch.float64, device="cuda")
    if c["kind"] == "attend":
        st["q"] = _randn(gen, *lead, c["H"], D, dtype=dtype)
    if own:
        from metaattention_b200 import PagedKVCache, RotaryEmbedding
        st["handle"] = PagedKVCache(st["pool_k"], st["pool_v"], st["k_scale"], st["v_scale"])
        st["rope"] = RotaryEmbedding(D) if c.get("rotary") else None
    return st


def prepare(case, seed):
    make = _prepare_rotary if case["kind"].startswith("rotary") else _prepare_cache
    return {**make(case, _gen(seed), DTYPES[case["dtype"]]), "case": case}


# ---------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------

def _turned(x, cos, sin, interleaved):
    """The first columns of x [..., heads, D] as pairs turned by angles [..., pairs]; the result is not rounded."""
    n = cos.shape[-1]
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    wide = x.to(cos.dtype)
    a, b = (wide[..., 0:2 * n:2], wide[..., 1:2 * n:2]) if interleaved else (wide[..., :n], wide[..., n:2 * n])
    left, right = a * cos - b * sin, b * cos + a * sin
    pairs = torch.stack((left, right), -1).flatten(-2) if interleaved else torch.cat((left, right), -1)
    return torch.cat((pairs, wide[..., 2 * n:]), -1)


def _angles(positions, freq, magnitude, dtype=torch.float32):
    angle = positions.double().unsqueeze(-1) * freq
    return (angle.cos() * magnitude).to(dtype), (angle.sin() * magnitude).to(dtype)


def _run_rotary(st):
    c = st["case"]
    both = [t for t in (st["q"], st["k"]) if t is not None]
    cos, sin = _angles(st["positions"], st["freq"], st["magnitude"])
    out = [_turned(t, cos, sin, c["interleaved"]).to(t.dtype) for t in both]
    if c["kind"] == "rotary_step":   # the transposed rotation of each pair is the rotation by the opposite angle
        out += [_turned(g, cos, -sin, c["interleaved"]).to(g.dtype) for g in st["grads"]]
    return out


def _new_tokens(st):
    """(sequence, position) of every new token, in the order of the rows of k, v and q."""
    c, lens = st["case"], st["cache_seqlens"].long()
    if not c["packed"]:
        seq = torch.arange(c["B"], device="cuda").repeat_interleave(c["new"])
        return seq, lens[seq] - c["new"] + torch.arange(c["new"], device="cuda").repeat(c["B"])
    cu = st["cu_seqlens"].long()
    row = torch.arange(sum(st["news"]), device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    return seq, lens[seq] + row - cu[seq + 1]


def _quantised(x):
    """(codes, scales) of rows x [..., D] in 32 bits: the scale is the least power of two with |x| <= 448 times it."""
    mantissa, exponent = torch.frexp(x.abs().amax(-1))
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    e = torch.where(mantissa == 0, -127, e).clamp(-127, 127)
    return torch.ldexp(x, -e.unsqueeze(-1)).to(E4M3), (e + 127).to(torch.uint8)


def _run_append(st):
    c = st["case"]
    seq, pos = _new_tokens(st)
    page, row = st["table"][seq, pos // c["page"]].long(), pos % c["page"]
    k, v = (st[n].flatten(0, -3).float() for n in ("k", "v"))
    if c["rotary"]:
        k = _turned(k, *_angles(pos, st["freq"], 1.0), False)
    for x, pool, scale in ((k, st["pool_k"], st["k_scale"]), (v, st["pool_v"], st["v_scale"])):
        if scale is None:
            pool[page, row] = x.to(pool.dtype)
        else:
            codes, e = _quantised(x)
            pool.view(torch.uint8)[page, row] = codes.view(torch.uint8)
            scale.view(torch.uint8)[page, row] = e
    return _pools(st)


def _pools(st):
    return [st["pool_k"], st["pool_v"]] + ([st["k_scale"], st["v_scale"]] if st["k_scale"] is not None else [])


def _gathered(st, name, dtype=torch.float32):
    """Keys or values of all sequences [B, tokens of whole pages, heads, D]."""
    def by_table(pool):
        return pool[st["table"].long()].flatten(1, 2)
    x = by_table(st["pool_" + name].view(torch.uint8)).view(E4M3) if st["k_scale"] is not None else by_table(st["pool_" + name])
    if st["k_scale"] is None:
        return x.to(dtype)
    e = by_table(st[name + "_scale"].view(torch.uint8)).to(torch.int32) - 127
    return torch.ldexp(x.to(dtype), e.unsqueeze(-1))


def _run_read(st):
    c, keep = st["case"], torch.arange(st["most"], device="cuda") < st["cache_seqlens"].unsqueeze(1)
    return [torch.where(keep[:, :, None, None], _gathered(st, n)[:, :st["most"]], 0.0).to(DTYPES[c["dtype"]]) for n in ("k", "v")]


def _run_attend(st):
    """Softmax over the kept keys of each row, all sequences padded to the longest; rows that keep none give 0 and -inf."""
    c, seq_pos = st["case"], _new_tokens(st)
    B, H, Hkv, D, n = c["B"], c["H"], c["Hkv"], c["D"], max(st["news"])
    q, slot = st["q"], None
    pos = st["cache_seqlens"].long().unsqueeze(1) - n + torch.arange(n, device="cuda")
    if c["packed"]:   # the rows of a sequence go to the end of its padded ones
        slot = seq_pos[0] * n + seq_pos[1] - pos[seq_pos[0], 0]
        q = q.new_zeros(B * n, H, D).index_copy_(0, slot, q).view(B, n, H, D)
    k, v = (_gathered(st, name).transpose(1, 2) for name in ("k", "v"))
    wide = q.float().view(B, n, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    s = torch.matmul(wide, k.transpose(2, 3)).mul_(D ** -0.5).view(B, Hkv, H // Hkv, n, -1)
    at = torch.arange(s.shape[-1], device="cuda")
    keep = at <= pos.unsqueeze(2)
    if c["window"]:
        keep &= at > pos.unsqueeze(2) - c["window"]
    s.masked_fill_(~keep[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    total = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_().sum(-1, keepdim=True)
    past = at >= st["cache_seqlens"].unsqueeze(1)   # what lies behind a sequence's end is no number to multiply by zero
    o = torch.matmul(s.view(B, Hkv, -1, s.shape[-1]), v.masked_fill_(past[:, None, :, None], 0.0)).view(B, Hkv, H // Hkv, n, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, n, H, D)
    lse = (total.log() + top).view(B, H, n)
    if c["packed"]:
        return [o.reshape(B * n, H, D)[slot].to(q.dtype), lse.transpose(0, 1).reshape(H, B * n)[:, slot]]
    return [o.to(q.dtype), lse]


def _run_own(st):
    c = st["case"]
    if c["kind"].startswith("rotary"):
        out = st["rope"](st["q"], st["k"], positions=st["positions"])
        out = list(out) if st["k"] is not None else [out]
        if c["kind"] == "rotary":
            return out
        leaves = [t for t in (st["q"], st["k"]) if t is not None]
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, st["grads"]))
    cache = st["handle"]
    if c["kind"] == "append":
        cache.append(st["k"], st["v"], st["table"], st["cache_seqlens"], cu_seqlens=st["cu_seqlens"], rotary=st["rope"])
        return _pools(st)
    if c["kind"] == "read":
        return list(cache.read(st["table"], st["cache_seqlens"], st["most"], dtype=DTYPES[c["dtype"]]))
    o, lse = cache.attention(st["q"], st["table"], st["cache_seqlens"], cu_seqlens=st["cu_seqlens"], window=c["window"] or None, return_lse=True)
    return [o, lse]


def run(st):
    if own:
        return _run_own(st)
    return {"rotary": _run_rotary, "rotary_step": _run_rotary, "append": _run_append, "read": _run_read, "attend": _run_attend}[st["case"]["kind"]](st)


# ---------------------------------------------------------------------------------------------------------------
# the same in 64 bits, token by token from the definitions
# ---------------------------------------------------------------------------------------------------------------

def _exact_rotation(x, positions, freq, magnitude, interleaved, sign=1.0):
    """x [..., heads, D] with the pair (a, b) of columns as the complex number a + ib, times magnitude * exp(i * angle)."""
    x, n = x.double().clone(), freq.numel()
    columns = torch.arange(n, device=x.device)
    first, second = (2 * columns, 2 * columns + 1) if interleaved else (columns, columns + n)
    turn = torch.polar(torch.full_like(freq, magnitude).expand(*positions.shape, n).contiguous(), sign * positions.double().unsqueeze(-1) * freq)
    z = torch.complex(x[..., first], x[..., second]) * turn.unsqueeze(-2)
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _sequence(st, b, name):
    """Keys or values of sequence b [tokens, heads, D] as the cache holds them."""
    page = st["case"]["page"]
    t = torch.arange(st["lens"][b], device="cuda")
    at = st["table"][b].long()[t // page], t % page
    if st["k_scale"] is None:
        return st["pool_" + name][at].double()
    return st["pool_" + name].view(torch.uint8)[at].view(E4M3).double() * torch.exp2(st[name + "_scale"].view(torch.uint8)[at].double() - 127.0).unsqueeze(-1)


def _exact_append(st):
    c = st["case"]
    pools = [t.double() for t in _pools(st)]
    first = 0
    for b, (n, length) in enumerate(zip(st["news"], st["lens"])):
        pos = torch.arange(length - n, length, device="cuda")
        at = st["table"][b].long()[pos // c["page"]], pos % c["page"]
        for i, name in enumerate(("k", "v")):
            x = (st[name][first:first + n] if c["packed"] else st[name][b]).double()
            if name == "k" and c["rotary"]:
                x = _exact_rotation(x, pos, st["freq"], 1.0, False)
            if c["cache"] == "e4m3":
                top = x.abs().amax(-1)
                e = torch.where(top > 0, torch.ceil(torch.log2(top / 448.0)), -127.0).clamp(-127, 127)
                pools[2 + i][at] = torch.exp2(e)
                x = x * torch.exp2(-e).unsqueeze(-1)
            pools[i][at] = x
        first += n
    return pools


def _exact_attend(st):
    c = st["case"]
    G, D, first, outs, sums = c["H"] // c["Hkv"], c["D"], 0, [], []
    for b, (n, length) in enumerate(zip(st["news"], st["lens"])):
        q = (st["q"][first:first + n] if c["packed"] else st["q"][b]).double()
        k, v = _sequence(st, b, "k"), _sequence(st, b, "v")
        ahead = torch.arange(length - n, length, device="cuda").unsqueeze(1) - torch.arange(length, device="cuda")
        keep = (ahead >= 0) & (ahead < (c["window"] or length + 1))
        o, lse = torch.empty_like(q), q.new_empty(c["H"], n)
        for h in range(c["H"]):
            s = (q[:, h] @ k[:, h // G].T * D ** -0.5).masked_fill(~keep, -math.inf)
            lse[h] = torch.logsumexp(s, 1)
            o[:, h] = torch.exp(s - lse[h].unsqueeze(1)) @ v[:, h // G]
        outs.append(o)
        sums.append(lse)
        first += n
    return [torch.cat(outs), torch.cat(sums, 1)] if c["packed"] else [torch.stack(outs), torch.stack(sums)]


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "append":
        return _exact_append(st)
    if kind == "attend":
        return _exact_attend(st)
    if kind == "read":
        out = [torch.zeros(case["B"], st["most"], case["Hkv"], case["D"], dtype=torch.float64, device="cuda") for _ in range(2)]
        for b, length in enumerate(st["lens"]):
            for t, name in zip(out, ("k", "v")):
                t[b, :length] = _sequence(st, b, name)
        return out
    def turned(t, sign):
        return _exact_rotation(t, st["positions"], st["freq"], st["magnitude"], case["interleaved"], sign)
    return [turned(t, 1.0) for t in (st["q"], st["k"]) if t is not None] + [turned(g, -1.0) for g in st.get("grads", ())]


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"].startswith("rotary"):
        tokens = max(c["B"], 1) * c["S"]
        values, passes = float(tokens * (c["H"] + c["Hkv"]) * c["D"]), 2 if c["kind"] == "rotary_step" else 1
        return {"bytes": passes * (2 * values * (4 if c["dtype"] == "fp32" else 2) + 8.0 * tokens),
                "flops": passes * 3.0 * tokens * (c["H"] + c["Hkv"]) * c["rotary_dim"]}
    news, lens = _lengths(c)
    row = 2.0 * c["Hkv"] * (c["D"] * 2 if c["cache"] == "16" else c["D"] + 1)   # k and v of one token in the cache
    plain = 4.0 * c["Hkv"] * c["D"]                                            # and in contiguous 16-bit rows
    if c["kind"] == "append":
        return {"bytes": sum(news) * (row + plain), "flops": sum(news) * c["Hkv"] * c["D"] * (8.0 if c["rotary"] else 2.0)}
    if c["kind"] == "read":
        return {"bytes": sum(lens) * row + c["B"] * max(lens) * plain, "flops": 2.0 * sum(lens) * c["Hkv"] * c["D"]}
    pairs = seen = 0.0
    for n, length in zip(news, lens):
        w = c["window"] or length
        kept = [min(length - n + i + 1, w) for i in range(n)]
        pairs += sum(kept)
        seen += min(length, n - 1 + kept[0] if n > 1 else kept[0])
    return {"bytes": seen * row + sum(news) * c["H"] * (4.0 * c["D"] + 4), "flops": 4.0 * c["H"] * pairs * c["D"]}
