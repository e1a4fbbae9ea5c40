"""A key's way from a fused projection's output into a cache of 8 bits and to the token that reads it, and the work
these operators are measured on:

* ``rotary``: rotary positions of queries and keys, by one axis (a text) or several (time, height and width of
  images and video), halves or neighbours as pairs, over all of a head or its first values.
* ``cache_write`` and ``cache_read``: keys and values in 8 bits, int8 or e4m3 with one fp32 scale for each token and
  head, written to slots of a paged or padded cache, and read back as rows for a prompt's next chunk. What a
  pass returns is what it read back: the values that the codes stand for.
* ``attention_decode`` over such a cache (``k_scale``, ``v_scale``): one token of every request against its cached
  keys, and a prefix that all requests share, which is not in 8 bits.

Types are the framework's own: fp16 and fp32. Lengths and pages' order come from a case's own ``spread`` and the seed;
every value comes from the seed.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16}
SIZE = {"f32": 4, "f16": 2}
DEVICE = "cuda"
MINUS_INF = float("-inf")
LEAST = 2.0 ** -96  # a row of smaller values is written as zeros


def _gtx():
    sys.path.insert(0, os.path.join(os.getcwd(), "gtx16-fp16_amd"))
    try:
        import gtx16_fp16
    finally:
        del sys.path[0]
    return gtx16_fp16


# ---- cases ------------------------------------------------------------------------------------------


def _rotary(seqs, tokens, hq, hkv, d, dtype="f16", pairs=0, sections="", past=0, interleaved=False, ragged=False, spread=0, name=None):
    """``seqs`` texts of ``tokens`` tokens (``ragged``: at most) from position ``past`` on, or, with ``sections`` (pairs
    of each of three axes), clips of that many patches; q and k are slices of one projection's output. ``pairs``: that
    are rotated (0: all)."""
    c = {"entry": "rotary", "seqs": seqs, "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype, "pairs": pairs or d // 2,
         "sections": sections, "past": past, "interleaved": interleaved, "ragged": ragged, "spread": spread}
    return c if name is None else dict(c, name=name)


def _cache(seqs, tokens, past, hkv, d, dtype="f16", code="int8", page=16, whole=False, idle=False, by_head=False, spread=0, name=None):
    """``tokens`` new tokens (where more than 1: at most) of each of ``seqs`` requests written after up to ``past`` cached ones, and
    read back: the new ones, or (``whole``) each request's all. ``page`` 0: a padded cache; ``idle``: some rows of the
    batch belong to no request; ``by_head``: the cache's memory is ordered by heads, then tokens."""
    c = {"entry": "cache", "seqs": seqs, "tokens": tokens, "past": past, "hkv": hkv, "d": d, "dtype": dtype, "code": code, "page": page,
         "whole": whole, "idle": idle, "by_head": by_head, "spread": spread}
    return c if name is None else dict(c, name=name)


def _decode(seqs, longest, hq, hkv, d, dtype="f16", code="int8", page=0, shared=0, cap=0.0, distance=False, by_head=False, spread=0,
            name=None):
    """One token of each of ``seqs`` requests against up to ``longest`` keys of its own, in pages of ``page`` keys (0: a
    padded cache), after ``shared`` common ones."""
    c = {"entry": "attention_decode", "seqs": seqs, "longest": longest, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype, "code": code,
         "page": page, "shared": shared, "cap": cap, "distance": distance, "by_head": by_head, "spread": spread}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one token of a small fp32 model, every position so far below 300: launches and the host path decide
        _rotary(1, 1, 12, 12, 64, dtype="f32", past=299, name="rotary_token"),
        # prompts of mixed lengths that continue far into a long text, grouped heads
        _rotary(9, 1531, 32, 8, 128, past=120000, ragged=True, spread=1, name="rotary_prompts"),
        # clips of patches at their time, height and width; the first 80 values of a head turn, neighbours as pairs
        _rotary(3, 4097, 16, 16, 128, pairs=40, sections="8,16,16", interleaved=True, name="rotary_clips"),
        # one token of the small fp32 model kept
        _cache(1, 1, 299, 12, 64, dtype="f32", page=0, name="cache_token"),
        # a batch of 64 slots, one token each, some of them idle
        _cache(64, 1, 900, 8, 128, idle=True, spread=2, name="cache_tokens_64"),
        # prompts of nine requests written, and read for their own attention
        _cache(9, 1000, 0, 8, 128, code="e4m3", spread=3, name="cache_prompts"),
        # a chunk of a long prompt written, and all of the prompt so far read for the chunk's attention
        _cache(1, 512, 32256, 8, 128, page=64, whole=True, by_head=True, name="cache_chunk_of_32k"),
        # one request of the small fp32 model
        _decode(1, 300, 12, 12, 64, dtype="f32", name="token_fp32"),
        # a serving batch on pages of 16 keys after a shared system prompt
        _decode(16, 1500, 32, 8, 128, page=16, shared=2048, spread=4, name="tokens_16_shared"),
        # one request about a whole book: the key axis has to be split
        _decode(1, 131072, 32, 8, 128, page=256, by_head=True, name="token_128k"),
        # a full batch of half-precision heads of 64 with keys of their own, capped and biased by the distance
        _decode(96, 2048, 12, 12, 64, page=16, cap=50.0, distance=True, spread=5, name="tokens_96_12x64"),
        # long chats on a padded cache in e4m3
        _decode(40, 8192, 32, 8, 128, code="e4m3", spread=6, name="tokens_40_e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    spread = rng.randrange(1 << 16)
    kind = rng.choice(("rotary", "cache", "attention_decode", "attention_decode"))
    while True:
        d = rng.choice((32, 64, 64, 72, 80, 96, 128, 128, 128))
        hkv = rng.choice((1, 2, 4, 5, 8, 12))
        group = rng.choice((1, 1, 3, 4, 4, 8, 20))
        dtype, code = rng.choice(("f16", "f16", "f32")), rng.choice(("int8", "int8", "e4m3"))
        page, by_head = rng.choice((0, 16, 16, 24, 64, 256)), rng.random() < 0.4
        if kind == "rotary":
            pairs = rng.choice((d // 2, d // 2, d // 4, 5))
            t = rng.randrange(1, pairs - 1)
            h = rng.randrange(1, pairs - t)
            c = _rotary(_log(rng, 1, 64), _log(rng, 1, 8192), hkv * group, hkv, d, dtype, pairs, rng.choice(("", "%d,%d,%d" % (t, h, pairs - t - h))),
                        rng.choice((0, _log(rng, 1, 1 << 20))), rng.random() < 0.4, rng.random() < 0.6, spread)
            if c["seqs"] * c["tokens"] * (c["hq"] + hkv) * d * SIZE[dtype] <= 9 * 1531 * 40 * 128 * 2:
                return c
        elif kind == "cache":
            c = _cache(_log(rng, 1, 128), rng.choice((1, _log(rng, 1, 4096))), rng.choice((0, _log(rng, 1, 32768))), hkv, d, dtype, code, page,
                       rng.random() < 0.5, rng.random() < 0.2, by_head, spread)
            if c["seqs"] * (c["tokens"] + c["past"]) * hkv * d * SIZE[dtype] <= 1 << 28:
                return c
        else:
            c = _decode(_log(rng, 1, 128), _log(rng, 1, 131072), hkv * group, hkv, d, dtype, code, page,
                        rng.choice((0, 0, _log(rng, 1, 4096))), rng.choice((0.0, 0.0, 20.0, 50.0)), rng.random() < 0.3, by_head, spread)
            keys = c["seqs"] * (c["longest"] + c["shared"])
            if keys * max(c["hq"], 4 * hkv) * d <= 40 * 8192 * 32 * 128:
                return c


def _lengths(case):
    """Tokens of every request: the longest first, now and then none (of texts and attended keys)."""
    n, rng = case["seqs"], random.Random(case["spread"])
    most = case["longest"] if case["entry"] == "attention_decode" else case["tokens"]
    if case["entry"] == "rotary" and not case["ragged"] or most == 1:
        return [most] * n
    none = 0.0 if case["entry"] == "cache" else 0.05
    return [most] + [0 if rng.random() < none else 1 + rng.randrange(most) for _ in range(n - 1)]


def _pasts(case):
    """Cached tokens of every request before a pass."""
    rng = random.Random(case["spread"] + 1)
    return [case["past"]] + [rng.randrange(case["past"] + 1) for _ in range(case["seqs"] - 1)]


def _idle(case):
    rng = random.Random(case["spread"] + 2)
    return [case["idle"] and rng.random() < 0.1 for _ in range(case["seqs"])]


# ---- inputs -----------------------------------------------------------------------------------------


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _positions(case):
    """int32 [rows], or [axes, rows]: a clip of n patches is about 12 frames of square pictures."""
    rows = torch.cat([torch.arange(n, dtype=torch.int32) for n in _lengths(case)])
    if not case["sections"]:
        return (rows + case["past"]).to(DEVICE)
    side = max(1, math.isqrt(case["tokens"] // 12))
    return torch.stack((rows // (side * side) + case["past"], rows // side % side, rows % side)).to(DEVICE)


def _freqs(pairs):
    return torch.tensor([10000.0 ** (-i / pairs) for i in range(pairs)], dtype=torch.float32, device=DEVICE)


def _slopes(h):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], dtype=torch.float32, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype, d = TYPES[case["dtype"]], case["d"]

    def normal(*shape, scale=1.0, type=dtype):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32).mul_(scale).to(type)

    loud = torch.where(torch.rand(d, generator=g, device=DEVICE) < 0.05, 6.0, 1.0)  # the few large channels that keys have

    def cache(blocks, page):
        """(codes, scales) [blocks, page, heads(, d)] of keys, then of values"""
        out = []
        for of in (loud, 1.0):
            codes, scale = _coded(normal(blocks, page, case["hkv"], d, type=torch.float32) * of, case["code"])
            if case["by_head"]:
                codes, scale = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (codes, scale))
            out += [codes, scale]
        return dict(zip(("k_cache", "k_scale", "v_cache", "v_scale"), out))

    def pages(longest):
        per = -(-longest // case["page"])
        return torch.randperm(case["seqs"] * per, generator=g, device=DEVICE).to(torch.int32).reshape(case["seqs"], per)

    s = {"entry": case["entry"]}
    if case["entry"] == "rotary":
        heads = case["hq"] + case["hkv"]
        fused = normal(sum(_lengths(case)), heads + case["hkv"], d)
        sections = tuple(int(n) for n in case["sections"].split(",")) if case["sections"] else None
        axis = torch.repeat_interleave(torch.arange(3), torch.tensor(sections)).to(DEVICE) if sections else None  # of every pair
        return s | {"x": fused[:, :heads], "positions": _positions(case), "freqs": _freqs(case["pairs"]), "interleaved": case["interleaved"],
                    "sections": sections, "axis": axis}

    if case["entry"] == "cache":
        seqs, page, new, past = case["seqs"], case["page"], _lengths(case), _pasts(case)
        longest = max(a + b for a, b in zip(new, past))
        table = pages(longest) if page else None
        s |= cache(table.numel(), page) if page else cache(seqs, longest)

        def slots(first, count):
            at = torch.cat([torch.arange(a, a + n, dtype=torch.int32) for a, n in zip(first, count)]).to(DEVICE)
            seq = torch.repeat_interleave(torch.arange(seqs), torch.tensor(count)).to(DEVICE)
            return (table[seq, at // page] * page + at % page if page else seq * longest + at).to(torch.int32)

        write = slots(past, new)
        if case["idle"]:
            write = torch.where(torch.repeat_interleave(torch.tensor(_idle(case)), torch.tensor(new)).to(DEVICE), -1, write).to(torch.int32)
        read = slots([0] * seqs, [a + b for a, b in zip(past, new)]) if case["whole"] else write
        fused = normal(len(write), 4 * case["hkv"], d)
        return s | {"k": fused[:, 2 * case["hkv"]:3 * case["hkv"]].mul_(loud), "v": fused[:, 3 * case["hkv"]:], "write": write, "read": read,
                    "code": case["code"], "idle": case["idle"]}

    seqs, longest, page, hq, hkv, shared = (case[n] for n in ("seqs", "longest", "page", "hq", "hkv", "shared"))
    table = pages(longest) if page else None
    s |= cache(table.numel(), page) if page else cache(seqs, longest)
    return s | {"q": normal(seqs, hq, d, scale=0.8), "lengths": _ints(_lengths(case)), "pages": table, "cap": case["cap"],
                "slopes": _slopes(hq) if case["distance"] else None, "shared_k": normal(shared, hkv, d).mul_(loud) if shared else None,
                "shared_v": normal(shared, hkv, d) if shared else None}


# ---- the operators ----------------------------------------------------------------------------------


def run(s):
    if own:
        return _own(s)
    if s["entry"] == "rotary":
        return _plain_rotary(s)
    return _plain_cache(s) if s["entry"] == "cache" else _plain_decode(s)


def _own(s):
    g = _GTX or _load()
    if s["entry"] == "rotary":
        return g.rotary(s["x"], s["positions"], s["freqs"], sections=s["sections"], interleaved=s["interleaved"])
    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if s["entry"] == "cache":
        g.cache_write(s["k"], s["v"], *cache, s["write"])
        return g.cache_read(*cache, s["read"], out_dtype=s["k"].dtype)
    return g.attention_decode(s["q"], s["k_cache"], s["v_cache"], s["lengths"], pages=s["pages"], shared_k=s["shared_k"],
                              shared_v=s["shared_v"], softcap=s["cap"], slopes=s["slopes"], k_scale=s["k_scale"], v_scale=s["v_scale"])


_GTX = None


def _load():
    global _GTX
    _GTX = _gtx()
    return _GTX


def _plain_rotary(s):
    x, positions, freqs = s["x"], s["positions"].double(), s["freqs"].double()
    pairs = freqs.shape[0]
    angle = (positions[:, None] if s["axis"] is None else positions[s["axis"]].t()) * freqs
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    turned, rest = x[..., :2 * pairs].float(), x[..., 2 * pairs:]
    if s["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :pairs], turned[..., pairs:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned.to(x.dtype), rest), -1)


def _coded(x, code):
    """x [.., d] -> codes of 8 bits [.., d] and fp32 scales [..]"""
    x = x.float()
    top = x.abs().amax(-1)
    none, lost = top < LEAST, ~torch.isfinite(top)
    safe = torch.where(none | lost, torch.ones_like(top), top)
    if code == "int8":  # (in 64 bits the product with the rounded inverse is exact)
        scale = safe / 127.0
        codes = torch.round(x.double() * (127.0 / safe).double()[..., None])
        kind = torch.int8
    else:
        part, power = torch.frexp(safe)  # safe = part * 2^power, part from 0.5 up
        scale = torch.exp2((power - torch.where(part <= 0.875, 9, 8)).float())  # to at most 448 = 0.875 * 2^9
        codes = x / scale[..., None]
        kind = torch.float8_e4m3fn
    codes = torch.where((none | lost)[..., None], torch.zeros_like(codes), codes).float().to(kind)
    return codes, torch.where(lost, torch.full_like(scale, float("nan")), torch.where(none, torch.zeros_like(scale), scale))


def _bytes(t):
    return t.view(torch.uint8)


def _plain_cache(s):
    page, write, read = s["k_cache"].shape[1], s["write"].long(), s["read"].long()
    k, v = s["k"], s["v"]
    if s["idle"]:
        rows = write >= 0
        write, k, v = write[rows], k[rows], v[rows]
    at = (write // page, write % page)
    codes, scale = _coded(k, s["code"])
    _bytes(s["k_cache"])[at], s["k_scale"][at] = _bytes(codes), scale
    codes, scale = _coded(v, s["code"])
    _bytes(s["v_cache"])[at], s["v_scale"][at] = _bytes(codes), scale
    kind, out = s["k_cache"].dtype, s["k"].dtype
    seen, at = (read >= 0)[:, None, None], (read.clamp_min(0) // page, read.clamp_min(0) % page)

    def values(cache, scale):
        x = _bytes(cache)[at].view(kind).float() * scale[at][..., None]
        return torch.where(seen, x, torch.zeros_like(x)).to(out) if s["idle"] else x.to(out)

    return values(s["k_cache"], s["k_scale"]), values(s["v_cache"], s["v_scale"])


def _plain_decode(s):
    q, kind = s["q"], s["k_cache"].dtype
    seqs, hq, d = q.shape
    hkv, dev = s["k_cache"].shape[-2], q.device
    group, shared = hq // hkv, 0 if s["shared_k"] is None else s["shared_k"].shape[0]

    def values(cache, scale):
        cache = _bytes(cache)
        if s["pages"] is not None:
            at = s["pages"].long()
            cache, scale = cache[at].flatten(1, 2), scale[at].flatten(1, 2)
        return cache.view(kind).float() * scale[..., None]

    k, v = values(s["k_cache"], s["k_scale"]), values(s["v_cache"], s["v_scale"])
    n = s["lengths"].long()[:, None, None, None]
    j = torch.arange(k.shape[1], device=dev)
    slopes = None if s["slopes"] is None else s["slopes"].view(hkv, group, 1)
    qf, scale = q.float().view(seqs, hkv, group, d), 1.0 / math.sqrt(d)

    def scored(x, ahead):
        x = x * scale
        if s["cap"]:
            x = s["cap"] * torch.tanh(x / s["cap"])
        return x if slopes is None else x - slopes * ahead.float()

    scores = scored(torch.matmul(qf, k.permute(0, 2, 3, 1)), n - 1 - j).masked_fill(j >= n, MINUS_INF)
    if shared:  # the shared keys in one product for all requests
        rows = qf.transpose(0, 1).reshape(hkv, seqs * group, d)
        front = torch.matmul(rows, s["shared_k"].float().permute(1, 2, 0)).view(hkv, seqs, group, shared).transpose(0, 1)
        scores = torch.cat((scored(front, shared + n - 1 - torch.arange(shared, device=dev)), scores), -1)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == MINUS_INF, torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-37)  # a row without any key gets zeros
    out = torch.matmul(p[..., shared:], v.transpose(1, 2))
    if shared:
        rows = p[..., :shared].transpose(0, 1).reshape(hkv, seqs * group, shared)
        out = out + torch.matmul(rows, s["shared_v"].float().transpose(0, 1)).view(hkv, seqs, group, d).transpose(0, 1)
    return out.reshape(seqs, hq, d).to(q.dtype)


# ---- what a pass cannot do without ------------------------------------------------------------------


def work(case):
    size, d, hkv = SIZE[case["dtype"]], case["d"], case["hkv"]
    if case["entry"] == "rotary":
        rows, heads = sum(_lengths(case)), case["hq"] + hkv
        axes = 3 if case["sections"] else 1
        return {"bytes": 2 * size * rows * heads * d + 4 * axes * rows + 4 * case["pairs"], "flops": 6 * rows * heads * case["pairs"]}
    if case["entry"] == "cache":
        new = _lengths(case)
        written = sum(n for n, idle in zip(new, _idle(case)) if not idle)
        read = sum(new) + sum(_pasts(case)) if case["whole"] else sum(new)
        seen = read if case["whole"] else written
        return {"bytes": 2 * hkv * (written * (size * d + d + 4) + seen * (d + 4) + read * size * d) + 4 * (sum(new) + read),
                "flops": 2 * hkv * d * (3 * written + read)}
    hq, shared, keys = case["hq"], case["shared"], sum(_lengths(case))
    return {"bytes": 2 * keys * hkv * (d + 4) + size * d * (2 * case["seqs"] * hq + 2 * shared * hkv) + 4 * case["seqs"]
            + (4 * case["seqs"] * -(-case["longest"] // case["page"]) if case["page"] else 0),
            "flops": 4 * d * hq * (keys + case["seqs"] * shared)}


# ---- the definitions in 64 bits ---------------------------------------------------------------------


def _exact_coded(x, code):
    """What a row's values become in 8 bits, in 64."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    if code == "int8":
        inverse, step = (127.0 / top).float().double(), (top / 127.0).float().double()
        return torch.where(top < LEAST, 0.0, torch.round(x * inverse) * step)
    step = torch.exp2(torch.ceil(torch.log2(top / 448.0) - 1e-12))
    y = x / step
    unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3.0)  # of 3 bits behind the point, or the smallest
    return torch.where(top < LEAST, 0.0, torch.round(y / unit) * unit * step)


def exact(case, seed):
    s = prepare(case, seed)
    if case["entry"] == "rotary":
        x, turned = s["x"].double(), s["x"].double()
        for i in range(case["pairs"]):
            if s["sections"] is None:
                at = s["positions"]
            else:
                t, h, _ = s["sections"]
                at = s["positions"][0 if i < t else 1 if i < t + h else 2]
            i0, i1 = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + case["pairs"])
            z = torch.polar(torch.ones_like(at, dtype=torch.float64), at.double() * float(s["freqs"][i]))[:, None]
            z = z * torch.complex(x[..., i0], x[..., i1])
            turned[..., i0], turned[..., i1] = z.real, z.imag
        return turned
    flat = {n: s[n + "_cache"].reshape(-1, *s[n + "_cache"].shape[2:]).double() * s[n + "_scale"].reshape(-1, case["hkv"]).double()[..., None]
            for n in "kv"}
    if case["entry"] == "cache":
        out = []
        for n in "kv":
            at = s["write"].long()
            flat[n][at[at >= 0]] = _exact_coded(s[n], case["code"])[at >= 0]
            got = flat[n][s["read"].long().clamp_min(0)]
            got[s["read"] < 0] = 0.0
            out.append(got)
        return tuple(out)
    hq, hkv, d, shared, page = (case[n] for n in ("hq", "hkv", "d", "shared", "page"))
    group = hq // hkv
    out = torch.zeros(case["seqs"], hkv, group, d, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(_lengths(case)):
        at = torch.arange(n, device=DEVICE)
        at = s["pages"][b].long()[at // page] * page + at % page if page else b * case["longest"] + at
        k, v = flat["k"][at], flat["v"][at]
        if shared:
            k, v = torch.cat((s["shared_k"].double(), k)), torch.cat((s["shared_v"].double(), v))
        if not k.shape[0]:
            continue
        score = s["q"][b].double().view(hkv, group, d) @ k.permute(1, 2, 0).contiguous() / math.sqrt(d)
        if case["cap"]:
            score = torch.tanh(score / case["cap"]) * case["cap"]
        if case["distance"]:
            slope = 2.0 ** (-8.0 * torch.arange(1, hq + 1, dtype=torch.float64, device=DEVICE) / hq).float().double()
            score = score - slope.view(hkv, group, 1) * (shared + n - 1 - torch.arange(shared + n, device=DEVICE)).abs()
        out[b] = torch.softmax(score, -1) @ v.transpose(0, 1).contiguous()
    return out.view(case["seqs"], hq, d)
