"""The operators that a program serving many requests calls around this framework's linear layers, and the
work they are measured on:

* ``attention``: the attention of prompts, packed one after another or in an equal batch. A score may be
  capped by a tanh and biased by the distance between its two tokens; a row sees its own sequence only,
  all of it or causally, a sequence's first keys (``visible``) by every row of it, and a prefix that all
  sequences share before their own keys.
* ``attention_decode``: one token of every request against the request's cached keys (a padded cache or
  pages) and a prefix that all requests share, read once for all of them.
* ``lora_mm_t``: a linear layer's product with, for each row, the low-rank adapter of that row's request
  beside it: ``x @ w_t + bias + scale * (x @ down.T) @ up.T``.

Types are the framework's own: fp16 and fp32 activations and outputs, fp16 weights and adapters. fp32
outputs of ``lora_mm_t`` are measured up to 8 rows, where the framework's products keep every bit of an
fp32 activation; past that it rounds activations to fp16, and the cases return fp16.

Lengths, and which request has which adapter, come from a case's own ``spread``; every value comes from
the seed.
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


def _gtx():
    sys.path.insert(0, os.path.join(os.getcwd(), "gtx16-fp16_amd"))
    try:
        import gtx16_fp16
    finally:
        del sys.path[0]
    return gtx16_fp16


# ---- cases ------------------------------------------------------------------------------------------


def _attention(seqs, tokens, hq, hkv, d, dtype="f16", ragged=False, past=0, shared=0, causal=True, visible=0,
               cap=0.0, distance=False, spread=0, name=None):
    """``seqs`` sequences of ``tokens`` new tokens (``ragged``: at most), each after ``past`` keys of its own
    and ``shared`` common ones; ``visible``: the first keys of a sequence that all of its rows see."""
    c = {"entry": "attention", "seqs": seqs, "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype,
         "ragged": ragged, "past": past, "shared": shared, "causal": causal, "visible": visible, "cap": cap,
         "distance": distance, "spread": spread}
    return c if name is None else dict(c, name=name)


def _decode(seqs, longest, hq, hkv, d, dtype="f16", shared=0, page=0, cap=0.0, distance=False, spread=0, name=None):
    """One token of each of ``seqs`` requests against up to ``longest`` keys of its own, in pages of ``page``
    keys (0: a padded cache), after ``shared`` common ones."""
    c = {"entry": "attention_decode", "seqs": seqs, "longest": longest, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype,
         "shared": shared, "page": page, "cap": cap, "distance": distance, "spread": spread}
    return c if name is None else dict(c, name=name)


def _lora(M, K, N, rank, adapters, requests, x="f16", out="f16", bias=False, spread=0, name=None):
    """``M`` rows of ``requests`` requests, each with one of ``adapters`` adapters or, now and then, none."""
    c = {"entry": "lora_mm_t", "M": M, "K": K, "N": N, "rank": rank, "adapters": adapters, "requests": requests,
         "x": x, "out": out, "bias": bias, "spread": spread}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # a one-line prompt in a small half-precision model, its instruction seen by every row: launches and
        # the host path decide
        _attention(1, 23, 8, 2, 64, visible=9, name="prompt_23"),
        # an encoder batch of packed texts of mixed lengths, BERT-base's heads: the document mask
        _attention(48, 512, 12, 12, 64, ragged=True, causal=False, spread=1, name="documents_12x64"),
        # the same heads in an fp32 model, with a bias that grows with the distance
        _attention(32, 256, 12, 12, 64, dtype="f32", causal=False, distance=True, name="encoder_fp32"),
        # prompts that continue a shared system prompt, capped scores, grouped heads
        _attention(9, 700, 32, 8, 128, ragged=True, shared=1536, cap=30.0, spread=2, name="prompts_shared_capped"),
        # a chunk of a long prompt: few rows against a long cache
        _attention(1, 128, 32, 8, 128, past=16000, distance=True, name="chunk_128_of_16k"),
        # one long prompt, causal
        _attention(1, 8192, 32, 8, 128, name="prompt_8192"),
        # one request in a small fp32 model
        _decode(1, 300, 12, 12, 64, dtype="f32", name="token_fp32"),
        # a serving batch on pages of 16 keys after a shared system prompt
        _decode(16, 1500, 32, 8, 128, shared=2048, page=16, spread=3, name="tokens_16_paged"),
        # many requests about one long document, short answers so far
        _decode(64, 400, 32, 8, 128, shared=32768, spread=4, cap=50.0, name="tokens_64_shared_32k"),
        # one token of one request of a 1024-wide fp32 model
        _lora(1, 1024, 1024, 8, 4, 1, x="f32", out="f32", bias=True, name="lora_token"),
        # a decode batch, nearly every row with an adapter of its own
        _lora(48, 4096, 4096, 16, 40, 48, spread=5, name="lora_tokens_48"),
        # prompts of nine requests through a wide projection
        _lora(4111, 4096, 4096, 32, 8, 9, bias=True, spread=6, name="lora_prompts"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    spread = rng.randrange(1 << 16)
    kind = rng.choice(("attention", "attention_decode", "lora_mm_t"))
    while True:
        d = rng.choice((32, 64, 64, 72, 80, 96, 128, 128, 128))
        hkv = rng.choice((1, 2, 4, 5, 8, 12))
        group = rng.choice((1, 1, 3, 4, 4, 8))
        cap, distance = rng.choice((0.0, 0.0, 20.0, 50.0)), rng.random() < 0.3
        if kind == "attention":
            c = _attention(_log(rng, 1, 64), _log(rng, 1, 8192), hkv * group, hkv, d, rng.choice(("f16", "f16", "f32")),
                           rng.random() < 0.6, rng.choice((0, 0, _log(rng, 1, 16384))), rng.choice((0, 0, _log(rng, 1, 4096))),
                           rng.random() < 0.7, rng.choice((0, 0, _log(rng, 1, 512))), cap, distance, spread)
            most = 8192.0 ** 2 * 32 * 128
            rows, keys = c["seqs"] * c["tokens"], c["tokens"] + c["past"] + c["shared"]
            if rows * keys * c["hq"] * max(d, 64) * (4 if c["dtype"] == "f32" else 1) <= most and c["seqs"] * keys * hkv * d <= 1 << 28:
                return c
        elif kind == "attention_decode":
            c = _decode(_log(rng, 1, 96), _log(rng, 1, 20000), hkv * group, hkv, d, rng.choice(("f16", "f16", "f32")),
                        rng.choice((0, _log(rng, 1, 32768), _log(rng, 1, 32768))), rng.choice((0, 16, 16, 24, 64, 256)), cap, distance, spread)
            keys = c["seqs"] * (c["shared"] + c["longest"])
            if keys * c["hq"] * d <= 64 * 33168 * 32 * 128 and c["seqs"] * c["longest"] * hkv * d <= 1 << 28:
                return c
        else:
            M, K, N = _log(rng, 1, 4096), 8 * _log(rng, 32, 1400), 8 * _log(rng, 32, 1400)
            x = rng.choice(("f16", "f16", "f32"))
            c = _lora(M, K, N, rng.choice((8, 16, 16, 32, 64)), _log(rng, 1, 64), rng.choice((M, max(1, min(M, _log(rng, 1, 64))))),
                      x, "f32" if x == "f32" and M <= 8 else "f16", rng.random() < 0.5, spread)
            if M * K * N <= 4111 * 4096 * 4096 and c["adapters"] * c["rank"] * (K + N) <= 1 << 25:
                return c


def _lengths(case):
    """New tokens of every sequence: the longest one first, now and then an empty one."""
    n, most = case["seqs"], case["tokens"] if case["entry"] == "attention" else case["longest"]
    rng = random.Random(case["spread"])
    if case["entry"] == "attention" and not case["ragged"]:
        return [most] * n
    return [most] + [0 if rng.random() < 0.05 else 1 + rng.randrange(most) for _ in range(n - 1)]


def _adapters_of(case):
    """The adapter of every row: rows of a request stand together; -1 is none."""
    rng = random.Random(case["spread"])
    M, requests = case["M"], case["requests"]
    if requests == M:
        cuts = list(range(M + 1))
    else:
        cuts = [0] + sorted(rng.sample(range(1, M), requests - 1)) + [M]
    got = []
    for a, b in zip(cuts, cuts[1:]):
        got += [-1 if requests > 4 and rng.random() < 0.1 else rng.randrange(case["adapters"])] * (b - a)
    return got


# ---- inputs -----------------------------------------------------------------------------------------


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=DEVICE)


def _slopes(h):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], dtype=torch.float32, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))

    def normal(*shape, scale=1.0, dtype=None):
        x = torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)
        return x.mul_(scale).to(TYPES[case["dtype"]] if dtype is None else TYPES[dtype])

    if case["entry"] == "lora_mm_t":
        M, K, N, r, n = (case[k] for k in ("M", "K", "N", "rank", "adapters"))
        x = normal(M, K, dtype=case["x"])
        if M >= 16:
            x[M // 3] *= 40.0  # a row of massive activations
        return {"entry": "lora_mm_t", "x": x, "w": normal(K, N, scale=0.02, dtype="f16"),
                "down": normal(n, r, K, scale=K ** -0.5, dtype="f16"), "up": normal(n, N, r, scale=0.05, dtype="f16"),
                "scale": 0.5 + torch.rand(n, generator=g, device=DEVICE),
                "index": torch.tensor(_adapters_of(case), dtype=torch.int32, device=DEVICE),
                "bias": normal(N, dtype="f32") if case["bias"] else None, "out": TYPES[case["out"]]}

    hq, hkv, d, shared = (case[k] for k in ("hq", "hkv", "d", "shared"))
    lengths = _lengths(case)
    s = {"entry": case["entry"], "cap": case["cap"], "slopes": _slopes(hq) if case["distance"] else None,
         "shared_k": normal(shared, hkv, d) if shared else None, "shared_v": normal(shared, hkv, d) if shared else None}
    if case["entry"] == "attention_decode":
        seqs, longest, page = case["seqs"], case["longest"], case["page"]
        s |= {"q": normal(seqs, hq, d, scale=1.5), "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEVICE),
              "pages": None}
        if page:
            per = -(-longest // page)
            s["pages"] = torch.randperm(seqs * per, generator=g, device=DEVICE).to(torch.int32).reshape(seqs, per)
            s |= {"k": normal(seqs * per, page, hkv, d), "v": normal(seqs * per, page, hkv, d)}
        else:
            s |= {"k": normal(seqs, longest, hkv, d), "v": normal(seqs, longest, hkv, d)}
        return s

    past, seqs, tokens = case["past"], case["seqs"], case["tokens"]
    rows = sum(lengths)
    if past:
        q, k, v = (normal(rows + n * seqs, h, d, scale=w) for n, h, w in ((0, hq, 1.5), (past, hkv, 1.0), (past, hkv, 1.0)))
    else:  # views of one projection's output
        fused = normal(rows, hq + 2 * hkv, d)
        fused[:, :hq] *= 1.5
        q, k, v = fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:]
    s |= {"q": q, "k": k, "v": v, "q_offsets": None, "k_offsets": None, "causal": case["causal"], "visible": None,
          "longest": max(lengths), "past": past}
    if case["ragged"]:
        s["q_offsets"] = _starts(lengths)
        s["k_offsets"] = _starts([n + past for n in lengths]) if past else s["q_offsets"]
    else:
        s |= {n: s[n].unflatten(0, (seqs, -1)) for n in ("q", "k", "v")}
    if case["visible"]:
        s["visible"] = torch.full((seqs,), case["visible"], dtype=torch.int32, device=DEVICE)
    return s


# ---- the operators ----------------------------------------------------------------------------------


def run(s):
    if own:
        return _own(s)
    if s["entry"] == "attention":
        return _plain_attention(s)
    return _plain_decode(s) if s["entry"] == "attention_decode" else _plain_lora(s)


def _own(s):
    g = _GTX or _load()
    if s["entry"] == "attention":
        return g.attention(s["q"], s["k"], s["v"], q_offsets=s["q_offsets"], k_offsets=s["k_offsets"], causal=s["causal"],
                           visible=s["visible"], shared_k=s["shared_k"], shared_v=s["shared_v"], softcap=s["cap"],
                           slopes=s["slopes"])
    if s["entry"] == "attention_decode":
        return g.attention_decode(s["q"], s["k"], s["v"], s["lengths"], pages=s["pages"], shared_k=s["shared_k"],
                                  shared_v=s["shared_v"], softcap=s["cap"], slopes=s["slopes"])
    return g.lora_mm_t(s["x"], s["w"], s["down"], s["up"], s["index"], scale=s["scale"], bias=s["bias"], out_dtype=s["out"])


_GTX = None


def _load():
    global _GTX
    _GTX = _gtx()
    return _GTX


def _softmax_parts(scores):
    """Weights of masked scores (-inf) in the last axis; a row with nothing to see gets zeros."""
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == MINUS_INF, torch.zeros_like(top), top))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-37)


def _scores(q, k, scale, cap, slopes, distance):
    """q [.., H, rows, d], k [.., H, keys, d]; slopes [H] with distance broadcastable to the scores."""
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    return s if slopes is None else s - slopes[:, None, None] * distance.abs().float()


def _grouped(x, group):
    """[B, L, Hkv, d] -> fp32 [B, Hkv * group, L, d]"""
    return x.float().transpose(1, 2).repeat_interleave(group, dim=1)


def _plain_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    hq, d = q.shape[-2:]
    group, dev = hq // k.shape[-2], q.device
    longest, shared = s["longest"], 0 if s["shared_k"] is None else s["shared_k"].shape[0]
    if s["q_offsets"] is None:
        nq = torch.full((q.shape[0],), q.shape[1], device=dev)
        nk = torch.full((k.shape[0],), k.shape[1], device=dev)
        qp, kp, vp = q, k, v
    else:  # packed: padded to the longest
        qo, ko = s["q_offsets"].long(), s["k_offsets"].long()
        nq, nk = qo[1:] - qo[:-1], ko[1:] - ko[:-1]
        qp = q[(qo[:-1, None] + torch.arange(longest, device=dev)).clamp_max(q.shape[0] - 1)]
        at = (ko[:-1, None] + torch.arange(longest + s["past"], device=dev)).clamp_max(k.shape[0] - 1)
        kp, vp = k[at], v[at]
    i = torch.arange(qp.shape[1], device=dev)[None, :, None]
    j = torch.arange(kp.shape[1], device=dev)[None, None, :]
    at_q = shared + i + (nk - nq)[:, None, None]
    seen = (j < nk[:, None, None]).expand(-1, qp.shape[1], -1)
    if s["causal"]:
        below = shared + j <= at_q
        if s["visible"] is not None:
            below = below | (shared + j < s["visible"][:, None, None])
        seen = seen & below
    qf = qp.float().transpose(1, 2)
    scale = 1.0 / math.sqrt(d)
    scores = _scores(qf, _grouped(kp, group), scale, s["cap"], s["slopes"], (at_q - shared - j)[:, None])
    scores = scores.masked_fill(~seen[:, None], MINUS_INF)
    if shared:
        c = torch.arange(shared, device=dev)[None, None, :]
        front = _scores(qf, _grouped(s["shared_k"][None], group), scale, s["cap"], s["slopes"], (at_q - c)[:, None])
        if s["causal"]:
            below = c <= at_q
            if s["visible"] is not None:
                below = below | (c < s["visible"][:, None, None])
            front = front.masked_fill(~below[:, None], MINUS_INF)
        scores = torch.cat((front, scores), -1)
    p = _softmax_parts(scores)
    out = torch.matmul(p[..., shared:], _grouped(vp, group))
    if shared:
        out = out + torch.matmul(p[..., :shared], _grouped(s["shared_v"][None], group))
    out = out.transpose(1, 2)
    if s["q_offsets"] is not None:
        seq = torch.repeat_interleave(torch.arange(nq.shape[0], device=dev), nq, output_size=q.shape[0])
        out = out[seq, torch.arange(q.shape[0], device=dev) - qo[seq]]
    return out.to(q.dtype)


def _plain_decode(s):
    q, k, v = s["q"], s["k"], s["v"]
    seqs, hq, d = q.shape
    hkv, dev = k.shape[-2], q.device
    group, shared = hq // hkv, 0 if s["shared_k"] is None else s["shared_k"].shape[0]
    if s["pages"] is not None:
        at = s["pages"].long()
        k, v = k[at].flatten(1, 2), v[at].flatten(1, 2)
    n = s["lengths"].long()[:, None, None, None]
    j = torch.arange(k.shape[1], device=dev)
    slopes = None if s["slopes"] is None else s["slopes"].view(hkv, group, 1)
    qf, scale = q.float().view(seqs, hkv, group, d), 1.0 / math.sqrt(d)

    def scored(x, ahead):
        x = x * scale
        if s["cap"]:
            x = s["cap"] * torch.tanh(x / s["cap"])
        return x if slopes is None else x - slopes * ahead.float()

    scores = scored(torch.matmul(qf, k.float().permute(0, 2, 3, 1)), n - 1 - j)
    scores = scores.masked_fill(j >= n, MINUS_INF)
    if shared:  # the shared keys in one product for all requests
        rows = qf.transpose(0, 1).reshape(hkv, seqs * group, d)
        front = torch.matmul(rows, s["shared_k"].float().permute(1, 2, 0)).view(hkv, seqs, group, shared).transpose(0, 1)
        front = scored(front, shared + n - 1 - torch.arange(shared, device=dev))
        scores = torch.cat((front, scores), -1)
    p = _softmax_parts(scores)
    out = torch.matmul(p[..., shared:], v.float().transpose(1, 2))
    if shared:
        rows = p[..., :shared].transpose(0, 1).reshape(hkv, seqs * group, shared)
        out = out + torch.matmul(rows, s["shared_v"].float().transpose(0, 1)).view(hkv, seqs, group, d).transpose(0, 1)
    return out.reshape(seqs, hq, d).to(q.dtype)


def _plain_lora(s):
    x, down, up, index = s["x"].float(), s["down"].float(), s["up"].float(), s["index"]
    n, r, K = down.shape
    y = torch.matmul(x, s["w"].float())
    if s["bias"] is not None:
        y = y + s["bias"]
    # every row through every adapter's first half, and only its own kept for the second
    low = torch.matmul(x, down.reshape(n * r, K).t()).view(-1, n, r)
    mine = (index[:, None] == torch.arange(n, device=x.device, dtype=torch.int32)).float() * s["scale"]
    low = (low * mine[:, :, None]).reshape(-1, n * r)
    return (y + torch.matmul(low, up.transpose(1, 2).reshape(n * r, -1))).to(s["out"])


# ---- what a pass cannot do without ------------------------------------------------------------------


def _pairs(case):
    """Query-key pairs of all sequences, of one head."""
    total, before = 0, case["past"] + case["shared"]
    for n in _lengths(case):
        if not case["causal"]:
            total += n * (n + before)
            continue
        see = min(case["visible"], n + before)
        early = max(0, min(n, see - before - 1))  # rows that see less than `see` causally
        total += early * see + (n - early) * (2 * before + 1 + early + n) // 2
    return total


def work(case):
    if case["entry"] == "lora_mm_t":
        M, K, N, r = (case[k] for k in ("M", "K", "N", "rank"))
        of = _adapters_of(case)
        distinct, rows = len({a for a in of if a >= 0}), sum(a >= 0 for a in of)
        return {"bytes": M * K * SIZE[case["x"]] + M * N * SIZE[case["out"]] + 2 * K * N + 2 * distinct * r * (K + N) + 4 * M
                + (4 * N if case["bias"] else 0),
                "flops": 2 * M * K * N + 2 * rows * r * (K + N)}
    size, d, hq, hkv = SIZE[case["dtype"]], case["d"], case["hq"], case["hkv"]
    lengths = _lengths(case)
    if case["entry"] == "attention":
        rows, keys = sum(lengths), sum(lengths) + case["past"] * case["seqs"] + case["shared"]
        return {"bytes": size * d * (2 * rows * hq + 2 * keys * hkv), "flops": 4 * d * hq * _pairs(case)}
    keys = sum(lengths) + case["shared"]
    return {"bytes": size * d * (2 * case["seqs"] * hq + 2 * keys * hkv) + 4 * case["seqs"],
            "flops": 4 * d * hq * (sum(lengths) + case["seqs"] * case["shared"])}


# ---- the definitions in 64 bits ---------------------------------------------------------------------


def _exact_rows(q, k, v, at_q, at_k, seen, cap, slope):
    """softmax(q k^T / sqrt(d), capped, biased) v of one head: q [rows, d], k and v [keys, d], positions of
    both, seen [rows, keys] or None."""
    if not k.shape[0]:
        return torch.zeros_like(q)
    s = (q @ k.T) / math.sqrt(q.shape[1])
    if cap:
        s = torch.tanh(s / cap) * cap
    if slope is not None:
        s = s - slope * (at_q[:, None] - at_k[None, :]).abs()
    if seen is not None:
        s[~seen] = MINUS_INF
    s = torch.exp(s - s.max(1, keepdim=True).values.nan_to_num(neginf=0.0))
    total = s.sum(1, keepdim=True)
    return torch.where(total > 0, (s @ v) / total.clamp_min(1e-300), torch.zeros_like(q))


def exact(case, seed):
    s = prepare(case, seed)
    if case["entry"] == "lora_mm_t":
        x = s["x"].double()
        y = x @ s["w"].double()
        if case["bias"]:
            y += s["bias"].double()
        of = torch.tensor(_adapters_of(case), device=DEVICE)
        for a in range(case["adapters"]):
            rows = (of == a).nonzero().flatten()
            if rows.numel():
                y[rows] += s["scale"][a].double() * ((x[rows] @ s["down"][a].double().T) @ s["up"][a].double().T)
        return y
    lengths, hq, hkv, d, shared = _lengths(case), case["hq"], case["hkv"], case["d"], case["shared"]
    group, decode = hq // hkv, case["entry"] == "attention_decode"
    past, size = (0, case["seqs"]) if decode else (case["past"], sum(lengths))
    out = torch.zeros(size, hq, d, dtype=torch.float64, device=DEVICE)
    flat = {n: s[n].reshape(-1, *s[n].shape[-2:]) for n in "qkv"}
    row = key = 0
    for b, n in enumerate(lengths):
        if decode:
            rows, keys = slice(b, b + 1), n
            if case["page"]:
                one = torch.arange(n, device=DEVICE)
                where = s["pages"][b].long()[one // case["page"]] * case["page"] + one % case["page"]
            else:
                where = b * case["longest"] + torch.arange(n, device=DEVICE)
            at_q = torch.tensor([shared + n - 1], device=DEVICE)
        else:
            rows, keys = slice(row, row + n), n + past
            where = key + torch.arange(keys, device=DEVICE)
            at_q = shared + past + torch.arange(n, device=DEVICE)
            row, key = row + n, key + keys
        at_k = torch.arange(shared + keys, device=DEVICE)
        seen = None
        if not decode and case["causal"]:
            seen = (at_k[None, :] <= at_q[:, None]) | (at_k < case["visible"])[None, :]
        for h in range(hkv):
            k, v = flat["k"][where, h].double(), flat["v"][where, h].double()
            if shared:
                k, v = torch.cat((s["shared_k"][:, h].double(), k)), torch.cat((s["shared_v"][:, h].double(), v))
            for i in range(h * group, (h + 1) * group):
                slope = 2.0 ** (-8.0 * (i + 1) / hq) if case["distance"] else None
                out[rows, i] = _exact_rows(flat["q"][rows, i].double(), k, v, at_q, at_k, seen, case["cap"], slope)
    return out if decode or case["ragged"] else out.unflatten(0, (case["seqs"], -1))
