"""Single tokens over a cache of 8 bits on the GPU, against attention over the numbers that its codes stand for, in 64 bits.

The bound is that of _attention.py but for the weights: fp16 queries' are multiplied to 2^-17 of each, in two parts (rounded
sums of them another 2^-17 at most), fp32 ones' to 2^-24, which the sums' own bound covers."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from _attention import check, one_sequence
from _cache8 import random_cache

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def expected(q, k, v, lengths, shared_k=None, shared_v=None, scale=None, softcap=0.0, slopes=None):
    """q [requests, hq, d] in its own type, k and v a list of each request's keys [n, hkv, d], doubles: (out, bound)."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    u = 2.0 ** -11 if q.dtype == F16 else 2.0 ** -24
    outs, bounds = [], []
    for b, n in enumerate(lengths):
        kk, vv, front = k[b][:n], v[b][:n], 0
        if shared_k is not None:
            front = shared_k.shape[0]
            kk, vv = torch.cat((shared_k.double(), kk)), torch.cat((shared_v.double(), vv))
        o, mean, err = one_sequence(q[b:b + 1].double(), kk, vv, torch.tensor([front + n - 1]), torch.arange(front + n),
                                    torch.ones(1, front + n, dtype=torch.bool), scale, softcap, slopes)
        outs.append(o)
        weights = 0.0 if q.dtype == F32 else (2.0 ** -16 if shared_k is None else u)  # (the shared keys' weights are fp16)
        bounds.append(u * o.abs() + (weights + err) * mean + (2.0 ** -25 if q.dtype == F16 else 1e-37))
    return torch.cat(outs), torch.cat(bounds)


def case(cuda, dtype, code, lengths, hq, hkv, d, page=0, capacity=None, shared=0, by_head=False, softcap=0.0, biased=False, scale=None, seed=0,
         spoil=True):
    """(call's arguments, expected) of a cache whose unused places hold NaN."""
    gen = torch.Generator().manual_seed(seed)
    seqs, longest = len(lengths), max(max(lengths), 1) if capacity is None else capacity
    per = -(-longest // page) if page else 1
    cache, k, v = random_cache(seqs * per + (3 if page else 0), page or longest, hkv, d, code, gen, by_head=by_head, loud=2.0)
    blocks = cache[0].shape[0]
    table = torch.randperm(blocks, generator=gen)[:seqs * per].view(seqs, per).to(torch.int32) if page else None
    used = torch.zeros(blocks, page or longest, dtype=torch.bool)
    keys, values = [], []
    for b, n in enumerate(lengths):
        at = torch.arange(max(0, n))
        rows = (table[b].long()[at // page], at % page) if page else (torch.full_like(at, b), at)
        used[rows] = True
        keys.append(k[rows])
        values.append(v[rows])
    if spoil:
        for t in cache[2:]:
            t[~used] = float("nan")
        if code == "e4m3":
            for t in cache[:2]:
                t.view(torch.uint8)[~used] = 0x7f
    q = torch.randn(seqs, hq, d, generator=gen).to(dtype)
    sk, sv = (torch.randn(shared, hkv, d, generator=gen).to(dtype) for _ in "kv") if shared else (None, None)
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)]) if biased else None
    move = lambda t: None if t is None else (t.to(cuda) if not by_head or t.dim() < 3 else t.transpose(1, 2).contiguous().to(cuda).transpose(1, 2))  # noqa: E731
    kc, vc, ks, vs = (move(t) for t in cache)
    plain = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    args = (q.to(cuda), kc, vc, torch.tensor(lengths, dtype=torch.int32, device=cuda))
    kw = dict(pages=plain(table), shared_k=plain(sk), shared_v=plain(sv), scale=scale, softcap=softcap, slopes=plain(slopes), k_scale=ks, v_scale=vs)
    return args, kw, expected(q, keys, values, [max(0, n) for n in lengths], sk, sv, scale, softcap, slopes)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lengths,hq,hkv,d,kw", [
    ([1], 1, 1, 8, {}), ([0], 2, 1, 64, {}), ([300], 12, 12, 64, {}), ([31, 32, 33, 1, 0], 4, 2, 128, {}), ([5, 129, 64], 6, 2, 72, dict(page=7)),
    ([100, 3, 0, 260], 8, 2, 128, dict(page=16)), ([77, 200], 20, 1, 128, dict(page=24)), ([40, 70], 40, 1, 64, dict(page=64, by_head=True)),
    ([33, 90], 17, 1, 96, dict(page=1)), ([200, 511, 17], 6, 3, 24, dict(by_head=True)), ([129, 0, 63], 5, 5, 40, dict(page=16, biased=True)),
    ([90, 300], 8, 4, 64, dict(softcap=20.0)), ([64, 65], 4, 1, 128, dict(page=256, softcap=50.0, biased=True)), ([33], 16, 1, 64, dict(scale=-0.3)),
    ([50, 20], 4, 4, 32, dict(scale=0.0)), ([45, 130], 4, 2, 80, dict(softcap=1000.0, page=16)), ([20, 5], 4, 2, 64, dict(capacity=500)),
], ids=str)
def test_against_64_bits(cuda, dtype, code, lengths, hq, hkv, d, kw):
    args, more, ref = case(cuda, dtype, code, lengths, hq, hkv, d, seed=sum(lengths), **kw)
    check(g.attention_decode(*args, **more), ref)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lengths,hq,hkv,d,kw", [
    ([2500], 2, 1, 128, {}), ([5000, 3], 4, 4, 64, dict(page=16)), ([700, 1900, 1, 0, 513], 8, 2, 128, dict(page=64, by_head=True)), ([4000], 24, 1, 80, dict(page=24)),
], ids=str)
def test_keys_split_over_workgroups(cuda, dtype, code, lengths, hq, hkv, d, kw):
    args, more, ref = case(cuda, dtype, code, lengths, hq, hkv, d, seed=7, **kw)
    y = g.attention_decode(*args, **more)
    check(y, ref)
    assert torch.equal(y, g.attention_decode(*args, **more))


@pytest.mark.parametrize("lengths,kw", [
    ([(37 * i) % 190 for i in range(150)], dict(capacity=600, page=16)),  # dealt in shares over more requests than a wavefront has lanes
    ([(7 * i) % 65 for i in range(40)], dict(capacity=600)),               # in more pieces than there are workgroups
    ([(7 * i) % 65 for i in range(140)], dict(capacity=600, page=24)),
    ([0] * 70 + [300] + [0] * 70, dict(capacity=600)),
], ids=lambda v: str(len(v)))
def test_many_requests(cuda, lengths, kw):
    args, more, ref = case(cuda, F16, "int8", lengths, 32, 32, 8, seed=len(lengths), **kw)
    check(g.attention_decode(*args, **more), ref)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lengths,hq,hkv,d,kw", [
    ([0, 1, 40], 4, 2, 64, dict(shared=1)), ([10, 0], 8, 1, 128, dict(shared=300, page=16)), ([5] * 40, 4, 2, 72, dict(shared=70)), ([3, 70], 2, 2, 64, dict(shared=40)),
    ([900, 0, 64], 16, 2, 128, dict(shared=65, page=16, by_head=True)), ([7] * 3, 12, 2, 64, dict(shared=200)),
    ([600, 30], 20, 1, 64, dict(shared=900, page=16, softcap=30.0, biased=True)), ([1200] * 2, 4, 2, 96, dict(shared=33, page=24, by_head=True)),
], ids=str)
def test_after_a_shared_prefix(cuda, dtype, code, lengths, hq, hkv, d, kw):
    args, more, ref = case(cuda, dtype, code, lengths, hq, hkv, d, seed=3, **kw)
    check(g.attention_decode(*args, **more), ref)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_pages_and_lengths_outside(cuda, dtype):
    (q, kc, vc, lengths), kw, _ = case(cuda, dtype, "int8", [40, 25, 64], 4, 2, 64, page=16, capacity=64, spoil=False)
    table = kw["pages"].clone()
    table[0, 1], table[0, 2], table[1, 0] = -1, kc.shape[0], 1 << 30
    kc2, vc2, ks, vs = (t.clone() for t in (kc, vc, kw["k_scale"], kw["v_scale"]))
    zero = torch.zeros(1, *kc.shape[1:], dtype=torch.int8, device=cuda)
    kc2, vc2 = torch.cat((kc2, zero)), torch.cat((vc2, zero))
    ks, vs = (torch.cat((t, t.new_ones(1, *t.shape[1:]))) for t in (ks, vs))
    zeros = torch.where((table < 0) | (table >= kc.shape[0]), kc.shape[0], table).to(torch.int32)
    a = g.attention_decode(q, kc, vc, lengths, **(kw | dict(pages=table)))
    b = g.attention_decode(q, kc2, vc2, lengths, **(kw | dict(pages=zeros, k_scale=ks, v_scale=vs)))
    assert torch.equal(a, b)
    # lengths past the capacity are the capacity, negative ones none
    whole = g.attention_decode(q, kc, vc, torch.full_like(lengths, 64), **kw)
    assert torch.equal(whole, g.attention_decode(q, kc, vc, torch.full_like(lengths, 1 << 30), **kw))
    assert not g.attention_decode(q, kc, vc, torch.full_like(lengths, -5), **kw).any()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_keys_and_values_that_are_nan(cuda, dtype):
    (q, kc, vc, lengths), kw, ref = case(cuda, dtype, "int8", [40, 40, 40], 4, 2, 64)
    kw["k_scale"][0, 7, 0] = kw["v_scale"][1, 39, 1] = float("nan")
    y = g.attention_decode(q, kc, vc, lengths, **kw)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[0, :2] = bad[1, 2:] = True
    assert (torch.isnan(y) == bad).all()
    clean, tol = ref
    assert ((y.cpu().double() - clean).abs() <= tol)[~bad.cpu()].all()


def test_large_and_small_scales(cuda):
    # fp32: values about the largest and about 2^-96, scores that leave one key, or all of them alike
    for factor_k, factor_v in ((2.0 ** 90, 2.0 ** 120), (2.0 ** -90, 2.0 ** -90)):
        gen = torch.Generator().manual_seed(1)
        cache, k, v = random_cache(2, 100, 2, 64, "int8", gen)
        q = torch.randn(2, 4, 64, generator=gen) / factor_k
        cache[2] *= factor_k
        cache[3] *= factor_v
        kw = dict(k_scale=cache[2].to(cuda), v_scale=cache[3].to(cuda))
        y = g.attention_decode(q.to(cuda), cache[0].to(cuda), cache[1].to(cuda), torch.tensor([100, 57], dtype=torch.int32, device=cuda), **kw)
        check(y, expected(q, [k[b] * factor_k for b in range(2)], [v[b] * factor_v for b in range(2)], [100, 57]))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_infinite_queries_are_nan_alone(cuda, dtype):
    (q, kc, vc, lengths), kw, ref = case(cuda, dtype, "e4m3", [70, 5], 4, 1, 128)
    q[0, 2, 5], q[1, 0, 0] = float("inf"), float("nan")
    y = g.attention_decode(q, kc, vc, lengths, **kw)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[0, 2] = bad[1, 0] = True
    assert (torch.isnan(y) == bad).all()


def test_views(cuda):
    # queries out of a fused projection, a cache in a larger tensor whose rows are only 8 bytes apart from alignment
    gen = torch.Generator().manual_seed(5)
    cache, k, v = random_cache(6, 16, 2, 72, "e4m3", gen)
    big = torch.zeros(6, 16, 2, 2, 88, dtype=torch.uint8, device=cuda)
    kc, vc = (big[:, :, i, :, 8:80].view(torch.float8_e4m3fn) for i in range(2))
    kc.view(torch.uint8).copy_(cache[0].view(torch.uint8)), vc.view(torch.uint8).copy_(cache[1].view(torch.uint8))
    scales = torch.stack(cache[2:], -1).to(cuda)
    fused = torch.randn(3, 8, 72, generator=gen).half()
    table = torch.randperm(6, generator=gen).view(3, 2).to(torch.int32)
    lengths = [32, 17, 9]
    y = g.attention_decode(fused.to(cuda)[:, 2:6], kc, vc, torch.tensor(lengths, dtype=torch.int32, device=cuda), pages=table.to(cuda),
                           k_scale=scales[..., 0], v_scale=scales[..., 1])
    flat = [[t[table[b].long()].reshape(-1, 2, 72) for b in range(3)] for t in (k, v)]
    check(y, expected(fused[:, 2:6], *flat, lengths))


def test_a_cache_past_32_bits(cuda):
    # the last request's keys start behind 4 GiB
    heads, d, capacity = 8, 128, 1 << 20
    seqs = (1 << 32) // (heads * d * capacity) + 1
    kc = torch.zeros(seqs, capacity, heads, d, dtype=torch.int8, device=cuda)
    vc = torch.zeros_like(kc)
    ks, vs = (torch.ones(seqs, capacity, heads, device=cuda) for _ in "kv")
    gen = torch.Generator().manual_seed(2)
    cache, k, v = random_cache(1, 100, heads, d, "int8", gen)
    for to, t in zip((kc, vc, ks, vs), cache):
        to[-1, :100] = t[0].to(cuda)
    q = torch.randn(seqs, 16, d, generator=gen).half()
    lengths = [0] * (seqs - 1) + [100]
    y = g.attention_decode(q.to(cuda), kc, vc, torch.tensor(lengths, dtype=torch.int32, device=cuda), k_scale=ks, v_scale=vs)
    check(y, expected(q, [k[0, :0]] * (seqs - 1) + [k[0]], [v[0, :0]] * (seqs - 1) + [v[0]], lengths))


def test_two_streams_and_graphs(cuda):
    (q, kc, vc, lengths), kw, _ = case(cuda, F16, "int8", [900, 1500, 40], 8, 2, 128, page=16, shared=200, spoil=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        g.attention_decode(q, kc, vc, lengths, **kw)
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(g.attention_decode(q, kc, vc, lengths, **kw))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(3):
        q.mul_(0.9)
        lengths.copy_(torch.tensor([900 - 100 * step, 1500, 41 + step], dtype=torch.int32))
        eager = g.attention_decode(q, kc, vc, lengths, **kw)
        for graph, y in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lengths,hq,hkv,d,kw", [
    ([700, 0, 64, 1, 513, 65], 4, 4, 64, dict(page=16)), ([600, 1300, 63, 2], 32, 8, 128, dict(page=24, shared=70)),
    ([1100, 0, 0, 5], 24, 12, 64, dict(softcap=20.0, biased=True)), ([900, 40], 64, 8, 128, dict(page=64, biased=True)),
    ([640, 129, 31], 20, 4, 64, dict(shared=33, softcap=30.0)),
    ([1500 - 31 * i for i in range(48)], 16, 16, 64, dict(page=16)), ([1200] * 23 + [0, 7], 8, 8, 128, {}),
])
def test_heads_next_to_each_other(cuda, dtype, code, lengths, hq, hkv, d, kw):
    # past 512 keys four heads of a token go together, by pieces of few tiles or (many keys) by equal shares
    args, kw, expect = case(cuda, dtype, code, lengths, hq, hkv, d, **kw)
    check(g.attention_decode(*args, **kw), expect)


def test_graphs_of_one_stream_at_once(cuda):
    # two graphs captured on one stream, replayed on two: neither uses the other's workspace
    cases = [case(cuda, F16, "int8", [3000, 1500, 40 + i], 8, 2, 128, page=16, shared=200, spoil=False) for i in range(2)]
    expect = [g.attention_decode(*args, **kw) for args, kw, _ in cases]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for args, kw, _ in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=streams[0]):
            outs.append([g.attention_decode(*args, **kw) for _ in range(8)])
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for ys, y in zip(outs, expect):
            assert all(torch.equal(x, y) for x in ys)
            for x in ys:
                x.zero_()


def test_refusals(cuda):
    (q, kc, vc, lengths), kw, _ = case(cuda, F16, "int8", [20, 30], 4, 2, 64, page=16, shared=5)
    args = dict(q=q, k=kc, v=vc, lengths=lengths)

    def call(**c):
        return g.attention_decode(*(args | {n: t for n, t in c.items() if n in args}).values(), **(kw | {n: t for n, t in c.items() if n not in args}))

    call()
    for bad in (dict(k_scale=None), dict(v_scale=None), dict(k_scale=kw["k_scale"].half()), dict(v_scale=kw["v_scale"][:1]), dict(q=q.bfloat16()), dict(q=q[0]),
                dict(q=q[:, :3]), dict(q=q[..., :56]), dict(k=kc.half()), dict(v=vc.view(torch.float8_e4m3fn)), dict(k=kc[:1]), dict(lengths=lengths.long()),
                dict(lengths=lengths[:1]), dict(pages=None), dict(pages=kw["pages"][:1]), dict(pages=kw["pages"].long()), dict(softcap=-1.0),
                dict(scale=float("nan")), dict(shared_k=None), dict(shared_k=kw["shared_k"].float()), dict(slopes=torch.ones(3, device=cuda)), dict(k=kc.cpu()),
                dict(k=kc.transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError):  # a cache of 16 bits has no scales, one of 8 needs them
        g.attention_decode(q, kc, vc, lengths, pages=kw["pages"])
    with pytest.raises(RuntimeError, match="no gradient"):
        call(q=q.clone().requires_grad_())
