"""A key's way, whole: rotated, written in 8 bits, read by single tokens and, as rows, by a prompt's next chunk; and the example that
serves so."""
from __future__ import annotations

import importlib.util
import threading
from pathlib import Path

import pytest
import torch

import gtx16_fp16 as g
from _attention import check, prompts
from _cache8 import empty, numbers
from test_gpu_attention8 import case, expected

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def freqs_of(pairs, device):
    return torch.tensor([10000.0 ** (-i / pairs) for i in range(pairs)], dtype=F32, device=device)


def held(cache, slots):
    """The keys and values of `slots` as doubles on the CPU, from the codes themselves."""
    heads, d = cache[0].shape[2:]
    return tuple((numbers(c).reshape(-1, heads, d) * s.cpu().double().reshape(-1, heads, 1))[slots.cpu().long()] for c, s in zip(cache[:2], cache[2:]))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 64, 16), (4, 4, 128, 24)])
def test_a_keys_way(cuda, code, dtype, hq, hkv, d, page):
    gen = torch.Generator().manual_seed(0)
    lengths, per = [37, 1, 64], 5
    cache = empty(3 * per, page, hkv, d, code, cuda)
    table = torch.randperm(3 * per, generator=gen).view(3, per).to(torch.int32)
    freqs = freqs_of(d // 2, cuda)
    slots_of = lambda b, at: table[b].long()[at // page] * page + at % page  # noqa: E731
    # the prompts, packed
    fused = torch.randn(sum(lengths), hq + 2 * hkv, d, generator=gen).to(dtype).to(cuda)
    at = torch.cat([torch.arange(n) for n in lengths])
    slots = torch.cat([slots_of(b, torch.arange(n)) for b, n in enumerate(lengths)]).to(torch.int32).to(cuda)
    qk = g.rotary(fused[:, :hq + hkv], at.to(torch.int32).to(cuda), freqs)
    g.cache_write(qk[:, hq:], fused[:, hq + hkv:], *cache, slots)
    for step in range(3):  # tokens after them
        fused = torch.randn(3, hq + 2 * hkv, d, generator=gen).to(dtype).to(cuda)
        now = torch.tensor(lengths)
        qk = g.rotary(fused[:, :hq + hkv], now.to(torch.int32).to(cuda), freqs)
        new = torch.stack([slots_of(b, n) for b, n in enumerate(now)]).to(torch.int32).to(cuda)
        g.cache_write(qk[:, hq:], fused[:, hq + hkv:], *cache, new)
        lengths = [n + 1 for n in lengths]
        y = g.attention_decode(qk[:, :hq], cache[0], cache[1], torch.tensor(lengths, dtype=torch.int32, device=cuda), pages=table.to(cuda),
                               k_scale=cache[2], v_scale=cache[3])
        keys = [held(cache, slots_of(b, torch.arange(n))) for b, n in enumerate(lengths)]
        check(y, expected(qk[:, :hq].cpu(), [k for k, _ in keys], [v for _, v in keys], lengths))
    # the next chunk of the first prompt, after what the cache has of it
    n, new = lengths[0], 20
    every = slots_of(0, torch.arange(n)).to(torch.int32).to(cuda)
    k, v = g.cache_read(*cache, every, out_dtype=dtype)
    assert all(torch.equal(a.cpu(), b.float().to(dtype)) for a, b in zip((k, v), held(cache, every)))
    fused = torch.randn(new, hq + 2 * hkv, d, generator=gen).to(dtype).to(cuda)
    qk = g.rotary(fused[:, :hq + hkv], torch.arange(n, n + new, dtype=torch.int32, device=cuda), freqs)
    k, v = torch.cat((k, qk[:, hq:])), torch.cat((v, fused[:, hq + hkv:]))
    off = lambda m: torch.tensor([0, m], dtype=torch.int32, device=cuda)  # noqa: E731
    y = g.attention(qk[:, :hq], k, v, q_offsets=off(new), k_offsets=off(n + new), causal=True)
    check(y, prompts(qk[:, :hq].cpu(), k.cpu(), v.cpu(), [new], [n + new], causal=True))


def test_a_step_replayed(cuda):
    # rotary, write and attention of a step as one graph, next to eager steps on another cache
    hq, hkv, d, page, n = 8, 2, 128, 16, 5
    caches = [empty(n * 4, page, hkv, d, "int8", cuda) for _ in range(2)]
    table = torch.randperm(n * 4).view(n, 4).to(torch.int32).to(cuda)
    freqs, lengths = freqs_of(d // 2, cuda), torch.zeros(n, dtype=torch.int32, device=cuda)
    fused = torch.randn(n, hq + 2 * hkv, d, device=cuda).half()

    def step(cache):
        qk = g.rotary(fused[:, :hq + hkv], lengths, freqs)
        slots = (table.gather(1, (lengths // page).long()[:, None])[:, 0] * page + lengths % page).to(torch.int32)
        g.cache_write(qk[:, hq:], fused[:, hq + hkv:], *cache, slots)
        return g.attention_decode(qk[:, :hq], cache[0], cache[1], lengths + 1, pages=table, k_scale=cache[2], v_scale=cache[3])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(caches[0])
        with torch.cuda.graph(graph, stream=side):
            y = step(caches[0])
    torch.cuda.current_stream().wait_stream(side)
    for i in range(40):
        fused.copy_(torch.randn_like(fused))
        graph.replay()
        z = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(y, z), i
        lengths.add_(1)


def test_threads_on_one_stream(cuda):
    # splits' sums of two threads' calls do not meet
    given = [case(cuda, F16, "int8", [900 + 300 * i, 40, 1500], 8, 2, 128, page=16, seed=i) for i in range(2)]
    alone = [g.attention_decode(*args, **kw) for args, kw, _ in given]
    wrong = []

    def body(i):
        args, kw, _ = given[i]
        for _ in range(60):
            y = g.attention_decode(*args, **kw)
            if not torch.equal(y, alone[i]):
                wrong.append(i)

    threads = [threading.Thread(target=body, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("argv", [["--rotary"], ["--cache", "int8"], ["--rotary", "--cache", "int8"], ["--rotary", "--cache", "e4m3"]])
def test_the_serving_example(cuda, argv):
    path = Path(__file__).resolve().parents[1] / "examples" / "serve_adapters.py"
    spec = importlib.util.spec_from_file_location("serve_adapters", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    # fp16 activations: as in test_gpu_serving. Codes are off by up to 1/254 of a head's largest value, or 2^-4 of a value.
    least = {"int8": 0.05, "e4m3": 0.2}.get(argv[-1], 2e-2)
    assert mod.main(["--layers", "2", "--requests", "5", "--tokens", "20", "--system", "70", *argv, "--check"]) < least
