"""GPU test: threads that call on one stream, each call of several launches, get what they would get alone."""
from __future__ import annotations

import threading

import pytest
import torch

import gtx16_fp16 as g

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def calls(dev):
    gen = torch.Generator().manual_seed(0)
    rand = lambda *s, dtype=F16, by=1.0: (by * torch.randn(*s, generator=gen)).to(dtype).to(dev)  # noqa: E731
    q, k, v = rand(60, 4, 128), rand(4000, 2, 128), rand(4000, 2, 128)
    q_off, k_off = (torch.tensor([0, n], dtype=torch.int32, device=dev) for n in (60, 4000))
    cache, n = rand(3, 2000, 2, 128), torch.tensor([2000, 17, 900], dtype=torch.int32, device=dev)
    x, w, b = rand(64, 4096, dtype=F32), rand(4096, 1024, by=0.02), rand(1024, dtype=F32)
    big, wide = rand(2304, 256, dtype=F32), rand(256, 4096, by=0.05)
    down, up, index = rand(6, 16, 4096, by=0.02), rand(6, 1024, 16, by=0.2), torch.arange(64, dtype=torch.int32, device=dev) % 6
    x16, odd = x.half(), rand(4096, 64).t()  # (the last: not contiguous, so the call is made in Python)
    return [lambda: g.attention(q, k, v, q_offsets=q_off, k_offsets=k_off, causal=True),
            lambda: g.attention_decode(q[:3], cache, cache, n, shared_k=k, shared_v=v),
            lambda: g.mm_t(x, w, b),
            lambda: g.mm_t(big, wide),
            lambda: g.lora_mm_t(x16, w, down, up, index, bias=b, out_dtype=F16),
            lambda: g.lora_mm_t(odd, w, down, up, index, bias=b, out_dtype=F16)]


def test_threads_share_a_stream(cuda):
    fns = calls(cuda)
    with torch.no_grad():
        want = [fn() for fn in fns]
    torch.cuda.synchronize()
    wrong, gate = [], threading.Barrier(6)

    def body(i):
        gate.wait()
        with torch.no_grad():
            got = [(j, fns[j]()) for r in range(60) for j in [(i + r) % len(fns)]]
        torch.cuda.synchronize()
        wrong.extend(j for j, y in got if not torch.equal(y, want[j]))

    threads = [threading.Thread(target=body, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, f"calls {sorted(set(wrong))} differed"


def test_a_capture_by_a_thread_without_buffers(cuda):
    # The thread that warmed the stream up is not the one that captures: the graph takes buffers of its own, which eager
    # calls of that thread, before and after replays, do not use.
    fns = calls(cuda)[:5]
    with torch.no_grad():
        want = [fn() for fn in fns]
    torch.cuda.synchronize()
    wrong = []

    def body():
        s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.stream(s):
            with torch.cuda.graph(graph, stream=s):
                captured = [fn() for fn in fns]
            for r in range(4):
                eager = [fn() for fn in fns]
                torch.cuda.synchronize()
                wrong.extend(("eager", r, j) for j, y in enumerate(eager) if not torch.equal(y, want[j]))
                for y in captured:
                    y.zero_()
                graph.replay()
                torch.cuda.synchronize()
                wrong.extend(("replay", r, j) for j, y in enumerate(captured) if not torch.equal(y, want[j]))

    t = threading.Thread(target=body)
    t.start()
    t.join()
    assert not wrong, wrong
