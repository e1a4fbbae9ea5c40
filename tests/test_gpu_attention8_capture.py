"""attention_decode over a cache in 8 bits, captured: what a graph's replays use besides the result stays the call's own."""
from __future__ import annotations

import ctypes

import pytest
import torch

import gtx16_fp16 as g
from test_gpu_attention8 import F16, F32, case

pytestmark = pytest.mark.gpu


def places(t):
    s = t.untyped_storage()
    return s.data_ptr(), s.data_ptr() + s.nbytes()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_the_workspace_lives_with_the_result(cuda, dtype):
    args, kw, _ = case(cuda, dtype, "int8", [900, 3000], 8, 2, 72, page=16, spoil=False)
    want = g.attention_decode(*args, **kw)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            ys = [g.attention_decode(*args, **kw) for _ in range(3)]
    own = 2 * 8 * 72 * ys[0].element_size()
    for y in ys:
        begin, end = places(y)
        # the parts of two requests' sums in 72 of 128 places for 8 rows at least
        assert y.shape == want.shape and y.is_contiguous() and y._base is None and y.data_ptr() == begin and end - begin >= own + 2 * 8 * 128 * 4
        for other in ys:
            assert other is y or end <= places(other)[0] or places(other)[1] <= begin
    for _ in range(3):
        for y in ys:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in ys)


def test_a_capture_that_torch_does_not_know(cuda):
    # begun through HIP itself: memory comes from where all tensors' does, and what is freed after the call goes to others
    hip = ctypes.CDLL("libamdhip64.so.7")

    def ok(status):
        assert status == 0, status

    args, kw, _ = case(cuda, F16, "int8", [900, 3000], 8, 2, 128, page=16, shared=100, spoil=False)
    want = g.attention_decode(*args, **kw)
    side, graph, run = torch.cuda.Stream(), ctypes.c_void_p(), ctypes.c_void_p()
    torch.cuda.synchronize()
    stream = ctypes.c_void_p(side.cuda_stream)
    with torch.cuda.stream(side):
        g.attention_decode(*args, **kw)
        torch.cuda.synchronize()
        ok(hip.hipStreamBeginCapture(stream, ctypes.c_int(2)))  # relaxed: allocations are allowed
        y = g.attention_decode(*args, **kw)
        ok(hip.hipStreamEndCapture(stream, ctypes.byref(graph)))
        ok(hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)))
        others = [torch.full((n,), 0x5a, dtype=torch.uint8, device=cuda) for n in (1 << 10, 1 << 14, 1 << 16, 1 << 18, 1 << 20, 1 << 22, 1 << 24) for _ in range(4)]
        begin, end = places(y)
        assert all(places(t)[1] <= begin or end <= places(t)[0] for t in others)
        for _ in range(3):
            y.zero_()
            ok(hip.hipGraphLaunch(run, stream))
            torch.cuda.synchronize()
            assert torch.equal(y, want) and all(bool((t == 0x5a).all()) for t in others)
        ok(hip.hipGraphExecDestroy(run))
        ok(hip.hipGraphDestroy(graph))


def test_in_inference_mode(cuda):
    args, kw, _ = case(cuda, F16, "e4m3", [900, 3000], 8, 2, 64, page=16, spoil=False)
    want = g.attention_decode(*args, **kw)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.inference_mode(), torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            y = g.attention_decode(*args, **kw)
        for _ in range(2):
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)
