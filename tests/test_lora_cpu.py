"""CPU tests of the adapters' entry points: what the library rejects before a launch, and the workspace it asks for."""
from __future__ import annotations

import weakref

import pytest
import torch

from gtx16_fp16 import _clib, lora

NAMES = ["x", "down", "up", "index", "scale", "y", "out", "M", "K", "N", "rank", "adapters", "x_is_f32", "out_is_f16", "num_cus"]
SHAPE, ALIGN, NULL, WORKSPACE, DTYPE = -1, -2, -3, -4, -6


def head(**changes) -> bytes:
    v = dict(x=4096, down=4096, up=4096, index=4096, scale=0, y=4096, out=4096, M=20, K=64, N=64, rank=16, adapters=3, x_is_f32=0,
             out_is_f16=1, num_cus=256)
    v.update(changes)
    return lora._ARGS.pack(*(v[n] for n in NAMES))


def call(name, **changes):
    return _clib.fast().args_call(_clib.address(name), head(**changes), None, 0, 0)


def size(**changes):
    return _clib.fast().args_size(_clib.address("g16_lora_workspace_bytes"), head(**changes))


@pytest.mark.parametrize("name", ["g16_lora_shrink", "g16_lora_expand"])
@pytest.mark.parametrize("changes,status", [
    (dict(M=-1), SHAPE), (dict(K=60), SHAPE), (dict(N=68), SHAPE), (dict(rank=12), SHAPE), (dict(rank=136), SHAPE), (dict(adapters=-1), SHAPE),
    (dict(x_is_f32=2), DTYPE), (dict(out_is_f16=3), DTYPE), (dict(x=0), NULL), (dict(down=0), NULL), (dict(up=0), NULL), (dict(index=0), NULL),
    (dict(y=0), NULL), (dict(out=0), NULL), (dict(x=4098), ALIGN), (dict(up=4100), ALIGN), (dict(y=4104), ALIGN), (dict(), WORKSPACE),
])
def test_rejected_before_a_launch(name, changes, status):
    assert call(name, **changes) == status
    if status != WORKSPACE:
        assert size(**changes) == 0


def test_nothing_to_do_is_no_error():
    for name in ("g16_lora_shrink", "g16_lora_expand"):
        assert call(name, M=0) == 0
        assert call(name, N=0) == 0
    assert call("g16_lora_shrink", rank=0) == 0
    assert _clib.load().g16_lora_shrink(None, None) == NULL
    assert _clib.load().g16_lora_expand(None, None) == NULL


def test_few_rows_need_no_workspace():
    assert size(M=1, K=8, rank=8) == 0


@pytest.mark.parametrize("M,K,rank", [(20, 4096, 16), (300, 4096, 40), (5000, 512, 128)])
def test_workspace_holds_whole_splits(M, K, rank):
    n = size(M=M, K=K, rank=rank)
    assert n > 0 and n % (4 * M * rank) == 0


@pytest.mark.parametrize("name", ["g16_lora_shrink", "g16_lora_expand"])
@pytest.mark.parametrize("side", ["K", "N"])
def test_sides_past_32_bit_offsets_are_rejected(name, side):
    assert call(name, **{side: lora.MAX_SIDE + 8}) == SHAPE
    assert size(**{side: lora.MAX_SIDE}) > 0


def test_the_workspace_lives_until_both_products_are_enqueued(monkeypatch):
    # past the size that is kept between calls, nothing but the call holds it
    made, seen = [], []

    def scratch(dev, stream, nbytes):
        t = torch.empty(nbytes, dtype=torch.uint8)
        made.append(weakref.ref(t))
        return t

    class Fast:
        lora_mm_t = staticmethod(lambda *args: None)
        args_size = staticmethod(lambda fn, head: 20 << 20)

        @staticmethod
        def args_call(fn, head, ws, nbytes, stream):
            seen.append(made[0]() is not None and made[0]().data_ptr() == ws and nbytes == 20 << 20)
            return 0

    monkeypatch.setattr(lora, "direct", Fast)
    monkeypatch.setattr(lora._clib, "fast", Fast)
    monkeypatch.setattr(lora, "scratch_buffer", scratch)
    monkeypatch.setattr(lora, "stream_handle", lambda index: 0)
    monkeypatch.setattr(lora, "_sm_count", lambda dev: 256)
    monkeypatch.setattr(lora, "mm_t", lambda x, w, bias, dtype: torch.zeros(x.shape[0], w.shape[1], dtype=dtype))
    x, w = torch.zeros(4, 8, dtype=torch.float16), torch.zeros(8, 8, dtype=torch.float16)
    index = torch.zeros(4, dtype=torch.int32)
    lora.lora_mm_t(x, w, torch.zeros(1, 8, 8, dtype=torch.float16), torch.zeros(1, 8, 8, dtype=torch.float16), index)
    assert seen == [True, True] and made[0]() is None


def test_expand_rejects_adapters_of_rank_0():
    # (few rows, where expand would compute both products, and many)
    for M in (1, 20, 5000):
        for out_is_f16 in (0, 1):
            assert call("g16_lora_expand", rank=0, M=M, out_is_f16=out_is_f16) == SHAPE
    assert call("g16_lora_expand", rank=0, M=0) == 0


def test_rows_past_32_bits_are_rejected():
    for name in ("g16_lora_shrink", "g16_lora_expand"):
        assert call(name, M=(1 << 31) - 2) == SHAPE
        assert call(name, M=1 << 30, K=8, N=8, rank=8) == WORKSPACE
