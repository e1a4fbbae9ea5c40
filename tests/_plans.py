"""Which shape of workgroup (query rows) and how many key splits a prompt takes, as the library plans it."""
from __future__ import annotations

import ctypes

from gtx16_fp16 import _clib, attn


def prompt_plan(rows, keys, hq, hkv, d, f32=False, sequences=1, packed=True, causal=False, shared=0, cus=256):
    """(rows of a workgroup, splits); rows and keys: of all sequences where packed, else of each."""
    # (strides and addresses the checks accept; nothing is launched)
    at, tok = 4096, hkv * d
    strides = (0, hq * d, d, keys * tok, tok, d, keys * tok, tok, d, tok, d, tok, d)
    head = attn._ARGS.pack(at, at, at, at, at, at, *((at, at) if packed else (0, 0)), 0, 0, 0, 0, *strides, sequences, rows, keys, hq, hkv, d,
                           shared, int(causal), 0, 0, 0, int(f32), cus, 1.0, 0.0, 0)
    tile, splits = ctypes.c_int(), ctypes.c_int()
    status = _clib.load().g16_attention_plan(ctypes.create_string_buffer(head + bytes(16)), ctypes.byref(tile), ctypes.byref(splits))
    assert status == 0, status
    return tile.value, splits.value
