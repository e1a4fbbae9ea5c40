"""Rotary positions of queries and keys, by one axis or several (``rotary``).

No counterpart in the reference; types, checks and streams follow ``attention``. The kernel is that of
``csrc/rotary.hip``.
"""
from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad

from . import _clib
from .attn import _ints, _rows
from .direct import direct, refuse_gradients, refuse_tangents
from .kernels import stream_handle
from .ops import _is_target

MAX_AXES = 4         # G16_ROTARY_MAX_AXES
MAX_HEAD_DIM = 4096  # G16_ROTARY_MAX_D

# g16_rotary_args
_ARGS = struct.Struct("@4P3q12i")
assert _ARGS.size == 4 * 8 + 3 * 8 + 12 * 4


def rotary(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, *, sections: tuple[int, ...] | None = None,
           interleaved: bool = False) -> torch.Tensor:
    """x with its heads' pairs of values turned by their rows' positions: pair i of a row at position p by the angle
    p * freqs[i], (a, b) -> (a cos - b sin, b cos + a sin).

    x is [rows, heads, d] or [sequences, tokens, heads, d], fp16 or fp32, d a multiple of 8 up to 4096; strides are free (the
    queries and keys of a fused projection's output, together, are read in place); views the kernel cannot read are
    copied. freqs fp32 [pairs], 2 * pairs up to d: pair i is the values i and i + pairs of a head, or, ``interleaved``,
    2 i and 2 i + 1, and values from 2 * pairs on stay as they are. positions int32, one a row (x's shape without the last
    two dimensions), of any sign: the negative ones turn back. With ``sections`` (pairs of each axis, up to 4 axes,
    pairs in all) positions are [axes, ..one a row..]: pairs 0 .. sections[0] - 1 go by the first axis, the next
    sections[1] by the second, and so on (time, height and width of images and video).

    Returns x's shape and type, contiguous. The angle is the exact product less whole turns (far positions keep their
    places; angles stay below 2^51); its cosine and sine, to 1e-7, and the rotation are fp32."""
    if forward_ad._current_level >= 0:
        refuse_tangents("rotary", x, freqs)
    out = direct().rotary(x, positions, freqs, sections, interleaved)
    if out is not None:
        return out
    dev, dt = x.device, x.dtype
    if not (x.is_cuda and (dt == torch.float16 or dt == torch.float32) and _is_target(dev.index or 0)):
        raise ValueError("rotary: x must be an fp16 or fp32 tensor on a gfx950 device")
    if x.dim() not in (3, 4):
        raise ValueError("rotary: x must be [rows, heads, d] or [sequences, tokens, heads, d]")
    lead, (heads, d) = x.shape[:-2], x.shape[-2:]
    if d % 8 or not 0 < d <= MAX_HEAD_DIM:
        raise ValueError(f"rotary: the head dimension must be a multiple of 8 up to {MAX_HEAD_DIM}, got {d}")
    if not (freqs.dtype == torch.float32 and freqs.dim() == 1 and freqs.device == dev):
        raise ValueError(f"rotary: freqs must be an fp32 vector on {dev}")
    pairs = freqs.shape[0]
    if 2 * pairs > d:
        raise ValueError(f"rotary: {pairs} pairs do not fit heads of {d} values")
    if sections is None:
        axes, parts, shape = 1, (pairs,), lead
    else:
        parts = tuple(int(n) for n in sections)
        axes = len(parts)
        if not 1 <= axes <= MAX_AXES or min(parts) < 0 or sum(parts) != pairs:
            raise ValueError(f"rotary: sections must be 1 to {MAX_AXES} numbers of pairs that add up to {pairs}, got {parts}")
        shape = (axes, *lead)
    positions = _ints("rotary", positions, shape, dev, "positions")
    refuse_gradients("rotary", x, freqs)
    x = _rows(x, x.element_size(), d, False)
    out = torch.empty(x.shape, dtype=dt, device=dev)
    if out.numel() == 0:
        return out
    freqs = freqs.contiguous()
    seqs, tokens = (1, lead[0]) if len(lead) == 1 else lead
    st = x.stride()
    head = _ARGS.pack(x.data_ptr(), out.data_ptr(), positions.data_ptr(), freqs.data_ptr(), st[0] if len(lead) == 2 else 0, st[-3], st[-2],
                      seqs, tokens, heads, d, pairs, axes, *parts, *(0,) * (MAX_AXES - axes), 1 if interleaved else 0, 1 if dt == torch.float32 else 0)
    status = _clib.fast().struct_call(_clib.address("g16_rotary"), head, stream_handle(dev.index or 0))
    if status != 0:
        _clib.check(status, "rotary")
    return out
