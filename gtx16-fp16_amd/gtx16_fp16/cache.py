"""A cache of keys and values in 8 bits: written as tokens arrive (``cache_write``), read back as rows
(``cache_read``) and by ``attention_decode``.

No counterpart in the reference; types, checks and streams follow ``attention``. The kernels are those of
``csrc/cache.hip``.
"""
from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _clib
from .attn import MAX_HEAD_DIM, _ints, _rows
from .direct import direct, refuse_gradients, refuse_tangents
from .kernels import stream_handle
from .ops import _is_target

CODES = {torch.int8: 1, torch.float8_e4m3fn: 2}  # G16_CODE_INT8, G16_CODE_E4M3

# g16_cache_args
_ARGS = struct.Struct("@7P16q8i")
assert _ARGS.size == 7 * 8 + 16 * 8 + 8 * 4


def check_cache(name: str, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> int:
    """The code of a cache that the kernels read in place; raises for any other."""
    dev, shape = k_cache.device, k_cache.shape
    code = CODES.get(k_cache.dtype)
    if code is None or v_cache.dtype != k_cache.dtype or k_cache.dim() != 4 or v_cache.shape != shape or v_cache.device != dev:
        raise ValueError(f"{name}: k_cache and v_cache must be int8 or float8_e4m3fn, [pages, page, heads, d], both of one type, shape and device")
    for t in (k_scale, v_scale):
        if not (t.dtype == torch.float32 and t.shape == shape[:3] and t.device == dev):
            raise ValueError(f"{name}: k_scale and v_scale must be fp32 tensors of shape {tuple(shape[:3])} on {dev}")
    d = shape[3]
    if d % 8 or not 0 < d <= MAX_HEAD_DIM:
        raise ValueError(f"{name}: the head dimension must be a multiple of 8 up to {MAX_HEAD_DIM}, got {d}")
    for t in (k_cache, v_cache):
        st = t.stride()
        if st[3] != 1 or (st[0] | st[1] | st[2] | t.data_ptr()) % 8:
            raise ValueError(f"{name}: a head's codes must be contiguous and start at a multiple of 8 bytes")
    return code


def _call(name: str, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
          v_scale: torch.Tensor, slots: torch.Tensor, code: int) -> None:
    pages, page, hkv, d = k_cache.shape
    dev = k_cache.device
    if pages * page > (1 << 31) - 1:
        raise ValueError(f"{name}: a cache may hold up to 2^31 - 1 tokens, got {pages * page}")
    head = _ARGS.pack(k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                      slots.data_ptr(), *k.stride()[:2], *v.stride()[:2], *k_cache.stride()[:3], *v_cache.stride()[:3], *k_scale.stride(),
                      *v_scale.stride(), slots.shape[0], pages, page, hkv, d, code, 1 if k.dtype == torch.float32 else 0, 0)
    status = _clib.fast().struct_call(_clib.address("g16_" + name), head, stream_handle(dev.index or 0))
    if status != 0:
        _clib.check(status, name)


def cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                v_scale: torch.Tensor, slots: torch.Tensor) -> None:
    """Write the keys and values of new tokens to their slots of a cache in 8 bits.

    k and v [.., heads, d], fp16 or fp32; the caches [pages, page, heads, d], int8 or float8_e4m3fn, their scales fp32
    [pages, page, heads] (a padded cache is [requests, capacity, heads, d]); slots int32, one a token, k's shape without
    the last two dimensions: token t of page p is slot p * page + t. A token whose slot is negative or past the cache is not
    written; of several with one slot the last one is. d a multiple of 8 up to 128; strides are free, but a head's codes
    are contiguous and start at a multiple of 8 bytes. Nothing else of the cache changes. To autograd all four tensors are
    changed in place.

    Every token's head has a scale of its own. int8: scale = max|x| / 127, codes nearest to x * (127 / max|x|), ties to
    even. e4m3: the smallest power of two that brings the values to at most 448 (another scale would gain a
    floating format nothing, and so the division is exact), codes nearest, ties to even. Values all below
    2^-96 are written as zeros; a head with a value that is not finite reads as NaN throughout."""
    name = "cache_write"
    if forward_ad._current_level >= 0:
        refuse_tangents(name, k, v, k_cache, v_cache, k_scale, v_scale)
    if direct().cache_write(k, v, k_cache, v_cache, k_scale, v_scale, slots):
        increment_version((k_cache, v_cache, k_scale, v_scale))  # (written in place, as autograd has to know)
        return
    dev = k.device
    if not (k.is_cuda and k.dtype in (torch.float16, torch.float32) and v.dtype == k.dtype and v.device == dev and _is_target(dev.index or 0)):
        raise ValueError(f"{name}: k and v must be fp16 or fp32 tensors of one type on one gfx950 device")
    code = check_cache(name, k_cache, v_cache, k_scale, v_scale)
    hkv, d = k_cache.shape[2:]
    if k.dim() < 2 or k.shape != v.shape or k.shape[-2:] != (hkv, d) or k_cache.device != dev:
        raise ValueError(f"{name}: k {tuple(k.shape)} and v {tuple(v.shape)} must be [.., {hkv}, {d}] on the cache's device")
    for t in (k_cache, v_cache, k_scale, v_scale):
        if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise ValueError(f"{name}: the cache's tokens must have memory of their own")
    slots = _ints(name, slots, k.shape[:-2], dev, "slots").reshape(-1)
    refuse_gradients(name, k, v, k_cache, v_cache, k_scale, v_scale)
    if k.numel() == 0 or k_cache.numel() == 0:
        return
    size = k.element_size()
    k, v = (_rows(t.reshape(-1, hkv, d), size, d, False) for t in (k, v))
    _call(name, k, v, k_cache, v_cache, k_scale, v_scale, slots, code)
    increment_version((k_cache, v_cache, k_scale, v_scale))


def cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, slots: torch.Tensor, *,
               out_dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that a cache in 8 bits (``cache_write``) holds at ``slots`` (int32, any shape), contiguous
    [*slots.shape, heads, d] in fp16 or fp32: code * scale, rounded once. A slot that is negative or past the cache reads
    as zeros. ``attention`` takes them as the keys of a prompt's earlier chunks."""
    name = "cache_read"
    if forward_ad._current_level >= 0:
        refuse_tangents(name, k_cache, v_cache, k_scale, v_scale)
    both = direct().cache_read(k_cache, v_cache, k_scale, v_scale, slots, out_dtype)
    if both is not None:
        return both
    if out_dtype not in (torch.float32, torch.float16):
        raise ValueError(f"out_dtype must be float32 or float16, got {out_dtype}")
    dev = k_cache.device
    if not (k_cache.is_cuda and _is_target(dev.index or 0)):
        raise ValueError(f"{name}: the cache must be on a gfx950 device")
    code = check_cache(name, k_cache, v_cache, k_scale, v_scale)
    slots = _ints(name, slots, slots.shape, dev, "slots")
    refuse_gradients(name, k_cache, v_cache, k_scale, v_scale)
    k, v = (torch.empty(*slots.shape, *k_cache.shape[2:], dtype=out_dtype, device=dev) for _ in "kv")
    if k.numel() != 0:
        hkv, d = k_cache.shape[2:]
        _call(name, k.view(-1, hkv, d), v.view(-1, hkv, d), k_cache, v_cache, k_scale, v_scale, slots.view(-1), code)
    return k, v
