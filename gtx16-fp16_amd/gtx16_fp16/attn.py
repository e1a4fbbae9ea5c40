"""Attention around the linear layers of a served model: of prompts (``attention``) and of one token per
request over a cache whose requests may share a prefix (``attention_decode``).

No counterpart in the reference, which replaces linear layers only; types, checks, streams and workspaces
follow this package's products. The kernels are those of ``csrc/attention.hip``.
"""
from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad

from . import _clib
from .direct import direct, refuse_gradients, refuse_tangents
from .kernels import scratch_buffer, stream_handle
from .ops import _is_target, _sm_count

MAX_HEAD_DIM = 128          # G16_ATTENTION_MAX_D
_MAX_STRIDE = 1 << 24       # G16_ATTENTION_MAX_STRIDE: bytes between a key row and the next
_F16, _F32 = torch.float16, torch.float32
_FLT_MAX = torch.finfo(torch.float32).max

# g16_attention_args without its workspace
_ARGS = struct.Struct("@12P13q13i2fi")
assert _ARGS.size == 12 * 8 + 13 * 8 + 16 * 4

_entry: dict[str, tuple[int, int]] = {}


def _entry_points(name: str) -> tuple[int, int]:
    e = _entry.get(name)
    if e is None:
        e = _entry[name] = (_clib.address(name + "_workspace_bytes"), _clib.address(name))
    return e


def _call(name: str, head: bytes, dev: torch.device) -> None:
    fast = _clib.fast()
    size, fn = _entry_points(name)
    stream = stream_handle(dev.index or 0)
    nbytes = fast.args_size(size, head)
    ws = scratch_buffer(dev, stream, nbytes) if nbytes else None
    status = fast.args_call(fn, head, None if ws is None else ws.data_ptr(), nbytes, stream)
    if status != 0:
        _clib.check(status, name)


def _rows(t: torch.Tensor, size: int, d: int, keys: bool) -> torch.Tensor:
    # [.., token, head, d] as the kernels read it: whole 16-byte pieces, the values of a head in a row, keys not
    # closer than their values nor further than the DMA reaches. Anything else is copied, like mm_t's
    # activations.
    st = t.stride()
    ok = (st[-1] == 1 or d == 1) and t.data_ptr() % 16 == 0
    for s in st[:-1]:
        ok = ok and s * size % 16 == 0
    if keys:
        ok = ok and d <= st[-3] and st[-3] * size < _MAX_STRIDE
    return t if ok else torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _ints(name: str, t: torch.Tensor, shape: tuple, dev: torch.device, what: str) -> torch.Tensor:
    if not (t.dtype == torch.int32 and t.shape == shape and t.device == dev):
        raise ValueError(f"{name}: {what} must be an int32 tensor of shape {tuple(shape)} on {dev}")
    return t if t.is_contiguous() else t.contiguous()


def _check(name: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, hq: int, hkv: int, d: int) -> None:
    dev, dt = q.device, q.dtype
    if not (q.is_cuda and (dt == _F16 or dt == _F32) and _is_target(dev.index or 0)):
        raise ValueError(f"{name}: q must be an fp16 or fp32 tensor on a gfx950 device")
    if k.dtype != dt or v.dtype != dt or k.device != dev or v.device != dev:
        raise ValueError(f"{name}: k and v must have q's type and device")
    if k.shape != v.shape or k.shape[-1] != d:
        raise ValueError(f"{name}: k {tuple(k.shape)} and v {tuple(v.shape)} must have one shape and q's head dimension {d}")
    if d % 8 or not 0 < d <= MAX_HEAD_DIM:
        raise ValueError(f"{name}: the head dimension must be a multiple of 8 up to {MAX_HEAD_DIM}, got {d}")
    if hq and (not hkv or hq % hkv):
        raise ValueError(f"{name}: {hq} query heads do not share {hkv} key heads evenly")


def _shared(name: str, shared_k, shared_v, q: torch.Tensor, hkv: int, d: int, size: int):
    """(k, v, keys, strides) of the shared prefix."""
    if (shared_k is None) != (shared_v is None):
        raise ValueError(f"{name}: shared_k and shared_v come together")
    if shared_k is None or shared_k.shape[0] == 0:
        return None, None, 0, (0, 0, 0, 0)
    for t in (shared_k, shared_v):
        if t.dtype != q.dtype or t.device != q.device or t.dim() != 3 or t.shape[1:] != (hkv, d) or t.shape != shared_k.shape:
            raise ValueError(f"{name}: shared_k and shared_v must be [keys, {hkv}, {d}] of q's type and device")
    sk, sv = _rows(shared_k, size, d, True), _rows(shared_v, size, d, True)
    return sk, sv, sk.shape[0], (*sk.stride()[:2], *sv.stride()[:2])


def _slopes(name: str, slopes, hq: int, dev: torch.device):
    if slopes is None:
        return None
    if not (slopes.dtype == _F32 and slopes.shape == (hq,) and slopes.device == dev):
        raise ValueError(f"{name}: slopes must be an fp32 tensor of shape ({hq},) on {dev}")
    return slopes if slopes.is_contiguous() else slopes.contiguous()


def _numbers(name: str, scale, softcap: float, d: int) -> tuple[float, float]:
    scale = d ** -0.5 if scale is None else float(scale)
    softcap = float(softcap or 0.0)
    if scale != scale or _FLT_MAX < abs(scale) < float("inf"):
        raise ValueError(f"{name}: scale must be a number that fp32 holds, got {scale}")
    if not 0.0 <= softcap <= _FLT_MAX or (softcap and not struct.unpack("f", struct.pack("f", softcap))[0]):
        raise ValueError(f"{name}: softcap must be 0 (none) or a positive number that fp32 holds, got {softcap}")
    return scale, softcap


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, q_offsets: torch.Tensor | None = None,
              k_offsets: torch.Tensor | None = None, causal: bool = False, visible: torch.Tensor | None = None,
              shared_k: torch.Tensor | None = None, shared_v: torch.Tensor | None = None, scale: float | None = None,
              softcap: float = 0.0, slopes: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of prompts: for every query row the softmax-weighted mean of the values that it sees.

    q is [sequences, tokens, heads, d] with k and v [sequences, keys, key heads, d], or all three are packed,
    [rows, heads, d], with ``q_offsets`` and ``k_offsets`` (int32, sequences + 1; k_offsets defaults to q_offsets):
    sequence b has rows q_offsets[b] .. q_offsets[b + 1] - 1 and keys k_offsets[b] .. (the document mask; rows
    of no sequence are not written). fp16 or fp32, d a multiple of 8 up to 128; query head h reads key head
    h // (heads / key heads). Strides are free (slices of a fused projection's output are read in place);
    views the kernels cannot read are copied.

    A sequence's rows are its last ones: row t of n, with m keys, stands at position m - n + t of its keys. With
    ``shared_k`` and ``shared_v`` [prefix, key heads, d] every sequence's keys follow that common prefix, and
    positions count from the prefix's first. ``causal``: a row sees the keys up to its own position, and the
    first ``visible[b]`` (int32, one a sequence) in any case (a prefix mask); otherwise all keys of its
    sequence, whatever ``visible`` says. Rows that see no key give zeros; values a row does not see do not reach it, whatever they are.

    Scores are ``scale * q.k`` (scale: 1 / sqrt(d)), then ``softcap * tanh(score / softcap)`` if softcap is not 0,
    then less ``slopes[head]`` (fp32) times the distance of the two positions. Returns q's shape and type,
    contiguous. Scores, softmax and sums are fp32. With fp16 inputs the weights are rounded to fp16 (2^-12 of each at
    most) for their product with the values; fp32 inputs are multiplied with all their bits, whatever their size."""
    if forward_ad._current_level >= 0:
        refuse_tangents("attention", q, k, v, shared_k, shared_v, slopes)
    out = direct().attention(q, k, v, q_offsets, k_offsets, causal, visible, shared_k, shared_v, scale, softcap, slopes)
    if out is not None:
        return out
    packed = q_offsets is not None
    if q.dim() != (3 if packed else 4) or k.dim() != q.dim() or v.dim() != q.dim():
        raise ValueError("attention: q, k and v must be [rows, heads, d] with q_offsets, [sequences, tokens, heads, d] without")
    hq, d = q.shape[-2:]
    hkv = k.shape[-2]
    _check("attention", q, k, v, hq, hkv, d)
    refuse_gradients("attention", q, k, v, shared_k, shared_v, slopes)
    dev, size = q.device, q.element_size()
    if packed:
        if q_offsets.dim() != 1 or q_offsets.shape[0] < 1:
            raise ValueError("attention: q_offsets must hold one value more than there are sequences")
        seqs = q_offsets.shape[0] - 1
        q_offsets = _ints("attention", q_offsets, (seqs + 1,), dev, "q_offsets")
        k_offsets = q_offsets if k_offsets is None else _ints("attention", k_offsets, (seqs + 1,), dev, "k_offsets")
    else:
        if k_offsets is not None or k.shape[0] != q.shape[0]:
            raise ValueError("attention: k and v must have q's sequences, and offsets come with packed tensors")
        seqs = q.shape[0]
    if visible is not None:
        visible = _ints("attention", visible, (seqs,), dev, "visible")
    scale, softcap = _numbers("attention", scale, softcap, d)
    slopes = _slopes("attention", slopes, hq, dev)
    q, k, v = _rows(q, size, d, False), _rows(k, size, d, True), _rows(v, size, d, True)
    sk, sv, shared, shared_strides = _shared("attention", shared_k, shared_v, q, hkv, d, size)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if out.numel() == 0 or seqs == 0:
        return out
    if packed:
        strides = (0, *q.stride()[:2], 0, *k.stride()[:2], 0, *v.stride()[:2])
        q_len, k_len = q.shape[0], k.shape[0]
    else:
        strides = (*q.stride()[:3], *k.stride()[:3], *v.stride()[:3])
        q_len, k_len = q.shape[1], k.shape[1]
    _call("g16_attention",
          _ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(sk), _ptr(sv), out.data_ptr(), _ptr(q_offsets),
                     _ptr(k_offsets), _ptr(visible), 0, 0, _ptr(slopes), *strides, *shared_strides, seqs, q_len, k_len,
                     hq, hkv, d, shared, 1 if causal else 0, 0, 0, 0, 1 if size == 4 else 0, _sm_count(dev), scale,
                     softcap, 0), dev)
    return out


def attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, *,
                     pages: torch.Tensor | None = None, shared_k: torch.Tensor | None = None,
                     shared_v: torch.Tensor | None = None, scale: float | None = None, softcap: float = 0.0,
                     slopes: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one token per request: q [requests, heads, d] over each request's cached keys, its own
    token's among them, and a prefix that all requests share (read once for all of them).

    The caches are [requests, capacity, key heads, d], or, with ``pages`` (int32, [requests, pages of each]),
    [all pages, keys of a page, key heads, d]: key j of request b is key j % page of page pages[b, j // page]. A
    request has ``lengths[b]`` (int32) keys, held to 0 .. its capacity; what lies behind them is not used, whatever
    it holds, and a page number outside the cache reads as zeros. ``shared_k`` and ``shared_v`` [prefix, key heads, d]
    come before every request's own keys. The token stands at its last key's position. Types, heads, scores
    and the result are ``attention``'s; a request without any key gives zeros."""
    if forward_ad._current_level >= 0:
        refuse_tangents("attention_decode", q, k_cache, v_cache, shared_k, shared_v, slopes)
    out = direct().attention_decode(q, k_cache, v_cache, lengths, pages, shared_k, shared_v, scale, softcap, slopes)
    if out is not None:
        return out
    if q.dim() != 3 or k_cache.dim() != 4 or v_cache.dim() != 4 or lengths.dim() != 1:
        raise ValueError("attention_decode: q must be [requests, heads, d], the caches have four dimensions, lengths one")
    seqs, hq, d = q.shape
    hkv = k_cache.shape[2]
    _check("attention_decode", q, k_cache, v_cache, hq, hkv, d)
    refuse_gradients("attention_decode", q, k_cache, v_cache, shared_k, shared_v, slopes)
    dev, size = q.device, q.element_size()
    lengths = _ints("attention_decode", lengths, (seqs,), dev, "lengths")
    page, max_pages = k_cache.shape[1], 0
    if pages is not None:
        if pages.dim() != 2:
            raise ValueError("attention_decode: pages must be [requests, pages of each]")
        max_pages = pages.shape[1]
        pages = _ints("attention_decode", pages, (seqs, max_pages), dev, "pages")
        capacity = page * max_pages
    else:
        if k_cache.shape[0] != seqs:
            raise ValueError("attention_decode: without pages, the caches' first dimension is the requests")
        capacity = page
    scale, softcap = _numbers("attention_decode", scale, softcap, d)
    slopes = _slopes("attention_decode", slopes, hq, dev)
    q, k, v = _rows(q, size, d, False), _rows(k_cache, size, d, True), _rows(v_cache, size, d, True)
    sk, sv, shared, shared_strides = _shared("attention_decode", shared_k, shared_v, q, hkv, d, size)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if out.numel() == 0:
        return out
    _call("g16_attention_decode",
          _ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(sk), _ptr(sv), out.data_ptr(), 0, 0, 0,
                     lengths.data_ptr(), _ptr(pages) if capacity else 0, _ptr(slopes), q.stride(0), 0, q.stride(1), *k.stride()[:3], *v.stride()[:3],
                     *shared_strides, seqs, 1, capacity, hq, hkv, d, shared, 0, page, max_pages, k.shape[0],
                     1 if size == 4 else 0, _sm_count(dev), scale, softcap, 0), dev)
    return out
