"""The usual calls of ``attention``, ``attention_decode`` and ``lora_mm_t``, made by the extension.

A small call is bound by the host: checked and packed in Python, one costs 8 us besides its launches, about
as long as its kernels run. ``_g16fast`` does the same for arguments that need no copy, and returns None for
any others; the Python functions then check them one by one, copy or raise. What it needs of this package
(the device, the buffers kept per stream and thread) it asks the functions here for.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _clib, ops
from .kernels import _MAX_CACHED_SCRATCH, SKINNY_MAX_M, scratch_buffer, split_buffers
from .ops import _is_target, _sm_count

_ENTRY_POINTS = ("g16_attention_workspace_bytes", "g16_attention", "g16_attention_decode_workspace_bytes", "g16_attention_decode",
                 "g16_mm_t_raw", "g16_mm_t_direct", "g16_lora_workspace_bytes", "g16_lora_shrink", "g16_lora_expand")


def _ready(device: int) -> int:
    return _sm_count(torch.device("cuda", device)) if _is_target(device) else -1


def _scratch_ptr(device: int, stream: int, nbytes: int) -> int:
    # 0 for a buffer that is not kept between calls (the caller has to hold it)
    if nbytes > _MAX_CACHED_SCRATCH:
        return 0
    return scratch_buffer(torch.device("cuda", device), stream, nbytes).data_ptr()


def _route(device: int, stream: int, M: int, N: int, K: int, x_is_f32: int):
    """How mm_t makes this product, with its buffers (see ``product_route`` in csrc/fastcall.c); None where
    it takes a buffer that is not kept between calls."""
    dev = torch.device("cuda", device)
    lib = _clib.load()
    if M <= SKINNY_MAX_M:
        ksplit, partials, counters = ops._skinny_plan(lib, M, N, K, dev)
        return (0, ksplit, 0.0, 0, 0, *split_buffers(dev, stream, partials, counters))
    if not x_is_f32:
        ops._enable_history(lib, device, stream)
    kind, scratch, ksplit, partials, counters, alone, raw, _ = ops._gemm_route(lib, M, N, K, dev)
    if (alone and ops._direct_thresh()) if x_is_f32 else raw:
        return 2, 1, ops.ROW_SCALE_THRESHOLD, 0, 0, 0, 0, 0, 0
    if scratch > _MAX_CACHED_SCRATCH:
        return None
    ptr = scratch_buffer(dev, stream, scratch).data_ptr() if scratch else 0
    bufs = split_buffers(dev, stream, partials, counters) if kind == "splitk" else (0, 0, 0, 0)
    return (1, ksplit, ops.ROW_SCALE_THRESHOLD, ptr, scratch, *bufs)


def refuse_tangents(name: str, *tensors) -> None:
    """Raise for the first of ``tensors`` (None among them) with a forward-mode tangent. Called only inside a
    ``forward_ad.dual_level()``; outside there are none."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative: pass it the tensors without their tangents")


def refuse_gradients(name: str, *tensors) -> None:
    """Raise for the first of ``tensors`` (None among them) that a gradient is wanted of: the kernels have none."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad()")


_bound = None


def direct():
    """``_g16fast``, bound to torch's types and this package's buffers."""
    global _bound
    if _bound is None:
        fast = _clib.fast()
        fast.bind_torch(torch.float16, torch.float32, torch.int32, torch._C._cuda_getCurrentRawStream, torch.is_grad_enabled, _ready,
                        _scratch_ptr, _route, [_clib.address(n) for n in _ENTRY_POINTS])
        _bound = fast
    return _bound
