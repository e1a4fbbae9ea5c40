"""The usual calls of ``attention``, ``attention_decode`` and ``lora_mm_t``, made by the extension.

A small call is bound by the host: checked and packed in Python, one costs 8 us besides its launches, about
as long as its kernels run. ``_g16fast`` does the same for arguments that need no copy, and returns None for
any others; the Python functions then check them one by one, copy or raise. What it needs of this package
(the device, the buffers kept per stream) it asks the functions here for.
"""
from __future__ import annotations

import torch

from . import _clib
from .kernels import _MAX_CACHED_SCRATCH, scratch_buffer, split_buffers
from .ops import _is_target, _sm_count

_ENTRY_POINTS = ("g16_attention_workspace_bytes", "g16_attention", "g16_attention_decode_workspace_bytes", "g16_attention_decode",
                 "g16_skinny_plan", "g16_skinny_workspace_bytes", "g16_skinny_counter_bytes", "g16_lora_workspace_bytes",
                 "g16_lora_shrink", "g16_lora_expand")


def _ready(device: int) -> int:
    return _sm_count(torch.device("cuda", device)) if _is_target(device) else -1


def _scratch_ptr(device: int, stream: int, nbytes: int) -> int:
    # 0 for a buffer that is not kept between calls (the caller has to hold it)
    if nbytes > _MAX_CACHED_SCRATCH:
        return 0
    return scratch_buffer(torch.device("cuda", device), stream, nbytes).data_ptr()


def _split_ptrs(device: int, stream: int, partial_bytes: int, counter_bytes: int) -> tuple:
    return split_buffers(torch.device("cuda", device), stream, partial_bytes, counter_bytes)


_bound = None


def direct():
    """``_g16fast``, bound to torch's types and this package's buffers."""
    global _bound
    if _bound is None:
        fast = _clib.fast()
        fast.bind_torch(torch.float16, torch.float32, torch.int32, torch._C._cuda_getCurrentRawStream, torch.is_grad_enabled, _ready,
                        _scratch_ptr, _split_ptrs, [_clib.address(n) for n in _ENTRY_POINTS])
        _bound = fast
    return _bound
