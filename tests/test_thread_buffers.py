"""CPU test of the buffers that a call's launches meet in: threads that share a stream have their own."""
from __future__ import annotations

import threading

import pytest
import torch

from gtx16_fp16 import kernels

CPU = torch.device("cpu")


@pytest.fixture
def fresh():
    kernels.release_workspaces()
    yield
    kernels.release_workspaces()


def in_threads(n, fn):
    """fn() in n threads that are all alive at once."""
    out, gate = [None] * n, threading.Barrier(n)

    def body(i):
        gate.wait()
        out[i] = fn()
        gate.wait()

    threads = [threading.Thread(target=body, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return out


def test_threads_on_one_stream_have_their_own_buffers(fresh):
    scratch = in_threads(6, lambda: kernels.scratch_buffer(CPU, 7, 1000).data_ptr())
    assert len(set(scratch)) == 6
    split = in_threads(6, lambda: kernels.split_buffers(CPU, 7, 1000, 64))
    assert len({s[0] for s in split}) == 6 and len({s[2] for s in split}) == 6


def test_a_thread_keeps_its_buffers(fresh):
    def twice():
        a, b = (kernels.scratch_buffer(CPU, 7, n).data_ptr() for n in (1000, 900))
        s, t = (kernels.split_buffers(CPU, 7, n, 64) for n in (1000, 900))
        return a == b and s == t and kernels.scratch_buffer(CPU, 8, 1000).data_ptr() != a

    assert all(in_threads(4, twice)) and twice()
