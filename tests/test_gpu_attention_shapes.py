"""GPU tests of prompts in the shape of workgroup that serves most of them, 128 rows, and of its splits over the keys,
against plain attention in 64 bits. Every test asks the library which shape it takes, so that another plan cannot move
them to the other shape unseen."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from _attention import check
from _attention_batched import prompts
from _plans import prompt_plan

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
DOCUMENTS = [140, 0, 129, 256, 1, 128, 127, 200, 64, 131, 0, 333, 140, 97, 250, 180]


def run(cuda, lens_q, lens_k, hq, hkv, d, dtype, splits=False, shared=0, seed=0, causal=False, visible=None, softcap=0.0, slopes=False):
    plan = prompt_plan(sum(lens_q), sum(lens_k), hq, hkv, d, dtype == F32, len(lens_q), causal=causal, shared=shared)
    assert plan[0] == 128 and (plan[1] > 1) == splits, plan
    gen = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    q, k, v = 1.5 * make(sum(lens_q), hq, d), make(sum(lens_k), hkv, d), make(sum(lens_k), hkv, d)
    rest = dict(causal=causal, softcap=softcap)
    if shared:
        rest.update(shared_k=make(shared, hkv, d), shared_v=make(shared, hkv, d))
    if slopes:
        rest["slopes"] = 0.5 * torch.rand(hq, generator=gen)
    if visible is not None:
        rest["visible"] = torch.tensor(visible, dtype=torch.int32)
    off = [torch.tensor([0] + torch.tensor(n).cumsum(0).tolist(), dtype=torch.int32, device=cuda) for n in (lens_q, lens_k)]
    put = {a: t.to(cuda) if isinstance(t, torch.Tensor) else t for a, t in rest.items()}
    y = g.attention(q.to(cuda), k.to(cuda), v.to(cuda), q_offsets=off[0], k_offsets=off[1], **put)
    check(y, prompts(q, k, v, lens_q, lens_k, **rest))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [8, 32, 64, 72, 96, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_documents(cuda, dtype, d, causal):
    run(cuda, DOCUMENTS, DOCUMENTS, 32, 16, d, dtype, causal=causal, seed=d)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq,hkv", [(32, 32), (40, 8), (48, 3), (50, 10)])
def test_groups_of_heads(cuda, dtype, hq, hkv):
    run(cuda, DOCUMENTS, DOCUMENTS, hq, hkv, 64, dtype, causal=True, seed=hq)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shared", [1, 31, 64, 65, 200])
@pytest.mark.parametrize("causal", [False, True])
def test_shared_prefix(cuda, dtype, shared, causal):
    lens_k = [n + (i % 3) * 20 for i, n in enumerate(DOCUMENTS)]
    run(cuda, DOCUMENTS, lens_k, 48, 6, 64, dtype, shared=shared, causal=causal, seed=shared)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shared", [0, 50])
@pytest.mark.parametrize("d", [64, 128])
def test_prefix_mask(cuda, dtype, shared, d):
    visible = [(0, 40, 64, 200, 1000, -5, 129)[i % 7] for i in range(len(DOCUMENTS))]
    run(cuda, DOCUMENTS, DOCUMENTS, 32, 16, d, dtype, shared=shared, causal=True, visible=visible)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("softcap", [0.0, 1.0, 30.0, 300.0])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("causal", [False, True])
def test_caps_and_distance(cuda, dtype, softcap, slopes, causal):
    run(cuda, DOCUMENTS, DOCUMENTS, 32, 16, 64, dtype, shared=33, softcap=softcap, slopes=slopes, causal=causal)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("causal", [False, True])
def test_rows_and_keys_differ(cuda, dtype, causal):
    # more rows than keys (the first see nothing), more keys than rows, none of either
    lens_k = [(n // 2, n + 70, 0, n)[i % 4] for i, n in enumerate(DOCUMENTS)]
    run(cuda, DOCUMENTS, lens_k, 32, 16, 64, dtype, causal=causal)
    run(cuda, DOCUMENTS, lens_k, 32, 16, 128, dtype, causal=causal, shared=70)


# (one sequence whose keys are split over workgroups, whose parts a second launch joins)
SPLIT = [([200], [4000], 32, 8, 64, F16), ([200], [8000], 32, 2, 128, F16), ([128], [1500], 32, 8, 32, F32), ([200], [4000], 48, 1, 64, F32),
         ([200], [1000], 16, 4, 96, F32), ([200], [2100], 16, 4, 128, F32)]


@pytest.mark.parametrize("case", SPLIT)
@pytest.mark.parametrize("causal", [False, True])
def test_split_keys(cuda, case, causal):
    run(cuda, *case, splits=True, causal=causal)


@pytest.mark.parametrize("case", SPLIT)
def test_split_keys_after_a_shared_prefix_capped_and_biased(cuda, case):
    run(cuda, *case, splits=True, causal=True, shared=333, softcap=30.0, slopes=True, visible=[450] * len(case[0]))
