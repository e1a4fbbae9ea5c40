"""GPU tests of infinities and NaN in values that some rows of a causal prompt see and others do not, in both shapes of
workgroup, split over the keys and not: rows that do not see them have their results, rows that do have what the formula
gives column by column, and the call takes about as long as any other."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from _attention_batched import prompts
from _plans import prompt_plan

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")
# sequences, rows, keys, query heads, key heads, d, shared keys: (rows of a workgroup, whether the keys are split)
CASES = [((2, 45, 50, 2, 1, 64, 0), (32, False)), ((1, 40, 2100, 2, 1, 128, 0), (32, True)), ((12, 140, 140, 24, 12, 64, 0), (128, False)),
         ((12, 140, 150, 24, 12, 128, 40), (128, False)), ((12, 140, 140, 24, 12, 32, 0), (128, False)),
         {F16: ((1, 200, 3000, 64, 8, 64, 0), (128, True)), F32: ((1, 200, 1000, 16, 4, 96, 0), (128, True))},
         ((12, 140, 140, 24, 12, 96, 0), (128, False))]


def case(case, dtype, seed=0):
    case = case[dtype] if isinstance(case, dict) else case
    (n, rows, keys, hq, hkv, d, shared), (tile, split) = case
    plan = prompt_plan(rows, keys, hq, hkv, d, dtype == F32, n, packed=False, causal=True, shared=shared)
    assert plan[0] == tile and (plan[1] > 1) == split, plan
    gen = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    return make(n, rows, hq, d), make(n, keys, hkv, d), make(n, keys, hkv, d), *((make(shared, hkv, d), make(shared, hkv, d)) if shared else (None, None))


def run(cuda, q, k, v, sk, sv, **rest):
    put = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    return g.attention(put(q), put(k), put(v), causal=True, shared_k=put(sk), shared_v=put(sv), **{a: put(t) for a, t in rest.items()}).cpu()


def expected(q, k, v, sk, sv, spots, visible=None):
    """The result with the values at `spots` (sequence, key, key head, column, value) and its bound."""
    n, rows = q.shape[:2]
    keys, hkv = k.shape[1:3]
    front = 0 if sk is None else sk.shape[0]
    out, tol = (t.unflatten(0, (n, rows)) for t in prompts(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), [rows] * n, [keys] * n, True, visible,
                                                          sk, sv))
    group = q.shape[2] // hkv
    for b, key, head, col, value in spots:
        at = front + key
        sees = at <= front + keys - rows + torch.arange(rows)
        if visible is not None:
            sees = sees | (at < visible[b])
        out[b, sees, head * group:(head + 1) * group, col] += value
    return out, tol


def check(y, out, tol):
    y = y.double()
    finite = torch.isfinite(out)
    assert torch.equal(y.isnan(), out.isnan()) and torch.equal(y[out.isinf()], out[out.isinf()])
    assert ((y - out).abs() / tol)[finite].max() <= 1.0


def spots_of(n, rows, keys, hkv, d):
    # about the first row's key, tile edges, the last key; signs that meet in a column
    first = keys - rows
    at = [first + 3, first + 31, first + 32, first + 33, first + rows // 2, keys - 1]
    return [(b, at[(b + i) % len(at)], (b + i) % hkv, (7 * i + b) % d, value)
            for b in range(n) for i, value in enumerate((INF, -INF, NAN, INF, -INF))] + [(0, at[2], 0, 5, INF), (0, at[4], 0, 5, -INF)]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("which", CASES)
def test_hidden_values(cuda, which, dtype):
    q, k, v, sk, sv = case(which, dtype)
    spots = spots_of(q.shape[0], q.shape[1], k.shape[1], k.shape[2], q.shape[3])
    for b, key, head, col, _ in spots:
        v[b, key, head, col] = 0
    out, tol = expected(q, k, v, sk, sv, spots)
    for b, key, head, col, value in spots:
        v[b, key, head, col] = value if not (b == 0 and col == 5) else (INF if key == spots[-2][1] else -INF)
    check(run(cuda, q, k, v, sk, sv), out, tol)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("which", [CASES[0], CASES[3]])
def test_hidden_values_behind_a_prefix_mask(cuda, which, dtype):
    q, k, v, sk, sv = case(which, dtype, 1)
    n, keys, front = q.shape[0], k.shape[1], 0 if sk is None else sk.shape[0]
    visible = torch.tensor([front + (0, 20, 33, keys)[b % 4] for b in range(n)], dtype=torch.int32)
    spots = [(b, (19, 20, 32, 33, keys - 2)[(b + i) % 5], b % k.shape[2], 3 * i, x) for b in range(n) for i, x in enumerate((INF, NAN, -INF))]
    for b, key, head, col, _ in spots:
        v[b, key, head, col] = 0
    out, tol = expected(q, k, v, sk, sv, spots, visible)
    for b, key, head, col, value in spots:
        v[b, key, head, col] = value
    check(run(cuda, q, k, v, sk, sv, visible=visible), out, tol)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("which", [CASES[0], CASES[2], CASES[1]])
def test_whole_rows_hidden(cuda, which, dtype):
    # keys and values from one position on are NaN: rows before it have their results, the others are NaN
    q, k, v, sk, sv = case(which, dtype, 2)
    n, rows, keys = q.shape[0], q.shape[1], k.shape[1]
    out, tol = expected(q, k, v, sk, sv, [])
    at = keys - rows + 35
    k[:, at:], v[:, at:] = NAN, NAN
    out[:, 35:] = NAN
    check(run(cuda, q, k, v, sk, sv), out, tol)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n", [600, 4096])
def test_infinities_cost_no_second_pass(cuda, dtype, n):
    # (a row at a time, key by key, would be hundreds of times as long)
    q, k, v = (torch.randn(1, n, h, 64, device=cuda).to(dtype) for h in (8, 4, 4))
    bad = v.clone()
    bad[0, 40, :, 3] = NAN

    def time(v):
        best = 1e9
        for _ in range(5):
            a, b = torch.cuda.Event(True), torch.cuda.Event(True)
            a.record()
            for _ in range(10):
                g.attention(q, k, v, causal=True)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    time(v)
    plain, with_nan = time(v), time(bad)
    assert with_nan <= 3 * plain, (plain, with_nan)
