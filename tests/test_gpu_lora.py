"""GPU tests of ``lora_mm_t`` against the formula in 64 bits.

Bounds: the output is rounded once to its type (2^-11 or 2^-24); sums over K and over the rank are fp32 (random
roundings: 4 sqrt(n) 2^-24 of the sum of magnitudes); past 8 rows the shared product rounds fp32 activations
to fp16 (2^-11 of each, at most 2^-11 of the sum of |x w|), as ``mm_t`` says; the adapters' part rounds nothing.
"""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from gtx16_fp16 import lora, ops

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def make(M, K, N, r, n, dtype=F16, seed=0, bias=True, scale=True):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s, by=1.0: by * torch.randn(*s, generator=gen)  # noqa: E731
    return dict(x=rand(M, K).to(dtype), w=rand(K, N, by=0.05).half(), down=rand(n, r, K, by=K ** -0.5 if K else 1.0).half(),
                up=rand(n, N, r, by=0.2).half(), index=torch.randint(-1, max(n, 1), (M,), generator=gen, dtype=torch.int32),
                bias=rand(N) if bias else None, scale=0.5 + torch.rand(n, generator=gen) if scale else None)


def reference(c, out):
    x, w = c["x"].double(), c["w"].double()
    K = x.shape[1]
    y, size = x @ w, x.abs() @ w.abs()
    err = (4 * K ** 0.5 * 2.0 ** -24 + (2.0 ** -11 if c["x"].dtype == F32 and x.shape[0] > 8 else 0.0)) * size
    if c["bias"] is not None:
        y = y + c["bias"].double()
    for a in range(c["down"].shape[0]):
        rows = (c["index"] == a).nonzero().flatten()
        if rows.numel():
            s = 1.0 if c["scale"] is None else float(c["scale"][a])
            d, u = c["down"][a].double(), c["up"][a].double()
            y[rows] += s * ((x[rows] @ d.T) @ u.T)
            low = s * (x[rows].abs() @ d.abs().T) @ u.abs().T
            err[rows] += 4 * (K ** 0.5 + d.shape[0] ** 0.5 + 2) * 2.0 ** -24 * low
    # (the last additions: the shared result, the bias and the adapters' part in fp32)
    u = 2.0 ** -11 if out == F16 else 2.0 ** -24
    return y, err + (u + 2 * 2.0 ** -24) * y.abs() + 2 * 2.0 ** -24 * size + (2.0 ** -25 if out == F16 else 1e-37)


def run(dev, c, out=F16):
    put = lambda t: None if t is None else t.to(dev)  # noqa: E731
    return g.lora_mm_t(put(c["x"]), put(c["w"]), put(c["down"]), put(c["up"]), put(c["index"]), scale=put(c["scale"]), bias=put(c["bias"]),
                       out_dtype=out)


def check(dev, c, out=F16):
    y = run(dev, c, out)
    assert y.dtype == out and y.is_contiguous()
    ref, tol = reference(c, out)
    over = ((y.double().cpu() - ref).abs() / tol).max().item() if ref.numel() else 0.0
    assert over <= 1.0, f"{over:.3g} times the bound"
    return y


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 15, 16, 17, 64, 130, 600])
@pytest.mark.parametrize("x,out", [(F16, F16), (F16, F32), (F32, F32), (F32, F16)])
def test_rows_and_types(cuda, M, x, out):
    check(cuda, make(M, 512, 384, 16, 5, x, seed=M), out)


@pytest.mark.parametrize("r", [8, 16, 24, 32, 40, 64, 72, 128])
@pytest.mark.parametrize("M", [3, 50, 300])
@pytest.mark.parametrize("x", [F16, F32])
def test_ranks(cuda, r, M, x):
    check(cuda, make(M, 264, 520, r, 4, x, seed=r))


@pytest.mark.parametrize("K,N", [(8, 8), (8, 4096), (4096, 8), (40, 72), (1000, 1048), (5000, 264)])
@pytest.mark.parametrize("M", [1, 33])
def test_odd_sizes(cuda, K, N, M):
    check(cuda, make(M, K, N, 8, 3, seed=K + N))
    check(cuda, make(M, K, N, 32, 3, F32, seed=K + N), F32)


@pytest.mark.parametrize("M,n", [(48, 48), (200, 64), (5000, 3)])
def test_every_row_its_own_adapter_or_long_runs(cuda, M, n):
    c = make(M, 256, 256, 16, n, seed=M)
    if n == 48:
        c["index"] = torch.randperm(48, dtype=torch.int32)
    elif n == 3:
        c["index"] = (torch.arange(M) // 1700).to(torch.int32)
    check(cuda, c)


def test_rows_without_an_adapter_equal_the_shared_product(cuda):
    c = make(100, 256, 512, 16, 4)
    c["index"][:] = -1
    c["index"][[3, 40]] = torch.tensor([4, 1 << 30], dtype=torch.int32)  # past the last adapter
    y = run(cuda, c, F32)
    assert torch.equal(y, ops.mm_t(c["x"].to(cuda), c["w"].to(cuda), c["bias"].to(cuda), F32))
    check(cuda, c, F16)


@pytest.mark.parametrize("n,r", [(0, 16), (3, 0)])
@pytest.mark.parametrize("out", [F16, F32])
def test_no_adapters(cuda, n, r, out):
    c = make(20, 64, 64, r, n)
    y = run(cuda, c, out)
    assert torch.equal(y, ops.mm_t(c["x"].to(cuda), c["w"].to(cuda), c["bias"].to(cuda), F32).to(out))


def test_empty_sizes(cuda):
    assert run(cuda, make(0, 64, 64, 8, 2)).shape == (0, 64)
    c = make(5, 0, 64, 8, 2)
    assert torch.equal(run(cuda, c, F32).cpu(), c["bias"].expand(5, 64))


def test_without_scale_and_bias(cuda):
    check(cuda, make(70, 256, 264, 24, 3, bias=False, scale=False))


def test_large_activations_keep_the_adapters_exact(cuda):
    # rows far past fp16's range: low-rank sums of 1e6 and more
    c = make(40, 256, 256, 16, 3, F32)
    c["x"][7] *= 1e6
    check(cuda, c, F32)


def test_infinite_and_nan_activations_stay_in_their_rows(cuda):
    for M in (5, 40, 600):
        c = make(M, 256, 264, 16, 3, F32)
        c["index"][:] = torch.arange(M, dtype=torch.int32) % 3
        ref, tol = reference(c, F32)
        c["x"][1, 5], c["x"][2, 9] = float("inf"), float("nan")
        y = run(cuda, c, F32).cpu().double()
        keep = [i for i in range(M) if i not in (1, 2)]
        assert ((y - ref).abs() / tol)[keep].max() <= 1.0
        assert not torch.isfinite(y[1:3]).any()


def test_views_are_copied(cuda):
    c = make(30, 128, 128, 8, 2)
    want = run(cuda, c)
    put = lambda t: t.to(cuda)  # noqa: E731
    wide = torch.zeros(30, 256, dtype=F16, device=cuda)
    wide[:, 3:131] = put(c["x"])
    down = put(c["down"]).transpose(1, 2).contiguous().transpose(1, 2)
    up = put(c["up"]).transpose(1, 2).contiguous().transpose(1, 2)
    idx = put(c["index"]).repeat_interleave(2)[::2]
    y = g.lora_mm_t(wide[:, 3:131], put(c["w"]), down, up, idx, scale=put(c["scale"]), bias=put(c["bias"]), out_dtype=F16)
    assert torch.equal(y, want)


def test_repeated_calls_streams_and_graphs(cuda):
    for M in (4, 40, 700):
        c = {k: None if v is None else v.to(cuda) for k, v in make(M, 512, 512, 16, 6).items()}
        call = lambda: g.lora_mm_t(c["x"], c["w"], c["down"], c["up"], c["index"], scale=c["scale"], bias=c["bias"], out_dtype=F16)  # noqa: E731,B023
        want = call()
        assert all(torch.equal(call(), want) for _ in range(4))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            y = call()
            with torch.cuda.graph(graph, stream=s):
                z = call()
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(y, want)
        for _ in range(3):
            z.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(z, want)
            assert torch.equal(call(), want)


def test_refusals(cuda):
    c = {k: v.to(cuda) for k, v in make(20, 64, 64, 8, 2).items()}

    def call(**changes):
        d = dict(c, out=F16, **{})
        d.update(changes)
        return g.lora_mm_t(d["x"], d["w"], d["down"], d["up"], d["index"], scale=d["scale"], bias=d["bias"], out_dtype=d["out"])

    call()
    for changes in (dict(x=c["x"].bfloat16()), dict(x=c["x"].cpu()), dict(x=c["x"][0]), dict(w=c["w"].float()), dict(w=c["w"][:32]),
                    dict(down=c["down"].float()), dict(down=c["down"][:1]), dict(down=c["down"][:, :, :32]), dict(up=c["up"][:, :, :4]),
                    dict(up=c["up"].transpose(1, 2)), dict(down=c["down"][:, :4], up=c["up"][:, :, :4]), dict(up=c["up"].cpu()),
                    dict(down=c["down"].repeat(1, 17, 1), up=c["up"].repeat(1, 1, 17)), dict(index=c["index"].long()),
                    dict(index=c["index"][:3]), dict(index=c["index"].cpu()), dict(scale=c["scale"].half()), dict(scale=c["scale"][:1]),
                    dict(bias=c["bias"][:3]), dict(out=torch.bfloat16)):
        with pytest.raises(ValueError):
            call(**changes)
            pytest.fail(f"{list(changes)} was taken")
    with pytest.raises(RuntimeError, match="no_grad"):
        call(x=c["x"].clone().requires_grad_())


def test_sides_past_32_bit_offsets_are_refused(cuda):
    n = lora.MAX_SIDE + 8
    index = torch.zeros(1, dtype=torch.int32, device=cuda)

    def zeros(*shape):
        return torch.zeros(*shape, device=cuda, dtype=F16)

    with pytest.raises(ValueError, match="up to"):
        g.lora_mm_t(zeros(1, 8), zeros(8, n), zeros(1, 8, 8), zeros(1, n, 8), index)
    with pytest.raises(ValueError, match="up to"):
        g.lora_mm_t(zeros(1, n), zeros(n, 8), zeros(1, 8, n), zeros(1, 8, 8), index)


@pytest.mark.parametrize("M,n", [(64, 2), (64, 5), (200, 3), (333, 40)])
def test_adapters_interleaved_row_by_row(cuda, M, n):
    c = make(M, 256, 136, 24, n)
    c["index"] = torch.arange(M, dtype=torch.int32) % (n + 1)
    check(cuda, c)


@pytest.mark.parametrize("M,K", [(5, 64), (16, 256), (40, 256), (300, 512)])
@pytest.mark.parametrize("x,out", [(F16, F16), (F32, F16), (F16, F32)])
def test_every_negative_index_means_no_adapter(cuda, M, K, x, out):
    c = make(M, K, 136, 16, 3, x, seed=M)
    c["index"][::2] = torch.tensor([-2, -1, -7, -(1 << 31)], dtype=torch.int32).repeat(M)[:c["index"][::2].numel()]
    rows = c["index"] < 0
    want = ops.mm_t(c["x"].to(cuda), c["w"].to(cuda), c["bias"].to(cuda), F32).to(out)
    for _ in range(2):
        torch.full((M, 136), float("nan"), dtype=out, device=cuda)  # (freed at once: likely the next output's memory)
        y = check(cuda, c, out)
        assert torch.equal(y[rows.to(cuda)], want[rows.to(cuda)])


@pytest.mark.parametrize("M,K,r", [(1, 512, 16), (7, 256, 24), (40, 256, 16), (300, 512, 48), (300, 264, 128)])
@pytest.mark.parametrize("x", [F16, F32])
def test_channels_of_the_rank_of_unlike_size(cuda, M, K, r, x):
    # large sums that meet small columns of `up` beside small ones that meet large columns, and make the result
    c = make(M, K, 136, r, 3, x, seed=M + r)
    c["w"] *= 2.0 ** -14
    c["bias"] *= 0
    c["down"] = (c["down"].float() * torch.where(torch.arange(r) % 3 == 0, 2.0 ** 15, 2.0 ** -13)[:, None]).half()
    c["up"] = (c["up"].float() * torch.where(torch.arange(r) % 3 == 0, 2.0 ** -22, 2.0 ** 13)).half()
    check(cuda, c, F32)


@pytest.mark.parametrize("M", [3, 40, 300])
def test_infinite_sums_of_an_adapter_stay_infinite(cuda, M):
    # one sum past fp32 beside a huge finite one of the other sign, from finite activations
    c = make(M, 64, 136, 16, 2, F32, seed=M, bias=False)
    c["index"][:] = 1
    c["down"].zero_()
    c["down"][1, 0, 3], c["down"][1, 1, 4] = 1000.0, -1.0
    c["up"] = c["up"].abs() + 0.1
    plain = c["x"].clone()
    c["x"][0, 3], c["x"][0, 4] = 1e38, 1e30
    y = run(cuda, c, F32).cpu()
    assert (y[0] == float("inf")).all()
    ref, tol = reference(dict(c, x=plain), F32)
    assert ((y.double() - ref).abs() / tol)[1:].max() <= 1.0


def test_a_workspace_that_is_not_kept(cuda):
    check(cuda, make(40000, 64, 64, 128, 3))


@pytest.mark.parametrize("M", [4, 40])
def test_a_gradient_of_any_operand_is_refused(cuda, M):
    c = {k: v.to(cuda) for k, v in make(M, 64, 64, 8, 2).items()}
    for view in (False, True):
        for name in ("x", "w", "down", "up", "scale", "bias"):
            d = dict(c, x=c["x"].t().contiguous().t()) if view else dict(c)
            d[name] = d[name].detach().clone(memory_format=torch.preserve_format).requires_grad_()
            call = lambda: g.lora_mm_t(d["x"], d["w"], d["down"], d["up"], d["index"], scale=d["scale"], bias=d["bias"])  # noqa: E731,B023
            with pytest.raises(RuntimeError, match="no_grad"):
                call()
                pytest.fail(f"{name} was taken")
            with torch.no_grad():
                call()


@pytest.mark.parametrize("M,K,rank", [((1 << 23) + 37, 64, 8), ((1 << 27) + 70, 8, 8)])
def test_more_rows_than_a_launch_has_threads_for(cuda, M, K, rank):
    # 2^32 threads a launch: workgroups of 512 for every 16 rows, several of them where a tile may hold several adapters
    gen = torch.Generator(cuda).manual_seed(0)
    x = torch.empty(M, K, dtype=F16, device=cuda).normal_(generator=gen)
    w, down = torch.randn(K, 8, generator=gen, device=cuda).half(), torch.randn(3, rank, K, generator=gen, device=cuda).half()
    up = torch.randn(3, 8, rank, generator=gen, device=cuda).half()
    index = (torch.arange(M, device=cuda) % 5 - 1).int()
    y = g.lora_mm_t(x, w, down, up, index, out_dtype=F16)
    for a in (0, 1 << 20, 1 << 22, (1 << 23) - 50, M // 2, (1 << 27) - 50, M - 100):
        if a + 100 <= M:
            rows = slice(a, a + 100)
            c = dict(x=x[rows].cpu(), w=w.cpu(), down=down.cpu(), up=up.cpu(), index=index[rows].cpu(), scale=None, bias=None)
            ref, tol = reference(c, F16)
            assert ((y[rows].double().cpu() - ref).abs() / tol).max() <= 1.0, a


@pytest.mark.parametrize("M,K,splits", [(300, 520, 1), (300, 1000, 1), (300, 2056, 4), (300, 4096, 4), (2000, 1032, 2), (2000, 4096, 4),
                                        (4200, 1000, 1), (4200, 4096, 2)])
@pytest.mark.parametrize("r", [8, 24, 32, 64, 128])
@pytest.mark.parametrize("x", [F16, F32])
def test_many_rows_by_way_of_lds(cuda, M, K, splits, r, x):
    # both operands through LDS, for every number of rank blocks: K split over workgroups and not, a multiple of a chunk and
    # not, rows of an adapter in runs, row by row and at random, one and several adapters to a workgroup
    head = lora._ARGS.pack(*([4096] * 7), M, K, 136, r, 6, x == F32, 1, torch.cuda.get_device_properties(cuda).multi_processor_count)
    nbytes = g._clib.fast().args_size(g._clib.address("g16_lora_workspace_bytes"), head)
    assert nbytes == splits * M * r * 4
    c = make(M, K, 136, r, 6, x, seed=M + K + r)
    m = torch.arange(M, dtype=torch.int32)
    for index in (m // 300, m % 7 - 1, torch.randint(-1, 6, (M,), generator=torch.Generator().manual_seed(r)).int()):
        c["index"] = index
        check(cuda, c, F32)


@pytest.mark.parametrize("x", [F16, F32])
def test_every_row_of_many_its_own_adapter(cuda, x):
    # 16 adapters to a tile, on fewer workgroups
    c = make(600, 1032, 136, 16, 600, x)
    c["index"] = torch.randperm(600, generator=torch.Generator().manual_seed(0)).int()
    check(cuda, c)
