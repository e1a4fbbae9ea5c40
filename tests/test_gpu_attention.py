"""GPU tests of ``attention`` and ``attention_decode`` against plain attention in 64 bits (``_attention``)."""
from __future__ import annotations

import pytest
import torch

import gtx16_fp16 as g
from _attention import check, prompts, tokens

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def normal(gen, *shape, dtype=F16, scale=1.0):
    return (scale * torch.randn(*shape, generator=gen)).to(dtype)


def offsets(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32)


def run_prompts(dev, lens_q, lens_k, hq, hkv, d, dtype, shared=0, seed=0, causal=False, visible=None, softcap=0.0, slopes=False,
                scale=None, what=""):
    gen = torch.Generator().manual_seed(seed)
    q = normal(gen, sum(lens_q), hq, d, dtype=dtype, scale=1.5)
    k, v = (normal(gen, sum(lens_k), hkv, d, dtype=dtype) for _ in "kv")
    sk, sv = (normal(gen, shared, hkv, d, dtype=dtype) if shared else None for _ in "kv")
    sl = 0.5 * torch.rand(hq, generator=gen) if slopes else None
    vis = None if visible is None else torch.tensor(visible, dtype=torch.int32)
    put = lambda t: None if t is None else t.to(dev)  # noqa: E731
    y = g.attention(put(q), put(k), put(v), q_offsets=put(offsets(lens_q)), k_offsets=put(offsets(lens_k)), causal=causal,
                    visible=put(vis), shared_k=put(sk), shared_v=put(sv), softcap=softcap, slopes=put(sl), scale=scale)
    assert y.shape == q.shape and y.dtype == dtype and y.is_contiguous()
    check(y, prompts(q, k, v, lens_q, lens_k, causal, vis, sk, sv, scale, softcap, sl), what)
    return y


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [8, 32, 64, 72, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (6, 2), (5, 1)])
def test_prompt_types_and_heads(cuda, dtype, d, hq, hkv):
    run_prompts(cuda, [37, 1, 70], [37, 1, 70], hq, hkv, d, dtype, causal=True, seed=d)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("causal", [False, True])
def test_prompt_lengths(cuda, dtype, n, causal):
    run_prompts(cuda, [n], [n], 2, 1, 64, dtype, causal=causal, seed=n)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("causal", [False, True])
def test_documents_of_all_lengths_and_empty_ones(cuda, dtype, causal):
    lens = [0, 17, 1, 0, 130, 64, 3, 0]
    run_prompts(cuda, lens, lens, 4, 2, 64, dtype, causal=causal)


def test_documents_past_one_wavefront_of_sequences(cuda):
    gen = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 6, (150,), generator=gen).tolist()
    run_prompts(cuda, lens, lens, 2, 2, 32, F16, causal=True)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lens_q,lens_k", [([5, 40], [300, 41]), ([70, 3], [20, 0]), ([1, 1, 1], [0, 1, 700]), ([64], [1]), ([9], [0])])
@pytest.mark.parametrize("causal", [False, True])
def test_rows_and_keys_differ(cuda, dtype, lens_q, lens_k, causal):
    # more rows than keys: under the causal mask the first rows stand before every key and see nothing
    y = run_prompts(cuda, lens_q, lens_k, 3, 1, 64, dtype, causal=causal)
    if causal and lens_q == [70, 3]:
        assert (y[:50] == 0).all() and (y[70:] == 0).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shared", [1, 31, 64, 65, 200])
@pytest.mark.parametrize("causal", [False, True])
def test_shared_prefix_of_prompts(cuda, dtype, shared, causal):
    run_prompts(cuda, [40, 0, 3], [50, 7, 0], 4, 2, 64, dtype, shared=shared, causal=causal)


def test_rows_before_the_end_of_the_shared_prefix(cuda):
    # rows that stand inside the prefix: more rows than own keys
    run_prompts(cuda, [90], [10], 2, 2, 64, F16, shared=100, causal=True)
    run_prompts(cuda, [90], [10], 2, 2, 64, F16, shared=40, causal=True)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("visible", [[0, 0], [5, 200], [33, 64], [1000, -3]])
@pytest.mark.parametrize("shared", [0, 20])
def test_prefix_mask(cuda, dtype, visible, shared):
    run_prompts(cuda, [100, 130], [100, 135], 2, 1, 64, dtype, shared=shared, causal=True, visible=visible)


def test_prefix_mask_without_a_causal_one_hides_nothing(cuda):
    run_prompts(cuda, [40, 50], [40, 55], 2, 1, 64, F16, visible=[3, 7])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("softcap", [0.0, 1.0, 30.0])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("causal", [False, True])
def test_caps_and_distance(cuda, dtype, softcap, slopes, causal):
    run_prompts(cuda, [50, 97], [80, 97], 4, 2, 64, dtype, shared=33, softcap=softcap, slopes=slopes, causal=causal)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0, 1e-30])
def test_scales(cuda, scale):
    run_prompts(cuda, [50], [50], 2, 1, 64, F32, scale=scale, causal=True)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rows", [3, 100])
@pytest.mark.parametrize("shared", [0, 1900])
def test_few_rows_and_many_keys(cuda, dtype, rows, shared):
    # keys split over workgroups and joined
    run_prompts(cuda, [rows], [2100], 2, 1, 128, dtype, shared=shared, causal=True)


def test_equal_sequences(cuda):
    gen = torch.Generator().manual_seed(3)
    q, k, v = (normal(gen, 3, n, h, 64).to(cuda) for n, h in ((130, 4), (150, 2), (150, 2)))
    y = g.attention(q, k, v, causal=True)
    packed = g.attention(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), q_offsets=offsets([130] * 3).to(cuda),
                         k_offsets=offsets([150] * 3).to(cuda), causal=True)
    check(y, prompts(q.flatten(0, 1).cpu(), k.flatten(0, 1).cpu(), v.flatten(0, 1).cpu(), [130] * 3, [150] * 3, True))
    assert torch.equal(y.flatten(0, 1), packed)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_strides(cuda, dtype):
    gen = torch.Generator().manual_seed(4)
    base = normal(gen, 70, 3 * 4 * 64 + 4, dtype=dtype)
    ref = prompts(*(base[:, i * 256:(i + 1) * 256].reshape(70, 4, 64) for i in range(3)), [70], [70])
    off = offsets([70]).to(cuda)
    x = base.to(cuda)
    q, k, v = (x[:, i * 256:(i + 1) * 256].unflatten(1, (4, 64)) for i in range(3))  # rows of an odd stride: copied
    check(g.attention(q, k, v, q_offsets=off), ref, "fused, odd stride")
    wide = x[:, :768].contiguous()
    q, k, v = (wide[:, i * 256:(i + 1) * 256].unflatten(1, (4, 64)) for i in range(3))
    check(g.attention(q, k, v, q_offsets=off), ref, "fused")
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]  # a token's stride is d
    check(g.attention(*heads_first, q_offsets=off), ref, "heads first")
    shifted = [torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape) for t in (q, k, v)]  # misaligned: copied
    check(g.attention(*shifted, q_offsets=off), ref, "misaligned")
    columns = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]  # values apart: copied
    check(g.attention(*columns, q_offsets=off), ref, "values apart")
    one = k[:1].expand(70, 4, 64)  # every key the same row: copied
    check(g.attention(q, one, one, q_offsets=off), prompts(q.cpu(), one.cpu(), one.cpu(), [70], [70]), "expanded")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("rows", [30, 150])
def test_hidden_infinities_and_nan_stay_hidden(cuda, dtype, bad, rows):
    # key `at` holds them: rows before it, and the other sequences, do not see it
    gen = torch.Generator().manual_seed(6)
    at, lens = rows - 10, [rows, 40]
    q, k, v = (normal(gen, sum(lens), h, 64, dtype=dtype) for h in (2, 1, 1))
    ref = prompts(q, k, v, lens, lens, True)
    k2, v2 = k.clone(), v.clone()
    k2[at], v2[at] = bad, bad
    off = offsets(lens).to(cuda)
    y = g.attention(q.to(cuda), k2.to(cuda), v2.to(cuda), q_offsets=off, causal=True).cpu()
    keep = [i for i in range(sum(lens)) if not at <= i < rows]
    check(y[keep], (ref[0][keep], ref[1][keep]))
    assert not torch.isfinite(y[at:rows]).any()
    # a split of the keys gives the same
    y = g.attention(q[:at].to(cuda), k2[:at + 1].to(cuda), v2[:at + 1].to(cuda), q_offsets=offsets([at]).to(cuda),
                    k_offsets=offsets([at + 1]).to(cuda), causal=True).cpu()
    assert not torch.isfinite(y[-1]).any()
    # without a mask every row sees the key
    y = g.attention(q.to(cuda), k.to(cuda), v2.to(cuda), q_offsets=off).cpu()
    assert not torch.isfinite(y[:rows]).any() and torch.isfinite(y[rows:]).all()


def test_hidden_nan_in_split_keys(cuda):
    gen = torch.Generator().manual_seed(16)
    q, k, v = (normal(gen, n, h, 128) for n, h in ((40, 2), (3000, 1), (3000, 1)))
    v[2980:] = float("nan")
    y = g.attention(q.to(cuda), k.to(cuda), v.to(cuda), q_offsets=offsets([40]).to(cuda), k_offsets=offsets([3000]).to(cuda),
                    causal=True).cpu()
    v0 = v.nan_to_num()
    ref = prompts(q, k, v0, [40], [3000], True)
    check(y[:20], (ref[0][:20], ref[1][:20]))
    assert y[20:].isnan().all()


def test_wide_ranges_of_scores(cuda):
    # scores rise by hundreds along the keys, so the running maximum moves in every tile; then they fall
    gen = torch.Generator().manual_seed(7)
    for order in (1, -1):
        q = normal(gen, 40, 2, 64, dtype=F32)
        k = q.mean(0)[None, :1] + (order * torch.linspace(-30, 30, 333))[:, None, None] * normal(gen, 1, 1, 64, dtype=F32)
        v = normal(gen, 333, 1, 64, dtype=F32)
        for dtype in (F16, F32):
            a, b, c = (t.to(dtype) for t in (q, k, v))
            y = g.attention(a.to(cuda), b.to(cuda), c.to(cuda), q_offsets=offsets([40]).to(cuda), k_offsets=offsets([333]).to(cuda))
            check(y, prompts(a, b, c, [40], [333]), f"{dtype} {order}")


@pytest.mark.parametrize("k_scale,v_scale", [(1e-6, 1.0), (1.0, 1e-6), (1e6, 1.0), (1.0, 1e6), (1e-30, 1e30), (1e6, 1e-12), (300.0, 1e-3)])
@pytest.mark.parametrize("rows", [20, 140])
def test_fp32_values_of_all_sizes(cuda, k_scale, v_scale, rows):
    # past fp16's range and far below it: the tiles that need them take the fp32 instructions
    gen = torch.Generator().manual_seed(17)
    q = normal(gen, rows, 2, 64, dtype=F32, scale=1 / max(k_scale, 1e-6))
    k, v = normal(gen, 150, 1, 64, dtype=F32, scale=k_scale), normal(gen, 150, 1, 64, dtype=F32, scale=v_scale)
    k[70:80] *= 7.0
    y = g.attention(q.to(cuda), k.to(cuda), v.to(cuda), q_offsets=offsets([rows]).to(cuda), k_offsets=offsets([150]).to(cuda))
    out, tol = prompts(q, k, v, [rows], [150])
    check(y, (out, tol + 2.0 ** -36 * min(v_scale, 1.0) * (v_scale >= 2.0 ** -12)))


def test_offsets_outside_the_tensors_are_held_to_them(cuda):
    gen = torch.Generator().manual_seed(8)
    q, k, v = (normal(gen, 50, h, 64) for h in (2, 1, 1))
    y = g.attention(q.to(cuda), k.to(cuda), v.to(cuda), q_offsets=torch.tensor([-7, 20, 900], dtype=torch.int32, device=cuda))
    check(y, prompts(q, k, v, [20, 30], [20, 30]))


# ---- single tokens ------------------------------------------------------------------------------------


def run_tokens(dev, lengths, hq, hkv, d, dtype, capacity=None, page=0, shared=0, softcap=0.0, slopes=False, seed=0, behind=float("nan")):
    """Keys past a length, and pages of no request, hold ``behind``."""
    gen = torch.Generator().manual_seed(seed)
    seqs, capacity = len(lengths), max(max(lengths), 1) if capacity is None else capacity
    q = normal(gen, seqs, hq, d, dtype=dtype, scale=1.5)
    held = [min(max(n, 0), capacity) for n in lengths]
    k, v = ([normal(gen, n, hkv, d, dtype=dtype) for n in held] for _ in "kv")
    sk, sv = (normal(gen, shared, hkv, d, dtype=dtype) if shared else None for _ in "kv")
    sl = 0.5 * torch.rand(hq, generator=gen) if slopes else None
    table = None
    if page:
        per = -(-capacity // page)
        capacity = per * page
        order = torch.randperm(seqs * per + 3, generator=gen)[:seqs * per].view(seqs, per)
        kc, vc = (torch.full((seqs * per + 3, page, hkv, d), behind, dtype=dtype) for _ in "kv")
        table = order.to(torch.int32)
        for b, n in enumerate(held):
            for j in range(0, n, page):
                m = min(page, n - j)
                kc[order[b, j // page], :m], vc[order[b, j // page], :m] = k[b][j:j + m], v[b][j:j + m]
            table[b, -(-n // page):] = -1  # entries past the length are not looked at
    else:
        kc, vc = (torch.full((seqs, capacity, hkv, d), behind, dtype=dtype) for _ in "kv")
        for b, n in enumerate(held):
            kc[b, :n], vc[b, :n] = k[b], v[b]
    put = lambda t: None if t is None else t.to(dev)  # noqa: E731
    y = g.attention_decode(put(q), put(kc), put(vc), torch.tensor(lengths, dtype=torch.int32, device=dev), pages=put(table),
                           shared_k=put(sk), shared_v=put(sv), softcap=softcap, slopes=put(sl))
    assert y.shape == q.shape and y.dtype == dtype
    check(y, tokens(q, k, v, held, sk, sv, softcap=softcap, slopes=sl))
    return y


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [8, 32, 64, 72, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (6, 2), (40, 1)])
def test_token_types_and_heads(cuda, dtype, d, hq, hkv):
    run_tokens(cuda, [33, 0, 130], hq, hkv, d, dtype, shared=40, seed=d)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("page", [0, 1, 3, 16, 24, 64])
@pytest.mark.parametrize("shared", [0, 70])
def test_pages(cuda, dtype, page, shared):
    run_tokens(cuda, [1, 0, 31, 32, 33, 100], 4, 2, 64, dtype, page=page, shared=shared, softcap=20.0, slopes=True)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("page", [0, 16])
def test_long_caches_split_over_workgroups(cuda, dtype, page):
    run_tokens(cuda, [4000, 5, 0, 1777], 4, 1, 128, dtype, page=page, shared=3000, slopes=True)
    run_tokens(cuda, [4000, 5, 0, 1777], 4, 1, 128, dtype, page=page)


def test_many_requests_share_a_prefix(cuda):
    run_tokens(cuda, [(7 * i) % 50 for i in range(70)], 4, 2, 64, F16, shared=500, slopes=True)


def test_lengths_are_held_to_the_cache(cuda):
    run_tokens(cuda, [60, -5, 50, 0], 2, 1, 64, F16, capacity=50)
    run_tokens(cuda, [60, -5, 48, 0], 2, 1, 64, F16, capacity=48, page=16)


def test_no_keys_at_all(cuda):
    q = torch.ones(3, 4, 64, dtype=F16, device=cuda)
    empty = torch.empty(3, 0, 2, 64, dtype=F16, device=cuda)
    n = torch.zeros(3, dtype=torch.int32, device=cuda)
    assert (g.attention_decode(q, empty, empty, n) == 0).all()
    assert g.attention_decode(q[:0], empty[:0], empty[:0], n[:0]).shape == (0, 4, 64)
    off = torch.tensor([0, 3], dtype=torch.int32, device=cuda)
    none = torch.empty(0, 2, 64, dtype=F16, device=cuda)
    assert (g.attention(q, none, none, q_offsets=off, k_offsets=torch.zeros_like(off)) == 0).all()
    assert g.attention(q[:0], none, none, q_offsets=torch.zeros(1, dtype=torch.int32, device=cuda)).shape == (0, 4, 64)


def test_cache_past_32_bit_offsets(cuda):
    # pages more than 2^32 bytes (and 2^31 values) into the cache
    page, hkv, d = 16, 2, 128
    num = (1 << 32) // (page * hkv * d * 2) + 40
    kc, vc = (torch.empty(num, page, hkv, d, dtype=F16, device=cuda) for _ in "kv")
    gen = torch.Generator().manual_seed(9)
    table = torch.tensor([[num - 1, 3, num - 7], [num - 20, num - 2, 0]], dtype=torch.int32)
    lengths = [45, 33]
    q = normal(gen, 2, 4, d)
    k, v = (normal(gen, 2, 3 * page, hkv, d) for _ in "kv")
    for b in range(2):
        for i in range(3):
            kc[table[b, i]], vc[table[b, i]] = k[b, i * page:(i + 1) * page].to(cuda), v[b, i * page:(i + 1) * page].to(cuda)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    y = g.attention_decode(q.to(cuda), kc, vc, n, pages=table.to(cuda))
    check(y, tokens(q, k, v, lengths))
    # the same as one run of keys per request, its sequences 2^32 bytes apart
    far_k, far_v = (t.view(-1).as_strided((2, 48, hkv, d), (1 << 31, hkv * d, d, 1)) for t in (kc, vc))
    far_k.copy_(k.to(cuda))
    far_v.copy_(v.to(cuda))
    check(g.attention_decode(q.to(cuda), far_k, far_v, n), tokens(q, k, v, lengths))
    prompt = g.attention(q.to(cuda)[:, None], far_k[:, :33], far_v[:, :33], causal=True)
    check(prompt, tokens(q, k, v, [33, 33]))


def test_unused_page_numbers_out_of_range_are_safe(cuda):
    gen = torch.Generator().manual_seed(10)
    q, k, v = normal(gen, 1, 2, 64), normal(gen, 4, 16, 1, 64), normal(gen, 4, 16, 1, 64)
    table = torch.tensor([[2, 1 << 30, -(1 << 31), 7]], dtype=torch.int32)
    y = g.attention_decode(q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor([16], dtype=torch.int32, device=cuda), pages=table.to(cuda))
    check(y, tokens(q, [k[2]], [v[2]], [16]))
    # within the length such a page reads as zeros
    z = torch.zeros(16, 1, 64, dtype=F16)
    y = g.attention_decode(q.to(cuda), k.to(cuda), v.to(cuda), torch.tensor([40], dtype=torch.int32, device=cuda), pages=table.to(cuda))
    check(y, tokens(q, [torch.cat((k[2], z, z))], [torch.cat((v[2], z, z))], [40]))


# ---- streams, graphs, repeated calls --------------------------------------------------------------------


def _calls(dev):
    gen = torch.Generator().manual_seed(11)
    q, k, v = (normal(gen, 60, h, 128).to(dev) for h in (4, 2, 2))
    long_k, long_v = (normal(gen, 3, 4000, 2, 128).to(dev) for _ in "kv")
    off = offsets([60]).to(dev)
    far = torch.tensor([0, 4000], dtype=torch.int32, device=dev)
    n = torch.tensor([4000, 17, 900], dtype=torch.int32, device=dev)
    return [lambda: g.attention(q, k, v, q_offsets=off, causal=True),
            lambda: g.attention(q, long_k[0], long_v[0], q_offsets=off, k_offsets=far, causal=True),
            lambda: g.attention_decode(q[:3], long_k, long_v, n, shared_k=k, shared_v=v)]


def test_repeated_calls_agree_bit_for_bit(cuda):
    for call in _calls(cuda):
        first = call()
        for _ in range(5):
            assert torch.equal(call(), first)


def test_other_streams_and_graphs(cuda):
    for call in _calls(cuda):
        want = call()
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


# ---- refusals ---------------------------------------------------------------------------------------------


def test_refusals(cuda):
    q, k = torch.zeros(2, 8, 4, 64, dtype=F16, device=cuda), torch.zeros(2, 8, 2, 64, dtype=F16, device=cuda)
    p, pk, off = q.flatten(0, 1), k.flatten(0, 1), torch.tensor([0, 8, 16], dtype=torch.int32, device=cuda)
    n = torch.tensor([1, 2], dtype=torch.int32, device=cuda)
    tok = q[:, 0]
    bad = [
        lambda: g.attention(q.cpu(), k.cpu(), k.cpu()),
        lambda: g.attention(q.bfloat16(), k.bfloat16(), k.bfloat16()),
        lambda: g.attention(q, k.float(), k),
        lambda: g.attention(q, k, k[:, :4]),
        lambda: g.attention(q, k[:1], k[:1]),
        lambda: g.attention(q, k[:, :, :1].expand(2, 8, 3, 64), k[:, :, :1].expand(2, 8, 3, 64)),
        lambda: g.attention(q[..., :60], k[..., :60], k[..., :60]),
        lambda: g.attention(*(torch.zeros(1, 8, 1, 136, dtype=F16, device=cuda) for _ in range(3))),
        lambda: g.attention(q, k, k, q_offsets=off),
        lambda: g.attention(p, pk, pk),
        lambda: g.attention(p, pk, pk, q_offsets=off.long()),
        lambda: g.attention(p, pk, pk, q_offsets=off.cpu()),
        lambda: g.attention(p, pk, pk, q_offsets=off, k_offsets=off[:2]),
        lambda: g.attention(q, k, k, k_offsets=off),
        lambda: g.attention(q, k, k, visible=n.long()),
        lambda: g.attention(q, k, k, causal=True, visible=n[:1]),
        lambda: g.attention(q, k, k, shared_k=pk),
        lambda: g.attention(q, k, k, shared_k=pk, shared_v=pk[:3]),
        lambda: g.attention(q, k, k, shared_k=p, shared_v=p),
        lambda: g.attention(q, k, k, softcap=-1.0),
        lambda: g.attention(q, k, k, scale=float("nan")),
        lambda: g.attention(q, k, k, slopes=torch.zeros(2, device=cuda)),
        lambda: g.attention(q, k, k, slopes=torch.zeros(4, device=cuda, dtype=F16)),
        lambda: g.attention_decode(q, k, k, n),
        lambda: g.attention_decode(tok, k, k, n.long()),
        lambda: g.attention_decode(tok, k, k, n[:1]),
        lambda: g.attention_decode(tok[:1], k, k, n[:1]),
        lambda: g.attention_decode(tok, k, k, n, pages=n),
        lambda: g.attention_decode(tok, k, k, n, pages=torch.zeros(3, 1, dtype=torch.int32, device=cuda)),
        lambda: g.attention_decode(tok, k, k, n, pages=torch.zeros(2, 1, dtype=torch.int64, device=cuda)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"refusal {i} was taken")
    with pytest.raises(RuntimeError, match="no_grad"):
        g.attention(q.requires_grad_(), k, k)
    with torch.no_grad():
        g.attention(q, k, k)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [8, 24, 32, 40, 72, 88, 96, 104])
def test_many_short_sequences_of_every_width(cuda, dtype, d):
    lengths = [(37 * i) % 70 for i in range(100)]
    run_prompts(cuda, lengths, lengths, 6, 6, d, dtype, causal=d % 16 == 0, seed=d)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lens_q,lens_k", [([130, 0, 7], [1500, 3, 40]), ([1], [3000]), ([300], [300])])
def test_few_tiles_split_over_the_keys(cuda, dtype, lens_q, lens_k):
    run_prompts(cuda, lens_q, lens_k, 2, 1, 72, dtype, causal=True, shared=100, slopes=True)


def test_a_gradient_of_any_operand_is_refused(cuda):
    q, k = torch.zeros(2, 8, 4, 64, dtype=F16, device=cuda), torch.zeros(2, 8, 2, 64, dtype=F16, device=cuda)
    given = dict(shared_k=k[0].clone(), shared_v=k[1].clone(), slopes=torch.zeros(4, device=cuda))
    n = torch.tensor([1, 2], dtype=torch.int32, device=cuda)
    odd = torch.zeros(2, 8, 2, 72, dtype=F16, device=cuda)[..., 4:68]  # (a view that is copied: checked in Python)
    for kk in (k, odd):
        for name in ("q", "k", "v", *given):
            ops = dict(q=q, k=kk, v=kk, **given)
            ops[name] = ops[name].detach().clone().requires_grad_()
            rest = {a: ops[a] for a in given}
            for call in (lambda: g.attention(ops["q"], ops["k"], ops["v"], **rest),  # noqa: B023
                         lambda: g.attention_decode(ops["q"][:, 0], ops["k"], ops["v"], n, **rest)):  # noqa: B023
                with pytest.raises(RuntimeError, match="no_grad"):
                    call()
                    pytest.fail(f"{name} was taken")
                with torch.no_grad():
                    call()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_caps_of_all_sizes(cuda, dtype):
    q, k = torch.zeros(1, 8, 4, 64, dtype=dtype, device=cuda), torch.zeros(1, 8, 2, 64, dtype=dtype, device=cuda)
    n = torch.ones(1, dtype=torch.int32, device=cuda)
    for bad in (1e39, 1e100, 1e299, 1e-60, float("inf")):
        for call in (lambda: g.attention(q, k, k, softcap=bad), lambda: g.attention_decode(q[:, 0], k, k, n, softcap=bad),  # noqa: B023
                     lambda: g.attention(q, k, k, scale=bad if 1 < bad < 1e300 else float("nan"))):  # noqa: B023
            with pytest.raises(ValueError):
                call()
                pytest.fail(f"{bad} was taken")
    for cap in (1e-44, 1e-38, 1e-6, 257.0, 1e6, 1e30, 3e38):
        run_prompts(cuda, [40, 1], [50, 3], 4, 2, 64, dtype, softcap=cap, causal=True, seed=3, what=str(cap))
        # (scores of exactly 0 have a weight, whatever the cap)
        assert (g.attention(q, k, k + 1, softcap=cap) == 1).all()
