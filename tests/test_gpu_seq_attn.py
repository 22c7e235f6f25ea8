"""Attention of new tokens over a paged cache and of packed prompts, against the formula in 64
bits (tests/seq_cases.py has it, with the tolerances)."""
import pytest
import torch

from tests.seq_cases import U, Cache, attention, check_packed, check_paged, gen, offsets, randn

pytestmark = pytest.mark.gpu

HALF = (torch.bfloat16, torch.float16)
CODES = (torch.int8, torch.float8_e4m3fn, None)


def _paged(srdit, g, cache, new, H, dtype, causal=True, q=None, **kw):
    cu = offsets(new)
    if q is None:
        q = randn(g, sum(new), H, cache.D).to(dtype)
    out = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                               causal=causal, **cache.scales, **kw)
    check_paged(cache, q, cu, out, causal, kw.get("scale", cache.D ** -0.5))
    return q, cu, out


# ------------------------------------------------------------------ single tokens, few rows
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("lens,H,Hkv,D,page,layout", [
    ([1], 1, 1, 64, 16, "tokens"), ([5, 0, 16, 17], 4, 4, 128, 16, "heads"),
    ([100, 2000, 1, 513, 64], 16, 2, 128, 32, "both"), ([777], 12, 1, 80, 128, "heads"),
    ([4000, 3999], 16, 1, 96, 64, "tokens"), ([5000], 2, 2, 16, 2304, "tokens"),
    ([9000], 5, 1, 112, 16, "heads"), ([33] * 40, 6, 3, 64, 16, "heads")])
def test_single_tokens(srdit, cuda_device, dtype, code, lens, H, Hkv, D, page, layout):
    g = gen(sum(lens) + H)
    cache = Cache(g, lens, Hkv, D, page, code or dtype, layout).fill(g, dtype)
    q = randn(g, len(lens), H, D).to(dtype)
    out = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, **cache.scales)
    check_paged(cache, q, torch.arange(len(lens) + 1), out, True, D ** -0.5)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("new,lens,H,Hkv,D,page", [
    ([3, 0, 4, 1], [3, 7, 300, 129], 8, 4, 128, 16), ([16], [1500], 3, 3, 64, 64),
    ([5, 5], [4, 2000], 3, 1, 128, 32), ([8, 1], [8, 17], 2, 1, 96, 16)])
def test_a_few_tokens(srdit, cuda_device, dtype, code, causal, new, lens, H, Hkv, D, page):
    """Up to 16 rows a key head; among them more new tokens than the cache has (5 of 4)."""
    g = gen(sum(lens) + H)
    cache = Cache(g, lens, Hkv, D, page, code or dtype, "heads").fill(g, dtype)
    q, cu, out = _paged(srdit, g, cache, new, H, dtype, causal, max_q=max(new))
    if lens[0] < new[0] and causal:
        assert (out[0] == 0).all()


# ------------------------------------------------------------------ chunks
CHUNKS = [
    ([17], [17], 1, 1, 64, 16, "tokens"), ([100, 0, 30], [131, 50, 30], 4, 2, 128, 16, "heads"),
    ([128, 256, 1, 257], [128, 300, 1000, 257], 2, 2, 64, 32, "both"),
    ([300], [2000], 8, 1, 128, 64, "heads"), ([65, 64, 63], [700, 65, 200], 12, 4, 80, 16, "tokens"),
    ([200], [5000], 6, 2, 112, 128, "tokens"), ([40, 0, 41], [30, 0, 2400], 5, 5, 32, 16, "heads"),
    ([513], [1025], 7, 1, 96, 16, "heads")]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("new,lens,H,Hkv,D,page,layout", CHUNKS)
def test_chunks(srdit, cuda_device, dtype, code, causal, new, lens, H, Hkv, D, page, layout):
    g = gen(sum(lens) + H)
    cache = Cache(g, lens, Hkv, D, page, code or dtype, layout).fill(g, dtype)
    _paged(srdit, g, cache, new, H, dtype, causal)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("causal", (True, False))
def test_many_sequences(srdit, cuda_device, code, causal):
    """More sequences than a warp has lanes, and more pieces of work than the GPU has SMs."""
    g, dt = gen(5), torch.bfloat16
    new = [(37 * i) % 61 if i % 5 else 0 for i in range(90)]
    lens = [n + (i * 71) % 400 for i, n in enumerate(new)]
    cache = Cache(g, lens, 4, 64, 16, code or dt, "heads").fill(g, dt)
    _paged(srdit, g, cache, new, 8, dt, causal)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("D", (64, 128))
def test_items_of_one_and_of_two_tiles(srdit, cuda_device, dtype, code, D):
    """Many short sequences in turn, with the second query tile of an item in use or not, whose
    query rows are of very different size."""
    g, n = gen(16), 260
    new = torch.randint(0, 2, (n,), generator=torch.Generator().manual_seed(3)).mul(160).add(40).tolist()
    cache = Cache(g, [100 + i % 29 for i in range(n)], 4, D, 16, code or dtype, "heads").fill(g, dtype)
    q = randn(g, sum(new), 4, D)
    q = q * torch.exp2(torch.randint(-12, 1, (sum(new), 4, 1), generator=g, device="cuda").float())
    _paged(srdit, g, cache, new, 4, dtype, False, q.to(dtype))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("new,lens,H,Hkv", [
    ([40, 900, 30], [60, 0, 200], 16, 2), ([300, 1400, 200, 1000, 50], [900, 0, 300, 0, 70], 8, 8),
    ([132, 9, 25, 391, 850], [3, 18, 277, 151, 2000], 16, 2), ([12000, 100, 9000], [0, 500, 10], 8, 1)])
def test_many_queries_without_keys(srdit, cuda_device, dtype, code, causal, new, lens, H, Hkv):
    """Long runs of queries that see no key, before, between and behind others that do."""
    g = gen(17)
    cache = Cache(g, lens, Hkv, 64, 32, code or dtype).fill(g, dtype)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, cu, out = _paged(srdit, g, cache, new, H, dtype, causal, status=status)
    assert status.item() == 0
    if code is None:
        kv = [torch.cat([cache.rows(b, w)[0] for b in range(len(lens))]).to(dtype) for w in "kv"]
        got = srdit.ops.packed_attn(q, *kv, cu, cu_k=offsets(lens), causal=causal, status=status)
        check_packed(q, *kv, cu, offsets(lens), got, causal, 64 ** -0.5)
        assert status.item() == 0


@pytest.mark.parametrize("code", CODES)
def test_a_chunk_of_frames(srdit, cuda_device, code):
    """Two frames of 2304 tokens over four, every token seen; pages of a frame."""
    g, dt = gen(6), torch.bfloat16
    cache = Cache(g, [4 * 2304], 3, 128, 2304, code or dt).fill(g, dt)
    _paged(srdit, g, cache, [2 * 2304], 3, dt, False)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("new", ([1, 1, 1], [70, 80, 90]))
def test_hidden_pages(srdit, cuda_device, code, new):
    """Keys in pages that the table does not have are not seen; one sequence has no other."""
    g, dt = gen(7), torch.bfloat16
    cache = Cache(g, [200, 90, 300], 2, 64, 16, code or dt, "heads").fill(g, dt)
    hide = [torch.zeros(n, dtype=torch.bool, device="cuda") for n in cache.lens]
    keep = cache.table.clone()
    for b, pages in ((0, (0, 5, 12)), (1, range(6)), (2, (7, 8, 18))):
        for p in pages:
            cache.table[b, p] = -1 if p % 2 else 1 << 29
            hide[b][p * 16:(p + 1) * 16] = True
    cu, H = offsets(new), 4
    q = randn(g, sum(new), H, 64).to(dt)
    out = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                               max_q=max(new), **cache.scales)
    cache.table = keep
    check_paged(cache, q, cu, out, True, 64 ** -0.5, hide)
    assert (out[int(cu[1]):int(cu[2])] == 0).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("new", ([1, 1], [50, 40]))
def test_rows_behind_the_last_sequence(srdit, cuda_device, code, new):
    g, dt = gen(8), torch.float16
    cache = Cache(g, [300, 70], 2, 128, 32, code or dt).fill(g, dt)
    n = sum(new)
    q = randn(g, n + 30, 4, 128).to(dt)
    q[n:] = float("nan")
    buf = torch.full((n + 30, 6, 136), 5.0, dtype=dt, device="cuda")
    out = buf[:, 1:5, :128]
    cu = offsets(new)
    srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, out, cu_q=cu,
                         max_q=max(new), **cache.scales)
    check_paged(cache, q, cu, out, True, 128 ** -0.5)
    buf[:n, 1:5, :128] = 5.0
    assert (buf == 5).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("code", (torch.int8, torch.float8_e4m3fn))
@pytest.mark.parametrize("new", ([1, 1], [60, 70]))
def test_scales_of_very_different_size(srdit, cuda_device, dtype, code, new):
    """Values from 2^-10 to 2^10 of the usual, keys too; queries of the type's large values."""
    g = gen(10)
    cache = Cache(g, [400, 1000], 2, 64, 16, code, "heads").fill(g, dtype, size=0.0)
    for s in (cache.ks, cache.vs):
        grow = torch.exp2(20 * torch.rand(s.shape, generator=g, device="cuda") - 10)
        s.mul_(grow if s is cache.vs else torch.rsqrt(1 + grow))
    q = randn(g, sum(new), 4, 64)
    q[0] *= 2.0 ** 14
    q[-1] = 0
    q = q.to(dtype)
    cache.ks.mul_(1.0)
    cu = offsets(new)
    # the first row's scores are far apart: its weights are one key's or a few
    out = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                               max_q=max(new), scale=0.125, **cache.scales)
    q2, out2 = q.clone(), out.clone()
    q2[0], out2[0] = 0, 0
    rows = torch.arange(1, sum(new), device="cuda")
    ref = srdit.ops.paged_attn(q2, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                               max_q=max(new), scale=0.125, **cache.scales)
    check_paged(cache, q2, cu, ref, True, 0.125)
    assert torch.equal(ref[rows], out2[rows]) and out[0].isfinite().all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("new", ([1, 1], [60, 70]))
def test_nan_of_a_seen_key_comes_out(srdit, cuda_device, code, new):
    g, dt = gen(14), torch.bfloat16
    cache = Cache(g, [100, 200], 2, 64, 16, code or dt).fill(g, dt)
    page, row = cache.places(0, 20, 21)
    if code is None:
        cache.k[page, row, 1, 5] = float("nan")
    else:
        cache.ks[page, row, 1] = float("nan")
    q = randn(g, sum(new), 4, 64).to(dt)
    cu = offsets(new)
    out = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                               max_q=max(new), **cache.scales)
    assert out[:new[0], 2:].isnan().all() and out[:new[0], :2].isfinite().all()
    assert out[new[0]:].isfinite().all()


def test_cache_beyond_32_bits(srdit, cuda_device):
    """Pages whose codes begin past 2^31 elements."""
    g, dt = gen(15), torch.bfloat16
    n, P, H, D = 9200, 128, 16, 128
    pool = torch.zeros(2, n, P, H, D, dtype=torch.int8, device="cuda")
    cache = Cache(g, [700], H, D, P, torch.int8, spare=0)
    scale = torch.full((2, n, P, H), float("nan"), device="cuda")
    cache.k, cache.v, cache.ks, cache.vs = pool[0], pool[1], scale[0], scale[1]
    cache.table[0, :6] = torch.tensor([n - 1, 0, n - 3, 5, n - 2, 17], dtype=torch.int32)
    cache.fill(g, dt)
    _paged(srdit, g, cache, [1], H, dt)
    _paged(srdit, g, cache, [40], H, dt)


# ------------------------------------------------------------------ packed prompts
PACKED = [
    ([1], 1, 1, 64), ([5, 0, 130, 1], 4, 2, 128), ([128, 128], 2, 2, 64), ([129, 127, 300], 8, 1, 80),
    ([700], 3, 3, 128), ([257, 0, 0, 40], 6, 2, 32), ([16] * 50, 4, 4, 96), ([1025], 16, 2, 112),
    ([33, 2000], 2, 1, 64)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("lens,H,Hkv,D", PACKED)
def test_packed(srdit, cuda_device, dtype, causal, lens, H, Hkv, D):
    g = gen(sum(lens) + H)
    T = sum(lens)
    q = randn(g, T, H, D).to(dtype)
    kv = randn(g, T, 2, Hkv, D).to(dtype)
    cu = offsets(lens)
    out = srdit.ops.packed_attn(q, kv[:, 0], kv[:, 1], cu, causal=causal)
    check_packed(q, kv[:, 0], kv[:, 1], cu, cu, out, causal, D ** -0.5)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("nq,nk,H,Hkv,D", [
    ([30, 300, 0, 5], [100, 10, 50, 0], 4, 2, 64), ([200, 300], [900, 301], 2, 2, 128),
    ([1, 2, 3], [1000, 3, 2], 8, 1, 96)])
def test_packed_keys_of_other_lengths(srdit, cuda_device, dtype, causal, nq, nk, H, Hkv, D):
    """More queries than keys (the first see none), no keys at all, views of wider buffers, rows
    before the first and behind the last sequence full of NaN and left as they were."""
    g = gen(sum(nq) + H)
    T, Tk = sum(nq) + 9, sum(nk) + 13
    q = randn(g, T, H, 2 * D).to(dtype)[..., D:]
    k = randn(g, Tk, Hkv + 1, D).to(dtype)[:, 1:]
    v = randn(g, Tk, Hkv, D).to(dtype)
    cu_q, cu_k = offsets(nq, 4), offsets(nk, 6)
    for t, cu in ((q, cu_q), (k, cu_k), (v, cu_k)):
        t[:int(cu[0])] = float("nan")
        t[int(cu[-1]):] = float("nan")
    buf = torch.full((T, H, D + 8), 5.0, dtype=dtype, device="cuda")
    out = srdit.ops.packed_attn(q, k, v, cu_q, buf[..., :D], cu_k=cu_k, causal=causal, scale=0.2)
    check_packed(q, k, v, cu_q, cu_k, out, causal, 0.2)
    for b, (n, L) in enumerate(zip(nq, nk)):
        if L == 0 or (causal and n > L):
            lo = int(cu_q[b])
            assert (out[lo:lo + (n - L if causal else n)] == 0).all()
    buf[4:4 + sum(nq), :, :D] = 5.0
    assert (buf == 5).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("causal", (True, False))
def test_repeated_key_heads(srdit, cuda_device, dtype, causal):
    """One key head for all by a stride of zero; heads of q are not read so."""
    g = gen(22)
    q = randn(g, 500, 6, 64).to(dtype)
    k, v = (randn(g, 500, 1, 64).to(dtype).expand(500, 3, 64) for _ in range(2))
    cu = offsets([200, 300])
    out = srdit.ops.packed_attn(q, k, v.contiguous(), cu, causal=causal)
    check_packed(q, k, v, cu, cu, out, causal, 64 ** -0.5)
    assert torch.equal(out, srdit.ops.packed_attn(q, k, v, cu, causal=causal))
    with pytest.raises(srdit._lib.SrditError):
        srdit.ops.packed_attn(q[:, :1].expand(500, 6, 64), k, v, cu, causal=causal)


@pytest.mark.parametrize("causal", (True, False))
def test_sequences_do_not_see_each_other(srdit, cuda_device, causal):
    """NaN in one sequence's keys and values leaves its neighbours as they are."""
    g, dt = gen(21), torch.bfloat16
    lens = [70, 90, 200]
    q, k, v = (randn(g, 360, 2, 64).to(dt) for _ in range(3))
    cu = offsets(lens)
    want = srdit.ops.packed_attn(q, k, v, cu, causal=causal)
    k[70:160] = float("nan")
    v[70:160] = float("inf")
    got = srdit.ops.packed_attn(q, k, v, cu, causal=causal)
    assert torch.equal(got[:70], want[:70]) and torch.equal(got[160:], want[160:])
    assert got[70:160].isnan().all()


# ------------------------------------------------------------------ calls
@pytest.mark.parametrize("code", CODES)
def test_together(srdit, cuda_device, code):
    """Prompts by packed_attn, their keys written, then chunks and single tokens over the cache:
    what a server does. Every answer is attention over all tokens so far."""
    g, dt = gen(30), torch.bfloat16
    H, Hkv, D, page = 8, 2, 128, 16
    prompt, steps = [50, 0, 211], ([20, 33, 0], [1, 1, 1], [1, 1, 1])
    total = [sum(x) for x in zip(prompt, *steps)]
    cache = Cache(g, total, Hkv, D, page, code or dt, "heads")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")

    def rows(n):
        return (randn(g, n, H, D).to(dt), *randn(g, 2, n, Hkv, D).to(dt))

    q, k, v = rows(sum(prompt))
    cu = offsets(prompt)
    out = srdit.ops.packed_attn(q, k, v, cu)
    check_packed(q, k, v, cu, cu, out, True, D ** -0.5)
    cache.lens = list(prompt)
    lens += cu[1:] - cu[:-1]
    srdit.ops.kv_write(k, v, cache.k, cache.v, cache.table, lens, cu_q=cu, **cache.scales)
    for new in steps:
        q, k, v = rows(sum(new))
        cu = offsets(new)
        lens += cu[1:] - cu[:-1]
        cache.lens = [a + b for a, b in zip(cache.lens, new)]
        one = max(new) == 1
        kw = dict() if one else dict(cu_q=cu)
        srdit.ops.kv_write(k, v, cache.k, cache.v, cache.table, lens, **kw, **cache.scales)
        out = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, lens, max_q=max(new), **kw,
                                   **cache.scales)
        check_paged(cache, q, cu, out, True, D ** -0.5)
    k, v = srdit.ops.kv_read(cache.k, cache.v, cache.table, offsets(total), total=sum(total),
                             **cache.scales)
    q = randn(g, sum(total), H, D).to(dt)
    out = srdit.ops.packed_attn(q, k, v, offsets(total))
    check_packed(q, k, v, offsets(total), offsets(total), out, True, D ** -0.5)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("new", ([1, 1], [200, 30]))
def test_graph_streams_and_repeats(srdit, cuda_device, code, new):
    """Two captured graphs whose replays overlap, another stream, the same answer every time;
    lengths that change between replays."""
    g, dt = gen(31), torch.bfloat16
    cache = Cache(g, [3000, 1700], 2, 128, 16, code or dt, "heads").fill(g, dt)
    cu, H = offsets(new), 8
    qs = [randn(g, sum(new), H, 128).to(dt) for _ in range(2)]
    outs = [torch.empty_like(q) for q in qs]
    lens = cache.lens_dev

    def call(i):
        return srdit.ops.paged_attn(qs[i], cache.k, cache.v, cache.table, lens, outs[i], cu_q=cu,
                                    max_q=max(new), **cache.scales)

    want = [call(i).clone() for i in range(2)]
    graphs = []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            call(i)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    lens.copy_(torch.tensor([900, 250], dtype=torch.int32))
    graphs[0].replay()
    cache.lens = [900, 250]
    check_paged(cache, qs[0], cu, outs[0], True, 128 ** -0.5)
    lens.copy_(torch.tensor([-4, 1 << 30], dtype=torch.int32))   # none, and all that pages hold
    graphs[0].replay()
    assert (outs[0][:new[0]] == 0).all()


def test_refusals(srdit, cuda_device):
    ops, err = srdit.ops, srdit._lib.SrditError
    g, dt = gen(40), torch.bfloat16
    c = Cache(g, [40, 50], 2, 64, 16, torch.int8).fill(g, dt)
    q = randn(g, 2, 4, 64).to(dt)
    k = randn(g, 2, 2, 64).to(dt)
    ok = lambda **kw: ops.paged_attn(**{**dict(q=q, k_pages=c.k, v_pages=c.v,  # noqa: E731
                                               page_table=c.table, kv_lens=c.lens_dev,
                                               **c.scales), **kw})
    ok()
    bad = [dict(q=q.float()), dict(q=q[0]), dict(q=q[..., :48]), dict(k_scale=None),
           dict(k_scale=c.ks.double()), dict(v_scale=c.vs[:1]), dict(page_table=c.table.long()),
           dict(page_table=c.table[:1]), dict(kv_lens=c.lens_dev.long()), dict(kv_lens=c.lens_dev[:1]),
           dict(cu_q=offsets([1])), dict(v_pages=c.v[:1]), dict(v_pages=c.v.view(torch.uint8)),
           dict(q=randn(g, 2, 3, 64).to(dt)), dict(out=q[:1]), dict(scale=0.0), dict(max_q=-1),
           dict(q=q.cpu()), dict(q=randn(g, 3, 4, 64).to(dt)),
           dict(k_pages=c.k[:, :15], v_pages=c.v[:, :15], k_scale=c.ks[:, :15], v_scale=c.vs[:, :15]),
           dict(k_pages=c.k[..., :56], v_pages=c.v[..., :56], q=q[..., :56])]
    for kw in bad:
        with pytest.raises(err):
            ok(**kw)
    wr = lambda **kw: ops.kv_write(**{**dict(k=k, v=k, k_pages=c.k, v_pages=c.v,  # noqa: E731
                                             page_table=c.table, kv_lens=c.lens_dev, **c.scales),
                                      **kw})
    wr()
    for kw in (dict(k=k.float(), v=k.float()), dict(v=k[:1]), dict(k=k[:, :1], v=k[:, :1]),
               dict(k_scale=None), dict(kv_lens=c.lens_dev.float()), dict(cu_q=offsets([2])),
               dict(k_pages=c.k.float(), v_pages=c.v.float()), dict(k=randn(g, 3, 2, 64).to(dt),
                                                                    v=randn(g, 3, 2, 64).to(dt))):
        with pytest.raises(err):
            wr(**kw)
    rd = lambda **kw: ops.kv_read(**{**dict(k_pages=c.k, v_pages=c.v, page_table=c.table,  # noqa: E731
                                            cu_k=offsets([4, 5]), total=9, **c.scales), **kw})
    rd()
    for kw in (dict(total=None), dict(v=k), dict(k=k, v=k), dict(dtype=torch.float32),
               dict(cu_k=offsets([9])), dict(v_scale=None)):
        with pytest.raises(err):
            rd(**kw)
    x = randn(g, 9, 2, 64).to(dt)
    pk = lambda **kw: ops.packed_attn(**{**dict(q=x, k=x, v=x, cu_q=offsets([9])), **kw})  # noqa: E731
    pk()
    for kw in (dict(k=x[:8], v=x[:8]), dict(v=x[:, :1]), dict(k=x.half()), dict(q=x[0]),
               dict(cu_q=offsets([9]).long()), dict(cu_k=offsets([4, 5])), dict(out=x.half()),
               dict(k=x[..., :60], v=x[..., :60], q=x[..., :60]), dict(scale=-1.0)):
        with pytest.raises(err):
            pk(**kw)


# ------------------------------------------------------------------ values that are not finite
def _poison(g, cache, code, b, token, what):
    """Make a cached token's value of key head 1 not finite: an element, a scale, a code."""
    page, row = cache.places(b, token, token + 1)
    if code is None:
        cache.v[page, row, 1, 3] = what
    elif code == torch.float8_e4m3fn and what != what:
        cache.v.view(torch.uint8)[page, row, 1, 3] = 0x7F
    else:
        cache.vs[page, row, 1] = what


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("what", (float("nan"), float("inf")))
@pytest.mark.parametrize("new,lens,at", [
    ([4, 3], [70, 35], 68), ([7, 1], [23, 9], 17), ([130, 20], [400, 90], 300),
    ([260, 5], [260, 300], 129), ([200, 77], [1000, 77], 999)])
def test_hidden_values_may_be_anything(srdit, cuda_device, code, what, new, lens, at):
    """A value that a causal mask hides from a query is not in its answer, finite or not; the
    queries that see it get no finite one."""
    g, dt = gen(50), torch.bfloat16
    cache = Cache(g, lens, 2, 64, 16, code or dt).fill(g, dt)
    cu, H = offsets(new), 4
    q = randn(g, sum(new), H, 64).to(dt)

    def call():
        return srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                                    max_q=max(new), **cache.scales)

    want = call()
    check_paged(cache, q, cu, want, True, 64 ** -0.5)
    _poison(g, cache, code, 0, at, what)
    got = call()
    see = at - (lens[0] - new[0])   # the first query that sees it
    rest = torch.ones(sum(new), H, dtype=torch.bool, device="cuda")
    rest[max(see, 0):new[0], 2:] = False
    assert torch.equal(got[rest], want[rest])
    assert (~got[~rest].isfinite()).any(-1).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("new,lens,at", [
    ([4, 3], [70, 35], 68), ([7, 1], [23, 9], 17), ([130, 20], [400, 90], 300),
    ([260, 5], [260, 300], 129), ([200, 77], [1000, 77], 999)])
@pytest.mark.parametrize("size", (20, 96))
@pytest.mark.parametrize("D", (64, 128))
def test_a_token_of_another_size(srdit, cuda_device, dtype, code, new, lens, at, size, D):
    """A token with values of 2^96 and keys of 2^20 or 2^96 (fp16: 2^14) times the others' size, which
    a causal mask hides from some queries: those get what they would without it. The others' score
    of it is beyond all others: it is all of their answer, or none (many rows over keys in 16 bits:
    where scores are below 2^28)."""
    g, big = gen(53), 96 if dtype == torch.bfloat16 else 14
    cache = Cache(g, lens, 2, D, 16, code or dtype).fill(g, dtype)
    k, v = randn(g, 2, 1, 2, D).clamp(-3, 3)
    cache.put(0, at, (k * 2.0 ** min(size, big)).to(dtype), (v * 2.0 ** big).to(dtype))
    cu, H, n, scale = offsets(new), 4, new[0], D ** -0.5
    q = randn(g, sum(new), H, D).to(dtype)
    out = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                               max_q=max(new), **cache.scales)
    K, _, _ = cache.rows(0, "k")
    V, codes, vs = cache.rows(0, "v")
    s = torch.stack([q[:n, h].double() @ K[at, h // 2] for h in range(H)], 1) * scale
    see = torch.arange(n, device="cuda")[:, None] >= at - (lens[0] - n)
    none, all_ = ~see | (s < -300), see & (s > 300)
    if code is None and max(new) > 8 and s.abs().max() > 2.0 ** 28:
        none, all_ = (~see).expand(n, H), torch.zeros_like(all_)
    else:
        assert (none | all_).sum() > 0.7 * n * H and (all_.any() or see.sum() < 8)
    # without the token: the formula, and no term of its size in the tolerance
    gone = torch.zeros(lens[0], dtype=torch.bool, device="cuda")
    gone[at] = True
    K0, V0 = (x.masked_fill(gone[:, None, None], 0) for x in (K, V))
    if vs is not None:
        vs = vs.masked_fill(gone[:, None], 0)
    u_p = U[dtype if code is None else torch.float16]
    ref, tol = attention(q[:n], K0, V0, scale, True, u_p, dtype, codes, vs, gone)
    err = (out[:n].double() - ref).abs()
    assert (err <= tol)[none].all(), float((err / tol)[none].max())
    # with it alone: its values, a weight of 1 rounded, the output rounded
    ref = V[at].repeat_interleave(2, 0).expand(n, H, D)
    tol = (u_p + 2.0 ** -11 + U[dtype] * (1 + 2.0 ** -6)) * ref.abs() + 2.0 ** -24
    if code is not None:
        tol = tol + 2.0 ** -11 * ref.abs() + 2.0 ** -24 * cache.rows(0, "v")[2][at].max()
    err = (out[:n].double() - ref).abs()
    assert (err <= tol)[all_].all(), float((err / tol)[all_].max())


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("what", (float("nan"), -float("inf")))
@pytest.mark.parametrize("at", (0, 100, 255, 256, 511))
def test_hidden_values_of_a_prompt(srdit, cuda_device, dtype, what, at):
    g = gen(51)
    q, k, v = (randn(g, 512, 2, 64).to(dtype) for _ in range(3))
    cu = offsets([512])
    want = srdit.ops.packed_attn(q, k, v, cu)
    v[at, 1, 7] = what
    got = srdit.ops.packed_attn(q, k, v, cu)
    rest = torch.ones(512, 2, dtype=torch.bool, device="cuda")
    rest[at:, 1] = False
    assert torch.equal(got[rest], want[rest])
    assert (~got[~rest].isfinite()).any(-1).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("new,lens,at", [
    ([4, 3], [70, 35], 0), ([4, 3], [70, 35], 66), ([7, 1], [200, 9], 192), ([130, 20], [400, 90], 12),
    ([130, 20], [400, 90], 390), ([260, 5], [300, 300], 299), ([90, 77], [128, 77], 127)])
def test_seen_values_that_are_not_finite(srdit, cuda_device, dtype, code, causal, new, lens, at):
    """A query that sees a value that is not finite does not get a finite answer, whatever else
    its block of keys has: ends of sequences, whole blocks."""
    g = gen(52)
    cache = Cache(g, lens, 2, 64, 16, code or dtype).fill(g, dtype)
    cu, H = offsets(new), 4
    q = randn(g, sum(new), H, 64).to(dtype)
    for what in (float("nan"), float("inf")):
        _poison(g, cache, code, 0, at, what)
        out = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                                   max_q=max(new), causal=causal, **cache.scales)
        see = max(at - (lens[0] - new[0]), 0) if causal else 0
        assert (~out[see:new[0], 2:].isfinite()).any(-1).all()
        assert out[:, :2].isfinite().all() and out[new[0]:].isfinite().all()
