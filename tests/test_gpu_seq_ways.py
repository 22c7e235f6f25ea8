"""Every way that attention of packed sequences is run in, at sizes that reach it (asked of the
library), against the formula in 64 bits."""
import ctypes

import pytest
import torch

from tests.seq_cases import Cache, check_packed, check_paged, gen, offsets, randn

pytestmark = pytest.mark.gpu

CODES = (torch.int8, torch.float8_e4m3fn, None)


@pytest.fixture
def way(srdit, monkeypatch):
    """The way of the last call."""
    seen = {}
    real = srdit.ops._launch

    def launch(name, *args, **kw):
        if name == "srdit_seq_attn":
            seen["way"] = srdit._lib.count("srdit_seq_attn_way", args[0])
        return real(name, *args, **kw)

    monkeypatch.setattr(srdit.ops, "_launch", launch)
    monkeypatch.setattr(srdit.ops, "_calls", None)   # by way of _launch
    return lambda: seen["way"]


def _paged(srdit, g, cache, new, H, dtype, causal=True, **kw):
    cu = offsets(new)
    q = randn(g, sum(new), H, cache.D).to(dtype)
    out = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                               causal=causal, **cache.scales, **kw)
    check_paged(cache, q, cu, out, causal, cache.D ** -0.5)
    return q, cu, out


# lengths that fill the shares of both kinds of codes; one sequence without new tokens, one
# without any, one shorter than a block
LONG = [9001, 0, 7, 30000, 12345, 100, 16, 8000]


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("new,H,D,page", [
    ([1, 0, 1, 1, 1, 0, 1, 1], 8, 128, 16), ([1, 1, 1, 1, 1, 1, 1, 1], 16, 64, 64),
    ([2, 0, 3, 1, 4, 4, 0, 2], 32, 80, 128)])
def test_shares_of_a_step(srdit, cuda_device, way, dtype, code, new, H, D, page):
    """Shares that end inside sequences, whole sequences within one; up to 16 rows a key head."""
    g = gen(60 + H)
    cache = Cache(g, LONG, 8, D, page, code or dtype, "heads").fill(g, dtype)
    _, _, out = _paged(srdit, g, cache, new, H, dtype, max_q=max(new))
    assert way() == srdit._lib.SRDIT_WAY_STEP_SHARES


def test_shares_of_one_key_head_and_of_many(srdit, cuda_device, way):
    g, dt = gen(61), torch.bfloat16
    for Hkv, lens in ((1, [100000, 250000, 33]), (24, [3000, 5000, 9000, 1, 4000])):
        cache = Cache(g, lens, Hkv, 64, 16, dt).fill(g, dt)
        _paged(srdit, g, cache, [1] * len(lens), 2 * Hkv, dt, max_q=1)
        assert way() == srdit._lib.SRDIT_WAY_STEP_SHARES


def test_shares_in_graphs_at_once(srdit, cuda_device, way):
    """Two graphs, whose workspaces are their own, replayed at the same time; lengths that change."""
    g, dt = gen(62), torch.bfloat16
    cache = Cache(g, [27000, 24000, 36000, 35000], 8, 64, 16, torch.int8).fill(g, dt)
    qs = [randn(g, 4, 16, 64).to(dt) for _ in range(2)]
    lens = [cache.lens_dev.clone() for _ in range(2)]
    lens[1] -= 700
    outs = [torch.empty_like(q) for q in qs]
    call = lambda i: srdit.ops.paged_attn(qs[i], cache.k, cache.v, cache.table, lens[i],  # noqa: E731
                                          outs[i], **cache.scales)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i in range(2):
        call(i)
        with torch.cuda.graph(graphs[i]):
            call(i)
    assert way() == srdit._lib.SRDIT_WAY_STEP_SHARES
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for i in range(2):
        cache.lens = lens[i].tolist()
        check_paged(cache, qs[i], torch.arange(5), outs[i], True, 0.125)
    lens[0].copy_(torch.tensor([0, 1, 5000, 17], dtype=torch.int32))
    graphs[0].replay()
    cache.lens = [0, 1, 5000, 17]
    check_paged(cache, qs[0], torch.arange(5), outs[0], True, 0.125)
    assert (outs[0][0] == 0).all()


def test_more_sequences_than_a_launch_by_shares_keeps(srdit, cuda_device, way):
    g, dt = gen(63), torch.bfloat16
    lens = [(7 * i) % 90 for i in range(1300)]
    cache = Cache(g, lens, 2, 64, 16, torch.int8, "heads").fill(g, dt)
    q = randn(g, 1300, 4, 64).to(dt)
    out = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, **cache.scales)
    assert way() == srdit._lib.SRDIT_WAY_STEP
    for b in list(range(0, 1300, 97)) + [1, 2, 1299]:
        one = Cache.__new__(Cache)
        one.__dict__.update(cache.__dict__, lens=[cache.lens[b]], table=cache.table[b:b + 1])
        check_paged(one, q[b:b + 1], [0, 1], out[b:b + 1], True, 0.125)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("new,lens", [([70], [20000]), ([33, 0, 90], [9000, 50, 14000])])
def test_shares_of_a_chunk(srdit, cuda_device, way, code, causal, new, lens):
    g, dt = gen(64), torch.bfloat16
    cache = Cache(g, lens, 2, 128, 16, code or dt, "heads").fill(g, dt)
    _paged(srdit, g, cache, new, 8, dt, causal)
    assert way() == srdit._lib.SRDIT_WAY_CHUNK_SHARES


@pytest.mark.parametrize("code", CODES)
def test_shares_of_the_last_round(srdit, cuda_device, way, code):
    g, dt = gen(65), torch.float16
    cache = Cache(g, [6912], 24, 64, 2304, code or dt).fill(g, dt)
    _paged(srdit, g, cache, [2304], 24, dt, False)
    assert way() == srdit._lib.SRDIT_WAY_CHUNK_REST


@pytest.mark.parametrize("causal", (True, False))
def test_more_pieces_than_are_kept(srdit, cuda_device, way, causal):
    """300 sequences, more than a warp finds at once or shared memory keeps, some empty."""
    g, dt = gen(66), torch.bfloat16
    lens = [(13 * i) % 70 if i % 7 else 0 for i in range(300)]
    T = sum(lens)
    q, k, v = randn(g, T, 4, 64).to(dt), randn(g, T, 2, 64).to(dt), randn(g, T, 2, 64).to(dt)
    cu = offsets(lens)
    out = srdit.ops.packed_attn(q, k, v, cu, causal=causal)
    check_packed(q, k, v, cu, cu, out, causal, 0.125)
    assert way() == srdit._lib.SRDIT_WAY_CHUNK


@pytest.mark.parametrize("code", (torch.float8_e4m3fn, None))
@pytest.mark.parametrize("what", (float("nan"), float("inf")))
@pytest.mark.parametrize("new,lens,at,H", [
    ([4, 1, 2], [26001, 14000, 9000], 25999, 32), ([60, 30], [15000, 9000], 14980, 8)])
def test_hidden_values_in_shares(srdit, cuda_device, way, code, what, new, lens, at, H):
    """A value that is not finite, hidden from some queries, in work that is cut."""
    g, dt = gen(67), torch.bfloat16
    Hkv = 8 if H == 32 else 2
    cache = Cache(g, lens, Hkv, 64, 16, code or dt).fill(g, dt)
    cu = offsets(new)
    q = randn(g, sum(new), H, 64).to(dt)
    call = lambda: srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev,  # noqa: E731
                                        cu_q=cu, max_q=max(new), **cache.scales)
    want = call()
    page, row = cache.places(0, at, at + 1)
    if code is None:
        cache.v[page, row, 1, 3] = what
    elif what != what:
        cache.v.view(torch.uint8)[page, row, 1, 3] = 0x7F
    else:
        cache.vs[page, row, 1] = what
    got = call()
    group, see = H // Hkv, at - (lens[0] - new[0])
    rest = torch.ones(sum(new), H, dtype=torch.bool, device="cuda")
    rest[see:new[0], group:2 * group] = False
    assert torch.equal(got[rest], want[rest]) and (~got[~rest].isfinite()).any(-1).all()
    assert way() in (srdit._lib.SRDIT_WAY_STEP_SHARES, srdit._lib.SRDIT_WAY_CHUNK_SHARES)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("D", (8, 24, 72, 120))
def test_odd_widths(srdit, cuda_device, dtype, D):
    """Widths in 16 bits that are no multiples of 16."""
    g = gen(68)
    cache = Cache(g, [70, 300], 2, D, 16, dtype).fill(g, dtype)
    _paged(srdit, g, cache, [1, 1], 8, dtype, max_q=1)
    _paged(srdit, g, cache, [60, 150], 8, dtype)
    q, k, v = (randn(g, 333, 2, D).to(dtype) for _ in range(3))
    cu = offsets([200, 133])
    check_packed(q, k, v, cu, cu, srdit.ops.packed_attn(q, k, v, cu), True, D ** -0.5)


def test_no_keys_at_all(srdit, cuda_device):
    """Packed keys of no rows, a cache of no pages, a table of no columns."""
    g, dt = gen(69), torch.bfloat16
    q = randn(g, 40, 4, 64).to(dt)
    k = torch.empty(0, 2, 64, dtype=dt, device="cuda")
    out = srdit.ops.packed_attn(q, k, k, offsets([10, 30]), cu_k=offsets([0, 0]))
    assert (out == 0).all()
    pool = torch.empty(0, 16, 2, 64, dtype=dt, device="cuda")
    for cols in (0, 3):
        table = torch.zeros(2, cols, dtype=torch.int32, device="cuda")
        for T, lens in ((2, [5, 40]), (40, [100, 3])):
            out = torch.full((T, 4, 64), 9.0, dtype=dt, device="cuda")
            srdit.ops.paged_attn(q[:T], pool, pool, table,
                                 torch.tensor(lens, dtype=torch.int32, device="cuda"), out,
                                 cu_q=offsets([T // 2, T // 2]), max_q=T // 2)
            assert (out == 0).all(), (cols, T)


def test_length_beyond_the_hint(srdit, cuda_device):
    """max_kv only says how work is split: sequences 50 times as long come out right."""
    g, dt = gen(70), torch.bfloat16
    cache = Cache(g, [5000, 300], 2, 64, 16, torch.float8_e4m3fn).fill(g, dt)
    for new in ([1, 1], [50, 60]):
        _paged(srdit, g, cache, new, 8, dt, max_q=max(new), max_kv=100)
