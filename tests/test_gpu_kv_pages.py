"""Writing tokens into a paged cache and reading them back, bit for bit, and what is beside them."""
import pytest
import torch

from tests.seq_cases import Cache, gen, offsets, quantise, randn

pytestmark = pytest.mark.gpu

HALF = (torch.bfloat16, torch.float16)
CODES = (torch.int8, torch.float8_e4m3fn, None)


def _bytes(t):
    return t.clone(memory_format=torch.contiguous_format).reshape(-1).view(torch.uint8)


def _clone(c):
    return [None if x is None else x.clone() for x in (c.k, c.v, c.ks, c.vs)]


def _same(a, b):
    return all((x is None) == (y is None) and (x is None or torch.equal(_bytes(x), _bytes(y)))
               for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("new,lens,Hkv,D,page,layout", [
    ([1], [1], 1, 16, 16, "tokens"), ([1, 1, 1], [5, 16, 17], 8, 128, 16, "heads"),
    ([0, 40, 7], [9, 131, 7], 3, 80, 32, "both"), ([130, 0, 1], [130, 0, 2304], 5, 64, 128, "heads"),
    ([2305], [4610], 2, 96, 2304, "tokens"), ([3, 0, 0, 0], [64, 3, 0, 1], 24, 112, 64, "both"),
    ([1] * 70, list(range(1, 71)), 2, 32, 16, "tokens")])
def test_write_then_read(srdit, cuda_device, dtype, code, new, lens, Hkv, D, page, layout):
    g = gen(sum(lens) + D)
    cache = Cache(g, lens, Hkv, D, page, code or dtype, layout)
    for b, n in enumerate(lens):   # what was there before
        old = n - new[b]
        cache.put(b, 0, randn(g, old, Hkv, D).to(dtype), randn(g, old, Hkv, D).to(dtype))
    T = sum(new)
    kv = (randn(g, T, 2, Hkv, D) * torch.exp(randn(g, T, 2, Hkv, 1))).to(dtype)
    if T > 4:
        kv[2] = 0
        kv[3] = 1e-30
    cu, state = offsets(new), _clone(cache)
    srdit.ops.kv_write(kv[:, 0], kv[:, 1], cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                       **cache.scales)
    got = _clone(cache)
    for x, old in zip((cache.k, cache.v, cache.ks, cache.vs), state):
        if x is not None:
            x.view(torch.uint8).copy_(old.view(torch.uint8)) if x.dtype in CODES else x.copy_(old)
    for b, n in enumerate(lens):
        rows = kv[int(cu[b]):int(cu[b + 1])]
        cache.put(b, n - new[b], rows[:, 0], rows[:, 1])
    assert _same(got, _clone(cache))   # every byte of the pool, those beside the rows too
    cu_k = offsets(lens)
    k, v = srdit.ops.kv_read(cache.k, cache.v, cache.table, cu_k, total=sum(lens), dtype=dtype,
                             **cache.scales)
    for which, x in (("k", k), ("v", v)):
        for b, n in enumerate(lens):
            _, codes, s = cache.rows(b, which)
            want = (cache.rows(b, which)[0].to(dtype) if codes is None
                    else (codes.float() * s.float()[..., None]).to(dtype))
            assert torch.equal(_bytes(x[int(cu_k[b]):int(cu_k[b + 1])]), _bytes(want)), (which, b)


@pytest.mark.parametrize("code", CODES)
def test_rows_behind_and_tokens_without_a_page(srdit, cuda_device, code):
    """A padded batch: rows behind the last sequence are nobody's. Tokens before the first, or in
    pages that the table does not have, are not written and read as zeros."""
    g, dt = gen(3), torch.bfloat16
    cache = Cache(g, [40, 20], 2, 64, 16, code or dt, "heads")
    cache.table[0, 1] = -1                        # tokens 16 to 31
    cache.table[1, 1] = cache.k.shape[0]          # tokens 16 to 19
    state = _clone(cache)
    k, v = randn(g, 100, 2, 64).to(dt), randn(g, 100, 2, 64).to(dt)
    cu = torch.tensor([2, 42, 72], dtype=torch.int32, device="cuda")
    lens = torch.tensor([40, 20], dtype=torch.int32, device="cuda")   # 30 new of 20: 10 left out
    srdit.ops.kv_write(k, v, cache.k, cache.v, cache.table, lens, cu_q=cu, **cache.scales)
    got = _clone(cache)
    for x, old in zip((cache.k, cache.v, cache.ks, cache.vs), state):
        if x is not None:
            x.view(torch.uint8).copy_(old.view(torch.uint8)) if x.dtype in CODES else x.copy_(old)
    good = cache.table.clone()
    cache.put(0, 0, k[2:18], v[2:18])
    cache.put(0, 32, k[34:42], v[34:42])
    cache.put(1, 0, k[52:68], v[52:68])
    assert _same(got, _clone(cache)) and torch.equal(good, cache.table)
    ko, vo = (torch.full((70, 2, 64), 7.0, dtype=dt, device="cuda") for _ in range(2))
    cu_k = torch.tensor([0, 40, 60], dtype=torch.int32, device="cuda")
    srdit.ops.kv_read(cache.k, cache.v, cache.table, cu_k, ko, vo, **cache.scales)
    for x in (ko, vo):
        assert (x[60:] == 7).all() and (x[16:32] == 0).all() and (x[56:60] == 0).all()
        assert (x[:16] != 0).any() and (x[32:56] != 0).any()


@pytest.mark.parametrize("code", (torch.int8, torch.float8_e4m3fn))
def test_rows_of_zeros_infinities_and_nan(srdit, cuda_device, code):
    g, dt = gen(9), torch.bfloat16
    cache = Cache(g, [6], 1, 32, 16, code)
    k = randn(g, 6, 1, 32).to(dt)
    k[0] = 0
    k[1, 0, 3] = float("nan")
    k[2, 0, 5] = -float("inf")
    k[3] = 3e38
    v = k.flip(0)
    srdit.ops.kv_write(k, v, cache.k, cache.v, cache.table, cache.lens_dev, **cache.scales)
    x, y = srdit.ops.kv_read(cache.k, cache.v, cache.table, offsets([6]), total=6, **cache.scales)
    assert torch.equal(_bytes(y), _bytes(x.flip(0)))
    assert (x[0] == 0).all() and x[1:3].isnan().all()
    assert (x[3].float() >= 2.9e38).all() and x[4:].isfinite().all()
    page, row = cache.places(0, 0, 6)
    s = cache.ks[page, row][:, 0]
    assert s[0] == 1e-12 and s[1].isnan() and s[2] == float("inf")


def test_without_offsets_and_rows_of_other_strides(srdit, cuda_device):
    """T / B tokens each; k, v as parts of a wider projection, one key head for all (stride 0)."""
    g, dt = gen(11), torch.float16
    cache = Cache(g, [20, 33, 48], 4, 64, 16, torch.int8)
    ref = Cache(gen(11), [20, 33, 48], 4, 64, 16, torch.int8)
    wide = randn(g, 9, 3, 8, 72).to(dt)
    k, v = wide[:, 1, 2:6, :64], wide[:, 2, 4:5, 8:].expand(9, 4, 64)
    srdit.ops.kv_write(k, v, cache.k, cache.v, cache.table, cache.lens_dev, **cache.scales)
    for b, n in enumerate(cache.lens):
        ref.put(b, n - 3, k[3 * b:3 * b + 3], v[3 * b:3 * b + 3])
    assert _same(_clone(cache), _clone(ref))


def test_offsets_beyond_32_bits(srdit, cuda_device):
    """A pool of 2.4e9 codes: its last pages."""
    g, dt = gen(12), torch.bfloat16
    n, P, H, D = 9200, 128, 16, 128
    pool = torch.zeros(2, n, P, H, D, dtype=torch.int8, device="cuda")
    scale = torch.zeros(2, n, P, H, device="cuda")
    table = torch.tensor([[n - 1, 0, n - 2]], dtype=torch.int32, device="cuda")
    k, v = randn(g, 300, H, D).to(dt), randn(g, 300, H, D).to(dt)
    lens = torch.tensor([300], dtype=torch.int32, device="cuda")
    srdit.ops.kv_write(k, v, pool[0], pool[1], table, lens, k_scale=scale[0], v_scale=scale[1])
    q, s = quantise(k, torch.int8)
    assert torch.equal(pool[0, n - 1], q[:128]) and torch.equal(pool[0, 0], q[128:256])
    assert torch.equal(pool[0, n - 2, :44], q[256:]) and torch.equal(scale[0, n - 2, :44], s[256:])
    assert not pool[:, 1:n - 2].any()
    x, y = srdit.ops.kv_read(pool[0], pool[1], table, offsets([300]), total=300, k_scale=scale[0],
                             v_scale=scale[1])
    assert torch.equal(x, (q.float() * s[..., None]).to(dt))
    qv, sv = quantise(v, torch.int8)
    assert torch.equal(y, (qv.float() * sv[..., None]).to(dt))


def test_in_a_graph_and_on_another_stream(srdit, cuda_device):
    g, dt = gen(13), torch.bfloat16
    cache = Cache(g, [17, 65], 2, 128, 16, torch.float8_e4m3fn).fill(g, dt)
    k, v = randn(g, 2, 2, 128).to(dt), randn(g, 2, 2, 128).to(dt)
    ko, vo = (torch.empty(82, 2, 128, dtype=dt, device="cuda") for _ in range(2))
    cu = offsets([17, 65])

    def step():
        srdit.ops.kv_write(k, v, cache.k, cache.v, cache.table, cache.lens_dev, **cache.scales)
        srdit.ops.kv_read(cache.k, cache.v, cache.table, cu, ko, vo, **cache.scales)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    k.copy_(randn(g, 2, 2, 128))
    v.copy_(randn(g, 2, 2, 128))
    graph.replay()
    got = ko.clone(), vo.clone()
    step()
    assert torch.equal(ko, got[0]) and torch.equal(vo, got[1])
    q, s = quantise(k, torch.float8_e4m3fn)
    want = (q.float() * s[..., None]).to(dt)
    assert torch.equal(ko[16], want[0]) and torch.equal(ko[81], want[1])


@pytest.mark.parametrize("code", (torch.int8, None))
@pytest.mark.parametrize("B", (32, 33, 1050))
def test_more_sequences_than_lanes(srdit, cuda_device, code, B):
    """Where a token's sequence is found in steps; many are empty."""
    g, dt = gen(70 + B), torch.bfloat16
    new = [(i * 7) % 3 for i in range(B)]
    lens = [n + i % 2 for i, n in enumerate(new)]
    cache = Cache(g, lens, 1, 16, 16, code or dt)
    T, cu = sum(new), offsets(new, 2)
    kv = randn(g, T + 5, 2, 1, 16).to(dt)
    for b in range(B):
        rows = kv[int(cu[b]):int(cu[b + 1])]
        cache.put(b, lens[b] - new[b], rows[:, 0], rows[:, 1])
    want = _clone(cache)
    for x in (cache.k, cache.v):
        x.view(torch.uint8).zero_()
    srdit.ops.kv_write(kv[:, 0], kv[:, 1], cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                       **cache.scales)
    got = _clone(cache)
    at = [cache.places(b, lens[b] - n, lens[b]) for b, n in enumerate(new) if n]
    pages, rows = (torch.cat(x) for x in zip(*at))
    for x, y in zip(got, want):
        if x is not None:
            assert torch.equal(x[pages, rows], y[pages, rows])
    cu_k = offsets(new, 1)
    k, v = (torch.full((T + 4, 1, 16), 5.0, dtype=dt, device="cuda") for _ in range(2))
    cache.put(0, 0, kv[:lens[0], 0], kv[:lens[0], 1])
    lo = [lens[b] - n for b, n in enumerate(new)]
    srdit.ops.kv_read(cache.k, cache.v, cache.table, cu_k, k, v, **cache.scales)
    for b, n in enumerate(new):
        if lo[b] == 0 and n:   # the first tokens, that were written
            first = int(cu_k[b])
            c = cache.rows(b, "k")[0][:n]
            assert torch.equal(k[first:first + n].double(), c.to(dt).double())
    assert (k[:1] == 5).all() and (k[1 + T:] == 5).all() and (v[1 + T:] == 5).all()
