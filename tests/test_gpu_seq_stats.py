"""What Stats says of the paged cache and packed attention: launches, and the work of the sequences as
they are, whatever the tensors and tables have room for."""
import pytest
import torch

from tests.seq_cases import Cache, gen, offsets, randn

pytestmark = pytest.mark.gpu
DT = torch.bfloat16


@pytest.fixture
def events(srdit, monkeypatch):
    monkeypatch.setattr(srdit.ops.Stats, "events", [])
    return srdit.ops.Stats.events


def _pairs(n, L, causal):
    return sum(1 for i in range(n) for j in range(L) if not causal or j <= L - n + i)


@pytest.mark.parametrize("code", (torch.int8, None))
def test_cache(srdit, cuda_device, events, code):
    g = gen(120)
    cache = Cache(g, [40, 0, 9], 2, 64, 16, code or DT, width=50).fill(g, DT)
    new = [5, 0, 9]
    k, v = randn(g, 17, 2, 64).to(DT), randn(g, 17, 2, 64).to(DT)   # 3 rows behind the last sequence
    srdit.ops.kv_write(k, v, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=offsets(new),
                       **cache.scales)
    srdit.ops.kv_read(cache.k, cache.v, cache.table, offsets([7, 0, 2]), k, v, **cache.scales)
    row = 64 * 2 + (64 + 4 if code else 64 * 2)
    assert [(e[0], e[3]) for e in events] == [("kv_write", 14 * 2 * 2 * row), ("kv_read", 9 * 2 * 2 * row)]


@pytest.mark.parametrize("causal", (True, False))
def test_paged(srdit, cuda_device, events, causal):
    g, lens, new = gen(121), [40, 0, 9, 30], [5, 0, 12, 1]   # 12 of 9: the first three see nothing
    cache = Cache(g, lens, 2, 64, 16, DT, width=50).fill(g, DT)
    q = randn(g, 20, 4, 64).to(DT)
    for kw in ({}, dict(max_q=12, max_kv=64)):
        srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=offsets(new),
                             causal=causal, **kw)
    want = 4 * 4 * 64 * sum(_pairs(n, L, causal) for n, L in zip(new, lens))
    assert [(e[0], e[3]) for e in events] == [("paged_attn", want)] * 2
    del events[:]
    srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, causal=causal)   # 5 each
    assert events[0][3] == 4 * 4 * 64 * sum(_pairs(5, L, causal) for L in lens)


@pytest.mark.parametrize("causal", (True, False))
def test_packed(srdit, cuda_device, events, causal):
    g, new, lens = gen(122), [30, 0, 50], [10, 4, 70]
    q, kv = randn(g, 85, 4, 64).to(DT), randn(g, 85, 2, 2, 64).to(DT)
    srdit.ops.packed_attn(q, kv[:, 0], kv[:, 1], offsets(new), causal=causal)
    srdit.ops.packed_attn(q, kv[:, 0], kv[:, 1], offsets(new), cu_k=offsets(lens), causal=causal)
    assert [(e[0], e[3]) for e in events] == [
        ("packed_attn", 4 * 4 * 64 * sum(_pairs(n, L, causal) for n, L in zip(new, ks)))
        for ks in (new, lens)]


def test_calls_are_counted_alike_with_and_without_events(srdit, cuda_device, monkeypatch):
    g, ops = gen(123), srdit.ops
    cache = Cache(g, [20000], 2, 64, 16, DT).fill(g, DT)
    for n in (1, 40):   # without and with a second kernel that joins parts
        q, counts = randn(g, n, 4, 64).to(DT), []
        for e in (None, []):
            monkeypatch.setattr(ops.Stats, "events", e)
            before = ops.Stats.launches
            ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev)
            counts.append(ops.Stats.launches - before)
        assert counts[0] == counts[1]
