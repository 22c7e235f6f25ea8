"""Attention over pages and packed rows with many query heads per key head: as many as fill a query
tile, or more, side by side with few tokens; and sequences with more new tokens than max_q says."""
import pytest
import torch

from tests.seq_cases import Cache, check_packed, check_paged, gen, offsets, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", (16, 17, 24, 32, 64, 96, 128, 256))
@pytest.mark.parametrize("code", (torch.int8, torch.float8_e4m3fn, None))
@pytest.mark.parametrize("dtype,D,Hkv", ((torch.bfloat16, 128, 1), (torch.float16, 64, 2)))
def test_groups_over_pages(srdit, cuda_device, group, code, dtype, D, Hkv):
    """Single tokens and a few of them."""
    g = gen(group + D)
    cache = Cache(g, [300, 0, 1, 515, 128], Hkv, D, 16, code or dtype, "heads").fill(g, dtype)
    for new in ([1] * 5, [3, 1, 1, 70, 0], [0, 2, 9, 5, 128]):
        cu, T = offsets(new), sum(new)
        q = randn(g, T + 2, Hkv * group, D).to(dtype)
        for causal in (True, False):
            out = torch.full_like(q, 7.0)
            srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, out, cu_q=cu,
                                 causal=causal, max_q=max(new), **cache.scales)
            check_paged(cache, q, cu, out, causal, D ** -0.5)
            assert (out[T:] == 7).all()


@pytest.mark.parametrize("group,Hkv", ((16, 2), (24, 1), (64, 1), (96, 2), (128, 1), (256, 1)))
@pytest.mark.parametrize("dtype,D", ((torch.bfloat16, 64), (torch.float16, 128)))
def test_groups_of_packed_rows(srdit, cuda_device, group, Hkv, dtype, D):
    g = gen(1000 + group)
    new, keys = [1, 40, 0, 7, 133], [130, 40, 5, 2, 300]
    cu_q, cu_k = offsets(new), offsets(keys)
    q, kv = randn(g, sum(new), Hkv * group, D).to(dtype), randn(g, sum(keys), Hkv, 2, D).to(dtype)
    k, v = kv[:, :, 0], kv[:, :, 1]
    for causal in (True, False):
        out = srdit.ops.packed_attn(q, k, v, cu_q, cu_k=cu_k, causal=causal)
        check_packed(q, k, v, cu_q, cu_k, out, causal, D ** -0.5)


@pytest.mark.parametrize("H,code", ((128, torch.float8_e4m3fn), (32, torch.int8), (32, None)))
def test_a_long_cache_shared_by_many_heads(srdit, cuda_device, H, code):
    """Key tiles in shares, whose parts are joined."""
    g, dt = gen(7 + H), torch.bfloat16
    cache = Cache(g, [9000, 20001], 1, 128, 64, code or dt).fill(g, dt)
    q = randn(g, 2, H, 128).to(dt)
    out = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, max_q=1, **cache.scales)
    check_paged(cache, q, torch.tensor([0, 1, 2]), out, True, 128 ** -0.5)


@pytest.mark.parametrize("H,keys", ((8, 200), (8, 40000), (64, 300), (64, 20000)))
@pytest.mark.parametrize("code", (torch.int8, None))
def test_more_new_tokens_than_max_q(srdit, cuda_device, H, keys, code):
    """A sequence's tokens up to max_q are answered, those of others too, and nothing is written that
    is no sequence's; what lies between may be left."""
    g, dt, most = gen(keys + H), torch.bfloat16, 2
    new, lens = [2, 9, 1, 70, 0], [keys, 77, keys // 2, keys, 5]
    cache = Cache(g, lens, 2, 64, 16, code or dt).fill(g, dt)
    cu, T = offsets(new, 1), sum(new)
    q = randn(g, T + 4, H, 64).to(dt)
    for causal in (True, False):
        out = torch.full_like(q, 7.0)
        srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, out, cu_q=cu, max_q=most,
                             causal=causal, **cache.scales)
        want = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                                    causal=causal, **cache.scales)
        check_paged(cache, q, cu, want, causal, 64 ** -0.5)
        for b, n in enumerate(new):   # the rows that may be left, as the answer
            x = slice(int(cu[b]) + min(n, most), int(cu[b]) + n)
            left = (out[x] == 7).all(-1, keepdim=True)
            out[x] = torch.where(left, want[x], out[x])
        check_paged(cache, q, cu, out, causal, 64 ** -0.5)
        assert (out[:1] == 7).all() and (out[1 + T:] == 7).all()
