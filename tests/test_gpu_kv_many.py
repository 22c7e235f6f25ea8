"""The paged cache with more sequences than a warp has lanes: everything that is stored and read."""
import pytest
import torch

from tests.seq_cases import Cache, gen, offsets, quantise, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", (torch.int8, torch.float8_e4m3fn, None))
@pytest.mark.parametrize("B", (32, 33, 1024, 1025, 1050))
def test_codes_scales_and_both_sides(srdit, cuda_device, code, B):
    """From a cache with nothing in it: codes and scales of k and v are stored by the call, and both
    are read back."""
    g, dt = gen(90 + B), torch.bfloat16
    new = [(i * 7) % 3 for i in range(B)]
    old = [i % 2 for i in range(B)]
    lens = [n + o for n, o in zip(new, old)]
    cache = Cache(g, lens, 2, 48, 16, code or dt)
    held = [x for x in (cache.k, cache.v, cache.ks, cache.vs) if x is not None]
    T, cu = sum(new), offsets(new, 2)
    kv = randn(g, T + 5, 2, 2, 48).to(dt)
    srdit.ops.kv_write(kv[:, 0], kv[:, 1], cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                       **cache.scales)
    at = [cache.places(b, o, o + n) for b, (o, n) in enumerate(zip(old, new)) if n]
    pages, rows = (torch.cat(x) for x in zip(*at))
    if code:
        (k, ks), (v, vs) = (quantise(kv[2:2 + T, i], code) for i in (0, 1))
        want = [k, v, ks, vs]
        values = [(x.float() * s[..., None]).to(dt) for x, s in ((k, ks), (v, vs))]
    else:
        want = values = [kv[2:2 + T, 0], kv[2:2 + T, 1]]
    for x, y in zip(held, want, strict=True):
        got = x[pages, rows] if x.itemsize > 1 else x.view(torch.uint8)[pages, rows].view(x.dtype)
        assert torch.equal(got.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))
    # the sequences whose new tokens are their first
    first = [n if o == 0 else 0 for o, n in zip(old, new)]
    mine = torch.cat([torch.arange(int(cu[b]) - 2, int(cu[b]) - 2 + n) for b, n in enumerate(first)])
    k, v = (torch.full((sum(first) + 4, 2, 48), 5.0, dtype=dt, device="cuda") for _ in range(2))
    srdit.ops.kv_read(cache.k, cache.v, cache.table, offsets(first, 1), k, v, **cache.scales)
    for x, y in zip((k, v), values):
        assert torch.equal(x[1:1 + len(mine)], y[mine.cuda()])
        assert (x[:1] == 5).all() and (x[1 + len(mine):] == 5).all()
