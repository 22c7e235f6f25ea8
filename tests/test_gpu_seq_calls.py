"""The two ways from tensors to the C entries of the paged cache and packed attention: the
extension's and the wrappers' own. They give the same bytes and refuse the same calls."""
import pytest
import torch

from tests.seq_cases import Cache, gen, offsets, randn

pytestmark = pytest.mark.gpu


@pytest.fixture
def both(srdit, monkeypatch):
    """f by the extension (which has to take it, where `taken`) and by the wrappers' own checks."""
    ops, lib = srdit.ops, srdit._lib
    ext = lib.calls()
    assert ext is not None

    def run(f, taken=True):
        out = []
        for calls in (ext, None):
            monkeypatch.setattr(ops, "_calls", calls)
            if calls is not None and taken:
                with monkeypatch.context() as m:
                    m.setattr(ops, "_same_device", None)   # the long way would fail
                    out.append(f())
            else:
                out.append(f())
        return out

    return run


def _same(a, b):
    for x, y in zip(a, b, strict=True):
        assert x.dtype == y.dtype and x.shape == y.shape
        assert torch.equal(x.reshape(-1).view(torch.uint8), y.reshape(-1).view(torch.uint8))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("code", (torch.int8, torch.float8_e4m3fn, None))
@pytest.mark.parametrize("cu", (True, False))
def test_cache(srdit, cuda_device, both, dtype, code, cu):
    ops, g = srdit.ops, gen(80)
    cache = Cache(g, [30, 17], 2, 64, 16, code or dtype, "both").fill(g, dtype)
    k, v = randn(g, 4, 2, 64).to(dtype), randn(g, 4, 2, 64).to(dtype)
    q = randn(g, 4, 4, 64).to(dtype)
    off = offsets([2, 2]) if cu else None
    start = [x.clone() for x in (cache.k, cache.v)]

    def call():
        for x, y in zip((cache.k, cache.v), start):
            x.view(torch.uint8).copy_(y.view(torch.uint8)) if code else x.copy_(y)
        n = ops.Stats.launches
        ops.kv_write(k, v, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=off, **cache.scales)
        a, b = ops.kv_read(cache.k, cache.v, cache.table, offsets([30, 17]), total=47, dtype=dtype,
                           **cache.scales)
        o = ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=off, max_q=2,
                           **cache.scales)
        o2 = ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, torch.empty_like(q),
                            cu_q=off, causal=False, scale=0.3, **cache.scales)
        assert ops.Stats.launches == n + 4
        return a, b, o, o2

    _same(*both(call))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_packed(srdit, cuda_device, both, dtype):
    g = gen(81)
    q = randn(g, 90, 4, 128).to(dtype)
    kv = randn(g, 90, 2, 2, 128).to(dtype)
    cu, cu_k = offsets([40, 50]), offsets([10, 80])
    out = torch.empty(90, 6, 128, dtype=dtype, device="cuda")[:, 1:5]
    _same(*both(lambda: (srdit.ops.packed_attn(q, kv[:, 0], kv[:, 1], cu),
                         srdit.ops.packed_attn(q, kv[:, 0], kv[:, 1], cu, out, cu_k=cu_k, scale=0.1,
                                               causal=False).clone())))


def test_calls_with_a_workspace_go_the_long_way(srdit, cuda_device, both):
    g, dt = gen(82), torch.bfloat16
    cache = Cache(g, [20000], 2, 64, 16, dt).fill(g, dt)
    q = randn(g, 40, 4, 64).to(dt)
    n = srdit.ops.Stats.launches
    _same(*[(x,) for x in both(lambda: srdit.ops.paged_attn(
        q, cache.k, cache.v, cache.table, cache.lens_dev, **cache.scales), taken=False)])
    assert srdit.ops.Stats.launches == n + 4


def test_refusals_are_the_same(srdit, cuda_device, monkeypatch):
    ops, err, g, dt = srdit.ops, srdit._lib.SrditError, gen(83), torch.bfloat16
    c = Cache(g, [40, 50], 2, 64, 16, torch.int8).fill(g, dt)
    q, k = randn(g, 2, 4, 64).to(dt), randn(g, 2, 2, 64).to(dt)
    lens, ext = c.lens_dev, srdit._lib.calls()
    bad = [
        lambda: ops.kv_write(k, k.half(), c.k, c.v, c.table, lens, **c.scales),
        lambda: ops.kv_write(k, k, c.k, c.v, c.table, lens.cpu(), **c.scales),
        lambda: ops.kv_write(k, k, c.k, c.v, c.table, lens[:1], **c.scales),
        lambda: ops.kv_write(k.transpose(1, 2).contiguous().transpose(1, 2), k, c.k, c.v, c.table,
                             lens, **c.scales),
        lambda: ops.kv_write(k, k, c.k[:, ::2], c.v[:, ::2], c.table, lens, k_scale=c.ks[:, ::2],
                             v_scale=c.vs[:, ::2]),
        lambda: ops.kv_read(c.k, c.v, c.table, offsets([1, 1]), k.expand(2, 2, 64), k[:1], **c.scales),
        lambda: ops.paged_attn(q, c.k, c.v, c.table.t(), lens, **c.scales),
        lambda: ops.paged_attn(q, c.k, c.v, c.table, lens, scale=-1.0, **c.scales),
        lambda: ops.paged_attn(q, c.k, c.v, c.table, lens, max_q=-3, **c.scales),
        lambda: ops.paged_attn(q, c.k, c.v, c.table, lens, q.half(), **c.scales),
        lambda: ops.paged_attn(q, c.k, c.v, c.table, lens, k_scale=c.ks, v_scale=None),
        lambda: ops.paged_attn(q[..., :48], c.k, c.v, c.table, lens, **c.scales),
        lambda: ops.packed_attn(k, k, k, offsets([1, 1]), scale=0.0),
        lambda: ops.packed_attn(k, k, k, offsets([1, 1])[::1].float()),
        lambda: ops.packed_attn(k, k[:1], k[:1], offsets([1, 1]))]
    for f in bad:
        said = []
        for calls in (ext, None):
            monkeypatch.setattr(ops, "_calls", calls)
            with pytest.raises(err) as e:
                f()
            said.append(str(e.value))
        assert said[0] == said[1]


def test_other_number_types(srdit, cuda_device, both):
    """Scales and sizes that are no plain float or int go the long way, with the same result."""
    g, dt = gen(84), torch.bfloat16
    c = Cache(g, [40], 2, 64, 16, dt).fill(g, dt)
    q = randn(g, 1, 4, 64).to(dt)
    for kw in (dict(scale=1), dict(max_q=True), dict(causal=1)):
        _same(*[(x,) for x in both(lambda: srdit.ops.paged_attn(q, c.k, c.v, c.table, c.lens_dev, **kw),
                                   taken=False)])
