"""Attention over pages and of packed prompts where numbers are large or far apart: scores of any
size, and values' scales from 2^-40 to 2^100 side by side, against the formula in 64 bits.

Nothing is added for scores: q and k are such that q.k is exact in 32 bits, and the factor
c = scale * log2(e) either is a power of two (a scale of ln(2) in fp32, whose product with log2(e)
in fp32 is 1), or large scores are equal or too far apart for any rounding of c to matter (2^-24 of
2^size, 2^-7 of it apart, which is 2^13 or more). With weights p_j of sum 1, u the rounding of the
output and u_p of a weight (its type's: the queries', or fp16 over codes), an answer is off by

  (u_p + 2^-11) sum_j p_j |v_j| + u |o|    weights, the exponential's approximation; the output
  2^-25 sum_j |v_j|                        fp16 weights over values in 16 bits that are below its
                                           steps (a weight is held over the largest one)
  2^-24 w sum_j |code_j|                   the same over codes: products of weight and scale are
                                           held over the largest of them, or over the largest
                                           weight of 32 keys times the largest scale among them;
                                           w is the larger, doubled as a unit is a power of two
  2^-11 sum_j p_j |v_j|                    many rows of bf16 over codes: code times scale in fp16
                                           (keys' products are exact here)
"""
import pytest
import torch

from tests.seq_cases import U, Cache, gen, offsets, randn

pytestmark = pytest.mark.gpu

HALF = (torch.bfloat16, torch.float16)
CODES = (torch.int8, torch.float8_e4m3fn)
LN2 = 0.6931471824645996   # ln(2) in fp32


def _answer(q, k, v, c, causal, codes=None, vs=None):
    """(answer, tolerance) of one sequence in 64 bits: q [n, H, D], k, v [L, Hkv, D]."""
    n, H, D = q.shape
    L, Hkv = k.shape[:2]
    u, u_p = U[q.dtype], U[q.dtype if codes is None else torch.float16]
    out = torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    seen = torch.ones(n, L, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(L - n)
    for h in range(H):
        g = h // (H // Hkv)
        s = (q[:, h].double() @ k[:, g].t() * c).masked_fill(~seen, float("-inf"))
        p = torch.exp2(s - s.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        o, a = p @ v[:, g], p @ v[:, g].abs()
        out[:, h] = o
        tol[:, h] = (u_p + 2.0 ** -11) * a + u * o.abs() * (1 + 2.0 ** -6)
        if codes is None and u_p == U[torch.float16]:
            tol[:, h] += 2.0 ** -25 * v[:, g].abs().sum(0)
        if codes is not None:
            pad = -L % 32
            groups = torch.nn.functional.pad(p, (0, pad)).view(n, -1, 32).amax(2)
            scales = torch.nn.functional.pad(vs[:, g], (0, pad)).view(-1, 32).amax(1)
            w = (groups * scales).amax(1, keepdim=True)
            tol[:, h] += 2.0 ** -24 * w * codes[:, g].abs().sum(0)
            if q.dtype == torch.bfloat16:
                tol[:, h] += 2.0 ** -11 * a
        if q.dtype == torch.float16:
            tol[:, h] += 2.0 ** -25
    return out, tol


def _check(got, ref, tol):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (float((err / tol)[~err.isnan()].max()), int(bad.sum()), bad.numel(),
                           bad.nonzero()[:5].tolist())


def _paged(srdit, cache, q, new, c, causal, each=None):
    cu = offsets(new)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = srdit.ops.paged_attn(q, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu,
                               max_q=max(new), causal=causal, scale=LN2 * c, status=status,
                               **cache.scales)
    assert status.item() == 0
    for b, n in enumerate(new):
        if n == 0:
            continue
        v, codes, vs = cache.rows(b, "v")
        lo = int(cu[b])
        ref, tol = _answer(q[lo:lo + n], cache.rows(b, "k")[0], v, c, causal, codes, vs)
        _check(out[lo:lo + n], ref, tol)
    return out


# ------------------------------------------------------------------ scores of any size
def _levels(g, q, k, size, sign, top):
    """Fill q [n, H, D] and k [L, Hkv, D] so that a key's score is sign * 2^size, or 1/128 of that
    less (7 of 8 keys, at random)."""
    a = min(size // 2, top)
    q.zero_()[..., 0] = sign * 2.0 ** a
    q[..., 17] = 1.0    # (of no weight beside the first, and k has zeros there)
    k.zero_()
    low = torch.rand(k.shape[:2], generator=g, device="cuda") < 0.875
    k[..., 0] = torch.where(low, 127 / 128, 1.0) * 2.0 ** min(size - a, top)
    return 1.1 * 2.0 ** (size - a - min(size - a, top))   # c: scores that no power of two divides


SIZES = [(torch.bfloat16, 20), (torch.bfloat16, 27), (torch.bfloat16, 29), (torch.bfloat16, 60),
         (torch.bfloat16, 120), (torch.float16, 20), (torch.float16, 28), (torch.float16, 40)]


@pytest.mark.parametrize("dtype,size", SIZES)
@pytest.mark.parametrize("sign", (1, -1))
@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("lens,H,Hkv,D", [([300, 40], 2, 2, 64), ([700], 8, 2, 128)])
def test_large_scores_of_prompts(srdit, cuda_device, dtype, size, sign, causal, lens, H, Hkv, D):
    g, T = gen(80 + size), sum(lens)
    q, k = (torch.empty(T, h, D, dtype=dtype, device="cuda") for h in (H, Hkv))
    c = _levels(g, q, k, size, sign, 15 if dtype == torch.float16 else 60)
    v = randn(g, T, Hkv, D).to(dtype)
    cu = offsets(lens)
    out = srdit.ops.packed_attn(q, k, v, cu, causal=causal, scale=LN2 * c)
    for b in range(len(lens)):
        at = slice(int(cu[b]), int(cu[b + 1]))
        ref, tol = _answer(q[at], k[at].double(), v[at].double(), c, causal)
        _check(out[at], ref, tol)


WAYS = [([1, 3], [37, 400], 4, 2, 64), ([1], [20000], 2, 1, 128), ([40, 30], [90, 300], 4, 2, 128),
        ([300], [700], 4, 4, 64), ([70], [20000], 8, 2, 128)]
STEP_SHARES = ([1, 0, 1, 2, 1, 0, 1, 1], [9001, 0, 7, 30000, 12345, 100, 16, 8000], 16, 8, 128)


@pytest.mark.parametrize("dtype,size", SIZES)
@pytest.mark.parametrize("sign", (1, -1))
@pytest.mark.parametrize("new,lens,H,Hkv,D", WAYS + [STEP_SHARES])
def test_large_scores_over_pages(srdit, cuda_device, dtype, size, sign, new, lens, H, Hkv, D):
    g = gen(81 + size)
    cache = Cache(g, lens, Hkv, D, 16, dtype).fill(g, dtype)
    q = torch.empty(sum(new), H, D, dtype=dtype, device="cuda")
    for b, n in enumerate(lens):
        k = torch.empty(n, Hkv, D, dtype=dtype, device="cuda")
        c = _levels(g, q, k, size, sign, 15 if dtype == torch.float16 else 60)
        cache.put(b, 0, k, cache.rows(b, "v")[0].to(dtype))
    _paged(srdit, cache, q, new, c, True)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("size", (24, 25, 26, 27))
@pytest.mark.parametrize("D", (64, 128))
def test_scores_a_step_apart(srdit, cuda_device, dtype, size, D):
    """Key tiles whose largest scores lie 1 to 6 of the smallest steps of fp32 apart, which are 2 to
    16 of an exponent."""
    g, n, step = gen(82), 900, 2.0 ** (size - 23)
    q, k = (torch.zeros(n, 1, D, dtype=dtype, device="cuda") for _ in range(2))
    q[..., 0], k[..., 0] = 2.0 ** (size - 13), 2.0 ** 13
    tile = torch.arange(n, device="cuda") // 128
    up = torch.tensor([1, 2, 3, 4, 6, 5, 9, 3], device="cuda")[tile]
    q[..., 33], k[..., 33] = step, up[:, None].to(dtype)
    v = randn(g, n, 1, D).to(dtype)
    out = srdit.ops.packed_attn(q, k, v, offsets([n]), causal=False, scale=LN2)
    ref, tol = _answer(q, k.double(), v.double(), 1.0, False)
    _check(out, ref, tol)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("size", (20, 27, 29, 40, 100))
@pytest.mark.parametrize("sign", (1, -1))
@pytest.mark.parametrize("new,lens,H,Hkv,D", WAYS + [STEP_SHARES])
def test_large_scores_over_codes(srdit, cuda_device, dtype, code, size, sign, new, lens, H, Hkv, D):
    """Keys of equal scores. Their values' scales are 1 to 2 times a power of two: its exponent and
    the score are rounded together, so that scores this large with other exponents need not stay
    equal."""
    g = gen(83 + size)
    cache = Cache(g, lens, Hkv, D, 16, code, "heads").fill(g, dtype)
    cache.vs.copy_(2.0 ** -7 * (1 + torch.rand(cache.vs.shape, generator=g, device="cuda")))
    q = torch.zeros(sum(new), H, D, dtype=dtype, device="cuda")
    q[..., 0] = sign * 2.0 ** 12
    q[..., 17] = 1.0
    for b, n in enumerate(lens):
        at = cache.places(b, 0, n)
        low = torch.rand(n, Hkv, generator=g, device="cuda") < 0.875
        codes = torch.zeros(n, Hkv, D, device="cuda")
        codes[..., 0] = torch.where(low, 56.0, 64.0)
        cache.k.view(torch.uint8)[at] = codes.to(code).view(torch.uint8)
        cache.ks[at] = 2.0 ** (size - 18)
    _paged(srdit, cache, q, new, 1.1, True)


# ------------------------------------------------------------------ scales far apart
def _scales(g, cache, lo, hi, zeros=0.1):
    """Every value's scale 2^lo to 2^hi, evenly over the exponents; a tenth as of rows of zeros."""
    for b, n in enumerate(cache.lens):
        at = cache.places(b, 0, n)
        s = torch.exp2(lo + (hi - lo) * torch.rand(n, cache.Hkv, generator=g, device="cuda"))
        none = torch.rand(n, cache.Hkv, generator=g, device="cuda") < zeros
        cache.vs[at] = torch.where(none, 1e-12, s)
        codes = cache.v.view(torch.uint8)[at]
        cache.v.view(torch.uint8)[at] = codes.masked_fill(none[..., None], 0)


@pytest.mark.parametrize("dtype,lo,hi", [
    (torch.bfloat16, -40, 100), (torch.bfloat16, 60, 110), (torch.bfloat16, -40, 40),
    (torch.bfloat16, -80, -40), (torch.float16, -40, 8)])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("size", (0.0, 0.5, 6.0))
@pytest.mark.parametrize("new,lens,H,Hkv,D", WAYS + [STEP_SHARES])
def test_scales_far_apart(srdit, cuda_device, dtype, lo, hi, code, size, new, lens, H, Hkv, D):
    """Equal scores, scores of the usual size, and some in which a few keys have all of the weight."""
    g = gen(84)
    cache = Cache(g, lens, Hkv, D, 16, code, "heads").fill(g, dtype)
    _scales(g, cache, lo, hi)
    q = torch.zeros(sum(new), H, D, dtype=dtype, device="cuda")
    q[..., 1] = size * torch.randint(-4, 5, (sum(new), H), generator=g, device="cuda").to(dtype)
    for b, n in enumerate(lens):   # (scores are multiples of 1/8: exact)
        at = cache.places(b, 0, n)
        codes = torch.zeros(n, Hkv, D, device="cuda")
        codes[..., 1] = torch.randint(-8, 9, (n, Hkv), generator=g, device="cuda").float()
        cache.k.view(torch.uint8)[at] = codes.to(code).view(torch.uint8)
        cache.ks[at] = 0.25
    _paged(srdit, cache, q, new, 1.0, True)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("rows", (1, 40))
@pytest.mark.parametrize("order", (0, 1))
def test_a_row_of_zeros_beside_one_of_huge_values(srdit, cuda_device, code, rows, order):
    """Two tokens of equal scores as kv_write leaves them: the answer is half of the huge one."""
    g, dt, D = gen(85), torch.bfloat16, 64
    cache = Cache(g, [rows + 1], 1, D, 16, code)
    k = torch.zeros(rows + 1, 1, D, dtype=dt, device="cuda")
    v = k.clone()
    v[order] = (randn(g, 1, D) * 2.0 ** 100).to(dt)
    cu = torch.tensor([0, rows + 1], dtype=torch.int32, device="cuda")
    srdit.ops.kv_write(k, v, cache.k, cache.v, cache.table, cache.lens_dev, cu_q=cu, **cache.scales)
    q = randn(g, rows, 2, D).to(dt)
    out = _paged(srdit, cache, q, [rows], 1.0, True)
    want = cache.rows(0, "v")[0][order, 0] / torch.arange(2, rows + 2, device="cuda")[:, None]
    assert ((out.double() - want[:, None]).abs() <= 2.0 ** -7 * want[:, None].abs() + 2.0 ** 80).all()
