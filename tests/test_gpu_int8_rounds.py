"""The int8 product and cross attention where a CTA goes through several tiles: more of them than
the GPU has SMs, so that accumulators, barriers' phases, staging and scales are used again.

Against the formulas in 64 bits, with the tolerances of the operators' other tests. What a shape
is here for (a tile width, a number of items, a shared last round) is asked of the library, so a
rule that changes does not take it out of the tests unseen."""
import ctypes

import pytest
import torch

from .test_gpu_int8_ops import DTYPES, _check_attn, _check_gemm, _codes, _gen, _qkv, _randn

pytestmark = pytest.mark.gpu


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


# ------------------------------------------------------------------ int8 product
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,columns", [
    (57001, 63, 130, 64), (57001, 127, 130, 128), (57001, 191, 130, 192), (57001, 255, 130, 256),
    (9221, 1025, 300, 192), (14113, 577, 300, 128), (18701, 579, 1100, 256),
    (2000, 10001, 260, 256)])
def test_int8_gemm_rounds_of_tiles(srdit, cuda_device, dtype, M, N, K, columns):
    """Three tiles a pair at least, of every width: a whole output of aligned rows, which TMA
    stores, and parts of wider ones, with what lies around them left alone."""
    assert srdit._lib.lib().srdit_int8_gemm_columns(M, N, K) == columns
    tiles = (M + 255) // 256 * ((N + columns - 1) // columns)
    assert tiles >= 3 * (_sms() // 2)
    g = _gen(M + N + K)
    a, w = _codes(srdit, g, M, K), _codes(srdit, g, N, K)
    full = N // 16 * 16 + 16   # as many columns as TMA stores
    assert srdit._lib.lib().srdit_int8_gemm_columns(M, full, K) == columns
    _check_gemm(srdit, a, _codes(srdit, g, full, K), dtype, True, g)
    for pitch, off in ((full + 16, 0), (N + 6, 3)):
        buf = torch.full((M, pitch), 5.0, dtype=dtype, device="cuda")
        _check_gemm(srdit, a, w, dtype, True, g, buf[:, off:off + N])
        assert (buf[:, :off] == 5).all() and (buf[:, off + N:] == 5).all()


# ------------------------------------------------------------------ cross attention
def _plan(srdit, q, k, v, lens):
    """(items, whether the last round is shared out) of a call."""
    B, Lq, H, D = q.shape
    a = srdit._lib.CrossAttnArgs()
    srdit._lib.CROSS_ATTN_LAYOUT.pack_into(
        a, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), q.data_ptr(),
        srdit.ops.HALF_TYPES[q.dtype], B, Lq, k.shape[1], H, k.shape[2], D, *q.stride()[:3],
        *k.stride()[:3], *v.stride()[:3], *q.stride()[:3], 0 if lens is None else lens.data_ptr(),
        0, 0, D ** -0.5, 0, 0, 0)
    L = srdit._lib.lib()
    return (L.srdit_cross_attn_items(ctypes.byref(a)),
            L.srdit_cross_attn_workspace(ctypes.byref(a)) > 0)


def _lens(B, Lk):
    """None, one, all, beyond, and all between."""
    return torch.tensor([(0, 1, Lk, Lk + 9, Lk // 2 + 7 * b, 128)[b % 6] for b in range(B)],
                        dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D,shared", [
    (20, 20, 257, 17, 17, 128, False), (20, 33, 300, 16, 16, 64, False),
    (4, 300, 129, 80, 40, 72, False), (10, 270, 130, 16, 16, 128, False),
    (20, 20, 1400, 16, 16, 128, True), (10, 300, 1290, 20, 10, 64, True),
    (3, 1100, 1290, 20, 20, 96, True), (31, 40, 1500, 10, 10, 128, True)])
def test_cross_attn_rounds_of_items(srdit, cuda_device, dtype, B, Lq, Lk, H, Hkv, D, shared):
    """More than two items an SM: whole rounds alone, and a last round whose keys are shared
    out; with lengths and a mask, samples without keys among them."""
    g = _gen(Lq * 7 + Lk)
    q, k, v = _qkv(g, B, Lq, Lk, H, Hkv, D, dtype)
    items, ranged = _plan(srdit, q, k, v, None)
    assert items > 2 * _sms() and items % _sms() != 0 and ranged == shared
    _check_attn(srdit, q, k, v)
    lens = _lens(B, Lk)
    assert _plan(srdit, q, k, v, lens) == (items, shared)
    mask = torch.rand(B, Lk, generator=g, device="cuda") < 0.6
    mask[:, 128:256] = False
    for m in (None, mask):
        y = _check_attn(srdit, q, k, v, lens, m)
        assert (y[0] == 0).all()


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D,rounds", [
    (33, 17, 300, 2, 2, 64, 0), (33, 130, 257, 10, 10, 128, 2), (100, 20, 140, 4, 4, 80, 2),
    (40, 1, 500, 8, 2, 128, None), (65, 8, 77, 2, 1, 64, None)])
def test_cross_attn_many_samples(srdit, cuda_device, dtype, B, Lq, Lk, H, Hkv, D, rounds):
    """More samples than have their key counts in shared memory, with lengths and a mask."""
    g = _gen(B + Lk)
    q, k, v = _qkv(g, B, Lq, Lk, H, Hkv, D, dtype)
    lens = _lens(B, Lk)
    items, shared = _plan(srdit, q, k, v, lens)
    assert not shared
    assert items == 0 if rounds is None else items > rounds * _sms()
    mask = torch.rand(B, Lk, generator=g, device="cuda") < 0.6
    for ln in (None, lens):
        for m in (None, mask):
            y = _check_attn(srdit, q, k, v, ln, m)
            if ln is not None:
                assert (y[0] == 0).all() and (y[6] == 0).all()


def test_repeats_are_bitwise_equal(srdit, cuda_device):
    """Many rounds and joins: the same bits every time, and beside other work."""
    g = _gen(3)
    q, k, v = _qkv(g, 10, 300, 1290, 20, 10, 64, torch.bfloat16)
    a, w = _codes(srdit, g, 9221, 300), _codes(srdit, g, 1025, 300)
    sa, sw = torch.rand(9221, device="cuda"), torch.rand(1025, device="cuda")
    first = srdit.ops.cross_attn(q, k, v), srdit.ops.int8_gemm(a, sa, w, sw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    noise = _randn(g, 2048, 2048)
    for _ in range(5):
        with torch.cuda.stream(side):
            noise @ noise
        again = srdit.ops.cross_attn(q, k, v), srdit.ops.int8_gemm(a, sa, w, sw)
        assert all(torch.equal(x, y) for x, y in zip(first, again))
    side.synchronize()
