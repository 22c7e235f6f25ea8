"""The integer operators at the edges of their operands: what lies past a row's end, past a cache's
length and beside an output, offsets beyond 2^31, repeated samples, strides of single entries.
Tolerances as in the operators' other tests."""
import pytest
import torch

from .test_gpu_int8_ops import (DTYPES, _check_attn, _check_codes, _check_gemm, _codes, _gen,
                                _norm_ref, _qkv, _randn)

pytestmark = pytest.mark.gpu

HALF = (torch.bfloat16, torch.float16)


# ------------------------------------------------------------------ int8 product
@pytest.mark.parametrize("M", (1, 20, 64, 70, 300))
@pytest.mark.parametrize("K", (1, 3, 15, 17, 33, 129, 200, 1001, 4099))
def test_codes_past_the_rows_end(srdit, cuda_device, M, K):
    """Bytes between K and the pitch take no part, whatever they are."""
    g = _gen(M + K)
    N = 136
    ops = []
    for rows in (M, N):
        t = torch.full((rows, (K + 47) // 16 * 16), 127, dtype=torch.int8, device="cuda")
        t[:, :K] = torch.randint(-128, 128, (rows, K), generator=g, device="cuda")
        ops.append(t[:, :K])
    _check_gemm(srdit, *ops, torch.float32, True, g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", [(70, 128), (255, 64), (129, 272), (300, 384)])
def test_rows_beside_the_output(srdit, cuda_device, dtype, M, N):
    """Whole 16-byte pieces: the output's neighbours on all sides."""
    g = _gen(M + N)
    buf = torch.full((M + 40, N + 32), 5.0, dtype=dtype, device="cuda")
    _check_gemm(srdit, _codes(srdit, g, M, 130), _codes(srdit, g, N, 130), dtype, True, g,
                buf[20:M + 20, 16:16 + N])
    buf[20:M + 20, 16:16 + N] = 5
    assert (buf == 5).all()


@pytest.mark.parametrize("M", (40, 70))
def test_rows_far_apart(srdit, cuda_device, M):
    """Rows whose offsets pass 2^31 elements: codes, outputs, and the row quantisers' rows."""
    g = _gen(M)
    K = N = 64
    pitch = (1 << 31) // 32
    big = torch.empty(M * pitch, dtype=torch.int8, device="cuda")
    a = big.as_strided((M, K), (pitch, 1))
    a.copy_(torch.randint(-128, 128, (M, K), generator=g, device="cuda"))
    y = _check_gemm(srdit, a, _codes(srdit, g, N, K), torch.bfloat16, True, g)
    del big, a
    big = torch.empty(M * pitch, dtype=torch.bfloat16, device="cuda")
    far = big.as_strided((M, K), (pitch, 1))
    far.copy_(y)
    q, s, _ = srdit.ops.add_rms_quant(far, torch.ones(K, device="cuda", dtype=far.dtype), 1e-6)
    _check_codes(_norm_ref(far, None, torch.ones(K, device="cuda"), 1e-6), q, s)
    _check_gemm(srdit, q, _codes(srdit, g, N, K), torch.bfloat16, True, g, far)


# ------------------------------------------------------------------ cross attention
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("Lq", (1, 7, 150, 300))
@pytest.mark.parametrize("D", (8, 40, 64, 72, 120))
@pytest.mark.parametrize("Lk", (77, 900))
def test_neighbours_of_every_operand(srdit, cuda_device, dtype, Lq, D, Lk):
    """Views into wider buffers of NaN: past each head's D, past the cache's Lk and beside the
    queries; what lies beside the output is left alone."""
    g = _gen(Lq + D)
    B, H, Hkv = 2, 4, 2

    def inside(x, fill):
        b, n, h, d = x.shape
        buf = torch.full((b, n + 40, h + 1, d + 24), fill, dtype=dtype, device="cuda")
        view = buf[:, :n, :h, 8:8 + d]
        view.copy_(x)
        return buf, view

    q, k, v = _qkv(g, B, Lq, Lk, H, Hkv, D, dtype)
    views = [inside(x, float("nan"))[1] for x in (q, k, v)]
    buf, out = inside(torch.zeros_like(q), 7.0)
    lens = torch.tensor([Lk, Lk // 2], dtype=torch.int32, device="cuda")
    for ln in (None, lens):
        _check_attn(srdit, *views, ln, out=out)
    out.fill_(7)
    assert (buf == 7).all()


@pytest.mark.parametrize("Lq", (1, 3, 200))
def test_repeated_samples_and_masks(srdit, cuda_device, Lq):
    """Queries, a mask and keys of one sample for all; lengths below zero are none."""
    g = _gen(Lq)
    B, Lk, D = 5, 333, 64
    q, k, v = _qkv(g, B, Lq, Lk, 4, 2, D, torch.bfloat16)
    mask = torch.rand(1, Lk, generator=g, device="cuda") < 0.6
    _check_attn(srdit, q[:1].expand_as(q), k, v, mask=mask.expand(B, Lk))
    _check_attn(srdit, q[:1].expand_as(q), k[:1].expand_as(k), v[:1].expand_as(v))
    lens = torch.tensor([-1, 0, 5, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    y = _check_attn(srdit, q, k, v, lens, mask.expand(B, Lk))
    assert (y[[0, 1, 3]] == 0).all()


@pytest.mark.parametrize("Lq", (1, 40))
def test_strides_of_single_entries(srdit, cuda_device, Lq):
    """Dimensions of one entry may have any stride."""
    g = _gen(Lq)
    q, k, v = _qkv(g, 1, Lq, 1, 1, 1, 64, torch.bfloat16)
    for bs, hs in ((3, 5), (0, 0), (1 << 40, 1 << 41)):
        qo = q.as_strided(q.shape, (bs, 64, hs, 1))
        kv = [x.as_strided(x.shape, (bs, 7, hs, 1)) for x in (k, v)]
        y = srdit.ops.cross_attn(qo, *kv)
        assert ((y - v).abs() <= 2.0 ** -8 * v.abs()).all()   # one key: its value


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [
    (1, 1, 300, 128, 1, 64), (2, 1, 513, 48, 2, 128), (1, 2, 700, 60, 3, 64),
    (2, 5, 257, 21, 3, 72), (1, 33, 400, 192, 1, 128), (3, 1, 140, 17, 1, 128),
    (2, 100, 300, 12, 1, 64), (1, 16, 2000, 1, 1, 128), (1, 17, 2000, 1, 1, 128),
    (1, 4, 2000, 4, 1, 64)])
def test_groups_of_any_size(srdit, cuda_device, dtype, B, Lq, Lk, H, Hkv, D):
    """One to 192 heads on a key head, powers of two and not, with lengths and a mask."""
    g = _gen(H + Lk)
    q, k, v = _qkv(g, B, Lq, Lk, H, Hkv, D, dtype)
    _check_attn(srdit, q, k, v)
    lens = torch.tensor([Lk - 77, Lk, 3][:B], dtype=torch.int32, device="cuda")
    mask = torch.rand(B, Lk, generator=g, device="cuda") < 0.5
    _check_attn(srdit, q, k, v, lens, mask)


@pytest.mark.parametrize("Lq", (1, 130))
def test_samples_and_heads_far_apart(srdit, cuda_device, Lq):
    """A cache whose samples lie 2^31 elements apart, and one whose heads do."""
    g = _gen(Lq)
    Lk, D, far = 300, 64, 1 << 31
    big = torch.empty(far + (1 << 16), dtype=torch.bfloat16, device="cuda")
    for shape, strides in (((2, Lk, 1, D), (far, D, D, 1)), ((1, Lk, 2, D), (far, D, far, 1))):
        q = _randn(g, shape[0], Lq, 2, D).to(torch.bfloat16)
        k = big.as_strided(shape, strides)
        v = big.as_strided(shape, strides, 32 * 1024)
        for t in (k, v):
            t.copy_(_randn(g, *shape))
        _check_attn(srdit, q, k, v)
    qshape, qstr = (2, Lq, 2, D), (far, 2 * D, D, 1)
    out = big.as_strided(qshape, qstr)
    q, k, v = _qkv(g, 2, Lq, Lk, 2, 1, D, torch.bfloat16)
    _check_attn(srdit, q, k, v, out=out)


@pytest.mark.parametrize("M", (1, 64, 300))
def test_status_words_stay_clear(srdit, cuda_device, M):
    g = _gen(M)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a, w = _codes(srdit, g, M, 256), _codes(srdit, g, 128, 256)
    one = torch.ones(300, device="cuda")
    srdit.ops.int8_gemm(a, one[:M], w, one[:128], status=status)
    srdit.ops.cross_attn(*_qkv(g, 1, M, 3000, 2, 1, 64, torch.bfloat16), status=status)
    assert status.item() == 0


@pytest.mark.parametrize("Lq,Lk,kernels", [(1, 300, 1), (1, 40000, 2), (300, 300, 1),
                                           (300, 9000, 2)])
def test_every_kernel_is_counted(srdit, cuda_device, Lq, Lk, kernels):
    """A call whose parts are joined by a second kernel counts as two launches."""
    q, k, v = _qkv(_gen(Lk), 1, Lq, Lk, 1, 1, 64, torch.bfloat16)
    before = srdit.ops.Stats.launches
    srdit.ops.cross_attn(q, k, v)
    assert srdit.ops.Stats.launches - before == kernels


@pytest.mark.parametrize("M,N,K", [
    (11, 4077, 2832), (57, 4452, 4934), (6, 2640, 4829), (22, 1362, 2675), (9, 2953, 2467),
    (64, 33, 3211), (33, 2, 3084), (1, 10, 4724), (45, 2296, 2789), (16, 4077, 4096)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_products_of_few_tokens_and_a_long_axis(srdit, cuda_device, dtype, M, N, K):
    """Sums shared out over the CTAs of a cluster, some of them without a token to join, of odd
    sizes and in rows wider than they are long; five times over, the same bits."""
    g = _gen(M + N + K)
    a, w = (torch.randint(-128, 128, (n, (K + 15) // 16 * 16 + 32), generator=g, device="cuda")
            .to(torch.int8)[:, :K] for n in (M, N))
    _check_gemm(srdit, a, w, dtype, True, g)
    s = torch.rand(max(M, N), generator=g, device="cuda")
    first = srdit.ops.int8_gemm(a, s[:M], w, s[:N], out_dtype=dtype)
    for _ in range(4):
        assert torch.equal(srdit.ops.int8_gemm(a, s[:M], w, s[:N], out_dtype=dtype), first)
