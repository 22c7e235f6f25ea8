"""RMS norm with the residual's addition and 8-bit codes, the int8 product, and cross
attention, each against its formula in 64 bits.

Tolerances, with u the unit roundoff of a type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32,
2^-4 e4m3):

- scale of a row: the sum of squares is a chain of at most 64 fp32 additions, so it is off
  by 64 u32, its root by 32 u32; the weight, the divisions and the products add 8 u32:
  40 u32 = 2.4e-6.
- codes: y / scale is off by twice that, so an int8 code is within 0.5 + 127 * 4.8e-6 of
  it, and an e4m3 code within 2^-4 of its size or 2^-10 (half the subnormal step).
- int8 product: the sum is exact; its conversion, two scalings and the bias are 4 u32 of
  the product's size, then one rounding to the output's type.
- attention: a weight p is rounded once to 16 bits (u of the type) and its exponential and
  score are off by less than 2^-11 together (scores of unit rows are below 12, summed in
  fp32; the exponential's approximation is 2^-22), so the output is off by
  (u + 2^-11) sum_j p_j |v_j| / sum_j p_j, plus one rounding u of the output; weights below
  the smallest fp16 step add 2^-25 |v_j| each.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
U32 = 2.0 ** -24
DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


# ------------------------------------------------------------------ rows to 8 bits
def _check_codes(y, q, scale):
    """q, scale against the unrounded rows y (64 bits)."""
    i8 = q.dtype == torch.int8
    ref = (y.abs().amax(1) / (127.0 if i8 else 448.0)).clamp_min(1e-12)
    assert ((scale.double() - ref).abs() <= 40 * U32 * ref).all()
    t = y / ref[:, None]
    err = (q.double() - t).abs()
    if i8:
        assert (err <= 0.5 + 127 * 80 * U32).all()
    else:
        assert (err <= torch.clamp(t.abs() * (2.0 ** -4 + 80 * U32), min=2.0 ** -10 * 1.001)).all()


def _norm_ref(x, r, w, eps):
    s = x.double() + (r.double() if r is not None else 0)
    return s / (s.pow(2).mean(1, keepdim=True) + eps).sqrt() * w.double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("qdtype", (torch.int8, torch.float8_e4m3fn))
@pytest.mark.parametrize("M,K,res", [(1, 1, True), (1, 64, False), (3, 7, True), (5, 96, True),
                                     (9, 1000, True), (2, 1026, False), (33, 513, True),
                                     (7, 3072, True), (4, 8200, True), (2, 16400, True),
                                     (3, 32768, True), (130, 256, False)])
def test_add_rms_quant(srdit, cuda_device, dtype, qdtype, M, K, res):
    g = _gen(M * 100003 + K)
    x = (_randn(g, M, K) * torch.exp(_randn(g, M, 1))).to(dtype)
    r = _randn(g, M, K).to(dtype) if res else None
    w = (1 + 0.2 * _randn(g, K)).to(dtype)
    q, scale, total = srdit.ops.add_rms_quant(x, w, 1e-6, residual=r, qdtype=qdtype)
    _check_codes(_norm_ref(x, r, w, 1e-6), q, scale)
    if res:
        assert torch.equal(total, (x.float() + r.float()).to(dtype))
    else:
        assert total is None
    assert K == 1 or q.stride(0) % 16 == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("qdtype", (torch.int8, torch.float8_e4m3fn))
@pytest.mark.parametrize("M,K", [(1, 1), (5, 72), (3, 1001), (2, 14336), (1, 32768)])
def test_quant_rows(srdit, cuda_device, dtype, qdtype, M, K):
    g = _gen(K)
    x = (3 * _randn(g, M, K)).to(dtype)
    q, scale = srdit.ops.quant_rows(x, qdtype=qdtype)
    _check_codes(x.double(), q, scale)


@pytest.mark.parametrize("off,pitch", [(0, 520), (8, 520), (1, 515), (2, 514), (4, 516)])
def test_norm_strided_views_and_in_place(srdit, cuda_device, off, pitch):
    """Rows of a wider buffer at every alignment; the sum written over the residual."""
    g = _gen(3)
    M, K = 6, 496
    big = _randn(g, M, pitch + 16).to(torch.bfloat16)
    x = big.view(-1)[off:off + M * pitch].view(M, pitch)[:, :K]
    r = _randn(g, M, pitch).to(torch.bfloat16)[:, :K]
    w = (1 + 0.2 * _randn(g, K)).to(torch.bfloat16)
    want, sum_want = _norm_ref(x, r, w, 1e-5), (x.float() + r.float()).to(torch.bfloat16)
    qbuf = torch.full((M, pitch), 77, dtype=torch.int8, device="cuda")
    q, scale, total = srdit.ops.add_rms_quant(x, w, 1e-5, residual=r, sum_out=r, q=qbuf[:, :K])
    _check_codes(want, q, scale)
    assert total.data_ptr() == r.data_ptr() and torch.equal(r, sum_want)
    assert (qbuf[:, K:] == 77).all()


@pytest.mark.parametrize("qdtype", (torch.int8, torch.float8_e4m3fn))
def test_norm_special_rows(srdit, cuda_device, qdtype):
    """Rows of zeros, of the type's extremes, and with a NaN or an infinity."""
    K = 264
    x = torch.ones(6, K, device="cuda")
    x[0] = 0
    x[1] = 1e-30
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    x[4, 9] = -float("inf")
    x[5, 3] = -50
    w = torch.ones(K, device="cuda")
    q, scale, _ = srdit.ops.add_rms_quant(x, w, 1e-6, qdtype=qdtype)
    v = q.float() * scale[:, None]
    assert (v[0] == 0).all() and scale[0] == 1e-12
    ref = _norm_ref(x[1:2], None, w, 1e-6)
    assert ((v[1].double() - ref[0]).abs() <= ref.abs().max() * 2.0 ** -4 + 1e-12).all()
    assert scale[2:5].isnan().all() and v[2:5].isnan().all()
    if qdtype == torch.int8:
        assert (q[2:5] == 0).all()
        assert q[5, 3] == -127
    else:
        assert q[5, 3].float() == -448


# ------------------------------------------------------------------ int8 product
def _codes(srdit, g, M, K):
    t = srdit.ops.code_rows(M, K, torch.int8, "cuda")
    t.copy_(torch.randint(-128, 128, (M, K), generator=g, device="cuda"))
    return t


def _check_gemm(srdit, a, w, dtype, bias, g, out=None):
    M, N = a.shape[0], w.shape[0]
    sa = (0.5 + torch.rand(M, generator=g, device="cuda")) / 127
    sw = (0.5 + torch.rand(N, generator=g, device="cuda")) / 127
    b = _randn(g, N).to(dtype) if bias else None
    y = srdit.ops.int8_gemm(a, sa, w, sw, b, out, out_dtype=None if out is not None else dtype)
    prod = (a.double() @ w.double().t()) * sa.double()[:, None] * sw.double()
    ref = prod + (b.double() if bias else 0)
    size = prod.abs() + (b.double().abs() if bias else 0)
    tol = 4 * U32 * size + U[dtype] * ref.abs() * (1 + 2.0 ** -7) + 2.0 ** -25 + 4 * U32 * U32
    assert y.dtype == dtype and ((y.double() - ref).abs() <= tol).all()
    return y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,bias", [
    (1, 1, 1, True), (1, 16, 64, False), (2, 7, 33, True), (8, 130, 512, True),
    (16, 128, 4096, False), (17, 257, 1000, True), (33, 128, 129, True), (64, 640, 2048, False),
    (65, 96, 160, True), (127, 384, 256, True), (129, 200, 96, True), (200, 264, 4128, False),
    (255, 129, 511, True), (300, 512, 128, True), (513, 1000, 700, True), (1030, 776, 320, False)])
def test_int8_gemm(srdit, cuda_device, dtype, M, N, K, bias):
    g = _gen(M * 31 + N * 7 + K)
    _check_gemm(srdit, _codes(srdit, g, M, K), _codes(srdit, g, N, K), dtype, bias, g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(33, 200, 1584), (33, 200, 1600), (48, 70, 2500), (61, 513, 3000),
                                   (64, 130, 4001), (64, 16400, 1540)])
def test_int8_gemm_of_33_to_64_rows(srdit, cuda_device, dtype, M, N, K):
    """Either side of where such products change kernels."""
    g = _gen(M + N + K)
    _check_gemm(srdit, _codes(srdit, g, M, K), _codes(srdit, g, N, K), dtype, True, g)


@pytest.mark.parametrize("M", (1, 5, 40, 300))
def test_int8_gemm_extremes(srdit, cuda_device, M):
    """-128 times -128 over the longest K: the int32 sum at its largest (2^31 - 2^14)."""
    K = 131071
    a = srdit.ops.code_rows(M, K, torch.int8, "cuda").fill_(-128)
    w = srdit.ops.code_rows(24, K, torch.int8, "cuda").fill_(-128)
    one = torch.ones(24, device="cuda")
    y = srdit.ops.int8_gemm(a, torch.ones(M, device="cuda"), w, one, out_dtype=torch.float32)
    assert (y.double() - 128.0 * 128 * K).abs().max() <= U32 * 128 * 128 * K


@pytest.mark.parametrize("M", (3, 70, 300))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
def test_int8_gemm_views(srdit, cuda_device, M, dtype):
    """Operands and output that are parts of wider buffers (an odd output pitch and offset);
    bytes of the operand rows past K, and around the output, are left alone."""
    g = _gen(M)
    K, N = 200, 136
    a = _codes(srdit, g, M, 512)[:, 16:16 + K]
    w = _codes(srdit, g, N, 256)[:, 32:32 + K]
    buf = torch.full((M, N + 11), 5.0, dtype=dtype, device="cuda")
    y = _check_gemm(srdit, a, w, dtype, True, g, buf[:, 3:3 + N])
    assert y.data_ptr() == buf.data_ptr() + 3 * buf.element_size()
    assert (buf[:, :3] == 5).all() and (buf[:, 3 + N:] == 5).all()


# ------------------------------------------------------------------ cross attention
def _attn_ref(q, k, v, keep, scale):
    """(output, sum p |v| / sum p, sum |v|) in 64 bits."""
    B, Lq, H, D = q.shape
    grp = H // k.shape[2]
    kd = k.double().repeat_interleave(grp, 2)
    vd = torch.where(keep[:, :, None, None], v.double(), 0.0).repeat_interleave(grp, 2)
    s = torch.einsum("bihd,bjhd->bhij", q.double(), kd) * scale
    s = s.masked_fill(~keep[:, None, None, :], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top.isinf(), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    o = torch.einsum("bhij,bjhd->bihd", p, vd)
    a = torch.einsum("bhij,bjhd->bihd", p, vd.abs())
    return o, a, vd.abs().sum(1)[:, None]


def _check_attn(srdit, q, k, v, lens=None, mask=None, scale=None, out=None):
    B, Lk = k.shape[:2]
    keep = torch.ones(B, Lk, dtype=torch.bool, device="cuda")
    if lens is not None:
        keep &= torch.arange(Lk, device="cuda")[None] < lens[:, None]
    if mask is not None:
        keep &= mask.bool()
    y = srdit.ops.cross_attn(q, k, v, out, kv_lens=lens, key_mask=mask, scale=scale)
    o, a, av = _attn_ref(q, k, v, keep, q.shape[-1] ** -0.5 if scale is None else scale)
    u = U[q.dtype]
    tol = (u + 2.0 ** -11) * a + u * (1 + 2.0 ** -7) * o.abs() + 2.0 ** -25 * (1 + av)
    assert y.shape == q.shape and ((y.double() - o).abs() <= tol).all()
    return y


def _qkv(g, B, Lq, Lk, H, Hkv, D, dtype):
    return (_randn(g, B, Lq, H, D).to(dtype), _randn(g, B, Lk, Hkv, D).to(dtype),
            _randn(g, B, Lk, Hkv, D).to(dtype))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [
    (1, 1, 1, 1, 1, 64), (2, 1, 77, 4, 4, 128), (1, 1, 4099, 8, 1, 128), (3, 2, 513, 6, 2, 64),
    (1, 5, 128, 4, 1, 80), (2, 16, 300, 2, 2, 96), (1, 17, 129, 3, 3, 128), (2, 64, 1000, 8, 2, 64),
    (1, 127, 127, 2, 2, 128), (1, 128, 128, 2, 1, 64), (2, 129, 257, 2, 1, 128),
    (1, 300, 640, 3, 1, 40), (1, 257, 33, 4, 4, 8), (2, 513, 384, 5, 5, 120),
    (1, 1000, 1030, 2, 2, 128), (1, 3, 20000, 2, 1, 128), (1, 130, 9000, 1, 1, 128)])
def test_cross_attn(srdit, cuda_device, dtype, B, Lq, Lk, H, Hkv, D):
    g = _gen(Lq * 131 + Lk)
    _check_attn(srdit, *_qkv(g, B, Lq, Lk, H, Hkv, D, dtype))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("Lq,H,Hkv,D", [(1, 4, 4, 128), (1, 16, 2, 64), (9, 4, 2, 80),
                                        (150, 4, 2, 128), (300, 2, 2, 64)])
@pytest.mark.parametrize("Lk", (1, 40, 384, 700, 5000))
def test_cross_attn_lengths_and_masks(srdit, cuda_device, dtype, Lq, H, Hkv, D, Lk):
    """Lengths from none to all (and beyond), holes, an empty mask, with NaN and infinities in
    every key and value that is not seen."""
    g = _gen(Lk + Lq)
    B = 6
    q, k, v = _qkv(g, B, Lq, Lk, H, Hkv, D, dtype)
    lens = torch.tensor([0, 1, (Lk + 1) // 2, Lk, Lk + 5, Lk], dtype=torch.int32, device="cuda")
    mask = torch.rand(B, Lk, generator=g, device="cuda") < 0.7
    mask[5] = False
    for m in (None, mask):
        keep = torch.arange(Lk, device="cuda")[None] < lens[:, None]
        if m is not None:
            keep = keep & m
        bad = torch.where(torch.rand(B, Lk, 1, 1, generator=g, device="cuda") < 0.5,
                          float("nan"), float("inf"))
        kb = torch.where(keep[:, :, None, None], k, bad.to(dtype))
        vb = torch.where(keep[:, :, None, None], v, bad.to(dtype))
        y = _check_attn(srdit, q, kb, vb, lens, m)
        assert (y[0] == 0).all()
        if m is not None:
            assert (y[5] == 0).all()
    only = torch.zeros(B, Lk, dtype=torch.uint8, device="cuda")
    only[:, Lk - 1] = 255   # one key seen: its value comes back
    y = srdit.ops.cross_attn(q, k, v, key_mask=only)
    want = v[:, Lk - 1:].repeat_interleave(H // Hkv, 2).expand_as(y)
    assert ((y.float() - want.float()).abs() <= U[dtype] * want.float().abs()).all()


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [(1, 512, 4000, 4, 4, 128), (2, 300, 2100, 4, 1, 64),
                                             (1, 130, 6000, 2, 2, 72), (7, 257, 900, 6, 3, 128)])
def test_cross_attn_shared_items(srdit, cuda_device, dtype, B, Lq, Lk, H, Hkv, D):
    """Few queries on many keys: query tiles whose keys are shared out over several CTAs and
    joined, with and without a sample that has none."""
    g = _gen(Lq + D)
    q, k, v = _qkv(g, B, Lq, Lk, H, Hkv, D, dtype)
    _check_attn(srdit, q, k, v)
    lens = torch.tensor([Lk - 130 * b if b != 1 else 0 for b in range(B)], dtype=torch.int32,
                        device="cuda")
    mask = torch.rand(B, Lk, generator=g, device="cuda") < 0.5
    mask[:, 128:384] = False   # whole key tiles without a seen key
    _check_attn(srdit, q, k, v, lens, mask)


@pytest.mark.parametrize("Lq", (1, 6, 200))
def test_cross_attn_layouts(srdit, cuda_device, Lq):
    """Fused k|v buffers, heads before tokens, a shared prompt (batch stride 0), one key head
    repeated by its stride, and an output inside a wider buffer."""
    g = _gen(Lq)
    B, Lk, H, Hkv, D = 2, 333, 4, 2, 64
    dt = torch.bfloat16
    q = _randn(g, B, H, Lq, D).to(dt).transpose(1, 2)
    kv = _randn(g, B, Lk, 2, Hkv, D).to(dt)
    buf = torch.full((B, Lq, H, 3 * D), 9.0, dtype=dt, device="cuda")
    _check_attn(srdit, q, kv[:, :, 0], kv[:, :, 1], out=buf[..., D:2 * D])
    assert (buf[..., :D] == 9).all() and (buf[..., 2 * D:] == 9).all()
    one = kv[:1].expand(B, Lk, 2, Hkv, D)
    _check_attn(srdit, q, one[:, :, 0], one[:, :, 1],
                torch.tensor([100, 333], dtype=torch.int32, device="cuda"))
    head = kv[:, :, :, :1].expand(B, Lk, 2, Hkv, D)
    _check_attn(srdit, q, head[:, :, 0], head[:, :, 1], scale=0.3)


@pytest.mark.parametrize("Lq", (1, 140))
def test_cross_attn_large_scores(srdit, cuda_device, Lq):
    """Scores in the hundreds, the largest last: the running maximum has to move."""
    g = _gen(5)
    q, k, v = _qkv(g, 1, Lq, 1025, 2, 2, 128, torch.float16)
    q = q.abs() * 4
    k = k * torch.linspace(0.1, 8, 1025, device="cuda")[None, :, None, None].to(k.dtype)
    k[:, -1] = k[:, -1].abs() + 4
    y = srdit.ops.cross_attn(q, k, v)
    keep = torch.ones(1, 1025, dtype=torch.bool, device="cuda")
    o, a, _ = _attn_ref(q, k, v, keep, 128 ** -0.5)
    # one key outweighs the rest by e^10 at least: scores of size 4000 are off by
    # 4000 * 128 u32 = 0.03 at most, which moves the others' weight, below e^-10, by 3%
    assert ((y.double() - o).abs() <= 2.0 ** -10 * a + 2.0 ** -10 * o.abs() + 1e-4).all()


@pytest.mark.parametrize("Lq", (1, 5, 200))
@pytest.mark.parametrize("Lk", (1, 300, 9000))
def test_cross_attn_seen_nan_stays_nan(srdit, cuda_device, Lq, Lk):
    """A NaN in a seen key reaches every row of its sample, one in a query its own row, one in
    a seen value its column; nothing else."""
    g = _gen(Lk)
    q, k, v = _qkv(g, 4, Lq, Lk, 2, 1, 64, torch.bfloat16)
    clean = srdit.ops.cross_attn(q, k, v)
    k[0, Lk // 2, 0, 3] = float("nan")
    q[1, Lq - 1, 1, 7] = float("nan")
    v[2, Lk - 1, 0, 9] = float("nan")
    y = srdit.ops.cross_attn(q, k, v)
    assert y[0].isnan().all()
    assert y[1, Lq - 1, 1].isnan().all() and y[2, :, :, 9].isnan().all()
    y[0] = clean[0]
    y[1, Lq - 1, 1] = clean[1, Lq - 1, 1]
    y[2, :, :, 9] = clean[2, :, :, 9]
    assert torch.equal(y, clean)


def test_cross_attn_empty(srdit, cuda_device):
    q = torch.randn(2, 3, 4, 64, device="cuda", dtype=torch.bfloat16)
    kv = torch.empty(2, 0, 4, 64, device="cuda", dtype=torch.bfloat16)
    assert (srdit.ops.cross_attn(q, kv, kv) == 0).all()
    y = srdit.ops.cross_attn(q[:, :0], q, q)
    assert y.shape == (2, 0, 4, 64)
    assert srdit.ops.cross_attn(q[:0], q[:0], q[:0]).shape == (0, 3, 4, 64)


# ------------------------------------------------------------------ streams, graphs, refusals
def _everything(srdit, s):
    ops = srdit.ops
    q, scale, total = ops.add_rms_quant(s["x"], s["w"], residual=s["r"])
    y = ops.int8_gemm(q, scale, s["wq"], s["ws"])
    qq, qs = ops.quant_rows(y)
    z = ops.int8_gemm(qq[:3], qs[:3].contiguous(), s["wk"], s["ws"][:256].contiguous())
    o = ops.cross_attn(y.view(1, 130, 4, 64), s["k"], s["v"])
    one = ops.cross_attn(y[:1].view(1, 1, 4, 64), s["k"], s["v"])
    return total, y, z, o, one


def _state(srdit):
    g = _gen(11)
    s = {"x": _randn(g, 130, 320).to(torch.bfloat16), "r": _randn(g, 130, 320).to(torch.bfloat16),
         "w": torch.ones(320, device="cuda", dtype=torch.bfloat16)}
    s["wq"], s["wk"] = _codes(srdit, g, 256, 320), _codes(srdit, g, 256, 256)
    s["ws"] = torch.full((256,), 1e-3, device="cuda")
    s["k"], s["v"] = (_randn(g, 1, 6000, 1, 64).to(torch.bfloat16) for _ in range(2))
    return s


def test_repeats_are_bitwise_equal_on_any_stream_and_in_a_graph(srdit, cuda_device):
    s = _state(srdit)
    first = _everything(srdit, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _everything(srdit, s)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _everything(srdit, s)
    for t in got:
        t.zero_()
    s["x"].neg_()
    s["r"].neg_()
    graph.replay()
    torch.cuda.synchronize()
    fresh = _everything(srdit, s)
    assert all(torch.equal(a, b) for a, b in zip(got, fresh))
    assert not torch.equal(got[1], first[1])


def test_refusals(srdit, cuda_device):
    ops, err = srdit.ops, srdit._lib.SrditError
    x = torch.randn(4, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    q, s, _ = ops.add_rms_quant(x, w)
    cases = [
        lambda: ops.add_rms_quant(x, w.float()),
        lambda: ops.add_rms_quant(x, w[:32]),
        lambda: ops.add_rms_quant(x.t(), w),
        lambda: ops.add_rms_quant(x, w, residual=x[:2]),
        lambda: ops.add_rms_quant(x, w, sum_out=x),
        lambda: ops.add_rms_quant(x, w, qdtype=torch.uint8),
        lambda: ops.add_rms_quant(x, w, float("nan")),
        lambda: ops.add_rms_quant(x.double(), w.double()),
        lambda: ops.add_rms_quant(torch.zeros(1, 40000, device="cuda"),
                                  torch.ones(40000, device="cuda")),
        lambda: ops.add_rms_quant(x.cpu(), w.cpu()),
        lambda: ops.add_rms_quant(x, w.cpu()),
        lambda: ops.quant_rows(x, q=q[:2]),
        lambda: ops.quant_rows(x, qscale=s[:2]),
        lambda: ops.int8_gemm(q.float(), s, q, s),
        lambda: ops.int8_gemm(q, s, q[:, :32], s),
        lambda: ops.int8_gemm(q, s[:2], q, s),
        lambda: ops.int8_gemm(q, s, q, s, w[:4].float()),
        lambda: ops.int8_gemm(q, s, q, s, out=x[:2]),
        lambda: ops.int8_gemm(q[:, 1:33], s, q[:, 1:33], s),
        lambda: ops.int8_gemm(q, s, q, s, out_dtype=torch.float64),
        lambda: ops.int8_gemm(torch.zeros(4, 72, device="cuda", dtype=torch.int8)[:, :64], s, q, s),
    ]
    a = torch.randn(2, 3, 4, 64, device="cuda", dtype=torch.bfloat16)
    lens = torch.ones(2, device="cuda", dtype=torch.int32)
    cases += [
        lambda: ops.cross_attn(a.float(), a.float(), a.float()),
        lambda: ops.cross_attn(a, a.half(), a.half()),
        lambda: ops.cross_attn(a, a, a[:, :2]),
        lambda: ops.cross_attn(a, a[:, :, :3], a[:, :, :3]),
        lambda: ops.cross_attn(a[..., :60], a[..., :60], a[..., :60]),
        lambda: ops.cross_attn(a[..., 4:60], a[..., 4:60], a[..., 4:60]),
        lambda: ops.cross_attn(a.transpose(2, 3), a.transpose(2, 3), a.transpose(2, 3)),
        lambda: ops.cross_attn(a, a, a, kv_lens=lens.long()),
        lambda: ops.cross_attn(a, a, a, kv_lens=lens[:1]),
        lambda: ops.cross_attn(a, a, a, key_mask=torch.ones(2, 2, device="cuda").bool()),
        lambda: ops.cross_attn(a, a, a, key_mask=torch.ones(2, 3, device="cuda")),
        lambda: ops.cross_attn(a, a, a, scale=-1.0),
        lambda: ops.cross_attn(a, a, a, scale=float("nan")),
        lambda: ops.cross_attn(a, a, a, out=a[:1].expand_as(a)),
        lambda: ops.cross_attn(a.repeat(1, 1, 1, 4), a.repeat(1, 1, 1, 4), a.repeat(1, 1, 1, 4)),
        lambda: ops.cross_attn(a.cpu(), a.cpu(), a.cpu()),
    ]
    for i, c in enumerate(cases):
        with pytest.raises(err):
            c()
            pytest.fail(f"case {i} was taken")
    torch.cuda.synchronize()   # nothing was launched that faults


# ------------------------------------------------------------------ modules
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,N", [((5, 96), 40), ((2, 3, 50), 33), ((1, 256), 128)])
def test_int8_linear(srdit, cuda_device, dtype, shape, N):
    """The module against its own codes: the activation's codes are those of quant_rows
    (checked above), the product that of int8_gemm."""
    g = _gen(N)
    lin = torch.nn.Linear(shape[-1], N, device="cuda", dtype=dtype)
    m = srdit.int8_linear.Int8Linear.from_linear(lin)
    x = _randn(g, *shape).to(dtype)
    y = m(x)
    assert y.shape == (*shape[:-1], N) and y.dtype == dtype
    q, s = srdit.ops.quant_rows(x.reshape(-1, shape[-1]))
    wq, ws = srdit.int8_linear.quantize_weight_int8(lin.weight)
    prod = (q.double() @ wq.double().t()) * s.double()[:, None] * ws.double()
    ref = (prod + lin.bias.double()).view(y.shape)
    size = prod.abs().view(y.shape) + lin.bias.double().abs()
    assert ((y.double() - ref).abs() <= 4 * U32 * size + U[dtype] * ref.abs() * (1 + 2.0 ** -7)
            + 2.0 ** -24).all()
    # and against the Linear itself: an int8 step is 1/127 of the largest value, half of it off
    # per value at most, in both operands
    full = x.double() @ lin.weight.double().t() + lin.bias.double()
    xs, w_abs = x.double().abs(), lin.weight.double().abs()
    half_x, half_w = xs.amax(-1, keepdim=True) / 254, w_abs.amax(1) / 254
    off = half_x * w_abs.sum(1) + xs.sum(-1, keepdim=True) * half_w + half_x * half_w * shape[-1]
    assert ((y.double() - full).abs() <= 1.01 * off + 2 * U[dtype] * full.abs() + 1e-4).all()


@pytest.mark.parametrize("B,L,heads,kv_heads", [(1, 1, 2, 2), (3, 1, 4, 2), (2, 70, 4, 1),
                                                (1, 300, 2, 2)])
def test_cross_stack(srdit, cuda_device, B, L, heads, kv_heads):
    """The blocks on the operators against the same blocks with the dequantised weights in 64
    bits. Each of a block's three quantisations is off by half a step of 1/127 of a row's
    largest value (4 to 5 sigma), 1% of a row's norm; with two blocks of a norm, an attention
    and products that keep such relative errors, 5% of the added part bounds their sum."""
    import importlib
    tb = importlib.import_module("dreamx-creator_b200.text_block")
    dim, text_dim, hd = heads * 64, 96, 64
    stack = tb.CrossStack.random_init(dim=dim, text_dim=text_dim, heads=heads, kv_heads=kv_heads,
                                      layers=2, seed=3)
    g = _gen(B + L)
    x = _randn(g, B, L, dim).to(torch.bfloat16)
    states = _randn(g, B, 77, text_dim).to(torch.bfloat16)
    lens = torch.tensor([77, 5, 0][:B], dtype=torch.int32, device="cuda")
    x0 = x.clone()
    out = stack(x, stack.text_kv(states), kv_lens=lens)
    assert torch.equal(x, x0)

    def lin(m, v):
        w = m.weight_int8[:, :m.in_features].double() * m.weight_scale.double()[:, None]
        return v @ w.t() + m.bias.double()

    ref = x.double()
    for b in stack.blocks:
        n = ref / (ref.pow(2).mean(-1, keepdim=True) + b.eps).sqrt() * b.norm.double()
        q = lin(b.q, n).view(B, L, heads, hd)
        kv = lin(b.kv, states.double()).view(B, 77, 2, kv_heads, hd).repeat_interleave(
            heads // kv_heads, 3)
        s = torch.einsum("bihd,bjhd->bhij", q, kv[:, :, 0]) * hd ** -0.5
        keep = torch.arange(77, device="cuda")[None] < lens[:, None]
        p = torch.softmax(s.masked_fill(~keep[:, None, None], -1e300), -1)
        p = p * keep[:, None, None]
        ref = ref + lin(b.o, torch.einsum("bhij,bjhd->bihd", p, kv[:, :, 1]).reshape(B, L, dim))
    added = ref - x.double()
    assert (out.double() - ref).norm() <= 0.05 * added.norm() + 2 * U[torch.bfloat16] * ref.norm()
