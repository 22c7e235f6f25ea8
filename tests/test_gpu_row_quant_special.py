"""The row quantisers on rows at the ends of fp32: against their formulas in 64 bits.

Tolerances, with u32 = 2^-24:

- scale of a row whose sum of squares is beyond fp32: that sum is then K / 32 fp32 additions a
  lane and 5 across the warp, its root half as far off, and 16 u32 cover the products and the
  root: (K / 64 + 20) u32. With a bf16 residual it is the sum of the rounded x + r, each off by
  2^-8 of its size at most, so the root is too.
- codes: the norm's factor cancels in y / scale, which leaves the products: less than 80 u32 of
  the largest code, as for other rows.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
CODES = (torch.int8, torch.float8_e4m3fn)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("qdtype", CODES)
@pytest.mark.parametrize("K", (1, 40, 300, 2570, 3072, 9000, 32768))
@pytest.mark.parametrize("res", ("none", "apart", "over x", "over r"))
def test_finite_rows_whose_squares_are_not(srdit, cuda_device, dtype, qdtype, K, res):
    """Rows of 2^57 to 2^125 between ordinary ones: codes and scales by the formula, not zeros."""
    g = _gen(K)
    size = torch.tensor([0, 57, 64, 1, 90, 120, 124, -3, 70], device="cuda")
    M = size.numel()
    x = (torch.rand(M, K, generator=g, device="cuda") - 0.5) * 2
    x[4, 1:] *= 2.0 ** -100   # a single large value
    x = torch.ldexp(x, size[:, None]).to(dtype)
    r = None
    if res != "none":
        r = torch.ldexp(torch.rand(M, K, generator=g, device="cuda"), size[:, None]).to(dtype)
    w = (1 + 0.2 * torch.rand(K, generator=g, device="cuda")).to(dtype)
    s = x.double() + (0 if r is None else r.double())
    y = s / (s.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    out = {"none": None, "apart": None, "over x": x, "over r": r}[res]
    q, scale, total = srdit.ops.add_rms_quant(x, w, 1e-6, residual=r, sum_out=out, qdtype=qdtype)
    i8 = qdtype == torch.int8
    ref = (y.abs().amax(1) / (127.0 if i8 else 448.0)).clamp_min(1e-12)
    tol = (K / 64 + 20) * U32
    if r is not None:
        assert torch.equal(total, s.float().to(dtype))
        if dtype == torch.bfloat16:
            tol += 2.0 ** -8
    tol = torch.where(size > 50, tol, 40 * U32)
    assert ((scale.double() - ref).abs() <= tol * ref).all()
    t = y / ref[:, None]
    err = (q.double() - t).abs()
    if i8:
        assert (err <= 0.5 + 127 * 80 * U32).all()
    else:
        assert (err <= torch.clamp(t.abs() * (2.0 ** -4 + 80 * U32), min=2.0 ** -10 * 1.001)).all()


@pytest.mark.parametrize("qdtype", CODES)
@pytest.mark.parametrize("K", (5, 264, 9000))
@pytest.mark.parametrize("norm", (False, True))
def test_special_rows(srdit, cuda_device, qdtype, K, norm):
    """Zeros, values below the smallest scale, a NaN, infinities."""
    x = torch.ones(6, K, device="cuda")
    x[0] = 0
    x[1] = 1e-30
    x[2, 3] = float("nan")
    x[3, 4] = float("inf")
    x[4, 0] = -float("inf")
    x[5, 2] = -50
    if norm:
        q, scale, _ = srdit.ops.add_rms_quant(x, torch.ones(K, device="cuda"), 1e-6, qdtype=qdtype)
    else:
        q, scale = srdit.ops.quant_rows(x, qdtype=qdtype)
    v = q.float() * scale[:, None]
    # 1e-30 is 1e-27 after the norm, far below half a step of the smallest scale
    assert (scale[:2] == 1e-12).all() and (q[:2].float() == 0).all()
    assert scale[2].isnan() and v[2:5].isnan().all()
    if norm:
        assert scale[3:5].isnan().all()
    else:
        assert scale[3:5].isposinf().all()
    if qdtype == torch.int8:
        assert (q[2:5] == 0).all() and q[5, 2] == -127
    else:
        assert q[5, 2].float() == -448
