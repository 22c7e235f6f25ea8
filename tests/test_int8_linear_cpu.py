"""Host-side logic of the integer operators (no GPU): weight preparation, module casts and
the module swap of Int8Linear, the struct layouts, and the refusals of the C entry points,
which return before anything is launched."""
import ctypes
import importlib
import re

import pytest
import torch
import torch.nn as nn


@pytest.fixture(scope="module")
def il(srdit):
    return importlib.import_module("dreamx-creator_b200.int8_linear")


@pytest.mark.parametrize("N,K", [(96, 160), (5, 33), (1, 1)])
def test_weight_codes(il, N, K):
    w = (torch.randn(N, K, generator=torch.Generator().manual_seed(1)) * 0.02).to(torch.bfloat16)
    w[0] = 0
    q, s = il.quantize_weight_int8(w)
    ref = (w.double().abs().amax(1) / 127).clamp_min(1e-12)
    assert q.dtype == torch.int8 and q.stride(0) % 16 == 0 and q.shape == (N, K)
    # the scale is one fp32 division; a code is within half a step and the division's rounding
    assert ((s.double() - ref).abs() <= 2.0 ** -23 * ref).all()
    assert ((q.double() - w.double() / ref[:, None]).abs() <= 0.5 + 127 * 2.0 ** -22).all()
    assert (q[0] == 0).all()


def test_module_casts_keep_codes_and_scales(il):
    lin = nn.Linear(50, 32).to(torch.bfloat16)
    m = il.Int8Linear.from_linear(lin)
    q0, s0 = m.weight_int8.clone(), m.weight_scale.clone()
    assert m.weight_int8.shape == (32, 64) and m.weight.dtype == torch.bfloat16
    for cast in (lambda t: t.half(), lambda t: t.float(), lambda t: t.to("cpu", torch.bfloat16)):
        assert cast(m) is m
        assert m.weight_int8.dtype == torch.int8 and torch.equal(m.weight_int8, q0)
        assert m.weight_scale.dtype == torch.float32 and torch.equal(m.weight_scale, s0)
    assert m.bias.dtype == torch.bfloat16
    with pytest.raises(ValueError):
        il.Int8Linear(torch.zeros(3))
    with pytest.raises(ValueError):
        m(torch.zeros(2, 51))


def test_no_cpu_path(srdit, il):
    err = srdit._lib.SrditError
    m = il.Int8Linear.from_linear(nn.Linear(32, 16))
    a = torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: m(torch.zeros(2, 32)),
                 lambda: srdit.ops.add_rms_quant(torch.zeros(2, 32), torch.ones(32)),
                 lambda: srdit.ops.cross_attn(a, a, a)):
        with pytest.raises(err):
            call()
    if not torch.cuda.is_available():
        tb = importlib.import_module("dreamx-creator_b200.text_block")
        with pytest.raises(err):
            il.convert_linears_to_int8(nn.Module())
        with pytest.raises(err):
            tb.CrossStack.random_init(dim=64, text_dim=64, heads=1)


def test_conversion_swaps_the_targets(il, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    block = nn.Module()
    block.ffn = nn.Sequential(nn.Linear(32, 64), nn.GELU(), nn.Linear(64, 32))
    model = nn.Module()
    model.blocks = nn.ModuleList([block])
    names = il.convert_linears_to_int8(model, targets=("ffn.0", "ffn.1", "ffn.2", "gone"))
    assert names == ["blocks.0.ffn.0", "blocks.0.ffn.2"]
    assert isinstance(block.ffn[0], il.Int8Linear) and isinstance(block.ffn[1], nn.GELU)
    assert il.convert_linears_to_int8(model, targets=("ffn.0",)) == []


def test_struct_matches_the_header(srdit):
    text = srdit._lib.HEADER.read_text()
    body = re.search(r"typedef struct srdit_cross_attn_args \{(.*?)\} srdit_cross_attn_args;", text,
                     re.S).group(1)
    names = re.findall(r"(\w+)(?:\[\d\])?\s*[,;]", body)
    assert names == [f[0] for f in srdit._lib.CrossAttnArgs._fields_]
    a = srdit._lib.CrossAttnArgs()
    srdit._lib.CROSS_ATTN_LAYOUT.pack_into(a, 0, *range(1, 24), 100, 200, 7, 0.5, 300, 9, 400)
    assert (a.q, a.out, a.dtype, a.D, list(a.q_stride), list(a.o_stride)) == (
        1, 4, 5, 11, [12, 13, 14], [21, 22, 23])
    assert (a.kv_lens, a.key_mask, a.mask_stride, a.scale, a.workspace, a.workspace_bytes,
            a.status) == (100, 200, 7, 0.5, 300, 9, 400)


EINVAL, EALIGN, EUNSUPPORTED = -1, -2, -3


def _norm(L, **kw):
    v = dict(x=4096, ldx=64, M=2, K=64, dtype=0, residual=None, ldr=0, weight=8192, eps=1e-6,
             sum=None, ld_sum=0, q=16384, ldq=64, q_type=0, scale=32768)
    v.update(kw)
    return L.srdit_add_rms_quant(*v.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(M=0), 0), (dict(x=None), EINVAL), (dict(weight=None), EINVAL), (dict(q=None), EINVAL),
    (dict(scale=None), EINVAL), (dict(M=-1), EINVAL), (dict(K=0), EINVAL), (dict(ldx=63), EINVAL),
    (dict(ldq=10), EINVAL), (dict(dtype=3), EINVAL), (dict(q_type=2), EINVAL),
    (dict(eps=-1.0), EINVAL), (dict(eps=float("nan")), EINVAL), (dict(residual=4096), EINVAL),
    (dict(sum=4096), EINVAL), (dict(residual=4096, ldr=64, sum=4096, ld_sum=2), EINVAL),
    (dict(x=4097), EALIGN), (dict(weight=8193), EALIGN), (dict(scale=32770), EALIGN),
    (dict(K=32769, ldx=32769, ldq=32769), EUNSUPPORTED)])
def test_norm_refusals(srdit, kw, rc):
    assert _norm(srdit._lib.lib(), **kw) == rc


def _gemm(L, **kw):
    v = dict(a=4096, a_scale=8192, w=16384, w_scale=32768, bias=None, out=65536, dtype=0, M=4, N=8,
             K=32, lda=32, ldw=32, ldo=8)
    v.update(kw)
    return L.srdit_int8_gemm(*v.values(), None, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(M=0), 0), (dict(N=0), 0), (dict(a=None), EINVAL), (dict(w_scale=None), EINVAL),
    (dict(out=None), EINVAL), (dict(K=0), EINVAL), (dict(M=-1), EINVAL), (dict(lda=16), EINVAL),
    (dict(ldo=7), EINVAL), (dict(dtype=7), EINVAL), (dict(lda=40), EALIGN), (dict(ldw=33), EALIGN),
    (dict(a=4100), EALIGN), (dict(out=65537), EALIGN), (dict(bias=1), EALIGN),
    (dict(dtype=2, out=65538), EALIGN),
    (dict(K=131072, lda=131072, ldw=131072), EUNSUPPORTED)])
def test_gemm_refusals(srdit, kw, rc):
    assert _gemm(srdit._lib.lib(), **kw) == rc


def _attn(L, workspace=False, **kw):
    a = srdit_args = kw.pop("cls")()
    v = dict(q=4096, k=8192, v=16384, out=32768, dtype=0, B=2, Lq=3, Lk=5, H=4, Hkv=2, D=64,
             q_stride=(768, 256, 64), k_stride=(640, 128, 64), v_stride=(640, 128, 64),
             o_stride=(768, 256, 64), scale=0.125)
    v.update(kw)
    for name, x in v.items():
        if isinstance(x, tuple):
            getattr(a, name)[:] = x
        else:
            setattr(a, name, x)
    fn = L.srdit_cross_attn_workspace if workspace else L.srdit_cross_attn
    return fn(ctypes.byref(srdit_args), *(() if workspace else (None,)))


@pytest.mark.parametrize("kw,rc", [
    (dict(B=0), 0), (dict(Lq=0), 0), (dict(q=None), EINVAL), (dict(k=None), EINVAL),
    (dict(out=None), EINVAL), (dict(B=-1), EINVAL), (dict(Hkv=0), EINVAL), (dict(Hkv=3), EINVAL),
    (dict(dtype=2), EINVAL), (dict(scale=0.0), EINVAL), (dict(scale=float("inf")), EINVAL),
    (dict(scale=float("nan")), EINVAL), (dict(D=60), EUNSUPPORTED), (dict(D=136), EUNSUPPORTED),
    (dict(D=0), EUNSUPPORTED), (dict(q=4104), EALIGN), (dict(kv_lens=2), EALIGN),
    (dict(q_stride=(768, 256, 60)), EALIGN), (dict(k_stride=(640, -128, 64)), EALIGN),
    (dict(o_stride=(0, 256, 64)), EINVAL), (dict(q_stride=(768, 0, 64)), EINVAL),
    (dict(k_stride=(640, 0, 64)), EINVAL), (dict(Lq=1 << 25), EUNSUPPORTED),
    (dict(B=40000), EUNSUPPORTED),
    (dict(B=1, Lk=1 << 20, H=1, Hkv=1, Lq=1), EINVAL)])   # split: the workspace is missing
def test_attention_refusals(srdit, kw, rc):
    assert _attn(srdit._lib.lib(), cls=srdit._lib.CrossAttnArgs, **kw) == rc


def test_attention_workspace(srdit):
    """Long contexts of few rows are split over their keys; short ones and refused ones not."""
    L, cls = srdit._lib.lib(), srdit._lib.CrossAttnArgs
    ws = lambda **kw: _attn(L, True, cls=cls, **kw)  # noqa: E731
    assert ws() == 0 and ws(D=60) == 0
    one = dict(B=1, H=1, Hkv=1, Lq=1, Lk=1 << 20)
    parts = ws(**one) * 1024 // (4 * (64 + 2))
    assert parts > 1 and ws(**dict(one, Lk=2048)) == 0
    tiles = ws(B=1, H=1, Hkv=1, Lq=300, Lk=1 << 16)
    assert tiles > 0 and ws(B=33, H=1, Hkv=1, Lq=300, Lk=1 << 16) == 0
