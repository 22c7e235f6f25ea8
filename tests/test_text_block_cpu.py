"""Host-side logic of the text-conditioning blocks (no GPU)."""
import pathlib
import subprocess
import sys

import pytest
import torch

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_the_package_brings_the_blocks():
    """``srdit.text_block`` after importing the package alone, as its documentation has it (in
    a process of its own: another test may have imported the submodule)."""
    code = ("import importlib; srdit = importlib.import_module('dreamx-creator_b200'); "
            "print(srdit.text_block.CrossStack.__name__, 'text_block' in srdit.__all__)")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-500:]
    assert r.stdout.split() == ["CrossStack", "True"]


# ------------------------------------------------------------------ on plain operators
def _add_rms_quant(x, weight, eps=1e-6, *, residual=None, sum_out=None, qdtype=None, q=None,
                   qscale=None):
    s = x if residual is None else x + residual
    if residual is not None:
        s = s if sum_out is None else sum_out.copy_(s)
    n = s.float() * (s.float().pow(2).mean(1, keepdim=True) + eps).rsqrt() * weight.float()
    q, scale = _quant_rows(n)
    return q, scale, None if residual is None else s


def _quant_rows(x, **_):
    scale = (x.float().abs().amax(1) / 127).clamp_min(1e-12)
    return torch.round(x.float() / scale[:, None]).to(torch.int8), scale


def _int8_gemm(a, sa, w, sw, bias=None, out=None, *, out_dtype=None, status=None):
    return ((a.float() @ w.float().t()) * sa[:, None] * sw + bias.float()).to(out_dtype)


def _cross_attn(q, k, v, out=None, *, kv_lens=None, key_mask=None, scale=None, status=None):
    if k.shape[1] == 0:
        return torch.zeros_like(q)
    s = torch.einsum("bihd,bjhd->bhij", q.float(), k.float()) * q.shape[-1] ** -0.5
    return torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v.float()).to(q.dtype).contiguous()


@pytest.fixture
def stack(srdit, monkeypatch):
    """Two blocks of two heads of 32 on plain operators."""
    for name, fn in (("add_rms_quant", _add_rms_quant), ("quant_rows", _quant_rows),
                     ("int8_gemm", _int8_gemm), ("cross_attn", _cross_attn)):
        monkeypatch.setattr(srdit.ops, name, fn)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    return srdit.text_block.CrossStack.random_init(dim=64, text_dim=48, heads=2, layers=3,
                                                   device="cpu", dtype=torch.float32)


def _inputs(L=5, Lk=7):
    g = torch.Generator().manual_seed(1)
    return tuple(torch.randn(2, n, d, generator=g) for n, d in ((L, 64), (L, 64), (Lk, 48)))


def test_a_block_leaves_its_arguments(stack):
    """x and y are the caller's: a block's sum is a tensor of its own, unless it is told that
    it may write it over y."""
    x, y, states = _inputs()
    x0, y0 = x.clone(), y.clone()
    kv = stack.text_kv(states)
    total, out = stack.blocks[0](x, y, kv[0])
    assert torch.equal(x, x0) and torch.equal(y, y0) and torch.equal(total, x0 + y0)
    over, out1 = stack.blocks[0](x, y, kv[0], into_y=True)
    assert over.data_ptr() == y.data_ptr() and torch.equal(over, total) and torch.equal(out, out1)
    assert torch.equal(x, x0)


def test_a_stack_adds_every_output(stack):
    x, _, states = _inputs()
    x0, kv = x.clone(), stack.text_kv(states)
    out = stack(x, kv)
    assert torch.equal(x, x0)
    total, y = x, None
    for block, bkv in zip(stack.blocks, kv):
        total, y = block(total, y, bkv)
    assert torch.equal(out, total + y)


@pytest.mark.parametrize("L,Lk", [(5, 0), (0, 7), (0, 0)])
def test_no_keys_or_no_tokens(stack, L, Lk):
    """A prompt without states adds the output Linears' biases; no tokens, no output."""
    x, _, states = _inputs(L, Lk)
    out = stack(x, stack.text_kv(states))
    assert out.shape == x.shape
    want = x + sum(b.o.bias for b in stack.blocks) if Lk == 0 else x
    assert torch.allclose(out, want, atol=1e-5)


# ------------------------------------------------------------------ rows of other layouts
@pytest.mark.parametrize("x", [
    torch.randn(1, 48).expand(4, 48), torch.randn(2, 1, 48).expand(2, 3, 48),
    torch.randn(1, 3, 48).expand(2, 3, 48), torch.randn(48, 3).t(), torch.randn(48, 1).t(),
    torch.randn(4, 6, 48)[:, 1], torch.randn(100).as_strided((4, 48), (5, 1)),
    torch.randn(0, 48), torch.randn(48)])
def test_the_linear_takes_rows_of_any_layout(srdit, stack, monkeypatch, x):
    """Expanded, transposed and overlapping rows reach the quantiser as rows a pitch of their
    width apart at least."""
    seen = []
    plain = srdit.ops.quant_rows
    monkeypatch.setattr(srdit.ops, "quant_rows", lambda r, **kw: (seen.append(r), plain(r))[1])
    lin = stack.blocks[0].kv
    y = lin(x)
    assert y.shape == (*x.shape[:-1], lin.out_features)
    rows = seen[0]
    assert srdit.ops._rows(rows) >= 48 or rows.shape[0] == 1   # whose pitch is not used
    assert torch.equal(rows, x.reshape(-1, 48))
    assert torch.equal(y, lin(x.clone(memory_format=torch.contiguous_format)))


def test_a_stack_takes_broadcast_inputs(stack, srdit, monkeypatch):
    x, _, states = _inputs()
    pitches = []
    for name in ("add_rms_quant", "quant_rows"):
        fn = getattr(srdit.ops, name)
        monkeypatch.setattr(srdit.ops, name, lambda r, *a, fn=fn, **kw: (
            pitches.append((srdit.ops._rows(r), r.shape[1])), fn(r, *a, **kw))[1])
    xe, se = x[:1, :1].expand(2, 5, 64), states[:1].expand(2, 7, 48)
    out = stack(xe, stack.text_kv(se))
    assert torch.equal(out, stack(xe.clone(), stack.text_kv(se.clone())))
    ye = x[:1, 1:2].expand(2, 5, 64)
    stack.blocks[0](xe, ye, stack.text_kv(se)[0])
    assert all(p >= k for p, k in pitches)
