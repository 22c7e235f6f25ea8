"""Text-conditioning blocks on the GPU where their inputs are empty, broadcast or views."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def stack(srdit, cuda_device):
    return srdit.text_block.CrossStack.random_init(dim=128, text_dim=96, heads=2, layers=3, seed=3)


def _inputs(B, L, Lk):
    g = torch.Generator(device="cuda").manual_seed(L + Lk)
    return tuple(torch.randn(B, n, d, generator=g, device="cuda").to(torch.bfloat16)
                 for n, d in ((L, 128), (Lk, 96)))


@pytest.mark.parametrize("L,Lk", [(1, 0), (300, 0), (0, 7), (0, 0)])
def test_no_keys_or_no_tokens(stack, L, Lk):
    """A prompt without states adds the output Linears' biases; no tokens, no output."""
    x, states = _inputs(2, L, Lk)
    out = stack(x, stack.text_kv(states))
    assert out.shape == x.shape and out.dtype == x.dtype
    want = x
    for b in stack.blocks:   # an output is the bias alone, each sum rounded to bf16
        want = want + b.o.bias
    assert torch.equal(out, want if L else x)


@pytest.mark.parametrize("L", (1, 70))
def test_a_block_leaves_its_arguments(stack, L):
    x, states = _inputs(2, L, 7)
    y = x.flip(1).contiguous() * 0.5
    x0, y0 = x.clone(), y.clone()
    kv = stack.text_kv(states)
    total, out = stack.blocks[0](x, y, kv[0])
    assert torch.equal(x, x0) and torch.equal(y, y0) and torch.equal(total, x0 + y0)
    over, again = stack.blocks[0](x, y, kv[0], into_y=True)
    assert over.data_ptr() == y.data_ptr() and torch.equal(over, total) and torch.equal(out, again)


def test_broadcast_inputs_and_single_rows(stack, srdit):
    """Rows expanded over tokens or samples, and single rows of any stride, as their copies."""
    x, states = _inputs(2, 5, 7)
    xe, se = x[:1, :1].expand(2, 5, 128), states[:1].expand(2, 7, 96)
    out = stack(xe, stack.text_kv(se))
    assert torch.equal(out, stack(xe.clone(), stack.text_kv(se.clone())))
    kv = stack.text_kv(states)
    for a, b in zip(stack.blocks[0](xe, x[:, 1:2].expand(2, 5, 128), kv[0]),
                    stack.blocks[0](xe.clone(), x[:, 1:2].expand(2, 5, 128).clone(), kv[0])):
        assert torch.equal(a, b)
    lin = stack.blocks[0].kv
    row = states[0, :1]
    want = lin(row)
    assert torch.equal(lin(row.expand(4, 96)), want.expand(4, -1))
    column = row.as_strided((1, 96), (1, 1))   # a transposed column
    assert column.stride() == (1, 1) and torch.equal(lin(column), want)
    one = x[0, :1]
    column = one.as_strided((1, 128), (1, 1))
    w = torch.ones(128, device="cuda", dtype=torch.bfloat16)
    for got, ref in zip(srdit.ops.add_rms_quant(column, w, residual=column),
                        srdit.ops.add_rms_quant(one, w, residual=one)):
        assert torch.equal(got, ref)


@pytest.mark.parametrize("K", (64, 100))
def test_products_of_single_rows(srdit, cuda_device, K):
    """One token, one output channel: a pitch that is not a multiple of 16 is not used."""
    g = torch.Generator(device="cuda").manual_seed(K)
    a, w = (torch.randint(-128, 128, (n, (K + 15) // 16 * 16), generator=g, device="cuda")
            .to(torch.int8)[:, :K] for n in (5, 7))
    one = torch.ones(7, device="cuda")
    y = srdit.ops.int8_gemm(a, one[:5], w, one, out_dtype=torch.float32)
    for pitch in (1, K, K + 1):
        row, column = a[2:3].as_strided((1, K), (pitch, 1)), w[:1].as_strided((1, K), (pitch, 1))
        out = torch.empty(7, device="cuda").as_strided((1, 7), (1, 1))
        srdit.ops.int8_gemm(row, one[:1], w, one, out=out)
        assert torch.equal(out[0], y[2])
        assert torch.equal(srdit.ops.int8_gemm(a, one[:5], column, one[:1],
                                               out_dtype=torch.float32), y[:, :1])
