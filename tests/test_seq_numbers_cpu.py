"""Sizes and numbers that the C structures do not hold are refused by the paged cache's and the
packed attention's wrappers, as everything else is, before anything is launched."""
import pytest
import torch

DT = torch.bfloat16


@pytest.fixture
def ops(srdit, monkeypatch):
    """The wrappers with tensors of the CPU let through: all that is called here is refused by
    them, or by the C entries from the sizes alone."""
    monkeypatch.setattr(srdit.ops, "_calls", None)
    monkeypatch.setattr(srdit.ops, "_same_device", lambda *t: 0)
    return srdit.ops


def _cache(size=16, width=1, pages=3):
    pool = torch.zeros(pages, size, 1, 16, dtype=DT)
    return pool, pool.clone(), torch.zeros(1, width, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)


@pytest.mark.parametrize("kw", (
    dict(max_q=2 ** 31), dict(max_q=-2 ** 31 - 1), dict(max_kv=2 ** 31), dict(max_kv=2 ** 70),
    dict(max_q=1.0), dict(max_kv="1"), dict(scale=1e39), dict(scale="1"), dict(max_q=-1), dict(max_kv=-1),
    dict(scale=float("inf")), dict(scale=float("nan"))))
def test_numbers(srdit, ops, kw):
    k, v, table, lens = _cache()
    with pytest.raises(srdit._lib.SrditError):
        ops.paged_attn(torch.zeros(1, 1, 16, dtype=DT), k, v, table, lens, **kw)


@pytest.mark.parametrize("scale", (2.4e38, 3.4e38))
def test_a_scale_without_a_factor_in_base_2(srdit, ops, scale):
    """scale log2(e) beyond fp32: rows whose scores are 0 would be NaN."""
    x, cu = torch.zeros(1, 1, 16, dtype=DT), torch.tensor([0, 1], dtype=torch.int32)
    with pytest.raises(srdit._lib.SrditError, match="-1"):
        ops.packed_attn(x, x, x, cu, scale=scale)


@pytest.mark.parametrize("max_kv", (None, 0, 7))
def test_a_table_of_more_than_the_kernels_count(srdit, ops, max_kv):
    k, v, table, lens = _cache(size=1 << 24, width=256, pages=0)   # 2^32 tokens
    with pytest.raises(srdit._lib.SrditError):
        ops.paged_attn(torch.zeros(1, 1, 16, dtype=DT), k, v, table, lens, max_kv=max_kv)


@pytest.mark.parametrize("tokens", (2 ** 31, 2 ** 32 + 5))
def test_more_rows_than_a_whole_number_of_32_bits(srdit, ops, tokens):
    """... whose low bits are not taken for the number."""
    k, v, table, lens = _cache()
    rows = torch.zeros(1, 1, 16, dtype=DT).expand(tokens, 1, 16)
    cu = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.kv_write(rows, rows, k, v, table, lens),
                 lambda: ops.kv_read(k, v, table, cu, rows, rows),
                 lambda: ops.paged_attn(rows, k, v, table, lens, rows),
                 lambda: ops.packed_attn(rows, rows, rows, cu, rows),
                 lambda: ops.packed_attn(rows[:1], rows, rows, cu, rows[:1], cu_k=cu)):
        with pytest.raises(srdit._lib.SrditError):
            call()
