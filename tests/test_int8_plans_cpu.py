"""How products and attention calls are run, asked of the library without a GPU (which then
goes by a B200's SMs)."""
import ctypes

import pytest


@pytest.mark.parametrize("M,N,K,columns", [
    (1, 16, 64, 0), (32, 4096, 4096, 0), (33, 200, 1584, 64), (33, 200, 1600, 0),
    (64, 1024, 1024, 64), (64, 4096, 4096, 0), (64, 16400, 1540, 0), (65, 96, 160, 64),
    (57001, 63, 130, 64),
    (57001, 127, 130, 128), (57001, 190, 130, 192), (57001, 255, 130, 256), (9527, 779, 300, 192),
    (6912, 14336, 3072, 256), (0, 8, 8, 0), (8, 0, 8, 0), (8, 8, 0, 0)])
def test_product_columns(srdit, M, N, K, columns):
    assert srdit._lib.lib().srdit_int8_gemm_columns(M, N, K) == columns


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,items", [
    (1, 6912, 512, 24, 24, 648), (1, 256, 100, 1, 1, 1), (1, 257, 100, 1, 1, 2),
    (3, 1, 100, 4, 1, 0), (2, 16, 9, 2, 2, 0), (2, 17, 9, 2, 2, 4), (1, 17, 9, 2, 1, 1),
    (1, 64, 9, 4, 1, 1), (1, 65, 9, 4, 1, 2), (1, 300, 0, 2, 2, 4), (0, 300, 9, 2, 2, 0), (1, 300, 9, 3, 2, 0)])
def test_attention_items(srdit, B, Lq, Lk, H, Hkv, items):
    """256 rows an item: tokens of one head, or heads of a group side by side."""
    a, D = srdit._lib.CrossAttnArgs(), 64
    kv = (Lk * Hkv * D, Hkv * D, D)
    srdit._lib.CROSS_ATTN_LAYOUT.pack_into(
        a, 0, 4096, 8192, 16384, 32768, 0, B, Lq, Lk, H, Hkv, D, Lq * H * D, H * D, D, *kv, *kv,
        Lq * H * D, H * D, D, 0, 0, 0, 0.125, 0, 0, 0)
    assert srdit._lib.lib().srdit_cross_attn_items(ctypes.byref(a)) == items
