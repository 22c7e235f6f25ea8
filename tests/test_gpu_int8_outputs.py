"""The int8 product into a part of a wider buffer: what lies beside it is left alone."""
import pytest
import torch

from .test_gpu_int8_ops import DTYPES, _check_gemm, _codes, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", (1, 40, 70, 300))
@pytest.mark.parametrize("N", (1, 61, 63, 66, 124, 255, 300))
@pytest.mark.parametrize("off", (0, 8))
def test_columns_beside_the_output(srdit, cuda_device, dtype, M, N, off):
    """Aligned rows (a pitch and an offset of whole 16-byte pieces) of a width that is not."""
    g = _gen(M + N)
    pitch = (N + 31) // 16 * 16
    buf = torch.full((M + 2, pitch), 5.0, dtype=dtype, device="cuda")
    _check_gemm(srdit, _codes(srdit, g, M, 130), _codes(srdit, g, N, 130), dtype, True, g,
                buf[1:M + 1, off:off + N])
    buf[1:M + 1, off:off + N] = 5
    assert (buf == 5).all()
