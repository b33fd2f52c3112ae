"""Sizes at the ends of what fss_quantize_fp8, fss_matmul_fp8 and fss_cross_attention take."""
import ctypes

import pytest
import torch

from fss import _lib
import fp8_attention_util as U

gpu = pytest.mark.gpu


@gpu
def test_quantize_more_than_2_to_32_threads():
    """Rows past what one launch holds: the first ones, those around the border and the last equal a small call's."""
    cols, per = 16, 1 << 29                         # 32 rows a workgroup of 256
    rows = per + 75
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device='cuda')               # 17 GB
    q = torch.full((rows, cols), 0x55, dtype=torch.uint8, device='cuda')
    scales = torch.full((1, rows), -77.0, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(1)
    spots = [(0, 384), (per - 384, 384), (per, 75)]
    for a, n in spots:
        x[a:a + n] = torch.randn(n, cols, generator=g, device='cuda').to(torch.bfloat16)
    _lib.call('fss_quantize_fp8', x.data_ptr(), cols, q.data_ptr(), cols, scales.data_ptr(), rows, rows, cols, 1, _lib.BF16,
              U.stream())
    for a, n in spots:
        q1, s1, _ = U.quantize(x[a:a + n].clone(), n, cols, 1, 'bf16')
        assert torch.equal(q[a:a + n].view(torch.float8_e4m3fn).float().cpu(), torch.from_numpy(q1))
        assert torch.equal(scales[0, a:a + n].cpu(), torch.from_numpy(s1[0]))
    assert int((scales == -77.0).sum()) == 0


def test_quantize_refuses_columns_past_one_launch():
    cols = (1 << 31) - 16
    with pytest.raises(_lib.FssError, match='columns'):
        _lib.call('fss_quantize_fp8', 4096, cols, 4096, cols, 4096, 1, 1, cols, 1, _lib.BF16, None)
