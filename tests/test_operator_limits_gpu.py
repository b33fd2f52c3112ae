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


# A launch of 2^32 threads or more would be cut off without an error.
@pytest.mark.parametrize('sizes', [dict(rows=1 << 32, cout=1, k=16), dict(rows=(1 << 31), cout=128, k=1024),
                                   dict(rows=1 << 27, cout=1 << 14, k=1024),
                                   dict(rows=(1 << 40) - 1, cout=1 << 25, k=1 << 17)])
def test_matmul_refuses_more_than_one_launch(sizes):
    d = U.matmul_desc(sizes['rows'], sizes['cout'], sizes['k'], 'bf16')
    with pytest.raises(_lib.FssError, match='too many tiles'):
        _lib.call('fss_matmul_fp8', ctypes.byref(d), *[4096] * 4, None, None, 4096, None, 0, None)


@pytest.mark.parametrize('batch,q_len,q_heads,kv_heads,head_dim', [
    (1024, 1 << 20, 4, 2, 64), (2, 1 << 30, 1, 1, 8), (1 << 24, 33, 1, 1, 8), (1 << 26, 1, 1, 1, 8), (2, (1 << 28), 4, 1, 256),
    ((1 << 24) // 3 + 1, 300, 1, 1, 32), ((1 << 23) // 2, 257, 1, 1, 200)])
def test_attention_refuses_more_than_one_launch(batch, q_len, q_heads, kv_heads, head_dim):
    d = U.attention_desc(batch, q_len, 5, q_heads, kv_heads, head_dim, 'bf16')
    size = ctypes.c_size_t()
    for call in (lambda: _lib.call('fss_cross_attention', ctypes.byref(d), *[4096] * 3, None, None, 4096, 4096, 1 << 60, None),
                 lambda: _lib.call('fss_cross_attention_workspace_bytes', ctypes.byref(d), ctypes.byref(size))):
        with pytest.raises(_lib.FssError, match='too many quer'):
            call()


@pytest.mark.parametrize('batch,q_len,q_heads,kv_heads,head_dim', [
    ((1 << 26) - 1, 1, 1, 1, 8), ((1 << 24) - 1, 33, 1, 1, 8), ((1 << 23) - 1, 129, 1, 1, 256), (1, 0x7fff0000 // 4, 1, 1, 8)])
def test_attention_takes_what_one_launch_holds(batch, q_len, q_heads, kv_heads, head_dim):
    d = U.attention_desc(batch, q_len, 5, q_heads, kv_heads, head_dim, 'bf16')
    size = ctypes.c_size_t(7)
    _lib.call('fss_cross_attention_workspace_bytes', ctypes.byref(d), ctypes.byref(size))
    assert size.value == 0
