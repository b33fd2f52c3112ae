"""fss_quantize_fp8 and fss_matmul_fp8 against plain 64-bit forms, and their refusals."""
import ctypes

import numpy as np
import pytest
import torch

from fss import _lib
import fp8_attention_util as U

gpu = pytest.mark.gpu


# ------------------------------------------------------------------------------------- quantize
@gpu
@pytest.mark.parametrize('rows,cols,block_rows,x_pad,q_pad,scale_pad', [
    (1, 16, 1, 0, 0, 0), (1, 512, 1, 0, 0, 0), (3, 144, 1, 16, 16, 1), (33, 128, 1, 0, 32, 7),
    (257, 1040, 1, 32, 0, 0), (2145, 2048, 1, 0, 0, 3),
    (1, 16, 128, 0, 0, 0), (127, 272, 128, 16, 16, 2), (129, 128, 128, 0, 0, 0), (512, 2064, 128, 0, 48, 1)])
@pytest.mark.parametrize('dt', ['f32', 'bf16', 'f16', 'f32x3'])
def test_quantize(rows, cols, block_rows, x_pad, q_pad, scale_pad, dt):
    x = U.features(rows, cols, seed=rows + cols)
    x[0, :16] = 0.0
    stored, value = U.store(x, dt, cols + x_pad)
    q, scales, raw = U.quantize(stored, rows, cols, block_rows, dt, q_pad, scale_pad)
    ref_q, ref_scales = U.quantize_ref(value, block_rows)
    # scale: one division, half a step of float
    np.testing.assert_allclose(scales, ref_scales, rtol=2.0 ** -24, atol=0)
    # values: within half an e4m3 step of x / scale (2^-4 relative, 2^-10 below the smallest normal
    # 2^-6), widened by the rounding of the scale (2^-24)
    spread = U.spread(ref_scales, block_rows, rows, cols)
    want = value.astype(np.float64) / spread
    assert np.all(np.abs(q - want) <= np.maximum(np.abs(want) * (2.0 ** -4 + 2.0 ** -22), 2.0 ** -10 * (1 + 2.0 ** -20)))
    # and equal to the exact quotient's rounding, ties included
    assert np.array_equal(q, ref_q)
    assert np.all(raw[:, cols:] == 0x55) and raw.shape[1] == cols + q_pad


@gpu
@pytest.mark.parametrize('block_rows', [1, 128])
def test_quantize_extremes(block_rows):
    rows, cols = 130, 384
    x = U.features(rows, cols, seed=5)
    x[2] = 0.0
    x[128:, 128:256] = 0.0                    # a whole block of zeros
    x[129, 256:] = 1e-38                      # below the smallest scale's range
    x[7, 3] = 3e38
    x[40, 130] = np.inf
    x[41, 131] = -np.nan
    x[50, 300] = -np.inf
    stored, value = U.store(x, 'f32', cols)
    q, scales, _ = U.quantize(stored, rows, cols, block_rows, 'f32')
    ref_q, ref_scales = U.quantize_ref(value, block_rows)
    np.testing.assert_array_equal(np.isnan(scales), np.isnan(ref_scales))
    np.testing.assert_array_equal(q, ref_q)
    assert np.isnan(scales).any() and not np.isnan(scales[0, -1])


@gpu
@pytest.mark.parametrize('dt', ['bf16', 'f16', 'f32'])
@pytest.mark.parametrize('top', [448.0, 7.0, 3.5, 1.3125, 0.013671875, 57344.0, 2.0 ** 127, 2.0 ** -90])
def test_quantize_ties(dt, top):
    """Quotients on and next to the midpoints of e4m3, in its normal and subnormal range."""
    k = np.arange(256, dtype=np.float64)
    mids = np.concatenate([(16 + k[:16] + 0.5) / 16 * 2.0 ** e for e in range(-6, 9)] + [(k[:16] + 0.5) * 2.0 ** -9])
    x = np.concatenate([mids * s * top / 448 for s in (1, -1, 1 + 2.0 ** -23, 1 - 2.0 ** -23, 1 + 2.0 ** -8)])
    x = np.resize(x[np.abs(x) <= top], (31, 128)).astype(np.float32)
    x[:, 5] = top
    if dt == 'f16' and not 2.0 ** -8 <= top <= 65504:
        return
    stored, value = U.store(x, dt, 128)
    for block_rows in (1, 128):
        q, _, _ = U.quantize(stored, 31, 128, block_rows, dt)
        assert np.array_equal(q, U.quantize_ref(value, block_rows)[0])


# --------------------------------------------------------------------------------------- matmul
MATMUL = [
    # rows, cout, k
    (1, 1, 16), (1, 512, 2048), (2, 19, 144), (7, 33, 128), (16, 64, 4096), (17, 129, 272), (33, 256, 512),
    (64, 64, 128), (100, 256, 256), (128, 128, 384), (129, 260, 1040), (255, 513, 528), (300, 72, 8192),
    (1000, 19, 512), (2145, 512, 64), (4097, 136, 160), (8385, 300, 272),
    # k split over the grid
    (128, 128, 16384), (500, 130, 4240), (700, 19, 4224),
    # the larger tiles
    (16500, 520, 144), (8100, 2049, 1040), (4093, 4090, 1040)]


@gpu
@pytest.mark.parametrize('rows,cout,k', MATMUL)
@pytest.mark.parametrize('dt,act,bias,residual', [
    ('f32', None, False, False), ('f32', 'relu6', True, True), ('bf16', 'relu', True, True), ('f16', None, True, True),
    ('bf16', None, True, False)])
def test_matmul(rows, cout, k, dt, act, bias, residual):
    U.check_matmul(rows, cout, k, dt, act, bias, residual)


@gpu
@pytest.mark.parametrize('rows,cout,k', [(1, 8, 16), (50, 136, 272), (1500, 264, 512), (300, 72, 8192)])
def test_matmul_split_bf16_output(rows, cout, k):
    U.check_matmul(rows, cout, k, 'f32x3', 'relu', True, True, y_pad=8)


@gpu
@pytest.mark.parametrize('y_pad,x_pad,w_pad,offset', [(1, 0, 0, 0), (3, 16, 32, 1), (8, 128, 16, 0), (0, 0, 0, 4)])
@pytest.mark.parametrize('rows,cout,k', [(5, 40, 176), (700, 130, 400), (1300, 256, 384)])
def test_matmul_strides(rows, cout, k, y_pad, x_pad, w_pad, offset):
    for dt in ('f32', 'bf16'):
        U.check_matmul(rows, cout, k, dt, None, True, True, y_pad=y_pad, x_pad=x_pad, w_pad=w_pad, offset=offset,
                       scale_pad=3)


@gpu
@pytest.mark.parametrize('rows,cout,k', [(3, 40, 256), (260, 270, 384)])
def test_matmul_carries_nan_and_infinity(rows, cout, k):
    """A NaN block reaches exactly the rows that hold it, relu included; half precision saturates."""
    x, xs, w, ws = U.operands(rows, cout, k, seed=3)
    xs[1, 2] = np.nan
    y = U.matmul(x, xs, w, ws, 'f32', act='relu')
    assert np.isnan(y[2]).all() and not np.isnan(np.delete(y, 2, 0)).any()
    xs[1, 2] = 1e8
    y = U.matmul(x, xs, w, ws, 'f16')
    assert np.isfinite(y).all() and np.abs(y[2]).max() == 65504.0
    y = U.matmul(x, xs, w, ws, 'f16', residual=np.full((rows, cout), np.inf, np.float32))
    assert (y == 65504.0).all()


@gpu
def test_matmul_is_repeatable_and_zero_rows():
    x, xs, w, ws = U.operands(500, 200, 4096, seed=9)
    a = U.matmul(x, xs, w, ws, 'f32')
    for _ in range(3):
        assert np.array_equal(a, U.matmul(x, xs, w, ws, 'f32'))
    d = U.matmul_desc(0, 200, 4096, 'f32')
    _lib.call('fss_matmul_fp8', ctypes.byref(d), *[None] * 8, 0, None)
    _lib.call('fss_quantize_fp8', None, 16, None, 16, None, 0, 0, 16, 1, _lib.F32, None)


# ------------------------------------------------------------------------- refusals (no GPU needed)
def _refused(name, *args):
    with pytest.raises(_lib.FssError):
        _lib.call(name, *args)


def test_quantize_refusals():
    good = dict(x=1 << 12, x_ld=64, q=1 << 13, q_ld=64, scales=1 << 14, scale_ld=4, rows=4, cols=64, block_rows=1,
                dtype=_lib.F32)
    for bad in (dict(x=None), dict(q=None), dict(scales=None), dict(x=4100), dict(q=8200), dict(scales=16386),
                dict(x_ld=48), dict(x_ld=65), dict(q_ld=48), dict(q_ld=72), dict(scale_ld=3), dict(rows=-1), dict(cols=0),
                dict(cols=60), dict(cols=-16), dict(block_rows=2), dict(block_rows=0), dict(dtype=_lib.F16_W2), dict(dtype=9),
                dict(dtype=_lib.F32_BF16X3, x_ld=68), dict(dtype=_lib.BF16, x_ld=68), dict(dtype=_lib.F32_BF16X3, x=4112),
                dict(rows=1 << 50, scale_ld=1 << 50)):
        a = dict(good, **bad)
        _refused('fss_quantize_fp8', a['x'], a['x_ld'], a['q'], a['q_ld'], a['scales'], a['scale_ld'], a['rows'], a['cols'],
                 a['block_rows'], a['dtype'], None)


def test_matmul_refusals():
    ptr = dict(x=1 << 12, xs=1 << 12, w=1 << 12, ws=1 << 12, bias=None, residual=None, y=1 << 12)
    for bad in (dict(x=None), dict(w=None), dict(xs=None), dict(ws=None), dict(y=None), dict(x=4104), dict(w=4097),
                dict(bias=4100), dict(y=4097), dict(residual=4098), dict(xs=4097), dict(ws=4098)):
        p = dict(ptr, **bad)
        d = U.matmul_desc(8, 24, 256, 'f32')
        _refused('fss_matmul_fp8', ctypes.byref(d), p['x'], p['xs'], p['w'], p['ws'], p['bias'], p['residual'], p['y'], None,
                 0, None)
    for bad in (dict(rows=-1), dict(cout=0), dict(cout=-3), dict(k=0), dict(k=100), dict(k=-16), dict(act=7), dict(out_dtype=4),
                dict(out_dtype=-1), dict(x_ld=128), dict(x_ld=260), dict(w_ld=240), dict(w_ld=264), dict(x_ld=1 << 23),
                dict(w_ld=1 << 23), dict(x_scale_ld=7), dict(w_scale_ld=0), dict(y_ld=23), dict(res_ld=23),
                dict(out_dtype=_lib.F32_BF16X3, y_ld=28), dict(out_dtype=_lib.F32_BF16X3, cout=20, w_scale_ld=1),
                dict(out_dtype=_lib.F32_BF16X3, res_ld=28), dict(rows=1 << 50, x_scale_ld=1 << 50),
                dict(rows=1 << 62, x_scale_ld=1 << 62), dict(cout=1 << 28, w_scale_ld=1 << 28, y_ld=1 << 28, res_ld=1 << 28)):
        d = U.matmul_desc(**dict(dict(rows=8, cout=24, k=256, dt='f32', x_scale_ld=8, w_scale_ld=1, x_ld=256, w_ld=256,
                                      y_ld=24, res_ld=24), **bad))
        _refused('fss_matmul_fp8', ctypes.byref(d), *[1 << 12] * 7, None, 0, None)
    size = ctypes.c_size_t()
    d = U.matmul_desc(300, 256, 8192, 'f32')
    _lib.call('fss_matmul_fp8_workspace_bytes', ctypes.byref(d), ctypes.byref(size))
    assert size.value > 0
    for ws, n in ((None, size.value), (1 << 12, size.value - 1), ((1 << 12) + 8, size.value), (None, 0)):
        _refused('fss_matmul_fp8', ctypes.byref(d), *[1 << 12] * 4, None, None, 1 << 12, ws, n, None)
    _refused('fss_matmul_fp8_workspace_bytes', ctypes.byref(U.matmul_desc(8, 24, 100, 'f32')), ctypes.byref(size))
    _refused('fss_matmul_fp8_workspace_bytes', ctypes.byref(U.matmul_desc(8, 24, 128, 'f32')), None)
    _refused('fss_matmul_fp8_workspace_bytes', None, ctypes.byref(size))
    _refused('fss_matmul_fp8', None, *[1 << 12] * 7, None, 0, None)
