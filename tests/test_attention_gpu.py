"""fss_cross_attention against a plain 64-bit form, and its refusals."""
import ctypes

import numpy as np
import pytest
import torch

from fss import _lib
import fp8_attention_util as U

gpu = pytest.mark.gpu


def tensors(b, lq, lk, hq, hk, d, dt, seed):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g).to(U.TORCH[dt]).cuda()
    return make(b, lq, hq, d), make(b, lk, hk, d), make(b, lk, hk, d)


def keys_mask(b, h, lq, lk, seed, share=0.5):
    m = torch.rand(b, h, lq, lk, generator=torch.Generator().manual_seed(seed)) < share
    return m.cuda()


SHAPES = [
    # batch, q_len, kv_len, q_heads, kv_heads, head_dim
    (1, 1, 1, 1, 1, 8), (1, 1, 2145, 8, 8, 32), (2, 1, 700, 8, 2, 64), (1, 3, 63, 2, 1, 128), (2, 5, 64, 6, 2, 40),
    (1, 32, 65, 1, 1, 256), (1, 33, 129, 2, 2, 72), (3, 100, 1000, 4, 4, 32), (1, 128, 127, 3, 3, 96),
    (1, 130, 50, 8, 8, 64), (2, 257, 191, 4, 1, 128), (1, 600, 320, 7, 1, 16), (1, 70, 515, 2, 1, 200), (1, 129, 1, 2, 2, 64),
    (1, 2000, 50, 8, 8, 64), (1, 31, 4000, 1, 1, 256), (4, 1, 33, 14, 2, 136),
    (1, 200, 2600, 2, 1, 256), (1, 64, 1500, 4, 4, 160), (2, 90, 1100, 3, 3, 24), (1, 150, 1200, 2, 2, 64)]


@gpu
@pytest.mark.parametrize('shape', SHAPES)
@pytest.mark.parametrize('dt', ['bf16', 'f16'])
def test_attention(shape, dt):
    q, k, v = tensors(*shape, dt, seed=sum(shape))
    U.check_attention(U.attend(q, k, v, dt), U.attention_ref(q, k, v), dt, shape[5], shape[2])


@gpu
@pytest.mark.parametrize('shape', SHAPES)
def test_attention_mask_and_lengths(shape):
    """Boolean masks with empty rows, ragged lengths (0 and more than kv_len among them), infinities
    and NaN in every place that is not seen."""
    b, lq, lk, hq, hk, d = shape
    dt = 'bf16'
    q, k, v = tensors(*shape, dt, seed=1 + sum(shape))
    lens = torch.tensor([[lk, lk // 2, 0, lk + 5][i % 4] for i in range(b)], dtype=torch.int32).cuda()
    for i in range(b):
        n = min(int(lens[i]), lk)
        k[i, n:] = float('nan')
        v[i, n:] = float('inf')
    mask = keys_mask(b, hq, lq, lk, seed=lk)
    mask[:, :, ::3] = False
    U.check_attention(U.attend(q, k, v, dt, lens=lens, mask=mask), U.attention_ref(q, k, v, lens=lens, mask=mask), dt, d, lk)
    # a key that nobody sees, and one that every second query sees
    mask[:, :, :, lk // 3] = False
    k[:, lk // 3] = float('nan')
    v[:, lk // 3] = float('nan')
    U.check_attention(U.attend(q, k, v, dt, lens=lens, mask=mask), U.attention_ref(q, k, v, lens=lens, mask=mask), dt, d, lk)
    mask[:, :, 1::2, lk // 2] = False
    mask[:, :, 0::2, lk // 2] = True
    v[:, lk // 2, :, :4] = float('inf')
    y = U.attend(q, k, v, dt, lens=lens, mask=mask)
    ref = U.attention_ref(q[:, 1::2], k, v, lens=lens, mask=mask[:, :, 1::2])
    U.check_attention(y[:, 1::2], ref, dt, d, lk)


@gpu
@pytest.mark.parametrize('lq,lk', [(5, 333), (200, 130)])
def test_attention_mask_strides(lq, lk):
    """One mask for all heads, for all queries, for the whole batch; a row stride that is odd."""
    shape = (2, lq, lk, 4, 2, 64)
    q, k, v = tensors(*shape, 'f16', seed=3)
    full = keys_mask(2, 4, lq, lk + 3, seed=4, share=0.3)
    for m in (full[:, :1, :, :lk].expand(2, 4, lq, lk), full[:, :, :1, 1:lk + 1].expand(2, 4, lq, lk),
              full[:1, :, :, 3:].expand(2, 4, lq, lk), full[:, :, :, :lk]):
        U.check_attention(U.attend(q, k, v, 'f16', mask=m), U.attention_ref(q, k, v, mask=m), 'f16', 64, lk)
    # any value but 0 counts
    m8 = full[:, :, :, :lk].to(torch.uint8) * 128
    assert torch.equal(U.attend(q, k, v, 'f16', mask=m8), U.attend(q, k, v, 'f16', mask=full[:, :, :, :lk]))


@gpu
@pytest.mark.parametrize('lq,lk,d', [(3, 300, 32), (140, 200, 64), (40, 90, 128)])
def test_attention_strides(lq, lk, d):
    """q, k and v as slices of one projection, heads before tokens, y inside a wider tensor."""
    b, hq, hk, dt = 2, 4, 2, 'bf16'
    g = torch.Generator().manual_seed(lq)
    kv = torch.randn(b, lk, 2, hk, d + 8, generator=g).to(torch.bfloat16).cuda()
    q = torch.randn(b, hq, lq, d, generator=g).to(torch.bfloat16).cuda().permute(0, 2, 1, 3)
    wide = torch.full((b, lq, hq + 1, d + 16), -77.0, dtype=torch.bfloat16, device='cuda')
    y = wide[:, :, 1:, 8:8 + d]
    k, v = kv[:, :, 0, :, :d], kv[:, :, 1, :, 8:]
    U.check_attention(U.attend(q, k, v, dt, y=y), U.attention_ref(q, k, v), dt, d, lk)
    wide[:, :, 1:, 8:8 + d] = -77.0
    assert (wide == -77.0).all()
    # one set of keys for the whole batch
    k1, v1 = k[:1].expand_as(k), v[:1].expand_as(v)
    U.check_attention(U.attend(q, k1, v1, dt), U.attention_ref(q, k1, v1), dt, d, lk)


@gpu
@pytest.mark.parametrize('lq', [2, 150])
@pytest.mark.parametrize('scale', [0.0, -0.3, 1e-4, 3.0])
def test_attention_scale(lq, scale):
    shape = (1, lq, 260, 2, 2, 32)
    q, k, v = tensors(*shape, 'f16', seed=8)
    U.check_attention(U.attend(q, k, v, 'f16', scale=scale), U.attention_ref(q, k, v, scale=scale), 'f16', 32, 260)


@gpu
@pytest.mark.parametrize('lq', [2, 150])
def test_attention_growing_scores(lq):
    """Scores that rise along the keys move the maximum in every tile; a lone huge one hides the rest."""
    lk, d = 520, 64
    q, k, v = tensors(1, lq, lk, 2, 2, d, 'bf16', seed=2)
    q = torch.ones_like(q)
    k = (torch.arange(lk, device='cuda')[None, :, None, None] * 0.05 * torch.ones_like(k)).to(torch.bfloat16)
    U.check_attention(U.attend(q, k, v, 'bf16'), U.attention_ref(q, k, v), 'bf16', d, lk)
    k[:, 300] = 1000.0
    y = U.attend(q, k, v, 'bf16')
    assert torch.equal(y, v[:, 300:301].expand_as(y))


@gpu
def test_attention_carries_seen_nan():
    for lq in (2, 150):
        q, k, v = tensors(1, lq, 200, 2, 2, 64, 'bf16', seed=2)
        v[0, 77, 1, 5] = float('nan')
        y = U.attend(q, k, v, 'bf16')
        assert torch.isnan(y[0, :, 1, 5]).all() and torch.isnan(y).sum() == lq
        k[0, 77, 0] = float('nan')
        assert torch.isnan(U.attend(q, k, v, 'bf16')[0, :, 0]).all()


@gpu
@pytest.mark.parametrize('lq,lk', [(1, 1000), (40, 40000), (1, 300)])
def test_attention_carries_a_piece_of_nan(lq, lk):
    """Where the key axis is cut into pieces: all keys of one are NaN, and a query that is."""
    q, k, v = tensors(1, lq, lk, 2, 2, 64, 'bf16', seed=2)
    n = lk // 3
    k[0, n:2 * n, 1] = float('nan')
    y = U.attend(q, k, v, 'bf16')
    assert torch.isnan(y[:, :, 1]).all() and not torch.isnan(y[:, :, 0]).any()
    q[0, 0, 0] = float('nan')
    assert torch.isnan(U.attend(q, k, v, 'bf16')[0, 0]).all()


@gpu
def test_attention_empty():
    q, k, v = tensors(2, 5, 0, 2, 2, 64, 'bf16', seed=1)
    assert (U.attend(q, k, v, 'bf16') == 0).all()
    d = U.attention_desc(0, 5, 5, 2, 2, 64, 'bf16')
    _lib.call('fss_cross_attention', ctypes.byref(d), *[None] * 7, 0, None)
    d = U.attention_desc(2, 0, 5, 2, 2, 64, 'bf16')
    _lib.call('fss_cross_attention', ctypes.byref(d), *[None] * 7, 0, None)


@gpu
def test_attention_far_tokens():
    """Key and value tensors whose batch entries and tokens lie more than 2^32 bytes apart."""
    d, lk, stride = 64, 300, 1 << 23                      # 16 MiB between tokens: 4.7 GiB per tensor
    k, v = (torch.empty(lk * stride, dtype=torch.bfloat16, device='cuda').as_strided((1, lk, 1, d), (0, stride, 0, 1))
            for _ in range(2))
    q, k0, v0 = tensors(1, 40, lk, 2, 1, d, 'bf16', seed=6)
    k.copy_(k0)
    v.copy_(v0)
    assert torch.equal(U.attend(q, k, v, 'bf16'), U.attend(q, k0, v0, 'bf16'))
    assert torch.equal(U.attend(q[:, :1], k, v, 'bf16'), U.attend(q[:, :1], k0, v0, 'bf16'))


@gpu
def test_attention_is_repeatable():
    for shape in ((1, 1, 5000, 8, 8, 32), (2, 300, 2000, 4, 2, 64)):
        q, k, v = tensors(*shape, 'bf16', seed=1)
        a = U.attend(q, k, v, 'bf16')
        for _ in range(3):
            assert torch.equal(a, U.attend(q, k, v, 'bf16'))


# ------------------------------------------------------------------------- refusals (no GPU needed)
def _refused(desc, args):
    with pytest.raises(_lib.FssError):
        _lib.call('fss_cross_attention', None if desc is None else ctypes.byref(desc), *args)


def test_attention_refusals():
    p = 1 << 12
    good = dict(batch=2, q_len=5, kv_len=4000, q_heads=4, kv_heads=2, head_dim=64, dt='bf16')
    args = [p, p, p, None, None, p, p, 1 << 40, None]
    for bad in (dict(batch=-1), dict(q_len=-1), dict(kv_len=-1), dict(q_heads=3), dict(q_heads=0), dict(kv_heads=0),
                dict(kv_heads=-2), dict(head_dim=0), dict(head_dim=60), dict(head_dim=264), dict(scale=float('nan')),
                dict(scale=float('inf')), dict(dtype=_lib.F32), dict(dtype=_lib.F32_BF16X3), dict(q_stride=(8, 4, 8)),
                dict(k_stride=(8, 8, 12)), dict(v_stride=(-8, 8, 8)), dict(y_stride=(8, 1 << 24, 8)),
                dict(k_stride=(8, 1 << 24, 8)), dict(mask_stride=(-1, 0, 0)), dict(q_len=1 << 30, q_heads=64),
                dict(batch=1 << 20, q_len=1 << 20)):
        a = list(args)
        if 'mask_stride' in bad:
            a[4] = p
        _refused(U.attention_desc(**dict(good, **bad)), a)
    d = U.attention_desc(**good)
    for i, value in ((0, None), (1, None), (2, None), (5, None), (0, p + 8), (1, p + 2), (2, p + 4), (5, p + 8), (3, p + 2),
                     (6, p + 8), (6, None), (7, 64)):
        a = list(args)
        a[i] = value
        _refused(d, a)
    _refused(None, args)
    size = ctypes.c_size_t()
    for fn_args in ((None, ctypes.byref(size)), (ctypes.byref(d), None),
                    (ctypes.byref(U.attention_desc(**dict(good, head_dim=4))), ctypes.byref(size))):
        with pytest.raises(_lib.FssError):
            _lib.call('fss_cross_attention_workspace_bytes', *fn_args)
