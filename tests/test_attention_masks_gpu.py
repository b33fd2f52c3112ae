"""fss_cross_attention: ends of masks inside a tile, non-finite values behind a mask, and what those cost."""
import pytest
import torch

import fp8_attention_util as U
from test_attention_gpu import tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('lq', [3, 40])
@pytest.mark.parametrize('stride', [140, 141, 150])
def test_attention_every_length(lq, stride):
    """Lengths from 0 to 140 in one batch: the masks say 'seen' behind each, where keys and values are NaN."""
    b, lk, d = 141, 140, 16
    q, k, v = tensors(b, lq, lk, 2, 1, d, 'f16', seed=lq)
    lens = torch.arange(b, dtype=torch.int32, device='cuda')
    behind = torch.arange(lk, device='cuda')[None, :] >= lens[:, None]
    k[behind], v[behind] = float('nan'), float('nan')
    mask = (torch.rand(b, 2, lq, stride, generator=torch.Generator().manual_seed(1)) < 0.5).cuda()[..., :lk]
    mask |= behind[:, None, None]
    y = U.attend(q, k, v, 'f16', lens=lens, mask=mask)
    U.check_attention(y, U.attention_ref(q, k, v, lens=lens, mask=mask), 'f16', d, lk)


@pytest.mark.parametrize('lk', list(range(1, 36)) + [63, 64, 65])
def test_attention_every_short_mask(lk):
    """Masks that end with their memory: the last byte of the last row is the tensor's last."""
    for lq, d in ((1, 8), (33, 72)):
        q, k, v = tensors(1, lq, lk, 1, 1, d, 'bf16', seed=lk)
        mask = (torch.rand(1, 1, lq, lk, generator=torch.Generator().manual_seed(lk)) < 0.6).cuda()
        U.check_attention(U.attend(q, k, v, 'bf16', mask=mask), U.attention_ref(q, k, v, mask=mask), 'bf16', d, lk)


@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('lq,lk,hq,hk,d', [(5, 90, 2, 2, 8), (5, 1500, 2, 1, 32), (70, 1500, 4, 2, 64), (300, 130, 2, 2, 128),
                                          (1, 2000, 3, 1, 200), (140, 1100, 2, 2, 256), (2, 64, 1, 1, 136)])
def test_attention_hidden_values_differ_by_query(lq, lk, hq, hk, d, dt):
    """Every query is barred from some keys whose values are infinite or NaN, another set for each; some see none of the
    rest either.  Large scores and negative scales take the same path."""
    for scale in (None, -0.2, 4.0):
        q, k, v = tensors(1, lq, lk, hq, hk, d, dt, seed=lq + lk)
        g = torch.Generator().manual_seed(d)
        bad = torch.rand(lk, generator=g) < 0.1
        v[:, bad.cuda(), :, ::3] = float('inf')
        v[:, bad.cuda(), :, 1::3] = float('nan')
        mask = (torch.rand(1, hq, lq, lk, generator=g) < 0.7) & ~bad
        mask[:, :, ::4] = False
        mask = mask.cuda()
        y = U.attend(q, k, v, dt, scale=scale, mask=mask)
        U.check_attention(y, U.attention_ref(q, k, v, scale=scale, mask=mask), dt, d, lk)
        assert (y[:, ::4] == 0).all()
        # a query that sees one of them carries it
        j = int(torch.nonzero(bad)[0]) if bad.any() else None
        if j is not None and scale is None and lq > 1:
            mask[:, :, 1, j] = True
            y = U.attend(q, k, v, dt, mask=mask)
            top = 65504.0 if dt == 'f16' else float('inf')           # half precision saturates
            assert torch.isnan(y[:, 1, :, 1::3]).all() and (y[:, 1, :, ::3] == top).all()
            assert torch.isfinite(y[:, 1, :, 2::3]).all()


def test_attention_scores_of_minus_infinity():
    for lq in (2, 150):
        for masked in (False, True):
            q, k, v = tensors(1, lq, 300, 2, 2, 64, 'bf16', seed=2)
            q[..., 0] = 1.0
            k[:, :, 1, 0] = float('-inf')                # every score of head 1
            k[:, 17, 0, 0] = float('-inf')               # one of head 0
            mask = torch.ones(1, 2, lq, 300, dtype=torch.bool, device='cuda') if masked else None
            y = U.attend(q, k, v, 'bf16', mask=mask)
            assert (y[:, :, 1] == 0).all()
            seen = torch.ones(1, 1, lq, 300, dtype=torch.bool, device='cuda')
            seen[..., 17] = False
            ref = U.attention_ref(q[:, :, :1], k[:, :, :1], v[:, :, :1], mask=seen)
            U.check_attention(y[:, :, :1], ref, 'bf16', 64, 300)


def test_attention_nan_queries_cost_nothing():
    """A NaN in a query, or in a key that it sees, makes all of its result NaN: no second pass over the keys, which would
    take some hundred times as long."""
    q, k, v = tensors(1, 512, 8000, 8, 8, 64, 'bf16', seed=1)
    mask = torch.ones(1, 1, 1, 8000, dtype=torch.bool, device='cuda').expand(1, 8, 512, 8000)
    times = []
    for nan in (False, True):
        if nan:
            q[:] = float('nan')
        y = U.attend(q, k, v, 'bf16', mask=mask)
        assert torch.isnan(y).all() if nan else torch.isfinite(y).all()
        best = float('inf')
        for _ in range(5):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            U.attend(q, k, v, 'bf16', mask=mask, y=y)
            end.record()
            end.synchronize()
            best = min(best, start.elapsed_time(end))
        times.append(best)
    assert times[1] < 10 * times[0], times
