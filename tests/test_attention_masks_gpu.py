"""fss_cross_attention: ends of masks inside a tile."""
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
