"""fss_cross_attention where the scores are far from zero.  Scores are exact in float here: few channels, powers of two."""
import numpy as np
import pytest
import torch

import fp8_attention_util as U

pytestmark = pytest.mark.gpu

# (queries, keys): single wave, its key axis whole and in pieces; four waves whole and in pieces
SIZES = [(2, 60), (3, 1500), (150, 260), (100, 2100)]


def plane(lq, lk, heads, d, dt, seed):
    g = torch.Generator().manual_seed(seed)
    v = torch.randn(1, lk, heads, d, generator=g).to(U.TORCH[dt]).cuda()
    return torch.zeros(1, lq, heads, d, dtype=U.TORCH[dt], device='cuda'), torch.zeros_like(v), v


@pytest.mark.parametrize('lq,lk', SIZES)
@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('dt,power', [('f16', 8), ('f16', 15), ('f16', 20), ('f16', 21), ('f16', 22), ('bf16', 12), ('bf16', 23),
                                      ('bf16', 40), ('bf16', 81), ('bf16', 119)])
def test_attention_far_scores(lq, lk, masked, dt, power):
    """Scores that are whole multiples of 2^power, at most 255 of them: everything but the largest has
    exp(score - largest) below 2^-300, so that a query's result is exactly the value of its best key."""
    heads, d = 2, 32
    q, k, v = plane(lq, lk, heads, d, dt, seed=power)
    r = np.random.default_rng(lq + lk + power)
    a = torch.from_numpy(r.integers(-255, 255, (1, lk, heads)).astype(np.float32)).cuda()
    best = int(r.integers(0, lk))
    a[:, best] = 255.0 if power % 2 else -1.0                # the largest may be negative
    if power % 2 == 0:
        a = torch.where((a < 0) & (torch.arange(lk, device='cuda') != best)[None, :, None], a - 1, -a.abs() - 2)
        a[:, best] = -1.0
    else:
        a[:, :best].clamp_(max=254)
        a[:, best + 1:].clamp_(max=254)
    k_power = min(power // 2, 7) if dt == 'f16' else power // 2
    k[..., 5] = a * 2.0 ** k_power
    q[..., 5] = 2.0 ** (power - k_power)
    assert torch.isfinite(q).all() and torch.equal(k[..., 5].float(), a * 2.0 ** k_power)
    mask = None
    if masked:
        mask = (torch.rand(1, heads, lq, lk, generator=torch.Generator().manual_seed(1)) < 0.5).cuda()
        mask[..., best] = True
    y = U.attend(q, k, v, dt, scale=1.0, mask=mask)
    assert torch.equal(y, v[:, best:best + 1].expand_as(y))


@pytest.mark.parametrize('lq,lk', SIZES)
@pytest.mark.parametrize('dt,offset', [(dt, s * o) for dt in ('f16', 'bf16') for s in (1, -1) for o in (64, 128, 256, 4096, 2 ** 16)])
def test_attention_offset_scores(lq, lk, dt, offset):
    """scores = offset + t with t in [-12, 0] in steps of 2^-4, exact in float: the softmax of t, whatever the
    offset."""
    heads, d = 2, 32
    q, k, v = plane(lq, lk, heads, d, dt, seed=abs(offset))
    r = np.random.default_rng(lq * lk)
    t = torch.from_numpy(-r.integers(0, 12 * 16 + 1, (1, lk, heads)).astype(np.float32) / 16).cuda()
    q[..., 0], k[..., 0] = 32.0, offset / 32.0
    q[..., 1], k[..., 1] = 1.0, t
    assert torch.equal(k[..., 1].float(), t)
    y = U.attend(q, k, v, dt, scale=1.0).double().cpu()
    w = torch.softmax(t.double().cpu(), 1)[..., None]
    want, size = (w * v.double().cpu()).sum(1), (w * v.double().cpu().abs()).sum(1)
    # p: its exponent, up to 12 log2(e), with two roundings, its base off by 2^-24 of at most 256 (farther
    # bases are exact), once in p and once between parts of the sum; an exponential of two steps; the
    # rounding to dt; sums over the keys; the result's rounding
    u = 2.0 ** -24
    p = 18 * 2 * u + 2 * 2.0 ** -16 + 4 * u
    tol = size * (U.HALF[dt] + 2 * p + 4 * u * (lk + 8)) + want.abs() * U.HALF[dt] + 2.0 ** -25
    bad = (y[0] - want[0]).abs() > tol[0]
    assert not bad.any(), (int(bad.sum()), float((y[0] - want[0]).abs().max()))


@pytest.mark.parametrize('lq', [3, 150, 66000])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('masked', [False, True])
def test_attention_many_weak_keys(lq, dt, masked):
    """One strong key, of value 0, above 33151 weak ones whose p are below half precision's subnormal numbers: they alone
    are the result."""
    if masked and lq > 1000:
        lq = 16500
    lk, d, strong = 33152, 8, 5
    q, k, v = plane(lq, lk, 1 if not masked else 4, d, dt, seed=0)
    heads = k.shape[2]
    q[..., 0] = 1.0
    for t in (-10.0, -14.0, -17.5, -20.0, -23.0):
        k[..., 0] = t
        v[:] = 1000.0
        k[:, strong, :, 0], v[:, strong] = 0.0, 0.0
        mask = torch.ones(1, 1, 1, lk, dtype=torch.bool, device='cuda').expand(1, heads, lq, lk) if masked else None
        y = U.attend(q, k, v, dt, scale=1.0, mask=mask).double()
        weak = (lk - 1) * np.exp(t)
        want = 1000 * weak / (1 + weak)
        # p: an exponent of up to 34 with two roundings, its base (2^-16, see above), an exponential of two steps, its
        # rounding to dt; the sum of the p takes two halves of the keys pair by pair, half a step each at
        # most; the output 16 keys at a time, a step each; its rounding
        u = 2.0 ** -24
        tol = want * (U.HALF[dt] + 2 * (34 * 2 * u + 2.0 ** -16 + 4 * u) + lk / 4 * u + lk / 16 * 2 * u + U.HALF[dt])
        if dt == 'f16':
            # Half precision has steps of 2^-24 below 2^-14, of 2^-39 of the largest p below 2^-29 of it as p is
            # carried: half a step for each weak key, at -23 (2^-33.2) 3.0e-5 in all for a result of 3.4e-3
            tol += 1000 * (lk - 1) * 2.0 ** -40
        assert float((y - want).abs().max()) <= tol, (t, float((y - want).abs().max()), tol)
