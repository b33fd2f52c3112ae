"""fss_quantize_fp8 on and next to the midpoints of e4m3, in every storage type."""
import numpy as np
import pytest
import torch

import fp8_attention_util as U

pytestmark = pytest.mark.gpu

# every midpoint of two neighbouring e4m3 values: normal (3 mantissa bits) and subnormal (steps of 2^-9)
MIDPOINTS = np.array([(8 + k + 0.5) / 8 * 2.0 ** e for e in range(-6, 9) for k in range(8) if (8 + k + 0.5) / 8 * 2.0 ** e < 448] +
                     [(k + 0.5) * 2.0 ** -9 for k in range(8)])
MIDPOINTS = np.concatenate([MIDPOINTS, MIDPOINTS[:-len(MIDPOINTS) % 8]])     # (split-bfloat16 comes in groups of 8)


def near(a, dt):
    """Values of `dt` whose quotient 448 x / a is a midpoint, or the nearest there is, and their neighbours on both
    sides: the floats next to them where the type holds those."""
    x = (MIDPOINTS * a / 448).astype(np.float32)
    out = [U.round_to(x, dt)]
    for steps in (1, 2, 5):
        up, down = x.copy(), x.copy()
        for _ in range(steps):
            up, down = np.nextafter(up, np.float32(np.inf)), np.nextafter(down, np.float32(-np.inf))
        out += [U.round_to(up, dt), U.round_to(down, dt)]
    if dt in ('bf16', 'f16'):
        step = np.maximum(np.abs(x) * 2 * U.HALF[dt], 2.0 ** -24).astype(np.float32)
        out += [U.round_to(x + step, dt), U.round_to(x - step, dt)]
    out = np.concatenate(out)
    return out[np.abs(out) <= a]


@pytest.mark.parametrize('dt', ['f32', 'bf16', 'f16', 'f32x3'])
@pytest.mark.parametrize('block_rows', [1, 128])
def test_quantize_next_to_midpoints(dt, block_rows):
    r = np.random.default_rng(11)
    tops = np.concatenate([[448.0, 7.0, 3.5, 28.0], np.exp(r.uniform(-4, 8, 44))])
    ties, seen = 0, 0
    rows_of = []
    for top in tops:
        a = U.round_to(np.array([top] * 8), dt)[0]
        x = near(a, dt)
        x = np.concatenate([x, -x])
        x = np.concatenate([x, np.zeros(-len(x) % 120, np.float32)]).reshape(-1, 120)
        rows = np.zeros((x.shape[0], 128), np.float32)
        rows[:, :120], rows[:, 127] = x, a
        quotient = rows.astype(np.float64) * 448 / float(a)
        ties += int(np.isin(np.abs(quotient), MIDPOINTS).sum())
        seen += int((np.abs(quotient) > 0).sum())
        rows_of.append(rows)
    # the powers of two times 7 among the maxima make every one of their midpoints a tie
    assert ties >= 4 * 100 and seen > 10000
    if block_rows == 1:
        rows_of = [np.concatenate(rows_of)]
    for rows in rows_of:
        stored, value = U.store(rows, dt, 128)
        assert np.array_equal(value, rows)
        q, _, _ = U.quantize(stored, rows.shape[0], 128, block_rows, dt)
        want = U.quantize_ref(value, block_rows)[0]
        bad = q != want
        assert not bad.any(), (int(bad.sum()), [(float(v).hex(), float(rows[i, 127]).hex(), float(g), float(w)) for i, j in
                                               np.argwhere(bad)[:4] for v, g, w in [(rows[i, j], q[i, j], want[i, j])]])


@pytest.mark.parametrize('a,x,want', [('0x1.9579p+0', '0x1.6a0778p-4', 26.0), ('0x1.461bp+0', '0x1.8bfc38p-2', 144.0),
                                      ('0x1.94298p+0', '0x1.4bfd84p-1', 176.0)])
def test_quantize_split_values_with_a_gap(a, x, want):
    """Split-bfloat16 values whose parts leave a gap: 24 significant bits, next to a midpoint."""
    a, x = np.float32(float.fromhex(a)), np.float32(float.fromhex(x))
    rows = np.zeros((1, 128), np.float32)
    rows[0, 0], rows[0, 1], rows[0, 2] = x, -x, a
    stored, value = U.store(rows, 'f32x3', 128)
    assert np.array_equal(value, rows)
    for block_rows in (1, 128):
        q, _, _ = U.quantize(stored, 1, 128, block_rows, 'f32x3')
        assert q[0, 0] == want and q[0, 1] == -want and U.quantize_ref(value, 1)[0][0, 0] == want
