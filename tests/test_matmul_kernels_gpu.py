"""Every kernel fss_matmul_fp8 chooses from, held to the exact result: e4m3 integers and scales that are powers of
two, whose products and sums are exact in any order, so that what is left is the one rounding of the output."""
import ctypes
import re

import numpy as np
import pytest
import torch

from fss import _lib
from fss.plan import split_bf16_decode, split_bf16_encode
import fp8_attention_util as U

pytestmark = pytest.mark.gpu

FEW, SPLIT, T64, T64K, T128, T256 = 'few', 'split', (64, 64, 2, 2, 1), (64, 64, 2, 2, 2), (128, 128, 2, 2, 1), (256, 256, 2, 4, 1)
# kernel, rows, channels (whole 16-byte pieces, then not), k
SIZES = [(FEW, 1, 512, 2048), (FEW, 5, 43, 176), (FEW, 33, 136, 272), (FEW, 1300, 19, 272),
         (SPLIT, 500, 136, 4240), (SPLIT, 500, 133, 4240), (SPLIT, 128, 128, 16384),
         (T64, 4097, 136, 176), (T64, 4097, 133, 176), (T64, 8385, 304, 1040),
         (T64K, 2145, 512, 2048), (T64K, 2145, 509, 1040),
         (T128, 16500, 1032, 144), (T128, 16500, 1029, 144),
         (T256, 4093, 4088, 1040), (T256, 4093, 4090, 1040)]
IDS = ['%s-%dx%d-%d' % ('x'.join(map(str, s[0])) if isinstance(s[0], tuple) else s[0], *s[1:]) for s in SIZES]
ACTS = {None: (-float('inf'), float('inf')), 'relu': (0.0, float('inf')), 'relu6': (0.0, 6.0)}
DTS = ['f32', 'bf16', 'f16', 'f32x3']


class Product:
    """Operands in padded buffers: NaN behind the columns, the scales and the channels."""

    def __init__(self, rows, cout, k, seed=0, x_pad=0, w_pad=0, scale_pad=0):
        g = torch.Generator(device='cuda').manual_seed(seed + rows + 7 * cout + 31 * k)
        ints = lambda top, *s: torch.randint(-top, top + 1, s, generator=g, device='cuda').float()
        two = lambda lo, hi, *s: torch.exp2(torch.randint(lo, hi + 1, s, generator=g, device='cuda').float())
        kb, nb = -(-k // 128), -(-cout // 128)
        self.sizes = rows, cout, k
        self.xv, self.wv = ints(3, rows, k), ints(2, cout, k)
        self.xsv, self.wsv = two(-2, 1, kb, rows), two(-1, 1, kb, nb)
        self.bias, self.residual = ints(30, cout) / 4, ints(30, rows, cout) / 4
        self.x, self.w = (self._padded(v.to(torch.float8_e4m3fn).view(torch.uint8), p, 0x7f)
                          for v, p in ((self.xv, x_pad), (self.wv, w_pad)))
        self.xs, self.ws = (self._padded(v, scale_pad, float('nan')) for v in (self.xsv, self.wsv))

    @staticmethod
    def _padded(v, pad, fill):
        t = torch.full((v.shape[0], v.shape[1] + pad), fill, dtype=v.dtype, device='cuda')
        t[:, :v.shape[1]] = v
        return t

    def desc(self, dt, act=None, **over):
        rows, cout, k = self.sizes
        return U.matmul_desc(rows, cout, k, dt, **dict(dict(x_ld=self.x.shape[1], w_ld=self.w.shape[1],
                                                             x_scale_ld=self.xs.shape[1], w_scale_ld=self.ws.shape[1],
                                                             act=_lib.ACT_CODES[act]), **over))

    def run(self, dt, act=None, bias=False, residual=False, y_pad=0, offset=0):
        """-> y as the call left it, in a buffer whose other elements are checked."""
        rows, cout, _ = self.sizes
        ld = cout + y_pad
        flat = torch.full((rows * ld + offset,), -77.0, dtype=U.TORCH[dt], device='cuda')
        y = flat[offset:].view(rows, ld)
        res = torch.zeros_like(flat)
        res_view = res[offset:].view(rows, ld)
        if dt == 'f32x3':
            wide = torch.zeros(rows, ld)
            wide[:, :cout] = self.residual.cpu()
            res_view.copy_(torch.from_numpy(split_bf16_encode(wide.numpy())))
        else:
            res_view[:, :cout] = self.residual.to(U.TORCH[dt])
        d = self.desc(dt, act, y_ld=ld, res_ld=ld)
        size = ctypes.c_size_t()
        _lib.call('fss_matmul_fp8_workspace_bytes', ctypes.byref(d), ctypes.byref(size))
        buf = torch.full((size.value + 256,), 0xff, dtype=torch.uint8, device='cuda')
        _lib.call('fss_matmul_fp8', ctypes.byref(d), self.x.data_ptr(), self.xs.data_ptr(), self.w.data_ptr(), self.ws.data_ptr(),
                  self.bias.data_ptr() if bias else None, res_view.data_ptr() if residual else None, y.data_ptr(),
                  buf.data_ptr() if size.value else None, size.value, U.stream())
        torch.cuda.synchronize()
        assert (buf[size.value:] == 0xff).all(), 'wrote behind the workspace'
        assert (flat[:offset] == -77.0).all() and (y[:, cout:] == -77.0).all(), 'wrote outside y'
        if dt == 'f32x3':
            return torch.from_numpy(split_bf16_decode(y.cpu().numpy())[:, :cout]).cuda()
        return y[:, :cout]

    def want(self, dt, act=None, bias=False, residual=False):
        rows, cout, k = self.sizes
        x = self.xv * self.xsv.t().repeat_interleave(128, 1)[:, :k]
        w = self.wv * self.wsv.t().repeat_interleave(128, 0)[:cout].repeat_interleave(128, 1)[:, :k]
        y = torch.mm(x.double(), w.double().t().contiguous())
        if bias:
            y += self.bias
        if residual:
            y += self.residual
        # every partial sum is a multiple of 2^-3 below 2^21: exact in a float
        assert float(y.abs().max()) < 2.0 ** 20
        y = y.clamp(*ACTS[act]).float()
        if dt == 'f32x3':
            return torch.from_numpy(U.round_to(y.cpu().numpy(), dt)).cuda()
        return y.to(U.TORCH[dt])

    def check(self, dt, y_pad=0, offset=0, **how):
        got, want = self.run(dt, y_pad=y_pad, offset=offset, **how), self.want(dt, **how)
        if not torch.equal(got, want):
            bad = got != want
            at = torch.nonzero(bad)[:4].tolist()
            raise AssertionError((int(bad.sum()), at, [(float(got[i, j]), float(want[i, j])) for i, j in at]))


def types_of(cout):
    return [dt for dt in DTS if dt != 'f32x3' or cout % 8 == 0]


@pytest.mark.parametrize('kernel,rows,cout,k', SIZES, ids=IDS)
def test_matmul_is_exact(kernel, rows, cout, k):
    p = Product(rows, cout, k)
    for dt in types_of(cout):
        p.check(dt)
        p.check(dt, bias=True, residual=True)
        p.check(dt, act='relu6' if dt == 'f16' else 'relu', bias=True)


@pytest.mark.parametrize('kernel,rows,cout,k', SIZES, ids=IDS)
def test_matmul_strides_are_exact(kernel, rows, cout, k):
    """NaN behind the columns of both operands and behind their scales; y and the residual in wider rows, at
    addresses that allow whole pieces and at others."""
    p = Product(rows, cout, k, seed=1, x_pad=48, w_pad=16, scale_pad=3)
    for dt in types_of(cout):
        if dt != 'f32x3':
            p.check(dt, y_pad=3, offset=1, bias=True, residual=True)
        p.check(dt, y_pad=-cout % 8 + 8, offset=16, bias=True, residual=True)
        p.check(dt, y_pad=8)


@pytest.mark.parametrize('kernel,rows,cout,k', [s for s in SIZES if s[1] > 100], ids=[i for i, s in zip(IDS, SIZES) if s[1] > 100])
def test_matmul_carries_nan_and_saturates(kernel, rows, cout, k):
    p = Product(rows, cout, k, seed=2)
    block, row = p.xs.shape[0] - 1, rows - 3
    for act in (None, 'relu', 'relu6'):
        p.xs[block, row] = float('nan')
        for dt in types_of(cout):
            y = p.run(dt, act=act)
            assert torch.isnan(y[row]).all() and int(torch.isnan(y).sum()) == cout
    p.xs[block, row] = 2.0 ** 60
    y = p.run('f16')
    assert torch.isfinite(y).all() and float(y[row].abs().max()) == 65504.0
    p.xs[block, row] = 1.0
    p.residual[5] = float('inf')
    y = p.run('f16', residual=True)
    assert (y[5] == 65504.0).all() and torch.isfinite(y).all()
    y = p.run('bf16', residual=True)
    assert (y[5] == float('inf')).all() and torch.isfinite(y[6:]).all()
    # a weight block of NaN: its 128 channels, all rows
    p.ws[0, -1] = float('nan')
    y = p.run('bf16')
    first = (cout - 1) // 128 * 128
    assert torch.isnan(y[:, first:]).all() and not torch.isnan(y[:, :first]).any()


def _kernels(names):
    """[(kernel, its template's numbers)] of this library's launches, from names mangled or not."""
    out = []
    for n in names:
        m = re.search(r'(matmul_fp8_\w+?_kernel)(?:<([^>]*)>|I(.*)E+v)', n)
        if m:
            args = m.group(2)
            numbers = re.findall(r'\b(true|false|\d+)\b', args) if args is not None else re.findall(r'L[bi](\d+)E', m.group(3))
            out.append((m.group(1), tuple({'true': 1, 'false': 0}.get(v, v) if v in ('true', 'false') else int(v) for v in numbers)))
    return out


def test_matmul_kernels_behind_the_sizes():
    """The sizes above reach the kernels they are listed under, in the form for whole 16-byte pieces or the other."""
    from torch.profiler import profile, ProfilerActivity
    calls = [(s, dt, Product(*s[1:])) for s in SIZES for dt in ('bf16', 'f16', 'f32')]
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        for _, dt, p in calls:
            p.run(dt)
    events = [e for e in prof.events() if 'matmul_fp8' in e.name]
    events.sort(key=lambda e: e.time_range.start)
    if not events:
        pytest.skip('the profiler saw no launch')
    got = iter(_kernels([e.name for e in events]))
    for (kernel, rows, cout, k), dt, _ in calls:
        vec = int(cout % 8 == 0)
        if kernel == FEW:
            want = [('matmul_fp8_few_kernel', ())]
        elif kernel == SPLIT:
            want = [('matmul_fp8_tile_kernel', (1, 1) + T64K), ('matmul_fp8_join_kernel', (vec,))]
        else:
            want = [('matmul_fp8_tile_kernel', (vec, 0) + kernel)]
        assert [next(got) for _ in want] == want, (rows, cout, k, dt)
    assert next(got, None) is None
