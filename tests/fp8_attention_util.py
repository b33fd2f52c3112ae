"""Callers of fss_quantize_fp8, fss_matmul_fp8 and fss_cross_attention for the tests (numpy in, numpy
out), and the plain 64-bit forms they are held to."""
import ctypes

import numpy as np
import torch

from fss import _lib
from fss.plan import split_bf16_decode, split_bf16_encode

TORCH = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16, 'f32x3': torch.float32}
CODE = {'f32': _lib.F32, 'bf16': _lib.BF16, 'f16': _lib.F16, 'f32x3': _lib.F32_BF16X3}
# half a step of the type, relative to the value
HALF = {'f32': 2.0 ** -24, 'bf16': 2.0 ** -8, 'f16': 2.0 ** -11}
# split-bfloat16: hi leaves a remainder of at most 2^-8 |v|, which lo holds to 2^-8 of itself
HALF['f32x3'] = 2.0 ** -16


def stream():
    return torch.cuda.current_stream().cuda_stream


def features(rows, cols, seed):
    r = np.random.default_rng(seed)
    return (r.standard_normal((rows, cols)) * np.exp(0.7 * r.standard_normal((1, cols)))).astype(np.float32)


def round_to(a, dt):
    """float array -> the nearest values of `dt`, as float32."""
    a = np.asarray(a, np.float32)
    if dt == 'f32x3':
        return split_bf16_decode(split_bf16_encode(a.reshape(-1, 8))).reshape(a.shape)
    return torch.from_numpy(a).to(TORCH[dt]).float().numpy()


def store(x, dt, ld):
    """[rows][cols] -> (device tensor [rows][ld] of `dt`, the values it holds as float32)."""
    rows, cols = x.shape
    wide = np.full((rows, ld), 777.0, np.float32)
    wide[:, :cols] = x
    if dt == 'f32x3':
        return torch.from_numpy(split_bf16_encode(wide)).cuda(), round_to(x, dt)
    return torch.from_numpy(wide).to(TORCH[dt]).cuda(), round_to(x, dt)


# ------------------------------------------------------------------------------------- quantize
def quantize(stored, rows, cols, block_rows, dt, q_pad=0, scale_pad=0):
    """-> (values float32 [rows][cols], scales [column blocks][row blocks], raw bytes [rows][cols + q_pad])"""
    blocks = -(-rows // block_rows)
    q = torch.full((rows, cols + q_pad), 0x55, dtype=torch.uint8, device='cuda')
    scales = torch.full((-(-cols // 128), blocks + scale_pad), -77.0, device='cuda')
    _lib.call('fss_quantize_fp8', stored.data_ptr(), stored.shape[1], q.data_ptr(), cols + q_pad, scales.data_ptr(),
              blocks + scale_pad, rows, cols, block_rows, CODE[dt], stream())
    torch.cuda.synchronize()
    assert (scales[:, blocks:] == -77.0).all()
    return (q[:, :cols].contiguous().view(torch.float8_e4m3fn).float().cpu().numpy(),
            scales[:, :blocks].cpu().numpy(), q.cpu().numpy())


def blocks_of(x, block_rows):
    rows, cols = x.shape
    p = np.zeros((-(-rows // block_rows) * block_rows, -(-cols // 128) * 128), x.dtype)
    p[:rows, :cols] = x
    return p.reshape(-1, block_rows, p.shape[1] // 128, 128)


def e4m3(v):
    """float array -> nearest e4m3 values (ties to even) as float32; NaN stays."""
    v = np.asarray(v, np.float64)
    with np.errstate(invalid='ignore'):
        e = np.maximum(np.frexp(v)[1] - 1, -6)
    step = np.exp2(e.astype(np.float64) - 3)
    return np.clip(np.rint(v / step) * step, -448, 448).astype(np.float32)


def quantize_ref(x, block_rows):
    """(values [rows][cols], scales [column blocks][row blocks]); the quotient 448 x / a of two floats is off a
    midpoint of e4m3 by 2^-29 at least or not at all, so 64 bits round it as the exact one."""
    rows, cols = x.shape
    b = blocks_of(x.astype(np.float32), block_rows)
    with np.errstate(all='ignore'):
        amax = np.maximum(np.abs(b).max(axis=(1, 3)), np.float32(2.0 ** -100))
        amax[~np.isfinite(amax)] = np.nan
        scales = amax / np.float32(448)
        q = e4m3(b.astype(np.float64) * 448.0 / amax.astype(np.float64)[:, None, :, None])
    return q.reshape(-1, b.shape[2] * 128)[:rows, :cols], np.ascontiguousarray(scales.T)


def spread(scales, block_rows, rows, cols):
    s = np.repeat(np.repeat(scales.T, block_rows, 0)[:rows], 128, 1)
    return s[:, :cols].astype(np.float64)


# --------------------------------------------------------------------------------------- matmul
def operands(rows, cout, k, seed):
    r = np.random.default_rng(seed)
    x, xs = quantize_ref(features(rows, k, seed), 1)
    w, ws = quantize_ref((r.standard_normal((cout, k)) / np.sqrt(k)).astype(np.float32), 128)
    return x, xs, w, ws


def matmul_desc(rows, cout, k, dt, **over):
    d = dict(rows=rows, cout=cout, k=k, x_ld=k, x_scale_ld=rows, w_ld=k, w_scale_ld=-(-cout // 128), res_ld=cout,
             y_ld=cout, act=0, out_dtype=CODE[dt])
    d.update(over)
    return _lib.MatmulFp8Desc(**d)


def _bytes(v, ld):
    """e4m3 values -> device bytes [rows][ld]; what lies behind the columns is NaN."""
    b = torch.full((v.shape[0], ld), 0x7f, dtype=torch.uint8)
    b[:, :v.shape[1]] = torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8)
    return b.cuda()


def _padded(a, ld):
    t = torch.full((a.shape[0], ld), float('nan'))
    t[:, :a.shape[1]] = torch.from_numpy(np.ascontiguousarray(a))
    return t.cuda()


def matmul(x, xs, w, ws, dt, act=None, bias=None, residual=None, y_pad=0, x_pad=0, w_pad=0, scale_pad=0, offset=0):
    """e4m3 values and scales -> y [rows][cout] as float32; checks that nothing else was written.
    offset: elements by which y and the residual start behind an aligned address."""
    (rows, k), cout = x.shape, w.shape[0]
    xd, wd = _bytes(x, k + x_pad), _bytes(w, k + w_pad)
    xsd, wsd = _padded(xs, xs.shape[1] + scale_pad), _padded(ws, ws.shape[1] + scale_pad)
    ld = cout + y_pad
    flat = torch.full((rows * ld + offset,), -77.0, dtype=TORCH[dt], device='cuda')
    y = flat[offset:].view(rows, ld)
    res = None
    if residual is not None:
        res_flat = torch.zeros(rows * ld + offset, dtype=TORCH[dt], device='cuda')
        res = res_flat[offset:].view(rows, ld)
        res.copy_(store(residual, dt, ld)[0])
    bd = None if bias is None else torch.from_numpy(bias).cuda()
    d = matmul_desc(rows, cout, k, dt, x_ld=k + x_pad, w_ld=k + w_pad, x_scale_ld=xsd.shape[1], w_scale_ld=wsd.shape[1],
                    y_ld=ld, res_ld=ld, act=_lib.ACT_CODES[act])
    size = ctypes.c_size_t()
    _lib.call('fss_matmul_fp8_workspace_bytes', ctypes.byref(d), ctypes.byref(size))
    ws_buf = torch.full((size.value + 256,), 0xff, dtype=torch.uint8, device='cuda')
    _lib.call('fss_matmul_fp8', ctypes.byref(d), xd.data_ptr(), xsd.data_ptr(), wd.data_ptr(), wsd.data_ptr(),
              None if bd is None else bd.data_ptr(), None if res is None else res.data_ptr(), y.data_ptr(),
              ws_buf.data_ptr() if size.value else None, size.value, stream())
    torch.cuda.synchronize()
    assert (ws_buf[size.value:] == 0xff).all(), 'wrote behind the workspace'
    assert (flat[:offset] == -77.0).all() and (y[:, cout:] == -77.0).all(), 'wrote outside y'
    if dt == 'f32x3':
        return split_bf16_decode(y.cpu().numpy())[:, :cout]
    return y[:, :cout].float().cpu().numpy()


def check_matmul(rows, cout, k, dt, act, bias, residual, **how):
    r = np.random.default_rng(rows + 7 * cout + 13 * k)
    x, xs, w, ws = operands(rows, cout, k, seed=rows * 31 + k)
    bv = r.standard_normal(cout).astype(np.float32) if bias else None
    rv = round_to(r.standard_normal((rows, cout)), dt) if residual else None
    got = matmul(x, xs, w, ws, dt, act, bv, rv, **how)
    xd = x.astype(np.float64) * spread(xs, 1, rows, k)
    wd = w.astype(np.float64) * spread(ws, 128, cout, k)
    want, size = xd @ wd.T, np.abs(xd) @ np.abs(wd).T
    if bias:
        want, size = want + bv, size + np.abs(bv)
    if residual:
        want, size = want + rv, size + np.abs(rv)
    # float sums: 128 products per block, then the blocks one by one, scale, bias, residual: each of
    # at most 128 + k / 128 + 4 additions or products loses half a step of a partial sum (a step where
    # the matrix core truncates), and no partial sum is above `size`
    tol = size * 2 * 2.0 ** -24 * (128 + k / 128 + 4)
    if dt in ('bf16', 'f16'):
        # the 8-bit matrix instructions align 8 products to the largest, of exponent e (at least a
        # quarter of 2^(e + 2)), and drop what lies below 2^(e - 13): each of the 7 others loses less than
        # 2^-13 of the largest, and the largest products of all groups together are at most `size`
        tol += size * 7 * 2.0 ** -13
    tol += np.abs(want) * HALF[dt] + (2.0 ** -25 if dt == 'f16' else 0)       # the one rounding; f16 below 2^-14
    if act:
        want = np.clip(want, 0, 6 if act == 'relu6' else np.inf)
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.abs(got - want).max()))


# ------------------------------------------------------------------------------------ attention
def attention_desc(batch, q_len, kv_len, q_heads, kv_heads, head_dim, dt, scale=None, **over):
    three = ctypes.c_int64 * 3
    d = dict(batch=batch, q_len=q_len, kv_len=kv_len, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, dtype=CODE[dt],
             scale=max(head_dim, 1) ** -0.5 if scale is None else scale,
             q_stride=(q_len * q_heads * head_dim, q_heads * head_dim, head_dim),
             k_stride=(kv_len * kv_heads * head_dim, kv_heads * head_dim, head_dim),
             v_stride=(kv_len * kv_heads * head_dim, kv_heads * head_dim, head_dim),
             y_stride=(q_len * q_heads * head_dim, q_heads * head_dim, head_dim), mask_stride=(0, 0, 0))
    d.update(over)
    return _lib.AttentionDesc(**{n: three(*v) if n.endswith('_stride') else v for n, v in d.items()})


def attend(q, k, v, dt, scale=None, lens=None, mask=None, y=None):
    """Device tensors [batch][tokens][heads][dim] of any strides, mask bool / uint8 [batch][heads][q][kv] of
    any strides (last 1) -> y, a device tensor."""
    b, lq, hq, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    if y is None:
        y = torch.full((b, lq, hq, d), -77.0, dtype=TORCH[dt], device='cuda')
    desc = attention_desc(b, lq, lk, hq, hk, d, dt, scale, q_stride=q.stride()[:3], k_stride=k.stride()[:3],
                          v_stride=v.stride()[:3], y_stride=y.stride()[:3],
                          mask_stride=(0, 0, 0) if mask is None else (mask.stride(0), mask.stride(2), mask.stride(1)))
    size = ctypes.c_size_t()
    _lib.call('fss_cross_attention_workspace_bytes', ctypes.byref(desc), ctypes.byref(size))
    ws = torch.full((size.value + 256,), 0xff, dtype=torch.uint8, device='cuda')
    _lib.call('fss_cross_attention', ctypes.byref(desc), q.data_ptr(), k.data_ptr(), v.data_ptr(),
              None if lens is None else lens.data_ptr(), None if mask is None else mask.data_ptr(), y.data_ptr(),
              ws.data_ptr() if size.value else None, size.value, stream())
    torch.cuda.synchronize()
    assert (ws[size.value:] == 0xff).all(), 'wrote behind the workspace'
    return y


def attention_ref(q, k, v, scale=None, lens=None, mask=None):
    """64-bit, on the CPU; keys that a query does not see are left out whatever they hold.  -> (y, bound)
    with bound = sum_j w_j |v_j|, the scale of the sums, and `top` = largest |scale q.k| per query."""
    q, k, v = (t.detach().cpu().double().numpy() for t in (q, k, v))
    b, lq, hq, d = q.shape
    lk, g = k.shape[1], hq // k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    y, size, top = np.zeros((b, lq, hq, d)), np.zeros((b, lq, hq, d)), np.zeros((b, lq, hq, 1))
    for i in range(b):
        n = lk if lens is None else min(max(int(lens[i]), 0), lk)
        for h in range(hq):
            kk, vv = k[i, :n, h // g], v[i, :n, h // g]
            seen = np.ones((lq, n), bool) if mask is None else mask[i, h, :, :n].cpu().numpy() != 0
            used = seen.any(0)
            kk, vv, seen = kk[used], vv[used], seen[:, used]
            if kk.shape[0] == 0:
                continue
            s = (q[i, :, h] @ kk.T) * scale
            reach = (np.abs(q[i, :, h]) @ np.abs(kk).T) * abs(scale)
            s = np.where(seen, s, -np.inf)
            m = s.max(1, keepdims=True)
            p = np.where(seen, np.exp(s - np.where(np.isfinite(m), m, 0)), 0.0)
            w = p / np.maximum(p.sum(1, keepdims=True), 1e-300)
            if np.isfinite(vv).all():
                y[i, :, h], size[i, :, h] = w @ vv, w @ np.abs(vv)
            else:
                for j in range(lq):
                    y[i, j, h] = w[j, seen[j]] @ vv[seen[j]]
                    size[i, j, h] = w[j, seen[j]] @ np.abs(vv[seen[j]])
            top[i, :, h, 0] = np.where(seen, reach, 0).max(1)
    return y, size, top


def check_attention(got, ref, dt, head_dim, keys):
    y, size, top = ref
    got = got.detach().float().cpu().numpy()
    assert np.isfinite(got).all()
    # p: a float score of head_dim products (a step of the partial sum each), times scale and log2 e, an
    # exponential of 2 steps; then rounded to dt for the product with v; sums over the keys in float
    # (at most one step per addition); one rounding of the result.  Errors of p enter the
    # numerator relative to sum w |v|, those of the sum relative to |y| <= sum w |v|.
    u = 2.0 ** -24
    score = top * (2 * u * (head_dim + 3)) + 4 * u
    tol = size * (HALF[dt] + 2 * score + 4 * u * (keys + 8)) + np.abs(y) * HALF[dt] + 2.0 ** -25
    bad = ~(np.abs(got - y) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.abs(got - y).max()))
