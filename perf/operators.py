"""Block-scaled 8-bit products and cross attention: the calls a decoder on top of the framework's feature maps makes.

Three operators, used one behind the other: `quantize` (fss_quantize_fp8: a tensor to e4m3 with a float
scale per 128 channels), `matmul` (fss_matmul_fp8: the product of two such tensors with the
convolutions' epilogue) and `attention` (fss_cross_attention: queries against the keys and values of
another, longer or shorter, set of tokens).  `run` computes them in plain torch operations, or, where
`own` is true, through the framework's entry points.

Sizes: 129 x 257 = 33153, 65 x 129 = 8385 and 33 x 65 = 2145 pixels are the 1/8, 1/16 and 1/32 maps of a
1025 x 2049 frame; 50 = 1 + 4 + 9 + 36 tokens are a pyramid of pooled maps with 1, 2, 3 and 6 bins;
100 is a set of object queries, 19 the classes.
"""
import ctypes
import math
import os
import sys

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BLOCK = 128
TINY = 2.0 ** -100           # a block of zeros gets the scale of this largest magnitude
E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------- cases
def _quantize(rows, cols, dtype, block_rows=1, **more):
    return dict(op='quantize', rows=rows, cols=cols, dtype=dtype, block_rows=block_rows, **more)


def _matmul(rows, cout, k, dtype, act='none', bias=True, residual=False, **more):
    return dict(op='matmul', rows=rows, cout=cout, k=k, dtype=dtype, act=act, bias=bias, residual=residual, **more)


def _attention(batch, q_len, kv_len, q_heads, kv_heads, head_dim, dtype, lens=False, mask=False, **more):
    return dict(op='attention', batch=batch, q_len=q_len, kv_len=kv_len, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, dtype=dtype, lens=lens, mask=mask, **more)


def listed():
    return [
        # one token of a decoder that produces its queries one after the other
        _quantize(1, 512, 'bf16', name='quantize one token'),
        # a float weight matrix when a program starts: 128 x 128 blocks
        _quantize(2048, 4096, 'f32', block_rows=128, name='quantize weights'),
        # the 1/8 map of four frames, 2048 channels
        _quantize(4 * 33153, 2048, 'bf16', name='quantize maps of 4 frames'),
        # the projection of that one token
        _matmul(1, 512, 2048, 'bf16', name='matmul one token'),
        # 1/32 map of one frame: few output tiles under a long K, half-precision residual stream
        _matmul(2145, 512, 2048, 'f16', residual=True, name='matmul 1/32 map'),
        # class scores of the 1/16 map: 19 columns, floats
        _matmul(8385, 19, 512, 'f32', name='matmul class scores'),
        # 1/8 map of one frame, the ordinary projection of a wide map to the attention's width
        _matmul(33153, 256, 512, 'bf16', act='relu', name='matmul 1/8 map'),
        # 1/8 maps of four frames, the widest layers
        _matmul(4 * 33153, 2048, 2048, 'bf16', name='matmul maps of 4 frames'),
        # one query token against the 1/32 map
        _attention(1, 1, 2145, 8, 8, 32, 'bf16', name='attend one token'),
        # object queries against the 1/8 map, each inside the region its mask leaves (some leave none)
        _attention(2, 100, 33153, 8, 8, 32, 'f16', mask=True, name='attend masked queries'),
        # every pixel of the 1/8 map against the pooled pyramid's tokens
        _attention(2, 33153, 50, 8, 8, 64, 'bf16', name='attend pyramid'),
        # every pixel of the 1/16 map against another frame's, padded batch, shared key / value heads
        _attention(2, 8385, 8385, 16, 4, 128, 'bf16', lens=True, name='attend frames'),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(['quantize', 'matmul', 'matmul', 'attention', 'attention'])
    if op == 'quantize':
        cols = 16 * _log(rng, 1, 256)
        rows = _log(rng, 1, min(4 * 33153, 4 * 33153 * 2048 // cols))
        return _quantize(rows, cols, rng.choice(['f32', 'bf16', 'f16']), rng.choice([1, 1, 128]))
    if op == 'matmul':
        cout, k = _log(rng, 1, 4096), 16 * _log(rng, 1, 256)
        rows = _log(rng, 1, min(4 * 33153, 4 * 33153 * 2048 * 2048 // (cout * k)))
        return _matmul(rows, cout, k, rng.choice(['f32', 'bf16', 'f16']), rng.choice(['none', 'relu', 'relu6']),
                       rng.random() < 0.7, rng.random() < 0.5)
    head_dim = 8 * rng.randint(1, 32) if rng.random() < 0.4 else rng.choice([32, 64, 128])
    kv_heads, group, batch = rng.randint(1, 8), rng.choice([1, 1, 2, 4, 7]), rng.randint(1, 4)
    most = 15 * 2 * 8385 * 8385                     # scores: just under the largest listed case
    kv_len = _log(rng, 1, 33153)
    q_len = _log(rng, 1, 33153)
    heads = kv_heads * group
    q_len = max(1, min(q_len, most * 128 // (batch * heads * kv_len * max(head_dim, 128))))
    return _attention(batch, q_len, kv_len, heads, kv_heads, head_dim, rng.choice(['bf16', 'f16']),
                      rng.random() < 0.4, rng.random() < 0.3 and q_len * kv_len < 1 << 26)


def _lens(case):
    """Tokens of each batch entry: the first is whole, the others are ever shorter."""
    b = case['batch']
    return [max(1, case['kv_len'] - i * case['kv_len'] // (2 * b) - (i > 0)) for i in range(b)] if case['lens'] \
        else [case['kv_len']] * b


def work(case):
    size = {'f32': 4, 'bf16': 2, 'f16': 2}[case['dtype']]
    if case['op'] == 'quantize':
        n, blocks = case['rows'] * case['cols'], -(-case['rows'] // case['block_rows']) * -(-case['cols'] // BLOCK)
        return {'bytes': n * (size + 1) + 4 * blocks, 'flops': 3 * n}
    if case['op'] == 'matmul':
        m, n, k = case['rows'], case['cout'], case['k']
        kb = -(-k // BLOCK)
        return {'bytes': m * k + n * k + m * n * size * (2 if case['residual'] else 1) + 4 * kb * (m + -(-n // BLOCK)) +
                (4 * n if case['bias'] else 0), 'flops': 2 * m * n * k}
    b, h, d, lq, keys = case['batch'], case['q_heads'], case['head_dim'], case['q_len'], sum(_lens(case))
    return {'bytes': size * d * (2 * b * lq * h + 2 * keys * case['kv_heads']) + (lq * keys if case['mask'] else 0),
            'flops': 4 * h * d * lq * keys}


# ----------------------------------------------------------------------------------------- prepare
def _features(g, rows, cols):
    """What a normalised layer leaves: near-normal values, some channels far louder than others."""
    x = torch.randn(rows, cols, generator=g, device='cuda')
    x *= torch.exp(0.7 * torch.randn(1, cols, generator=g, device='cuda'))
    return x


def _blocks(x, block_rows):
    """[rows][cols] as [row blocks][block rows][column blocks][128], zero filled."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, -rows % block_rows))
    return x.reshape(-1, block_rows, x.shape[1] // BLOCK, BLOCK)


def _to_fp8(x, block_rows):
    """Plain form of the conversion: (e4m3 [rows][cols], float scales [column blocks][row blocks])."""
    rows, cols = x.shape
    xb = _blocks(x.float(), block_rows)
    amax = xb.abs().amax(dim=(1, 3)).clamp_min(TINY)
    q = (xb * (E4M3_MAX / amax)[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.reshape(-1, q.shape[2] * BLOCK)[:rows, :cols].contiguous(), (amax / E4M3_MAX).t().contiguous()


def _spread(scales, block_rows, rows, cols):
    """Scales [column blocks][row blocks] as one value per element."""
    return scales.t().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dt = DTYPES[case['dtype']]
    s = {'case': case}
    if case['op'] == 'quantize':
        s['x'] = _features(g, case['rows'], case['cols']).to(dt)
    elif case['op'] == 'matmul':
        m, n, k = case['rows'], case['cout'], case['k']
        s['x'], s['x_scales'] = _to_fp8(_features(g, m, k), 1)
        s['w'], s['w_scales'] = _to_fp8(torch.randn(n, k, generator=g, device='cuda') / math.sqrt(k), BLOCK)
        s['bias'] = 0.5 * torch.randn(n, generator=g, device='cuda') if case['bias'] else None
        s['residual'] = torch.randn(m, n, generator=g, device='cuda').to(dt) if case['residual'] else None
    else:
        b, lq, lk, d = case['batch'], case['q_len'], case['kv_len'], case['head_dim']
        s['q'] = torch.randn(b, lq, case['q_heads'], d, generator=g, device='cuda').to(dt)
        # keys and values leave one projection side by side
        kv = torch.randn(b, lk, 2, case['kv_heads'], d, generator=g, device='cuda').to(dt)
        s['k'], s['v'] = kv[:, :, 0], kv[:, :, 1]
        s['scale'] = 1.0 / math.sqrt(d)
        s['lens'] = torch.tensor(_lens(case), dtype=torch.int32, device='cuda') if case['lens'] else None
        s['mask'] = None
        if case['mask']:
            # a query may look at a run of keys; one query in eight has an empty region
            at = torch.rand(b, lq, 1, generator=g, device='cuda') * lk
            wide = torch.rand(b, lq, 1, generator=g, device='cuda') * lk * 0.6 + 1
            wide[torch.rand(b, lq, 1, generator=g, device='cuda') < 0.125] = 0
            j = torch.arange(lk, device='cuda')
            s['mask'] = ((j >= at - wide / 2) & (j < at + wide / 2))
    return s


# --------------------------------------------------------------------------------------------- run
def _plain(s):
    case = s['case']
    if case['op'] == 'quantize':
        return _to_fp8(s['x'], case['block_rows'])
    if case['op'] == 'matmul':
        m, n, k = case['rows'], case['cout'], case['k']
        x = s['x'].float() * _spread(s['x_scales'], 1, m, k)
        w = s['w'].float() * _spread(s['w_scales'], BLOCK, n, k)
        y = x @ w.t()
        if s['bias'] is not None:
            y += s['bias']
        if s['residual'] is not None:
            y += s['residual'].float()
        if case['act'] != 'none':
            y = y.clamp(0.0, 6.0 if case['act'] == 'relu6' else math.inf)
        return y.to(DTYPES[case['dtype']])
    b, lq, lk, h, hk, d = (case[n] for n in ('batch', 'q_len', 'kv_len', 'q_heads', 'kv_heads', 'head_dim'))
    q = s['q'].float().reshape(b, lq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, h // hk * lq, d)
    k = s['k'].float().permute(0, 2, 3, 1).contiguous()
    v = s['v'].float().permute(0, 2, 1, 3).contiguous()
    p = (q @ k).mul_(s['scale']).view(b, hk, h // hk, lq, lk)
    if s['lens'] is not None:
        p.masked_fill_((torch.arange(lk, device=p.device) >= s['lens'][:, None])[:, None, None, None], -math.inf)
    if s['mask'] is not None:
        p.masked_fill_(~s['mask'][:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    y = p.view(b, hk, h // hk * lq, lk) @ v
    y = (y.view(b, hk, h // hk, lq, d) / total.clamp_min_(1e-30)).permute(0, 3, 1, 2, 4)
    return y.reshape(b, lq, h, d).to(s['q'].dtype)


_L = None


def _lib():
    global _L
    if _L is None:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'fast-semantic-segmentation_amd')
        if root not in sys.path:
            sys.path.insert(0, root)
        from fss import _lib as L
        _L = L
    return _L


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own(s):
    L, case = _lib(), s['case']
    stream = torch.cuda.current_stream().cuda_stream
    codes = {'f32': L.F32, 'bf16': L.BF16, 'f16': L.F16}
    if case['op'] == 'quantize':
        rows, cols, br = case['rows'], case['cols'], case['block_rows']
        q = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device='cuda')
        scales = torch.empty(-(-cols // BLOCK), -(-rows // br), device='cuda')
        L.call('fss_quantize_fp8', s['x'].data_ptr(), cols, q.data_ptr(), cols, scales.data_ptr(), scales.shape[1],
               rows, cols, br, codes[case['dtype']], stream)
        return q, scales
    if case['op'] == 'matmul':
        m, n, k = case['rows'], case['cout'], case['k']
        y = torch.empty(m, n, dtype=DTYPES[case['dtype']], device='cuda')
        desc = L.MatmulFp8Desc(rows=m, cout=n, k=k, x_ld=k, x_scale_ld=s['x_scales'].shape[1], w_ld=k,
                               w_scale_ld=s['w_scales'].shape[1], res_ld=n, y_ld=n,
                               act=L.ACT_CODES[None if case['act'] == 'none' else case['act']],
                               out_dtype=codes[case['dtype']])
        size = ctypes.c_size_t()
        L.call('fss_matmul_fp8_workspace_bytes', ctypes.byref(desc), ctypes.byref(size))
        ws = torch.empty(size.value, dtype=torch.uint8, device='cuda') if size.value else None
        L.call('fss_matmul_fp8', ctypes.byref(desc), s['x'].data_ptr(), s['x_scales'].data_ptr(), s['w'].data_ptr(),
               s['w_scales'].data_ptr(), _ptr(s['bias']), _ptr(s['residual']), y.data_ptr(), _ptr(ws), size.value, stream)
        return y
    q, k, v, mask = s['q'], s['k'], s['v'], s['mask']
    y = torch.empty_like(q)
    three = ctypes.c_int64 * 3
    desc = L.AttentionDesc(batch=case['batch'], q_len=case['q_len'], kv_len=case['kv_len'], q_heads=case['q_heads'],
                           kv_heads=case['kv_heads'], head_dim=case['head_dim'], dtype=codes[case['dtype']],
                           scale=s['scale'], q_stride=three(*q.stride()[:3]), k_stride=three(*k.stride()[:3]),
                           v_stride=three(*v.stride()[:3]), y_stride=three(*y.stride()[:3]),
                           mask_stride=three(mask.stride(0), mask.stride(1), 0) if mask is not None else three())
    size = ctypes.c_size_t()
    L.call('fss_cross_attention_workspace_bytes', ctypes.byref(desc), ctypes.byref(size))
    ws = torch.empty(size.value, dtype=torch.uint8, device='cuda') if size.value else None
    L.call('fss_cross_attention', ctypes.byref(desc), q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(s['lens']),
           _ptr(mask), y.data_ptr(), _ptr(ws), size.value, stream)
    return y


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------- exact
def _e4m3(v):
    """float64 -> the nearest e4m3 value (ties to even): 3 mantissa bits, exponents from 2^-6, at most 448."""
    exponent = torch.frexp(v)[1] - 1                       # |v| in [2^exponent, 2^(exponent + 1))
    step = torch.exp2(exponent.clamp_min(-6).double() - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'quantize':
        x, br = s['x'], case['block_rows']
        rows, cols = x.shape
        values = torch.empty(rows, cols, dtype=torch.float32, device=x.device)      # e4m3 values are exact in it
        scales = torch.empty(-(-cols // 128), -(-rows // br), dtype=torch.float64, device=x.device)
        for c in range(0, cols, 128):
            xc = x[:, c:c + 128].double()
            top = torch.nn.functional.pad(xc.abs().amax(1), (0, -rows % br)).view(-1, br).amax(1)
            scale = torch.maximum(top, torch.full_like(top, 2.0 ** -100)) / 448.0
            scales[c // 128] = scale
            values[:, c:c + 128] = _e4m3(xc / scale.repeat_interleave(br)[:rows, None])
        return values, scales
    if case['op'] == 'matmul':
        m, n, k = case['rows'], case['cout'], case['k']
        w = s['w'].double()
        for j in range(-(-n // 128)):
            for i in range(-(-k // 128)):
                w[j * 128:(j + 1) * 128, i * 128:(i + 1) * 128] *= s['w_scales'][i, j].double()
        y = torch.empty(m, n, dtype=torch.float64, device='cuda')
        for a in range(0, m, 16384):
            x = s['x'][a:a + 16384].double()
            for i in range(-(-k // 128)):
                x[:, i * 128:(i + 1) * 128] *= s['x_scales'][i, a:a + 16384, None].double()
            y[a:a + 16384] = torch.mm(x, w.t().contiguous())
            if s['bias'] is not None:
                y[a:a + 16384] += s['bias'].double()
            if s['residual'] is not None:
                y[a:a + 16384] += s['residual'][a:a + 16384].double()
        if case['act'] != 'none':
            y = torch.relu(y)
        if case['act'] == 'relu6':
            y = torch.minimum(y, torch.full_like(y, 6.0))
        return y
    b, lq, lk, h, hk, d = (case[n] for n in ('batch', 'q_len', 'kv_len', 'q_heads', 'kv_heads', 'head_dim'))
    y = torch.zeros(b, lq, h, d, dtype=torch.float64, device='cuda')
    part = max(1, (1 << 28) // lk)                          # queries at a time: 2 GiB of scores
    for i in range(b):
        n = int(s['lens'][i]) if s['lens'] is not None else lk
        for j in range(h):
            keys, values = s['k'][i, :n, j // (h // hk)].double(), s['v'][i, :n, j // (h // hk)].double()
            for a in range(0, lq, part):
                t = torch.mm(s['q'][i, a:a + part, j].double(), keys.t().contiguous()) * s['scale']
                if s['mask'] is not None:
                    t = torch.where(s['mask'][i, a:a + part, :n], t, -math.inf)
                seen = t.amax(1) > -math.inf
                weights = torch.softmax(t, dim=1)
                y[i, a:a + part, j] = torch.where(seen[:, None], torch.mm(weights, values), 0.0)
    return y
