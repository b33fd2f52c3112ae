"""fss_quantize_fp8, fss_matmul_fp8 and fss_cross_attention used together behind a convolution, as a decoder
on a feature map uses them: eagerly, captured, on two streams; and tensors past 2^32 bytes."""
import ctypes

import numpy as np
import pytest
import torch

from fss import _lib
import gpu_util as gu
import fp8_attention_util as U

pytestmark = pytest.mark.gpu

C, HEADS, KV_HEADS, D = 256, 8, 2, 32                 # map channels, heads, shared key / value heads


class Decoder:
    """y = queries + W_o attention(W_q queries, W_kv map), map = relu(conv3x3(frame features)); every buffer is
    its own, so two of them can run at once."""

    def __init__(self, q_len, h, w, seed):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g)
        self.h, self.w, self.q_len, self.kv_len = h, w, q_len, h * w
        self.feat = rand(1, h, w, 64).to(torch.bfloat16).cuda()
        self.queries = rand(q_len, C).to(torch.bfloat16).cuda()
        self.lens = torch.tensor([self.kv_len], dtype=torch.int32).cuda()
        self.mask = (torch.rand(q_len, self.kv_len, generator=g) < 0.6).cuda()
        self.mask[::5] = False
        wp, self.k_pad, self.cout_pad = gu.pack_conv_weights((rand(3, 3, 64, C) / 24).numpy(), 'bf16')
        self.conv_w, self.bias = wp, rand(C).cuda()
        empty = lambda *s, dt=torch.bfloat16: torch.full(s, -77.0).to(dt).cuda()
        self.map = empty(self.kv_len, C)
        self.weights = {}
        for name, cout, k in (('q', HEADS * D, C), ('kv', 2 * KV_HEADS * D, C), ('o', C, HEADS * D)):
            f = (rand(cout, k) / k ** 0.5).cuda()
            q8, s8 = torch.empty(cout, k, dtype=torch.uint8, device='cuda'), empty(k // 128, -(-cout // 128), dt=torch.float32)
            self.call('fss_quantize_fp8', f.data_ptr(), k, q8.data_ptr(), k, s8.data_ptr(), s8.shape[1], cout, k, 128, _lib.F32)
            self.weights[name] = (q8, s8, rand(cout).cuda())
        self.q, self.kv, self.a = empty(q_len, HEADS, D), empty(self.kv_len, 2, KV_HEADS, D), empty(q_len, HEADS, D)
        self.y = empty(q_len, C)
        self.small = {n: (torch.empty(r, C, dtype=torch.uint8, device='cuda'), empty(C // 128, r, dt=torch.float32))
                      for n, r in (('q', q_len), ('kv', self.kv_len), ('o', q_len))}
        s = (0, HEADS * D, D)
        kvs = (0, 2 * KV_HEADS * D, D)
        self.adesc = U.attention_desc(1, q_len, self.kv_len, HEADS, KV_HEADS, D, 'bf16', q_stride=s, y_stride=s, k_stride=kvs,
                                      v_stride=kvs, mask_stride=(0, self.mask.stride(0), 0))
        self.ws = {}
        torch.cuda.synchronize()

    def call(self, name, *args):
        _lib.call(name, *args, U.stream())

    def workspace(self, name, desc):
        size = ctypes.c_size_t()
        _lib.call('fss_%s_workspace_bytes' % name, ctypes.byref(desc), ctypes.byref(size))
        return torch.empty(size.value + 16, dtype=torch.uint8, device='cuda'), size.value

    def project(self, name, x, out, residual=None):
        rows, (q8, s8), (w, ws, bias) = x.shape[0], self.small[name], self.weights[name]
        cout = w.shape[0]
        self.call('fss_quantize_fp8', x.data_ptr(), C, q8.data_ptr(), C, s8.data_ptr(), rows, rows, C, 1, _lib.BF16)
        d = U.matmul_desc(rows, cout, C, 'bf16')
        if name not in self.ws:
            self.ws[name] = self.workspace('matmul_fp8', d)
        buf, size = self.ws[name]
        self.call('fss_matmul_fp8', ctypes.byref(d), q8.data_ptr(), s8.data_ptr(), w.data_ptr(), ws.data_ptr(), bias.data_ptr(),
                  None if residual is None else residual.data_ptr(), out.data_ptr(), buf.data_ptr(), size)

    def run(self):
        d = _lib.ConvDesc(n=1, h=self.h, w=self.w, cin=64, cout=C, kh=3, kw=3, stride=1, dilation=1, pad_top=1, pad_left=1,
                          ho=self.h, wo=self.w, act=_lib.ACT_RELU, in_dtype=_lib.BF16, out_dtype=_lib.BF16, y_ld=C, res_ld=C,
                          k_pad=self.k_pad, cout_pad=self.cout_pad, config=0)
        self.call('fss_conv2d_nhwc', ctypes.byref(d), self.feat.data_ptr(), self.conv_w.data_ptr(), self.bias.data_ptr(), None,
                  self.map.data_ptr())
        self.project('q', self.queries, self.q)
        self.project('kv', self.map, self.kv)
        if 'a' not in self.ws:
            self.ws['a'] = self.workspace('cross_attention', self.adesc)
        buf, size = self.ws['a']
        self.call('fss_cross_attention', ctypes.byref(self.adesc), self.q.data_ptr(), self.kv.data_ptr(),
                  self.kv[:, 1].data_ptr(), self.lens.data_ptr(), self.mask.data_ptr(), self.a.data_ptr(), buf.data_ptr(), size)
        self.project('o', self.a.view(self.q_len, C), self.y, self.queries)
        return self.y

    def state(self):
        return [t.clone() for t in (self.map, self.q, self.kv, self.a, self.y)]


def _check_stages(m):
    """Every stage against its 64-bit form on the stage's own inputs."""
    torch.cuda.synchronize()
    for name, x, out, residual in (('q', m.queries, m.q, None), ('kv', m.map, m.kv, None), ('o', m.a, m.y, m.queries)):
        x = x.reshape(-1, C).float().cpu().numpy()
        xq, xs = U.quantize_ref(x, 1)
        np.testing.assert_array_equal(m.small[name][0].view(torch.float8_e4m3fn).float().cpu().numpy(), xq)
        np.testing.assert_allclose(m.small[name][1].cpu().numpy(), xs, rtol=2.0 ** -24)
        w, ws, bias = m.weights[name]
        wd = w.view(torch.float8_e4m3fn).float().cpu().numpy() * U.spread(ws.cpu().numpy(), 128, w.shape[0], C)
        xd = xq * U.spread(m.small[name][1].cpu().numpy(), 1, x.shape[0], C)
        want, size = xd @ wd.T + bias.cpu().numpy(), np.abs(xd) @ np.abs(wd).T + np.abs(bias.cpu().numpy())
        if residual is not None:
            want, size = want + residual.float().cpu().numpy(), size + np.abs(residual.float().cpu().numpy())
        # the terms of check_matmul
        tol = size * (2 * 2.0 ** -24 * (128 + C / 128 + 4) + 7 * 2.0 ** -13) + np.abs(want) * U.HALF['bf16']
        assert (np.abs(out.reshape(want.shape).float().cpu().numpy() - want) <= tol).all(), name
    q, kv = m.q[None], m.kv[None]
    mask = m.mask[None, None].expand(1, HEADS, -1, -1)
    ref = U.attention_ref(q, kv[:, :, 0], kv[:, :, 1], lens=m.lens, mask=mask)
    U.check_attention(m.a[None], ref, 'bf16', D, m.kv_len)
    assert (m.a[::5] == 0).all()                       # queries without a region


@pytest.mark.parametrize('q_len,h,w', [(1, 33, 65), (100, 33, 65), (515, 17, 33)])
def test_decoder_step_by_step(q_len, h, w):
    m = Decoder(q_len, h, w, seed=q_len)
    m.run()
    _check_stages(m)


@pytest.mark.parametrize('q_len,h,w', [(1, 33, 65), (100, 33, 65)])
def test_decoder_captured(q_len, h, w):
    """Replays with eager work and synchronisations between them, inputs and lengths changing in place."""
    m = Decoder(q_len, h, w, seed=5)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        m.run()
        s.synchronize()
        _lib.call('fss_capture_begin', U.stream())
        m.run()
        graph = ctypes.c_void_p()
        _lib.call('fss_capture_end', U.stream(), ctypes.byref(graph))
        for i, n in enumerate((m.kv_len, 1, 0, m.kv_len - 70, m.kv_len)):
            m.lens.fill_(n)
            m.queries.add_(0.25 * i)
            m.feat.neg_()
            m.run()
            want = m.state()
            for t in (m.map, m.q, m.kv, m.a, m.y):
                t.fill_(-77.0)
            s.synchronize()
            for _ in range(2):
                _lib.call('fss_graph_launch', graph, U.stream())
            s.synchronize()
            for a, b in zip(want, m.state()):
                assert torch.equal(a, b), (i, n)
        s.synchronize()
        torch.cuda.synchronize()
        _lib.call('fss_graph_destroy', graph)


def test_two_decoders_at_once():
    """Two captured decoders on two streams, each with its own buffers and workspaces."""
    made = [(Decoder(100, 33, 65, seed=1), torch.cuda.Stream()), (Decoder(7, 33, 65, seed=2), torch.cuda.Stream())]
    want, graphs = [], []
    for m, s in made:
        with torch.cuda.stream(s):
            m.run()
            s.synchronize()
            want.append(m.state())
            _lib.call('fss_capture_begin', U.stream())
            m.run()
            graphs.append(ctypes.c_void_p())
            _lib.call('fss_capture_end', U.stream(), ctypes.byref(graphs[-1]))
    for _ in range(10):
        for (m, s), g in zip(made, graphs):
            with torch.cuda.stream(s):
                m.y.fill_(-77.0)
                _lib.call('fss_graph_launch', g, U.stream())
    torch.cuda.synchronize()
    for (m, _), w, g in zip(made, want, graphs):
        for a, b in zip(w, m.state()):
            assert torch.equal(a, b)
        _lib.call('fss_graph_destroy', g)


def test_first_call_under_capture():
    """No warm-up call on these sizes: the largest tiles and the widest heads, which ask for more than 64 KiB of LDS."""
    g = torch.Generator(device='cuda').manual_seed(4)
    q, k, v = (torch.randn(1, n, 2, 248, generator=g, device='cuda').to(torch.float16) for n in (300, 700, 700))
    y = torch.zeros_like(q)
    ad = U.attention_desc(1, 300, 700, 2, 2, 248, 'f16')
    rows, cout, k8 = 4096, 4096, 1024
    x8 = torch.randint(0, 120, (rows, k8), generator=g, device='cuda', dtype=torch.uint8)
    w8 = torch.randint(0, 120, (cout, k8), generator=g, device='cuda', dtype=torch.uint8)
    xs, ws = torch.full((8, rows), 1e-3, device='cuda'), torch.full((8, 32), 1e-3, device='cuda')
    out = torch.zeros(rows, cout, dtype=torch.float16, device='cuda')
    md = U.matmul_desc(rows, cout, k8, 'f16')
    size = ctypes.c_size_t()
    _lib.call('fss_cross_attention_workspace_bytes', ctypes.byref(ad), ctypes.byref(size))
    buf = torch.empty(size.value + 16, dtype=torch.uint8, device='cuda')
    torch.cuda.synchronize()

    def run():
        _lib.call('fss_matmul_fp8', ctypes.byref(md), x8.data_ptr(), xs.data_ptr(), w8.data_ptr(), ws.data_ptr(), None, None,
                  out.data_ptr(), None, 0, U.stream())
        _lib.call('fss_cross_attention', ctypes.byref(ad), q.data_ptr(), k.data_ptr(), v.data_ptr(), None, None, y.data_ptr(),
                  buf.data_ptr(), size.value, U.stream())

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _lib.call('fss_capture_begin', U.stream())
        run()
        graph = ctypes.c_void_p()
        _lib.call('fss_capture_end', U.stream(), ctypes.byref(graph))
        got = []
        for _ in range(3):
            y.zero_()
            out.zero_()
            _lib.call('fss_graph_launch', graph, U.stream())
            s.synchronize()
            got.append((y.clone(), out.clone()))
        run()
        s.synchronize()
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, y) and torch.equal(b, out) and out.abs().max() > 0
    U.check_attention(y, U.attention_ref(q, k, v), 'f16', 248, 700)
    _lib.call('fss_graph_destroy', graph)


def test_matmul_and_quantize_past_4_gib():
    """Row offsets past 2^32 bytes: the last rows equal those of a small call on the same rows."""
    rows, k, cout = (1 << 20) + 70, 4096 + 128, 24
    g = torch.Generator(device='cuda').manual_seed(3)
    x = torch.randn(rows, k, generator=g, device='cuda', dtype=torch.bfloat16)            # 8.9 GB
    q = torch.empty(rows, k, dtype=torch.uint8, device='cuda')                            # 4.4 GB
    xs = torch.empty(k // 128, rows, device='cuda')
    w, ws = U.quantize_ref(U.features(cout, k, 1), 128)
    wd, wsd = U._bytes(w, k), torch.from_numpy(ws).cuda()
    tail = 70
    for first, n in ((0, rows), (rows - tail, tail)):
        qq, ss = (q, xs) if first == 0 else (torch.empty(n, k, dtype=torch.uint8, device='cuda'),
                                             torch.empty(k // 128, n, device='cuda'))
        y = torch.empty(n, cout, device='cuda')
        _lib.call('fss_quantize_fp8', x[first:].data_ptr(), k, qq.data_ptr(), k, ss.data_ptr(), n, n, k, 1, _lib.BF16, U.stream())
        d = U.matmul_desc(n, cout, k, 'f32')
        size = ctypes.c_size_t()
        _lib.call('fss_matmul_fp8_workspace_bytes', ctypes.byref(d), ctypes.byref(size))
        buf = torch.empty(size.value + 16, dtype=torch.uint8, device='cuda')
        _lib.call('fss_matmul_fp8', ctypes.byref(d), qq.data_ptr(), ss.data_ptr(), wd.data_ptr(), wsd.data_ptr(), None, None,
                  y.data_ptr(), buf.data_ptr(), size.value, U.stream())
        if first == 0:
            whole, whole_q, whole_s = y[-tail:].clone(), q[-tail:].clone(), xs[:, -tail:].clone()
    assert torch.equal(whole_q, qq) and torch.equal(whole_s, ss)
    # the two calls may use kernels that add the blocks of k in another order: 33 blocks, a step each
    bound = (qq.view(torch.float8_e4m3fn).double().abs() * U_spread(ss, k)) @ (
        wd.view(torch.float8_e4m3fn).double().abs() * U_spread_w(wsd, cout, k)).t()
    assert ((whole - y).double().abs() <= bound * 2.0 ** -23 * 2 * 40).all()


def U_spread(s, k):
    return s.t().repeat_interleave(128, 1)[:, :k].double()


def U_spread_w(s, cout, k):
    return s.t().repeat_interleave(128, 0)[:cout].repeat_interleave(128, 1)[:, :k].double()
