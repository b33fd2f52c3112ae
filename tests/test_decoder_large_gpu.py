"""The decoder of test_fp8_attention_chain_gpu on a larger map: projections by the LDS-tiled product, attention in pieces and
whole, step by step against the 64-bit forms and captured."""
import ctypes

import pytest
import torch

from fss import _lib
import fp8_attention_util as U
from test_fp8_attention_chain_gpu import C, Decoder, _check_stages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('q_len,h,w', [(100, 65, 129), (2700, 65, 65)])
def test_large_decoder(q_len, h, w):
    m = Decoder(q_len, h, w, seed=q_len)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        m.run()
        s.synchronize()
        _check_stages(m)
        _lib.call('fss_capture_begin', U.stream())
        m.run()
        graph = ctypes.c_void_p()
        _lib.call('fss_capture_end', U.stream(), ctypes.byref(graph))
        for n in (m.kv_len, m.kv_len - 70, 31):
            m.lens.fill_(n)
            m.queries.neg_()
            m.run()
            want = m.state()
            for t in (m.map, m.q, m.kv, m.a, m.y):
                t.fill_(-77.0)
            for _ in range(2):
                _lib.call('fss_graph_launch', graph, U.stream())
                s.synchronize()
                for a, b in zip(want, m.state()):
                    assert torch.equal(a, b), n
        s.synchronize()
        _lib.call('fss_device_sync')
        _lib.call('fss_graph_destroy', graph)
    # the widest projection is past the few-row kernel's share of the work
    assert (m.kv_len + 15) // 16 * (C // 32) * (C // 128) > 2560
