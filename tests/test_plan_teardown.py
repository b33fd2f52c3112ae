"""End of a plan's life: its executable graph is destroyed and its memory returned only once the device is
drained, and never while a stream is being captured, whenever Python happens to collect it."""
import contextlib
import ctypes
import gc
import weakref

import numpy as np
import pytest
import torch

from fss import _lib, plan, plan_schedule


gpu = pytest.mark.gpu


class Recorder(object):
    """The entry points a capture and a teardown use, with the runtime's rule that a device
    cannot be synchronised while a stream of it is being captured."""

    def __init__(self):
        self.log, self.capturing, self.pending, self.errors = [], False, set(), []

    def _note(self, what):
        self.log.append(what)
        if self.capturing and what[0] in ('sync', 'destroy', 'event'):
            self.errors.append('%s %s during a capture' % what)

    def fss_capture_begin(self, stream):
        self.capturing = True
        return 0

    def fss_capture_end(self, stream, out):
        self.capturing = False
        out._obj.value = 4096
        return 0

    def fss_device_sync(self):
        self._note(('sync', None))
        if self.capturing:
            return 2
        self.pending.clear()
        return 0

    def fss_graph_destroy(self, graph):
        self._note(('destroy', graph.value))
        if graph.value in self.pending:
            self.errors.append('graph %d destroyed with a launch in flight' % graph.value)
        return 0

    def fss_event_destroy(self, event):
        self._note(('event', event.value))
        return 0


@pytest.fixture
def runtime(monkeypatch):
    r = Recorder()
    for module in (_lib, plan, plan_schedule):
        monkeypatch.setattr(module, 'lib', r)
    monkeypatch.setattr(torch.cuda, 'device', lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    gc.collect()
    gc.disable()
    monkeypatch.setattr(plan_schedule, '_retired', [], raising=False)
    yield r
    gc.enable()


def bare_plan(graph=None):
    cg = plan.CompiledGraph.__new__(plan.CompiledGraph)
    cg.device, cg.sh = 0, ctypes.c_void_p(1)
    cg.graph_exec = None if graph is None else ctypes.c_void_p(graph)
    cg.events, cg.two_streams, cg.steps = [], False, []
    cg.temps = [np.zeros(1)]           # stands for the device tensors
    return cg


def test_teardown_drains_first(runtime):
    cg = bare_plan(7)
    cg.events = [ctypes.c_void_p(8)]
    runtime.pending.add(7)
    del cg
    assert runtime.log == [('sync', None), ('destroy', 7), ('event', 8)] and not runtime.errors


def test_plan_collected_during_a_capture(runtime):
    """A plan in a reference cycle ends when the cyclic collector runs, here in the middle of another
    plan's capture: its graph, whose last launch is in flight, and its memory stay until the capture is over."""
    old = bare_plan(7)
    old.events = [ctypes.c_void_p(8)]
    old.cycle = old
    memory = weakref.ref(old.temps[0])
    runtime.pending.add(7)
    del old
    new = bare_plan()

    def run_eager():
        gc.collect()
        assert runtime.capturing and plan_schedule._retired and memory() is not None
    new.run_eager = run_eager
    new._capture()
    assert runtime.errors == []
    assert runtime.log == [('sync', None), ('destroy', 7), ('event', 8)]
    assert memory() is None
    assert new.graph_exec.value == 4096


def test_plan_dropped_during_a_capture_of_the_caller(runtime):
    """The same in a capture this package did not begin: what the refusal or torch's own state says
    puts the teardown off, and the next plan that ends makes up for it."""
    first, second = bare_plan(7), bare_plan(9)
    runtime.pending |= {7, 9}
    torch.cuda.is_current_stream_capturing = lambda: True          # (the fixture puts the original back)
    del first
    assert runtime.log == []
    torch.cuda.is_current_stream_capturing = lambda: False
    del second
    assert [e for e in runtime.log if e[0] == 'destroy'] in ([('destroy', 7), ('destroy', 9)],
                                                            [('destroy', 9), ('destroy', 7)])
    assert runtime.errors == []


def test_refused_drain_keeps_the_graph(runtime):
    """A synchronisation that is refused (any reason) leaves the graph alone until one succeeds."""
    cg = bare_plan(7)
    runtime.pending.add(7)
    runtime.fss_device_sync = lambda: 2
    del cg
    assert runtime.log == []
    del runtime.fss_device_sync
    plan_schedule.release_retired()
    assert runtime.log == [('sync', None), ('destroy', 7)] and not runtime.errors


# ------------------------------------------------------------------------------------- on the device
def small_plan():
    from test_models_gpu import build
    g, _, outs, weights = build('icnet', 'dilated_resnet50', 0.5, [1.0, 2.0, 3.0, 4.0], (1, 256, 512, 3), (257, 513))
    return plan.CompiledGraph(g, outs, weights, dtype='bfloat16', autotune=False)


@gpu
def test_device_sync_is_refused_during_a_capture():
    """... by the library itself, so that the capture goes on."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = torch.randn(64, device='cuda')
        y = torch.zeros(64, dtype=torch.float16, device='cuda')
        h = s.cuda_stream
        want = x.half()
        s.synchronize()
        _lib.call('fss_capture_begin', h)
        assert _lib.lib.fss_device_sync() != 0
        _lib.call('fss_to_half', x.data_ptr(), y.data_ptr(), 64, _lib.F32, h)
        graph = ctypes.c_void_p()
        _lib.call('fss_capture_end', h, ctypes.byref(graph))
        _lib.call('fss_device_sync')
        for _ in range(3):
            y.zero_()
            _lib.call('fss_graph_launch', graph, h)
            s.synchronize()
            assert torch.equal(y, want)
        _lib.call('fss_device_sync')
        _lib.call('fss_graph_destroy', graph)


@gpu
def test_plans_collected_during_the_capture_of_others():
    """Plans whose last pass nobody waited for, collected in the middle of another plan's capture."""
    img = np.random.default_rng(0).integers(0, 256, (1, 256, 512, 3)).astype(np.uint8)
    want = small_plan().run(img)
    for _ in range(2):
        old = small_plan()
        old.set_input(img)
        old.launch()
        old.cycle = old
        new = small_plan()
        eager = new.run_eager
        del old

        def run_eager():
            gc.collect()
            assert plan_schedule._retired
            eager()
        new.run_eager = run_eager
        new._capture()
        assert not plan_schedule._retired
        for a, b in zip(want, new.run(img)):
            assert np.array_equal(a, b)
        del new, eager, run_eager
        gc.collect()


@gpu
def test_plan_ends_with_its_last_reference():
    """... and not when the cyclic collector gets round to it."""
    img = np.random.default_rng(0).integers(0, 256, (1, 256, 512, 3)).astype(np.uint8)
    gc.collect()
    gc.disable()
    try:
        cg = small_plan()
        cg.run(img)
        ended, held, own = weakref.ref(cg), torch.cuda.memory_allocated(), cg.activation_bytes
        del cg
        assert ended() is None and own > 0 and held - torch.cuda.memory_allocated() >= own
    finally:
        gc.enable()
