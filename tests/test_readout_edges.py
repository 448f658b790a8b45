"""The read-out of a trained map (pink_hip_readout_*) at its edges: recorded graphs and the workspace, what is not finite or very
small, and the forms that only large maps and long batches take.  References and bounds are those of test_readout.py unless a
test says otherwise."""
import ctypes as C

import numpy as np
import pytest

from pink_amd import capi
from test_readout import Element, experts_inputs, gpu  # noqa: F401  (gpu: fixture)


# -------------------------------------------------------------------------------------------- graphs and the workspace

class Recording:
    """Calls of a handle recorded on a stream of their own."""

    def __init__(self, gpu, ro):
        self.gpu, self.ro, self.stream, self.graph, self.run = gpu, ro, C.c_void_p(), C.c_void_p(), C.c_void_p()
        gpu.ok(gpu.rt.hipStreamCreateWithFlags(C.byref(self.stream), 1))
        ro.set_stream(self.stream.value)

    def __enter__(self):
        self.gpu.ok(self.gpu.rt.hipStreamBeginCapture(self.stream, 0))
        return self

    def __exit__(self, *a):
        self.gpu.ok(self.gpu.rt.hipStreamEndCapture(self.stream, C.byref(self.graph)))
        self.gpu.ok(self.gpu.rt.hipGraphInstantiate(C.byref(self.run), self.graph, None, None, 0))

    def launch(self):
        self.gpu.ok(self.gpu.rt.hipGraphLaunch(self.run, self.stream))

    def close(self):
        self.ro.set_stream(capi.OWN_STREAM)
        self.gpu.rt.hipGraphExecDestroy(self.run)
        self.gpu.rt.hipGraphDestroy(self.graph)
        self.gpu.rt.hipStreamDestroy(self.stream)


@pytest.mark.gpu
def test_a_graph_keeps_its_workspace_when_later_calls_take_a_larger_one(gpu):  # noqa: F811
    rng = np.random.default_rng(23)
    element, t, n, k, f, h, o, more = Element(False), 300, 6, 2, 40, 24, 16, 16
    stored, _, neuron, gates = experts_inputs(rng, element, t, n, k, f, h, o)
    with capi.Readout(n, k, f, h, o) as ro:
        weights, x, y = [gpu.up(stored[i]) for i in ("w1", "b1", "w2", "b2")], gpu.up(stored["x"]), gpu.new((t, o), np.float32)
        at, g = gpu.up(neuron), gpu.up(gates)
        ro.experts(x, t, at, g, weights, y)
        ro.synchronize()
        want = gpu.down(y, (t, o), np.float32)
        ro.reserve(t)
        recording = Recording(gpu, ro)
        with recording:
            ro.experts(x, t, at, g, weights, y)
        large = [gpu.up(np.tile(a, (more, 1))) for a in (stored["x"], neuron, gates)]
        y_large = gpu.new((more * t, o), np.float32)
        for i in range(4):
            gpu.write(y, np.zeros((t, o), np.float32))
            recording.launch()
            ro.synchronize()
            assert np.array_equal(gpu.down(y, (t, o), np.float32), want)
            ro.experts(large[0], (1 + i * (more - 1) // 3) * t, large[1], large[2], weights, y_large)       # grows between the launches
            ro.synchronize()
            assert np.array_equal(gpu.down(y_large, (more * t, o), np.float32)[:t], want)
            # memory that would be where a freed workspace was stays as it is
            others = [gpu.up(np.full(1 << s, 7, np.uint8)) for s in range(16, 24)]
            recording.launch()
            ro.synchronize()
            for s, p in zip(range(16, 24), others):
                assert (gpu.down(p, 1 << s, np.uint8) == 7).all()
        recording.close()


@pytest.mark.gpu
def test_recorded_calls_do_not_grow_the_workspace(gpu):  # noqa: F811
    rng = np.random.default_rng(29)
    t, n, k, f, h, o = 200, 6, 2, 40, 24, 16
    stored, _, neuron, gates = experts_inputs(rng, Element(False), t, n, k, f, h, o)
    with capi.Readout(n, k, f, h, o) as ro:
        weights, x, y, saved = [gpu.up(stored[i]) for i in ("w1", "b1", "w2", "b2")], gpu.up(stored["x"]), gpu.new((t, o), np.float32), gpu.new(ro.saved_bytes(t), np.int8)
        at, g, d, one = gpu.up(neuron), gpu.up(gates), gpu.new((t, n), np.float32), gpu.up(np.ones(n, np.float32))
        ro.reserve(t // 2)
        recording = Recording(gpu, ro)
        with recording:                                    # refused before anything is launched; the recording goes on
            for call in (lambda: ro.experts(x, t, at, g, weights, y), lambda: ro.experts_backward(x, t, g, weights, saved, y, [x, None, None, None, None, None]),
                         lambda: ro.reserve(t)):
                with pytest.raises(capi.PinkError) as e:
                    call()
                assert e.value.status == -4 and "reserve" in str(e.value)
            ro.experts(x, t // 2, at, g, weights, y)
        recording.launch()
        ro.synchronize()
        got = gpu.down(y, (t, o), np.float32)[:t // 2]
        ro.experts(x, t // 2, at, g, weights, y)
        ro.synchronize()
        assert np.array_equal(gpu.down(y, (t, o), np.float32)[:t // 2], got)
        recording.close()
    with capi.Readout(n, k) as ro:
        chosen, weighed = gpu.new((t, k), np.int32), gpu.new((t, k), np.float32)
        recording = Recording(gpu, ro)
        with recording:
            with pytest.raises(capi.PinkError) as e:
                ro.route_backward(d, t, one, one, None, at, g, g, d)
            assert e.value.status == -4 and "reserve" in str(e.value)
            ro.route(d, t, one, one, None, chosen, weighed)                                                  # has no workspace
        recording.launch()
        ro.synchronize()
        recording.close()
