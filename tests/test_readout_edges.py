"""The read-out of a trained map (pink_hip_readout_*) at its edges: recorded graphs and the workspace, what is not finite or very
small, and the forms that only large maps and long batches take.  References and bounds are those of test_readout.py unless a
test says otherwise."""
import ctypes as C

import numpy as np
import pytest

import test_readout as base
from pink_amd import capi
from test_readout import ACT, BENT, S, STEEP, Element, assert_within, experts_inputs, experts_reference, f_and_slope, gpu, pack, to_bf16  # noqa: F401  (gpu: fixture)


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


@pytest.mark.gpu
def test_the_workspace_takes_what_calls_need(gpu):  # noqa: F811
    """No rows to be added up where one neuron answers, no second place for what a caller's buffer holds."""
    def free():
        now, all_ = C.c_size_t(), C.c_size_t()
        gpu.ok(gpu.rt.hipMemGetInfo(C.byref(now), C.byref(all_)))
        return now.value

    t, wide, allowed = 65536, 4096, 64 << 20               # wide rows in float32 would take 1 GiB
    with capi.Readout(4, 1, 8, 8, wide) as ro:
        before = free()
        ro.reserve(t)
        assert before - free() < allowed
    with capi.Readout(4, 1, 8, wide, 8) as ro:
        x, y, at, g = gpu.new((t, 8), np.float32), gpu.new((t, 8), np.float32), gpu.up(np.arange(t, dtype=np.int32) % 4), gpu.new(t, np.float32)
        weights, saved = [gpu.new((4, wide, 8), np.float32)] * 4, gpu.new(ro.saved_bytes(t), np.int8)
        before = free()
        ro.experts(x, t, at, g, weights, y, dev_saved=saved)
        ro.synchronize()
        assert before - free() < allowed


# --------------------------------------------------------------------------------------------------------------- AdamW

F = np.float32


def adamw_tensor(gpu, value, grad, bits, m=None, v=None, decay=0.0):  # noqa: F811
    """(the descriptor, pointers to the two states' values)"""
    n = value.size
    m, v = (np.zeros(n, F) if x is None else x for x in (m, v))
    t = dict(value=gpu.up(value), gradient=gpu.up(grad), size=n, decay=decay)
    if bits == 8:
        (mc, ms), (vc, vs) = pack(m, False), pack(v, True)
        t.update(first=gpu.up(mc), second=gpu.up(vc), first_scale=gpu.up(ms), second_scale=gpu.up(vs), first_values=gpu.new(n, F), second_values=gpu.new(n, F))
        return t, ("first_values", "second_values")
    t.update(first=gpu.up(m), second=gpu.up(v))
    return t, ("first", "second")


@pytest.mark.gpu
@pytest.mark.parametrize("epsilon", [1e-45, 1e-40, 2.0 ** -126, 1e-30, 1e-20, 2.0 ** -39, 2.0 ** -38, 1e-8, 1.0])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_small_gradients_and_epsilons(gpu, bits, epsilon):  # noqa: F811
    # whole blocks of gradients of one size, from those that are no gradient at all to those whose square is subnormal, or 0
    rng = np.random.default_rng(3)
    sizes = np.array([0, 1e-37, 1e-30, 1e-24, 3e-23, 1e-21, 1e-20, 1e-19, 1e-18, 1e-8, 1], F)
    grad = (np.repeat(sizes, 256) * rng.choice([-1, 1], sizes.size * 256)).astype(F)
    value = rng.standard_normal(grad.size).astype(F)
    lr, b1, b2, step = F(2e-3), F(0.9), F(0.99), 1
    with capi.Readout(4) as ro:
        t, _ = adamw_tensor(gpu, value, grad, bits)
        ro.adamw(ro.tensors([t]), step, learning_rate=lr, beta_first=b1, beta_second=b2, epsilon=epsilon, bits=bits)
        ro.synchronize()
        got = gpu.down(t["value"], grad.size, F).astype(np.float64)
    m, v = (grad * (F(1) - b1)).astype(F).astype(np.float64), ((grad * grad) * (F(1) - b2)).astype(F).astype(np.float64)
    eps, c1, c2 = float(F(epsilon)), 1 / (1 - float(b1) ** step), 1 / (1 - float(b2) ** step)
    root = np.sqrt(v * c2)
    # c2 second is rounded, below 2^-126 to multiples of 2^-149; a root moves by no more than d / root, nor than sqrt(d)
    d = 2 * S * v * c2 + 2.0 ** -150
    off_root = np.minimum(np.sqrt(d), d / np.maximum(root, 1e-300)) * (v > 0)
    change = m * c1 / (root + eps)
    off = np.abs(change) * (16 * S + off_root / (np.maximum(root - off_root, 0) + eps)) + 2.0 ** -148 * c1 / (root + eps)
    want = value.astype(np.float64) - float(lr) * change
    assert_within(got, want, float(lr) * off + 2 * S * np.abs(want), "value")
    assert np.array_equal(got[:256], value[:256])          # where there was no gradient nothing moves


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_gradients_that_are_not_finite(gpu, bits):  # noqa: F811
    """They go into the value and the states; of 8-bit states a block's scale is its largest magnitude, so the block holds NaN from then on."""
    rng = np.random.default_rng(4)
    n, options = 5 * 256 + 100, dict(learning_rate=2e-3, beta_first=0.9, beta_second=0.99, epsilon=1e-8)
    value, grad = rng.standard_normal(n).astype(F), rng.standard_normal(n).astype(F)
    m, v = (0.1 * rng.standard_normal(n)).astype(F), (0.01 * rng.standard_normal(n) ** 2).astype(F)
    bad = {300: np.nan, 256 * 2 + 255: np.inf, 256 * 3: -np.inf, n - 1: np.nan}
    for at, x in bad.items():
        grad[at] = x
    with capi.Readout(4) as ro:
        t, states = adamw_tensor(gpu, value, grad, bits, m, v)
        clean = grad.copy()
        clean[list(bad)] = 0
        other, _ = adamw_tensor(gpu, value, clean, bits, m, v)
        table, without = ro.tensors([t]), ro.tensors([other])
        hurt = np.isin(np.arange(n), list(bad))
        block = np.isin(np.arange(n) // 256, [at // 256 for at in bad])
        for step in (1, 2):
            for x in (table, without):
                ro.adamw(x, step, bits=bits, **options)
                if bits == 8:
                    ro.adamw_unpack(x)
            ro.synchronize()
            got, want = gpu.down(t["value"], n, F), gpu.down(other["value"], n, F)
            of_value = block if bits == 8 and step == 2 else hurt
            assert np.isnan(got[of_value]).all() and np.array_equal(got[~of_value], want[~of_value])
            for name in states:
                got, want = gpu.down(t[name], n, F), gpu.down(other[name], n, F)
                of_state = block if bits == 8 else hurt
                assert not np.isfinite(got[of_state]).any() and np.array_equal(got[~of_state], want[~of_state])
                if bits == 8:
                    assert np.isnan(got[of_state]).all()


# ----------------------------------------------------------------------------------------------- what is kept of a model

KEPT_GATES = [0.0, -0.0, 1e-45, 1e-25, 1e-21, 1e-19, 1e-10, 0.5, -0.75]


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("act", ["identity", "relu", "gelu", "silu"])
@pytest.mark.parametrize("size", [1.0, 1e3, 1e5, 1e20])
def test_gradients_of_gates_that_are_small(gpu, act, bf16, size):  # noqa: F811
    """A gate's gradient does not depend on the gate: right at any gate, and for values before the activation of any size."""
    rng = np.random.default_rng(6)
    element, t, n, k, f, h, o = Element(bf16), 90, 3, 3, 16, 24, 8
    stored, value, neuron, _ = experts_inputs(rng, element, t, n, k, f, h, o)
    for i in ("w1", "b1"):
        stored[i], value[i] = element.store(value[i] * size)
    gates = np.resize(np.array(KEPT_GATES, np.float32), (t, k))
    dy_stored, dy = element.store(rng.standard_normal((t, o)))
    with np.errstate(over="ignore", under="ignore"):
        want = experts_reference(value, element, act, neuron, gates, dy)
    with capi.Readout(n, k, f, h, o, activation=ACT[act], element=element.id) as ro:
        p = {i: gpu.up(v) for i, v in stored.items()}
        weights, saved, y = [p[i] for i in ("w1", "b1", "w2", "b2")], gpu.new(ro.saved_bytes(t), np.int8), gpu.new((t, o), element.dtype)
        g, dgates = gpu.up(gates), gpu.new((t, k), element.dtype)
        ro.experts(p["x"], t, gpu.up(neuron), g, weights, y, dev_saved=saved)
        ro.experts_backward(p["x"], t, g, weights, saved, gpu.up(dy_stored), [None, dgates, None, None, None, None])
        ro.synchronize()
        assert_within(element.values(gpu.down(dgates, (t, k), element.dtype)), *want["dgates"], "of gates")


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_slopes_from_what_bfloat16_models_keep(gpu, act):  # noqa: F811
    """Of a before GELU and SILU 11 bits are kept, so a slope near zero is off by 2^-11 of a, not by 2^-8; a value comes from gate f(a),
    rounded once.  One image a neuron and one hidden value: bias gradients are da itself."""
    element, n = Element(True), 2048
    rng = np.random.default_rng(8)
    # a = x w1 + b1 is a number of 32 bits; slopes cross zero at -0.75 (GELU) and -1.28 (SILU)
    _, x = element.store(np.ones((n, 1)))
    w1s, w1 = element.store(rng.uniform(-2, 1, (n, 1, 1)))
    b1s, b1 = element.store(rng.uniform(-0.25, 0.25, (n, 1)))
    w2s, w2 = element.store(rng.uniform(0.5, 1, (n, 1, 1)))
    dys, dy = element.store(rng.uniform(0.5, 1, (n, 1)))
    gates = rng.uniform(0.1, 1, (n, 1)).astype(np.float32)
    a, g, back = w1[:, 0, 0] + b1[:, 0], gates[:, 0].astype(np.float64), dy[:, 0] * w2[:, 0, 0]
    v, slope = f_and_slope(act, a)
    off_a = 4 * S * np.abs(a) + 2.0 ** -11 * np.abs(a)
    da = g * back * slope
    off_da = np.abs(g * back) * (BENT[act] * off_a + 8 * S * (1 + np.abs(a))) + 4 * S * np.abs(da)
    dg = back * v
    off_dg = np.abs(back) * (8 * S * (np.abs(a) + np.abs(v)) + element.u * np.abs(v)) + 8 * S * np.abs(dg)
    assert (np.abs(g * back) * BENT[act] * 2.0 ** -9 * np.abs(a) > 1.5 * (off_da + element.u * np.abs(da))).any()        # 8 bits would show
    with capi.Readout(n, 1, 1, 1, 1, activation=ACT[act], element=element.id) as ro:
        weights = [gpu.up(w1s), gpu.up(b1s), gpu.up(w2s), None]
        saved, y, db1, dgates = gpu.new(ro.saved_bytes(n), np.int8), gpu.new((n, 1), np.uint16), gpu.new((n, 1), np.uint16), gpu.new((n, 1), np.uint16)
        xs, at, gd = gpu.up(to_bf16(x)), gpu.up(np.arange(n, dtype=np.int32)[:, None]), gpu.up(gates)
        ro.experts(xs, n, at, gd, weights, y, dev_saved=saved)
        ro.experts_backward(xs, n, gd, weights, saved, gpu.up(dys), [None, dgates, None, db1, None, None])
        ro.synchronize()
        # (da is rounded as it is kept, and a sum of one term of that is the same number)
        assert_within(element.values(gpu.down(db1, (n, 1), np.uint16))[:, 0], da, off_da + element.u * (np.abs(da) + off_da), "da")
        assert_within(element.values(gpu.down(dgates, (n, 1), np.uint16))[:, 0], dg, off_dg + element.u * (np.abs(dg) + off_dg), "of gates")


# ------------------------------------------------------------------------------------------ large maps and long batches

LARGE_ROUTES = [  # images, neurons, chosen, sigmoid, renormalise, groups, kept, bias, ties; one for every number of registers
    (9, 200, 3, False, False, 1, 1, True, False), (9, 200, 64, True, True, 1, 1, False, True),
    (5, 380, 7, False, False, 1, 1, False, True), (9, 500, 5, False, True, 1, 1, True, True),
    (9, 700, 64, False, False, 1, 1, False, True), (9, 768, 2, True, False, 1, 1, True, False),
    (6, 1000, 9, False, True, 1, 1, True, True), (6, 1024, 64, False, False, 1, 1, True, False),
    (6, 1200, 33, True, True, 1, 1, False, True), (6, 1280, 8, False, False, 1, 1, False, False),
    (5, 1500, 64, False, True, 1, 1, True, True), (5, 1536, 1, False, False, 1, 1, True, True),
    (5, 1600, 8, True, False, 1, 1, True, False), (5, 1600, 64, False, False, 1, 1, False, True),
    (5, 1700, 17, False, True, 1, 1, True, True), (5, 1800, 64, False, False, 1, 1, True, True),
    (4, 2048, 64, True, True, 1, 1, False, True), (4, 2047, 5, False, False, 1, 1, True, False),
    # groups whose kept neurons are more than eight registers, and fewer, beside as many of all neurons
    (4, 1600, 64, False, True, 40, 20, True, True), (4, 2000, 9, False, False, 10, 9, False, False), (4, 700, 64, True, True, 7, 7, True, True),
    (4, 700, 20, False, False, 35, 5, True, True), (4, 1000, 6, False, True, 50, 3, False, False), (4, 1270, 4, False, False, 64, 2, True, True),
    (4, 1500, 8, True, False, 2, 1, False, True), (4, 2048, 8, False, True, 64, 16, True, False), (4, 2040, 8, False, True, 2, 2, True, False),
    (2, 32768, 64, False, False, 1, 1, True, False), (2, 20000, 9, True, True, 1000, 30, False, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", LARGE_ROUTES, ids=lambda c: "-".join(str(int(x)) for x in c))
def test_route_of_large_maps(gpu, case):  # noqa: F811
    base.test_route(gpu, *case)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [c for c in LARGE_ROUTES if c[1] <= 2048 and not c[2] == 64] + [
    # blocks of up to 64 images each
    (16500, 9, 2, False, False, 1, 1, True, False), (16384, 9, 3, False, True, 3, 2, False, False), (16400, 5, 2, True, True, 1, 1, False, False),
    (20001, 9, 1, True, False, 1, 1, True, False), (4099, 260, 2, False, False, 1, 1, False, False),
], ids=lambda c: "-".join(str(int(x)) for x in c))
def test_route_backward_of_large_maps_and_long_batches(gpu, case):  # noqa: F811
    base.test_route_backward(gpu, *case, bf16=case[1] % 2 == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("t, n, k", [(20000, 32768, 3), (70000, 1600, 4), (3, 32768, 64)])
def test_balance_of_large_maps(gpu, t, n, k):  # noqa: F811
    rng = np.random.default_rng(t)
    neuron = (n * rng.random((t, k)) ** 3).astype(np.int32)
    neuron[rng.random((t, k)) < 0.1] = -1
    load = np.bincount(neuron[neuron >= 0], minlength=n)
    bias = rng.standard_normal(n).astype(np.float32)
    with capi.Readout(n, k) as ro:
        p, got = gpu.up(bias), gpu.new(n, np.int32)
        ro.balance(gpu.up(neuron), t, 0.01, p, got)
        ro.synchronize()
        assert np.array_equal(gpu.down(got, n, np.int32), load)
        assert np.array_equal(gpu.down(p, n, np.float32), bias + np.float32(0.01) * np.sign(load.sum() - load * n).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("t, n, k, f, h, o", [
    # rows sorted by one block, and by several, where a thread has several neurons; fewer waves to a block from 2048 neurons on
    (300, 1600, 2, 24, 16, 8), (3000, 1600, 2, 24, 16, 8), (300, 1024, 3, 8, 8, 8), (1400, 1025, 3, 9, 7, 5), (300, 5000, 2, 16, 8, 4), (1600, 5000, 2, 15, 9, 3),
    (100, 32768, 2, 3, 2, 2), (350, 32768, 2, 8, 8, 8),
])
def test_models_of_large_maps(gpu, t, n, k, f, h, o, bf16):  # noqa: F811
    def spread(rng, shape):                                # most on few neurons, the others anywhere; some places unused
        neuron = np.where(rng.random(shape) < 0.5, rng.integers(n - 3, n, shape), rng.integers(0, n, shape))
        return np.where(rng.random(shape) < 0.1, -1, neuron)

    base.test_experts(gpu, t, n, k, f, h, o, "silu", True, True, spread, 0, bf16)


@pytest.mark.gpu
def test_calls_of_more_threads_than_a_launch_has(gpu):  # noqa: F811
    buffer = gpu.new(4096, np.float32)
    with capi.Readout(3, 1) as ro, capi.Readout(3000, 1) as large:
        calls = [lambda: ro.route(buffer, 2 ** 28, buffer, buffer, None, buffer, buffer),
                 lambda: large.route(buffer, 2 ** 24, buffer, buffer, None, buffer, buffer),
                 lambda: ro.adamw(ro.tensors([dict(value=buffer, gradient=buffer, first=buffer, second=buffer, size=2 ** 36)]), 1)]
        for call in calls:
            with pytest.raises(capi.PinkError) as e:
                call()
            assert e.value.status == -1 and "too many" in str(e.value)
