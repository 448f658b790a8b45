"""The read-out of a trained map (pink_hip_readout_*): routing, the neurons' models and AdamW against plain restatements in
64 bits, through the C ABI.

Tolerances are bounds, computed next to each expected value from the roundings that the operators make: u is half a unit in the
last place of what is stored (2^-24 float32, 2^-8 bfloat16), s = 2^-24 that of the sums, a sum of K terms is off by at most
(K + 2) s times the sum of their magnitudes, and errors of an operand go through as the formulas say.
"""
import ctypes as C
import math

import numpy as np
import pytest

from pink_amd import capi

S = 2.0 ** -24
ACT = {"identity": capi.ACT_IDENTITY, "relu": capi.ACT_RELU, "gelu": capi.ACT_GELU, "silu": capi.ACT_SILU}


# ------------------------------------------------------------------------------------------------------------ refusals

@pytest.mark.parametrize("change, text", [
    (dict(neurons=0), "Number of neurons"), (dict(neurons=32769), "Number of neurons"),
    (dict(chosen=0), "Number of chosen neurons"), (dict(chosen=101), "Number of chosen neurons"), (dict(neurons=500, chosen=65), "Number of chosen neurons"),
    (dict(score=2), "unknown score"), (dict(groups=0), "Number of groups"), (dict(groups=101), "Number of groups"),
    (dict(neurons=10, groups=7), "group without neurons"), (dict(groups_kept=0), "kept groups"), (dict(groups=4, groups_kept=5), "kept groups"),
    (dict(activation=4), "unknown activation"), (dict(element=2), "unknown element"),
    (dict(features=8), "all zero or none"), (dict(features=8, hidden=8), "all zero or none"),
    (dict(features=8, hidden=2 ** 20 + 1, outputs=1), "at most 1048576"),
])
def test_configurations_that_are_refused(change, text):
    with pytest.raises(capi.PinkError) as e:
        capi.Readout.check(**{**dict(neurons=100, chosen=2), **change})
    assert e.value.status == -1 and text in str(e.value)


def test_configurations_that_are_taken():
    for good in (dict(neurons=1), dict(neurons=32768, chosen=64), dict(neurons=331, groups=21, groups_kept=4), dict(neurons=10, groups=5),
                 dict(neurons=3, chosen=3, features=1, hidden=1, outputs=1, element=capi.ELEMENT_BF16)):
        capi.Readout.check(**good)


# ------------------------------------------------------------------------------------------------------ device buffers

class Gpu:
    """Device memory and streams straight from the HIP runtime that the library runs on."""

    def __init__(self):
        capi.lib()
        self.rt = C.CDLL("libamdhip64.so.7")
        vp = C.c_void_p
        self.rt.hipMalloc.argtypes = [C.POINTER(vp), C.c_size_t]
        self.rt.hipMemcpy.argtypes = [vp, vp, C.c_size_t, C.c_int]
        self.rt.hipFree.argtypes = [vp]
        self.rt.hipStreamCreateWithFlags.argtypes = [C.POINTER(vp), C.c_uint]
        self.rt.hipStreamBeginCapture.argtypes = [vp, C.c_int]
        self.rt.hipStreamEndCapture.argtypes = [vp, C.POINTER(vp)]
        self.rt.hipGraphInstantiate.argtypes = [C.POINTER(vp), vp, vp, vp, C.c_size_t]
        self.rt.hipGraphLaunch.argtypes = [vp, vp]
        self.rt.hipGraphExecDestroy.argtypes = [vp]
        self.rt.hipGraphDestroy.argtypes = [vp]
        self.rt.hipStreamDestroy.argtypes = [vp]
        self.held = []

    def ok(self, rc):
        assert rc == 0, "HIP error %d" % rc

    def up(self, a):
        """A copy on the device, as an address; None stays None."""
        if a is None:
            return None
        a = np.ascontiguousarray(a)
        p = C.c_void_p()
        self.ok(self.rt.hipMalloc(C.byref(p), max(a.nbytes, 256)))
        if a.nbytes:
            self.ok(self.rt.hipMemcpy(p, a.ctypes.data, a.nbytes, 1))
        self.held.append(p)
        return p.value

    def new(self, shape, dtype):
        return self.up(np.full(shape, -77, np.int8).astype(dtype) if dtype != np.uint16 else np.full(shape, 0x7fc0, np.uint16))

    def write(self, p, a):
        a = np.ascontiguousarray(a)
        self.ok(self.rt.hipMemcpy(p, a.ctypes.data, a.nbytes, 1))

    def down(self, p, shape, dtype):
        out = np.empty(shape, dtype)
        if out.nbytes:
            self.ok(self.rt.hipMemcpy(out.ctypes.data, p, out.nbytes, 2))
        return out

    def release(self):
        for p in self.held:
            self.rt.hipFree(p)
        self.held = []


@pytest.fixture
def gpu():
    g = Gpu()
    yield g
    g.release()


def to_bf16(a):
    """float -> bfloat16 bits, nearest, ties to even."""
    bits = np.ascontiguousarray(a, np.float32).view(np.uint32)
    return ((bits + 0x7fff + ((bits >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


class Element:
    def __init__(self, bf16):
        self.id = capi.ELEMENT_BF16 if bf16 else capi.ELEMENT_F32
        self.bf16, self.u, self.dtype = bf16, 2.0 ** -8 if bf16 else S, np.uint16 if bf16 else np.float32

    def store(self, a):
        """(what goes to the device, what it stands for in 64 bits)"""
        if a is None:
            return None, None
        b = to_bf16(a) if self.bf16 else np.ascontiguousarray(a, np.float32)
        return b, self.values(b)

    def values(self, b):
        return (from_bf16(b) if self.bf16 else b).astype(np.float64)


def assert_within(got, want, bound, what):
    off = np.abs(got - want)
    assert np.all(np.isfinite(got)), what + ": not finite"
    worst = np.unravel_index(np.argmax(off - bound), off.shape) if off.size else None
    assert worst is None or off[worst] <= bound[worst], "%s: off by %g at %s, bound %g" % (what, off[worst], worst, bound[worst])


# ------------------------------------------------------------------------------------------------------------- routing

def route_reference(d, a, r, b, k, sigmoid, renormalise, groups, kept):
    """One image after the other, from the definition: 32-bit logits decide, the rest is in 64 bits."""
    t, n = d.shape
    size = -(-n // groups)
    neuron, gates = np.full((t, k), -1, np.int32), np.zeros((t, k))
    with np.errstate(all="ignore"):
        z = (a * (r - d)).astype(np.float32)
        key = z if b is None else (z + b).astype(np.float32)
    part = np.isfinite(z) & np.isfinite(key)
    for i in range(t):
        in_play = [int(m) for m in range(n) if part[i, m]]
        scores = []
        for g in range(groups):
            best = sorted((key[i, m] for m in in_play if m // size == g), reverse=True)[:2]
            with np.errstate(over="ignore"):
                scores.append(-math.inf if not best else best[0] if len(best) == 1 else np.float32(best[0] + best[1]))
        keep = sorted(range(groups), key=lambda g: (-scores[g], g))[:kept]
        order = sorted((m for m in in_play if m // size in keep), key=lambda m: (-key[i, m], m))[:k]
        if not order:
            continue
        zi = z[i].astype(np.float64)
        level = [-np.logaddexp(0, -zi[m]) if sigmoid else zi[m] for m in order]
        if renormalise:
            e = np.exp(np.array(level) - max(level))
            g = e / e.sum()
        elif sigmoid:
            g = np.exp(level)
        else:
            top = max(zi[m] for m in in_play)
            g = np.exp(np.array(level) - top) / sum(math.exp(zi[m] - top) for m in in_play)
        neuron[i, :len(order)], gates[i, :len(order)] = order, g
    return neuron, gates, z, part


def route_inputs(rng, t, n, ties=False):
    d = (6 + 2 * rng.random((t, 1)) + rng.standard_normal((t, n))).astype(np.float32)
    if ties:
        d = np.round(d)                                    # many equal distances
    d[:, rng.random(n) < 0.1] = np.inf
    d[rng.random((t, n)) < 0.02] = np.nan
    if t > 2:
        d[1] = np.inf                                      # nothing left
        d[2] = np.inf
        d[2, n // 2] = 5.0                                 # one neuron left
    a, r = (1.5 + 0.5 * rng.random(n)).astype(np.float32), (5 + 0.5 * rng.standard_normal(n)).astype(np.float32)
    if ties:
        a[:], r[:] = 1.5, 5.0
    return d, a, r


ROUTES = [  # images, neurons, chosen, sigmoid, renormalise, groups, kept, bias, ties
    (1, 1, 1, False, True, 1, 1, False, False), (1, 100, 2, False, True, 1, 1, False, False), (5, 64, 64, True, False, 1, 1, True, False),
    (9, 331, 4, False, False, 1, 1, True, False), (9, 331, 5, False, False, 21, 3, True, False), (4, 1600, 8, True, True, 40, 8, True, False),
    (7, 100, 6, True, True, 10, 2, False, True), (3, 65, 3, False, True, 13, 13, True, True), (6, 10, 3, False, False, 5, 1, False, True),
    (3, 2049, 9, False, False, 98, 7, True, False), (2, 5000, 64, True, True, 1, 1, False, True), (130, 37, 2, True, False, 37, 5, True, False),
    (3, 2048, 33, False, True, 1024, 40, True, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("t, n, k, sigmoid, renormalise, groups, kept, bias, ties", ROUTES)
def test_route(gpu, t, n, k, sigmoid, renormalise, groups, kept, bias, ties):
    rng = np.random.default_rng(t * 7919 + n)
    d, a, r = route_inputs(rng, t, n, ties)
    b = (rng.integers(-1, 2, n) if ties else 0.3 * rng.standard_normal(n)).astype(np.float32) if bias else None
    want_n, want_g, z, part = route_reference(d, a, r, b, k, sigmoid, renormalise, groups, kept)
    wide = np.full((t, n + 5), 1.0, np.float32)
    wide[:, :n] = d
    with capi.Readout(n, k, score=int(sigmoid), renormalise=renormalise, groups=groups, groups_kept=kept) as ro:
        for rows, stride in ((d, 0), (wide, n + 5)):
            out_n, out_g = gpu.new((t, k), np.int32), gpu.new((t, k), np.float32)
            ro.route(gpu.up(rows), t, gpu.up(a), gpu.up(r), gpu.up(b), out_n, out_g, distance_stride=stride)
            ro.synchronize()
            assert np.array_equal(gpu.down(out_n, (t, k), np.int32), want_n)
            got = gpu.down(out_g, (t, k), np.float32).astype(np.float64)
            # a gate's exponent is a difference of two levels of at most `span`, rounded; exp, log and the sum add some units
            span = 2 * (np.abs(z[part]).max() if part.any() else 0)
            assert_within(got, want_g, want_g * S * (2 * span + n / 8 + 32) + 1e-38, "gates")


@pytest.mark.gpu
@pytest.mark.parametrize("score, renormalise", [(0, True), (0, False), (1, True), (1, False)])
def test_route_of_extreme_distances(gpu, score, renormalise):
    # the type's largest values as masks, overflow to infinity, minus zero against zero, levels that underflow one by one
    big = np.float32(3.4028235e38)
    d = np.array([[big, big, big, big], [1, big, np.inf, -np.inf], [200, 201, 1000, big], [0.0, -0.0, 0.0, -0.0], [-big, 0, big, np.nan]], np.float32)
    a, r = np.ones(4, np.float32), np.zeros(4, np.float32)
    want_n, want_g, z, part = route_reference(d, a, r, None, 3, bool(score), renormalise, 1, 1)
    with capi.Readout(4, 3, score=score, renormalise=renormalise) as ro:
        out_n, out_g = gpu.new((5, 3), np.int32), gpu.new((5, 3), np.float32)
        ro.route(gpu.up(d), 5, gpu.up(a), gpu.up(r), None, out_n, out_g)
        ro.synchronize()
        assert np.array_equal(gpu.down(out_n, (5, 3), np.int32), want_n)
        got = gpu.down(out_g, (5, 3), np.float32).astype(np.float64)
        assert_within(got, want_g, want_g * S * 2000 + 1e-38, "gates")       # exponents up to 1000 that count


def route_gradients(d, a, r, neuron, gates, grad, z, part, sigmoid, renormalise):
    """(dz of every entry, sum of the magnitudes that went into it), in 64 bits."""
    t, n = d.shape
    dz, size = np.zeros((t, n)), np.zeros((t, n))
    for i in range(t):
        at = [int(m) for m in neuron[i] if m >= 0]
        if not at:
            continue
        g, w = grad[i, :len(at)].astype(np.float64), gates[i, :len(at)]
        zi = z[i].astype(np.float64)
        pull, weight = (w * g).sum(), (w * np.abs(g)).sum()
        below = 1 / (1 + np.exp(np.minimum(zi[at], 700)))
        if renormalise:
            dz[i, at], size[i, at] = w * (g - pull) * (below if sigmoid else 1), w * (np.abs(g) + weight)
        elif sigmoid:
            dz[i, at], size[i, at] = w * g * below, w * np.abs(g)
        else:
            play = np.flatnonzero(part[i])
            e = np.exp(zi[play] - zi[play].max())
            share = e / e.sum()
            dz[i, play], size[i, play] = -share * pull, share * weight
            dz[i, at] += w * g
            size[i, at] += w * np.abs(g)
    return dz, size


@pytest.mark.gpu
@pytest.mark.parametrize("t, n, k, sigmoid, renormalise, groups, kept, bias, ties", [r for r in ROUTES if r[0] * r[1] < 20000] + [
    (700, 21, 3, False, False, 1, 1, False, False), (2100, 9, 2, True, True, 1, 1, True, False)])
@pytest.mark.parametrize("bf16", [False, True])
def test_route_backward(gpu, t, n, k, sigmoid, renormalise, groups, kept, bias, ties, bf16):
    rng = np.random.default_rng(t * 31 + n)
    element = Element(bf16)
    d, a, r = route_inputs(rng, t, n, ties)
    b = (0.3 * rng.standard_normal(n)).astype(np.float32) if bias else None
    neuron, gates, z, part = route_reference(d, a, r, b, k, sigmoid, renormalise, groups, kept)
    gates32 = gates.astype(np.float32)
    stored, grad = element.store(rng.standard_normal((t, k)))
    dz, size = route_gradients(d, a, r, neuron, gates, grad, z, part, sigmoid, renormalise)
    a64, gap = a.astype(np.float64), np.where(part, r.astype(np.float64) - d, 0.0)
    span = 2 * np.abs(z[part]).max() if part.any() else 0
    off = size * S * (2 * span + n / 8 + k + 40)
    with capi.Readout(n, k, score=int(sigmoid), renormalise=renormalise, groups=groups, groups_kept=kept, element=element.id) as ro:
        dd, da, dr = gpu.new((t, n), np.float32), gpu.new(n, np.float32), gpu.new(n, np.float32)
        args = (gpu.up(d), t, gpu.up(a), gpu.up(r), gpu.up(b), gpu.up(neuron), gpu.up(gates32), gpu.up(stored))
        ro.route_backward(*args, dd, da, dr)
        ro.synchronize()
        got = gpu.down(dd, (t, n), np.float32)
        assert_within(got.astype(np.float64), -a64 * dz, a64 * (off + 2 * S * np.abs(dz)) + 1e-37, "of distances")
        sums = [gpu.down(p, n, np.float32) for p in (da, dr)]
        assert_within(sums[0].astype(np.float64), (dz * gap).sum(0), (np.abs(gap) * (off + (t + 4) * S * np.abs(dz))).sum(0) + 1e-37, "of sharpness")
        assert_within(sums[1].astype(np.float64), (dz * a64).sum(0), (a64 * (off + (t + 4) * S * np.abs(dz))).sum(0) + 1e-37, "of radius")
        # the sums alone, and each output alone, are the same bits
        again = [gpu.new(n, np.float32), gpu.new(n, np.float32), gpu.new((t, n), np.float32)]
        ro.route_backward(*args, None, again[0], None)
        ro.route_backward(*args, None, None, again[1])
        ro.route_backward(*args, again[2], None, None)
        ro.synchronize()
        assert np.array_equal(gpu.down(again[0], n, np.float32), sums[0]) and np.array_equal(gpu.down(again[1], n, np.float32), sums[1])
        assert np.array_equal(gpu.down(again[2], (t, n), np.float32), got)


@pytest.mark.gpu
@pytest.mark.parametrize("sigmoid, renormalise", [(False, True), (False, False), (True, True), (True, False)])
def test_route_gradients_against_differences(gpu, sigmoid, renormalise):
    # central differences of a weighted sum of the 64-bit gates along random directions; the choice stays as it is
    rng = np.random.default_rng(5)
    t, n, k = 6, 30, 4
    d, a, r = (6 + rng.standard_normal((t, n))).astype(np.float32), np.full(n, 1.25, np.float32), (5 + rng.random(n)).astype(np.float32)
    neuron, gates, z, part = route_reference(d, a, r, None, k, sigmoid, renormalise, 1, 1)
    grad = rng.standard_normal((t, k)).astype(np.float32)

    def loss(d, a, r):
        z = a * (r - d)
        zc = np.take_along_axis(z, neuron, 1)
        if renormalise:
            level = -np.logaddexp(0, -zc) if sigmoid else zc
            g = np.exp(level) / np.exp(level).sum(1, keepdims=True)
        else:
            g = 1 / (1 + np.exp(-zc)) if sigmoid else np.exp(zc) / np.exp(z).sum(1, keepdims=True)
        return (g * grad).sum()

    with capi.Readout(n, k, score=int(sigmoid), renormalise=renormalise) as ro:
        dd, da, dr = gpu.new((t, n), np.float32), gpu.new(n, np.float32), gpu.new(n, np.float32)
        ro.route_backward(gpu.up(d), t, gpu.up(a), gpu.up(r), None, gpu.up(neuron), gpu.up(gates.astype(np.float32)), gpu.up(grad), dd, da, dr)
        ro.synchronize()
        got = [gpu.down(dd, (t, n), np.float32), gpu.down(da, n, np.float32), gpu.down(dr, n, np.float32)]
    at = [v.astype(np.float64) for v in (d, a, r)]
    for i in range(3):
        v, h = rng.standard_normal(at[i].shape), 1e-4
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * v, at[i] - h * v
        slope = (loss(*up) - loss(*down)) / (2 * h)
        # h^2 times third derivatives of order |v|^3 (about 10 of size |grad|), and float32 gradients
        assert abs((got[i] * v).sum() - slope) < 1e-4 * (1 + np.abs(got[i] * v).sum())


@pytest.mark.gpu
def test_balance(gpu):
    rng = np.random.default_rng(3)
    for t, n, k in ((1, 1, 1), (500, 37, 3), (4, 2000, 8), (0, 5, 2)):
        neuron = rng.integers(-1, n + 1, (t, k)).astype(np.int32)          # -1 and n are no neurons
        load = np.bincount(neuron[(neuron >= 0) & (neuron < n)], minlength=n)
        bias = rng.standard_normal(n).astype(np.float32)
        want = bias + np.float32(0.01) * np.sign(load.sum() - load * n).astype(np.float32)
        with capi.Readout(n, min(k, n)) as ro:
            if k > n:
                neuron = neuron[:, :n].copy()
            p, l = gpu.up(bias), gpu.new(n, np.int32)
            ro.balance(gpu.up(neuron), t, 0.01, p, l)
            ro.synchronize()
            assert np.array_equal(gpu.down(l, n, np.int32), load) and np.array_equal(gpu.down(p, n, np.float32), want)


# -------------------------------------------------------------------------------------------------------------- models

def f_and_slope(kind, a):
    if kind == "identity":
        return a, np.ones_like(a)
    if kind == "relu":
        return np.maximum(a, 0), (a > 0).astype(np.float64)
    if kind == "gelu":
        e = np.vectorize(math.erf)(a * math.sqrt(0.5)) if a.size else a
        return 0.5 * a * (1 + e), 0.5 * (1 + e) + a * np.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    s = 1 / (1 + np.exp(-a))
    return a * s, s * (1 + a * (1 - s))


STEEP, BENT = {"identity": 1, "relu": 1, "gelu": 1.13, "silu": 1.1}, {"identity": 0, "relu": 0, "gelu": 0.8, "silu": 0.5}


def experts_reference(m, element, act, neuron, gates, dy):
    """{name: (value, bound)} of the answer and all gradients, one neuron after the other, in 64 bits; `m` holds x, w1, b1, w2, b2, residual."""
    x, w1, b1, w2, b2 = (m[i] for i in ("x", "w1", "b1", "w2", "b2"))
    (t, k), (n, h, f), o, u = neuron.shape, w1.shape, w2.shape[1], element.u
    out = {i: [np.zeros(s), np.zeros(s)] for i, s in dict(y=(t, o), dx=(t, f), dgates=(t, k), dw1=w1.shape, db1=(n, h), dw2=w2.shape, db2=(n, o)).items()}
    size_y, size_x = np.zeros((t, o)), np.zeros((t, f))
    for e in range(n):
        img, slot = np.nonzero(neuron == e)
        if not len(img):
            continue
        xe, g = x[img], gates[img, slot].astype(np.float64)[:, None]
        c1, c2 = (b1[e] if b1 is not None else np.zeros(h)), (b2[e] if b2 is not None else np.zeros(o))
        a = xe @ w1[e].T + c1
        off_a = (f + 2) * S * (np.abs(xe) @ np.abs(w1[e]).T + np.abs(c1))
        v, slope = f_and_slope(act, a)
        off_v = STEEP[act] * off_a + 8 * S * (np.abs(a) + np.abs(v))
        after = g * v
        off_after = np.abs(g) * off_v + (u + S) * np.abs(after) * 1.01
        answer, mag = after @ w2[e].T + g * c2, np.abs(after) @ np.abs(w2[e]).T + np.abs(g * c2)
        off = off_after @ np.abs(w2[e]).T + (h + 3) * S * mag
        np.add.at(out["y"][0], img, answer)
        np.add.at(out["y"][1], img, off)
        np.add.at(size_y, img, np.abs(answer))
        if dy is None:
            continue
        dye = dy[img]
        back, off_back = dye @ w2[e], (o + 2) * S * (np.abs(dye) @ np.abs(w2[e]))
        off_b = off_a + u * np.abs(a) * 1.01               # the value before the activation as it is kept
        off_v = STEEP[act] * off_b + 8 * S * (np.abs(a) + np.abs(v))
        off_slope = BENT[act] * off_b + (8 * S * (1 + np.abs(a)) if act in ("gelu", "silu") else 0)
        if act == "relu":
            off_slope = off_slope + (np.abs(a) <= off_b)   # on which side of the kink is open there
        dg = (back * v).sum(1) + dye @ c2
        out["dgates"][0][img, slot] = dg
        out["dgates"][1][img, slot] = (off_back * (np.abs(v) + off_v) + np.abs(back) * off_v).sum(1) + (h + o + 8) * S * (
            (np.abs(back * v)).sum(1) + np.abs(dye) @ np.abs(c2)) + u * np.abs(dg) * 1.01
        da = g * back * slope
        off_da = np.abs(g) * (off_back * (np.abs(slope) + off_slope) + np.abs(back) * off_slope) + (u + 2 * S) * np.abs(da) * 1.01
        dx, mag = da @ w1[e], np.abs(da) @ np.abs(w1[e])
        np.add.at(out["dx"][0], img, dx)
        np.add.at(out["dx"][1], img, off_da @ np.abs(w1[e]) + (h + 3) * S * mag)
        np.add.at(size_x, img, np.abs(dx))
        sums = (len(img) + 3) * S
        for name, left, right, off in (("dw1", da, xe, off_da.T @ np.abs(xe)), ("dw2", dye, after, np.abs(dye).T @ off_after)):
            out[name][0][e] = left.T @ right
            out[name][1][e] = off + sums * (np.abs(left).T @ np.abs(right))
        out["db1"][0][e], out["db1"][1][e] = da.sum(0), off_da.sum(0) + sums * np.abs(da).sum(0)
        gdy = g * dye
        out["db2"][0][e], out["db2"][1][e] = gdy.sum(0), (sums + (2.0 ** -16 if element.bf16 else 0)) * np.abs(gdy).sum(0)
    if m["residual"] is not None:
        out["y"][0] += m["residual"]
        size_y += np.abs(m["residual"])
    out["y"][1] += (k + 2) * S * size_y
    out["dx"][1] += (k + 2) * S * size_x
    for name, (value, bound) in out.items():
        bound += u * np.abs(value) * 1.02 + u * bound
    return out


def experts_inputs(rng, element, t, n, k, f, h, o, bias=True, residual=False, spread=None):
    draw = {"x": rng.standard_normal((t, f)), "w1": rng.standard_normal((n, h, f)) * 1.5 / math.sqrt(f),
            "b1": 0.3 * rng.standard_normal((n, h)) if bias else None, "w2": rng.standard_normal((n, o, h)) * 1.5 / math.sqrt(h),
            "b2": 0.3 * rng.standard_normal((n, o)) if bias else None, "residual": rng.standard_normal((t, o)) if residual else None}
    stored, value = {}, {}
    for name, v in draw.items():
        stored[name], value[name] = element.store(v)
    neuron = (rng.integers(0, n, (t, k)) if spread is None else spread(rng, (t, k))).astype(np.int32)
    return stored, value, neuron, rng.random((t, k)).astype(np.float32)


def some_unused(rng, shape):
    # a neuron that does not exist, of either sign, in a third of the places; the third image has none
    neuron = np.where(rng.random(shape) < 0.2, -1, rng.integers(0, 5, shape))
    neuron = np.where(rng.random(shape) < 0.1, 5, neuron)
    neuron[2 % shape[0]] = -1
    return neuron


def all_on_one(rng, shape):
    return np.full(shape, 3)


def none_at_all(rng, shape):
    return np.full(shape, -1)


MODELS = [  # images, neurons, chosen, features, hidden, outputs, activation, bias, residual, spread, padding of rows
    (1, 1, 1, 1, 1, 1, "identity", True, False, None, 0),
    (1, 100, 2, 64, 32, 16, "gelu", True, False, None, 0),
    (2, 7, 4, 45, 19, 5, "silu", True, True, None, 3),
    (9, 5, 2, 129, 65, 33, "relu", False, True, some_unused, 1),
    (65, 5, 3, 200, 72, 10, "gelu", True, True, some_unused, 8),
    (130, 5, 1, 48, 136, 129, "silu", True, False, some_unused, 0),
    (300, 5, 1, 31, 24, 40, "relu", True, False, all_on_one, 0),
    (40, 12, 2, 128, 256, 64, "identity", True, True, None, 0),
    (5, 5, 2, 33, 17, 9, "gelu", True, True, none_at_all, 2),
    (333, 9, 4, 96, 40, 24, "gelu", True, True, None, 4),
    (17, 300, 3, 72, 144, 200, "silu", True, False, None, 0),
    # tiles of every size, each with whole chunks and without: rows a neuron 12, 40, 100, 350; more rows than are looked up at a time
    (60, 10, 2, 64, 40, 48, "silu", True, True, None, 0),
    (60, 10, 2, 61, 41, 47, "silu", True, True, None, 0),
    (200, 5, 1, 264, 72, 136, "silu", True, False, None, 0),
    (200, 5, 1, 263, 71, 135, "silu", True, False, None, 1),
    (300, 6, 2, 520, 136, 72, "silu", False, False, None, 0),
    (300, 6, 2, 519, 137, 73, "silu", False, False, None, 0),
    (700, 2, 1, 136, 264, 520, "silu", True, True, None, 0),
    (700, 2, 1, 135, 263, 519, "silu", True, True, None, 3),
    (5000, 1, 1, 40, 24, 16, "gelu", True, False, None, 0),
    (4300, 2, 2, 39, 23, 17, "relu", True, False, None, 0),
    # few hidden values or outputs: narrow tiles
    (200, 5, 1, 264, 16, 8, "gelu", True, False, None, 0),
    (200, 5, 1, 263, 17, 3, "gelu", True, True, None, 1),
    (300, 6, 2, 136, 24, 32, "silu", True, False, None, 0),
    (300, 6, 2, 137, 15, 10, "silu", True, False, None, 0),
    (700, 2, 1, 136, 32, 16, "silu", True, True, None, 0),
    (700, 2, 1, 135, 31, 1, "silu", True, True, None, 0),
    # so many neurons that gradients of weights take the largest tiles
    (8400, 256, 2, 264, 264, 16, "silu", True, False, None, 0),
]


def padded(a, pad, fill):
    """Rows `pad` elements further apart, with `fill` between them."""
    out = np.full((a.shape[0], a.shape[1] + pad), fill, a.dtype)
    out[:, :a.shape[1]] = a
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("t, n, k, f, h, o, act, bias, residual, spread, pad", MODELS)
def test_experts(gpu, t, n, k, f, h, o, act, bias, residual, spread, pad, bf16):
    rng = np.random.default_rng(t * 131 + f)
    element = Element(bf16)
    stored, value, neuron, gates = experts_inputs(rng, element, t, n, k, f, h, o, bias, residual, spread)
    nan = 0x7fc0 if bf16 else np.nan
    dy_stored, dy = element.store(rng.standard_normal((t, o)))
    unused = (neuron < 0) | (neuron >= n)
    gates[unused] = np.nan                                 # what lies in unused places must not matter
    want = experts_reference(value, element, act, np.where(unused, -1, neuron), np.where(unused, 0, gates), dy)
    x = stored["x"].copy()
    x[unused.all(1)] = nan                                 # nor what an image without a neuron holds, its residual aside
    p = {i: gpu.up(v) for i, v in stored.items()}
    p["x"], weights = gpu.up(padded(x, pad, nan)), [p[i] for i in ("w1", "b1", "w2", "b2")]
    p["residual"] = gpu.up(padded(stored["residual"], pad, nan)) if residual else None
    where = gpu.up(neuron), gpu.up(gates)
    names = dict(dx=(t, f), dgates=(t, k), dw1=(n, h, f), db1=(n, h), dw2=(n, o, h), db2=(n, o))
    with capi.Readout(n, k, f, h, o, activation=ACT[act], element=element.id) as ro:
        saved = gpu.new(ro.saved_bytes(t), np.int8)
        answers = []
        for keep in (None, None, saved, saved):
            y = gpu.new((t, o + pad), element.dtype)
            ro.experts(p["x"], t, *where, weights, y, dev_residual=p["residual"], dev_saved=keep, x_stride=f + pad, residual_stride=o + pad, y_stride=o + pad)
            ro.synchronize()
            answers.append(gpu.down(y, (t, o + pad), element.dtype)[:, :o])
            assert_within(element.values(answers[-1]), *want["y"], "y")
        # the same call gives the same bits (few images are summed in another order when nothing is kept for a backward pass)
        assert np.array_equal(answers[0], answers[1]) and np.array_equal(answers[2], answers[3])
        grads = {i: gpu.new(s if i != "dx" else (t, f + pad), element.dtype) for i, s in names.items()}
        dy_dev = gpu.up(padded(dy_stored, pad, nan))
        for _ in range(2):                                 # twice: the same bits
            ro.experts_backward(p["x"], t, where[1], weights, saved, dy_dev, [grads[i] for i in names], x_stride=f + pad, y_gradient_stride=o + pad,
                                x_gradient_stride=f + pad)
            ro.synchronize()
            got = {i: gpu.down(grads[i], s if i != "dx" else (t, f + pad), element.dtype) for i, s in names.items()}
            got["dx"] = got["dx"][:, :f]
            first = got if _ == 0 else first
            for i in names:
                assert np.array_equal(got[i], first[i])
                assert_within(element.values(got[i]), *want[i], i)
        for i in names:                                    # each gradient alone: the same bits
            alone = gpu.new(names[i], element.dtype)
            ro.experts_backward(p["x"], t, where[1], weights, saved, dy_dev, [alone if j == i else None for j in names], x_stride=f + pad,
                                y_gradient_stride=o + pad)
            ro.synchronize()
            assert np.array_equal(gpu.down(alone, names[i], element.dtype), got[i]), i


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["identity", "gelu", "silu"])
def test_experts_gradients_against_differences(gpu, act):
    rng = np.random.default_rng(17)
    element = Element(False)
    t, n, k, f, h, o = 12, 4, 2, 10, 9, 7
    stored, value, neuron, gates = experts_inputs(rng, element, t, n, k, f, h, o)
    dy_stored, dy = element.store(rng.standard_normal((t, o)))

    def loss(x, gates, w1, b1, w2, b2):
        total = 0.0
        for i in range(t):
            for s in range(k):
                e = neuron[i, s]
                total += gates[i, s] * dy[i] @ (w2[e] @ f_and_slope(act, w1[e] @ x[i] + b1[e])[0] + b2[e])
        return total

    at = [value["x"], gates.astype(np.float64), value["w1"], value["b1"], value["w2"], value["b2"]]
    with capi.Readout(n, k, f, h, o, activation=ACT[act], element=element.id) as ro:
        p = {i: gpu.up(v) for i, v in stored.items()}
        weights, saved, y = [p[i] for i in ("w1", "b1", "w2", "b2")], gpu.new(ro.saved_bytes(t), np.int8), gpu.new((t, o), np.float32)
        ro.experts(p["x"], t, gpu.up(neuron), gpu.up(gates), weights, y, dev_saved=saved)
        grads = [gpu.new(v.shape, np.float32) for v in at]
        ro.experts_backward(p["x"], t, gpu.up(gates), weights, saved, gpu.up(dy_stored), grads)
        ro.synchronize()
        got = [gpu.down(q, v.shape, np.float32).astype(np.float64) for q, v in zip(grads, at)]
    for i, v in enumerate(at):
        direction, step = rng.standard_normal(v.shape), 1e-5
        up, down = list(at), list(at)
        up[i], down[i] = v + step * direction, v - step * direction
        slope = (loss(*up) - loss(*down)) / (2 * step)
        # differences: step^2 times third derivatives; gradients: some hundred roundings of 2^-24
        assert abs((got[i] * direction).sum() - slope) < 2e-5 * np.abs(got[i] * direction).sum() + 1e-6


@pytest.mark.gpu
def test_experts_adds_to_its_residual_in_place(gpu):
    rng = np.random.default_rng(2)
    element = Element(True)
    stored, value, neuron, gates = experts_inputs(rng, element, 20, 6, 2, 24, 16, 24, residual=True)
    with capi.Readout(6, 2, 24, 16, 24, element=element.id) as ro:
        p = {i: gpu.up(v) for i, v in stored.items()}
        weights, y, inplace = [p[i] for i in ("w1", "b1", "w2", "b2")], gpu.new((20, 24), np.uint16), gpu.up(stored["residual"])
        where = gpu.up(neuron), gpu.up(gates)
        ro.experts(p["x"], 20, *where, weights, y, dev_residual=p["residual"])
        ro.experts(p["x"], 20, *where, weights, inplace, dev_residual=inplace)
        ro.synchronize()
        assert np.array_equal(gpu.down(y, (20, 24), np.uint16), gpu.down(inplace, (20, 24), np.uint16))


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("t, h, f", [(20, 33, 64), (90, 33, 128), (300, 42, 256), (700, 9, 136)])
def test_experts_read_nothing_that_they_did_not_write(gpu, t, h, f, bf16):
    """Workspace and saved rows are padded; what lies there, NaN from a larger call before, takes part in nothing."""
    rng = np.random.default_rng(t)
    element, n, k, o = Element(bf16), 2, 1, 16
    stored, value, neuron, gates = experts_inputs(rng, element, t, n, k, f, h, o)
    dy_stored, dy = element.store(rng.standard_normal((t, o)))
    want = experts_reference(value, element, "silu", neuron, gates, dy)
    nan = 0x7fc0 if bf16 else np.nan
    names = dict(dx=(t, f), dgates=(t, k), dw1=(n, h, f), db1=(n, h), dw2=(n, o, h), db2=(n, o))
    with capi.Readout(n, k, f, h, o, activation=capi.ACT_SILU, element=element.id) as ro, \
            capi.Readout(n, 2, f, h, o, activation=capi.ACT_SILU, element=element.id) as before:
        p = {i: gpu.up(v) for i, v in stored.items()}
        weights = [p[i] for i in ("w1", "b1", "w2", "b2")]
        ro.reserve(8 * t)
        big = 8 * t                                        # two slots' rows of NaN each, wherever this handle puts them
        for handle, c in ((ro, 1), (before, 2)):
            where = gpu.up(np.tile(np.arange(n, dtype=np.int32), big * c)[:big * c]), gpu.up(np.ones(big * c, np.float32))
            x_nan, dy_nan = gpu.up(np.full((big, f), nan, element.dtype)), gpu.up(np.full((big, o), nan, element.dtype))
            junk = [gpu.new(s, element.dtype) for s in ((big, f), (big, c), (n, h, f), (n, h), (n, o, h), (n, o))]
            keep = gpu.new(handle.saved_bytes(big), np.int8)
            handle.experts(x_nan, big, *where, weights, gpu.new((big, o), element.dtype), dev_saved=keep)
            handle.experts(x_nan, big, *where, weights, gpu.new((big, o), element.dtype))
            handle.experts_backward(x_nan, big, where[1], weights, keep, dy_nan, junk)
        saved = gpu.up(np.full(ro.saved_bytes(t) // 2, 0x7fff, np.uint16))     # NaN in either type
        y, grads, where = gpu.new((t, o), element.dtype), {i: gpu.new(s, element.dtype) for i, s in names.items()}, (gpu.up(neuron), gpu.up(gates))
        ro.experts(p["x"], t, *where, weights, y, dev_saved=saved)
        ro.experts_backward(p["x"], t, where[1], weights, saved, gpu.up(dy_stored), [grads[i] for i in names])
        ro.synchronize()
        assert_within(element.values(gpu.down(y, (t, o), element.dtype)), *want["y"], "y")
        for i, s in names.items():
            assert_within(element.values(gpu.down(grads[i], s, element.dtype)), *want[i], i)


@pytest.mark.gpu
def test_no_images(gpu):
    with capi.Readout(5, 2, 8, 4, 3) as ro:
        weights = [gpu.new(60, np.float32)] * 4
        ro.route(None, 0, None, None, None, None, None)
        ro.experts(None, 0, None, None, weights, None)
        shapes = [(5, 4, 8), (5, 4), (5, 3, 4), (5, 3)]
        grads = [gpu.new(s, np.float32) for s in shapes]
        da, dr = gpu.new(5, np.float32), gpu.new(5, np.float32)
        ro.experts_backward(None, 0, None, weights, None, None, [None, None] + grads)
        ro.route_backward(None, 0, None, None, None, None, None, None, None, da, dr)
        ro.synchronize()
        for p, s in zip(grads + [da, dr], shapes + [5, 5]):
            assert not gpu.down(p, s, np.float32).any()


@pytest.mark.gpu
def test_calls_that_are_refused(gpu):
    buffer = gpu.new(1024, np.float32)
    with capi.Readout(5, 2) as ro:
        for call in (lambda: ro.route(None, 1, buffer, buffer, None, buffer, buffer), lambda: ro.route(buffer, 1, buffer, buffer, None, None, buffer),
                     lambda: ro.route(buffer, 1, buffer, buffer, None, buffer, buffer, distance_stride=4),
                     lambda: ro.route(buffer, 2 ** 31 - 1, buffer, buffer, None, buffer, buffer),
                     lambda: ro.route_backward(buffer, 1, buffer, buffer, None, buffer, buffer, None, buffer),
                     lambda: ro.balance(None, 1, 0.1, buffer), lambda: ro.balance(buffer, 1, 0.1, None)):
            with pytest.raises(capi.PinkError) as e:
                call()
            assert e.value.status == -1 and str(e.value)
        with pytest.raises(capi.PinkError) as e:
            ro.experts(buffer, 1, buffer, buffer, [buffer] * 4, buffer)
        assert e.value.status == -4 and ro.saved_bytes(1) == 0
        one = dict(value=buffer, gradient=buffer, first=buffer, second=buffer, size=16)
        for tensors, step, options in (([one], 0, {}), ([one], 1, dict(bits=16)), ([one], 1, dict(bits=8)), ([one], 1, dict(epsilon=0.0)),
                                       ([one], 1, dict(beta_first=1.0)), ([one], 1, dict(beta_second=-0.1)), ([dict(one, first=None)], 1, {})):
            with pytest.raises(capi.PinkError) as e:
                ro.adamw(ro.tensors(tensors), step, **options)
            assert e.value.status == -1
    with capi.Readout(5, 2, 8, 4, 3) as ro:
        for change in (dict(x=None), dict(y=None), dict(weights=[None] + [buffer] * 3), dict(x_stride=7), dict(y_stride=2), dict(saved=buffer + 4)):
            c = {**dict(x=buffer, y=buffer, weights=[buffer] * 4, x_stride=0, y_stride=0, saved=None), **change}
            with pytest.raises(capi.PinkError) as e:
                ro.experts(c["x"], 1, buffer, buffer, c["weights"], c["y"], dev_saved=c["saved"], x_stride=c["x_stride"], y_stride=c["y_stride"])
            assert e.value.status == -1
            if "y" not in change:
                with pytest.raises(capi.PinkError):
                    ro.experts_backward(c["x"], 1, buffer, c["weights"], c["saved"], buffer, [buffer] * 6, x_stride=c["x_stride"],
                                        y_gradient_stride=c["y_stride"])
    with pytest.raises(capi.PinkError):
        capi.Readout(5, 6)


@pytest.mark.gpu
def test_graph_on_a_given_stream(gpu):
    """Router and models, forward and backward, recorded once and replayed on new inputs with other work between the replays."""
    rng = np.random.default_rng(11)
    element, t, n, k, f, h, o = Element(True), 70, 30, 3, 40, 24, 16
    stored, value, neuron, gates = experts_inputs(rng, element, t, n, k, f, h, o)
    stream, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    gpu.ok(gpu.rt.hipStreamCreateWithFlags(C.byref(stream), 1))
    with capi.Readout(n, k, f, h, o, element=element.id) as ro:
        p = {i: gpu.up(v) for i, v in stored.items()}
        weights, d = [p[i] for i in ("w1", "b1", "w2", "b2")], gpu.new((t, n), np.float32)
        a, r = gpu.up(np.ones(n, np.float32)), gpu.up(np.full(n, 5, np.float32))
        at, g, y, saved = gpu.new((t, k), np.int32), gpu.new((t, k), np.float32), gpu.new((t, o), np.uint16), gpu.new(ro.saved_bytes(t), np.int8)
        shapes = dict(dx=(t, f), dgates=(t, k), dw1=(n, h, f), db1=(n, h), dw2=(n, o, h), db2=(n, o))
        grads = {i: gpu.new(s, np.uint16) for i, s in shapes.items()}
        dd, da, dr = gpu.new((t, n), np.float32), gpu.new(n, np.float32), gpu.new(n, np.float32)

        def calls():
            ro.route(d, t, a, r, None, at, g)
            ro.experts(p["x"], t, at, g, weights, y, dev_saved=saved)
            ro.experts_backward(p["x"], t, g, weights, saved, y, list(grads.values()))
            ro.route_backward(d, t, a, r, None, at, g, grads["dgates"], dd, da, dr)

        def results():
            return [gpu.down(at, (t, k), np.int32), gpu.down(g, (t, k), np.float32), gpu.down(y, (t, o), np.uint16)] + [
                gpu.down(grads[i], s, np.uint16) for i, s in shapes.items()] + [
                gpu.down(dd, (t, n), np.float32), gpu.down(da, n, np.float32), gpu.down(dr, n, np.float32)]

        inputs = [(5 + rng.standard_normal((t, n))).astype(np.float32) for _ in range(4)]
        eager = []
        ro.reserve(t)
        for v in inputs:
            gpu.write(d, v)
            calls()
            ro.synchronize()
            eager.append(results())
        ro.set_stream(stream.value)
        gpu.ok(gpu.rt.hipStreamBeginCapture(stream, 0))
        calls()
        gpu.ok(gpu.rt.hipStreamEndCapture(stream, C.byref(graph)))
        gpu.ok(gpu.rt.hipGraphInstantiate(C.byref(run), graph, None, None, 0))
        for i in (2, 0, 3, 1):
            gpu.write(d, inputs[i])
            gpu.ok(gpu.rt.hipGraphLaunch(run, stream))
            ro.synchronize()
            for got, want in zip(results(), eager[i]):
                assert np.array_equal(got, want)
            calls()                                        # eager work between the replays, on the other inputs' buffers
            ro.synchronize()
        ro.set_stream(capi.OWN_STREAM)
        gpu.rt.hipGraphExecDestroy(run)
        gpu.rt.hipGraphDestroy(graph)
    gpu.rt.hipStreamDestroy(stream)


# --------------------------------------------------------------------------------------------------------------- AdamW

F = np.float32
OPTIONS = dict(learning_rate=2e-3, beta_first=0.9, beta_second=0.99, epsilon=1e-8)


def unpack(codes, scale, second):
    i = np.arange(codes.size) // 256
    u = codes.astype(F) * (F(1) / F(255) if second else F(1) / F(127))
    if second:
        u = u * u
        return (u * u) * scale[i]
    return (u * np.abs(u)) * scale[i]


def pack(x, second):
    """(codes, scales) in 32-bit arithmetic, as the definition says."""
    padded_ = np.pad(x, (0, -x.size % 256)).reshape(-1, 256)
    scale = np.abs(padded_).max(1)
    scale = np.where(scale < F(2.0 ** -126), F(0), scale).astype(F)
    with np.errstate(divide="ignore"):
        over = np.where(scale > 0, F(1) / scale, F(0)).astype(F)
    ratio = np.abs(padded_) * over[:, None]
    root = np.sqrt(ratio)
    if second:
        codes = np.rint(np.sqrt(root) * F(255))
        codes = np.where(ratio > 0, np.maximum(codes, 1), codes)
    else:
        codes = np.rint(root * F(127)) * np.sign(padded_)
    return codes.reshape(-1)[:x.size].astype(np.uint8 if second else np.int8), scale


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", [[1], [255, 256, 257, 2047, 2048, 2049, 5], [7, 0, 3] * 30, [70001]])
@pytest.mark.parametrize("bf16", [False, True])
def test_adamw(gpu, bits, sizes, bf16):
    rng = np.random.default_rng(sum(sizes) + bits)
    element = Element(bf16)
    tensors, held = [], []
    for i, n in enumerate(sizes):
        stored, grad = element.store(rng.standard_normal(n) * 10.0 ** rng.integers(-6, 1))
        value = rng.standard_normal(n).astype(F)
        m, v = (0.1 * rng.standard_normal(n)).astype(F), (0.01 * rng.standard_normal(n) ** 2).astype(F)
        if n > 300:
            m[:256] = v[:256] = 0                          # a block of zeros
            stored[:256] = 0
            grad[:256] = 0
            v[256:300] = F(1e-44)                          # far below the block's largest: never zero once packed
        t = dict(value=gpu.up(value), gradient=gpu.up(stored), size=n, decay=0.1 * (i % 2), gradient_bf16=bf16, rounded=gpu.new(n, np.uint16) if bf16 else None)
        s = dict(value=value, grad=grad.astype(F), decay=F(0.1 * (i % 2)))
        if bits == 8:
            s["m"], s["ms"] = pack(m, False)
            s["v"], s["vs"] = pack(v, True)
            t.update(first=gpu.up(s["m"]), second=gpu.up(s["v"]), first_scale=gpu.up(s["ms"]), second_scale=gpu.up(s["vs"]),
                     first_values=gpu.new(n, F), second_values=gpu.new(n, F))
        else:
            s["m"], s["v"] = m, v
            t.update(first=gpu.up(m), second=gpu.up(v))
        tensors.append(t)
        held.append(s)
    with capi.Readout(4) as ro:
        table = ro.tensors(tensors)
        for step in (1, 2, 3):
            ro.adamw(table, step, bits=bits, **OPTIONS)
            if bits == 8:
                ro.adamw_unpack(table)
            ro.synchronize()
            for t, s in zip(tensors, held):
                n = t["size"]
                # the states follow in 32-bit arithmetic, every operation rounded: the same bits
                m, v = (unpack(s["m"], s["ms"], False), unpack(s["v"], s["vs"], True)) if bits == 8 else (s["m"], s["v"])
                b1, b2 = F(OPTIONS["beta_first"]), F(OPTIONS["beta_second"])
                m, v = m * b1 + s["grad"] * (F(1) - b1), v * b2 + (s["grad"] * s["grad"]) * (F(1) - b2)
                # the values in 64 bits: three products, a sum, a root, a quotient, and the subtraction's own rounding
                m64, v64, p64 = m.astype(np.float64), v.astype(np.float64), s["value"].astype(np.float64)
                change = m64 / (1 - float(b1) ** step) / (np.sqrt(v64 / (1 - float(b2) ** step)) + OPTIONS["epsilon"])
                want = p64 - float(F(OPTIONS["learning_rate"])) * (change + float(s["decay"]) * p64)
                got = gpu.down(t["value"], n, F)
                bound = S * (np.abs(want) * 1.01 + 16 * OPTIONS["learning_rate"] * (np.abs(change) + np.abs(s["decay"] * p64))) + 1e-40
                assert_within(got.astype(np.float64), want, bound, "value")
                s["value"] = got
                if bf16:
                    assert np.array_equal(gpu.down(t["rounded"], n, np.uint16), to_bf16(got))
                if bits == 8:
                    s["m"], s["ms"] = pack(m, False)
                    s["v"], s["vs"] = pack(v, True)
                    assert np.array_equal(gpu.down(t["first"], n, np.int8), s["m"]) and np.array_equal(gpu.down(t["second"], n, np.uint8), s["v"])
                    assert np.array_equal(gpu.down(t["first_scale"], s["ms"].size, F), s["ms"])
                    assert np.array_equal(gpu.down(t["second_scale"], s["vs"].size, F), s["vs"])
                    assert np.array_equal(gpu.down(t["first_values"], n, F), unpack(s["m"], s["ms"], False))
                    assert np.array_equal(gpu.down(t["second_values"], n, F), unpack(s["v"], s["vs"], True))
                    assert not np.any((v > 0) & (s["vs"][np.arange(n) // 256] > 0) & (v / np.maximum(s["vs"][np.arange(n) // 256], F(1e-38)) > 0) & (s["v"] == 0))
                else:
                    s["m"], s["v"] = m, v
                    assert np.array_equal(gpu.down(t["first"], n, F), m) and np.array_equal(gpu.down(t["second"], n, F), v)


@pytest.mark.gpu
def test_adamw_at_addresses_of_single_elements(gpu):
    """Tensors that start anywhere in a buffer, as views do."""
    rng = np.random.default_rng(9)
    n = 1000
    value, grad = rng.standard_normal(n + 3).astype(F), rng.standard_normal(n + 3).astype(F)
    zeros = np.zeros(n + 3, F)
    with capi.Readout(4) as ro:
        got = []
        for skip in (0, 1, 3):
            p = [gpu.up(np.roll(a, skip)) for a in (value, to_bf16(grad), zeros, zeros)]
            rounded = gpu.new(n + 3, np.uint16)
            ro.adamw(ro.tensors([dict(value=p[0] + 4 * skip, gradient=p[1] + 2 * skip, first=p[2] + 4 * skip, second=p[3] + 4 * skip,
                                      rounded=rounded + 2 * skip, size=n, decay=0.0, gradient_bf16=True)]), 1, **OPTIONS)
            ro.synchronize()
            all_ = gpu.down(p[0], n + 3, F)
            assert np.array_equal(np.roll(all_, -skip)[n:], value[n:])         # nothing outside is touched
            got.append(all_[skip:skip + n])
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


# ------------------------------------------------------------------------------------------------------- all together

@pytest.mark.gpu
@pytest.mark.parametrize("options", [[], ["--state-bits", "8", "--chosen", "3"]])
def test_read_out_of_a_small_map_learns(options):
    # in a process of its own: PyTorch has to come before the library
    import os
    import re
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-u", "-m", "pink_amd.readout", "--steps", "200"] + options, cwd=root, capture_output=True, text=True, timeout=100)
    assert run.returncode == 0, run.stderr[-2000:]
    error, alone = map(float, re.search(r"new sources: mean squared error ([\d.]+) \(of the mean alone: ([\d.]+)\)", run.stdout).groups())
    assert error < 0.25 * alone, run.stdout
