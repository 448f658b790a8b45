"""The read-out's blocks and its loss on classes (pink_hip_readout_norm*, _gated*, _distil*) against plain restatements in 64 bits, through the
C ABI.

Tolerances are bounds, computed next to each expected value from the roundings that the operators make: u is half a step of what
is stored (2^-24 float32, 2^-8 bfloat16), s = 2^-24 that of sums.  A sum of K terms in any order is off by at most (K + 2) s times the sum
of their magnitudes; where a row's terms are added up a few a thread and then by a tree, K is the number of additions that one
term goes through.
"""
import ctypes as C
import math
import types

import numpy as np
import pytest

from pink_amd import capi
from test_readout import ACT, BENT, S, STEEP, Element, assert_within, f_and_slope, gpu, padded  # noqa: F401  (gpu: fixture)
from test_readout_edges import Recording


def nan_of(element):
    return 0x7fc0 if element.bf16 else np.nan


# ---------------------------------------------------------------------------------------------------------- layer norm

EPSILON = 1e-5


def norm_reference(x, w, b, dy, residual, element, epsilon=EPSILON):
    """{name: (value, bound)} of the forward and backward pass."""
    t, n = x.shape
    u, one = element.u, np.ones(n)
    path = (64 + n // 1024 + 5) * S                       # additions that a term of a row goes through
    w_, b_ = (one if w is None else w), (0 * one if b is None else b)
    mean = x.mean(1, keepdims=True)
    off_mean = path * np.abs(x).mean(1, keepdims=True)
    off = x - mean
    e_off = off_mean + S * np.abs(off)
    var = (off * off).mean(1, keepdims=True)
    e_var = (2 * np.abs(off) * e_off + e_off ** 2).mean(1, keepdims=True) + path * var
    scale = 1 / np.sqrt(var + epsilon)
    assert (e_var < 0.1 * (var + epsilon)).all()
    e_scale = scale * (0.6 * e_var / (var + epsilon) + 6 * S)
    form = off * scale
    e_form = e_off * scale + np.abs(off) * e_scale + 2 * S * np.abs(form)
    y = form * w_ + b_
    out = {"y": (y, e_form * np.abs(w_) + 3 * S * (np.abs(form * w_) + np.abs(b_)) + 1.01 * u * np.abs(y)), "mean": (mean[:, 0], off_mean[:, 0]),
           "scale": (scale[:, 0], e_scale[:, 0])}
    if dy is None:
        return out
    g = dy * w_
    c1, c2 = g.mean(1, keepdims=True), (g * form).mean(1, keepdims=True)
    e1 = path * np.abs(g).mean(1, keepdims=True)
    e2 = (np.abs(g) * e_form).mean(1, keepdims=True) + path * np.abs(g * form).mean(1, keepdims=True)
    inner, mag = g - c1 - form * c2, np.abs(g) + np.abs(c1) + np.abs(form * c2)
    dx = scale * inner + (0 if residual is None else residual)
    e_dx = scale * (e1 + np.abs(form) * e2 + e_form * np.abs(c2) + e_form * e2 + 5 * S * mag) + e_scale * (np.abs(inner) + 5 * S * mag)
    out["dx"] = dx, e_dx + S * np.abs(dx) + 1.01 * u * np.abs(dx)
    down = (t + 70) * S
    dw, db = (dy * form).sum(0), dy.sum(0)
    out["dw"] = dw, (np.abs(dy) * e_form).sum(0) + down * np.abs(dy * form).sum(0) + 1.01 * u * np.abs(dw) + u * down * np.abs(dy * form).sum(0)
    out["db"] = db, (1 + u) * down * np.abs(dy).sum(0) + 1.01 * u * np.abs(db)
    return out


NORMS = [  # images, width, weight, bias, residual, padding of rows: every number of threads a row, whole chunks and not
    (1, 1, True, True, False, 0), (1, 7, True, True, True, 1), (3, 16, False, True, False, 0), (37, 128, True, True, True, 0), (9, 129, True, False, False, 3),
    (20, 256, True, True, False, 8), (1100, 33, True, True, True, 0), (5, 331, True, True, True, 0), (17, 512, False, False, False, 0),
    (6, 1000, True, True, True, 0), (9, 1024, True, True, False, 8), (301, 2025, True, True, True, 0), (13, 2048, True, True, False, 0), (3, 2049, True, True, True, 1),
    (530, 4096, True, True, True, 0), (5, 4999, True, False, True, 0), (3, 8192, True, True, False, 0), (2, 8200, False, True, True, 8),
    (2, 16384, True, True, True, 0), (1030, 1000, True, True, False, 0), (8195, 1030, True, True, True, 0),
    (70, 16385, True, True, True, 0), (2, 40003, True, True, False, 5), (1, 2 ** 20, True, True, True, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("t, n, weight, bias, residual, pad", NORMS)
def test_norm(gpu, t, n, weight, bias, residual, pad, bf16):  # noqa: F811
    rng, element = np.random.default_rng(t * 37 + n), Element(bf16)
    nan = nan_of(element)
    draw = {"x": rng.standard_normal((t, n)) * rng.uniform(0.2, 2, (t, 1)) + 3 * rng.standard_normal((t, 1)), "w": 1 + 0.3 * rng.standard_normal(n) if weight else None,
            "b": 0.3 * rng.standard_normal(n) if bias else None, "dy": rng.standard_normal((t, n)), "r": rng.standard_normal((t, n)) if residual else None}
    stored, value = {}, {}
    for i, v in draw.items():
        stored[i], value[i] = element.store(v)
    want = norm_reference(value["x"], value["w"], value["b"], value["dy"], value["r"], element)
    rows = {i: gpu.up(padded(stored[i], pad, nan)) if stored[i] is not None else None for i in ("x", "dy", "r")}
    w, b = gpu.up(stored["w"]), gpu.up(stored["b"])
    with capi.Readout(1, element=element.id) as ro:
        y, mean, scale = gpu.up(np.full((t, n + pad), nan, element.dtype)), gpu.new(t, np.float32), gpu.new(t, np.float32)
        dx, dw, db = gpu.up(np.full((t, n + pad), nan, element.dtype)), gpu.new(n, element.dtype), gpu.new(n, element.dtype)
        first = None
        for _ in range(2):                                 # twice: the same bits
            ro.norm(rows["x"], t, n, w, b, EPSILON, y, mean, scale, x_stride=n + pad, y_stride=n + pad)
            ro.norm_backward(rows["x"], t, n, w, mean, scale, rows["dy"], dx, dw, db, dev_residual=rows["r"], x_stride=n + pad, dy_stride=n + pad,
                             residual_stride=n + pad, dx_stride=n + pad)
            ro.synchronize()
            got = {"y": gpu.down(y, (t, n + pad), element.dtype), "mean": gpu.down(mean, t, np.float32), "scale": gpu.down(scale, t, np.float32),
                   "dx": gpu.down(dx, (t, n + pad), element.dtype), "dw": gpu.down(dw, n, element.dtype), "db": gpu.down(db, n, element.dtype)}
            for i, v in got.items():
                if i in ("y", "dx"):                       # what lies between rows stays as it was
                    assert np.array_equal(v[:, n:], np.full((t, pad), nan, element.dtype), equal_nan=not bf16)
                    v = v[:, :n]
                assert_within(v.astype(np.float64) if i in ("mean", "scale") else element.values(v), *want[i], i)
            first = first or got
            assert all(np.array_equal(first[i], got[i], equal_nan=not bf16) for i in got)
        # each gradient alone, and in the place of an argument that allows it
        alone = gpu.new(n, element.dtype)
        ro.norm_backward(rows["x"], t, n, w, mean, scale, rows["dy"], None, alone, None, x_stride=n + pad, dy_stride=n + pad)
        ro.synchronize()
        assert np.array_equal(gpu.down(alone, n, element.dtype), got["dw"])
        ro.norm_backward(rows["x"], t, n, w, mean, scale, rows["dy"], None, None, alone, x_stride=n + pad, dy_stride=n + pad)
        ro.synchronize()
        assert np.array_equal(gpu.down(alone, n, element.dtype), got["db"])
        place = rows["r"] if residual else rows["dy"]
        ro.norm_backward(rows["x"], t, n, w, mean, scale, rows["dy"], place, dw, None, dev_residual=rows["r"], x_stride=n + pad, dy_stride=n + pad,
                         residual_stride=n + pad, dx_stride=n + pad)
        ro.norm(rows["x"], t, n, w, b, EPSILON, rows["x"], x_stride=n + pad, y_stride=n + pad)
        ro.synchronize()
        assert np.array_equal(gpu.down(place, (t, n + pad), element.dtype)[:, :n], got["dx"][:, :n])
        assert np.array_equal(gpu.down(dw, n, element.dtype), got["dw"])
        assert np.array_equal(gpu.down(rows["x"], (t, n + pad), element.dtype)[:, :n], got["y"][:, :n])


def test_norm_gradients_of_the_restatement_against_differences():
    rng, element = np.random.default_rng(5), Element(False)
    x, w, b, dy, d = rng.standard_normal((3, 17)) + 2, 1 + rng.standard_normal(17), rng.standard_normal(17), rng.standard_normal((3, 17)), 1e-5
    out = norm_reference(x, w, b, dy, None, element)
    for name, at in (("dx", x), ("dw", w), ("db", b)):
        for i in np.ndindex(*at.shape):
            kept, loss = at[i], []
            for sign in (1, -1):
                at[i] = kept + sign * d
                loss.append((norm_reference(x, w, b, None, None, element)["y"][0] * dy).sum())
            at[i] = kept
            # truncated at d^2 (third derivatives of some tens), rounded to 1e-16 / d
            assert abs((loss[0] - loss[1]) / (2 * d) - out[name][0][i]) < 1e-7


@pytest.mark.gpu
def test_norm_of_rows_at_the_edges(gpu):  # noqa: F811
    """Constant rows give the bias; a level far above the spread costs no more than its own digits; a row that is not finite gives NaN and
    no other does."""
    rng, element, n = np.random.default_rng(6), Element(False), 300
    x = np.stack([np.full(n, 7.0), np.zeros(n), 1000 + rng.standard_normal(n), rng.standard_normal(n) * 1e-15, rng.standard_normal(n) * 1e15,
                  rng.standard_normal(n), rng.standard_normal(n), rng.standard_normal(n)]).astype(np.float32)
    x[5, 3], x[6, 299] = np.nan, np.inf
    w, b = rng.standard_normal(n).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    with capi.Readout(1, element=element.id) as ro:
        y, args = gpu.new(x.shape, np.float32), [gpu.up(a) for a in (x, w, b)]
        ro.norm(args[0], len(x), n, args[1], args[2], EPSILON, y)
        ro.synchronize()
        got = gpu.down(y, x.shape, np.float32).astype(np.float64)
        part = [0, 1, 3, 4, 7]
        # (a constant row's mean is a rounding off, by path |x|, which its scale of 1 / sqrt(epsilon) enlarges; bound[2]: as derived)
        value, bound = norm_reference(x[[2, 7, 3, 4]].astype(np.float64), w.astype(np.float64), b.astype(np.float64), None, None, element)["y"]
        assert_within(got[[2, 7, 3, 4]], value, bound, "y")
        assert np.array_equal(got[1], b.astype(np.float64))
        assert (np.abs(got[0] - b) <= np.abs(w) * 70 * S * 7 / math.sqrt(EPSILON) + S * np.abs(b) * 2).all()
        assert np.isnan(got[5]).all() and np.isnan(got[6]).all() and np.isfinite(got[part]).all()
        ro.norm(args[0], len(x), n, None, None, 0.0, y)    # no epsilon, no weights: rows of a spread
        ro.synchronize()
        got = gpu.down(y, x.shape, np.float32).astype(np.float64)
        value, bound = norm_reference(x[[2, 7]].astype(np.float64), None, None, None, None, element, 0.0)["y"]
        assert_within(got[[2, 7]], value, bound, "y")


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 260, 1000])
def test_norm_gradients_at_a_level_near_the_largest(gpu, n):  # noqa: F811
    """Threads that have nothing of a row add nothing, also where a level of 2^120 by a scale of 2^10 is past float32."""
    rng, element, t = np.random.default_rng(n), Element(False), 3
    x, dy = np.full((t, n), 2.0 ** 120, np.float32), rng.standard_normal((t, n)).astype(np.float32)
    args = [gpu.up(a) for a in (x, np.full(t, 2.0 ** 120, np.float32), np.full(t, 2.0 ** 10, np.float32), dy)]
    out = [gpu.new(s, np.float32) for s in ((t, n), n, n)]
    with capi.Readout(1, element=element.id) as ro:
        ro.norm_backward(args[0], t, n, None, args[1], args[2], args[3], *out)
        ro.synchronize()
    dx, dw, db = (gpu.down(p, s, np.float32).astype(np.float64) for p, s in zip(out, ((t, n), n, n)))
    d = dy.astype(np.float64)
    value = 2.0 ** 10 * (d - d.mean(1, keepdims=True))     # x' is 0
    # (a mean of n terms, at most 74 additions each: norm_reference's path; then a subtraction, a product, a rounding)
    bound = 2.0 ** 10 * (74 * S * np.abs(d).mean(1, keepdims=True) + 3 * S * (np.abs(d) + np.abs(d).mean(1, keepdims=True)))
    assert_within(dx, value, bound, "dx")
    assert (dw == 0).all()
    assert_within(db, d.sum(0), 5 * S * np.abs(d).sum(0), "db")


# -------------------------------------------------------------------------------------------------------- gated block

def gated_reference(m, element, act, dy):
    """{name: (value, bound)} of the answer and all gradients; `m` holds x, gate, gate_bias, up, up_bias, down, down_bias, residual."""
    x, gate, up, down = (m[i] for i in ("x", "gate", "up", "down"))
    (t, f), h, o, u = x.shape, gate.shape[0], down.shape[0], element.u
    c1, c2, c3 = (0 if m[i] is None else m[i] for i in ("gate_bias", "up_bias", "down_bias"))
    a, b = x @ gate.T + c1, x @ up.T + c2
    off_a, off_b = ((f + 2) * S * (np.abs(x) @ np.abs(w).T + np.abs(c)) for w, c in ((gate, c1), (up, c2)))
    v, slope = f_and_slope(act, a)
    # (bfloat16's activations: within 1.5e-7 and a few roundings of the formula's)
    off_v = STEEP[act] * off_a + 8 * S * (np.abs(a) + np.abs(v))
    off_slope = BENT[act] * off_a + (8 * S * (1 + np.abs(a)) if act in ("gelu", "silu") else 0)
    if act == "relu":
        off_slope = off_slope + (np.abs(a) <= off_a)       # on which side of the kink is open there
    def product(p, q, off_p, off_q, more):
        return p * q, off_p * np.abs(q) + np.abs(p) * off_q + off_p * off_q + more * np.abs(p * q) * 1.01
    hidden, off_h = product(v, b, off_v, off_b, u + S)
    y, mag = hidden @ down.T + c3, np.abs(hidden) @ np.abs(down).T + np.abs(c3)
    off = off_h @ np.abs(down).T + (h + 3) * S * mag
    if m["residual"] is not None:
        y, off = y + m["residual"], off + 2 * S * (np.abs(y) + np.abs(m["residual"]))
    out = {"y": (y, off)}
    if dy is not None:
        dh, off_dh = dy @ down, (o + 2) * S * (np.abs(dy) @ np.abs(down))
        kept = 2.0 ** -15 if element.bf16 else 0                         # (cut off after 16 bits, or all of float32's)
        k1, off_k1 = product(slope, b, off_slope, off_b, kept + S)
        off_k2 = off_v + kept * np.abs(v) * 1.01
        da, off_da32 = product(dh, k1, off_dh, off_k1, S)
        db, off_db32 = product(dh, v, off_dh, off_k2, S)
        off_da, off_db = off_da32 + u * np.abs(da) * 1.01 + u * off_da32, off_db32 + u * np.abs(db) * 1.01 + u * off_db32
        out["dx"] = da @ gate + db @ up, off_da @ np.abs(gate) + off_db @ np.abs(up) + (2 * h + 4) * S * (np.abs(da) @ np.abs(gate) + np.abs(db) @ np.abs(up))
        sums = (t + 40) * S
        out["dgate"] = da.T @ x, off_da.T @ np.abs(x) + sums * (np.abs(da).T @ np.abs(x))
        out["dup"] = db.T @ x, off_db.T @ np.abs(x) + sums * (np.abs(db).T @ np.abs(x))
        out["ddown"] = dy.T @ hidden, np.abs(dy).T @ off_h + sums * (np.abs(dy).T @ np.abs(hidden))
        out["dgate_bias"] = da.sum(0), off_da32.sum(0) + sums * np.abs(da).sum(0)
        out["dup_bias"] = db.sum(0), off_db32.sum(0) + sums * np.abs(db).sum(0)
        out["ddown_bias"] = dy.sum(0), sums * np.abs(dy).sum(0)
    return {i: (value, bound + u * np.abs(value) * 1.02 + u * bound) for i, (value, bound) in out.items()}


WEIGHTS = ("gate", "gate_bias", "up", "up_bias", "down", "down_bias")


def gated_inputs(rng, element, t, f, h, o, bias, residual):
    draw = {"x": rng.standard_normal((t, f)), "gate": rng.standard_normal((h, f)) / math.sqrt(f), "gate_bias": 0.3 * rng.standard_normal(h) if bias else None,
            "up": rng.standard_normal((h, f)) / math.sqrt(f), "up_bias": 0.3 * rng.standard_normal(h) if bias else None,
            "down": rng.standard_normal((o, h)) / math.sqrt(h), "down_bias": 0.3 * rng.standard_normal(o) if bias else None,
            "residual": rng.standard_normal((t, o)) if residual else None, "dy": rng.standard_normal((t, o))}
    stored, value = {}, {}
    for name, v in draw.items():
        stored[name], value[name] = element.store(v)
    return stored, value


GATED = [  # images, features, hidden, outputs, activation, bias, residual, padding of rows
    (1, 1, 1, 1, "identity", True, False, 0),
    (1, 64, 32, 16, "silu", True, False, 0),
    (1, 130, 33, 7, "gelu", False, True, 1),
    (2, 1024, 200, 72, "silu", True, True, 8),
    (4, 77, 19, 5, "silu", True, True, 3),
    (5, 264, 136, 129, "relu", False, True, 0),
    (16, 520, 72, 40, "gelu", True, False, 0),
    (16, 331, 71, 41, "silu", True, True, 0),
    (17, 96, 48, 24, "silu", True, True, 0),
    (33, 95, 47, 23, "relu", True, False, 1),
    (70, 200, 1024, 1, "silu", True, False, 0),
    (100, 16, 2048, 16, "gelu", True, True, 0),
    (130, 40, 2000, 264, "silu", True, True, 0),
    (130, 41, 2001, 263, "silu", True, True, 3),
    (300, 264, 520, 264, "silu", True, True, 0),
    (301, 263, 519, 265, "gelu", False, True, 1),
    (1500, 24, 16, 8, "silu", True, False, 0),
    (1501, 23, 17, 9, "silu", True, True, 0),
    (2100, 520, 1096, 520, "silu", True, True, 0),
    (2099, 519, 1095, 521, "relu", True, False, 1),
    # few rows and a long summed axis, in whole chunks and not; the same cut into runs
    (3, 2312, 2120, 40, "silu", True, True, 0),
    (25, 2313, 2121, 41, "gelu", True, True, 2),
    (32, 4104, 40, 4104, "silu", False, True, 0),
    (40, 72, 4104, 136, "silu", True, True, 0),
    (41, 71, 4101, 135, "silu", True, True, 1),
    # the last three products in one launch, in tiles of 16 x 32, 32 x 32 and 64 x 64; not, for one's long axis
    (90, 328, 248, 328, "silu", True, True, 0),
    (400, 520, 400, 520, "gelu", True, False, 8),
    (401, 519, 401, 521, "gelu", True, False, 0),
    (600, 1032, 1000, 520, "silu", True, True, 0),
    (1600, 520, 136, 264, "silu", True, True, 0),
    (2047, 72, 64, 40, "silu", True, True, 0),
    (2048, 72, 64, 40, "silu", True, True, 0),
    (2600, 331, 331, 331, "relu", True, True, 0),
    (3000, 72, 64, 40, "silu", True, True, 0),
    (97, 1544, 3001, 32, "silu", True, False, 0),
    (65, 2112, 2200, 72, "gelu", True, True, 8),
    (200, 1544, 800, 32, "silu", True, False, 0),
    (200, 1545, 801, 33, "relu", True, True, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("t, f, h, o, act, bias, residual, pad", GATED)
def test_gated(gpu, t, f, h, o, act, bias, residual, pad, bf16):  # noqa: F811
    rng, element = np.random.default_rng(t * 131 + f), Element(bf16)
    stored, value = gated_inputs(rng, element, t, f, h, o, bias, residual)
    want, nan = gated_reference(value, element, act, value["dy"]), nan_of(element)
    p = {i: gpu.up(v) for i, v in stored.items()}
    for i in ("x", "residual", "dy"):
        p[i] = gpu.up(padded(stored[i], pad, nan)) if stored[i] is not None else None
    weights, shape = [p[i] for i in WEIGHTS], (f, h, o, ACT[act])
    names = {"dx": (t, f), **{"d" + i: stored[i].shape for i in WEIGHTS if stored[i] is not None}}
    given = ["dx"] + ["d" + i for i in WEIGHTS]
    with capi.Readout(1, element=element.id) as ro:
        saved = gpu.new(ro.gated_saved_bytes(shape, t), np.int8)
        answers = []
        for keep in (None, None, saved, saved):
            y = gpu.up(np.full((t, o + pad), nan, element.dtype))
            ro.gated(shape, p["x"], t, weights, y, dev_residual=p["residual"], dev_saved=keep, x_stride=f + pad, residual_stride=o + pad, y_stride=o + pad)
            ro.synchronize()
            answers.append(gpu.down(y, (t, o + pad), element.dtype))
            assert np.array_equal(answers[-1][:, o:], np.full((t, pad), nan, element.dtype), equal_nan=not bf16)
            assert_within(element.values(answers[-1][:, :o]), *want["y"], "y")
        assert np.array_equal(answers[0][:, :o], answers[1][:, :o]) and np.array_equal(answers[2][:, :o], answers[3][:, :o])
        grads = {i: gpu.new(s if i != "dx" else (t, f + pad), element.dtype) for i, s in names.items()}
        for again in range(2):
            ro.gated_backward(shape, p["x"], t, weights, saved, p["dy"], [grads.get(i) for i in given], x_stride=f + pad, y_gradient_stride=o + pad,
                              x_gradient_stride=f + pad)
            ro.synchronize()
            got = {i: gpu.down(grads[i], s if i != "dx" else (t, f + pad), element.dtype) for i, s in names.items()}
            got["dx"] = got["dx"][:, :f]
            first = got if not again else first
            for i in names:
                assert np.array_equal(got[i], first[i])
                assert_within(element.values(got[i]), *want[i], i)
        for i in names:                                    # each gradient alone: the same bits
            alone = gpu.new(names[i], element.dtype)
            ro.gated_backward(shape, p["x"], t, weights, saved, p["dy"], [alone if j == i else None for j in given], x_stride=f + pad, y_gradient_stride=o + pad)
            ro.synchronize()
            assert np.array_equal(gpu.down(alone, names[i], element.dtype), got[i]), i


@pytest.mark.gpu
@pytest.mark.parametrize("t, f, h, o, act, bias, residual, pad", [
    # each product in tiles of 256 x 256: with last tiles and stages that are not full
    (4100, 328, 3080, 264, "silu", True, True, 8),
    (4097, 64, 3328, 64, "gelu", False, False, 0),
    (4100, 3080, 192, 3080, "silu", True, True, 0),
    (72, 1544, 4104, 4104, "relu", True, False, 8),
    (130, 3080, 4104, 3080, "silu", True, True, 0),
])
def test_gated_in_large_tiles(gpu, t, f, h, o, act, bias, residual, pad):  # noqa: F811
    test_gated(gpu, t, f, h, o, act, bias, residual, pad, True)


@pytest.mark.gpu
@pytest.mark.parametrize("t, f, h, o, bf16", [(2200, 1930, 1150, 24, False), (2201, 1931, 1151, 23, False), (12000, 1200, 2000, 8, True)])
def test_gated_with_weights_gradients_in_runs_of_large_tiles(gpu, t, f, h, o, bf16):  # noqa: F811
    test_gated(gpu, t, f, h, o, "silu", False, False, 0, bf16)


@pytest.mark.parametrize("act", ["identity", "gelu", "silu"])
def test_gated_gradients_of_the_restatement_against_differences(act):
    rng, element, d = np.random.default_rng(8), Element(False), 1e-5
    value = {i: None if v is None else v.astype(np.float64) for i, v in gated_inputs(rng, element, 3, 5, 4, 2, True, True)[1].items()}
    out = gated_reference(value, element, act, value["dy"])
    for name in ("x",) + WEIGHTS:
        at = value[name]
        for i in np.ndindex(*at.shape):
            kept, loss = at[i], []
            for sign in (1, -1):
                at[i] = kept + sign * d
                loss.append((gated_reference(value, element, act, None)["y"][0] * value["dy"]).sum())
            at[i] = kept
            assert abs((loss[0] - loss[1]) / (2 * d) - out["d" + name][0][i]) < 1e-7


@pytest.mark.gpu
def test_gated_in_place(gpu):  # noqa: F811
    """The answer may lie where the residual or the images do; images outside the batch stay as they were."""
    rng, element, (t, f, h) = np.random.default_rng(9), Element(True), (200, 136, 72)
    stored, _ = gated_inputs(rng, element, t, f, h, f, True, True)
    weights, shape = [gpu.up(stored[i]) for i in WEIGHTS], (f, h, f, capi.ACT_SILU)
    more = np.concatenate([stored["x"], np.full((3, f), 0x4242, np.uint16)])
    with capi.Readout(1, element=element.id) as ro:
        x, y = gpu.up(more), gpu.new((t, f), np.uint16)
        ro.gated(shape, x, t, weights, y, dev_residual=x)
        ro.gated(shape, x, t, weights, x, dev_residual=x)
        ro.synchronize()
        got = gpu.down(x, more.shape, np.uint16)
        assert np.array_equal(got[:t], gpu.down(y, (t, f), np.uint16)) and (got[t:] == 0x4242).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("t, f, h", [(200, 136, 72), (70, 33, 2100), (600, 520, 400), (1400, 72, 40)])
def test_gated_gradients_in_place(gpu, t, f, h, bf16):  # noqa: F811
    """The gradients of the features may lie where the images or those of the answers do: none of the others change."""
    rng, element = np.random.default_rng(19), Element(bf16)
    stored, _ = gated_inputs(rng, element, t, f, h, f, True, False)
    weights, shape = [gpu.up(stored[i]) for i in WEIGHTS], (f, h, f, capi.ACT_SILU)
    with capi.Readout(1, element=element.id) as ro:
        saved, got = gpu.new(ro.gated_saved_bytes(shape, t), np.int8), []
        for place in ("apart", "x", "dy"):
            at = {"x": gpu.up(stored["x"]), "dy": gpu.up(stored["dy"]), "apart": gpu.new((t, f), element.dtype)}
            grads = [gpu.new(stored[i].shape, element.dtype) for i in WEIGHTS]
            ro.gated(shape, at["x"], t, weights, gpu.new((t, f), element.dtype), dev_saved=saved)
            ro.gated_backward(shape, at["x"], t, weights, saved, at["dy"], [at[place]] + grads)
            ro.synchronize()
            got.append([gpu.down(at[place], (t, f), element.dtype)] + [gpu.down(p, stored[i].shape, element.dtype) for p, i in zip(grads, WEIGHTS)])
        for other in got[1:]:
            assert all(np.array_equal(a, b) for a, b in zip(other, got[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("t, h, f", [(1, 33, 64), (20, 33, 64), (90, 33, 128), (300, 42, 256), (2100, 519, 520)])
def test_gated_reads_nothing_that_it_did_not_write(gpu, t, h, f, bf16):  # noqa: F811
    """Hidden values in whole chunks: what pads a row is zeros, whatever the workspace and `saved` held."""
    rng, element = np.random.default_rng(10), Element(bf16)
    stored, value = gated_inputs(rng, element, t, f, h, f, True, False)
    weights, shape = [gpu.up(stored[i]) for i in WEIGHTS], (f, h, f, capi.ACT_SILU)
    want = gated_reference(value, element, "silu", value["dy"])
    with capi.Readout(1, element=element.id) as ro:
        n = ro.gated_saved_bytes(shape, t)
        saved, y, dx = gpu.up(np.full(n, 0xff, np.uint8)), gpu.new((t, f), element.dtype), gpu.new((t, f), element.dtype)
        dgate = gpu.new((h, f), element.dtype)
        x, dy = gpu.up(stored["x"]), gpu.up(stored["dy"])
        ro.gated_reserve(shape, t)
        poison = [gpu.up(np.full(1 << s, 0xff, np.uint8)) for s in range(14, 26)]
        ro.gated(shape, x, t, weights, y, dev_saved=saved)
        ro.gated_backward(shape, x, t, weights, saved, dy, [dx, dgate, None, None, None, None, None])
        ro.synchronize()
        assert len(poison) == 12
        assert_within(element.values(gpu.down(y, (t, f), element.dtype)), *want["y"], "y")
        assert_within(element.values(gpu.down(dx, (t, f), element.dtype)), *want["dx"], "dx")
        assert_within(element.values(gpu.down(dgate, (h, f), element.dtype)), *want["dgate"], "dgate")


# -------------------------------------------------------------------------------------------------------- distillation

def distil_reference(z, at, teacher, normaliser, label, weights, temperature, a, b, element):
    """(losses, bound, gradients, bound): one image after the other, by the definition, in 64 bits."""
    (t, v), u = z.shape, element.u
    losses, grads, off_l, off_g = np.zeros(t), np.zeros((t, v)), np.zeros(t), np.zeros((t, v))
    for i in range(t):
        w = 1.0 if weights is None else float(weights[i])
        part = ~np.isneginf(z[i])
        if w == 0 or not part.any():
            continue
        def soft(temp):
            top = z[i][part].max()
            e = np.where(part, np.exp((np.where(part, z[i], top) - top) / temp), 0.0)
            return e / e.sum(), (np.where(part, z[i], 0) - top) / temp - math.log(e.sum())
        dz, e_dz, loss, e_loss = np.zeros(v), np.zeros(v), 0.0, 0.0
        # A power is off by what its exponent is, two roundings of it in float32 and one of the hardware's each, and by one of its own; a sum of them by as
        # much, and 200 additions (128 in a thread, then in 64 bits).
        def e_power(temp):
            return np.abs(np.where(part, z[i] - z[i][part].max(), 0)) / temp * 1.4427 * 4 * S + 4 * S
        if a and (at.shape[1] or normaliser is not None):
            q, logq = soft(temperature)
            e_q = q * (e_power(temperature) + (q * e_power(temperature)).sum() + 200 * S)
            e_logq = (q * e_power(temperature)).sum() + 200 * S
            places, seen = [], set()
            for c, x in zip(at[i], teacher[i]):
                if 0 <= c < v and part[c] and not np.isneginf(x) and c not in seen:
                    places.append((int(c), float(x)))
                    seen.add(int(c))
            p, left, free = np.zeros(v), 0.0, part.copy()
            free[list(seen)] = False
            if places:
                cs, xs = np.array([c for c, _ in places]), np.array([x for _, x in places]) / temperature
                if normaliser is None:
                    e = np.exp(xs - xs.max())
                    p[cs] = e / e.sum()
                else:
                    p[cs] = np.exp(xs - float(normaliser[i]))
            whole = p.sum()
            for c in seen:
                if p[c]:
                    loss += p[c] * (math.log(p[c]) - logq[c])
                e_loss += p[c] * e_logq
            dz[list(seen)] -= p[list(seen)]
            if normaliser is not None and free.any():
                left = max(0.0, 1 - whole)
                if left:
                    top = z[i][part].max()             # (all relative to it, as lowest values swallow small logarithms)
                    zf = (z[i][free] - top) / temperature
                    log_free = zf.max() + math.log(np.exp(zf - zf.max()).sum())
                    loss += left * (math.log(left) - log_free + math.log(np.exp((z[i][part] - top) / temperature).sum()))
                    of = np.where(free, np.exp((np.where(free, z[i], z[i][free].max()) - top) / temperature - log_free), 0.0)
                    dz -= left * of
                    e_dz += left * of * (e_power(temperature) + e_logq + (of * e_power(temperature)).sum() + 200 * S)
                    e_loss += left * (e_logq + (of * e_power(temperature)).sum() + 200 * S)
                whole += left
            dz += whole * q
            e_dz += whole * e_q + 4 * S * (whole * q + np.abs(dz))
            dz, e_dz, loss, e_loss = dz * a * temperature, e_dz * abs(a) * temperature, loss * a * temperature ** 2, e_loss * abs(a) * temperature ** 2
        c = -1 if label is None else int(label[i])
        if b and 0 <= c < v and part[c]:
            q, logq = soft(1.0)
            loss -= b * logq[c]
            e_loss += abs(b) * ((q * e_power(1.0)).sum() + 200 * S)
            dz += b * q
            dz[c] -= b
            e_dz += abs(b) * q * (e_power(1.0) + (q * e_power(1.0)).sum() + 204 * S)
        losses[i], off_l[i], grads[i], off_g[i] = w * loss, abs(w) * (e_loss + 2 * S * abs(loss)) + 1e-300, w * dz, abs(w) * (e_dz + 4 * S * np.abs(dz)) + 2.0 ** -126
    return losses, off_l + 2 * S * np.abs(losses), grads, off_g + 1.01 * u * np.abs(grads) + (2.0 ** -133 if element.bf16 else 2.0 ** -149)


def distil_inputs(rng, element, t, v, k, masked=True, spread=2.0):
    z = rng.standard_normal((t, v)) * spread
    if masked and v > 4:
        z[rng.random((t, v)) < 0.1] = -np.inf
    stored, value = element.store(z)
    full = np.where(np.isneginf(z), 0, z) + rng.standard_normal((t, v))
    at = np.argsort(-full, axis=1)[:, :k].astype(np.int32)
    teacher = np.take_along_axis(full, at, 1).astype(np.float32)
    return stored, value, full, at, teacher


DISTILS = [  # images, classes, places, temperature, rest, teacher's weight, label's weight, image weights, padding of rows
    (1, 1, 1, 1.0, False, 1.0, 0.0, False, 0), (3, 2, 1, 2.0, True, 0.5, 0.5, True, 1), (70, 10, 3, 4.0, True, 0.7, 0.3, True, 0), (5, 10, 10, 2.0, True, 1.0, 1.0, False, 0),
    (9, 31, 0, 1.0, False, 1.0, 1.0, True, 3), (6, 31, 0, 3.0, True, 1.0, 1.0, False, 0), (4, 256, 17, 0.5, False, 1.0, 0.0, False, 0), (4, 257, 16, 2.0, True, 1.0, 0.4, True, 0),
    (5, 1000, 300, 2.0, True, 1.0, 0.4, False, 8), (6, 1025, 8, 1.0, True, 1.0, 0.4, False, 0), (3, 2049, 64, 2.0, False, 1.0, 0.4, True, 1), (3, 4097, 1024, 2.0, True, 1.0, 0.4, False, 0),
    (2, 8193, 64, 2.0, True, 1.0, 0.4, False, 0), (3, 20000, 40, 2.0, True, 1.0, 0.4, True, 0), (2, 50001, 64, 0.7, True, 0.3, 0.4, False, 0), (70, 33000, 20, 1.0, False, 1.0, 0.0, True, 0),
    (66, 40001, 33, 2.0, True, 1.0, 0.3, False, 3), (65, 70000, 8, 2.0, True, 1.0, 0.3, False, 0), (2, 131072, 20, 1.0, False, 1.0, 0.0, False, 0), (1, 2 ** 20, 50, 2.0, True, 1.0, 0.3, False, 0),
    (4, 100, 12, 2.0, True, 0.0, 1.0, False, 0), (4, 100, 12, 2.0, False, -0.5, 2.0, True, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("t, v, k, temperature, rest, a, b, weighted, pad", DISTILS)
def test_distil(gpu, t, v, k, temperature, rest, a, b, weighted, pad, bf16):  # noqa: F811
    rng, element = np.random.default_rng(t * 17 + v), Element(bf16)
    nan = nan_of(element)
    stored, value, full, at, teacher = distil_inputs(rng, element, t, v, k)
    # places that take no part: none, out of range, of the lowest logit; and classes named again
    if k > 3:
        odd = rng.random((t, k))
        at = np.where(odd < 0.05, -1, np.where(odd < 0.1, v, np.where(odd < 0.2, at[:, :1], at))).astype(np.int32)
        teacher[rng.random((t, k)) < 0.05] = -np.inf
        teacher[(at < 0) | (at >= v)] = np.nan             # what lies in unused places must not matter
    normaliser = np.logaddexp.reduce(full / temperature, axis=1).astype(np.float32) if rest else None
    label = rng.integers(-1, v + 1, t).astype(np.int32)
    label[:: 2] = np.where(at[:: 2, 0] < v, at[:: 2, 0], 0) if k else label[:: 2]
    weights = rng.uniform(-1, 2, t).astype(np.float32) if weighted else None
    if weighted:
        weights[t // 2] = 0
        stored[t // 2], value[t // 2] = nan, np.nan        # an image of weight 0 may hold anything
    loss, off_loss, grad, off_grad = distil_reference(value, at, teacher, normaliser, label, weights, temperature, a, b, element)
    where = [gpu.up(x) for x in (padded(stored, pad, nan), at if k else None, teacher if k else None, normaliser, label, weights)]
    options = dict(dev_teacher_class=where[1], dev_teacher_logits=where[2], places=k, dev_teacher_normaliser=where[3], dev_label=where[4], dev_image_weights=where[5],
                   temperature=temperature, teacher_weight=a, label_weight=b, logit_stride=v + pad)
    with capi.Readout(1, element=element.id) as ro:
        losses, grads = gpu.new(t, np.float32), gpu.up(np.full((t, v + pad), nan, element.dtype))
        ro.distil(where[0], t, v, losses, None, **options)
        ro.synchronize()
        alone = gpu.down(losses, t, np.float32)
        assert_within(alone.astype(np.float64), loss, off_loss, "losses")
        for _ in range(2):
            ro.distil(where[0], t, v, losses, grads, gradient_stride=v + pad, **options)
            ro.synchronize()
            assert np.array_equal(gpu.down(losses, t, np.float32), alone)
            got = gpu.down(grads, (t, v + pad), element.dtype)
            assert np.array_equal(got[:, v:], np.full((t, pad), nan, element.dtype), equal_nan=not bf16)
            assert_within(element.values(got[:, :v]), grad, off_grad, "gradients")
            first = got if not _ else first
            assert np.array_equal(got, first, equal_nan=not bf16)
        ro.distil(where[0], t, v, None, grads, gradient_stride=v + pad, **options)
        ro.synchronize()
        assert np.array_equal(gpu.down(grads, (t, v + pad), element.dtype), got, equal_nan=not bf16)


def test_distil_gradients_of_the_restatement_against_differences():
    rng, element, d = np.random.default_rng(11), Element(False), 1e-5
    for rest, temperature in ((False, 1.0), (True, 2.0), (True, 0.7)):
        _, z, full, at, teacher = distil_inputs(rng, element, 4, 9, 3)
        at[1, 1], at[2, 2], teacher[3, 0] = -1, at[2, 0], -np.inf
        normaliser = np.logaddexp.reduce(full / temperature, axis=1).astype(np.float32) if rest else None
        label, weights = rng.integers(0, 9, 4), np.array([1.0, -0.5, 2.0, 0.3])
        grad = distil_reference(z, at, teacher, normaliser, label, weights, temperature, 0.7, 0.4, element)[2]
        for i in np.ndindex(*z.shape):
            if np.isneginf(z[i]):
                assert grad[i] == 0
                continue
            kept, loss = z[i], []
            for sign in (1, -1):
                z[i] = kept + sign * d
                loss.append(distil_reference(z, at, teacher, normaliser, label, weights, temperature, 0.7, 0.4, element)[0].sum())
            z[i] = kept
            assert abs((loss[0] - loss[1]) / (2 * d) - grad[i]) < 1e-7


@pytest.mark.gpu
@pytest.mark.parametrize("v", [10, 700, 9000, 140000])
def test_distil_of_rows_at_the_edges(gpu, v):  # noqa: F811
    """Rows whose mask leaves nothing or one class, of the type's lowest value, far apart, not finite; teachers that leave nothing."""
    rng, element, k = np.random.default_rng(12), Element(False), 3
    lowest = np.finfo(np.float32).min
    z = rng.standard_normal((10, v)).astype(np.float32)
    z[0] = -np.inf
    z[1, 1:] = -np.inf
    z[2] = lowest
    z[3, 1:] = lowest
    z[4, :2] = 1000, -1000
    z[5, v // 2], z[6, v - 1] = np.nan, np.inf
    at = np.tile(np.array([0, 1, 2], np.int32), (10, 1))
    teacher = np.tile(np.array([3, 1, 2], np.float32), (10, 1))
    at[3] = 0, -1, -1
    at[7], teacher[8], teacher[9, 1] = -1, -np.inf, np.nan
    label = np.array([0, 0, 1, 0, 0, 0, 0, -1, v, 0], np.int32)
    with capi.Readout(1) as ro:
        p = [gpu.up(a) for a in (z, at, teacher, label)]
        for rest in (False, True):
            norm = (np.full(10, 3.5, np.float32)) if rest else None
            losses, grads = gpu.new(10, np.float32), gpu.new((10, v), np.float32)
            ro.distil(p[0], 10, v, losses, grads, dev_teacher_class=p[1], dev_teacher_logits=p[2], places=k, dev_teacher_normaliser=gpu.up(norm), dev_label=p[3],
                      temperature=2.0, teacher_weight=1.0, label_weight=1.0)
            ro.synchronize()
            l, g = gpu.down(losses, 10, np.float32), gpu.down(grads, (10, v), np.float32).astype(np.float64)
            good = [0, 1, 2, 3, 4, 7, 8]
            want = distil_reference(z[good].astype(np.float64), at[good], teacher[good], None if norm is None else norm[good], label[good], None, 2.0, 1.0, 1.0, element)
            # (the fourth has a part of what is left against a probability of exp(-1.7e38): past float32's range where that is more than half)
            assert l[3] == (np.inf if want[0][3] > np.finfo(np.float32).max else l[3])
            l[3], want[0][3] = (0, 0) if np.isinf(l[3]) else (l[3], want[0][3])
            assert_within(l[good].astype(np.float64), want[0], want[1], "losses")
            assert_within(g[good], want[2], want[3], "gradients")
            assert l[0] == 0 and (g[0] == 0).all()
            assert np.isnan(l[[5, 6, 9]]).all() and np.isnan(g[[5, 6, 9]]).all()


# ------------------------------------------------------------------------------------------- calls that are refused, graphs

def refused(call, text):
    with pytest.raises(capi.PinkError) as e:
        call()
    assert e.value.status == -1 and text in str(e.value), str(e.value)


@pytest.mark.gpu
def test_calls_that_are_refused(gpu):  # noqa: F811
    shape = (8, 8, 8, 1)
    with capi.Readout(1) as ro:
        x = gpu.up(np.zeros((64, 64), np.float32))
        w = [x] * 6
        for width in (0, 2 ** 20 + 1):
            refused(lambda: ro.norm(x, 1, width, x, x, 1e-5, x), "width")
            refused(lambda: ro.norm_backward(x, 1, width, x, x, x, x, x), "width")
            refused(lambda: ro.norm_reserve(1, width), "width")
            refused(lambda: ro.distil(x, 1, width, x), "classes")
            refused(lambda: ro.distil_reserve(1, width), "classes")
        for epsilon in (-1.0, float("nan"), float("inf")):
            refused(lambda: ro.norm(x, 1, 8, x, x, epsilon, x), "epsilon")
        refused(lambda: ro.norm(None, 1, 8, x, x, 1e-5, x), "null")
        refused(lambda: ro.norm(x, 1, 8, x, x, 1e-5, None), "null")
        refused(lambda: ro.norm(x, 2, 8, x, x, 1e-5, x, x_stride=7), "overlap")
        refused(lambda: ro.norm(x, 2, 8, x, x, 1e-5, x, x_stride=9), "overlap")
        refused(lambda: ro.norm_backward(x, 2, 8, x, x, x, x + 1024, x + 1024, dx_stride=9), "overlap")
        refused(lambda: ro.norm(x, 2 ** 31, 8, x, x, 1e-5, x), "too many")
        refused(lambda: ro.norm_backward(x, 1, 8, x, None, x, x, x), "null")
        refused(lambda: ro.norm_backward(x, 1, 8, x, x, x, x, x, dx_stride=4), "overlap")
        for bad in ((0, 8, 8, 1), (8, 0, 8, 1), (8, 8, 0, 1), (2 ** 20 + 1, 8, 8, 1)):
            refused(lambda: ro.gated(bad, x, 1, w, x), "between 1 and")
            assert ro.gated_saved_bytes(bad, 1) == 0
        refused(lambda: ro.gated((8, 8, 8, 4), x, 1, w, x), "unknown activation")
        refused(lambda: ro.gated(shape, None, 1, w, x), "null")
        refused(lambda: ro.gated(shape, x, 1, [None] * 6, x), "null")
        refused(lambda: ro.gated(shape, x, 1, w, x, dev_saved=x + 16), "aligned")
        refused(lambda: ro.gated(shape, x, 2, w, x, y_stride=7), "overlap")
        refused(lambda: ro.gated(shape, x, 2 ** 31, w, x), "too many")
        refused(lambda: ro.gated_backward(shape, x, 1, w, None, x, [x] * 7), "null")
        refused(lambda: ro.gated_backward(shape, x, 1, w, x, x, [x] * 7, x_stride=7), "overlap")
        for options, text in ((dict(places=1025), "places"), (dict(temperature=0.0), "temperature"), (dict(temperature=float("inf")), "temperature"),
                              (dict(temperature=float("nan")), "temperature"), (dict(temperature=1e-40), "temperature"), (dict(teacher_weight=float("nan")), "finite"), (dict(label_weight=float("inf")), "finite"),
                              (dict(places=2), "null"), (dict(logit_stride=3), "overlap"), (dict(gradient_stride=3), "overlap")):
            refused(lambda: ro.distil(x, 1, 8, x, None, **options), text)
        refused(lambda: ro.distil(None, 1, 8, x), "null")
        refused(lambda: ro.distil(x, 4, 8, x, x), "may not lie")
        refused(lambda: ro.distil(x, 4, 8, x, x + 4 * 31), "may not lie")
        refused(lambda: ro.distil(x, 2 ** 31, 8, x), "too many")


@pytest.mark.gpu
def test_no_images(gpu):  # noqa: F811
    """Nothing to do; gradients of weights are sums over nothing."""
    with capi.Readout(1) as ro:
        ro.norm(None, 0, 8, None, None, 1e-5, None)
        ro.gated((8, 8, 8, 1), None, 0, [None] * 6, None)
        ro.distil(None, 0, 8, None)
        ro.norm_reserve(0, 8)
        ro.gated_reserve((8, 8, 8, 1), 0)
        ro.distil_reserve(0, 8)
        assert ro.gated_saved_bytes((8, 8, 8, 1), 0) == 0
        grads = [gpu.new(64, np.float32) for _ in range(8)]
        ro.norm_backward(None, 0, 8, None, None, None, None, None, grads[0], grads[1])
        ro.gated_backward((8, 8, 8, 1), None, 0, [None] * 6, None, None, [None] + grads[2:])
        ro.synchronize()
        for p, n in zip(grads, (8, 8, 64, 8, 64, 8, 64, 8)):
            assert (gpu.down(p, n, np.float32) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
def test_a_step_as_it_is_used(gpu, bf16):  # noqa: F811
    """Layer norm, a block on it, its answers as logits, and back: called, recorded on a given stream, and recorded on another handle's workspace."""
    rng, element = np.random.default_rng(13), Element(bf16)
    t, f, h, v, k = 300, 200, 136, 40, 4
    stored, value = gated_inputs(rng, element, t, f, h, v, True, False)
    w, b = element.store(1 + 0.2 * rng.standard_normal(f))[0], element.store(0.2 * rng.standard_normal(f))[0]
    _, _, full, at, teacher = distil_inputs(rng, element, t, v, k, masked=False)
    label, shape = rng.integers(0, v, t).astype(np.int32), (f, h, v, capi.ACT_SILU)
    p = {i: gpu.up(stored[i]) for i in ("x",) + WEIGHTS} | {"w": gpu.up(w), "b": gpu.up(b), "at": gpu.up(at), "teacher": gpu.up(teacher), "label": gpu.up(label)}
    weights = [p[i] for i in WEIGHTS]
    sizes = {"n": (t, f), "y": (t, v), "dy": (t, v), "dn": (t, f), "dx": (t, f), "dw": f, "db": f, **{"d" + i: stored[i].shape for i in WEIGHTS}}
    out = {i: gpu.new(s, element.dtype) for i, s in sizes.items()} | {i: gpu.new(t, np.float32) for i in ("mean", "scale", "losses")}

    def step(ro, saved):
        ro.norm(p["x"], t, f, p["w"], p["b"], EPSILON, out["n"], out["mean"], out["scale"])
        ro.gated(shape, out["n"], t, weights, out["y"], dev_saved=saved)
        ro.distil(out["y"], t, v, out["losses"], out["dy"], dev_teacher_class=p["at"], dev_teacher_logits=p["teacher"], places=k, dev_label=p["label"], temperature=2.0, label_weight=0.5)
        ro.gated_backward(shape, out["n"], t, weights, saved, out["dy"], [out["dn"]] + [out["d" + i] for i in WEIGHTS])
        ro.norm_backward(p["x"], t, f, p["w"], out["mean"], out["scale"], out["dn"], out["dx"], out["dw"], out["db"])

    def results():
        return {i: gpu.down(out[i], s, element.dtype) for i, s in sizes.items()} | {"losses": gpu.down(out["losses"], t, np.float32)}

    with capi.Readout(1, element=element.id) as ro, capi.Readout(1, element=element.id) as other:
        saved = gpu.new(ro.gated_saved_bytes(shape, t), np.int8)
        step(ro, saved)
        ro.synchronize()
        want = results()
        n = norm_reference(value["x"], element.values(w), element.values(b), None, None, element)["y"]
        assert_within(element.values(want["n"]), *n, "n")
        y = gated_reference({**value, "x": element.values(want["n"])}, element, "silu", element.values(want["dy"]))
        for i in ("y", "dgate", "dup", "ddown", "dgate_bias", "dup_bias", "ddown_bias"):
            assert_within(element.values(want[i]), *y[i], i)
        assert_within(element.values(want["dn"]), *y["dx"], "dn")
        loss = distil_reference(element.values(want["y"]), at, teacher, None, label, None, 2.0, 1.0, 0.5, element)
        assert_within(want["losses"].astype(np.float64), loss[0], loss[1], "losses")
        assert_within(element.values(want["dy"]), loss[2], loss[3], "dy")
        back = norm_reference(value["x"], element.values(w), element.values(b), element.values(want["dn"]), None, element)
        for i in ("dx", "dw", "db"):
            assert_within(element.values(want[i]), *back[i], i)
        for handle in (ro, other):
            handle.gated_reserve(shape, t)
            handle.norm_reserve(t, f)
            handle.distil_reserve(t, v)
        recordings = [Recording(gpu, handle) for handle in (ro, other)]
        for recording in recordings:
            with recording:
                step(recording.ro, saved)
        for _ in range(3):
            for recording in recordings:
                for i, s in sizes.items():
                    gpu.write(out[i], np.zeros(s, element.dtype))
                recording.launch()
                recording.ro.synchronize()
                got = results()
                assert all(np.array_equal(got[i], want[i]) for i in want)
        for recording in recordings:
            recording.close()


@pytest.mark.gpu
def test_recorded_calls_do_not_grow_the_workspace(gpu):  # noqa: F811
    shape, x = (64, 64, 64, capi.ACT_SILU), gpu.up(np.zeros((3000, 64), np.float32))
    w, saved = [x, None, x, None, x, None], gpu.new(3000 * 64 * 12, np.int8)
    calls = [lambda ro: ro.gated(shape, x, 3000, w, x), lambda ro: ro.gated_backward(shape, x, 3000, w, saved, x, [x, None, None, None, None, None, None]),
             lambda ro: ro.norm_backward(x, 3000, 64, None, x, x, x, None, x, None), lambda ro: ro.distil(x, 1, 100000, None, x + 4 * 100000)]
    for call in calls:
        with capi.Readout(1) as ro:
            recording = Recording(gpu, ro)
            with recording:
                with pytest.raises(capi.PinkError) as e:
                    call(ro)
                assert e.value.status == -4 and "larger workspace" in str(e.value)
            recording.close()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
def test_a_reserved_workspace_is_enough_for_fewer_images(gpu, bf16):  # noqa: F811
    """Fewer images than were reserved for may be worked on otherwise: a recorded call of theirs does not have to grow the workspace."""
    element, (f, h, o, v, most) = Element(bf16), (1600, 640, 24, 70000, 3000)
    shape, zeros = (f, h, o, capi.ACT_SILU), lambda *s: gpu.up(np.zeros(s, element.dtype))
    x, dy, dx, weights = zeros(most, f), zeros(most, o), zeros(most, f), [zeros(h, f), zeros(h), zeros(h, f), zeros(h), zeros(o, h), zeros(o)]
    grads, z, dz, m = [zeros(h, f), zeros(h), zeros(h, f), zeros(h), zeros(o, h), zeros(o)], zeros(80, v), zeros(80, v), gpu.up(np.zeros(most, np.float32))
    for t in (1, 17, 40, 64, 100, 200, 320, 600, 1000, 1100, 2000):
        with capi.Readout(1, element=element.id) as ro:
            saved = gpu.new(ro.gated_saved_bytes(shape, t), np.int8)
            for calls in (1, 2):
                if calls == 1:
                    ro.gated_reserve(shape, most)
                else:
                    ro.norm_reserve(most, f)
                    ro.distil_reserve(80, v)
                recording = Recording(gpu, ro)
                with recording:
                    if calls == 1:
                        ro.gated(shape, x, t, weights, dy, dev_saved=saved)
                        ro.gated_backward(shape, x, t, weights, saved, dy, [dx] + grads)
                    else:
                        ro.norm_backward(x, t, f, None, m, m, dx, dx, grads[0], grads[2])
                        ro.distil(z, min(t, 80), v, m, dz)
                recording.close()


@pytest.mark.gpu
def test_gated_over_a_residual_of_other_strides(gpu):  # noqa: F811
    """Answers take the residual's place row by row, or not at all."""
    rng, element, (t, f, h) = np.random.default_rng(20), Element(False), (40, 24, 16)
    stored, _ = gated_inputs(rng, element, t, f, h, f, True, True)
    weights, shape = [gpu.up(stored[i]) for i in WEIGHTS], (f, h, f, capi.ACT_SILU)
    x, wide = gpu.up(stored["x"]), padded(stored["residual"], 5, np.nan)
    with capi.Readout(1) as ro:
        for images in (2, t):
            for strides in ((0, f + 5), (f + 5, 0), (f + 5, f + 6)):
                place = gpu.up(wide)
                refused(lambda: ro.gated(shape, x, images, weights, place, dev_residual=place, residual_stride=strides[0], y_stride=strides[1]), "overlap")
                assert np.array_equal(gpu.down(place, wide.shape, np.float32), wide, equal_nan=True)
        for images, strides in ((t, (f + 5, f + 5)), (1, (0, f + 5)), (1, (f + 5, 0))):
            place, y = gpu.up(wide), gpu.new((images, f), np.float32)
            ro.gated(shape, x, images, weights, y, dev_residual=place, residual_stride=f + 5)
            ro.gated(shape, x, images, weights, place, dev_residual=place, residual_stride=strides[0], y_stride=strides[1])
            ro.synchronize()
            got = gpu.down(place, wide.shape, np.float32)
            assert np.array_equal(got[:images, :f], gpu.down(y, (images, f), np.float32))
            assert np.isnan(got[:, f:]).all() and np.array_equal(got[images:, :f], wide[images:, :f])
        # x has been read when answers are written, whatever its stride
        place, y = gpu.up(padded(stored["x"], 5, np.nan)), gpu.new((t, f), np.float32)
        ro.gated(shape, place, t, weights, y, x_stride=f + 5)
        ro.gated(shape, place, t, weights, place, x_stride=f + 5)
        ro.synchronize()
        assert np.array_equal(gpu.down(place, (t, f), np.float32), gpu.down(y, (t, f), np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("v", [10, 700, 9000, 140000])
def test_distil_of_rows_that_are_not_finite_and_have_nothing_to_learn(gpu, v, bf16):  # noqa: F811
    """Without a label, and without a place that takes part: NaN all the same, and rows that are finite 0."""
    rng, element = np.random.default_rng(21), Element(bf16)
    z = rng.standard_normal((6, v)).astype(np.float32)
    z[1, v // 2], z[2, v - 1], z[3, 0], z[4], z[5] = np.nan, np.inf, np.nan, np.nan, -np.inf
    teachers = {"out of range": (np.full((6, 2), -1, np.int32), np.ones((6, 2), np.float32)), "lowest": (np.tile(np.array([0, v - 1], np.int32), (6, 1)), np.full((6, 2), -np.inf, np.float32)),
                "none": (None, None)}
    logits = gpu.up(element.store(z)[0])
    with capi.Readout(1, element=element.id) as ro:
        for name, (at, teacher) in teachers.items():
            p, k = (gpu.up(at), gpu.up(teacher)), 0 if at is None else 2
            for label in (None, np.full(6, -1, np.int32), np.full(6, v, np.int32)):
                for weight in (0.0, 1.0):
                    for grads in (None, gpu.new((6, v), element.dtype)):
                        losses = gpu.up(np.full(6, 7.0, np.float32))
                        ro.distil(logits, 6, v, losses, grads, dev_teacher_class=p[0], dev_teacher_logits=p[1], places=k, dev_label=gpu.up(label), temperature=2.0,
                                  teacher_weight=weight, label_weight=1.0)
                        ro.synchronize()
                        got = gpu.down(losses, 6, np.float32)
                        assert (got[[0, 5]] == 0).all() and np.isnan(got[1:5]).all(), (name, weight, got)
                        if grads:
                            g = element.values(gpu.down(grads, (6, v), element.dtype))
                            assert (g[[0, 5]] == 0).all() and np.isnan(g[1:5]).all(), (name, weight)


def few_images(rng, t, f, h, o):
    """A bfloat16 block's inputs with the residual nearly the rest's opposite, so that what is left shows the sum's own roundings; and answers with a bound for
    hidden values that go on as two bfloat16 values: what the second leaves of a half step is a half step of that, or of the least number."""
    element = Element(True)
    stored, value = gated_inputs(rng, element, t, f, h, o, True, False)
    stored["residual"], value["residual"] = element.store(-gated_reference(value, element, "silu", None)["y"][0])
    y, off = gated_reference(value, types.SimpleNamespace(u=element.u ** 2, bf16=True), "silu", None)["y"]
    off = off + 2.0 ** -126 * np.abs(value["down"]).sum(1)
    return element, stored, value, y, off + element.u * (np.abs(y) * 1.02 + off)


FEW = [(1, 24, 16, 40), (3, 130, 33, 41), (16, 40, 24, 64), (17, 33, 31, 39), (32, 136, 64, 24), (16, 64, 2040, 2048), (16, 64, 2056, 2048), (32, 48, 4104, 1032)]


@pytest.mark.parametrize("t, f, h, o", FEW[:5])
def test_the_bound_of_few_images_tells_one_rounding_of_hidden_values_from_two(t, f, h, o):
    element, stored, value, y, off = few_images(np.random.default_rng(22), t, f, h, o)
    a, b = value["x"] @ value["gate"].T + value["gate_bias"], value["x"] @ value["up"].T + value["up_bias"]
    hidden = a / (1 + np.exp(-a)) * b
    once = element.store(hidden)[1]
    twice = once + element.store(hidden - once)[1]
    more = value["down_bias"] + value["residual"]
    assert (np.abs(twice @ value["down"].T + more - y) <= off).all() and (np.abs(once @ value["down"].T + more - y) > off).any()


@pytest.mark.gpu
@pytest.mark.parametrize("t, f, h, o", FEW)
def test_few_images_without_a_backward_pass_have_one_rounding(gpu, t, f, h, o):  # noqa: F811
    """Whatever the number of weights; with what a backward pass needs, as the block's bound says."""
    element, stored, value, y, off = few_images(np.random.default_rng(22), t, f, h, o)
    shape, p = (f, h, o, capi.ACT_SILU), {i: gpu.up(v) for i, v in stored.items()}
    with capi.Readout(1, element=element.id) as ro:
        out = gpu.new((t, o), np.uint16)
        for keep in (None, gpu.new(ro.gated_saved_bytes(shape, t), np.int8)):
            ro.gated(shape, p["x"], t, [p[i] for i in WEIGHTS], out, dev_residual=p["residual"], dev_saved=keep)
            ro.synchronize()
            assert_within(element.values(gpu.down(out, (t, o), np.uint16)), *((y, off) if keep is None else gated_reference(value, element, "silu", None)["y"]), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 16, 30])
def test_few_images_by_weights_that_are_not_finite(gpu, t):  # noqa: F811
    """An infinite weight gives infinite answers, not NaN, also where the second part of a hidden value is 0 or of the other sign; so does an infinite hidden
    value; what is NaN stays NaN, and other answers are as they would be."""
    rng, element, (f, h, o) = np.random.default_rng(23), Element(True), (40, 24, 16)
    stored, value = gated_inputs(rng, element, t, f, h, o, True, False)
    shape, p = (f, h, o, capi.ACT_SILU), {i: gpu.up(v) for i, v in stored.items()}
    a, b = value["x"] @ value["gate"].T + value["gate_bias"], value["x"] @ value["up"].T + value["up_bias"]
    hidden = a / (1 + np.exp(-a)) * b
    down = stored["down"].copy()
    down[3, 5], down[7, 2], down[9, 0] = 0x7f80, 0xff80, 0x7fc0          # infinity, minus infinity, NaN
    with capi.Readout(1, element=element.id) as ro:
        y, wrong = gpu.new((t, o), np.uint16), gpu.new((t, o), np.uint16)
        ro.gated(shape, p["x"], t, [p[i] for i in WEIGHTS], y)
        ro.gated(shape, p["x"], t, [gpu.up(down) if i == "down" else p[i] for i in WEIGHTS], wrong)
        ro.synchronize()
        want, got = (element.values(gpu.down(v, (t, o), np.uint16)) for v in (y, wrong))
        want[:, 3], want[:, 7], want[:, 9] = np.sign(hidden[:, 5]) * np.inf, -np.sign(hidden[:, 2]) * np.inf, np.nan
        assert np.array_equal(got, want, equal_nan=True)
        # h past what is finite: a and b of 2^100 in its fourth place
        gate_bias, up_bias = stored["gate_bias"].copy(), stored["up_bias"].copy()
        gate_bias[3] = up_bias[3] = element.store(np.array([2.0 ** 100]))[0][0]
        ro.gated(shape, p["x"], t, [gpu.up(gate_bias) if i == "gate_bias" else gpu.up(up_bias) if i == "up_bias" else p[i] for i in WEIGHTS], wrong)
        ro.synchronize()
        assert np.array_equal(element.values(gpu.down(wrong, (t, o), np.uint16)), np.tile(np.sign(value["down"][:, 3]) * np.inf, (t, 1)))


def free_bytes(gpu):
    free, total = C.c_size_t(), C.c_size_t()
    gpu.ok(gpu.rt.hipMemGetInfo(C.byref(free), C.byref(total)))
    return free.value


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
def test_a_workspace_reserved_for_few_images_is_small(gpu, bf16):  # noqa: F811
    """Hidden values and their gradients of 16 images take 4 MB at most, and runs of few tiles 1536 of 64 x 64 float32 numbers; the weights' gradients, of 134 MB
    each, are cut from 1024 images on."""
    with capi.Readout(1, element=Element(bf16).id) as ro:
        before = free_bytes(gpu)
        ro.gated_reserve((4096, 8192, 4096, capi.ACT_SILU), 16)
        assert before - free_bytes(gpu) <= 4 * 2 ** 20 + 1536 * 64 * 64 * 4 + 2 * 2 ** 20        # (an allocation is of whole 2 MiB)


@pytest.mark.gpu
@pytest.mark.parametrize("f, h, o, most, bf16", [(1930, 1150, 24, 2300, False), (24, 1930, 2300, 2300, False), (1200, 2000, 8, 12000, True)])
def test_a_reserved_workspace_is_enough_for_gradients_in_runs(gpu, f, h, o, most, bf16):  # noqa: F811
    """Weights' gradients of some hundred tiles of 128 x 128, which go by the number of images into runs: none of these calls has to grow what was reserved."""
    element, shape = Element(bf16), (f, h, o, capi.ACT_SILU)
    x, dy, dx, weights, grads = (gpu.new(s, element.dtype) for s in ((most, f), (most, o), (most, f), (3, h, max(f, o)), (3, h, max(f, o))))
    for t in (1, 33, 500, 1023, 1024, 1536, 2200, most):
        with capi.Readout(1, element=element.id) as ro:
            saved = gpu.new(ro.gated_saved_bytes(shape, t), np.int8)
            ro.gated_reserve(shape, most)
            recording = Recording(gpu, ro)
            with recording:
                ro.gated(shape, x, t, [weights] * 6, dy, dev_saved=saved)
                ro.gated_backward(shape, x, t, [weights] * 6, saved, dy, [dx] + [grads] * 6)
            recording.close()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("t, v, k, temperature, rest, a, b, weighted, pad", [
    # rows that a block of 1024 threads holds in 4, 8 and 16 chunks each, of either type, odd and exactly full
    (66, 20001, 33, 2.0, True, 1.0, 0.3, True, 3), (66, 32768, 20, 0.7, True, 1.0, 0.4, False, 0), (65, 65536, 8, 4.0, True, 1.0, 0.3, True, 0), (67, 16384, 300, 1.0, False, 0.5, 1.0, False, 8),
])
def test_distil_of_many_long_rows(gpu, t, v, k, temperature, rest, a, b, weighted, pad, bf16):  # noqa: F811
    test_distil(gpu, t, v, k, temperature, rest, a, b, weighted, pad, bf16)


@pytest.mark.gpu
def test_calls_after_one_that_found_no_memory(gpu):  # noqa: F811
    """A workspace that there is no memory for is refused, and the calls after that are as they were."""
    rng, (t, n) = np.random.default_rng(24), (40, 100)
    x = rng.standard_normal((t, n)).astype(np.float32)
    with capi.Readout(1) as ro:
        at, y, again, dw = gpu.up(x), gpu.new((t, n), np.float32), gpu.new((t, n), np.float32), gpu.new(n, np.float32)
        mean, scale = gpu.new(t, np.float32), gpu.new(t, np.float32)
        ro.norm(at, t, n, None, None, EPSILON, y, mean, scale)
        for _ in range(2):
            with pytest.raises(capi.PinkError) as e:
                ro.gated_reserve((2 ** 20, 2 ** 20, 2 ** 20, capi.ACT_SILU), 2 ** 30)            # (2^53 bytes)
            assert e.value.status == -2 and "memory" in str(e.value), (e.value.status, str(e.value))
            ro.norm(at, t, n, None, None, EPSILON, again)
            with pytest.raises(capi.PinkError) as e:
                capi.Context(4000, 1, 64, 10000, 1, False, 32)                                   # (1.6 TB of neurons)
            assert e.value.status == -2, (e.value.status, str(e.value))
            ro.norm(at, t, n, None, None, EPSILON, again)
            ro.norm_backward(at, t, n, None, mean, scale, at, None, dw)                          # (with a workspace)
        ro.synchronize()
        assert np.array_equal(gpu.down(again, (t, n), np.float32), gpu.down(y, (t, n), np.float32))
