"""What is timed of a read-out's blocks and of its loss on classes: layer norm, the gated feed-forward block, distillation.

Before the neurons' own models a read-out may refine its features by blocks that all neurons share, x + gated(norm(x)); its answers may be
logits of classes, learned from labels and from a teacher of which the top logits of every image were kept.  A case is one
call pattern of one operator, `op`:

  norm      layer norm of rows of features; with "train" also the gradients of the rows, of the weight and of the bias
  gated     D (f(G x + g) * (U x + u)) + d, added to a residual where there is one; with "train" also all gradients
  distil    an image's loss against its teacher and its label; with "train" also the gradients of the logits

The plain forms hold all in 32 bits and round once at the end.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_EPSILON = 1e-5


# ---------------------------------------------------------------------------------------------------------------- cases

def _norm(name, images, width, type="bf16", train=False, pad=0):
    c = dict(op="norm", images=images, width=width, type=type, train=train, pad=pad)
    return dict(c, name=name) if name else c


def _gated(name, images, features, hidden, outputs, activation="silu", type="bf16", bias=True, residual=False, train=False, pad=0):
    c = dict(op="gated", images=images, features=features, hidden=hidden, outputs=outputs, activation=activation, type=type, bias=bias,
             residual=residual, train=train, pad=pad)
    return dict(c, name=name) if name else c


def _distil(name, images, classes, places, type="bf16", rest=False, label=False, train=True, temperature=2.0, pad=0):
    c = dict(op="distil", images=images, classes=classes, places=places, type=type, rest=rest, label=label, train=train,
             temperature=temperature, pad=pad)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one image's 32 x 32 region: latency counts
        _norm("norm-1", 1, 1024),
        # a batch's 45 x 45 regions in float32, a training step: rows of an odd length
        _norm("norm-train-301-f32-odd", 301, 2025, "f32", True),
        # a training step over many wide rows
        _norm("norm-train-16384", 16384, 8192, train=True),
        # one image through a block
        _gated("gated-1", 1, 1024, 2048, 1024),
        # a handful of images through a wide block: its weights have to be read
        _gated("gated-16", 16, 4096, 8192, 4096, bias=False, residual=True),
        # a batch's 45 x 45 regions to the distances of a hexagonal map of 331 neurons, odd sizes throughout
        _gated("gated-301-f32-odd", 301, 2025, 1000, 331, "gelu", "f32"),
        # small pictures (28 x 28), a training step in float32
        _gated("gated-train-500-f32", 500, 784, 256, 784, "relu", "f32", residual=True, train=True),
        # a training step over many images
        _gated("gated-train-8192", 8192, 2048, 8192, 2048, residual=True, train=True),
        # one image's answer among a thousand classes
        _distil("distil-1", 1, 1000, 10, "f32"),
        # a batch of small pictures, ten classes, labels beside the teacher
        _distil("distil-500-f32", 500, 10, 3, "f32", rest=True, label=True, temperature=4.0),
        # many classes, an odd number, and what the teacher's top logits leave
        _distil("distil-4001-odd", 4001, 50001, 64, rest=True, label=True),
        # the longest rows
        _distil("distil-2048-long", 2048, 131072, 20, temperature=1.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MAX_VALUES = {"norm": 16384 * 8192, "distil": 2048 * 131072}
_MAX_FLOPS = 2.0e12          # of a drawn pass: the largest listed one has 2.5e12


def draw(rng):
    op = rng.choice(("norm", "gated", "gated", "distil"))
    type, pad = rng.choice(("bf16", "bf16", "f32")), rng.choice((0, 0, 0, 3, 8))
    most = 2 if type == "f32" else 1
    if op == "norm":
        width = rng.choice((784, 1024, 1936, 2025, 331, _log(rng, 1, 16384), 8 * _log(rng, 1, 2048)))
        return _norm(None, _log(rng, 1, max(1, min(16384, _MAX_VALUES["norm"] // (width * most)))), width, type, rng.random() < 0.6, pad)
    if op == "distil":
        classes = rng.choice((10, 1000, _log(rng, 2, 131072), 8 * _log(rng, 1, 16384)))
        images = _log(rng, 1, max(1, min(16384, _MAX_VALUES["distil"] // (classes * most))))
        return _distil(None, images, classes, min(classes, _log(rng, 1, 128)), type, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.7,
                       rng.choice((1.0, 2.0, 4.0, 0.7)), pad)
    features = rng.choice((784, 1024, 1936, 2025, 64 * _log(rng, 1, 64), _log(rng, 16, 4096)))
    hidden = rng.choice((64 * _log(rng, 1, 128), _log(rng, 16, 8192)))
    outputs = rng.choice((features, features, 8 * _log(rng, 1, 512), _log(rng, 1, 4096)))
    residual, train = rng.random() < 0.5, rng.random() < 0.5
    each = (6.0 if train else 2.0) * hidden * (2 * features + outputs)
    images = _log(rng, 1, max(1, min(16384, int(_MAX_FLOPS / each / (4 if type == "f32" else 1)))))
    return _gated(None, images, features, hidden, outputs, rng.choice(("identity", "relu", "gelu", "silu", "silu")), type, rng.random() < 0.5,
                  residual, train, pad)


def work(case):
    """Inputs read once, outputs written once."""
    c, size = case, 2.0 if case["type"] == "bf16" else 4.0
    t = c["images"]
    if c["op"] == "norm":
        n = c["width"]
        return {"bytes": size * (2 * t * n + 2 * n + ((2 * t * n + 2 * n) if c["train"] else 0)), "flops": (20.0 if c["train"] else 8.0) * t * n}
    if c["op"] == "gated":
        f, h, o = c["features"], c["hidden"], c["outputs"]
        weights = h * (2 * f + o) + ((2 * h + o) if c["bias"] else 0)
        moved = size * (t * f + weights + t * o * (2 if c["residual"] else 1))
        if c["train"]:
            moved += size * (t * o + t * f + weights)
        return {"bytes": moved, "flops": (6.0 if c["train"] else 2.0) * t * h * (2 * f + o)}
    v, k = c["classes"], c["places"]
    moved = size * t * v * (2 if c["train"] else 1) + 8.0 * t * k + 8.0 * t + (4.0 * t if c["rest"] else 0) + (4.0 * t if c["label"] else 0)
    return {"bytes": moved, "flops": (14.0 if c["train"] else 6.0) * t * v}


# --------------------------------------------------------------------------------------------------------------- inputs

_readouts = {}


def _readout(c):
    """The handle that a program keeps for its read-out, on PyTorch's stream."""
    if not own:
        return None
    from pink_amd import capi
    if c["type"] not in _readouts:
        r = capi.Readout(1, element=capi.ELEMENT_BF16 if c["type"] == "bf16" else capi.ELEMENT_F32)
        r.set_stream(torch.cuda.current_stream().cuda_stream)
        _readouts[c["type"]] = r
    return _readouts[c["type"]]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, scale=1.0, type=torch.float32):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(type)


def _rand(gen, *shape):
    return torch.rand(shape, device="cuda", generator=gen)


def _prepare_norm(c, seed):
    gen, type = _generator(seed), _TYPES[c["type"]]
    t, n = c["images"], c["width"]
    # rows with a level and a spread of their own, as images have
    wide = (_randn(gen, t, n + c["pad"]) * (0.2 + _rand(gen, t, 1)) + 2 * _randn(gen, t, 1)).to(type)
    s = {"case": c, "x": wide[:, :n], "weight": (1 + _randn(gen, n, scale=0.2)).to(type), "bias": _randn(gen, n, scale=0.2, type=type),
         "y": torch.empty((t, n), dtype=type, device="cuda"), "readout": _readout(c)}
    if c["train"]:
        s["dy"] = _randn(gen, t, n, type=type)
        s["dx"] = torch.empty((t, n), dtype=type, device="cuda")
        s["dweight"], s["dbias"] = torch.empty(n, dtype=type, device="cuda"), torch.empty(n, dtype=type, device="cuda")
        s["mean"], s["scale"] = torch.empty(t, device="cuda"), torch.empty(t, device="cuda")
    return s


_GATED = (("gate", "hidden", "features"), ("gate_bias", "hidden"), ("up", "hidden", "features"), ("up_bias", "hidden"), ("down", "outputs", "hidden"),
          ("down_bias", "outputs"))


def _prepare_gated(c, seed):
    gen, type = _generator(seed), _TYPES[c["type"]]
    t, f, o = c["images"], c["features"], c["outputs"]
    wide = _randn(gen, t, f + c["pad"], type=type)                     # as a layer norm leaves them
    s = {"case": c, "x": wide[:, :f], "y": torch.empty((t, o), dtype=type, device="cuda"), "readout": _readout(c),
         "residual": _randn(gen, t, o, type=type) if c["residual"] else None}
    for name, *shape in _GATED:
        shape = [c[x] for x in shape]
        if len(shape) == 2:
            s[name] = _randn(gen, *shape, scale=1.2 / math.sqrt(shape[1]), type=type)
        else:
            s[name] = _randn(gen, *shape, scale=0.3, type=type) if c["bias"] else None
    if c["train"]:
        s["dy"], s["dx"] = _randn(gen, t, o, type=type), torch.empty((t, f), dtype=type, device="cuda")
        for name, *_ in _GATED:
            s["d" + name] = None if s[name] is None else torch.empty_like(s[name])
    return s


def _prepare_distil(c, seed):
    gen, type = _generator(seed), _TYPES[c["type"]]
    t, v, k = c["images"], c["classes"], c["places"]
    student = _randn(gen, t, v + c["pad"], scale=2.0)
    teacher = student[:, :v] + _randn(gen, t, v)                       # the student is on its way to its teacher
    top = teacher.topk(k, dim=1)
    # classes that take no part; not in the smallest questions
    if v >= 100:
        student[:, :v].masked_fill_(_rand(gen, 1, v) < 0.01, -math.inf)
    student = student.to(type)
    at = top.indices.to(torch.int32)
    # a tenth of the images have fewer places, one has none
    kept = torch.where(_rand(gen, t, 1) < 0.1, 1 + (k - 1) // 2, k)
    if t > 8:
        kept[t // 2] = 0
    at = torch.where(torch.arange(k, device="cuda")[None, :] < kept, at, -1).contiguous()
    weights = (0.5 + _rand(gen, t)) / t
    if t > 8:
        weights[t // 3] = 0                                            # rows that fill up a batch
    s = {"case": c, "logits": student[:, :v], "class": at, "teacher": top.values.contiguous(), "weights": weights, "readout": _readout(c),
         "normaliser": torch.logsumexp(teacher / c["temperature"], 1) if c["rest"] else None, "label": None,
         "losses": torch.empty(t, device="cuda"), "dlogits": torch.empty((t, v), dtype=type, device="cuda") if c["train"] else None}
    if c["label"]:
        label = (teacher - torch.log(-torch.log(_rand(gen, t, v).clamp(1e-7, 1 - 1e-7)))).argmax(1).to(torch.int32)
        s["label"] = torch.where(_rand(gen, t) < 0.05, -1, label)      # some images have none
    return s


_TEACHER_WEIGHT, _LABEL_WEIGHT = 0.7, 0.3


def prepare(case, seed):
    return {"norm": _prepare_norm, "gated": _prepare_gated, "distil": _prepare_distil}[case["op"]](case, seed)


# ---------------------------------------------------------------------------------------------------------- plain forms

def _plain_norm(s):
    type = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    off = x - x.mean(1, keepdim=True)
    scale = 1 / torch.sqrt((off * off).mean(1, keepdim=True) + _EPSILON)
    form = off * scale
    out = {"y": form * w + s["bias"].float()}
    if s["case"]["train"]:
        dy = s["dy"].float()
        g = dy * w
        out["dx"] = scale * (g - g.mean(1, keepdim=True) - form * (g * form).mean(1, keepdim=True))
        out["dweight"], out["dbias"] = (dy * form).sum(0), dy.sum(0)
    return {name: v.to(type) for name, v in out.items()}


_ROOT_HALF, _ROOT_TWO_PI = math.sqrt(0.5), math.sqrt(2 * math.pi)


def _activate(kind, a):
    if kind == "identity":
        return a
    if kind == "relu":
        return a.clamp(min=0)
    if kind == "gelu":
        return 0.5 * a * (1 + torch.erf(a * _ROOT_HALF))
    return a / (1 + torch.exp(-a))


def _slope(kind, a):
    if kind == "identity":
        return torch.ones_like(a)
    if kind == "relu":
        return (a > 0).to(a.dtype)
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(a * _ROOT_HALF)) + a * torch.exp(-0.5 * a * a) / _ROOT_TWO_PI
    sig = 1 / (1 + torch.exp(-a))
    return sig * (1 + a * (1 - sig))


def _plain_gated(s):
    c, type = s["case"], s["x"].dtype
    x, gate, up, down = (s[name].float() for name in ("x", "gate", "up", "down"))
    a, u = x @ gate.t(), x @ up.t()
    if c["bias"]:
        a, u = a + s["gate_bias"].float(), u + s["up_bias"].float()
    f = _activate(c["activation"], a)
    h = f * u
    y = h @ down.t()
    if c["bias"]:
        y = y + s["down_bias"].float()
    if c["residual"]:
        y = y + s["residual"].float()
    out = {"y": y}
    if c["train"]:
        dy = s["dy"].float()
        dh = dy @ down
        da, du = dh * u * _slope(c["activation"], a), dh * f
        out |= {"dx": da @ gate + du @ up, "dgate": da.t() @ x, "dup": du.t() @ x, "ddown": dy.t() @ h}
        if c["bias"]:
            out |= {"dgate_bias": da.sum(0), "dup_bias": du.sum(0), "ddown_bias": dy.sum(0)}
    return {name: v.to(type) for name, v in out.items()}


def _powers(z, temperature):
    """exp((z - its row's largest) / temperature) over the classes that take part, those above minus infinity; their sum in 64 bits."""
    top = z.amax(1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    e = torch.exp((z - top) / temperature)
    return top, e, e.sum(1, keepdim=True, dtype=torch.float64)


def _plain_distil(s):
    """What a loss is a small difference of, places' logarithms and sums, is held in 64 bits; all that is as long as a row in 32."""
    c, z, temperature = s["case"], s["logits"].float(), s["case"]["temperature"]
    t, v = c["images"], c["classes"]
    at = s["class"].long()
    named = at.clamp(0, v - 1)
    part = (at >= 0) & (z.gather(1, named) > -math.inf)
    top, e, total = _powers(z, temperature)
    logq = (z.gather(1, named) - top).double() / temperature - torch.log(total)
    teacher = torch.where(part, s["teacher"].double() / temperature, -math.inf)
    if c["rest"]:
        logp = teacher - s["normaliser"].double()[:, None]
    else:
        most = teacher.amax(1, keepdim=True)
        logp = teacher - torch.where(torch.isinf(most), 0.0, most)
        logp = logp - torch.log(torch.exp(logp).sum(1, keepdim=True))
    p = torch.where(part, torch.exp(logp), 0.0)
    share = p.sum(1, keepdim=True)
    loss = torch.where(part, p * (logp - logq), 0.0).sum(1)
    if c["rest"]:
        held = torch.zeros((t, v + 1), dtype=torch.bool, device=z.device).scatter_(1, torch.where(part, at, v), True)[:, :v]
        others = torch.where(held, 0.0, e).sum(1, keepdim=True, dtype=torch.float64)
        left = torch.where(others > 0, (1 - share).clamp(min=0), 0.0)
        loss = loss + torch.where(left > 0, left * (torch.log(left) - torch.log(others / total)), 0.0).view(-1)
        share = share + left
        factor = torch.where(held, (share / total).float(), (share / total - left / torch.where(others > 0, others, 1.0)).float())
    else:
        factor = (share / total).float()
    if c["train"]:
        # (a place without a class adds nothing to class 0)
        dz = torch.where(e > 0, e * factor, 0.0).scatter_add_(1, named, -p.float()) * (_TEACHER_WEIGHT * temperature)
    loss = loss * (_TEACHER_WEIGHT * temperature * temperature)
    if c["label"]:
        label = s["label"].long()
        of = label.clamp(0, v - 1)[:, None]
        has = (label[:, None] >= 0) & (z.gather(1, of) > -math.inf)
        top, e, total = _powers(z, 1.0)
        loss = loss + torch.where(has, (torch.log(total) - (z.gather(1, of) - top)) * _LABEL_WEIGHT, 0.0).view(-1)
        if c["train"]:
            dz = dz + torch.where(has, e * (_LABEL_WEIGHT / total).float(), 0.0)
            dz = dz.scatter_add_(1, of, torch.where(has, -_LABEL_WEIGHT, 0.0))
    out = {"losses": loss.float() * s["weights"]}
    if c["train"]:
        out["dlogits"] = (dz * s["weights"][:, None]).to(s["logits"].dtype)
    return out


# ----------------------------------------------------------------------------------------------------- the framework's

def _at(x):
    return None if x is None else x.data_ptr()


def _own_norm(s):
    c, r = s["case"], s["readout"]
    r.norm(_at(s["x"]), c["images"], c["width"], _at(s["weight"]), _at(s["bias"]), _EPSILON, _at(s["y"]), dev_mean=_at(s.get("mean")),
           dev_scale=_at(s.get("scale")), x_stride=s["x"].stride(0))
    if not c["train"]:
        return {"y": s["y"]}
    r.norm_backward(_at(s["x"]), c["images"], c["width"], _at(s["weight"]), _at(s["mean"]), _at(s["scale"]), _at(s["dy"]), _at(s["dx"]),
                    _at(s["dweight"]), _at(s["dbias"]), x_stride=s["x"].stride(0))
    return {name: s[name] for name in ("y", "dx", "dweight", "dbias")}


def _own_gated(s):
    from pink_amd import capi
    c, r = s["case"], s["readout"]
    act = {"identity": capi.ACT_IDENTITY, "relu": capi.ACT_RELU, "gelu": capi.ACT_GELU, "silu": capi.ACT_SILU}[c["activation"]]
    shape = (c["features"], c["hidden"], c["outputs"], act)
    weights = [_at(s[name]) for name, *_ in _GATED]
    saved = torch.empty(r.gated_saved_bytes(shape, c["images"]), dtype=torch.uint8, device="cuda") if c["train"] else None
    r.gated(shape, _at(s["x"]), c["images"], weights, _at(s["y"]), dev_residual=_at(s["residual"]), dev_saved=_at(saved), x_stride=s["x"].stride(0))
    out = {"y": s["y"]}
    if c["train"]:
        grads = ["dx"] + ["d" + name for name, *_ in _GATED]
        r.gated_backward(shape, _at(s["x"]), c["images"], weights, _at(saved), _at(s["dy"]), [_at(s[name]) for name in grads], x_stride=s["x"].stride(0))
        out |= {name: s[name] for name in grads if s[name] is not None}
    return out


def _own_distil(s):
    c, r = s["case"], s["readout"]
    r.distil(_at(s["logits"]), c["images"], c["classes"], _at(s["losses"]), _at(s["dlogits"]), dev_teacher_class=_at(s["class"]),
             dev_teacher_logits=_at(s["teacher"]), places=c["places"], dev_teacher_normaliser=_at(s["normaliser"]), dev_label=_at(s["label"]),
             dev_image_weights=_at(s["weights"]), temperature=c["temperature"], teacher_weight=_TEACHER_WEIGHT,
             label_weight=_LABEL_WEIGHT if c["label"] else 0.0, logit_stride=s["logits"].stride(0))
    return {"losses": s["losses"], "dlogits": s["dlogits"]} if c["train"] else {"losses": s["losses"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "gated": _own_gated, "distil": _own_distil}[op](state)
    return {"norm": _plain_norm, "gated": _plain_gated, "distil": _plain_distil}[op](state)


# ------------------------------------------------------------------------------------------------------- in 64 bits

def _exact_norm(c, s):
    """In runs of rows, gradients by automatic differentiation."""
    w, b = s["weight"].double().requires_grad_(c["train"]), s["bias"].double().requires_grad_(c["train"])
    y, dx, sums = [], [], [torch.zeros_like(w), torch.zeros_like(b)]
    for at in range(0, c["images"], 2048):
        x = s["x"][at:at + 2048].double().requires_grad_(c["train"])
        with torch.set_grad_enabled(c["train"]):
            variance = x.var(1, keepdim=True, unbiased=False)
            of = (x - x.mean(1, keepdim=True)) * (variance + _EPSILON).rsqrt() * w + b
        y.append(of.detach())
        if c["train"]:
            d = torch.autograd.grad(of, (x, w, b), s["dy"][at:at + 2048].double())
            dx.append(d[0])
            sums = [sums[0] + d[1], sums[1] + d[2]]
    out = {"y": torch.cat(y)}
    return out | {"dx": torch.cat(dx), "dweight": sums[0].detach(), "dbias": sums[1].detach()} if c["train"] else out


def _exact_gated(c, s):
    """In 64 bits, gradients by automatic differentiation."""
    act = {"identity": lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[c["activation"]]
    names = ["x"] + [name for name, *_ in _GATED if s[name] is not None]
    d = {name: s[name].double().requires_grad_(c["train"]) for name in names}
    with torch.set_grad_enabled(c["train"]):
        linear = torch.nn.functional.linear
        h = act(linear(d["x"], d["gate"], d.get("gate_bias"))) * linear(d["x"], d["up"], d.get("up_bias"))
        y = linear(h, d["down"], d.get("down_bias"))
        if c["residual"]:
            y = y + s["residual"].double()
    if not c["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [d[name] for name in names], s["dy"].double())
    out = {"d" + name: v for name, v in zip(names, grads)}
    return {name: (out | {"y": y.detach()})[name] for name in ["y", "dx", "dgate", "dup", "ddown"] + (["dgate_bias", "dup_bias", "ddown_bias"] if c["bias"] else [])}


def _exact_distil(c, s):
    """In 64 bits, in runs of rows, gradients by automatic differentiation.  The teacher's share of every class is laid out in full."""
    t, v, k, temperature = c["images"], c["classes"], c["places"], c["temperature"]
    losses, grads, step = [], [], max(1, (1 << 24) // v)
    for at in range(0, t, step):
        rows = slice(at, at + step)
        raw = s["logits"][rows].double()
        live = ~torch.isneginf(raw)
        z = torch.where(live, raw, -1e30).requires_grad_(c["train"])
        n = len(raw)
        where = torch.where(s["class"][rows] >= 0, s["class"][rows].long(), v)
        full = torch.full((n, v + 1), -math.inf, dtype=torch.float64, device="cuda").scatter_(1, where, s["teacher"][rows].double() / temperature)[:, :v]
        full = torch.where(live, full, -math.inf)
        named = ~torch.isneginf(full)
        if c["rest"]:
            p = torch.exp(full - s["normaliser"][rows].double()[:, None])
        else:
            p = torch.where(named.any(1, keepdim=True), torch.softmax(torch.where(named, full, -1e30), 1), 0.0) * named
        entropy = torch.special.xlogy(p, p).sum(1)
        with torch.set_grad_enabled(c["train"]):
            scaled = z / temperature
            total = torch.logsumexp(scaled, 1)
            loss = entropy - (p * torch.where(named, scaled - total[:, None], 0.0)).sum(1)
            if c["rest"]:
                free = live & ~named
                left = torch.where(free.any(1), (1 - p.sum(1)).clamp(min=0), 0.0)
                others = torch.logsumexp(torch.where(free, scaled, -1e30), 1) - total
                loss = loss + torch.special.xlogy(left, left) - left * torch.where(free.any(1), others, 0.0)
            loss = loss * (_TEACHER_WEIGHT * temperature ** 2)
            if c["label"]:
                label = s["label"][rows].long()
                of = label.clamp(min=0)[:, None]
                has = (label >= 0) & live.gather(1, of).view(-1)
                loss = loss + _LABEL_WEIGHT * torch.where(has, torch.logsumexp(z, 1) - z.gather(1, of).view(-1), 0.0)
            loss = loss * s["weights"][rows].double()
        losses.append(loss.detach())
        if c["train"]:
            grads.append(torch.where(live, torch.autograd.grad(loss, z, torch.ones_like(loss))[0], 0.0))
    return {"losses": torch.cat(losses), "dlogits": torch.cat(grads)} if c["train"] else {"losses": torch.cat(losses)}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "gated": _exact_gated, "distil": _exact_distil}[c["op"]](c, s)
