"""What is timed of the read-out of a map: routing images to neurons, the neurons' own models, and the optimiser that trains them.

A trained map answers an image with its distance to every neuron.  The read-out lets the nearest neurons answer a question
about the image, each with a two-layer model of its own.  A case is one call pattern of one operator, `op`:

  route     images' distances to neurons -> the `chosen` neurons of every image and their gates; with "train" also the gradients of
            the distances and of every neuron's sharpness and radius
  experts   the chosen neurons' models on the images' features, added up by their gates; with "train" also all gradients
  adamw     one AdamW step over the read-out's tensors, states in 32 or 8 bits

The plain forms hold all in 32 bits and round once at the end; 8-bit states come back as the values they stand for.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_BLOCK = 256        # values that share one scale of an 8-bit state


# ---------------------------------------------------------------------------------------------------------------- cases

def _route(name, images, neurons, chosen, score="softmax", renormalise=True, groups=1, kept=1, bias=False, train=False):
    c = dict(op="route", images=images, neurons=neurons, chosen=chosen, score=score, renormalise=renormalise, groups=groups, kept=kept,
             bias=bias, train=train)
    return dict(c, name=name) if name else c


def _experts(name, images, neurons, chosen, features, hidden, outputs, activation="gelu", type="bf16", residual=False, train=False, pad=0):
    c = dict(op="experts", images=images, neurons=neurons, chosen=chosen, features=features, hidden=hidden, outputs=outputs,
             activation=activation, type=type, residual=residual, train=train, pad=pad)
    return dict(c, name=name) if name else c


def _adamw(name, neurons, features, hidden, outputs, bits=32, type="f32"):
    c = dict(op="adamw", neurons=neurons, features=features, hidden=hidden, outputs=outputs, bits=bits, type=type)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one image looked up on a 10 x 10 map, the two nearest neurons answer: latency counts
        _route("route-1", 1, 100, 2),
        # a survey's worth of images on a 40 x 40 map, eight of its forty rows kept, balanced by a bias
        _route("route-16000-groups", 16000, 1600, 8, "sigmoid", True, 40, 8, True),
        # a training batch on a hexagonal map of 331 neurons, full softmax, with gradients
        _route("route-train-1001-hex", 1001, 331, 4, "softmax", False, train=True),
        # one image's 32 x 32 region through its two neurons' models
        _experts("experts-1", 1, 100, 2, 1024, 256, 64),
        # float32, hexagonal map, 45 x 45 region: few images for each neuron, odd sizes throughout
        _experts("experts-301-f32-odd", 301, 331, 2, 2025, 200, 45, "relu", "f32"),
        # a survey's worth of images cleaned up: the answer has the size of the region and is added to it
        _experts("experts-16000-residual", 16000, 100, 2, 1024, 512, 1024, "silu", residual=True),
        # small pictures (28 x 28), one neuron each, ten classes, a training step in float32
        _experts("experts-train-500-f32", 500, 64, 1, 784, 96, 10, "relu", "f32", train=True),
        # a training step over many images: 44 x 44 neurons, four answer
        _experts("experts-train-16000", 16000, 100, 4, 1936, 1024, 256, train=True),
        # the tensors of a small read-out: launches count
        _adamw("adamw-small", 64, 784, 16, 10),
        # a hexagonal map's read-out in float32
        _adamw("adamw-f32-hex", 331, 2025, 64, 45),
        # the largest read-out, bfloat16 gradients and 8-bit states
        _adamw("adamw-8bit", 100, 1936, 1024, 256, 8, "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MAX_FLOPS = 8.0e11          # of a drawn pass: what the largest listed one has
_MAX_PARAMETERS = 1.6e8


def draw(rng):
    op = rng.choice(("route", "experts", "experts", "adamw"))
    neurons = rng.choice((64, 100, 331, 1600, _log(rng, 9, 1600)))
    if op == "route":
        groups = rng.choice((1, 1, _log(rng, 1, 40)))
        while (groups - 1) * -(-neurons // groups) >= neurons:
            groups -= 1
        return _route(None, _log(rng, 1, 16000), neurons, rng.choice((1, 2, 3, 4, 6, 8)), rng.choice(("softmax", "sigmoid")),
                      rng.random() < 0.6, groups, max(1, groups // rng.choice((1, 2, 4))), rng.random() < 0.5, rng.random() < 0.5)
    while True:
        features = rng.choice((784, 1024, 1936, 2025, _log(rng, 64, 2048)))
        hidden = rng.choice((_log(rng, 8, 1024), 16 * _log(rng, 1, 64)))
        outputs = rng.choice((_log(rng, 1, 1024), 8 * _log(rng, 1, 128)))
        per_neuron = hidden * (features + 1) + outputs * (hidden + 1)
        if neurons * per_neuron > _MAX_PARAMETERS:
            neurons = rng.choice((64, 100, 331))
            continue
        if op == "adamw":
            bits = rng.choice((8, 32))
            return _adamw(None, neurons, features, hidden, outputs, bits, rng.choice(("f32", "bf16")))
        chosen, train, type = rng.choice((1, 2, 3, 4)), rng.random() < 0.5, rng.choice(("bf16", "bf16", "f32"))
        most = _MAX_FLOPS / ((6.0 if train else 2.0) * chosen * per_neuron) / (4 if type == "f32" else 1)
        images = _log(rng, 1, max(1, min(16000, int(most))))
        residual = rng.random() < 0.3
        return _experts(None, images, neurons, chosen, features, hidden, outputs, rng.choice(("identity", "relu", "gelu", "silu")), type,
                        residual, train, rng.choice((0, 0, 0, 3, 8)))


def _shapes(c):
    """The trained tensors of a read-out, in the order that an optimiser is given them; the first two belong to the router."""
    n, f, h, o = c["neurons"], c["features"], c["hidden"], c["outputs"]
    return [(n,), (n,), (n, h, f), (n, h), (n, o, h), (n, o)]


def work(case):
    """Inputs read once, outputs written once.  Of the models' weights those of neurons that at least one image can have chosen."""
    c = case
    if c["op"] == "route":
        t, n, k = c["images"], c["neurons"], c["chosen"]
        moved = 4.0 * t * n + 8.0 * t * k + 12.0 * n
        if c["train"]:
            moved += 4.0 * t * n + 4.0 * t * k + 8.0 * n
        return {"bytes": moved, "flops": (16.0 if c["train"] else 8.0) * t * n}
    size = 2 if c["type"] == "bf16" else 4
    if c["op"] == "experts":
        t, k, f, h, o = c["images"], c["chosen"], c["features"], c["hidden"], c["outputs"]
        rows, n = t * k, min(c["neurons"], t * k)
        moved = size * (t * f + n * (h * f + h + o * h + o) + t * o * (2 if c["residual"] else 1)) + 8.0 * rows
        flops = 2.0 * rows * h * (f + o)
        if c["train"]:
            moved += size * (t * o + t * f + rows + c["neurons"] * (h * f + h + o * h + o))
            flops *= 3
        return {"bytes": moved, "flops": flops}
    total = float(sum(math.prod(s) for s in _shapes(c)))
    state = 16.0 if c["bits"] == 32 else 4.0 + 16.0 / _BLOCK + 8.0        # unpacked ones are an output too
    return {"bytes": total * (8.0 + size + (2.0 if c["type"] == "bf16" else 0.0) + state), "flops": 20.0 * total}


# --------------------------------------------------------------------------------------------------------------- inputs

_readouts = {}


def _readout(c):
    """The handle that a program keeps for its read-out: one per configuration, on PyTorch's stream."""
    if not own:
        return None
    from pink_amd import capi
    key = tuple((k, v) for k, v in sorted(c.items()) if k not in ("name", "images", "pad", "residual", "train", "bits"))
    if key not in _readouts:
        element = capi.ELEMENT_BF16 if c.get("type") == "bf16" else capi.ELEMENT_F32
        if c["op"] == "route":
            r = capi.Readout(c["neurons"], c["chosen"], score={"softmax": capi.SCORE_SOFTMAX, "sigmoid": capi.SCORE_SIGMOID}[c["score"]],
                             renormalise=c["renormalise"], groups=c["groups"], groups_kept=c["kept"])
        elif c["op"] == "experts":
            r = capi.Readout(c["neurons"], c["chosen"], c["features"], c["hidden"], c["outputs"], element=element,
                             activation={"identity": capi.ACT_IDENTITY, "relu": capi.ACT_RELU, "gelu": capi.ACT_GELU, "silu": capi.ACT_SILU}[c["activation"]])
        else:
            r = capi.Readout(c["neurons"], 1)
        r.set_stream(torch.cuda.current_stream().cuda_stream)
        _readouts[key] = r
    return _readouts[key]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, scale=1.0, type=torch.float32):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(type)


def _rand(gen, *shape):
    return torch.rand(shape, device="cuda", generator=gen)


def _prepare_route(c, seed):
    gen = _generator(seed)
    t, n, k = c["images"], c["neurons"], c["chosen"]
    # distances as a mapper gives them: a level of the image's own, near neurons stand out
    distances = (6 + 2 * _rand(gen, t, 1)) + _randn(gen, t, n) - 2 * _rand(gen, t, n) ** 8
    dead = _rand(gen, n) < 0.01                                        # neurons taken out of the competition
    distances = torch.where(dead[None, :], math.inf, distances)
    distances = torch.where(_rand(gen, t, n) < 1e-4, math.nan, distances)
    if t > 8:
        distances[t // 2] = math.inf                                   # an image that no neuron may answer for
    s = {"case": c, "distances": distances.contiguous(), "sharpness": 1.5 + 0.5 * _rand(gen, n), "radius": 5 + 0.5 * _randn(gen, n),
         "bias": _randn(gen, n, scale=0.3) if c["bias"] else None, "neuron": torch.empty((t, k), dtype=torch.int32, device="cuda"),
         "gates": torch.empty((t, k), device="cuda"), "readout": _readout(c)}
    if c["train"]:
        s["dgates"] = _randn(gen, t, k)
        s["ddistances"] = torch.empty((t, n), device="cuda")
        s["dsharpness"], s["dradius"] = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    return s


def _prepare_experts(c, seed):
    gen, type = _generator(seed), _TYPES[c["type"]]
    t, n, k, f, h, o = (c[x] for x in ("images", "neurons", "chosen", "features", "hidden", "outputs"))
    # neurons are chosen unevenly, each at most once by an image; a few images have a neuron less, one has none
    popular = _randn(gen, 1, n, scale=0.5) - torch.log(-torch.log(_rand(gen, t, n).clamp(1e-7, 1 - 1e-7)))
    neuron = popular.topk(k, dim=1).indices.to(torch.int32)
    gates = torch.softmax(_randn(gen, t, k), dim=1)
    none = _rand(gen, t) < 0.02
    neuron[:, k - 1] = torch.where(none, -1, neuron[:, k - 1]) if t > 8 else neuron[:, k - 1]
    if t > 8:
        neuron[t // 2] = -1
    gates = torch.where(neuron < 0, 0.0, gates)
    wide = (0.5 * _rand(gen, t, f + c["pad"]) + _randn(gen, t, f + c["pad"], scale=0.25)).to(type)
    s = {"case": c, "neuron": neuron.contiguous(), "gates": gates.contiguous(), "x": wide[:, :f],
         "w1": _randn(gen, n, h, f, scale=1.5 / math.sqrt(f), type=type), "b1": _randn(gen, n, h, scale=0.3, type=type),
         "w2": _randn(gen, n, o, h, scale=1.5 / math.sqrt(h), type=type), "b2": _randn(gen, n, o, scale=0.3, type=type),
         "residual": (_rand(gen, t, o).to(type) if c["residual"] else None), "y": torch.empty((t, o), dtype=type, device="cuda"), "readout": _readout(c)}
    if c["train"]:
        s["dy"] = _randn(gen, t, o, type=type)
        s["dx"], s["dgates"] = torch.empty((t, f), dtype=type, device="cuda"), torch.empty((t, k), dtype=type, device="cuda")
        for x in ("w1", "b1", "w2", "b2"):
            s["d" + x] = torch.empty_like(s[x])
    return s


_OPTIONS = dict(learning_rate=1e-3, beta_first=0.9, beta_second=0.99, epsilon=1e-8)


def _decode_first(codes, scale, n):
    u = _blocks(codes.to(torch.float32), n) * np.float32(1 / 127)
    return ((u * u.abs()) * scale[:, None]).reshape(-1)[:n]


def _decode_second(codes, scale, n):
    u = _blocks(codes.to(torch.float32), n) * np.float32(1 / 255)
    u = u * u
    return ((u * u) * scale[:, None]).reshape(-1)[:n]


def _blocks(x, n):
    return torch.nn.functional.pad(x.reshape(-1), (0, -n % _BLOCK)).view(-1, _BLOCK)


def _codes(x, n, top):
    """Roots of the values over their block's largest, as fractions of `top`, and the scales; a block below the smallest normal number holds zeros."""
    b = _blocks(x, n)
    scale = b.abs().amax(1)
    small = scale < np.float32(2.0 ** -126)
    scale = torch.where(small, 0.0, scale)
    ratio = b.abs() * torch.where(small, 0.0, 1.0 / scale)[:, None]
    root = torch.sqrt(ratio)
    if top == 127:
        codes = torch.round(root * 127.0) * torch.sign(b)
    else:
        codes = torch.round(torch.sqrt(root) * 255.0)
        codes = torch.where(ratio > 0, codes.clamp(min=1.0), codes)
    return codes.reshape(-1)[:n].to(torch.int8 if top == 127 else torch.uint8), scale


def _prepare_adamw(c, seed):
    gen, tensors = _generator(seed), []
    for i, shape in enumerate(_shapes(c)):
        n = math.prod(shape)
        size = 10.0 ** (-4 + 2 * _rand(gen, 1))                        # gradients' size differs from tensor to tensor
        p = {"value": _randn(gen, n, scale=0.05), "decay": 0.01 if len(shape) == 3 else 0.0}
        # of many rows of a batch few reach one neuron: a part of the gradients is zero
        p["gradient"] = (_randn(gen, n) * size * (_rand(gen, n) < 0.9)).to(_TYPES[c["type"]] if i >= 2 else torch.float32)
        p["rounded"] = p["value"].to(torch.bfloat16) if c["type"] == "bf16" and i >= 2 else None
        first, second = _randn(gen, n) * size * 0.3, (_randn(gen, n) * size) ** 2
        if c["bits"] == 8:
            p["first"], p["first_scale"] = _codes(first, n, 127)
            p["second"], p["second_scale"] = _codes(second, n, 255)
            p["first_values"], p["second_values"] = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        else:
            p["first"], p["second"] = first, second
        tensors.append(p)
    return {"case": c, "tensors": tensors, "step": 10, "readout": _readout(c)}


def prepare(case, seed):
    return {"route": _prepare_route, "experts": _prepare_experts, "adamw": _prepare_adamw}[case["op"]](case, seed)


# ---------------------------------------------------------------------------------------------------------- plain forms

def _plain_route(s):
    c, d = s["case"], s["distances"]
    t, n = d.shape
    z = s["sharpness"] * (s["radius"] - d)
    biased = z if s["bias"] is None else z + s["bias"]
    part = torch.isfinite(z) & torch.isfinite(biased)
    key = torch.where(part, biased, -math.inf)
    if c["groups"] > 1:
        size = -(-n // c["groups"])
        member = torch.nn.functional.pad(key, (0, c["groups"] * size - n), value=-math.inf).view(t, c["groups"], size)
        best = member.sort(dim=2, descending=True, stable=True).values[:, :, :2]
        score = torch.where(torch.isinf(best), 0.0, best).sum(2)
        score = torch.where(torch.isinf(best[:, :, 0]), -math.inf, score)
        kept = score.sort(dim=1, descending=True, stable=True).indices[:, : c["kept"]]
        keep = torch.zeros((t, c["groups"]), dtype=torch.bool, device=d.device).scatter_(1, kept, True)
        key = torch.where(keep.repeat_interleave(size, 1)[:, :n], key, -math.inf)
    best = key.sort(dim=1, descending=True, stable=True)
    k = c["chosen"]
    valid = torch.isfinite(best.values[:, :k])
    at = best.indices[:, :k]
    zc = torch.where(valid, z.gather(1, at), -math.inf)
    zall = torch.where(part, z, -math.inf)
    if c["renormalise"]:
        level = zc if c["score"] == "softmax" else torch.minimum(zc, torch.zeros_like(zc)) - torch.log(1 + torch.exp(-zc.abs()))
        top = level.amax(1, keepdim=True)
        e = torch.where(valid, torch.exp(level - torch.where(torch.isinf(top), 0.0, top)), 0.0)
        gates = e / torch.where(valid.any(1, keepdim=True), e.sum(1, keepdim=True), 1.0)
    elif c["score"] == "softmax":
        top = zall.amax(1, keepdim=True)
        share = torch.where(part, torch.exp(zall - torch.where(torch.isinf(top), 0.0, top)), 0.0)
        share = share / torch.where(part.any(1, keepdim=True), share.sum(1, keepdim=True), 1.0)
        gates = torch.where(valid, share.gather(1, at), 0.0)
    else:
        gates = torch.where(valid, 1 / (1 + torch.exp(-zc)), 0.0)
    out = {"neuron": torch.where(valid, at, -1).to(torch.int32), "gates": gates}
    if not c["train"]:
        return out
    g = torch.where(valid, s["dgates"], 0.0)
    if c["renormalise"]:
        dzc = gates * (g - (gates * g).sum(1, keepdim=True))
        if c["score"] == "sigmoid":
            dzc = dzc / (1 + torch.exp(zc))
    elif c["score"] == "softmax":
        dzc = gates * g
    else:
        dzc = g * gates / (1 + torch.exp(zc))
    dz = torch.zeros_like(d).scatter_(1, at, torch.where(valid, dzc, 0.0))
    if c["score"] == "softmax" and not c["renormalise"]:
        dz = dz - share * (gates * g).sum(1, keepdim=True)
    out["ddistances"] = -s["sharpness"] * dz
    out["dsharpness"] = torch.where(part, dz * (s["radius"] - d), 0.0).sum(0)
    out["dradius"] = (s["sharpness"] * dz).sum(0)
    return out


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


def _plain_experts(s):
    """Rows sorted by neuron and padded to the largest number that one neuron has, so that a layer is one batched product."""
    c, type = s["case"], _TYPES[s["case"]["type"]]
    t, n, k, f, h, o = (c[x] for x in ("images", "neurons", "chosen", "features", "hidden", "outputs"))
    w1, b1, w2, b2 = (s[x].float() for x in ("w1", "b1", "w2", "b2"))
    x = s["x"].float()
    flat = s["neuron"].reshape(-1).long()
    slots = torch.nonzero((flat >= 0) & (flat < n)).view(-1)
    e, order = flat[slots].sort(stable=True)
    slots = slots[order]
    count = torch.bincount(e, minlength=n)
    rank = torch.arange(len(e), device=e.device) - (count.cumsum(0) - count)[e]
    most = int(count.max())
    image, gate = slots // k, s["gates"].reshape(-1)[slots][:, None]
    rows = torch.zeros((n, most, f), device=x.device)
    rows[e, rank] = x[image]
    before = torch.bmm(rows, w1.transpose(1, 2).contiguous()) + b1[:, None]
    after = _activate(c["activation"], before)
    answer = (torch.bmm(after, w2.transpose(1, 2).contiguous()) + b2[:, None])[e, rank]
    each = torch.zeros((t * k, o), device=x.device)
    each[slots] = gate * answer
    y = each.view(t, k, o).sum(1)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(type)}
    if not c["train"]:
        return out
    dy = s["dy"].float()[image]
    dgates = torch.zeros(t * k, device=x.device)
    dgates[slots] = (dy * answer).sum(1)
    scaled = torch.zeros((n, most, o), device=x.device)
    scaled[e, rank] = gate * dy
    dbefore = torch.bmm(scaled, w2) * _slope(c["activation"], before)
    dx = torch.zeros((t * k, f), device=x.device)
    dx[slots] = torch.bmm(dbefore, w1)[e, rank]
    out |= {"dx": dx.view(t, k, f).sum(1), "dgates": dgates.view(t, k), "dw2": torch.bmm(scaled.transpose(1, 2).contiguous(), after),
            "db2": scaled.sum(1), "dw1": torch.bmm(dbefore.transpose(1, 2).contiguous(), rows), "db1": dbefore.sum(1)}
    return {name: v.to(type) for name, v in out.items()}


def _plain_adamw(s):
    c, o = s["case"], _OPTIONS
    s["step"] += 1
    lr, b1, b2, eps = (np.float32(o[x]) for x in ("learning_rate", "beta_first", "beta_second", "epsilon"))
    rest1, rest2 = np.float32(1) - b1, np.float32(1) - b2
    c1, c2 = np.float32(1 / (1 - float(b1) ** s["step"])), np.float32(1 / (1 - float(b2) ** s["step"]))
    for p in s["tensors"]:
        n, g = p["value"].numel(), p["gradient"].float()
        if c["bits"] == 8:
            m, v = _decode_first(p["first"], p["first_scale"], n), _decode_second(p["second"], p["second_scale"], n)
        else:
            m, v = p["first"], p["second"]
        m = m * float(b1) + g * float(rest1)
        v = v * float(b2) + (g * g) * float(rest2)
        step = (m * float(c1)) / (torch.sqrt(v * float(c2)) + float(eps))
        p["value"].copy_(p["value"] - (step + p["value"] * p["decay"]) * float(lr))
        if p["rounded"] is not None:
            p["rounded"].copy_(p["value"])
        if c["bits"] == 8:
            for name, x, top in (("first", m, 127), ("second", v, 255)):
                codes, scale = _codes(x, n, top)
                p[name].copy_(codes)
                p[name + "_scale"].copy_(scale)
            p["first_values"] = _decode_first(p["first"], p["first_scale"], n)
            p["second_values"] = _decode_second(p["second"], p["second_scale"], n)
        else:
            p["first"].copy_(m)
            p["second"].copy_(v)
    return _adamw_outputs(s) if c["bits"] == 32 else _adamw_outputs(s, "first_values", "second_values")


def _adamw_outputs(s, first="first", second="second"):
    return [{"value": p["value"], "rounded": p["rounded"], "first": p[first], "second": p[second]} for p in s["tensors"]]


# ----------------------------------------------------------------------------------------------------- the framework's

def _at(x):
    return None if x is None else x.data_ptr()


def _own_route(s):
    c, r = s["case"], s["readout"]
    r.route(_at(s["distances"]), c["images"], _at(s["sharpness"]), _at(s["radius"]), _at(s["bias"]), _at(s["neuron"]), _at(s["gates"]))
    out = {"neuron": s["neuron"], "gates": s["gates"]}
    if c["train"]:
        r.route_backward(_at(s["distances"]), c["images"], _at(s["sharpness"]), _at(s["radius"]), _at(s["bias"]), _at(s["neuron"]), _at(s["gates"]),
                         _at(s["dgates"]), _at(s["ddistances"]), _at(s["dsharpness"]), _at(s["dradius"]))
        out |= {"ddistances": s["ddistances"], "dsharpness": s["dsharpness"], "dradius": s["dradius"]}
    return out


def _own_experts(s):
    c, r = s["case"], s["readout"]
    weights = [_at(s[x]) for x in ("w1", "b1", "w2", "b2")]
    saved = torch.empty(r.saved_bytes(c["images"]), dtype=torch.uint8, device="cuda") if c["train"] else None
    r.experts(_at(s["x"]), c["images"], _at(s["neuron"]), _at(s["gates"]), weights, _at(s["y"]), dev_residual=_at(s["residual"]),
              dev_saved=_at(saved), x_stride=s["x"].stride(0))
    out = {"y": s["y"]}
    if c["train"]:
        grads = ("dx", "dgates", "dw1", "db1", "dw2", "db2")
        r.experts_backward(_at(s["x"]), c["images"], _at(s["gates"]), weights, _at(saved), _at(s["dy"]), [_at(s[x]) for x in grads],
                           x_stride=s["x"].stride(0))
        out |= {x: s[x] for x in grads}
    return out


def _own_adamw(s):
    s["step"] += 1
    r, bits = s["readout"], s["case"]["bits"]
    fields = ("value", "gradient", "rounded", "first", "second") + (("first_scale", "second_scale", "first_values", "second_values") if bits == 8 else ())
    tensors = r.tensors([dict(size=p["value"].numel(), decay=p["decay"], gradient_bf16=p["gradient"].dtype == torch.bfloat16,
                              **{x: _at(p[x]) for x in fields}) for p in s["tensors"]])
    r.adamw(tensors, s["step"], bits=bits, **_OPTIONS)
    if bits == 32:
        return _adamw_outputs(s)
    r.adamw_unpack(tensors)                            # as the values that the codes stand for
    return _adamw_outputs(s, "first_values", "second_values")


def run(state):
    op = state["case"]["op"]
    if own:
        return {"route": _own_route, "experts": _own_experts, "adamw": _own_adamw}[op](state)
    return {"route": _plain_route, "experts": _plain_experts, "adamw": _plain_adamw}[op](state)


# ------------------------------------------------------------------------------------------------------- in 64 bits

def _exact_route(c, s):
    """Which neurons are chosen goes by the logits as 32-bit numbers (that is their definition); all else in 64 bits, one image after the other's rules
    written as numpy array operations."""
    d, a, r = (s[x].cpu().numpy() for x in ("distances", "sharpness", "radius"))
    with np.errstate(all="ignore"):
        z32 = a * (r - d)
        key = z32 if s["bias"] is None else z32 + s["bias"].cpu().numpy()
        part = np.isfinite(z32) & np.isfinite(key)
        z = a.astype(np.float64) * (r.astype(np.float64) - d)
    t, n, k = c["images"], c["neurons"], c["chosen"]
    lowest = np.float32(-np.inf)
    key = np.where(part, key, lowest)
    if c["groups"] > 1:
        size = -(-n // c["groups"])
        score = np.full((t, c["groups"]), lowest)
        for g in range(c["groups"]):
            own_ = np.sort(key[:, g * size:(g + 1) * size], axis=1)[:, ::-1]
            two = own_[:, :2] if own_.shape[1] > 1 else np.concatenate([own_, np.full((t, 1), lowest)], 1)
            score[:, g] = np.where(np.isinf(two[:, 1]), two[:, 0], two[:, 0] + two[:, 1])
        kept = np.argsort(-score, axis=1, kind="stable")[:, : c["kept"]]
        ok = np.zeros((t, c["groups"]), bool)
        np.put_along_axis(ok, kept, True, 1)
        key = np.where(ok[:, np.arange(n) // size], key, lowest)
    at = np.argsort(-key, axis=1, kind="stable")[:, :k]
    valid = np.isfinite(np.take_along_axis(key, at, 1))
    row = np.arange(t)[:, None]
    chosen = np.zeros((t, n), bool)
    chosen[row, at] = valid
    zz = np.where(part, z, 0.0)
    if c["score"] == "softmax":
        level, below = zz, np.ones_like(zz)
    else:
        level, below = -np.logaddexp(0, -zz), 1 / (1 + np.exp(zz))     # log of the score, and its slope
    over = chosen if c["renormalise"] else part if c["score"] == "softmax" else None
    if over is None:
        total = np.zeros((t, 1))
    else:
        top = np.where(over, level, -np.inf).max(1, keepdims=True)
        top = np.where(np.isfinite(top), top, 0.0)
        total = top + np.log(np.maximum(np.where(over, np.exp(level - top), 0.0).sum(1, keepdims=True), 1e-300))
    gate = np.where(part, np.exp(np.minimum(level - total, 0.0)), 0.0)
    out = {"neuron": torch.from_numpy(np.where(valid, at, -1).astype(np.int32)), "gates": torch.from_numpy(np.where(valid, gate[row, at], 0.0))}
    if not c["train"]:
        return out
    g = np.zeros((t, n))
    g[row, at] = np.where(valid, s["dgates"].cpu().numpy().astype(np.float64), 0.0)
    dlevel = np.where(chosen, gate * g, 0.0)
    if over is not None:
        dlevel = dlevel - np.where(over, gate, 0.0) * dlevel.sum(1, keepdims=True)
    dz = dlevel * below
    with np.errstate(all="ignore"):
        distance = np.where(part, r.astype(np.float64) - d, 0.0)
    return out | {"ddistances": torch.from_numpy(-a.astype(np.float64) * dz), "dsharpness": torch.from_numpy((dz * distance).sum(0)),
                  "dradius": torch.from_numpy((a.astype(np.float64) * dz).sum(0))}


def _exact_experts(c, s):
    """One neuron after the other, in 64 bits, gradients by automatic differentiation."""
    double = {x: s[x].double().requires_grad_(c["train"]) for x in ("x", "gates", "w1", "b1", "w2", "b2")}
    act = {"identity": lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[c["activation"]]
    y = torch.zeros(c["images"], c["outputs"], dtype=torch.float64, device="cuda")
    if s["residual"] is not None:
        y = y + s["residual"].double()
    grads = {x: torch.zeros_like(v) for x, v in double.items()} if c["train"] else {}
    for n in torch.unique(s["neuron"]).tolist():
        if n < 0:
            continue
        image, slot = torch.nonzero(s["neuron"] == n, as_tuple=True)
        x, g = double["x"].detach()[image].requires_grad_(c["train"]), double["gates"].detach()[image, slot].requires_grad_(c["train"])
        w = [double[v].detach()[n].requires_grad_(c["train"]) for v in ("w1", "b1", "w2", "b2")]
        with torch.set_grad_enabled(c["train"]):
            answer = g[:, None] * (act(x @ w[0].T + w[1]) @ w[2].T + w[3])
        y.index_add_(0, image, answer.detach())
        if c["train"]:
            of = torch.autograd.grad(answer, [x, g] + w, s["dy"].double()[image])
            grads["x"].index_add_(0, image, of[0])
            grads["gates"][image, slot] = of[1]
            for name, v in zip(("w1", "b1", "w2", "b2"), of[2:]):
                grads[name][n] = v
    return {"y": y, **{"d" + x: v.detach() for x, v in grads.items()}}


def _exact_adamw(c, s):
    """In 64 bits from the states as they stand; of states that are held in 8 bits, what they are before they are packed."""
    step, o, out = s["step"] + 1, _OPTIONS, []
    for p in s["tensors"]:
        g = p["gradient"].double()
        if c["bits"] == 8:
            i = torch.arange(g.numel(), device="cuda") // _BLOCK
            q = p["first"].double() / 127
            m, v = q * q.abs() * p["first_scale"].double()[i], (p["second"].double() / 255) ** 4 * p["second_scale"].double()[i]
        else:
            m, v = p["first"].double(), p["second"].double()
        b1, b2 = float(np.float32(o["beta_first"])), float(np.float32(o["beta_second"]))
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        value = p["value"].double()
        change = m / (1 - b1 ** step) / ((v / (1 - b2 ** step)).sqrt() + o["epsilon"]) + p["decay"] * value
        value = value - o["learning_rate"] * change
        out.append({"value": value, "rounded": None if p["rounded"] is None else value, "first": m, "second": v})
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    with torch.no_grad():
        return {"route": _exact_route, "experts": _exact_experts, "adamw": _exact_adamw}[c["op"]](c, s)
