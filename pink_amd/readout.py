"""A read-out of a trained map: what is asked about an image is answered by the neurons nearest to it.

    from pink_amd import pink, readout
    answers = readout.MapReadout(som, outputs=2, chosen=2, number_of_rotations=180, euclidean_distance_dim=22)
    for images, targets in batches:
        loss = answers.step(images, targets)
    y = answers(images)

An image's heatmap routes it to its neurons and is what their models see, so answers do not change when the image is turned or
mirrored, as the map's distances do not.  Everything between the images and the answers stays on the GPU: mapping
(pink_hip_map_device), routing, the neurons' models, their gradients and AdamW (pink_hip_readout_*).  PyTorch holds the device memory and
has to be imported before the library is loaded, so that both run on one HIP runtime and share a stream (importing this
module first does that).

Answers may be logits of classes instead, learned from labels and from what a larger read-out answers:

    teacher.learn(images, labels)
    student.learn(images, labels, teacher.teach(images, places=8))

    python -m pink_amd.readout [--steps N] [--blocks N] [--distil]

trains a small map on synthetic sources and a read-out of their size and axis ratio (with --distil: of classes of both, and a smaller one
from it).
"""
import argparse
import collections
import functools
import math
import types

import numpy as np
import torch

from . import capi, pink


def _check_one_runtime():
    """PyTorch's wheels carry a HIP runtime of their own; a library loaded before PyTorch is bound to the system's, and streams of one mean
    nothing to the other."""
    capi.lib()
    with open("/proc/self/maps") as maps:
        runtimes = {line.split()[-1] for line in maps if "libamdhip64" in line}
    if len(runtimes) > 1:
        raise pink.exception(-4, "import torch (or this module) before the library is first used: two HIP runtimes are loaded, " + ", ".join(sorted(runtimes)))


def _on_its_device(call):
    @functools.wraps(call)
    def run(self, *args, **options):
        with torch.cuda.device(self.device):
            self._follow_stream()
            return call(self, *args, **options)
    return run


# What a read-out answered about images: its largest logits and their classes, and the logarithm of the sum over all classes of
# exp(logit / temperature).
Teacher = collections.namedtuple("Teacher", "classes logits normaliser temperature")

_EPSILON = 1e-5              # of the blocks' layer norm


class MapReadout:
    """Two-layer models of a map's neurons on its heatmap; `chosen` of them answer for an image, weighted by the softmax of
    sharpness * (radius - distance).

    With `blocks` the features go through as many blocks first, x + gated(norm(x)), which all neurons share: layer norm and a gated
    feed-forward block of `block_hidden` hidden values (twice the neurons unless given), nothing but x to start with.

    The map is copied when it is made, as a pink.Mapper does: its models are trained on that map.  The first step's images set `level`,
    the scale of the features, and where sharpness and radius start; answers asked for before go by the scale of their own images.
    What a trained read-out consists of (parameters, states, bias, level and steps) is saved by state_dict() and put back by
    load_state_dict() of one that was made alike; its tensors can be written to but not replaced, as AdamW holds their addresses.

    It lives on the device that is current when it is made.  Calls run on that device's stream that is current when they are made, and
    what they return is that stream's; a call on another stream than the last one's waits for that one first, so a stream that
    was used has to exist until then."""

    def __init__(self, som, outputs, hidden=32, chosen=2, activation=capi.ACT_GELU, learning_rate=3e-3, weight_decay=1e-3, balance_rate=1e-3,
                 state_bits=32, number_of_rotations=360, use_flip=True, euclidean_distance_dim=None,
                 euclidean_distance_type=pink.DataType.UINT8, seed=0, blocks=0, block_hidden=None):
        self.som, self.outputs, self.hidden, self.chosen, self.state_bits = som, outputs, hidden, chosen, state_bits
        self.learning_rate, self.weight_decay, self.balance_rate = learning_rate, weight_decay, balance_rate
        self._map_args = (int(number_of_rotations), bool(use_flip), int(euclidean_distance_dim))
        self._map_type = int(euclidean_distance_type)
        n = som.number_of_neurons
        self._rows = som._rows().copy()
        self._neuron_channels, self._neuron_dim = pink._image_geometry(som.neuron_shape, som.neuron_layout, "neuron")
        self.blocks, self.block_hidden = int(blocks), int(2 * n if block_hidden is None else block_hidden)
        if self.blocks < 0 or not 1 <= self.block_hidden <= 2 ** 20:
            raise pink.exception(-1, "blocks must be 0 or more, and their hidden values between 1 and 1048576")
        self._shape = (n, self.block_hidden, n, capi.ACT_SILU)
        _check_one_runtime()
        capi.Readout.check(n, chosen, n, hidden, outputs, activation=activation)
        torch.cuda.init()
        self.device = torch.device("cuda", torch.cuda.current_device())
        self.readout = capi.Readout(n, chosen, n, hidden, outputs, activation=activation, device=self.device.index)
        self._stream = None
        self._follow_stream()
        self._mapper = None
        gen = torch.Generator(device=self.device).manual_seed(seed)

        def zeros(shape, dtype=torch.float32):
            return torch.zeros(shape, dtype=dtype, device=self.device)

        def randn(*shape, scale):
            return torch.randn(shape, device=self.device, generator=gen) * scale

        self.parameters = {"sharpness": zeros(n) + 1, "radius": zeros(n),
                           "first": randn(n, hidden, n, scale=1 / math.sqrt(n)), "first_bias": zeros((n, hidden)),
                           "second": randn(n, outputs, hidden, scale=1 / math.sqrt(hidden)), "second_bias": zeros((n, outputs))}
        for b in range(self.blocks):
            h = self.block_hidden
            self.parameters |= {"block%d.%s" % (b, k): v for k, v in {
                "weight": zeros(n) + 1, "bias": zeros(n), "gate": randn(h, n, scale=1 / math.sqrt(n)), "gate_bias": zeros(h),
                "up": randn(h, n, scale=1 / math.sqrt(n)), "up_bias": zeros(h), "down": zeros((n, h)), "down_bias": zeros(n)}.items()}
        self.gradients = {k: torch.zeros_like(v) for k, v in self.parameters.items()}
        state, blocks = (lambda v, t: zeros(v.numel(), t)), lambda v: zeros(-(-v.numel() // 256))
        if state_bits == 8:
            self.states = {k: dict(first=state(v, torch.int8), second=state(v, torch.uint8), first_scale=blocks(v), second_scale=blocks(v))
                           for k, v in self.parameters.items()}
        else:
            self.states = {k: dict(first=state(v, torch.float32), second=state(v, torch.float32)) for k, v in self.parameters.items()}
        self._tensors = self.readout.tensors([
            dict(value=v.data_ptr(), gradient=self.gradients[k].data_ptr(), size=v.numel(),
                 decay=weight_decay if k.split(".")[-1] in ("first", "second", "gate", "up", "down") else 0.0,
                 **{s: x.data_ptr() for s, x in self.states[k].items()}) for k, v in self.parameters.items()])
        self.parameters, self.gradients = types.MappingProxyType(self.parameters), types.MappingProxyType(self.gradients)
        self.states = types.MappingProxyType({k: types.MappingProxyType(v) for k, v in self.states.items()})
        self.bias = zeros(n)                               # for an even load; takes part in the choice of neurons only
        self.steps, self.level = 0, None                   # level: mean and spread of the distances

    def _held(self):
        return {**{"parameters." + k: v for k, v in self.parameters.items()},
                **{"states.%s.%s" % (k, name): v for k, held in self.states.items() for name, v in held.items()}, "bias": self.bias}

    def _follow_stream(self):
        """What was queued for the read-out so far is complete, and the handle works on the caller's current stream."""
        stream = torch.cuda.current_stream(self.device)
        if stream != self._stream:
            self.readout.set_stream(stream.cuda_stream)    # waits for the stream that it leaves, PyTorch's work there too
            self._stream = stream

    @_on_its_device
    def state_dict(self):
        """Copies of all that a trained read-out consists of, by name: tensors, the number of steps, and the level (None before the first step)."""
        return {**{k: v.clone() for k, v in self._held().items()}, "level": None if self.level is None else self.level.clone(), "steps": self.steps}

    @_on_its_device
    def load_state_dict(self, saved):
        """Goes on from what state_dict() gave, of a read-out with as many neurons, hidden values, outputs and blocks and the same state_bits."""
        held = self._held()
        if set(saved) != set(held) | {"level", "steps"}:
            raise pink.exception(-1, "not the state of such a read-out: " + ", ".join(sorted(set(saved) ^ (set(held) | {"level", "steps"}))))
        wrong = [k for k, v in held.items() if saved[k].shape != v.shape or saved[k].dtype != v.dtype]
        if wrong or (saved["level"] is not None and tuple(saved["level"].shape) != (2,)):
            raise pink.exception(-1, "not the state of such a read-out: shape or type of " + ", ".join(wrong or ["level"]))
        for k, v in held.items():
            v.copy_(saved[k])
        self.level = None if saved["level"] is None else saved["level"].to(self.device, torch.float32, copy=True)
        self.steps = int(saved["steps"])

    @_on_its_device
    def distances(self, images):
        """The images' heatmaps, (images, neurons) on the GPU.  Images: a float32 array or CUDA tensor (images[, channels], edge, edge)."""
        images = torch.as_tensor(images, dtype=torch.float32, device=self.device).contiguous()
        channels, edge = self._geometry(images)
        if self._mapper is None or self._mapper.I != edge:
            rotations, flip, region = self._map_args
            self._mapper = capi.Context(len(self._rows), channels, edge, self._neuron_dim, rotations, flip, region, ed_type=self._map_type,
                                        device=self.device.index)
            self._mapper.set_som(self._rows)
        heat = torch.empty((images.shape[0], len(self._rows)), device=self.device)
        torch.cuda.synchronize()                           # the mapper runs on a stream of its own
        self._mapper.map_device(images.data_ptr(), images.shape[0], heat.data_ptr())
        self._mapper.synchronize()
        return heat

    def _geometry(self, images):
        channels = 1 if images.dim() == 3 else images.shape[1]
        if images.dim() not in (3, 4) or images.shape[-1] != images.shape[-2] or channels != self._neuron_channels:
            raise pink.exception(-1, "images must be (images, edge, edge) or (images, channels, edge, edge) with the neurons' channels")
        return int(channels), int(images.shape[-1])

    def _levels(self, heat):
        """(mean and spread of the images' distances, sharpness and radius to start from).  Distances that are not finite take no part."""
        part = torch.isfinite(heat)
        count, known = part.sum(), torch.where(part, heat, 0.0)
        mean = known.sum() / count.clamp(min=1)
        spread = (torch.where(part, heat - mean, 0.0).square().sum() / (count - 1).clamp(min=1)).sqrt() + 1e-6
        each = part.sum(0)
        return torch.stack((mean, spread)), (1 / spread).repeat(heat.shape[1]), torch.where(each > 0, known.sum(0) / each.clamp(min=1), mean)

    def _scale(self, heat):
        """Level, sharpness and radius: the read-out's, or before its first step those that the images would set."""
        return (self.level, self.parameters["sharpness"], self.parameters["radius"]) if self.level is not None else self._levels(heat)

    def _weights(self):
        return [self.parameters[k].data_ptr() for k in ("first", "first_bias", "second", "second_bias")]

    def _block(self, b, which=None):
        """Addresses of a block's parameters, or of their gradients: the layer norm's, and the gated block's."""
        of = self.parameters if which is None else which
        at = [of["block%d.%s" % (b, k)].data_ptr() for k in ("weight", "bias", "gate", "gate_bias", "up", "up_bias", "down", "down_bias")]
        return at[:2], at[2:]

    def _through_blocks(self, x, keep):
        """The features that the neurons' models see, and what a backward pass through the blocks needs."""
        r, (t, n), kept = self.readout, x.shape, []
        for b in range(self.blocks):
            norm, weights = self._block(b)
            normed, out = torch.empty_like(x), torch.empty_like(x)
            mean, scale, saved = None, None, None
            if keep:
                mean, scale = torch.empty(t, device=self.device), torch.empty(t, device=self.device)
                saved = torch.empty(r.gated_saved_bytes(self._shape, t), dtype=torch.uint8, device=self.device)
                kept.append((x, mean, scale, normed, saved))
            r.norm(x.data_ptr(), t, n, *norm, _EPSILON, normed.data_ptr(), mean.data_ptr() if keep else None, scale.data_ptr() if keep else None)
            r.gated(self._shape, normed.data_ptr(), t, weights, out.data_ptr(), dev_residual=x.data_ptr(), dev_saved=saved.data_ptr() if keep else None)
            x = out
        return x, kept

    def _back_through_blocks(self, kept, dx):
        """The blocks' gradients for those of the features that the models saw."""
        r, (t, n) = self.readout, dx.shape
        for b in reversed(range(self.blocks)):
            x, mean, scale, normed, saved = kept[b]
            (norm_weight, _), weights = self._block(b)
            (dweight, dbias), grads = self._block(b, self.gradients)
            dnormed = torch.empty_like(dx)
            r.gated_backward(self._shape, normed.data_ptr(), t, weights, saved.data_ptr(), dx.data_ptr(), [dnormed.data_ptr()] + grads)
            # (what came in needs none: distances are not trained)
            r.norm_backward(x.data_ptr(), t, n, norm_weight, mean.data_ptr(), scale.data_ptr(), dnormed.data_ptr(), dx.data_ptr() if b else None, dweight,
                            dbias, dev_residual=dx.data_ptr())

    def _forward(self, heat, keep):
        r, t = self.readout, heat.shape[0]
        level, sharpness, radius = scale = self._scale(heat)
        x = torch.where(torch.isfinite(heat), (heat - level[0]) / level[1], 0.0)
        neuron = torch.empty((t, self.chosen), dtype=torch.int32, device=self.device)
        gates, y = torch.empty((t, self.chosen), device=self.device), torch.empty((t, self.outputs), device=self.device)
        saved = torch.empty(r.saved_bytes(t), dtype=torch.uint8, device=self.device) if keep else None
        x, kept = self._through_blocks(x, keep)
        r.route(heat.data_ptr(), t, sharpness.data_ptr(), radius.data_ptr(), self.bias.data_ptr(), neuron.data_ptr(), gates.data_ptr())
        r.experts(x.data_ptr(), t, neuron.data_ptr(), gates.data_ptr(), self._weights(), y.data_ptr(), dev_saved=saved.data_ptr() if keep else None)
        return types.SimpleNamespace(x=x, neuron=neuron, gates=gates, y=y, saved=saved, kept=kept, scale=scale)

    @_on_its_device
    def __call__(self, images):
        """Answers, (images, outputs) on the GPU."""
        return self._forward(self.distances(images), False).y

    def _train(self, images, loss_of):
        """One step of AdamW; loss_of(answers) gives the loss and its gradient for the answers."""
        r, p, g = self.readout, self.parameters, self.gradients
        heat = self.distances(images)
        t = heat.shape[0]
        if t == 0:
            raise pink.exception(-1, "a step needs images")
        if self.level is None and not torch.isfinite(heat).any():
            raise pink.exception(-1, "the first step needs an image with a finite distance")
        f = self._forward(heat, True)
        loss, dy = loss_of(f.y)
        level, sharpness, radius = f.scale
        dgates, dx = torch.empty_like(f.gates), torch.empty_like(f.x) if self.blocks else None
        r.experts_backward(f.x.data_ptr(), t, f.gates.data_ptr(), self._weights(), f.saved.data_ptr(), dy.data_ptr(),
                           [dx.data_ptr() if self.blocks else None, dgates.data_ptr()] + [g[k].data_ptr() for k in ("first", "first_bias", "second", "second_bias")])
        if self.blocks:
            self._back_through_blocks(f.kept, dx)
        r.route_backward(heat.data_ptr(), t, sharpness.data_ptr(), radius.data_ptr(), self.bias.data_ptr(), f.neuron.data_ptr(),
                         f.gates.data_ptr(), dgates.data_ptr(), None, g["sharpness"].data_ptr(), g["radius"].data_ptr())
        if self.level is None:
            p["sharpness"].copy_(sharpness)
            p["radius"].copy_(radius)
        r.adamw(self._tensors, self.steps + 1, learning_rate=self.learning_rate, bits=self.state_bits)
        self.level, self.steps = level, self.steps + 1     # (a step that is refused sets neither)
        r.balance(f.neuron.data_ptr(), t, self.balance_rate, self.bias.data_ptr())
        return loss()

    @_on_its_device
    def step(self, images, targets):
        """One step of AdamW on the mean squared error of a batch; returns the error before the step, on the GPU."""
        def squared(y):
            off = y - torch.as_tensor(targets, dtype=torch.float32, device=self.device).reshape(y.shape)
            return lambda: (off * off).mean(), off * (2.0 / off.numel())
        return self._train(images, squared)

    @_on_its_device
    def teach(self, images, places, temperature=2.0):
        """What a smaller read-out learns from this one's answers, logits of classes: the `places` largest of each image and their normaliser."""
        if not 1 <= places <= min(self.outputs, 1024) or not torch.finfo(torch.float32).tiny <= temperature <= torch.finfo(torch.float32).max:
            raise pink.exception(-1, "a teacher gives between 1 and 1024 of its classes, at a temperature of 2^-126 or larger that float32 holds")
        y = self(images)
        top = y.topk(places, dim=1)
        return Teacher(top.indices.to(torch.int32), top.values.contiguous(), torch.logsumexp(y / temperature, 1), float(temperature))

    def _class_numbers(self, of):
        """As 32-bit numbers; what these cannot hold is past all classes, or before them, as it was."""
        of = torch.as_tensor(of, device=self.device)
        return (of if of.dtype == torch.int32 else of.to(torch.int64).clamp(-1, 2 ** 31 - 1).to(torch.int32)).contiguous()

    @_on_its_device
    def learn(self, images, labels=None, teacher=None, teacher_weight=1.0, label_weight=1.0):
        """One step of AdamW for answers that are logits of classes: on the cross entropy of `labels` (a class each, -1: none), on the distance from what a
        teacher's teach() gave for these images (the divergence at its temperature, times its square), or on both by their weights.  Returns the mean
        loss before the step, on the GPU."""
        if labels is None and teacher is None:
            raise pink.exception(-1, "classes are learned from labels or a teacher")

        def distilled(y):
            t, classes = y.shape
            given = dict(label_weight=0.0, teacher_weight=0.0)
            if labels is not None:
                label = self._class_numbers(labels)
                if label.shape != (t,):
                    raise pink.exception(-1, "labels must be a class for each image")
                given |= dict(dev_label=label.data_ptr(), label_weight=label_weight)
            if teacher is not None:
                at, (logits, normaliser) = self._class_numbers(teacher.classes), (v.to(self.device, torch.float32).contiguous() for v in teacher[1:3])
                if at.shape != logits.shape or at.shape[0] != t or normaliser.shape != (t,):
                    raise pink.exception(-1, "a teacher's places must be of these images")
                given |= dict(dev_teacher_class=at.data_ptr(), dev_teacher_logits=logits.data_ptr(), places=at.shape[1], temperature=teacher.temperature,
                              dev_teacher_normaliser=normaliser.data_ptr(), teacher_weight=teacher_weight)
            losses, dy, each = torch.empty(t, device=self.device), torch.empty_like(y), torch.full((t,), 1.0 / t, device=self.device)
            self.readout.distil(y.data_ptr(), t, classes, losses.data_ptr(), dy.data_ptr(), dev_image_weights=each.data_ptr(), **given)
            return losses.sum, dy
        return self._train(images, distilled)


def synthetic_sources(count, edge, rng):
    """(images, targets): one elliptical source each, turned anyhow; its size and axis ratio, scaled to about one."""
    size, ratio, angle = rng.uniform(1.5, 5.0, count), rng.uniform(0.3, 1.0, count), rng.uniform(0, math.pi, count)
    y, x = np.mgrid[:edge, :edge] - (edge - 1) / 2
    a = np.cos(angle)[:, None, None] * x + np.sin(angle)[:, None, None] * y
    b = np.cos(angle)[:, None, None] * y - np.sin(angle)[:, None, None] * x
    images = np.exp(-0.5 * ((a / size[:, None, None]) ** 2 + (b / (size * ratio)[:, None, None]) ** 2))
    images = np.clip(images + rng.normal(0, 0.02, images.shape), 0, 1).astype(np.float32)
    return images, np.stack([(size - 3.25) / 1.0, (ratio - 0.65) / 0.2], 1).astype(np.float32)


def distil_small_sources(som, images, targets, new, truth, steps, batch, rng, options):
    """Sixteen classes of size and axis ratio: a read-out is trained on labels, and a smaller one on labels and the first one's answers."""
    def classes(values):
        edges = np.quantile(targets, (0.25, 0.5, 0.75), axis=0)
        return sum((values[:, i, None] > edges[:, i]).sum(1) * 4 ** i for i in range(2)).astype(np.int32)
    label, right = classes(targets), classes(truth)
    teacher = MapReadout(som, outputs=16, hidden=64, **{**options, "blocks": max(1, options["blocks"])})
    student = MapReadout(som, outputs=16, hidden=8, **{**options, "blocks": 0})
    for name, learner, learn in (("teacher", teacher, lambda pick: teacher.learn(images[pick], label[pick])),
                                 ("student", student, lambda pick: student.learn(images[pick], label[pick], teacher.teach(images[pick], places=4)))):
        for step in range(steps):
            loss = learn(rng.integers(0, len(images), batch))
            if step % 50 == 0 or step + 1 == steps:
                print("%s, step %4d: loss %.4f" % (name, step + 1, float(loss)), flush=True)
        print("%s, new sources: %.3f of the classes right" % (name, float((learner(new).argmax(1).cpu().numpy() == right).mean())), flush=True)


def main(argv=None):
    parser = argparse.ArgumentParser(prog="pink_amd.readout", description="trains a small map on synthetic sources and a read-out of their size and axis ratio")
    parser.add_argument("--steps", type=int, default=300)
    parser.add_argument("--batch", type=int, default=256)
    parser.add_argument("--chosen", type=int, default=2)
    parser.add_argument("--state-bits", type=int, default=32, choices=(8, 32))
    parser.add_argument("--blocks", type=int, default=0, help="blocks that the neurons' models share")
    parser.add_argument("--distil", action="store_true", help="sixteen classes instead: a read-out on labels, and a smaller one from it")
    args = parser.parse_args(argv)
    rng = np.random.default_rng(0)
    edge, region = 32, 22
    torch.cuda.init()
    images, targets = synthetic_sources(4096, edge, rng)
    som = pink.SOM(rng.random((6, 6, edge, edge), dtype=np.float32) * 0.1)
    trainer = pink.Trainer(som, pink.GaussianFunctor(1.1, 0.2), number_of_rotations=92, euclidean_distance_dim=region)
    trainer.train(images)
    trainer.update_som()
    options = dict(chosen=args.chosen, state_bits=args.state_bits, number_of_rotations=92, euclidean_distance_dim=region, blocks=args.blocks)
    if args.distil:
        new, truth = synthetic_sources(1024, edge, rng)
        return distil_small_sources(som, images, targets, new, truth, args.steps, args.batch, rng, options)
    answers = MapReadout(som, outputs=2, **options)
    for step in range(args.steps):
        pick = rng.integers(0, len(images), args.batch)
        loss = answers.step(images[pick], targets[pick])
        if step % 50 == 0 or step + 1 == args.steps:
            print("step %4d: mean squared error %.4f" % (step + 1, float(loss)), flush=True)
    new, truth = synthetic_sources(1024, edge, rng)
    off = answers(new).cpu().numpy() - truth
    print("new sources: mean squared error %.4f (of the mean alone: %.4f)" % (float((off * off).mean()), float(truth.var(0).mean())), flush=True)


if __name__ == "__main__":
    main()
