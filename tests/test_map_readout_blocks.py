"""MapReadout with blocks that all neurons share, and with answers that are classes: against PyTorch's automatic differentiation in 64 bits, and what is refused."""
import subprocess
import sys

import pytest

from test_map_readout import ROOT, made, run  # noqa: F401  (made: fixture)


def test_read_outs_and_steps_that_are_refused(made):  # noqa: F811
    from pink_amd import pink, readout
    answers, recorder, torch = made
    for wrong in (dict(blocks=-1), dict(blocks=1, block_hidden=0), dict(blocks=1, block_hidden=2 ** 20 + 1)):
        with pytest.raises(pink.exception) as e:
            readout.MapReadout(answers.som, outputs=2, euclidean_distance_dim=3, **wrong)
        assert "blocks" in str(e.value)
    heat = torch.rand(5, 6)
    good = readout.Teacher(torch.zeros(5, 2, dtype=torch.int32), torch.zeros(5, 2), torch.zeros(5), 2.0)
    for options, text in ((dict(), "labels or a teacher"), (dict(labels=[0, 1]), "a class for each image"), (dict(teacher=good._replace(normaliser=torch.zeros(4))), "of these images"),
                          (dict(teacher=good._replace(logits=torch.zeros(5, 3))), "of these images"),
                          (dict(teacher=good._replace(classes=torch.zeros(4, 2), logits=torch.zeros(4, 2))), "of these images")):
        before = {k: v.clone() for k, v in answers._held().items() if k not in ("parameters.sharpness", "parameters.radius")}
        with pytest.raises(pink.exception) as e:
            answers.learn(heat, **options)
        assert text in str(e.value) and answers.steps == 0 and all(torch.equal(v, before[k]) for k, v in answers._held().items() if k in before)
    for places, temperature in ((0, 2.0), (3, 2.0), (1, 0.0), (1, float("inf")), (1, float("nan"))):
        with pytest.raises(pink.exception):
            answers.teach(heat, places, temperature)
    recorder.calls.clear()
    answers.learn(heat, labels=[0, 1, -1, 0, 1], teacher=good)
    assert [name for name, *_ in recorder.calls] == ["route", "experts", "distil", "experts_backward", "route_backward", "adamw", "balance"]


def test_a_first_step_that_is_refused_sets_nothing(made):  # noqa: F811
    """Neither level, sharpness and radius nor anything else: the next step's images are the first then."""
    from pink_amd import capi, pink, readout
    answers, recorder, torch = made
    heat = torch.rand(5, 6)
    good = readout.Teacher(torch.zeros(5, 2, dtype=torch.int32), torch.zeros(5, 2), torch.zeros(5), 2.0)
    before = {k: v.clone() for k, v in answers._held().items()}
    def unchanged():
        return answers.level is None and answers.steps == 0 and all(torch.equal(v, before[k]) for k, v in answers._held().items())
    for options in (dict(), dict(labels=[0, 1]), dict(teacher=good._replace(normaliser=torch.zeros(4))), dict(labels=[0] * 5, teacher=good._replace(logits=torch.zeros(5, 3)))):
        with pytest.raises(pink.exception):
            answers.learn(heat, **options)
        assert unchanged()
    for targets in (torch.zeros(4, 2), torch.zeros(5, 3), torch.zeros(3)):
        with pytest.raises(Exception):
            answers.step(heat, targets)
        assert unchanged()
    with pytest.raises(pink.exception):
        answers.step(torch.full((5, 6), float("inf")), torch.zeros(5, 2))
    assert unchanged()
    def refuse(*args, **options):                          # as the library does what only it looks at: weights, a temperature
        raise capi.PinkError(-1, "weights must be finite")
    recorder.distil = refuse
    with pytest.raises(capi.PinkError):
        answers.learn(heat, labels=[0] * 5, label_weight=float("nan"))
    assert unchanged()
    recorder.adamw = refuse
    with pytest.raises(capi.PinkError):
        answers.step(heat, torch.zeros(5, 2))
    assert answers.level is None and answers.steps == 0
    del recorder.adamw
    later = heat * 3 + 1
    level, sharpness, radius = answers._levels(later)
    answers.step(later, torch.zeros(5, 2))
    assert answers.steps == 1 and torch.equal(answers.level, level)
    assert torch.equal(answers.parameters["sharpness"], sharpness) and torch.equal(answers.parameters["radius"], radius)
    answers.step(heat, torch.zeros(5, 2))
    assert answers.steps == 2 and torch.equal(answers.level, level) and torch.equal(answers.parameters["radius"], radius)


def test_teachers_are_of_temperatures_that_are_learned_at(made):  # noqa: F811
    """learn() hands the temperature on as a float32 that is not subnormal: teach() gives no answers at any other."""
    from pink_amd import pink
    answers, _, torch = made
    for temperature in (1e-40, 2.0 ** -127, 2.0 ** 128 * (1 - 2.0 ** -30), 2.0 ** 128, 1e39, -1.0):
        with pytest.raises(pink.exception):
            answers.teach(torch.rand(5, 6), 1, temperature)
    for temperature in (2.0 ** -126, 1, 2.0 ** 127):
        assert answers.teach(torch.rand(5, 6), 1, temperature).temperature == temperature


def test_class_numbers_that_32_bits_do_not_hold_are_no_classes(made):  # noqa: F811
    from pink_amd import readout
    import ctypes
    answers, recorder, torch = made
    taken = {}

    def distil(*args, dev_label, dev_teacher_class, places, **options):      # (on the CPU here: addresses that can be read)
        taken["label"] = list((ctypes.c_int32 * 5).from_address(dev_label))
        taken["teacher"] = list((ctypes.c_int32 * (5 * places)).from_address(dev_teacher_class))
    recorder.distil = distil
    far = [1, -1, 2 ** 32 + 1, -2 ** 32 + 1, 2 ** 31]
    teacher = readout.Teacher(torch.tensor([far, [0, 1, 2 ** 40, 1, 0]]).T, torch.zeros(5, 2), torch.zeros(5), 2.0)
    answers.learn(torch.rand(5, 6), labels=far, teacher=teacher)
    assert taken["label"] == [1, -1, 2 ** 31 - 1, -1, 2 ** 31 - 1]
    assert taken["teacher"] == [1, 0, -1, 1, 2 ** 31 - 1, 2 ** 31 - 1, -1, 1, 2 ** 31 - 1, 0]
    for labels in (torch.tensor([0, 1, 1, 0, 1], dtype=torch.uint8), torch.tensor([False, True, True, False, True]), torch.tensor([0, 1, 1, 0, 1], dtype=torch.int32)):
        answers.learn(torch.rand(5, 6), labels=labels, teacher=teacher)
        assert taken["label"] == [0, 1, 1, 0, 1]


# What a step's gradients are, in 64 bits; every product of K terms is off by (K + 2) 2^-24 of its magnitudes at most, K <= 256 here, and ten of them follow each other:
# 2e-4 of a tensor's largest entry, with sums of magnitudes no more than a few times that.
REFERENCE = """
def restated(answers, heat, images_loss):
    d = {k: v.double().clone().requires_grad_() for k, v in before.items()}
    heat = heat.double()
    level = answers.level.double()
    x = (heat - level[0]) / level[1]
    for b in range(answers.blocks):
        q = {k.split(".")[1]: v for k, v in d.items() if k.startswith("block%d." % b)}
        n = (x - x.mean(1, keepdim=True)) * (x.var(1, keepdim=True, unbiased=False) + 1e-5).rsqrt() * q["weight"] + q["bias"]
        x = x + (torch.nn.functional.silu(n @ q["gate"].T + q["gate_bias"]) * (n @ q["up"].T + q["up_bias"])) @ q["down"].T + q["down_bias"]
    z = d["sharpness"] * (d["radius"] - heat)
    top = (z.float() + bias).topk(answers.chosen, dim=1).indices       # (the bias takes part in the choice alone)
    gates = torch.softmax(z.gather(1, top), 1)
    hidden = torch.nn.functional.gelu(torch.einsum("tf,tkhf->tkh", x, d["first"][top]) + d["first_bias"][top])
    y = ((torch.einsum("tkh,tkoh->tko", hidden, d["second"][top]) + d["second_bias"][top]) * gates[..., None]).sum(1)
    loss = images_loss(y)
    loss.backward()
    return loss.item(), {k: v.grad for k, v in d.items()}
def check(answers, loss, want):
    value, grads = want
    assert abs(float(loss) - value) <= 2e-4 * abs(value), (float(loss), value)
    for k, v in grads.items():
        off, size = (answers.gradients[k].double() - v).abs().max().item(), v.abs().max().item()
        assert off <= 2e-4 * size, (k, off, size)
def randomised(answers):
    gen = torch.Generator(device="cuda").manual_seed(5)
    for k, v in answers.parameters.items():
        if k.startswith("block"):
            v.copy_(torch.randn(v.shape, device="cuda", generator=gen) * (0.3 if v.dim() == 1 else 1 / v.shape[-1] ** 0.5) + (1 if k.endswith(".weight") else 0))
"""


@pytest.mark.gpu
@pytest.mark.parametrize("blocks", [0, 1, 2])
def test_gradients_of_a_step(blocks):
    run(REFERENCE + """
answers = made(a_map(), blocks=%d, block_hidden=40)
randomised(answers)
answers.step(images[64:128], targets[64:128])              # (the first step sets the scale)
before, bias = {k: v.clone() for k, v in answers.parameters.items()}, answers.bias.clone()
heat, goal = answers.distances(images[:64]), torch.as_tensor(targets[:64], device="cuda").double()
loss = answers.step(images[:64], targets[:64])
check(answers, loss, restated(answers, heat, lambda y: ((y - goal) ** 2).mean()))
""" % blocks)


@pytest.mark.gpu
@pytest.mark.parametrize("blocks, labelled, taught", [(0, True, False), (1, False, True), (2, True, True)])
def test_gradients_of_learning(blocks, labelled, taught):
    run(REFERENCE + """
blocks, labelled, taught = %r, %r, %r
teacher, answers = made(a_map(), outputs=9, hidden=48, seed=3), made(a_map(), outputs=9, blocks=blocks, block_hidden=40)
randomised(answers)
rng = np.random.default_rng(6)
label = rng.integers(-1, 9, 192).astype(np.int32)
answers.learn(images[64:128], label[64:128])
before, bias = {k: v.clone() for k, v in answers.parameters.items()}, answers.bias.clone()
heat, taken = answers.distances(images[:64]), teacher.teach(images[:64], places=3, temperature=1.5)
full = teacher(images[:64]).double()
loss = answers.learn(images[:64], label[:64] if labelled else None, taken if taught else None, teacher_weight=0.7, label_weight=0.4)
def of(y):
    total = 0
    if labelled:
        goal = torch.as_tensor(label[:64], device="cuda").long()
        total = total + 0.4 * torch.nn.functional.cross_entropy(y, goal, ignore_index=-1, reduction="sum") / 64
    if taught:
        t = 1.5
        p, q, at = torch.softmax(full / t, 1), torch.softmax(y / t, 1), taken.classes.long()
        pk, qk = p.gather(1, at), q.gather(1, at)
        rest, others = 1 - pk.sum(1), 1 - qk.sum(1)
        total = total + 0.7 * t * t * ((pk * (pk / qk).log()).sum(1) + rest * (rest / others).log()).mean()
    return total
check(answers, loss, restated(answers, heat, of))
assert torch.equal(taken.classes.long(), full.float().topk(3, dim=1).indices) and taken.temperature == 1.5
""" % (blocks, labelled, taught))


@pytest.mark.gpu
def test_blocks_start_as_nothing_and_leave_other_parameters_as_they_are():
    run("""
    plain, with_blocks = made(a_map()), made(a_map(), blocks=2)
    for k, v in plain.parameters.items():
        assert torch.equal(v, with_blocks.parameters[k])
    assert torch.equal(plain(images[:50]), with_blocks(images[:50]))
    assert with_blocks.block_hidden == 32
    """)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_training_with_blocks_on_changing_streams_and_from_what_was_saved(bits):
    run("""
    options = dict(blocks=2, block_hidden=24, outputs=5, state_bits=%d)
    label = np.random.default_rng(7).integers(0, 5, 192).astype(np.int32)
    teacher = made(a_map(), outputs=5, seed=4)
    def train(answers, streams, steps):
        for i in steps:
            with torch.cuda.stream(streams[i %% len(streams)]):
                at = slice(i %% 3 * 64, i %% 3 * 64 + 64)
                answers.learn(images[at], label[at], teacher.teach(images[at], 2))
    one, two, default = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.default_stream()
    whole, parts, again = made(a_map(), **options), made(a_map(), **options), made(a_map(), **options)
    train(whole, [default], range(9))
    train(parts, [one, two, default], range(5))
    again.load_state_dict(parts.state_dict())
    train(again, [two, one], range(5, 9))
    torch.cuda.synchronize()
    for a, b in zip(state(whole), state(again)):
        assert np.array_equal(a, b)
    for other in (made(a_map(), outputs=5, state_bits=%d), made(a_map(), **{**options, "block_hidden": 25})):
        try:
            other.load_state_dict(parts.state_dict())
        except pink.exception:
            continue
        assert False, "the state of another read-out was taken"
    """ % (bits, bits))


@pytest.mark.gpu
@pytest.mark.parametrize("options, lines", [(["--blocks", "1"], ["new sources: mean squared error"]),
                                            (["--distil"], ["teacher, new sources:", "student, new sources:"])])
def test_the_command_runs(options, lines):
    done = subprocess.run([sys.executable, "-u", "-m", "pink_amd.readout", "--steps", "20"] + options, cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stderr[-2000:]
    assert all(line in done.stdout for line in lines), done.stdout
