"""MapReadout, the read-out of a map from images to answers: on which stream it works, and what it keeps of its map and its first images."""
import contextlib
import os
import subprocess
import sys
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ------------------------------------------------------------------------------------------------------- without a GPU

class Recorder:
    """In the place of capi.Readout and of PyTorch's streams: what was called on which stream."""

    def __init__(self):
        self.calls, self.at, self.current = [], "own", "first"

    def set_stream(self, stream):
        self.at = stream

    def saved_bytes(self, images):
        return 16

    def __getattr__(self, name):
        if name.startswith("_"):
            raise AttributeError(name)
        return lambda *args, **options: self.calls.append((name, self.at, self.current))


class Stream:
    def __init__(self, name):
        self.cuda_stream = name

    def __eq__(self, other):
        return isinstance(other, Stream) and other.cuda_stream == self.cuda_stream


@pytest.fixture
def made(monkeypatch):
    """A MapReadout on the CPU, whose handle only records."""
    torch = pytest.importorskip("torch")
    from pink_amd import capi, pink, readout
    import numpy as np
    recorder = Recorder()
    monkeypatch.setattr(capi, "Readout", type("Readout", (), dict(check=staticmethod(lambda *a, **o: None), __new__=lambda cls, *a, **o: recorder)))
    recorder.tensors = lambda described: described
    monkeypatch.setattr(readout, "_check_one_runtime", lambda: None)
    monkeypatch.setattr(torch.cuda, "init", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(recorder.current))
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    real = torch.device
    monkeypatch.setattr(torch, "device", lambda *a: real("cpu"))
    som = pink.SOM(np.zeros((2, 3, 4, 4), np.float32))
    answers = readout.MapReadout(som, outputs=2, euclidean_distance_dim=3)
    monkeypatch.setattr(torch, "device", real)
    answers.distances = lambda images: torch.as_tensor(images)
    return answers, recorder, torch


def test_calls_go_to_the_stream_that_is_current_when_they_are_made(made):
    answers, recorder, torch = made
    heat = torch.rand(5, 6)
    for stream in ("first", "second", "second", "first", "third"):
        recorder.current = stream
        answers.step(heat, targets=torch.zeros(5, 2))
        answers(heat)
    assert {name for name, *_ in recorder.calls} == {"route", "experts", "experts_backward", "route_backward", "adamw", "balance"}
    assert all(at == current for _, at, current in recorder.calls)


def test_what_the_optimiser_holds_is_not_replaced(made):
    answers, _, torch = made
    for held in (answers.parameters, answers.gradients, answers.states, answers.states["first"]):
        with pytest.raises(TypeError):
            held["first"] = torch.zeros(1)
    answers.parameters["first"].fill_(2.0)


def test_states_that_are_refused(made):
    from pink_amd import pink
    answers, _, torch = made
    good = answers.state_dict()
    before = {k: v.clone() for k, v in answers._held().items()}
    for change in ({"bias": torch.zeros(7)}, {"parameters.first": good["parameters.first"].double()}, {"more": torch.zeros(1)}, {"level": torch.zeros(3)}):
        with pytest.raises(pink.exception):
            answers.load_state_dict({**{k: v if not torch.is_tensor(v) else v + 1 for k, v in good.items()}, **change})
    with pytest.raises(pink.exception):
        answers.load_state_dict({k: v for k, v in good.items() if k != "steps"})
    assert all(torch.equal(v, before[k]) for k, v in answers._held().items()) and answers.level is None
    answers.load_state_dict(good)


# ------------------------------------------------------------------------------------------------------------ on a GPU

def run(code):
    """In a process of its own: PyTorch has to come before the library."""
    code = """
import numpy as np, torch
from pink_amd import capi, pink, readout
EDGE, REGION = 32, 22
images, targets = readout.synthetic_sources(192, EDGE, np.random.default_rng(1))
def a_map(seed=2):
    return pink.SOM(np.random.default_rng(seed).random((4, 4, EDGE, EDGE), dtype=np.float32))
def made(som, **options):
    return readout.MapReadout(som, **{**dict(outputs=2, number_of_rotations=36, euclidean_distance_dim=REGION), **options})
def state(answers):
    return [v.cpu().numpy() for v in answers.parameters.values()] + [v.cpu().numpy() for s in answers.states.values() for v in s.values()]
""" + textwrap.dedent(code) + "\nprint('ok', flush=True)\n"
    done = subprocess.run([sys.executable, "-u", "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and done.stdout.strip().endswith("ok"), done.stdout[-1000:] + done.stderr[-2000:]


@pytest.mark.gpu
def test_steps_on_changing_streams_are_the_steps_on_one():
    run("""
    def train(streams, made_on):
        with torch.cuda.stream(made_on):
            answers = made(a_map())
        out = []
        for i in range(9):
            with torch.cuda.stream(streams[i % len(streams)]):
                at = slice(i % 3 * 64, i % 3 * 64 + 64)
                loss = answers.step(images[at], targets[at])
                out.append((loss + 0).cpu().numpy())           # the caller's own work, on its stream
                out.append(answers(images[at]).cpu().numpy())
        torch.cuda.synchronize()
        return out + state(answers)
    one, two, default = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.default_stream()
    want = train([default], default)
    for streams, first in (([one], default), ([one, two], one), ([default, one, two, one], two)):
        for a, b in zip(train(streams, first), want):
            assert np.array_equal(a, b)
    """)


@pytest.mark.gpu
def test_the_callers_device_stays_current():
    run("""
    answers = made(a_map())
    assert answers.device == torch.device("cuda", 0)
    answers.step(images=images[:32], targets=targets[:32])
    assert torch.cuda.current_device() == 0
    assert answers(images[:3]).device == answers.device and answers.distances(images[:3]).device == answers.device
    """)


@pytest.mark.gpu
def test_the_map_is_the_one_it_was_made_with():
    run("""
    som = a_map()
    answers, same = made(som), made(a_map())
    answers.step(images[:64], targets[:64])
    want = answers(images[:32]).cpu().numpy()
    small = images[:32, 2:-2, 2:-2].copy()
    np.asarray(som)[...] = np.asarray(a_map(7))                # the map is trained further
    assert np.array_equal(answers(images[:32]).cpu().numpy(), want)
    assert np.array_equal(answers.distances(small).cpu().numpy(), same.distances(small).cpu().numpy())     # images of another edge
    assert np.array_equal(answers(images[:32]).cpu().numpy(), want)
    assert not np.array_equal(made(som).distances(small).cpu().numpy(), same.distances(small).cpu().numpy())
    """)


@pytest.mark.gpu
def test_answers_before_the_first_step_change_nothing():
    run("""
    asked, not_asked = made(a_map()), made(a_map())
    assert np.isfinite(asked(images[100:103]).cpu().numpy()).all() and tuple(asked(images[:0]).shape) == (0, 2)
    assert asked.level is None
    for answers in (asked, not_asked):
        for i in range(3):
            answers.step(images[:64], targets[:64])
    heat = not_asked.distances(images[:64]).cpu().numpy().astype(np.float64)
    assert np.allclose(not_asked.level.cpu().numpy(), [heat.mean(), heat.std(ddof=1) + 1e-6], rtol=1e-5)
    for a, b in zip(state(asked), state(not_asked)):
        assert np.array_equal(a, b)
    """)


@pytest.mark.gpu
def test_distances_that_are_not_finite():
    # a neuron out of the competition, an image without any distance, a few entries: of the first images, and of later ones
    run("""
    clean, masked = made(a_map(), chosen=3), made(a_map(), chosen=3)
    heat = clean.distances(images[:64])
    hurt = heat.clone()
    hurt[:, 5], hurt[9], hurt[3, 7], hurt[4, 8] = float("inf"), float("nan"), float("nan"), float("-inf")
    for answers in (clean, masked):
        answers.distances = lambda images: torch.as_tensor(images, device="cuda")
    part = np.isfinite(hurt.cpu().numpy())
    known = hurt.cpu().numpy().astype(np.float64)[part]
    for i in range(4):
        loss = masked.step(hurt, targets[:64])
        assert np.isfinite(float(loss))
        if i == 0:
            assert np.allclose(masked.level.cpu().numpy(), [known.mean(), known.std(ddof=1) + 1e-6], rtol=1e-5)
    assert all(np.isfinite(x).all() for x in state(masked) if x.dtype == np.float32)
    assert not masked.states["second"]["first"].reshape(16, -1)[5].any()     # the neuron answered for nobody
    y = masked(hurt).cpu().numpy()
    assert np.isfinite(y).all() and not y[9].any()
    clean.step(heat, targets[:64])
    before = clean(heat).cpu().numpy()
    far = int(heat[0].argmax())                                # not among the three that answer for image 0
    one = heat[:1].clone()
    one[0, far] = float("inf")
    assert np.isfinite(clean(one).cpu().numpy()).all() and np.isfinite(before).all()
    """)


@pytest.mark.gpu
def test_steps_that_are_refused():
    run("""
    answers = made(a_map())
    real, none = answers.distances, torch.full((4, 16), float("inf"), device="cuda")
    for heat, text in ((none[:0], "needs images"), (none, "finite distance")):
        answers.distances = lambda images: heat
        try:
            answers.step(None, targets[:len(heat)])
        except pink.exception as e:
            assert text in str(e)
        else:
            raise AssertionError("taken")
        assert answers.level is None and answers.steps == 0
    answers.distances = real
    one = readout.MapReadout(pink.SOM(np.ones((1, 1, EDGE, EDGE), np.float32)), outputs=2, chosen=1, number_of_rotations=36, euclidean_distance_dim=REGION)
    assert np.isfinite(float(one.step(images[:1], targets[:1]))) and np.isfinite(one(images[:5]).cpu().numpy()).all()       # one distance in all
    assert np.isfinite(float(answers.step(images[:64], targets[:64])))
    """)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_training_goes_on_from_what_was_saved(bits):
    run("""
    import os, tempfile
    def train(answers, steps):
        for i in steps:
            at = slice(i %% 3 * 64, i %% 3 * 64 + 64)
            answers.step(images[at], targets[at])
        return state(answers) + [answers(images[:40]).cpu().numpy()]
    one, two = made(a_map(), state_bits=%d), made(a_map(), state_bits=%d, seed=5)
    train(one, range(4))
    with tempfile.TemporaryDirectory() as folder:
        torch.save(one.state_dict(), os.path.join(folder, "read-out"))
        two.load_state_dict(torch.load(os.path.join(folder, "read-out"), weights_only=True))
    assert two.steps == 4
    for a, b in zip(train(one, range(4, 8)), train(two, range(4, 8))):
        assert np.array_equal(a, b)
    """ % (bits, bits))
