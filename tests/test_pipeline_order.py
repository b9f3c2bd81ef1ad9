"""What StreamPipeline's waits order, on streams that only keep account: of any depth model and velocity model of one pipeline, one is behind the other."""
import contextlib
import itertools

import pytest
import torch

from evfly_amd.pipeline import StreamPipeline


class _Stream:
    """Work is a name; `seen` is all that ends before what this stream is given next."""

    def __init__(self):
        self.seen = set()

    def wait_stream(self, other):
        self.seen |= other.seen


class _Tensor:
    is_cuda = False

    def record_stream(self, stream):
        pass


class _Device:
    def __init__(self, monkeypatch):
        self.now, self.before = _Stream(), {}
        monkeypatch.setattr(torch.cuda, "current_stream", lambda: self.now)
        monkeypatch.setattr(torch.cuda, "stream", self.on)

    @contextlib.contextmanager
    def on(self, stream):
        old, self.now = self.now, stream
        try:
            yield
        finally:
            self.now = old

    def launch(self, kind):
        name = f"{kind}{len(self.before)}"
        self.before[name] = set(self.now.seen)
        self.now.seen.add(name)

    def together(self):
        return [(a, b) for a, b in itertools.combinations(self.before, 2) if a[0] != b[0] and a not in self.before[b] and b not in self.before[a]]


@pytest.fixture
def device(monkeypatch):
    return _Device(monkeypatch)


def _pipe(device):
    class Unet:
        def forward_streams(self, *a):
            device.launch("D")
            return _Tensor(), None, None

    class Vit:
        def _run(self, *a, **k):
            device.launch("P")
            return _Tensor(), None

    pipe = StreamPipeline.__new__(StreamPipeline)
    pipe.unet, pipe.vit, pipe.side = Unet(), Vit(), _Stream()
    return pipe


def test_steps_of_one_stream(device):
    pipe = _pipe(device)
    for _ in range(3):
        pipe.step(None, None, 1, 1)
    assert len(device.before) == 6 and device.together() == []


def test_steps_of_two_streams(device):
    pipe = _pipe(device)
    for stream in (_Stream(), _Stream(), device.now):
        with device.on(stream):
            pipe.step(None, None, 1, 1)
    assert device.together() == []


def test_a_step_whose_after_raises(device):
    pipe = _pipe(device)

    def after(vel):
        raise RuntimeError("no room")

    with pytest.raises(RuntimeError, match="no room"):
        pipe.step(None, None, 1, 1, after=after)
    device.launch("D")                                # the model itself, called on the same stream
    pipe.step(None, None, 1, 1)
    assert device.together() == []
