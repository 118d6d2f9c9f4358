"""The calls that perf/operators.py makes as a user's program: in order with the other work of the current stream and with a context and workspace for each device.
torch is stood in for by records of what was asked of its streams, so no GPU is needed."""
import importlib
import importlib.util
import os
import sys
import types

import pytest

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")


class Stream:
    def __init__(self, log, name):
        self.log, self.name, self.stream_id = log, name, id(self)

    def wait_stream(self, other):
        self.log.append((self.name, "waits for", other.name))


class Rows:
    """a tensor's address and stride; where it was made"""

    def __init__(self, made=None):
        self.made, self.used, self.dtype = made, [], None

    def data_ptr(self):
        return 4096

    def stride(self, _):
        return 8

    def numel(self):
        return 0

    def record_stream(self, stream):
        self.used.append(stream.name)


@pytest.fixture
def program(monkeypatch):
    """(module, log, torch.cuda as it was asked)"""
    log = []
    cuda = types.SimpleNamespace(device=0, current=Stream(log, "the caller's"), contexts=[])

    class Within:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            self.before, cuda.current = cuda.current, self.stream

        def __exit__(self, *_):
            cuda.current = self.before

    class Context:
        def __init__(self, device):
            self.device = device
            cuda.contexts.append(device)

        def stream(self):
            return "the context's of %d" % self.device

        def rotate(self, *_):
            log.append((self.stream(), "rotates"))

    cuda.current_device = lambda: cuda.device
    cuda.current_stream = lambda: cuda.current
    cuda.ExternalStream = lambda handle, device=None: Stream(log, handle)
    cuda.stream = Within

    def set_stream(stream):
        cuda.current = stream
    cuda.set_stream = set_stream
    torch = types.SimpleNamespace(cuda=cuda, accelerator=types.SimpleNamespace(current_stream=cuda.current_stream), Tensor=Rows, device=lambda *a: a, empty=lambda *a, **k: Rows(cuda.current.name), float32=0, float16=1, bfloat16=2, uint8=3, int32=4)
    framework = types.SimpleNamespace(Context=Context, RotateSpec=lambda *a: a, LV_F32=0, LV_F16=1, LV_BF16=30, LV_Q8_0=8, LV_Q4_0=2)
    spec = importlib.util.spec_from_file_location("operator_cases", PATH)
    module = importlib.util.module_from_spec(spec)
    with monkeypatch.context() as m:
        m.setitem(sys.modules, "torch", torch)
        spec.loader.exec_module(module)
    load = importlib.import_module
    monkeypatch.setattr(importlib, "import_module", lambda name, *a: framework if name == "llama-vulkan_amd" else load(name, *a))
    module.own = True
    return module, log, cuda


def rotation():
    return dict(c=dict(kind="rotate", tokens=1, heads=1, dim=8, rot=8, type="f32", pairs="halves", axes=1, base=1e4), x=Rows(), positions=Rows())


def test_calls_wait_for_the_current_stream_and_it_for_them(program):
    module, log, cuda = program
    out = module.run(rotation())
    ours, theirs = "the context's of 0", "the caller's"
    assert log == [(ours, "waits for", theirs), (ours, "rotates"), (theirs, "waits for", ours)]
    assert out.made == ours and out.used == [theirs]      # memory of the stream that writes it, not given back before the other has read it
    assert cuda.current.name == theirs


def test_a_program_whose_stream_is_the_contexts_waits_for_nothing(program):
    module, log, cuda = program
    try:
        module.prepare(rotation()["c"], 1)      # makes it so before anything is computed, which needs torch
    except AttributeError:
        pass
    assert cuda.current.name == "the context's of 0"
    module.run(rotation())
    assert log == [("the context's of 0", "rotates")]


def test_every_device_has_a_context_and_a_workspace(program):
    module, log, cuda = program
    module.run(rotation())
    cuda.device = 1
    module.run(rotation())
    module.run(rotation())
    cuda.device = 0
    module.run(rotation())
    assert cuda.contexts == [0, 1]
    assert [x[0] for x in log if x[1] == "rotates"] == ["the context's of %d" % i for i in (0, 1, 1, 0)]
