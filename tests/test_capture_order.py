"""A step is captured on a stream of its own, which has to wait for what the caller's stream still does to the state."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

import bench
from shiftaddllm_b200 import decoder, shard_decoder


@pytest.fixture()
def log(monkeypatch):
    """The calls of a capture, in order, on a host without a GPU."""
    seen, current = [], object()

    class Stream:
        def __init__(self, device=None):
            self.cuda_stream = 1

        def wait_stream(self, other):
            seen.append("wait" if other is current else "wait for another stream")

    @contextlib.contextmanager
    def on(name):
        seen.append(name)
        yield

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: on("side stream"))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: current)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: seen.append("synchronize"))
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: SimpleNamespace(replay=None))
    monkeypatch.setattr(torch.cuda, "graph", lambda g, stream=None: on("capture"))
    return seen


def state(log, **more):
    model = SimpleNamespace(device=torch.device("cpu"), token=torch.zeros(1), pos=torch.zeros(1), logits=torch.zeros(5), **more)

    def step():
        log.append("step")
        for t in (model.token, model.pos, model.logits):
            t.add_(1)

    model.step = step
    return model


def in_order(log, model):
    assert log[:3] == ["wait", "side stream", "step"] and log[-1] == "synchronize" and log.count("step") == 2
    assert not model.token.any() and not model.pos.any() and not model.logits.any()


def test_decoder(log):
    model = state(log)
    decoder.BcqLlamaDecoder.capture(model)
    in_order(log, model)


def test_column_parallel_decoder(log):
    model = state(log, _slot=0, blocks=[None] * shard_decoder.NSLOTS)
    shard_decoder.ColumnParallelDecoder.capture(model)
    in_order(log, model)


def test_the_benchmark_s_steps(log):
    args = SimpleNamespace(warmup=3)
    timer = bench.Timer(args, torch.device("cpu"), 1, torch.cuda.Stream())
    timer.capture(lambda: log.append("step"))
    assert log[:3] == ["wait", "side stream", "step"] and log.count("step") == 2
