"""Calls on one context from several streams: scratch and counters are the context's, so a stream bound later
waits for what went to the one before."""
import numpy as np
import pytest
import torch


class _Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(ptr, stream):
            self.calls.append((name, stream))
            return 0
        return call


def test_a_change_of_stream_is_ordered(monkeypatch):
    from shardlm_b200 import runtime

    class Stream:
        def __init__(self, raw):
            self.cuda_stream = raw

    rec = _Recorder()
    monkeypatch.setattr(runtime, "lib", lambda: rec)
    c = runtime.Context.__new__(runtime.Context)
    c.device, c.ptr, c._bound_stream = 0, None, None
    for raw in (7, 7, 9, 9, 7, 0):
        c.bind_stream(Stream(raw))
    assert rec.calls == [("shd_set_stream", 7), ("shd_switch_stream", 9), ("shd_switch_stream", 7), ("shd_switch_stream", 0)]


class Calls:
    """Attention calls that are cut and joined in scratch, with the results they give alone."""

    def __init__(self, ctx):
        from shardlm_b200.kv4 import Kv4Cache

        g = torch.Generator(device="cuda")
        g.manual_seed(3)
        heads, d, n = 2, 128, 6000
        self.cache = Kv4Cache(ctx, 2, heads, n, d)
        x = [torch.randn(n, heads * d, device="cuda", generator=g) for _ in range(4)]
        self.cache.write_prompt(x[0], None, x[1], None, slot=0, pos0=0)
        self.cache.write_prompt(x[2], None, x[3], None, slot=1, pos0=0)
        self.q = torch.randn(64, 8 * d, device="cuda", generator=g)
        self.slot = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        self.pos = torch.tensor([n - 1, n - 300], dtype=torch.int32, device="cuda")
        self.alone = [self.run(i) for i in range(4)]
        torch.cuda.synchronize()

    def run(self, i):
        if i % 2:
            return self.cache.attend(self.q[i:i + 2], slot=self.slot, pos=self.pos)[0]
        return self.cache.attend_prompt(self.q[i:i + 40], slot=i // 2, pos0=5900)[0]


@pytest.mark.gpu
def test_two_streams_take_turns_without_synchronisation(ctx):
    calls = Calls(ctx)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for k in range(24):
        with torch.cuda.stream(streams[k % 2]):
            got.append(calls.run(k % 4))
    torch.cuda.synchronize()
    for k, y in enumerate(got):
        assert torch.equal(y, calls.alone[k % 4]), k
    ctx.bind_stream()
    ctx.sync()


@pytest.mark.gpu
def test_streams_around_and_within_a_capture(ctx):
    calls = Calls(ctx)
    side, branch = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        before = calls.run(0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        here = torch.cuda.current_stream()
        one = calls.run(1)
        branch.wait_stream(here)
        with torch.cuda.stream(branch):  # a second branch, whose work needs the same scratch
            two = calls.run(2)
        three = calls.run(3)
        here.wait_stream(branch)
    with torch.cuda.stream(side):
        after = calls.run(3)
    torch.cuda.synchronize()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for y, i in ((before, 0), (one, 1), (two, 2), (three, 3), (after, 3)):
        assert torch.equal(y, calls.alone[i]), i
    ctx.bind_stream()
    ctx.sync()


@pytest.mark.gpu
def test_an_idle_stream_is_left_alone(ctx):
    """After sync() the stream that was bound is not touched any more, as its owner may have destroyed it."""
    calls = Calls(ctx)
    with torch.cuda.stream(torch.cuda.Stream()):
        calls.run(1)
        ctx.sync()
    y = calls.run(1)
    ctx.sync()
    assert torch.equal(y, calls.alone[1])
    assert np.isfinite(y.cpu().numpy()).all()
