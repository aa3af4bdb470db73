"""The serving calls on a stream that is not the current one, while the current one is busy
with work that the call must not wait for: what the calls make for themselves (scratch that
starts as zeros, results) belongs to the call's stream."""
import contextlib

import pytest
import torch

from mini_tensorrt_b200 import matmulq, serving
from tests.test_serving import BF16, F32, Paged, check_select, make_gen, randn

gpu = pytest.mark.gpu


def busy(seconds=0.2):
    """Work of about that long on the current stream (8192^3 products of some 0.8 ms)."""
    a = torch.zeros((8192, 8192), dtype=BF16, device="cuda")
    torch.cuda.synchronize()
    for _ in range(int(seconds / 0.0008)):
        a @ a


def other_stream(raw):
    s = torch.cuda.Stream()
    return s, (s.cuda_stream if raw else s)


@pytest.fixture
def fresh(cuda_device):
    """No kept workspaces, and memory whose next owner finds ones, not zeros."""
    kept = dict(serving._workspaces)
    serving._workspaces.clear()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.full((1 << 28,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    yield
    torch.cuda.synchronize()
    serving._workspaces.clear()
    serving._workspaces.update(kept)


@gpu
@pytest.mark.parametrize("raw", [False, True], ids=["stream", "address"])
@pytest.mark.parametrize("own", [False, True], ids=["kept", "handed_in"])
@pytest.mark.parametrize("kind", ["f32", "mixed"])
def test_attention_workspace_is_zeroed_on_the_calls_stream(fresh, raw, own, kind):
    """A first call and one that needs more, both with cut tiles, which are joined by tickets
    that have to start at zero."""
    calls = [Paged([1, 1], [3000, 800], 4, 2, 64, 32, kind, seed=1), Paged([200, 1], [3000, 900], 8, 2, 128, 32, kind, seed=2)]
    side, stream = other_stream(raw)
    ws = matmulq.Workspace("cuda") if own else None
    for s in calls:  # kernels are loaded by their first call
        s.run(workspace=torch.zeros(1 << 26, dtype=torch.uint8, device="cuda"))
    for s in calls:
        out = torch.full(s.q.shape, 9.0, dtype=s.kp.dtype, device="cuda")
        torch.full((1 << 26,), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        busy()
        s.run(out=out, workspace=ws, stream=stream)
        side.synchronize()
        assert not torch.cuda.current_stream().query(), "the current stream was to be busy for longer"
        got = out.cpu()  # (waits for the current stream)
        torch.cuda.synchronize()
        s.verify(got.cuda())


@gpu
def test_beam_workspace_is_zeroed_on_the_calls_stream(fresh):
    logits, scores = randn(make_gen(3), 12, 20000), -torch.rand((3, 4), device="cuda")
    done = torch.zeros((3, 4), dtype=torch.uint8, device="cuda")
    out = (torch.zeros_like(scores), *(torch.zeros((3, 4), dtype=torch.int32, device="cuda") for _ in range(2)),
           torch.zeros_like(done))
    side, stream = other_stream(False)
    serving.beam_select(logits, scores, done, 7, workspace=torch.zeros(1 << 22, dtype=torch.uint8, device="cuda"))
    torch.full((1 << 26,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    busy()
    serving.beam_select(logits, scores, done, 7, out=out, stream=stream)
    side.synchronize()
    assert not torch.cuda.current_stream().query()
    torch.cuda.synchronize()
    check_select(logits, scores, done, 7, out)


@gpu
@pytest.mark.parametrize("raw", [False, True], ids=["stream", "address"])
def test_results_belong_to_the_calls_stream(cuda_device, raw):
    """Memory that the current stream has been given back, but not yet written for the last
    time, is not where another stream's result goes."""
    s = Paged([1] * 4, [300, 40, 2, 77], 8, 2, 64, 32, "f32", seed=4)
    logits, scores = randn(make_gen(5), 4, 3000), -torch.rand((1, 4), device="cuda")
    done = torch.zeros((1, 4), dtype=torch.uint8, device="cuda")
    side, stream = other_stream(raw)
    s.run(stream=stream), serving.beam_select(logits, scores, done, 7, stream=stream)  # workspaces
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    busy()
    late = [torch.empty(s.q.shape, dtype=F32, device="cuda"), torch.empty((1, 4), device="cuda"),
            torch.empty((1, 4), dtype=torch.int32, device="cuda"), torch.empty((1, 4), dtype=torch.int32, device="cuda"),
            torch.empty((1, 4), dtype=torch.uint8, device="cuda")]
    for x in late:
        x.fill_(7)
    late.clear()
    del x
    out = s.run(stream=stream)
    picked = serving.beam_select(logits, scores, done, 7, stream=stream)
    side.synchronize()
    assert not torch.cuda.current_stream().query()
    torch.cuda.synchronize()
    s.verify(out)
    check_select(logits, scores, done, 7, picked)


@gpu
def test_results_outlive_their_readers_on_the_current_stream(cuda_device):
    """A result that the current stream still has to read is not handed out again by the
    other stream's memory when its last name goes."""
    s = Paged([1] * 4, [300, 40, 2, 77], 8, 2, 64, 32, "f32", seed=6)
    side = torch.cuda.Stream()
    s.run(stream=side)
    torch.cuda.synchronize()
    out = s.run(stream=side)
    want = out.clone()
    side.synchronize()
    torch.cuda.synchronize()
    busy()
    read = out.clone()
    del out
    with torch.cuda.stream(side):
        again = [torch.full(s.q.shape, 5.0, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(read, want) and len(again) == 4


@gpu
def test_address_of_the_default_stream(cuda_device):
    """stream=0 is the default stream, also where another is current."""
    s = Paged([1] * 4, [300, 40, 2, 77], 8, 2, 64, 32, "f32", seed=7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = s.run(stream=0)
    torch.cuda.synchronize()
    s.verify(out)


@gpu
def test_capture_without_a_workspace(fresh):
    """A capture that finds no kept workspace, or a small one, makes none that later calls
    would use: its memory is the graph's, and zeros are there from its first replay on."""
    small, large = Paged([1, 1], [300, 80], 4, 2, 64, 32, "f32", seed=1), Paged([200, 1], [3000, 900], 8, 2, 128, 32, "f32", seed=2)
    side = torch.cuda.Stream()
    for s in (small, large):
        s.run(workspace=torch.zeros(1 << 26, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    small.run(stream=side)
    side.synchronize()
    kept = {key: ws.buf for key, ws in serving._workspaces.items()}
    out = torch.zeros(large.q.shape, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        large.run(out=out)
    assert {key: ws.buf for key, ws in serving._workspaces.items()} == kept
    large.verify(large.run(stream=side))
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        large.verify(out)


@pytest.fixture
def fake_streams(monkeypatch):
    """Stream 7 is the current one; notes where each buffer is made, on the CPU."""
    made, now = [], [7]

    @contextlib.contextmanager
    def on(stream):
        before = now[0]
        now[0] = before if stream is None else stream[1]
        yield
        now[0] = before

    class Buffer:
        def __init__(self, n):
            self.n, self.recorded = n, []

        def numel(self):
            return self.n

        def record_stream(self, s):
            self.recorded.append(s)

    def zeros(n, dtype, device):
        made.append((now[0], Buffer(n)))
        return made[-1][1]

    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now[0])
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda ptr, device: ("external", ptr))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] == 11)
    monkeypatch.setattr(torch, "zeros", zeros)
    monkeypatch.setattr(serving, "_workspaces", {})
    return made


def scratch(ptr, nbytes, workspace=None):
    device = torch.device("cuda", 0)
    return serving._workspace(workspace, device, ptr, serving._other_stream(ptr, ptr, 0), nbytes)


def test_where_kept_workspaces_are_made(fake_streams):
    made = fake_streams
    a = scratch(9, 100)
    assert [at for at, _ in made] == [9]
    assert scratch(9, 100) is a and scratch(7, 50) is not a and len(made) == 2
    assert [at for at, _ in made] == [9, 7]
    b = scratch(9, 200)
    assert b is not a and [at for at, _ in made] == [9, 7, 9]
    assert a.recorded == [9]  # not given out again before stream 9 is done with it


def test_where_a_workspace_handed_in_grows(fake_streams):
    made, ws = fake_streams, matmulq.Workspace("cuda")
    a = scratch(7, 100, ws)
    assert scratch(9, 100, ws) is a
    b = scratch(9, 101, ws)
    assert b is not a and [at for at, _ in made] == [7, 9] and a.recorded == [9]
    mine = object()
    assert scratch(9, 10 ** 6, mine) is mine


@pytest.mark.parametrize("own", [False, True])
def test_what_a_capture_needs_is_not_kept(fake_streams, own):
    """Stream 11 is being captured."""
    made, ws = fake_streams, matmulq.Workspace("cuda") if own else None
    a = scratch(11, 100, ws)
    b = scratch(11, 100, ws)
    assert a is not b and [at for at, _ in made] == [11, 11]
    assert all(w.buf is None for w in serving._workspaces.values()) and (ws is None or ws.buf is None)


def test_a_capture_uses_what_is_there(fake_streams):
    ws = matmulq.Workspace("cuda")
    a = scratch(9, 100, ws)
    assert scratch(11, 100, ws) is a and scratch(11, 101, ws) is not a and ws.buf is a
