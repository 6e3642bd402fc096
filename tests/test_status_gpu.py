"""Status words and workspaces whose first call is a captured one: zero before the first
replay, untouched by replays, and kept while a captured launch holds their address."""

import pytest
import torch

from batchstream_inference_engine_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture
def fresh(monkeypatch):
    """No stream has a status word or a workspace yet."""
    source = lambda i, s: ops._status_words.get(i, s).data_ptr()  # noqa: E731
    with monkeypatch.context() as m:
        m.setattr(ops, "_status_words", ops._StatusWords())
        m.setattr(ops, "_workspaces", ops._Workspaces())
        ops._native.set_status_source(source)
        # Words and buffers start in memory that held something else.
        junk = [torch.full((1 << 20,), 255, dtype=torch.uint8, device=DEV) for _ in range(8)]
        torch.cuda.synchronize()
        del junk
        yield
        torch.cuda.synchronize()
    ops._native.set_status_source(source)


def captured(stream, call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    return graph


def status(stream):
    with torch.cuda.stream(stream):
        return ops.take_status(torch.device(DEV))


def attention(op, rows=2):
    q = torch.randn(rows, 4, 64, device=DEV).bfloat16()
    pool = torch.randn(2, 8, 16, 64, device=DEV).bfloat16()
    table = torch.arange(2 * rows, dtype=torch.int32, device=DEV).view(rows, 2) % 8
    lens = torch.full((rows,), 20, dtype=torch.int32, device=DEV)
    if op == "window":
        return table, lambda: ops.window_attention_batched(q, pool, pool, table, lens, 0.125, 8, 1)
    return table, lambda: ops.paged_attention_batched(q, pool, pool, table, lens, 0.125)


@pytest.mark.parametrize("op", ["window", "full"])
def test_first_call_of_a_stream_is_captured(fresh, op):
    table, call = attention(op)
    call()  # kernels are loaded (on another stream)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graph = captured(stream, call)
    assert status(stream) == 0  # nothing ran
    table[1, 1] = 99
    graph.replay()
    torch.cuda.synchronize()
    table[1, 1] = 3
    graph.replay()  # reports nothing, and clears nothing
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="block table entry"):
        status(stream)
    assert status(stream) == 0
    graph.replay()
    torch.cuda.synchronize()
    assert status(stream) == 0


def test_a_captured_call_keeps_its_workspace(fresh):
    # A larger call on the stream moves its workspace; the graph still uses the old one.
    table, call = attention("full")
    stream = torch.cuda.Stream()
    graph = captured(stream, call)
    held = ops._workspaces.get(torch.device(DEV), stream.cuda_stream, 0)
    with torch.cuda.stream(stream):
        grown = ops.workspace_for(torch.device(DEV), 2 * held.numel())
    assert grown.data_ptr() != held.data_ptr()
    address, size = held.data_ptr(), held.numel()
    del held
    with torch.cuda.stream(stream):
        others = [torch.full((size,), 7, dtype=torch.uint8, device=DEV) for _ in range(4)]
        assert all(o.data_ptr() != address for o in others)
    table[1, 1] = 99
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(bool((o == 7).all()) for o in others)
    with pytest.raises(RuntimeError, match="block table entry"):
        status(stream)
    assert status(stream) == 0


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_a_workspace_grows_inside_a_capture(fresh):
    _, call = attention("full")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call()
        small = ops.workspace_for(torch.device(DEV), 0)
        small[:4].view(torch.int32).fill_(1)  # a status bit that nobody has taken
    torch.cuda.synchronize()
    graph = captured(stream, lambda: ops.workspace_for(torch.device(DEV), 2 * small.numel()))
    graph.replay()
    torch.cuda.synchronize()
    grown = ops._workspaces.get(torch.device(DEV), stream.cuda_stream, 0)
    assert grown.numel() >= 2 * small.numel() and not bool(grown.any())
    with pytest.raises(RuntimeError, match="block table entry"):
        status(stream)
    assert status(stream) == 0
