"""The attention workspace: what it holds on to, and for whom."""
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops():
    from litert_b200 import ops as o

    return o


def test_growth_takes_what_is_needed_and_keeps_what_graphs_hold(ops, monkeypatch):
    """On the CPU, with a stand-in for the stream's state."""
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    ws = ops.Workspace.__new__(ops.Workspace)
    ws.device = torch.device("cpu")
    ws._no_attention_yet()
    assert ws.sdpa_bytes(1000).numel() == 1000
    assert ws.sdpa_bytes(1100).numel() == 1100 and not ws.outgrown  # not twice the size, and nothing kept
    assert ws.sdpa_bytes(500).numel() == 1100
    capturing[0] = True
    held = ws.sdpa_bytes(1100)
    capturing[0] = False
    assert ws.sdpa_bytes(900) is held
    assert ws.sdpa_bytes(1200).numel() == 1200 and len(ws.outgrown) == 1 and ws.outgrown[0] is held
    assert ws.sdpa_bytes(1300).numel() == 1300 and len(ws.outgrown) == 1  # (1200 was in no graph)
    capturing[0] = True
    grown = ws.sdpa_bytes(1400)  # a graph's own call outgrows it
    capturing[0] = False
    assert len(ws.outgrown) == 1 and ws.sdpa_bytes(1500).numel() == 1500 and ws.outgrown[1] is grown


def attend(ops, cache, ws, t=1, scores=None):
    q = torch.ones((cache[0].shape[0], t, 4, 64), device="cuda")
    return ops.sdpa_decode_int4(q, *cache, scores=scores, ws=ws)


def attend_float(ops, cache, ws, b=2):
    k = torch.ones((b, cache[0].shape[1], 2, 64), device="cuda")
    return ops.sdpa_decode(torch.ones((b, 1, 4, 64), device="cuda"), k, k, ws=ws)


@pytest.mark.gpu
@pytest.mark.parametrize("call", [attend, attend_float])
def test_a_captured_call_marks_the_workspace(ops, call):
    """Through the extension too, which takes the buffer that is there."""
    cache, ws = ops.int4_kv_cache(2, 9000, 2, 64), ops.Workspace("cuda")
    for _ in range(2):
        call(ops, cache, ws)
    assert not ws.captured and not ws.outgrown
    first, size = ws.sdpa, ws.sdpa.numel()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(ops, cache, ws)
    assert ws.captured and ws.sdpa is first
    call(ops, cache, ws)
    assert ws.captured
    need = 4 * size
    assert ws.sdpa_bytes(need).numel() == need and ws.outgrown[0] is first and not ws.captured
    call(ops, cache, ws)
    assert not ws.captured
    graph.replay()
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_growing_calls_hold_one_workspace(ops):
    """Batches that grow one sequence at a time: the memory of the largest call's workspace, not of twice that and of all
    before."""
    cache = ops.int4_kv_cache(24, 9000, 2, 64)
    ws = ops.Workspace("cuda")
    from litert_b200 import _lib

    for b in range(8, 25):
        scores = torch.zeros((b, 2, 9000), device="cuda")
        attend(ops, [x[:b] for x in cache], ws, t=4, scores=scores)
        need = _lib.load().b200_kv4_sdpa_workspace_bytes(b, 4, 4, 2, 64, 64, 9000, 1)
        assert ws.sdpa.numel() == need and not ws.outgrown


def test_a_workspace_of_another_device_is_refused(ops, monkeypatch):
    """The kernel would read and write the other device's addresses. On the CPU, with stand-ins for devices."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    ws = ops.Workspace.__new__(ops.Workspace)
    ws.device = torch.device("cpu")
    ws._no_attention_yet()
    assert ws.sdpa_bytes(100, torch.device("cpu")).numel() == 100
    with pytest.raises(ops.B200Error, match="device"):
        ws.sdpa_bytes(100, torch.device("meta"))
    with pytest.raises(ops.B200Error, match="device"):
        ws.sdpa_bytes(200, torch.device("meta"))
    assert ws.sdpa.numel() == 100
