"""PagedAttention's workspace over streams: what a call's `stream` is ordered
behind, and what a host read of the plan is."""
import pytest

from test_paged import _Many, _Paged

pytestmark = pytest.mark.gpu


def _busy(torch, dev, times=40):
    """Tens of milliseconds of work for the current stream."""
    a = torch.ones(4096, 4096, device=dev)
    for _ in range(times):
        a = a @ a * 0.0
    return a


def test_a_read_of_the_plan_waits_for_the_plan(gpu):
    import torch
    p = _Many(gpu, [40, 333, 0], [50, 33, 200], 8, 2, 128, "bf16", 16, seed=6)
    att = p.attention()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        keep = _busy(torch, gpu)
    att.plan(p.cu, p.lengths, stream=s)
    assert int(att.work[12:16].view(torch.int32)) > 0  # workgroups of the second list
    s.synchronize()
    del keep


@pytest.mark.parametrize("wrapped", [False, True])
def test_a_plan_on_a_new_stream_waits_for_the_workspace(gpu, wrapped):
    """The zeros that the object is made with are still queued when another stream plans."""
    import torch
    p = _Paged(gpu, [700, 40, 2000], [1, 33, 5], 8, 2, 128, "bf16", 16, seed=13, pad=3)
    want = p.run()
    s = torch.cuda.Stream()
    stream = type("Handle", (), {"cuda_stream": s.cuda_stream})() if wrapped else s
    out = torch.full_like(p.q, 5.0)
    torch.cuda.synchronize()
    keep = _busy(torch, gpu)
    att = p.attention()
    att.plan(p.cu, p.lengths, stream=stream)
    torch.cuda.synchronize()  # the zeros, had they come after the plan
    att(p.q, p.k, p.v, p.table, out=out, stream=stream)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    del keep


def test_a_workspace_is_held_until_its_stream_is_done(gpu):
    """An object that is gone while its calls are queued on another stream: its memory is not given out before they ran."""
    import torch
    p = _Paged(gpu, [700, 40, 2000], [1, 33, 5], 8, 2, 128, "bf16", 16, seed=13, pad=3)
    want = p.run()
    s = torch.cuda.Stream()
    out = torch.full_like(p.q, 5.0)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        keep = _busy(torch, gpu)
    att = p.attention()
    size, at = att.work.numel(), att.work.data_ptr()
    att.plan(p.cu, p.lengths, stream=s)
    att(p.q, p.k, p.v, p.table, out=out, stream=s)
    del att
    other = torch.zeros(size, dtype=torch.uint8, device=gpu)
    assert other.data_ptr() != at
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    del keep


def test_a_captured_step_of_an_object_made_before(gpu):
    """Its first use on a stream of its own is in a capture; replayed with eager steps between."""
    import torch
    p = _Paged(gpu, [700, 40, 2000], [1, 33, 5], 8, 2, 128, "bf16", 16, seed=13, pad=3)
    want = p.run()
    att, out, s = p.attention(), torch.full_like(p.q, 5.0), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        att.plan(p.cu, p.lengths, stream=s)
        att(p.q, p.k, p.v, p.table, out=out, stream=s)
    for _ in range(3):
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(p.run(), want)
        torch.cuda.synchronize()


def test_objects_that_share_a_workspace(gpu):
    """Two objects of one shape take turns in one workspace, the second one's own given up."""
    import torch
    p = _Paged(gpu, [700, 40, 2000], [1, 33, 5], 8, 2, 128, "bf16", 16, seed=13, pad=3)
    want, windowed = p.run(), p.run(window=30)
    a, b = p.attention(), p.attention(window=30)
    b.work = a.work
    assert b.work.data_ptr() == a.work.data_ptr()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for att, expected in ((a, want), (b, windowed), (a, want)):
        out = torch.full_like(p.q, 5.0)
        s.wait_stream(torch.cuda.current_stream())
        att.plan(p.cu, p.lengths, stream=s)
        att(p.q, p.k, p.v, p.table, out=out, stream=s)
        s.synchronize()
        assert torch.equal(out, expected)
