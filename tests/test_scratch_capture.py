"""The kept scratch buffer of the Python half of the binding, and stream capture."""
import pytest
import torch


def test_a_capture_gets_scratch_of_its_own(monkeypatch):
    """Host logic only: tensors on the CPU stand in for the device's."""
    from actnn_b200 import _lib
    capturing = False
    monkeypatch.setattr(_lib, "_scratch", {})
    monkeypatch.setattr(_lib, "stream_of_index", lambda idx: 77)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    dev = torch.device("cpu")
    kept = _lib.scratch(dev, 5000)
    assert _lib.scratch(dev, 100) is kept and kept.numel() >= 5000
    capturing = True
    one, two = _lib.scratch(dev, 5000), _lib.scratch(dev, 0)
    assert len({t.data_ptr() for t in (kept, one, two)}) == 3 and one.numel() >= 5000 and two.numel() > 0
    assert list(_lib._scratch.values()) == [kept]                # nothing of a capture is kept
    _lib.scratch(dev, 1 << 24)
    assert list(_lib._scratch.values()) == [kept]                # and no capture takes the kept one's place
    capturing = False
    assert _lib.scratch(dev, 5000) is kept


@pytest.mark.gpu
def test_graphs_of_calls_that_need_scratch(cuda_device):
    """Two graphs, replayed at once on two streams beside calls that are not captured and after the kept buffer has grown: the backward
    pass of the norms around a residual branch, by the functions of the Python half."""
    from actnn_b200 import _lib
    from actnn_b200.cpp_extension import residual_norm as rn
    rows, c = 3000, 520
    g = torch.Generator().manual_seed(3)
    x, f, dr, dh = (torch.randn(rows, c, generator=g).to(torch.bfloat16).cuda() for _ in range(4))
    w, pw = (torch.randn(c, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    _, _, codes, stats = rn.run(x, f, w, None, pw, codes=True)

    def run(scale):
        return [t for t in rn.backward(dr * scale, dh, codes, stats, w, None, pw) if t is not None]

    def captured(scale, stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = run(scale)
        return graph, out

    streams = [torch.cuda.Stream() for _ in range(2)]
    want = [run(1.0), run(-2.0)]
    torch.cuda.synchronize()
    graphs = [captured(s, streams[0]) for s in (1.0, -2.0)]
    with torch.cuda.stream(streams[0]):
        run(1.0)                                                 # the stream's kept buffer; then a larger one, and tensors where it was
        _lib.scratch(x.device, _lib.scratch(x.device, 1).numel() * 4)
        others = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(64)]
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, out), ref in zip(graphs, want):
        assert len(out) == len(ref) and all(torch.equal(a, b) for a, b in zip(out, ref))
    assert all(bool((t == 7).all()) for t in others)
