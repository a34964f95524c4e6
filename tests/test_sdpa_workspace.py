"""The scratch of the split-KV attention kernels is one buffer per stream for calls of every shape: what a call leaves in it is
never taken for another call's tickets."""
import pytest
import torch

from kuipy import _ffi


def test_tickets_take_the_same_place_in_every_workspace():
    """With the split count fixed the records grow with the batch alone, so what the sizes have in common is the tickets' share."""
    L = _ffi.lib()
    need = lambda n: L.kuiops_sdpa_workspace_bytes(_ffi.BF16, n, 32, 8, 1, 4096, 128, 128)        # noqa: E731
    L.kuiops_debug_sdpa_splits(32)
    try:
        share = {2 * need(n) - need(2 * n) for n in (1, 4, 8, 16, 60)}
        assert len(share) == 1 and share.pop() >= 4 * 8 * 120
        assert need(200) == 0                                  # more units than there are tickets: not split
    finally:
        L.kuiops_debug_sdpa_splits(0)


def _want(q, k, v):
    g = q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    return torch.softmax(q @ k.transpose(2, 3) * q.shape[3] ** -0.5, -1) @ v


@pytest.mark.gpu
@pytest.mark.parametrize("calls", [
    [("bf16", 8, 4096), ("bf16", 16, 4096), ("bf16", 30, 4096)],             # batches that grow
    [("f32", 4, 2048), ("f32", 16, 2048), ("f32", 30, 1024)],
    [("bf16", 1, 6000), ("f32", 20, 1500), ("bf16", 28, 3000), ("f32", 1, 3000), ("f32", 33, 1024)],     # both kernels in turn
], ids=["bf16", "f32", "both"])
def test_calls_of_growing_batches_share_a_workspace(cuda, calls):
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}
    tol = {"bf16": 3 * 2.0 ** -8, "f32": 1e-5}                 # weights and result rounded once each, and a little for the sums
    g = torch.Generator(device="cuda").manual_seed(1)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for kind, n, s in calls + calls:
            q, k, v = (torch.randn(n, hh, ll, 128, generator=g, device="cuda").to(dt[kind]) for hh, ll in ((16, 1), (8, s), (8, s)))
            assert _ffi.lib().kuiops_sdpa_workspace_bytes(_ffi.dtype_code(dt[kind]), n, 16, 8, 1, s, 128, 128) > 0, "a split case"
            out = torch.full((n, 16, 1, 128), float("nan"), device="cuda", dtype=dt[kind])
            _ffi.sdpa(q, k, v, out=out)
            want = _want(q, k, v)
            assert torch.isfinite(out).all() and float((out.double() - want).abs().max()) <= tol[kind] * float(v.abs().max())
    stream.synchronize()
    assert _ffi.tc_error() == 0


def test_a_workspace_made_inside_a_capture_stays_with_its_graph(monkeypatch):
    """Memory of a capture holds zeros only once the graph has run: it is not kept for calls outside."""
    dev = torch.device("cpu", 0)
    monkeypatch.setattr(_ffi, "_stream", lambda: 12345)
    monkeypatch.setattr(_ffi, "_scratch", {})
    monkeypatch.setattr(_ffi, "_capturing", lambda: True)
    first, second = _ffi.workspace("sdpa", dev, 5000), _ffi.workspace("sdpa", dev, 5000)
    assert first.data_ptr() != second.data_ptr() and first.numel() >= 5000 and int(first.sum()) == 0 and not _ffi._scratch
    monkeypatch.setattr(_ffi, "_capturing", lambda: False)
    kept = _ffi.workspace("sdpa", dev, 5000)
    assert kept.data_ptr() == _ffi.workspace("sdpa", dev, 7000).data_ptr()
    monkeypatch.setattr(_ffi, "_capturing", lambda: True)
    assert _ffi.workspace("sdpa", dev, 5000).data_ptr() == kept.data_ptr()          # made before: zero already
    assert _ffi.workspace("sdpa", dev, 2 << 20).data_ptr() != kept.data_ptr() and len(_ffi._scratch) == 1


@pytest.mark.gpu
def test_attention_first_called_inside_a_capture(cuda):
    """Split attention captured on a fresh stream without a warm-up, replayed, and called eagerly on that stream before and after."""
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(2, hh, ll, 128, generator=g, device="cuda").bfloat16() for hh, ll in ((16, 1), (8, 4096), (8, 4096)))
    want = _want(q, k, v)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        outs = [_ffi.sdpa(q, k, v)[0] for _ in range(3)]

    def eager():
        with torch.cuda.stream(side):
            out = torch.full((2, 16, 1, 128), float("nan"), device="cuda", dtype=torch.bfloat16)
            return _ffi.sdpa(q, k, v, out=out)[0]
    got = [eager()]
    for _ in range(3):
        for out in outs:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got += [eager()] + [out.clone() for out in outs]
    torch.cuda.synchronize()
    for out in got:
        assert torch.isfinite(out).all() and float((out.double() - want).abs().max()) <= 3 * 2.0 ** -8 * float(v.abs().max())
    del graph
