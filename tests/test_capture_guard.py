"""The query/key norm's guard against captures next to live eager graphs, where the host
extension did not load.
"""

import pytest
import torch

from mlx_primitives import _native
from mlx_primitives.kernels import precompute_rope_cache, qk_norm_rope


def test_leaves_count_without_the_extension(monkeypatch):
    monkeypatch.setattr(_native, "_host", _native._GeneralPath())
    leaf, plain = torch.ones(4, requires_grad=True), torch.ones(4)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert not _native.live_leaf(plain, leaf)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert _native.live_leaf(plain, leaf)
    assert not _native.live_leaf(plain, leaf * 2)
    assert not _native.live_leaf(plain)


@pytest.mark.gpu
def test_a_capture_without_the_extension(device, monkeypatch):
    _native.load()
    q = torch.randn(1, 4, 2, 64, device=device)
    w = torch.ones(64, device=device, requires_grad=True)
    cos, sin = precompute_rope_cache(4, 64, device=device)
    want = qk_norm_rope(q, q, w.detach(), w.detach(), cos, sin)
    monkeypatch.setattr(_native, "_host", _native._GeneralPath())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="same leaf"):
            qk_norm_rope(q, q, w, w, cos, sin)
        with torch.no_grad():
            out = qk_norm_rope(q, q, w, w, cos, sin)
    for _ in range(3):
        out[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    qk_norm_rope(q, q, w, w, cos, sin)[0].sum().backward()  # (not captured)
    assert w.grad.any()
