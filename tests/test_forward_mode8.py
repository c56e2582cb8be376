"""Dual tensors of forward-mode differentiation are refused by the 8-bit cache and by the
query/key norm: their outputs would lack the tangents.
"""

import pytest
import torch
from torch.autograd import forward_ad

from mlx_primitives import _native
from mlx_primitives.cache import load_kv, paged_attention, set_block_data, store_kv
from mlx_primitives.kernels import precompute_rope_cache, qk_norm_rope


def dual(x):
    return forward_ad.make_dual(x, torch.ones_like(x))


def test_tangents_are_seen():
    x = torch.ones(3)
    _native.require_no_tangent(x, None)
    with forward_ad.dual_level():
        _native.require_no_tangent(x, None)
        d = dual(x)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _native.require_no_tangent(None, d)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            _native.require_no_tangent(d)
    _native.require_no_tangent(d)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_dual_tensors_are_refused(device, monkeypatch, native):
    _native.load()
    if not native:
        monkeypatch.setattr(_native, "_host", _native._GeneralPath())
    q, w = torch.randn(1, 2, 4, 64, device=device), torch.ones(64, device=device)
    cos, sin = (t.to(device) for t in precompute_rope_cache(8, 64))
    kp = torch.zeros((2, 16, 4, 64), dtype=torch.int8, device=device)
    vp, scales = kp.clone(), tuple(torch.zeros((2, 4), device=device) for _ in range(2))
    tab = torch.tensor([[0, 1]], dtype=torch.int32, device=device)
    one, two = (torch.tensor([n], dtype=torch.int32, device=device) for n in (0, 2))
    slopes = torch.ones(4, device=device)

    def calls(f):
        # (each with one tensor of its own as f makes it)
        for i in range(6):
            args = [q, q, w, w, cos, sin]
            args[i] = f(args[i])
            yield lambda args=args: qk_norm_rope(*args)
        for k, v in ((f(q), q), (q, f(q))):
            yield lambda k=k, v=v: store_kv(kp, vp, tab, k, v, one, check=False, kv_scales=scales)
            yield lambda k=k, v=v: set_block_data(kp, vp, 0, k[0], v[0], kv_scales=scales)
        for rope in ((f(cos), sin), (cos, f(sin))):
            yield lambda rope=rope: store_kv(kp, vp, tab, q, q, one, check=False, kv_scales=scales,
                                             rope=rope)
        for s in ((f(scales[0]), scales[1]), (scales[0], f(scales[1]))):
            yield lambda s=s: load_kv(kp, vp, tab, one, two, max_tokens=2, kv_scales=s)
            yield lambda s=s: paged_attention(q, kp, vp, tab, two, kv_scales=s)
        yield lambda: paged_attention(f(q), kp, vp, tab, two, kv_scales=scales)
        yield lambda: paged_attention(q, kp, vp, tab, two, kv_scales=scales, alibi_slopes=f(slopes))
    for call in calls(lambda x: x):
        call()
    with forward_ad.dual_level():
        for call in calls(lambda x: x):
            call()
        for call in calls(dual):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
