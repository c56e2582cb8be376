"""The query/key norm with weights that are not finite, and in calls of very many tokens."""

import pytest
import torch

from mlx_primitives.kernels import precompute_rope_cache, qk_norm_rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_rows_outside_the_tables_with_weights_that_are_not_finite(device, bad):
    # Such rows come out as zeros and get zeros, whatever the weights hold.
    q, k = (torch.randn(3, 2, h, 64, device=device) for h in (4, 2))
    w = torch.ones(64, device=device)
    w[5] = bad
    cos, sin = precompute_rope_cache(4, 64, device=device)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, w, w)]
    out = qk_norm_rope(*leaves, cos, sin, positions=torch.tensor([0, 3, -2]), check=False)
    grads = torch.autograd.grad(out, leaves, [torch.ones_like(x) for x in out])
    for y, dx in zip(out, grads):
        assert not y[1, 1].any() and not y[2].any()
        assert not dx[1, 1].any() and not dx[2].any()
    # the weights' gradients are those of the rows inside
    inside = [x.detach().clone().requires_grad_(True) for x in (q[:2], k[:2], w, w)]
    out = qk_norm_rope(*inside, cos, sin, positions=torch.tensor([0, 3]), check=False)
    for a, b in zip(grads[2:], torch.autograd.grad(out, inside, [torch.ones_like(x) for x in out])[2:]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("positions", [False, True])
def test_very_many_tokens(device, positions):
    # More than 2^26 tokens, the threads of whose waves a grid has no room for in one dimension:
    # head rows of 16 values, every sequence of 1025 tokens the same as the first or second.
    B, S, D = 65536, 1025, 16
    gen = torch.Generator(device=device).manual_seed(1)
    base = torch.randn(2, S, 1, D, device=device, generator=gen).to(torch.bfloat16)
    q = base.repeat(B // 2, 1, 1, 1)
    w = torch.rand(D, device=device, generator=gen)
    cos, sin = precompute_rope_cache(S + 1, D, device=device)
    pos = torch.ones(B, dtype=torch.int32, device=device) if positions else None
    errors = torch.full((1,), 5, dtype=torch.int32, device=device) if positions else None
    with torch.no_grad():
        got = qk_norm_rope(q, q, w, w, cos, sin, positions=pos, check=False, errors=errors)
        want = qk_norm_rope(base, base, w, w, cos, sin, offset=int(positions))
    assert not positions or errors.item() == 0
    for a, b in zip(got, want):
        assert torch.equal(a.view(B // 2, 2, S, 1, D), b.expand(B // 2, -1, -1, -1, -1))
    if positions:  # one row outside, of the last sequence
        pos[-1] = 2
        qk_norm_rope(q, q, w, w, cos, sin, positions=pos, check=False, errors=errors)
        assert errors.item() == 1
