"""RMS norm of queries and keys for each head, with the rotary rotation in the
same pass, on MI355X (an extension: the reference norms and rotates with
separate array operations).

One gfx950 kernel takes both tensors, normalises every head row, weights it,
rotates it to its position and rounds once; its backward is one kernel more
(and the sum of the weights' gradients).
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from mlx_primitives import _native


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x (B, S, H, D) as the kernels read it: 16-byte rows."""
    vec = 4 if x.dtype == torch.float32 else 8
    if x.stride(-1) != 1 or any(st % vec for st in x.stride()[:3]) or x.data_ptr() % 16:
        return _native.contiguous16(x)
    return x


class _QkNormRopeFn(torch.autograd.Function):
    """Saves the inputs; the backward computes the rows' norms again (they cost
    less than reading them back)."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, offset, positions, eps, errors):
        q, k = _rows(q), _rows(k)
        q_weight, k_weight = map(_native.contiguous16, (q_weight, k_weight))
        out = _forward(q, k, q_weight, k_weight, cos, sin, offset, positions, eps, errors)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.cfg = (offset, eps)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        offset, eps = ctx.cfg
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        dqw, dkw = torch.empty_like(q_weight), torch.empty_like(k_weight)
        _native.qk_norm_rope_bwd(q, k, q_weight, k_weight, cos, sin, _rows(dq_out), _rows(dk_out),
                                 dq, dk, dqw, dkw, offset, positions, eps)
        return dq, dk, dqw, dkw, None, None, None, None, None, None


def _forward(q, k, q_weight, k_weight, cos, sin, offset, positions, eps, errors):
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    if errors is not None and q.numel() + k.numel() == 0:
        errors.zero_()  # (no kernel runs, which would write them)
    _native.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, q_out, k_out, offset, positions, eps,
                         errors)
    return q_out, k_out


def _raise_outside(errors: torch.Tensor, seq: int, rows: int) -> None:
    if int(errors.item()):
        raise ValueError(f"a position in positions .. positions + {seq - 1} lies outside the "
                         f"cache's {rows} rows")


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    cos_cache: torch.Tensor,
    sin_cache: torch.Tensor,
    offset: int = 0,
    eps: float = 1e-6,
    positions: Optional[Union[torch.Tensor, list]] = None,
    check: bool = True,
    errors: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """(rope(rms_norm(q) * q_weight), rope(rms_norm(k) * k_weight)), each head row
    of dim values normalised by itself, in float32 and rounded once.

    q: (batch, seq, heads, dim), k: (batch, seq, kv_heads, dim), one dtype
    (float32, float16 or bfloat16); q_weight, k_weight: (dim,), one dtype of
    the three; cos_cache, sin_cache: (positions, dim // 2) as built by
    precompute_rope_cache. dim is a multiple of 16 up to 256. Slices of a wider
    projection are read in place.

    Row s of sequence b stands at position offset + s, or with positions (int
    (batch,) tensor or sequence) at positions[b] + s. With positions the call
    is that of rope_at: with ``check`` it waits and raises ValueError if a row's
    position falls outside the tables; otherwise such rows come out as zeros
    and ``errors`` (int32 (1,) device tensor, cleared here; a temporary when
    None) is set.

    Returns new contiguous tensors. Differentiable in q, k and both weights
    (the tables get no gradient, and there are no forward-mode derivatives); the
    weights' gradients are summed in float32 in a fixed order. A call that is captured
    into a HIP graph with gradients is refused (RuntimeError) while an eager autograd
    graph of one of its leaves, made on the default stream, is alive, and for any leaf
    where the host extension is not loaded, which could tell.
    """
    if positions is None or errors is not None or not check:
        # the ordinary call, checked and launched in native code
        out = _native.qk_norm_rope_new(q, k, q_weight, k_weight, cos_cache, sin_cache, offset, eps,
                                       positions, errors)
        if out is not None:
            if positions is not None and check:
                _raise_outside(errors, q.shape[1], cos_cache.shape[0])
            return out
    for name, x in (("q", q), ("k", k)):
        if x.ndim != 4:
            raise ValueError(f"Expected {name} of shape (batch, seq, heads, dim), got {x.ndim}D")
    B, S, H, D = q.shape
    if k.shape[:2] != q.shape[:2] or k.shape[3] != D:
        raise ValueError(f"q and k must agree in batch, seq and dim, got {tuple(q.shape)} and "
                         f"{tuple(k.shape)}")
    if k.dtype != q.dtype:
        raise ValueError(f"q/k dtype mismatch: {q.dtype}, {k.dtype}")
    _native.dtype_code(q.dtype)
    if D % 2:
        raise ValueError(f"head_dim must be even for RoPE, got {D}")
    if D % 16 or D > 256:
        raise NotImplementedError("qk_norm_rope: the MI355X kernel needs head_dim to be a "
                                  f"multiple of 16 up to 256, got {D}")
    if q_weight.shape != (D,) or k_weight.shape != (D,):
        raise ValueError(f"q_weight and k_weight must both be ({D},); got "
                         f"{tuple(q_weight.shape)} and {tuple(k_weight.shape)}")
    if k_weight.dtype != q_weight.dtype:
        raise ValueError(f"weight dtype mismatch: {q_weight.dtype}, {k_weight.dtype}")
    _native.dtype_code(q_weight.dtype)
    if cos_cache.shape != sin_cache.shape or cos_cache.ndim != 2 or cos_cache.shape[1] != D // 2:
        raise ValueError(f"cos/sin caches must both be (positions, {D // 2}); got "
                         f"{tuple(cos_cache.shape)} and {tuple(sin_cache.shape)}")
    if cos_cache.dtype != sin_cache.dtype:
        raise ValueError(f"cos/sin dtype mismatch: {cos_cache.dtype}, {sin_cache.dtype}")
    _native.dtype_code(cos_cache.dtype)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    dev = _native.require_device(q, k, q_weight, k_weight, cos_cache, sin_cache)
    _native.require_no_tangent(q, k, q_weight, k_weight, cos_cache, sin_cache)
    if torch.is_grad_enabled() and (cos_cache.requires_grad or sin_cache.requires_grad):
        raise NotImplementedError("qk_norm_rope: the cos/sin tables get no gradient; pass "
                                  "detached tables")
    if positions is None:
        if offset < 0 or offset + S > cos_cache.shape[0]:
            raise ValueError(f"positions {offset}..{offset + S - 1} exceed the cache's "
                             f"{cos_cache.shape[0]} rows")
        if errors is not None:
            raise ValueError("errors goes with positions")
        pos = None
    else:
        if offset != 0:
            raise ValueError("give offset or positions, not both")
        pos = torch.as_tensor(positions, dtype=torch.int32, device=dev).reshape(-1).contiguous()
        if pos.numel() != B:
            raise ValueError(f"positions must have {B} entries, got {pos.numel()}")
        if errors is None:
            errors = torch.empty(1, dtype=torch.int32, device=dev)
        elif errors.dtype != torch.int32 or errors.numel() != 1 or errors.device != dev:
            raise ValueError("errors must be an int32 tensor of 1 entry on q's device")
    cos, sin = _native.contiguous16(cos_cache), _native.contiguous16(sin_cache)
    if torch.is_grad_enabled() and any(x.requires_grad for x in (q, k, q_weight, k_weight)):
        if _native.live_leaf(q, k, q_weight, k_weight):
            raise RuntimeError("qk_norm_rope: a graph is being captured while an eager autograd "
                               "graph of the same leaf, made on the default stream, is alive (or, "
                               "without the host extension, may be); its gradient could not be "
                               "captured. Delete that graph's outputs first, or make it on a side "
                               "stream")
        out = _QkNormRopeFn.apply(q, k, q_weight, k_weight, cos, sin, offset, pos, float(eps),
                                  errors)
    else:
        weights = map(_native.contiguous16, (q_weight, k_weight))
        out = _forward(_rows(q), _rows(k), *weights, cos, sin, offset, pos, float(eps), errors)
    if pos is not None and check:
        _raise_outside(errors, S, cos_cache.shape[0])
    return out
