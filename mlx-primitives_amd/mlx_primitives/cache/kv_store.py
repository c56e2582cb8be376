"""Writes of new K/V tokens into a paged KV cache on MI355X.

Drop-in for the page writes of the reference's KV cache:
KVCache._store_kv (mlx_primitives/cache/kv_cache.py:194-264) and
BlockAllocator.set_block_data (mlx_primitives/cache/block_allocator.py:299-331),
over the same pools (num_blocks, block_size, H, D) and int32 block tables
padded with -1. One gfx950 scatter kernel writes every new token of every
sequence into its page slot; the allocator bookkeeping (which pages a sequence
owns, eviction, copy-on-write) stays with the caller.

Pools may also hold 8-bit codes with a scale for each page and head: store_kv
quantises on the way in, load_kv gives tokens back as values.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from mlx_primitives import _native


def _i32(x, device, n: int, what: str) -> torch.Tensor:
    if type(x) is int and n > 0 and -2**31 <= x < 2**31:
        # filled on the device: a copy from the host would wait for the stream
        # (as_tensor refuses what int32 does not hold)
        return torch.full((n,), x, dtype=torch.int32, device=device)
    t = torch.as_tensor(x, dtype=torch.int32, device=device).reshape(-1)
    if t.numel() == 1 and n > 1:
        t = t.expand(n)
    if t.numel() != n:
        raise ValueError(f"{what} must have {n} entries, got {t.numel()}")
    return t.contiguous()


def _raise_errors(flags) -> None:
    neg, past, bad = (int(x) for x in flags[:3])
    if len(flags) > 3 and int(flags[3]):
        raise ValueError("RoPE position out of range: a token's position lies past the "
                         "cos/sin tables")
    if neg:
        raise ValueError("Invalid write_start position: a start position is negative")
    if past:
        raise RuntimeError("Block index out of range: a token's position lies past its "
                           "sequence's block table")
    if bad:
        raise ValueError("Invalid block_id: a block table entry is outside the pool")


def check_pools8(k_pool: torch.Tensor, v_pool: torch.Tensor,
                 kv_scales: Tuple[torch.Tensor, torch.Tensor]) -> None:
    """Pools of 8-bit codes and their scales, as the kernels take them."""
    if k_pool.dtype not in _native.CODE8_FORMATS or v_pool.dtype != k_pool.dtype:
        raise ValueError("pools with kv_scales hold torch.float8_e4m3fn or torch.int8 codes, one "
                         f"format; got {k_pool.dtype} and {v_pool.dtype}")
    if k_pool.shape[3] % 16 or k_pool.shape[3] > 256:
        raise NotImplementedError("8-bit pools need head_dim to be a multiple of 16 up to 256, "
                                  f"got {k_pool.shape[3]}")
    if k_pool.shape[1] > _native.MAX_BLOCK_SIZE8:
        raise ValueError(f"8-bit pools need block_size up to {_native.MAX_BLOCK_SIZE8}, got "
                         f"{k_pool.shape[1]}")
    if not isinstance(kv_scales, (tuple, list)) or len(kv_scales) != 2:
        raise ValueError("kv_scales must be (k_scales, v_scales)")
    want = (k_pool.shape[0], k_pool.shape[2])
    for s in kv_scales:
        if tuple(s.shape) != want or s.dtype != torch.float32 or not s.is_contiguous():
            raise ValueError(f"k_scales and v_scales must be contiguous float32 {want} tensors; "
                             f"got {s.dtype} {tuple(s.shape)}")
    if not (k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError("k_pool and v_pool must be contiguous")
    if k_pool.data_ptr() % 16 or v_pool.data_ptr() % 16:
        raise ValueError("8-bit pools must be 16-byte aligned")


def store_kv(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_tables: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    start_positions: Union[int, torch.Tensor],
    num_tokens: Optional[Union[int, torch.Tensor]] = None,
    check: bool = True,
    errors: Optional[torch.Tensor] = None,
    rope: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
    kv_scales: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
) -> Optional[torch.Tensor]:
    """Write new tokens into their pages, in place.

    k, v: (batch, T, heads, dim), or (T, heads, dim) for one sequence as in
    KVCache._store_kv; block_tables: (batch, max_blocks) or (max_blocks,);
    start_positions: position of each sequence's first new token (int or
    (batch,)); num_tokens: tokens to write per sequence (default T), for
    ragged appends. Token t of sequence b lands at position p = start + t,
    page block_tables[b, p // block_size], slot p % block_size.

    With ``check`` (the default) the call waits for the kernel and raises like
    the reference: ValueError for a negative start, RuntimeError for a
    position past the block table, ValueError for a page id outside the pool.
    Unlike the reference, which stops at the failing chunk, every token that
    can be placed is written. With ``check=False`` nothing waits and the int32
    (3,) error words [negative start, past table, bad page] are returned.

    errors: optional int32 (3,) device tensor that receives the error words
    (cleared by a fill kernel, then set by the append kernel), so that a call
    allocates nothing, e.g. inside a captured HIP graph; without it a
    temporary is allocated per call.

    rope (keyword-only extension): (cos_cache, sin_cache) tables as built by
    precompute_rope_cache, (positions, dim // 2). Each K token is stored
    rotated to its position p (the values rope(k, cos, sin, p) gives, in the
    same kernel that writes the pages), V as given, so attention over the
    cache rotates only its queries. The error words are then 4, the fourth
    set for a position at or past the tables' rows (ValueError with check).

    kv_scales (keyword-only extension): (k_scales, v_scales), float32
    (num_blocks, heads) tensors, for pools of 8-bit codes (torch.float8_e4m3fn
    or torch.int8); k and v are then float32, float16 or bfloat16. A code c of
    page p and head h stands for c * scales[p, h]. The scale is the least power
    of two that holds the largest finite value the call brings to the page and
    head (K after rotation, which is exact here: codes are rounded once), or the
    page's old one where that is larger; where it grew, the page's earlier codes
    are brought to it. A call that writes slot 0 of a page starts the page anew,
    and the slots behind the last one written stand for nothing: a sequence ends
    where it was last written. A page is written for one sequence per call and
    stands once in its row of the table. Values past the largest code saturate;
    NaN stays NaN in float8_e4m3fn and becomes 0 in int8.
    """
    if kv_scales is not None:
        if type(start_positions) is int and k.ndim == 4 and k.shape[0] > 0:
            start_positions = _i32(start_positions, k_pool.device, k.shape[0], "start_positions")
        # the ordinary call, checked and launched in native code
        words = _native.store8_new(k_pool, v_pool, block_tables, k, v, start_positions, num_tokens,
                                   errors, rope, kv_scales)
        if words is not None:
            if not check:
                return words
            _raise_errors(words.tolist())
            return None
    return _store(k_pool, v_pool, block_tables, k, v, start_positions, num_tokens, check, errors,
                  rope, kv_scales)


def _store(k_pool, v_pool, block_tables, k, v, start_positions, num_tokens=None, check=True,
           errors=None, rope=None, kv_scales=None, keep_rest=False) -> Optional[torch.Tensor]:
    """store_kv's general path; keep_rest (8-bit pools): slots that the call does not write
    keep their values, also behind the last one written."""
    if k.ndim == 3:
        k, v = k[None], v[None]
        block_tables = block_tables.reshape(1, -1)
    if k.ndim != 4 or v.shape != k.shape:
        raise ValueError(
            f"k and v must both be (batch, T, heads, dim); got {tuple(k.shape)} and "
            f"{tuple(v.shape)}")
    if k_pool.ndim != 4 or v_pool.shape != k_pool.shape:
        raise ValueError(
            f"k_pool and v_pool must both be (num_blocks, block_size, heads, dim); got "
            f"{tuple(k_pool.shape)} and {tuple(v_pool.shape)}")
    batch, T, heads, dim = k.shape
    num_blocks, block_size = k_pool.shape[:2]
    if k_pool.shape[2:] != (heads, dim):
        raise ValueError(f"pool heads/dim {tuple(k_pool.shape[2:])} do not match k ({heads}, {dim})")
    if kv_scales is not None:
        check_pools8(k_pool, v_pool, kv_scales)
        if k.dtype != v.dtype:
            raise ValueError(f"k/v dtype mismatch: {k.dtype}, {v.dtype}")
        _native.dtype_code(k.dtype)
    elif k.dtype != k_pool.dtype or v.dtype != k_pool.dtype or v_pool.dtype != k_pool.dtype:
        raise ValueError(f"k/v/pool dtype mismatch: {k.dtype}, {v.dtype}, {k_pool.dtype}")
    if block_tables.ndim != 2 or block_tables.shape[0] != batch:
        raise ValueError(f"block_tables must be (batch, max_blocks), got {tuple(block_tables.shape)}")
    if not (k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError("k_pool and v_pool must be contiguous (they are written in place)")
    dev = _native.require_device(k_pool, v_pool, k, v, block_tables)
    starts = _i32(start_positions, dev, batch, "start_positions")
    counts = _i32(T if num_tokens is None else num_tokens, dev, batch, "num_tokens")
    tables = block_tables if block_tables.dtype == torch.int32 else block_tables.to(torch.int32)
    tables = tables.contiguous()
    es = k.element_size()
    if kv_scales is not None:
        _native.require_device(k_pool, *kv_scales)
        _native.require_no_grad(k, v)
        _native.require_no_tangent(k, v, *kv_scales, *(rope or ()))
    elif (dim * es) % 16:
        raise NotImplementedError(
            f"store_kv: head_dim * element size must be a multiple of 16 bytes (dim={dim})")
    vec = 16 // es

    def fit(x: torch.Tensor) -> torch.Tensor:
        if x.stride(-1) != 1 or any(s % vec for s in x.stride()[:3]) or x.data_ptr() % 16:
            return _native.contiguous16(x)
        return x
    k, v = fit(k), fit(v)
    n_err = 3 if rope is None else 4
    if rope is not None:
        cos_cache, sin_cache = rope
        if (cos_cache.shape != sin_cache.shape or cos_cache.ndim != 2
                or cos_cache.shape[1] != dim // 2):
            raise ValueError(
                f"rope cos/sin caches must both be (positions, {dim // 2}); got "
                f"{tuple(cos_cache.shape)} and {tuple(sin_cache.shape)}")
        if dim % 16:
            raise NotImplementedError(
                f"store_kv(rope=...): head_dim must be a multiple of 16, got {dim}")
        _native.require_device(cos_cache, sin_cache)
        cos_cache, sin_cache = map(_native.contiguous16, (cos_cache, sin_cache))
        if kv_scales is not None:
            _native.require_device(k_pool, cos_cache)
            if cos_cache.dtype != sin_cache.dtype:
                raise ValueError(f"cos/sin dtype mismatch: {cos_cache.dtype}, {sin_cache.dtype}")
    if errors is None:
        errors = torch.empty(n_err, dtype=torch.int32, device=dev)
    elif (errors.dtype != torch.int32 or errors.numel() != n_err or errors.device != dev
            or not errors.is_contiguous()):
        raise ValueError(f"errors must be a contiguous int32 tensor of {n_err} entries on "
                         "the pools' device")
    if kv_scales is not None:
        if k.numel() == 0:
            errors.zero_()  # (no kernel runs, which would write them)
        _native.kv_append8(k, v, k_pool, v_pool, *kv_scales, tables, starts, counts, errors,
                           None if rope is None else (cos_cache, sin_cache), keep_rest)
    elif not _native.kv_append_clear(k, v, k_pool, v_pool, tables, starts, counts, errors,
                                   None if rope is None else (cos_cache, sin_cache)):
        errors.zero_()
        if rope is None:
            _native.kv_append(k, v, k_pool, v_pool, tables, starts, counts, errors,
                              k.stride()[:3], v.stride()[:3], batch, T, heads, dim, num_blocks,
                              block_size, tables.shape[1])
        else:
            _native.kv_append_rope(k, v, k_pool, v_pool, tables, starts, counts, errors,
                                   k.stride()[:3], v.stride()[:3], batch, T, heads, dim,
                                   num_blocks, block_size, tables.shape[1], cos_cache, sin_cache)
    if not check:
        return errors
    _raise_errors(errors.tolist())
    return None


def load_kv(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_tables: torch.Tensor,
    start_positions: Union[int, torch.Tensor],
    num_tokens: Union[int, torch.Tensor],
    *,
    kv_scales: Tuple[torch.Tensor, torch.Tensor],
    max_tokens: Optional[int] = None,
    dtype: torch.dtype = torch.bfloat16,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Values of cached tokens of 8-bit pools: (k, v), each (batch, max_tokens,
    heads, dim) of ``dtype`` (bfloat16 and float32 hold every value that store_kv
    makes exactly; values past float16's largest become infinite there).

    block_tables: (batch, max_blocks); row t of sequence b is the token at
    start_positions[b] + t, for t < num_tokens[b]; the rows behind, and rows
    that have no page, are zeros. max_tokens defaults to num_tokens where that
    is an int and must be given otherwise (a tensor's largest entry is only
    known on the device). The pools and kv_scales are those of store_kv.
    """
    if max_tokens is not None and dtype in _native.DTYPE_CODES:
        # the ordinary call, checked and launched in native code
        out = _native.load8_new(k_pool, v_pool, block_tables, start_positions, num_tokens,
                                max_tokens, kv_scales, _native.DTYPE_CODES[dtype])
        if out is not None:
            return out
    if k_pool.ndim != 4 or v_pool.shape != k_pool.shape:
        raise ValueError(
            f"k_pool and v_pool must both be (num_blocks, block_size, heads, dim); got "
            f"{tuple(k_pool.shape)} and {tuple(v_pool.shape)}")
    check_pools8(k_pool, v_pool, kv_scales)
    _native.dtype_code(dtype)
    if block_tables.ndim != 2:
        raise ValueError(f"block_tables must be (batch, max_blocks), got {tuple(block_tables.shape)}")
    if max_tokens is None:
        if not isinstance(num_tokens, int):
            raise ValueError("max_tokens must be given where num_tokens is not an int")
        max_tokens = num_tokens
    if max_tokens < 0:
        raise ValueError(f"max_tokens must not be negative, got {max_tokens}")
    dev = _native.require_device(k_pool, v_pool, block_tables, *kv_scales)
    _native.require_no_tangent(*kv_scales)
    batch = block_tables.shape[0]
    starts = _i32(start_positions, dev, batch, "start_positions")
    counts = _i32(num_tokens, dev, batch, "num_tokens")
    tables = block_tables if block_tables.dtype == torch.int32 else block_tables.to(torch.int32)
    shape = (batch, max_tokens) + tuple(k_pool.shape[2:])
    k, v = (torch.empty(shape, dtype=dtype, device=dev) for _ in range(2))
    _native.kv_load8(k_pool, v_pool, *kv_scales, tables.contiguous(), starts, counts, k, v)
    return k, v


def set_block_data(k_pool: torch.Tensor, v_pool: torch.Tensor, block_id: int, k: torch.Tensor,
                   v: torch.Tensor, start_pos: int = 0, length: Optional[int] = None, *,
                   kv_scales: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> None:
    """Write k, v (length, heads, dim) into page block_id from slot start_pos.

    Same arguments and errors as BlockAllocator.set_block_data
    (block_allocator.py:299-331, without the allocator's copy-on-write).

    kv_scales as in store_kv, but that the slots which are not written keep their
    values, before and behind the written ones: the page's scale stays or grows, and
    where it grew their codes are rounded to it once. Writing all slots starts the page
    anew. A page that holds nothing yet has to have the scale 0 (a new pool's, and what
    BlockAllocator gives a block it hands out).
    """
    num_blocks, block_size = k_pool.shape[:2]
    if not 0 <= int(block_id) < num_blocks:
        raise ValueError(f"Invalid block_id {block_id} (pool has {num_blocks} blocks)")
    if length is None:
        length = k.shape[0]
    if start_pos < 0 or start_pos + length > block_size or length > k.shape[0]:
        raise ValueError(
            f"slots [{start_pos}, {start_pos + length}) do not fit a block of {block_size}")
    table = torch.full((1, 1), int(block_id), dtype=torch.int32, device=k_pool.device)
    _store(k_pool, v_pool, table, k[:length][None], v[:length][None], start_pos, check=False,
           kv_scales=kv_scales, keep_rest=kv_scales is not None)
