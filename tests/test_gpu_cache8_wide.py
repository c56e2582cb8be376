"""The 8-bit cache at the far ends of its sizes: attention in block tables that are far wider than
what is in them (static tables of captured programs, ragged batches), partitions, rows and
appends of any length. Oracle and bounds are those of test_gpu_cache8.
"""

import math

import numpy as np
import pytest
import torch

from mlx_primitives.cache import load_kv, paged_attention, store_kv
from test_gpu_cache8 import CODES, DTYPES, check_attend, make, random_cache, spread_tables
from test_gpu_cache8_paths import i32, wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("width", [40000, 1 << 20])
@pytest.mark.parametrize("D,bs,Sq,H,H_kv,form", [
    (128, 16, 1, 8, 2, "decode"), (64, 24, 1, 4, 4, "decode"), (80, 5, 3, 4, 2, "behind"),
    (128, 16, 70, 4, 2, "behind"), (64, 7, 45, 4, 2, "behind"), (256, 16, 37, 2, 1, "behind"),
    (128, 16, 150, 2, 1, "prompt"), (64, 16, 9, 4, 2, "prompt"), (128, 16, 70, 4, 2, "open")])
def test_wide_tables(device, dt, width, D, bs, Sq, H, H_kv, form):
    rng = np.random.default_rng(D + Sq)
    lens = [2900, 257, Sq, 0, 1300]
    first = [n - Sq for n in lens] if form == "behind" else None
    tables, nb = spread_tables(rng, lens, bs)
    tables[0, 2] = nb
    tables = wide(tables, -(-width // bs))
    code = "int8" if bs == 16 else "e4m3"
    kp, vp, scales = random_cache(rng, nb, bs, H_kv, D, code, device)
    q = make(rng, (len(lens), Sq, H, D), DTYPES[dt]).to(device)
    causal = form != "open"
    out = paged_attention(q, kp, vp, torch.from_numpy(tables).to(device), i32(lens, device),
                          block_size=bs, causal=causal, enable_gqa=True, kv_scales=scales,
                          query_start=None if first is None else i32(first, device))
    check_attend(out, q, kp, vp, scales, tables, lens, 1 / math.sqrt(D), causal, None, first, dt)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("code", CODES)
def test_waves_that_take_heads_in_wide_tables(device, dt, code):
    # More than 64 partitions of 512 tokens in the tables: two sequences spread over all of them.
    rng = np.random.default_rng(12)
    B, H, H_kv, D, bs = 16, 8, 4, 64, 16
    lens = [int(x) for x in rng.integers(0, 40, B)]
    lens[3], lens[15] = 33001, 40000
    tables, nb = spread_tables(rng, lens, bs)
    tables = wide(tables, (1 << 17) // bs)
    kp, vp, scales = random_cache(rng, nb, bs, H_kv, D, code, device)
    q = make(rng, (B, 1, H, D), DTYPES[dt]).to(device)
    out = paged_attention(q, kp, vp, torch.from_numpy(tables).to(device), i32(lens, device),
                          block_size=bs, enable_gqa=True, kv_scales=scales)
    check_attend(out, q, kp, vp, scales, tables, lens, 1 / math.sqrt(D), True, None, None, dt)


@pytest.mark.parametrize("bs", [16, 24, 7, 1, 32768])
@pytest.mark.parametrize("Sq,H", [(2048, 32), (1, 1), (20, 1)])
def test_partitions_of_more_than_65536_tokens(device, bs, Sq, H):
    # One partition holds all 70001 tokens of many rows (512 row blocks fill the chip); few rows
    # spread over it. A row against the softmax of the same values in 64 bits: the scores are off
    # by (D + 8) 2^-24 of sums of at most 4 D terms' sizes, their weights and sums by that, by
    # 2^-22 of the score and by n 2^-24; bf16 rounds weights and output by 2^-8 each.
    rng = np.random.default_rng(bs)
    n, D = 70001, 64
    tables, nb = spread_tables(rng, [n], bs)
    kp = torch.randint(-127, 128, (nb, bs, 1, D), dtype=torch.int8, device=device,
                       generator=torch.Generator(device=device).manual_seed(bs))
    vp = kp.flip(0).contiguous()
    scales = tuple(torch.full((nb, 1), 2.0 ** -6, device=device) for _ in range(2))
    q = make(rng, (1, Sq, H, D), torch.bfloat16).to(device)
    first = n - Sq
    out = paged_attention(q, kp, vp, torch.from_numpy(tables).to(device), i32([n], device),
                          block_size=bs, enable_gqa=True, kv_scales=scales,
                          query_start=i32([first], device))
    pages = torch.from_numpy(tables[0, :-(-n // bs)]).long().to(device)
    k, v = (p[pages].flatten(0, 1)[:n, 0].double() * 2.0 ** -6 for p in (kp, vp))
    for i in sorted({0, Sq // 2, Sq - 1}):
        rows = q[0, i].double()
        x = (rows @ k.t() / 8).masked_fill(torch.arange(n, device=device) > first + i, -math.inf)
        w = torch.softmax(x, -1)
        ref, size = w @ v, w @ v.abs()
        E = (rows.abs() @ (k.abs() + 2.0).t() / 8).max()  # (int8 codes as k + 128: 2 in units)
        off = 2 * ((D + 8) * 2.0 ** -24 * E + 2.0 ** -22 * (1 + E) + n * 2.0 ** -24) + 2.0 ** -8
        bound = off * size + 2.0 ** -8 * ref.abs() + n * 2.0 ** -24 * 4
        assert ((out[0, i].double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("dt,Sq,G", [("f32", 131073, 8), ("bf16", 65536, 8), ("f16", 3, 7)])
@pytest.mark.parametrize("behind", [False, True])
def test_rows_in_any_number(device, dt, Sq, G, behind):
    # More than 65535 blocks of 16 float32 rows; a table of 2^20 tokens. All rows against the
    # formula in 64 bits, bounds as in check_attend (values of unit scale).
    rng = np.random.default_rng(Sq)
    n, D, bs = 75, 16, 16
    tables, nb = spread_tables(rng, [n], bs)
    tables = wide(tables, (1 << 20) // bs)
    kp, vp, _ = random_cache(rng, nb, bs, 1, D, "e4m3", device)
    scales = tuple(torch.full((nb, 1), 2.0 ** -8, device=device) for _ in range(2))
    q = torch.randn((1, Sq, G, D), device=device,
                    generator=torch.Generator(device=device).manual_seed(Sq)).to(DTYPES[dt])
    first = 30 if behind else 0
    out = paged_attention(q, kp, vp, torch.from_numpy(tables).to(device), i32([n], device),
                          enable_gqa=True, kv_scales=scales,
                          query_start=i32([first], device) if behind else None)
    pages = torch.from_numpy(tables[0, :-(-n // bs)]).long().to(device)
    k, v = (p[pages].flatten(0, 1)[:n, 0].double() * 2.0 ** -8 for p in
            (kp.float(), vp.float()))
    u = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dt]
    for lo in range(0, Sq, 16384):
        rows = q[0, lo:lo + 16384].double()
        at = first + lo + torch.arange(len(rows), device=device)
        x = (rows @ k.t() / 4).masked_fill(
            torch.arange(n, device=device) > at[:, None, None], -math.inf)
        w = torch.softmax(x, -1)
        ref, size = w @ v, w @ v.abs()
        E = (rows.abs() @ k.abs().t() / 4).amax(-1, keepdim=True)
        off = 2 * ((D + 8) * 2.0 ** -24 * E + 2.0 ** -22 * (1 + E) + n * 2.0 ** -24)
        bound = (off + u) * size + u * ref.abs() + n * 2.0 ** -38 * 448 * 2.0 ** -8 + 2.0 ** -24
        assert ((out[0, lo:lo + 16384].double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("bs,T", [(1, 70001), (16, 16 * 65600 + 5), (16, 1)])
def test_appends_of_any_length(device, bs, T):
    # More pages than 65535 in one call, and the pages of many sequences: what comes back is what
    # went in, values that codes hold exactly.
    H, D, B = 1, 16, 3
    counts = [T, 1, max(1, T // 3)]
    starts = [0, bs // 2, 3]
    pages = [-(-(s + n) // bs) for s, n in zip(starts, counts)]
    nb = sum(pages)
    gen = torch.Generator(device=device).manual_seed(T)
    perm = torch.randperm(nb, device=device, generator=gen).int()
    tables = torch.full((B, max(pages)), -1, dtype=torch.int32, device=device)
    at = 0
    for b, n in enumerate(pages):
        tables[b, :n] = perm[at:at + n]
        at += n
    k, v = (torch.randint(-8, 9, (B, T, H, D), device=device, generator=gen).float() for _ in "kv")
    for x in (k, v):
        x[..., 0] = 127.0  # (the scale of every page is 1)
    kp = torch.zeros((nb, bs, H, D), dtype=torch.int8, device=device)
    vp = torch.zeros_like(kp)
    scales = tuple(torch.zeros((nb, H), device=device) for _ in range(2))
    store_kv(kp, vp, tables, k, v, i32(starts, device), i32(counts, device), kv_scales=scales)
    got = load_kv(kp, vp, tables, i32(starts, device), i32(counts, device), max_tokens=T,
                  kv_scales=scales, dtype=torch.float32)
    for x, y in zip(got, (k, v)):
        for b, n in enumerate(counts):
            assert torch.equal(x[b, :n], y[b, :n]) and not x[b, n:].any()
    with pytest.raises(RuntimeError, match="Block index"):  # one token past the tables
        store_kv(kp, vp, tables[:1], k[:1, -1:], v[:1, -1:], tables.shape[1] * bs, kv_scales=scales)
