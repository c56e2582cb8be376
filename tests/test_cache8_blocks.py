"""Writes of single slots into 8-bit blocks (set_block_data): the slots that a write
leaves out keep their values, and a block that is handed out again starts empty.
"""

import numpy as np
import pytest
import torch

from mlx_primitives.cache import BlockAllocator, BlockConfig, load_kv, set_block_data
from oracle import cache8 as o8

CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def held(pool):
    return (pool if pool.dtype == torch.int8 else pool.float()).double().cpu().numpy()


def write64(c, scale, first, x, code):
    """x (n, H, D) into slots first.. of one block: codes c (bs, H, D) and scale (H,), in place."""
    n = len(x)
    for h in range(c.shape[1]):
        s = o8.need(float(np.abs(x[:, h]).max()), code)
        if n < len(c):
            s = max(s, scale[h])
        c[:, h] = o8.encode(c[:, h] * (scale[h] / s), code)
        c[first:first + n, h] = o8.encode(x[:, h] / s, code)
        scale[h] = s


@pytest.mark.parametrize("dtype", CODES.values())
def test_blocks_are_handed_out_empty(dtype):
    a = BlockAllocator(BlockConfig(16, 3, 32, dtype), 6, device="cpu")
    for s in a.get_scales():
        s.fill_(7.0)
    ids = a.allocate(2)
    for s in a.get_scales():
        assert not s[ids].any() and (s[[i for i in range(6) if i not in ids]] == 7.0).all()
        s.fill_(5.0)
    a.allocate(1)
    a.free([ids[0]])
    ids = a.allocate(3)  # (ids that are no run)
    assert max(ids) - min(ids) > 2
    for s in a.get_scales():
        assert not s[ids].any() and (s == 5.0).sum() == 2 * 3
    assert a.allocate(0) == []
    # a private copy has its source's scales, not empty ones
    for s in a.get_scales():
        s[ids[0]] = 3.0
    a.increment_ref(ids[0])
    new = a.copy_on_write(ids[0])
    assert new != ids[0] and all((s[new] == 3.0).all() for s in a.get_scales())
    # who only appends does without
    a = BlockAllocator(BlockConfig(16, 3, 32, dtype), 2, device="cpu", clear_scales=False)
    a.get_scales()[0].fill_(7.0)
    assert (a.get_scales()[0][a.allocate(2)] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [50.0, 1.0, 0.02])
@pytest.mark.parametrize("bs,D,first,n", [(16, 64, 0, 5), (16, 64, 4, 6), (16, 64, 10, 6),
                                          (16, 64, 0, 16), (24, 80, 0, 1), (24, 80, 23, 1),
                                          (40, 256, 7, 21), (1, 16, 0, 1)])
def test_other_slots_keep_their_values(device, code, dt, size, bs, D, first, n):
    rng = np.random.default_rng(bs + first)
    H, nb, page = 3, 3, 1
    pools, scales, ref = [], [], []
    for _ in range(2):
        x = rng.standard_normal((nb, bs, H, D))
        s = np.array([[o8.need(np.abs(x[p, :, h]).max(), code) for h in range(H)]
                      for p in range(nb)])
        c = o8.encode(x / s[:, None, :, None], code)
        pools.append(torch.from_numpy(c.astype(np.float32)).to(CODES[code]).to(device))
        scales.append(torch.from_numpy(s.astype(np.float32)).to(device))
        ref.append((c, s))
    new = [torch.from_numpy((rng.standard_normal((n, H, D)) * size).astype(np.float32)).to(dt)
           for _ in range(2)]
    for (c, s), x in zip(ref, new):
        write64(c[page], s[page], first, x.double().numpy(), code)
    set_block_data(*pools, page, *(x.to(device) for x in new), first, n, kv_scales=tuple(scales))
    for pool, scale, (c, s) in zip(pools, scales, ref):
        np.testing.assert_array_equal(scale.double().cpu().numpy(), s)
        np.testing.assert_array_equal(held(pool), c)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
def test_a_block_filled_in_pieces(device, code):
    # Written back to front, in the middle and again, after an owner whose values were louder.
    rng = np.random.default_rng(3)
    bs, H, D = 16, 2, 64
    a = BlockAllocator(BlockConfig(bs, H, D, CODES[code]), 2, device=device)

    def rows(n, size):
        return torch.from_numpy((rng.standard_normal((n, H, D)) * size).astype(np.float32))
    page, = a.allocate(1)
    a.set_block_data(page, *(rows(bs, 1e6).to(device) for _ in range(2)))
    a.free([page])
    assert a.allocate(1) == [page]
    refs = [(np.zeros((bs, H, D)), np.zeros(H)) for _ in range(2)]
    for first, n, size in ((12, 4, 0.1), (0, 3, 1.0), (5, 2, 30.0), (1, 2, 0.01), (3, 9, 3.0)):
        new = [rows(n, size) for _ in range(2)]
        for (c, s), x in zip(refs, new):
            write64(c, s, first, x.double().numpy(), code)
        assert a.set_block_data(page, *(x.to(device) for x in new), first, n) == page
        for pool, scale, (c, s) in zip(a.get_pools(), a.get_scales(), refs):
            np.testing.assert_array_equal(scale[page].double().cpu().numpy(), s)
            np.testing.assert_array_equal(held(pool[page]), c)
    table = torch.tensor([[page]], dtype=torch.int32, device=device)
    got = load_kv(*a.get_pools(), table, 0, bs, kv_scales=a.get_scales(), dtype=torch.float32)
    for x, (c, s) in zip(got, refs):
        np.testing.assert_array_equal(x[0].double().cpu().numpy(), c * s[:, None])
