"""What rounding the weights of 16-bit attention over 8-bit pages leaves in its outputs."""

import numpy as np
import pytest
import torch

from mlx_primitives.cache import paged_attention
from test_gpu_cache8 import CODES, DTYPES, make, random_cache, spread_tables
from test_gpu_cache8_paths import i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D,bs,Sq,H,H_kv", [(64, 16, 1, 4, 2), (128, 5, 1, 4, 4), (256, 16, 1, 2, 1),
                                            (128, 16, 3, 16, 2), (64, 24, 40, 2, 2)])
def test_one_token_is_its_value(device, code, dt, D, bs, Sq, H, H_kv):
    # A row that sees one token returns its value: numerator and denominator carry the same weight,
    # rounded or not, up to float32 (relative errors of a few 2^-24, for int8 of 255 times that),
    # and the value, a code times a power of two, is a number of the type or within 2^-20 of one.
    rng = np.random.default_rng(D + Sq)
    B = 30
    tables, nb = spread_tables(rng, [1] * B, bs)
    kp, vp, scales = random_cache(rng, nb, bs, H_kv, D, code, device)
    q = make(rng, (B, Sq, H, D), DTYPES[dt]).to(device)
    out = paged_attention(q, kp, vp, torch.from_numpy(tables).to(device), i32([1] * B, device),
                          block_size=bs, enable_gqa=True, kv_scales=scales)
    pages = torch.from_numpy(tables[:, 0]).long().to(device)
    v = (vp.float()[pages, 0] * scales[1][pages][:, :, None]).repeat_interleave(H // H_kv, dim=1)
    want = v[:, None].expand(-1, Sq, -1, -1)
    if dt == "f32":
        assert ((out - want).abs() <= 2.0 ** -21 * want.abs()).all()
    else:
        assert torch.equal(out, want.to(out.dtype))
