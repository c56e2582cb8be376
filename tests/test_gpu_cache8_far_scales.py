"""Attention over 8-bit pages whose V scales are far apart, as an outlier among the values makes
them: pages with small scales keep their bits where the rows look at them, wherever the large
ones stand.
"""

import math

import numpy as np
import pytest
import torch

from mlx_primitives.cache import paged_attention
from oracle import cache8 as o8
from test_gpu_cache8 import CODES, DTYPES, held, spread_tables
from test_gpu_cache8_paths import i32, wide

pytestmark = pytest.mark.gpu


def cache(rng, nb, bs, H, D, code, spread):
    """Pages whose V scales and scores go together in several ways: a scale of 2^s (s up to
    `spread`) comes with scores that are lower by none, all or twice of s log 2. Returns pools,
    scales and the direction that queries have to have."""
    u = rng.standard_normal((H, D))
    u /= np.sqrt((u * u).sum(-1, keepdims=True))
    s = rng.integers(0, 4, (nb, H)) * (spread / 3)
    s = np.round(s) * (rng.random((nb, H)) < 0.6)
    level = -s * math.log(2) * rng.choice([1.0, 2.0, 2.0, 0.0], (nb, H))
    k = level[:, None, :, None] * u + 0.1 * rng.standard_normal((nb, bs, H, D))
    v = rng.standard_normal((nb, bs, H, D)) * 2.0 ** s[:, None, :, None]
    out = []
    for x in (k, v):
        need = np.vectorize(lambda a: o8.need(a, code))(np.abs(x).max(axis=(1, 3)))
        c = o8.encode(x / need[:, None, :, None], code)
        out.append((torch.from_numpy(c.astype(np.float32)).to(CODES[code]), need))
    return out, u


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("spread", [45, 180])
@pytest.mark.parametrize("B,Sq,H,H_kv,D,bs,n,width", [
    (2, 1, 4, 2, 64, 16, 300, 0), (2, 9, 4, 2, 128, 16, 290, 0), (1, 2, 4, 4, 64, 5, 200, 0),
    (2, 1, 4, 1, 128, 16, 3000, 0), (1, 1, 2, 2, 256, 24, 700, 0), (64, 1, 4, 4, 64, 16, 600, 16384),
    (2, 20, 4, 2, 64, 16, 300, 0)])
def test_far_scales(device, code, dt, spread, B, Sq, H, H_kv, D, bs, n, width):
    # Scores and weights: bounds as in test_gpu_cache8.check_attend. What is lost beyond them is
    # under 2^-38 (16-bit queries; float32 2^-80) of the row's largest weight times scale, for each
    # token and the largest code; for int8 the sums that 128 is taken off of again round by 2^-24
    # of 255 of that.
    if dt == "f16" and Sq * H // H_kv > 32:
        pytest.skip("float16 rows in the many-rows form take V's scales within float16's range")
    if dt == "f16" and spread > 100:
        spread = 100  # (what is large and seen passes float16's largest number anyway)
    rng = np.random.default_rng(n + Sq + spread)
    lens = [n] + [int(x) for x in rng.integers(1, 40, B - 1)]
    tables, nb = spread_tables(rng, lens, bs)
    if width:
        tables = wide(tables, -(-width // bs))
    ((kp, ks), (vp, vs)), u = cache(rng, nb, bs, H_kv, D, code, spread)
    g = H // H_kv
    q = math.sqrt(D) * u.repeat(g, 0) + 0.05 * rng.standard_normal((B, Sq, H, D))
    q = torch.from_numpy(q.astype(np.float32)).to(DTYPES[dt])
    first = [m - Sq for m in lens]
    out = paged_attention(
        q.to(device), kp.to(device), vp.to(device), torch.from_numpy(tables).to(device),
        i32(lens, device), block_size=bs, enable_gqa=True, query_start=i32(first, device),
        kv_scales=tuple(torch.from_numpy(s.astype(np.float32)).to(device) for s in (ks, vs)))
    got, qn = out.double().cpu().numpy(), q.double().numpy()
    kc, vc = held(kp) * ks[:, None, :, None], held(vp) * vs[:, None, :, None]
    r = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dt]
    for b, m in enumerate(lens):
        pages = tables[b, :-(-m // bs)]
        k, v = (x[pages].reshape(-1, H_kv, D)[:m] for x in (kc, vc))
        t = np.arange(m)
        scale = vs[pages].repeat(bs, 0)[:m]
        kscale = ks[pages].repeat(bs, 0)[:m]
        for i in range(Sq):
            see = t <= first[b] + i
            for h in range(H):
                if not see.any():
                    assert np.isnan(got[b, i, h]).all()
                    continue
                x = k[see, h // g] @ qn[b, i, h] / math.sqrt(D)
                w = np.exp(x - x.max())
                w /= w.sum()
                ref, A = w @ v[see, h // g], w @ np.abs(v[see, h // g])
                E = np.abs(k[see, h // g]) @ np.abs(qn[b, i, h])
                if code == "int8" and dt != "f32":
                    E = E + 128 * kscale[see, h // g] * np.abs(qn[b, i, h]).sum()
                E = E.max() / math.sqrt(D)
                err = 2 * ((D + 8) * 2.0 ** -24 * E + 2.0 ** -22 * (1 + E) + m * 2.0 ** -24)
                top = (w * scale[see, h // g]).max()
                lost = m * (2.0 ** -80 if dt == "f32" else 2.0 ** -38) * 448 * top
                if code == "int8" and dt != "f32":
                    lost += m * 2.0 ** -24 * 255 * m * top
                bound = (min(err, 2.0) + r) * A + r * np.abs(ref) + lost + 2.0 ** -24 * (dt == "f16")
                # (float16: what its error may carry past the largest number may be infinite)
                ok = np.abs(ref) + bound < (65504 if dt == "f16" else np.inf)
                with np.errstate(invalid="ignore"):
                    off = np.abs(got[b, i, h] - ref)
                assert (off <= bound * (1 + 2.0 ** -7))[ok].all(), (
                    b, i, h, (off / bound)[ok].max(), ref[ok][:4], bound[ok][:4])
