"""What attention over 8-bit pages asks of the host before it launches: workspace that follows
what the rows can see, not the width of the block tables.
"""

import os
import random

import pytest

from mlx_primitives import _native

MOST = 256 << 20  # bytes of a call's workspace


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_native.library_path()):
        pytest.skip("libmpx_attn.so not built")
    return _native.load()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("width", [256, 2048, 8192, 1 << 16])
def test_prompts_in_wide_tables_need_none(lib, width, dtype):
    # Causal rows from position 0 on see Sq tokens at most.
    need = lib.mpx_paged_attend8_call_workspace_bytes
    assert need(4, 4096, 32, 8, 128, 16, width, dtype, 1, 0) == 0
    assert need(1, 32768, 64, 8, 128, 16, width, dtype, 1, 0) == 0


def test_turns_in_wide_tables(lib):
    # 65 queries behind a prefix: 64 partitions at most, however wide the table (one has the
    # sums of 2 x 65 x 32 rows, 130 floats each).
    need = lib.mpx_paged_attend8_call_workspace_bytes
    narrow = need(2, 65, 32, 8, 128, 16, 259, 2, 1, 1)
    assert narrow > 0
    for width in (512, 2048, 8192, 1 << 16, 1 << 24):
        assert narrow <= need(2, 65, 32, 8, 128, 16, width, 2, 1, 1) <= 64 * 4160 * 130 * 4


def test_workspaces_are_bounded(lib):
    rng = random.Random(5)
    call, most = lib.mpx_paged_attend8_call_workspace_bytes, lib.mpx_paged_attend8_workspace_bytes
    for _ in range(4000):
        H_kv = rng.choice([1, 2, 4, 8, 32])
        shape = (int(2 ** rng.uniform(0, 13)), rng.choice([1, 1, 2, 5, 65, 300, 4096, 65536]),
                 H_kv * rng.choice([1, 4, 8]), H_kv, rng.choice([16, 64, 80, 128, 256]),
                 rng.choice([1, 7, 16, 64]))
        shape += (int(2 ** rng.uniform(0, 29)) // shape[5], rng.choice([0, 1, 2]))
        enough = most(*shape)
        for causal in (0, 1):
            for positions in (0, 1):
                need = call(*shape, causal, positions)
                assert need <= enough <= MOST, (shape, causal, positions)


def test_sizes_that_are_none(lib):
    call = lib.mpx_paged_attend8_call_workspace_bytes
    assert call(0, 1, 4, 4, 64, 16, 8, 2, 1, 0) == 0
    assert call(1, 1, 5, 4, 64, 16, 8, 2, 1, 0) == 0
    # sizes that the launch refuses ask for nothing first
    assert call(65536, 1, 4, 4, 64, 16, 1 << 16, 2, 1, 0) == 0
    assert call(1, 1 << 26, 8, 1, 64, 16, 1 << 16, 0, 0, 0) == 0
