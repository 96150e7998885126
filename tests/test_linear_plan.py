"""Which kernel an 8-bit product takes, by the host-only query (no GPU)."""

from __future__ import annotations

import random
import re

import pytest

from fast_mimi_amd import _native as nat

pytestmark = pytest.mark.skipif(not nat.LIBRARY_PATH.is_file(), reason="library not built")


@pytest.mark.parametrize("rows,k,n,plan", [
    (1, 4096, 6144, "linear_rows_kernel<1>"), (32, 1008, 1000, "linear_rows_kernel<2>"),
    (32, 8192, 2048, "linear_tile_kernel<64, 64> splits=8"), (500, 4096, 6144, "linear_tile_kernel<64, 128> splits=1"),
    (1001, 2048, 8192, "linear_tile_kernel<128, 128> splits=1"), (8192, 8192, 8192, "linear_tile_kernel<256, 256> splits=1"),
    # Few outputs, or few rows beside them: no tile that is mostly empty.
    (65536, 1024, 64, "linear_tile_kernel<64, 64> splits=1"), (65536, 4096, 16, "linear_tile_kernel<64, 64> splits=1"),
    (65536, 1024, 128, "linear_tile_kernel<128, 128> splits=1"), (20000, 1024, 64, "linear_tile_kernel<64, 64> splits=1"),
    (64, 2048, 65536, "linear_tile_kernel<64, 128> splits=1"), (129, 2048, 65536, "linear_tile_kernel<256, 256> splits=1"),
])
def test_plans(rows, k, n, plan):
    assert nat.linear_fp8_plan(rows, k, n) == plan


def test_large_tiles_are_more_than_half_full():
    rng = random.Random(1)
    for _ in range(3000):
        rows, k, n = (max(1, int(2 ** rng.uniform(0, 17))) for _ in range(3))
        found = re.fullmatch(r"linear_tile_kernel<(\d+), (\d+)> splits=(\d+)", nat.linear_fp8_plan(rows, 16 * k, n))
        if not found:
            assert rows <= 32
            continue
        bm, bn, splits = map(int, found.groups())
        padded = -(-rows // bm) * bm * (-(-n // bn) * bn)
        assert (bm, bn) == (64, 64) or 2 * rows * n > padded, (rows, k, n)
        need = nat.library().fm_linear_fp8_workspace_bytes(rows, 16 * k, n)
        assert need == (4 * splits * rows * n if splits > 1 else 0)


def test_refusals():
    plan, buf = nat.library().fm_linear_fp8_plan, b" " * 80
    for args in ((0, 16, 16, buf, 80), (1, 0, 16, buf, 80), (1, 16, 0, buf, 80), (1, 16, 16, None, 80), (1, 16, 16, buf, 0)):
        assert plan(*args) == 1000
