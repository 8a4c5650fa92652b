"""add_rms_norm of rows far longer than its registers hold (GPU), to the bounds of its
other tests: a lane then sums K / 1024 squares one after the other."""
from __future__ import annotations

import pytest

from tests.test_gpu_add_rms_norm import check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dst,k", [("f32", (1 << 20) + 5), ("f32", 1 << 22), ("f16", (1 << 21) + 3), ("q8_0", 1 << 20),
                                   ("q8_1", (1 << 20) + 32), ("q8_k", 1 << 22)])
@pytest.mark.parametrize("total", ["own", None])
def test_long_rows(hip, dst, k, total):
    raw, y = run(hip, 2, k, dst, total=total, seed=k % 1000)
    check(raw, y, dst, k)
