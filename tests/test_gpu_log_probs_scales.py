"""log_probs of logits near the largest 32-bit number, at scales that make ordinary ones of them (GPU): differences
that no 32-bit number holds before the scale is on them, and sums of such differences.  The bounds are those of
tests/test_gpu_log_probs.py: halves of both logits and twice the scale round as the whole ones do."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_log_probs import asked, check
from weft_amd import ggml as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("v", [5, 700, 9001, 40000])
@pytest.mark.parametrize("scale", [1e-38, 1.5e-38, 4e-38, 1e-37])
def test_logits_near_the_largest_number(hip, v, scale):
    rng = np.random.default_rng(v)
    x = (rng.uniform(-3.3e38, 3.3e38, (3, v))).astype(np.float32)
    x[1] = 1e38 * np.round(rng.uniform(-3, 3, v))
    x[2] = np.where(rng.random(v) < 0.5, np.finfo(np.float32).min, np.finfo(np.float32).max)
    check(hip, x, asked(3, v, 3), min(v, 20), scale)


@pytest.mark.parametrize("v", [700, 40000])
def test_barred_beside_them(hip, v):
    x = np.random.default_rng(v).uniform(-3.3e38, 3.3e38, (4, v)).astype(np.float32)
    x[0, ::3] = -np.inf
    x[1, 5:] = -np.inf
    x[2, v // 2] = np.nan
    x[3, v // 3] = np.inf
    check(hip, x, asked(4, v, 3), 9, 1e-38)


def test_the_lowest_and_largest_at_ordinary_scales(hip):
    """Differences past the largest number whose log probabilities (up to 1.7e38) are not."""
    x = np.full((3, 300), np.finfo(np.float32).min)
    x[0, 7] = np.finfo(np.float32).max
    x[1, 7], x[1, 8] = 1e38, 1e38
    x[2] = 3
    for scale in (0.25, 1e-3):
        check(hip, x, np.tile(np.int32([3, 7, 8]), (3, 1)), 5, scale)
