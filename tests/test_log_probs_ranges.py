"""Ranges of log_probs for rows that do not begin on 16 bytes.  A range of a few rows is a chunk of 256 x 32 values; a row
that begins late has up to 16 bytes more, and where they make one more chunk, the call needs one more range, not
half of them with two chunks and the others with none."""
from __future__ import annotations

import pytest

from weft_amd import ggml as G

CHUNK = 256 * 32


@pytest.mark.parametrize("t,late", [(G.F32, 3), (G.F16, 7)])
@pytest.mark.parametrize("v,rows", [(131072, 3), (131071, 3), (65536, 1), (262143, 8), (524288, 10)])
@pytest.mark.parametrize("top", [0, 20, 64])
def test_a_range_a_chunk(v, rows, top, t, late):
    chunks = -(-(v + late) // CHUNK)
    assert chunks <= 64 + 1 and chunks * rows <= 1024
    size = G.log_probs_work_size(G.tensor(t, (v, rows)), top)
    # past 64 ranges two chunks a range; an aligned row of 64 chunks keeps its 64
    assert size == rows * min(chunks, 64) * (16 + 8 * top)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [G.F32, G.F16])
@pytest.mark.parametrize("v,rows,offset", [(131071, 3, 0), (131072, 3, 1), (65536, 2, 1), (262143, 8, 0), (524288, 2, 1)])
def test_rows_off_their_alignment(hip, v, rows, offset, t):
    from tests.test_gpu_log_probs import asked, check, logits

    x = logits(rows, v, t)
    x[0] = x[0].round()
    x[1, -9:] += 20
    for top in (0, 20, 64):
        check(hip, x, asked(rows, v, 2), top, offset=offset)
