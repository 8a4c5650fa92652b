"""The most rows a call of the attention may have (GPU): 2^31 - 1 queries of one head,
which share memory, as their outputs do.  The table has one key, so every output is its
value."""
from __future__ import annotations

import numpy as np
import pytest

from tests._layer import encode
from weft_amd import ggml as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [(1 << 31) - 1, (1 << 31) - 127])
def test_one_key(hip, tokens):
    d = 64
    k, v = np.random.default_rng(1).standard_normal((2, 1, d)).astype(np.float32)
    dev = [hip.to_dev(encode("f16", x)) for x in (k, v)]
    pools = [G.tensor(G.F16, (d, 1, 1, 1), x.ptr) for x in dev]
    ints = [hip.to_dev(np.array(x, np.int32)) for x in ([[0]], [0, tokens], [tokens])]
    batch = G.kv_batch(G.tensor(G.I32, (1, 1), ints[0].ptr), G.tensor(G.I32, (2,), ints[1].ptr),
                       G.tensor(G.I32, (1,), ints[2].ptr))
    qd, out = hip.to_dev(np.ones(d, np.float32)), hip.empty(4 * d, fill=0xFF)
    qt = G.tensor(G.F32, (d, 1, tokens), qd.ptr, [4, 0, 0, 0])
    assert G.attention_work_size(qt, *pools, batch) == 0
    print(f"attention tokens={tokens}", flush=True)
    G.attention(qt, *pools, batch, G.tensor(G.F32, (d, 1, tokens), out.ptr, [4, 0, 0, 0]), 0.125)
    hip.torch.cuda.synchronize()
    assert hip.last_error() == 0
    got = out.numpy(np.float32)
    # one weight over itself: the division's rounding
    assert (np.abs(got - v[0].astype(np.float16)) <= np.abs(v[0]) * 2.0 ** -22).all()
