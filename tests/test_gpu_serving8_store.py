"""Stores into blocks of an 8-bit cache that hold NaN."""
import copy

import numpy as np
import pytest

from test_gpu_serving import F32
from test_gpu_serving8 import E4M3, Pages8, run_store

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,rope_dim", [(64, 64), (128, 128), (256, 256), (128, 64), (64, 0)])
@pytest.mark.parametrize("size", [2.0 ** -4, 2.0 ** 6])
def test_bytes_of_nan_stay_when_a_block_grows(native, hd, rope_dim, size):
    """e4m3 bytes of NaN at earlier positions (a cache filled by someone else) outlast a store into their block, whether its
    exponent rises or not; every other byte is what it would be without them."""
    rng = np.random.default_rng(hd + rope_dim)
    nh, n_kv, n, m = 4, 2, 43, 5
    clean = Pages8(rng, [n], 16, n_kv, hd, E4M3, fill=False)
    clean.put(rng, 0, n - m, spread=0)
    spots = [(p, h, d, b) for p, h, d, b in ((32, 0, 0, 0x7F), (33, 1, hd - 1, 0xFF), (37, 0, hd // 2 + 3, 0xFF), (35, 1, 7, 0x7F))]
    odd = copy.deepcopy(clean)
    for pg in (clean, odd):
        for name in ("k", "v"):
            for p, h, d, b in spots:
                x = pg.raw(0, [p], name)
                x[0, h, d] = b if pg is odd else 0
                pg.set(0, [p], name, x)
    qkv = (rng.normal(0, 1, (m, (nh + 2 * n_kv) * hd)) * size).astype(np.float32)
    one, zero = np.ones((m, rope_dim // 2), np.float32), np.zeros((m, rope_dim // 2), np.float32)
    was = {name: odd.exp_bytes(0, [32], name).copy() for name in ("k", "v")}
    for pg in (clean, odd):
        run_store(native, pg, qkv, m, [m], nh, rope_dim, False, one, zero, None, None, 0.0, F32)
        assert pg.status() == 0
    for name in ("k", "v"):
        now = odd.exp_bytes(0, [32], name)
        assert (now > was[name]).all() if size > 1 else (now == was[name]).all()
        assert (now == clean.exp_bytes(0, [32], name)).all() and (now < 255).all()
        for p, h, d, b in spots:
            assert odd.raw(0, [p], name)[0, h, d] == b, (name, p)
            x = odd.raw(0, [p], name)
            x[0, h, d] = clean.raw(0, [p], name)[0, h, d]
            odd.set(0, [p], name, x)
        assert ((odd.k if name == "k" else odd.v) == (clean.k if name == "k" else clean.v)).all(), name
    assert (odd.ke == clean.ke).all() and (odd.ve == clean.ve).all()
