"""Prompts over an 8-bit cache cut into pieces in each of the ways that their sizes and lengths lead to, against 64 bits.
References and tolerances are those of test_gpu_serving8."""
import math

import numpy as np
import pytest

from test_gpu_serving import BF16, F16, F32, typed
from test_gpu_serving8 import E4M3, I8, Pages8, attention8_reference, check_attention8, run_attention8

pytestmark = pytest.mark.gpu

CASES = [
    # nh, n_kv, hd, lens, new, page, q type, kv type, positions that the table has room for
    (16, 8, 64, [1100, 1030, 1200], [1100, 1030, 1200], 16, F32, I8, None),              # from nothing, whole segments
    (8, 8, 128, [1100, 1050, 1, 1060, 1100], [1100, 1050, 1, 1060, 1100], 64, BF16, E4M3, 8192),  # by the lengths
    (8, 8, 128, [1700, 1300, 1150], [1100, 900, 1000], 32, F16, I8, 4096),               # a few positions before
    (24, 8, 64, [512], [512], 16, BF16, I8, 2048),                                       # few segments, from nothing
    (24, 8, 64, [2048], [512], 32, F16, E4M3, None),                                     # pieces of 8 tiles
    (24, 8, 64, [6200], [512], 16, BF16, I8, None),                                      # as many pieces as fit at once
    (24, 8, 64, [6200], [512], 16, F32, E4M3, None),
    (16, 8, 128, [1500, 2100], [520, 470], 16, BF16, I8, None),
    (32, 8, 128, [1500], [1024], 128, F16, E4M3, None),
    (4, 4, 256, [1200, 1100], [1200, 1100], 16, BF16, I8, None),
]


@pytest.mark.parametrize("nh,n_kv,hd,lens,new,ps,qt,kv,room", CASES)
def test_prompts_in_pieces(native, nh, n_kv, hd, lens, new, ps, qt, kv, room):
    rng = np.random.default_rng(nh + hd + len(lens) + lens[0])
    pg = Pages8(rng, lens, ps, n_kv, hd, kv)
    if room:
        pg.table = np.pad(pg.table, ((0, 0), (0, room // ps - pg.stride)))
        pg.stride = room // ps
    q = typed(rng.normal(0, 1.7, (pg.n * max(new), nh * hd)), qt)
    scale = float(np.float32(1 / math.sqrt(hd)))
    out = run_attention8(native, pg, q, qt, max(new), new, nh, scale)
    assert pg.status() == 0
    check_attention8(out, attention8_reference(pg, q, qt, max(new), new, nh, scale, one_term=qt != F32), qt)
    again = run_attention8(native, pg, q, qt, max(new), new, nh, scale, upload=False)
    assert (out == again).all()
