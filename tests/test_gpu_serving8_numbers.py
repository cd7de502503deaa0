"""What the 8-bit cache's attention keeps of its weights, against 64 bits.

Tolerance.  Queries with one dim that is not zero: a score is one product, exact in f32 (f16 and bf16 queries of at most
11 bits, 8-bit keys), times a factor that takes two roundings and one for itself: off by at most 4 u |score|,
u = 2^-24, counted from the row's reference.  A weight is then exp(+-2 d) - 1 off relatively with d = 4 u max |score|, 2^-21 more for its
own rounding to a pair of f16, 2^-20 for the exponential, and f16's smallest step, 2^-39 of the row's largest weight times
its block's scale, against numbers of up to 448.  Sums run in chains of n / 32 + 64 steps of u, numerator and denominator.  All against
sum_p w_p |v_p|, plus half a step of the result's type."""
import numpy as np
import pytest

from test_gpu_serving import BF16, F16, HALF_STEP, U, typed, value
from test_gpu_serving8 import E4M3, I8, Pages8, run_attention8

pytestmark = pytest.mark.gpu

CASES = [
    # nh, n_kv, hd, length, new, page, q type, kv type
    (8, 2, 128, 300, 8, 16, F16, I8),        # up to 8 new tokens
    (8, 2, 128, 300, 40, 16, F16, I8),       # more
    (8, 2, 128, 301, 40, 16, BF16, E4M3),
    (4, 1, 64, 260, 64, 32, F16, E4M3),
    (4, 4, 64, 400, 200, 16, BF16, I8),
    (4, 2, 256, 150, 70, 64, F16, I8),
    (2, 1, 256, 700, 65, 16, BF16, E4M3),
    (6, 1, 128, 1700, 130, 16, F16, E4M3),   # pieces joined
]


@pytest.mark.parametrize("nh,n_kv,hd,n,m,ps,qt,kv", CASES)
def test_weights_where_values_cancel(native, nh, n_kv, hd, n, m, ps, qt, kv):
    """A few heavy positions with values of both signs: some of the sums are small against their terms, and what the
    weights' rounding leaves there must be, too."""
    rng = np.random.default_rng(n + m + hd)
    pg = Pages8(rng, [n], ps, n_kv, hd, kv)
    g, scale, d0 = nh // n_kv, 1.5, hd - 3
    q = np.zeros((m, nh, hd))
    q[..., d0] = rng.normal(0, 1.5, (m, nh))
    q = typed(q.reshape(m, nh * hd), qt)
    out = value(run_attention8(native, pg, q, qt, m, [m], nh, scale), qt).reshape(m, nh, hd)
    x = value(q, qt).reshape(m, nh, hd)
    pos = np.arange(n)
    k, v = pg.get(0, pos, "k"), pg.get(0, pos, "v")
    ve = 2.0 ** (pg.exp_bytes(0, pos, "v").astype(np.float64) - 127)
    for t in range(m):
        see = n - m + t + 1
        for h in range(n_kv):
            score = x[t, h * g:(h + 1) * g, d0, None] * k[None, :see, h, d0] * scale
            w = np.exp(score - score.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            y = w @ v[:see, h]
            d = 4 * U * np.abs(score).max(-1, keepdims=True)
            rel = np.expm1(2 * d) + 2.0 ** -21 + 2.0 ** -20 + 2 * (see / 32 + 64) * U
            tol = rel * (w @ np.abs(v[:see, h])) + 2.0 ** -38 * 448 * see * (w * ve[:see, h]).max(-1, keepdims=True)
            near = np.abs(out[t, h * g:(h + 1) * g] - y) <= tol + HALF_STEP[qt] * (np.abs(y) + tol) + (2.0 ** -25 if qt == F16 else 0)
            assert near.all(), (t, h, float(np.abs(out[t, h * g:(h + 1) * g] - y).max()), float(tol.max()))
