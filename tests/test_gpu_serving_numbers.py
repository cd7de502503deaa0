"""Batched serving over a paged cache on the GPU: the bits that its numbers keep, and values at the ends of their
types."""
import math

import numpy as np
import pytest

from test_gpu_serving import (BF16, F16, F32, HALF_STEP, U, Pages, attention_reference, from16, run_attention, to16,
                              typed, value)

pytestmark = pytest.mark.gpu


def cancelling(kv, n=64, n_kv=2, g=4, hd=64):
    """Two positions a sequence whose values are each other's negatives and whose scores are 2^-11 apart: an
    output is v tanh(2^-12), a difference of weights near 1/2, so that an error of a weight is one of the
    output 2^12 times as large relative to it.  Every row has a score of its own."""
    rng = np.random.default_rng(81)
    pg = Pages(rng, [2] * n, 8, n_kv, hd, kv)
    v = rng.uniform(0.5, 1, (n, n_kv, hd))
    k = np.zeros((2, hd))
    k[:, 0], k[:, 1] = (1.0, 1.0 + 2.0 ** -7), 1.0
    for s in range(n):
        pg.set(s, [0, 1], to16(np.broadcast_to(k[:, None], (2, n_kv, hd)), kv), to16(np.stack([-v[s], v[s]]), kv))
    q = np.zeros((n, n_kv * g, hd))
    q[..., 0], q[..., 1] = 2.0 ** -4, rng.uniform(-2, 2, (n, n_kv * g))
    return pg, typed(q.reshape(n, -1), kv)


# Weights as sums of 16-bit numbers: three bf16 hold 24 bits (half a step of each term's 8 bits is left to the
# next), two f16 hold 22.
WEIGHT_BITS = {BF16: 2.0 ** -24, F16: 2.0 ** -22}


@pytest.mark.parametrize("kv", [BF16, F16])
def test_weights_of_16_bit_rows_keep_their_bits(native, kv):
    pg, q = cancelling(kv)
    nh = 8
    out, _ = run_attention(native, pg, q, kv, 1, [1] * pg.n, nh, 1.0)
    ref = attention_reference(pg, q, kv, 1, [1] * pg.n, nh, 1.0, None)[0]
    for r in range(pg.n):
        want, got = ref[r][0], value(out[r], kv)
        # |score| < 2.5: its two products and sum are exact, log2(e) rounded and the fma off by 2^-24 of less than 4
        # each; the exponential by 2^-23; the weight's terms; sums and quotient: 8 roundings at most of a single tile's
        # two positions.  All relative to the sum of p |v|, which is at most 1
        tol = 2 * 4 * U + 2.0 ** -23 + WEIGHT_BITS[kv] + 8 * U + HALF_STEP[kv] * np.abs(want)
        assert (np.abs(got - want) <= tol).all(), (r, np.abs(got - want).max(), tol.max())


def rows_near(got, ref, qt):
    for r, want in enumerate(ref):
        y, tol = want
        x = value(got[r], qt)
        assert (np.abs(x - y) <= tol + HALF_STEP[qt] * (np.abs(y) + tol) + 2.0 ** -25).all(), (r, x, y)


@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("size,scale,keys", [(1e37, 1e-37, 1.0), (3e38, 1e-37, 0.05), (1.5 * 2.0 ** 117, 2.0 ** -118, 1.0),
                                             (1.0, 0.125, 1.0), (1e-30, 1e29, 1.0), (1e-37, 1e37, 1.0),
                                             (1e-40, 3e38, 20.0)])
def test_f32_queries_of_any_size(native, kv, size, scale, keys):
    """Queries from subnormal to the largest f32, with a scale that brings their scores near 1."""
    rng = np.random.default_rng(82)
    nh, n_kv, hd, lens = 8, 2, 64, [70, 300]
    pg = Pages(rng, lens, 16, n_kv, hd, kv, rows=lambda *sh: rng.normal(0, keys, sh))
    q = np.clip(rng.normal(0, 1, (2, nh * hd)), -1.1, 1.1) * size
    if size == 3e38:
        q[0, 5], q[1, 100] = np.finfo(np.float32).max, -np.finfo(np.float32).max
    q = q.astype(np.float32)
    assert np.isfinite(q).all()
    scale = float(np.float32(scale))
    out, _ = run_attention(native, pg, q, F32, 1, [1, 1], nh, scale)
    rows_near(out, attention_reference(pg, q, F32, 1, [1, 1], nh, scale, None)[0], F32)


@pytest.mark.parametrize("scale", [1.0, 2.3e38, 3e38, -3.4e38])
def test_scales_near_the_largest(native, scale):
    """f32 rows with every finite scale: keys so small that the scores are near 1."""
    rng = np.random.default_rng(89)
    nh, n_kv, hd, lens = 4, 2, 64, [70, 300]
    pg = Pages(rng, lens, 16, n_kv, hd, BF16)
    for s, n in enumerate(lens):
        k = np.zeros((n, n_kv, hd))
        k[..., 0] = (1 + rng.integers(0, 128, (n, n_kv)) / 128) * 2.0 ** -125 * (3e38 if scale == 1.0 else 1.0)
        pg.set(s, np.arange(n), to16(k, BF16), pg.get(s, np.arange(n))[1])
    q = np.zeros((2, nh, hd), np.float32)
    q[..., 0] = rng.choice([0.5, 1.0], (2, nh)) * rng.choice([1, -1], (2, nh))
    q = q.reshape(2, -1)
    scale = float(np.float32(scale))
    out, _ = run_attention(native, pg, q, F32, 1, [1, 1], nh, scale)
    rows_near(out, attention_reference(pg, q, F32, 1, [1, 1], nh, scale, None)[0], F32)


@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** 13, 2.0 ** 40, 2.0 ** 80])
def test_scores_of_any_size(native, kv, wide, scale):
    """Scores from 1e4 to 1e32 in size, of either sign: the positions of the largest share the row (three, far
    apart), the others are e^-64 or less beside them, and a row's weights add up to 1."""
    rng = np.random.default_rng(83)
    nh, n_kv, hd = 4, 2, 64
    lens = [1200, 70, 333]
    pg = Pages(rng, lens, 16, n_kv, hd, kv)
    qt = F32 if wide else kv
    best = {}
    for s, n in enumerate(lens):
        kb, vb = pg.get(s, np.arange(n))
        k = np.zeros((n, n_kv, hd))
        k[..., 0] = 1024 + 8 * rng.integers(1, 100, (n, n_kv))
        for h in range(n_kv):
            at = rng.permutation(n)[:6]
            k[at[:3], h, 0], k[at[3:], h, 0] = 2040, 1024  # the largest, the smallest
            best[s, h] = at[:3], at[3:]
        pg.set(s, np.arange(n), to16(k, kv), vb)
    q = np.zeros((3, nh, hd))
    q[..., 0] = np.exp2(rng.integers(3, 15, (3, nh))) * [1, -1, 1, -1]
    weights = np.zeros((3, n_kv, pg.cap), np.float32)
    out, got_w = run_attention(native, pg, typed(q.reshape(3, -1), qt), qt, 1, [1] * 3, nh, scale, weights)
    for s, n in enumerate(lens):
        v = from16(pg.get(s, np.arange(n))[1], kv)
        chain = (n / 32 + 64) * U  # with the weights' bits, 2^-22, and the exponentials', 2^-23
        for h in range(nh):
            at = best[s, h // 2][h % 2]
            want = v[at, h // 2].mean(0)
            tol = (chain + 2.0 ** -21) * np.abs(v[at, h // 2]).mean(0) + HALF_STEP[qt] * np.abs(want)
            assert (np.abs(value(out[s], qt).reshape(nh, hd)[h] - want) <= tol).all(), (s, h)
        for h in range(n_kv):
            want = np.zeros(pg.cap)
            want[np.r_[best[s, h]]] = 1 / 3
            assert (np.abs(got_w[s, h] - want) <= chain + 2.0 ** -21).all(), (s, h)


@pytest.mark.parametrize("qt", [F32, BF16])
@pytest.mark.parametrize("lens,new", [([70, 200, 1], [1, 1, 1]), ([3000, 1900, 40], [5, 2, 4])])
def test_values_near_the_largest(native, qt, lens, new):
    """Rows that average values of bf16's largest sizes: every one finite, whatever the number of positions."""
    rng = np.random.default_rng(84)
    nh, n_kv, hd = 8, 2, 128
    pg = Pages(rng, lens, 16, n_kv, hd, BF16)
    for s, n in enumerate(lens):
        kb, vb = pg.get(s, np.arange(n))
        pg.set(s, np.arange(n), to16(rng.normal(0, 0.1, (n, n_kv, hd)), BF16),
               to16(rng.uniform(2.5e38, 3.3e38, (n, n_kv, hd)) * rng.choice([1, 1, -1], (1, n_kv, hd)), BF16))
    n_new = max(new)
    q = typed(rng.normal(0, 1, (len(lens) * n_new, nh * hd)), qt)
    out, _ = run_attention(native, pg, q, qt, n_new, new, nh, 0.125)
    ref = attention_reference(pg, q, qt, n_new, new, nh, 0.125, None)[0]
    rows = [r for r in range(len(ref)) if ref[r] is not None]
    rows_near(out[rows], [ref[r] for r in rows], qt)


def test_values_near_the_smallest(native):
    """bf16 values down to its smallest normal ones: off by f32's smallest normal number at most."""
    rng = np.random.default_rng(85)
    nh, n_kv, hd, lens = 8, 2, 64, [70, 1000]
    pg = Pages(rng, lens, 16, n_kv, hd, BF16, rows=lambda *sh: rng.normal(0, 1, sh) * 2.0 ** -118)
    q = typed(rng.normal(0, 1, (2, nh * hd)), F32)
    out, _ = run_attention(native, pg, q, F32, 1, [1, 1], nh, 0.125)
    for r, (y, tol) in enumerate(attention_reference(pg, q, F32, 1, [1, 1], nh, 0.125, None)[0]):
        assert (np.abs(value(out[r], F32) - y) <= tol + 2.0 ** -126).all(), r


def test_bad_draft_logits_leave_the_engine_as_it_was(native):
    """A draft's row of logits without a distribution is the caller's mistake: refused, nothing of the engine's
    cache lost.  Rows that are not needed (T = 0, drafts behind a rejected one) may hold anything."""
    from camelid_amd._native import HipError
    from camelid_amd.model import ResidentSession, SyntheticModel, prompt_tokens, rope_tables, tiny_config
    cfg = tiny_config(prompt_len=12)
    model = SyntheticModel.generate(cfg)
    sess = ResidentSession(model, 32)
    prompt = prompt_tokens(cfg)
    sess.prefill(prompt[:-1])
    eng, base = sess.engine, len(prompt) - 1
    step = [int(prompt[-1]), 3, 5]
    cos, sin = rope_tables(cfg, base, 3)

    def call(draft_logits, temp=1.0, u=(0.4, 0.5, 0.6)):
        return [x.tolist() for x in eng.verify_sampled(model.embed(step), cos, sin, base, cfg.scale(), step[1:], u, temp,
                                                       draft_logits)]

    good = np.random.default_rng(86).normal(0, 1, (2, cfg.vocab)).astype(np.float32)
    want = call(good)
    for bad in (np.nan, np.inf, -np.inf):
        rows = good.copy()
        rows[0, slice(None) if bad == -np.inf else 7] = bad
        with pytest.raises(HipError, match="draft_logits"):
            call(rows)
        assert eng.filled() == base and call(good) == want
        assert call(rows, temp=0.0) == call(None, temp=0.0)
    rows = good.copy()
    rows[0, 3] = 1e4          # the first draft certain of itself: rejected by any number above its probability
    rows[1, 9] = np.nan
    assert len(call(rows, u=(0.9999, 0.5, 0.6))[0]) == 1
    assert eng.filled() == base and call(good) == want
    sess.close()


@pytest.mark.parametrize("kv", [F16, BF16])
def test_infinite_keys_of_16_bit_rows(native, kv):
    """An infinity in K that a row sees: a weight of zero where it makes the score -infinity, NaN where
    +infinity, whichever of its sequence's tiles it is in; not seen by a row: nothing."""
    rng = np.random.default_rng(87)
    nh, n_kv, hd, m = 8, 2, 64, 3
    lens = [45, 45, 700, 700]
    at = [10, 43, 5, 698]  # the last but one of the new tokens' positions: seen by two of the three rows
    pg = Pages(rng, lens, 16, n_kv, hd, kv)
    q = rng.normal(0, 1, (4 * m, nh, hd))
    q[:, :4, 3], q[:, 4:, 3] = -np.abs(q[:, :4, 3]) - 0.1, np.abs(q[:, 4:, 3]) + 0.1  # KV head 0 below zero, 1 above
    q = typed(q.reshape(4 * m, -1), kv)
    for s, p in enumerate(at):
        kb, vb = pg.get(s, [p])
        kb[0, :, 3] = 0x7C00 if kv == F16 else 0x7F80
        pg.set(s, [p], kb, vb)
    out, _ = run_attention(native, pg, q, kv, m, [m] * 4, nh, 0.125)
    masked = attention_reference(pg, q, kv, m, [m] * 4, nh, 0.125, None, {(s, p) for s, p in enumerate(at)})[0]
    for s, p in enumerate(at):
        for t in range(m):
            got = value(out[s * m + t], kv).reshape(nh, hd)
            y, tol = (z.reshape(nh, hd) for z in masked[s * m + t])
            sees = p <= lens[s] - m + t
            near = np.abs(got - y) <= tol + HALF_STEP[kv] * (np.abs(y) + tol) + 2.0 ** -25
            assert near[:4].all(), (s, t)
            assert np.isnan(got[4:]).all() if sees else near[4:].all(), (s, t)


@pytest.mark.parametrize("qt", [F32, F16])
def test_subnormal_keys_and_values(native, qt):
    """f16 K and V below its smallest normal number count with all their bits."""
    rng = np.random.default_rng(88)
    nh, n_kv, hd, lens = 8, 2, 64, [70, 1000]
    pg = Pages(rng, lens, 16, n_kv, hd, F16, rows=lambda *sh: rng.normal(0, 1, sh) * 2.0 ** -17)
    q = typed(rng.normal(0, 1, (2, nh * hd)) * 256, qt)
    scale = 2.0 ** 6  # scores near 1
    out, _ = run_attention(native, pg, q, qt, 1, [1, 1], nh, scale)
    for r, (y, tol) in enumerate(attention_reference(pg, q, qt, 1, [1, 1], nh, scale, None)[0]):
        half = np.maximum(HALF_STEP[qt] * np.abs(y), 2.0 ** -25 if qt == F16 else 0.0)  # (f16 results are subnormal)
        assert (np.abs(value(out[r], qt) - y) <= tol + half).all(), r
