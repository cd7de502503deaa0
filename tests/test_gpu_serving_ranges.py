"""Batched serving over a paged cache on the GPU, in the ranges that tests of single pieces do not reach:
waves that take several tiles, kernels that pass the caches by, batches of thousands of sequences, waves with
several shares of a row of logits.  Tolerances as in test_gpu_serving.py."""
import math

import numpy as np
import pytest

from test_gpu_serving import (BF16, F16, F32, Pages, attention_reference, check_attention, check_verify, from16,
                              run_attention, run_verify, softmax64, to16, typed, value, verify_reference)

pytestmark = pytest.mark.gpu


def shared_pages(rng, lens, ps, n_kv, hd, kv, distinct, rows=None):
    """Sequences whose table rows are drawn from the pages of one sequence of `distinct` positions (reading
    only: a small cache serves a large batch)."""
    pg = Pages(rng, [distinct], ps, n_kv, hd, kv, extra_stride=0, rows=rows)
    pool = pg.table[0, :distinct // ps]  # whole pages
    pg.n, pg.lens = len(lens), np.array(lens, np.uint32)
    pg.stride = max(1, -(-int(max(lens)) // ps))
    pg.table = rng.choice(pool, (pg.n, pg.stride)).astype(np.uint32)
    return pg


def longer_table(pg, stride):
    """The same sequences with room for `stride` pages each: entries behind the lengths name no page."""
    table = np.full((pg.n, stride), 0xFFFFFFFF, np.uint32)
    table[:, :pg.stride] = pg.table
    pg.table, pg.stride = table, stride


def tiles_a_piece(pg, new, nh):
    """The largest number of 32-position tiles of a workgroup's piece, worked out as the kernels' plan does."""
    rows = max(new) * (nh // pg.n_kv)
    nr = 2 if rows > 16 and pg.hd <= 128 else 1
    per_cu = {64: 5 - nr, 128: 4 - nr, 256: 2}[pg.hd]
    at_once = 256 * per_cu * 7 // 8
    total = sum(-(-int(n) // 32) * -(-m * (nh // pg.n_kv) // (16 * nr)) * pg.n_kv for n, m in zip(pg.lens, new) if m)
    one = -(-total // at_once)
    return max(4, (one + 3) & ~3) if one <= 16 else max(16, -(-total // 2048))


SEVERAL_TILES = [
    # nh, n_kv, hd, sequences, length, new, page, q type, kv type, weights, tiles a piece
    (32, 8, 128, 12, 1500, 5, 16, F32, F16, True, 12),
    (32, 8, 128, 12, 1500, 5, 32, BF16, BF16, True, 12),
    (8, 8, 64, 16, 4000, 1, 64, F16, F16, False, 16),
    (16, 8, 64, 33, 4400, 1, 32, F32, F16, True, 18),
    (16, 8, 128, 24, 4100, 2, 128, F32, BF16, False, 16),
    (16, 4, 256, 20, 2500, 1, 8, BF16, BF16, False, 16),
    (16, 4, 256, 9, 1700, 3, 16, F32, F16, True, 8),
]


@pytest.mark.parametrize("nh,n_kv,hd,n,length,new,ps,qt,kv,keep_w,tiles", SEVERAL_TILES)
@pytest.mark.parametrize("rising", [False, True])
def test_attention_of_several_tiles_a_wave(native, nh, n_kv, hd, n, length, new, ps, qt, kv, keep_w, tiles, rising):
    """Waves that take several tiles one after the other; rising: every page's scores beyond the one's before,
    so that the reference of the exponents moves with each tile."""
    rng = np.random.default_rng(n + hd + length)
    lens = [length - (i * 7) % (64 if tiles > 12 else length // 3) for i in range(n)]
    news = [max(1, new - i % 2) for i in range(n)]
    pg = shared_pages(rng, lens, ps, n_kv, hd, kv, 1024)
    q = rng.normal(0, 1.5, (n * new, nh * hd))
    if rising:
        q = np.abs(q)
        order = np.sort(pg.table, axis=1)
        pg.table = np.ascontiguousarray(order)
        pool = np.unique(pg.table)
        k = np.abs(rng.normal(0, 0.2, (len(pool), n_kv, hd * ps))) * (0.2 + np.arange(len(pool))[:, None, None] / 16 / len(pool) * 80)
        pg.k[pool] = to16(k, kv)
    q = typed(q, qt)
    assert tiles_a_piece(pg, news, nh) == tiles
    weights = rng.uniform(0, 2, (n, n_kv, pg.cap)).astype(np.float32) if keep_w else None
    scale = float(np.float32(1 / math.sqrt(hd)))
    out, got_w = run_attention(native, pg, q, qt, new, news, nh, scale, weights)
    assert pg.status() == 0
    check_attention(out, got_w, attention_reference(pg, q, qt, new, news, nh, scale, weights), weights, pg, new, news, qt)


@pytest.mark.parametrize("qt,kv", [(F32, F16), (BF16, BF16)])
def test_attention_of_several_tiles_with_bad_positions(native, qt, kv):
    """In a wave's later tiles: pages that do not exist, and an infinity or NaN at a draft's position, which
    reaches that draft's row and the later ones only."""
    rng = np.random.default_rng(71)
    nh, n_kv, hd, n, m, ps = 32, 8, 128, 12, 5, 16
    inf, nan = (0x7C00, 0x7E00) if kv == F16 else (0x7F80, 0x7FC0)
    lens = [1500 - 3 * i for i in range(n)]
    pg = Pages(rng, lens, ps, n_kv, hd, kv, extra_stride=0)
    assert tiles_a_piece(pg, [m] * n, nh) == 12
    q = typed(rng.normal(0, 1, (n * m, nh * hd)), qt)
    where = {2: (inf, 3), 5: (nan, 2), 7: (inf, 0)}  # sequence: bits, from the end
    for s, (bits, back) in where.items():
        kb, vb = pg.get(s, [lens[s] - 1 - back])
        vb[0, :, 9] = bits
        pg.set(s, [lens[s] - 1 - back], kb, vb)
    good = pg.table.copy()
    holes = {0: 60, 3: 1, 8: 92}                     # sequence: a page that does not exist
    bad = {(s, p) for s, page in holes.items() for p in range(page * ps, min(lens[s], (page + 1) * ps))}
    weights = np.zeros((n, n_kv, pg.cap), np.float32)
    ref, w, werr = attention_reference(pg, q, qt, m, [m] * n, nh, 0.1, weights, bad)
    for s, page in holes.items():
        pg.table[s, page] = pg.n_pages + s
    out, got_w = run_attention(native, pg, q, qt, m, [m] * n, nh, 0.1, weights)
    pg.table = good
    assert pg.status() == 1
    got = value(out, qt)
    for s in range(n):
        for t in range(m):
            y, tol = ref[s * m + t]
            y, tol, x = (z.reshape(nh, hd) for z in (y, tol, got[s * m + t]))
            if s in where and t >= m - 1 - where[s][1]:
                assert not np.isfinite(x[:, 9]).any(), (s, t)
                y, tol, x = (np.delete(z, 9, 1) for z in (y, tol, x))
            half = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}[qt]
            assert (np.abs(x - y) <= tol + half * (np.abs(y) + tol) + 2.0 ** -25).all(), (s, t)
    assert (np.abs(got_w - w) <= werr + 1e-30).all()


PASSING = [
    # nh, n_kv, hd, lens, new, page, q type, kv type, weights, positions of a table row
    (32, 8, 128, [700, 33, 1, 2000], [1, 1, 1, 1], 16, F32, F16, False, 17000),
    (32, 8, 128, [700, 33, 5, 2000], [5, 2, 5, 4], 32, BF16, BF16, True, 17024),
    (8, 8, 64, [900, 31, 32, 0, 1025, 64], [2, 1, 2, 0, 1, 2], 64, F16, F16, True, 22400),
    (64, 8, 64, [900, 77], [4, 1], 16, F32, BF16, False, 66000),
    (4, 4, 256, [50, 3000], [1, 1], 8, F32, F16, True, 33000),
    (16, 4, 256, [50, 1300], [4, 3], 4096, BF16, BF16, False, 36864),
]


@pytest.mark.parametrize("nh,n_kv,hd,lens,new,ps,qt,kv,keep_w,cap", PASSING)
def test_attention_that_passes_the_caches_by(native, nh, n_kv, hd, lens, new, ps, qt, kv, keep_w, cap):
    """Tables that could hold more than 256 MB of K and V: other kernels, the same rows."""
    rng = np.random.default_rng(hd + cap)
    pg = Pages(rng, lens, ps, n_kv, hd, kv, extra_stride=0)
    longer_table(pg, -(-cap // ps))
    assert pg.n * n_kv * hd * 4 * pg.cap > 256 << 20 and max(new) * (nh // n_kv) <= (32 if hd < 256 else 16)
    n_new = max(new)
    q = typed(rng.normal(0, 1.7, (len(lens) * n_new, nh * hd)), qt)
    weights = rng.uniform(0, 2, (len(lens), n_kv, pg.cap)).astype(np.float32) if keep_w else None
    scale = float(np.float32(1 / math.sqrt(hd)))
    out, got_w = run_attention(native, pg, q, qt, n_new, new, nh, scale, weights)
    assert pg.status() == 0
    check_attention(out, got_w, attention_reference(pg, q, qt, n_new, new, nh, scale, weights), weights, pg, n_new, new, qt)


def test_attention_beside_a_padding_sequence(native):
    """A batch with a sequence of no tokens among the real ones, and the batch without it: the same rows,
    and weights, within the bounds of either."""
    rng = np.random.default_rng(72)
    nh, n_kv, hd = 32, 8, 128
    pg = Pages(rng, [900, 0, 4000, 17], 32, n_kv, hd, F16)
    new = [2, 0, 1, 2]
    q = typed(rng.normal(0, 1, (8, nh * hd)), F32)
    w = rng.uniform(0, 1, (4, n_kv, pg.cap)).astype(np.float32)
    ref = attention_reference(pg, q, F32, 2, new, nh, float(np.float32(0.1)), w)
    out, got_w = run_attention(native, pg, q, F32, 2, new, nh, 0.1, w)
    check_attention(out, got_w, ref, w, pg, 2, new, F32)
    assert (got_w[1].view(np.uint32) == w[1].view(np.uint32)).all()
    real = [0, 2, 3]
    pg.n, pg.lens, pg.table = 3, pg.lens[real], np.ascontiguousarray(pg.table[real])
    rows = [r for s in real for r in (2 * s, 2 * s + 1)]
    out, got_w = run_attention(native, pg, q[rows], F32, 2, [2, 1, 2], nh, 0.1, w[real])
    check_attention(out, got_w, ([ref[0][r] for r in rows], ref[1][real], ref[2][real]), w[real], pg, 2, [2, 1, 2], F32)


@pytest.mark.parametrize("n", [1000, 4099])
def test_attention_of_thousands_of_sequences(native, n):
    rng = np.random.default_rng(73)
    nh, n_kv, hd = 4, 2, 64
    lens = [(i * 37) % 131 for i in range(n)]
    new = [min(x, i % 3) for i, x in enumerate(lens)]
    pg = shared_pages(rng, lens, 8, n_kv, hd, F16, 1024)
    q = typed(rng.normal(0, 1, (n * 2, nh * hd)), F32)
    w = np.zeros((n, n_kv, pg.cap), np.float32)
    out, got_w = run_attention(native, pg, q, F32, 2, new, nh, 0.125, w)
    assert pg.status() == 0
    check_attention(out, got_w, attention_reference(pg, q, F32, 2, new, nh, 0.125, w), w, pg, 2, new, F32)


SEVERAL_SHARES = [
    # seqs, drafts, vocab, draft logits, type: sequences x rows x shares of 2048 logits past 8192, 12288 and 16384,
    # shares no multiple of what a workgroup takes
    (40, 3, 70001, True, F32), (50, 3, 75000, True, BF16), (64, 3, 80001, True, F16), (140, 3, 70001, False, F32),
    (70, 1, 151936, False, BF16),
]


@pytest.mark.parametrize("n,k,vocab,has_draft,lt", SEVERAL_SHARES)
def test_verify_of_several_shares_a_wave(native, n, k, vocab, has_draft, lt):
    rng = np.random.default_rng(n + vocab)
    rows = 2 * k + 1 if has_draft else k + 1
    shares = -(-vocab // 2048)
    per = min(4, n * rows * shares // 4096)
    assert per >= 2 and shares % (4 * per)
    target = value(typed(rng.normal(0, 2.5, (n, k + 1, vocab)).astype(np.float32), lt), lt).reshape(n, k + 1, vocab)
    draft = None
    tokens = rng.integers(0, vocab, (n, k))
    if has_draft:
        draft = value(typed(target[:, :k] + rng.normal(0, 0.7, (n, k, vocab)), lt), lt).reshape(n, k, vocab)
        for s in range(n):
            for t in range(k):
                c = np.cumsum(softmax64(draft[s, t], 0.9))
                tokens[s, t] = min(vocab - 1, int(np.searchsorted(c, rng.random() * c[-1], side="right")))
    else:
        best = target[:, :k].argmax(-1)
        tokens = np.where(rng.random((n, k)) < 0.7, best, tokens)
        np.put_along_axis(target[:, :k], best[..., None], 24.0, -1)
    # the largest logits of some rows in the last share, and rows of masks
    target[1::5, :, vocab - 1] = 20.0
    target[2::5, :, :vocab - 3000] = -np.inf
    temps = np.array([0.0 if s % 6 == 3 else 0.5 + 0.3 * (s % 3) for s in range(n)], np.float32)
    lens = np.array([k if s == 0 else s % (k + 1) for s in range(n)])
    u = rng.random((n, k + 1)).astype(np.float32)
    want = verify_reference(target, draft, tokens, lens, temps, u)
    check_verify(run_verify(native, target, draft, tokens, lens, temps, u, lt), want)
