"""The 8-bit cache's calls where they can go wrong: numbers far apart, NaN, bad pages, large pools, streams and graphs,
and a run of all calls as a server makes them.  References and tolerances are those of test_gpu_serving8."""
import ctypes as C
import math

import numpy as np
import pytest

from test_gpu_pages import Book, reserve_reference
from test_gpu_logits import reference as logits_reference
from test_gpu_serving import (BF16, F16, F32, HALF_STEP, _buf, _dev, _hip, _ok, check_verify, rope_reference, run_verify,
                              typed, value, verify_reference)
from test_gpu_serving8 import (E4M3, I8, Pages8, attention8_buffers, attention8_reference, call_attention8, check_attention8,
                               check_stored, run_attention8, run_store)

pytestmark = pytest.mark.gpu


def _case(rng, pg, qt, new, nh, size=1.7):
    return typed(rng.normal(0, size, (pg.n * max(new), nh * pg.hd)), qt)


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("kv", [I8, E4M3])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 3, 8], [40, 33, 17]])
def test_scales_far_apart(native, qt, kv, new):
    """Blocks whose scales differ by many powers of two: what is heavy has small values and the other way round."""
    rng = np.random.default_rng(qt + kv + new[0])
    nh, n_kv, hd, lens = 8, 2, 64, [300, 700, 129]
    for spread_k, spread_v in ((6, 0), (0, 60), (3, 110)):
        pg = Pages8(rng, lens, 32, n_kv, hd, kv)
        near = 127 - (5 if kv == I8 else 7)
        for s, n in enumerate(lens):
            for b in range(-(-n // 16)):
                page, i = pg.table[s, 16 * b // 32], 16 * b % 32 // 16
                pg.ke[page, :, i] = near - rng.integers(0, spread_k + 1, n_kv)
                pg.ve[page, :, i] = near + rng.integers(-spread_v, 1, n_kv)
        q = _case(rng, pg, qt, new, nh)
        out = run_attention8(native, pg, q, qt, max(new), new, nh, 0.125)
        check_attention8(out, attention8_reference(pg, q, qt, max(new), new, nh, 0.125, one_term=qt != F32 and max(new) > 8), qt)


@pytest.mark.parametrize("kv", [I8, E4M3])
@pytest.mark.parametrize("new", [1, 40])
def test_values_at_the_ends(native, kv, new):
    """V near the largest f32 and near the smallest, K zero, rows of equal weights, all in f32."""
    rng = np.random.default_rng(kv + new)
    nh, n_kv, hd, n = 4, 1, 128, 500
    for ve in (246 if kv == E4M3 else 248, 1, 127):
        pg = Pages8(rng, [n], 16, n_kv, hd, kv)
        pg.ve[pg.table[0, :-(-n // 16)]] = ve
        if ve == 127:
            pg.k[:] = 0
        v = pg.raw(0, np.arange(n), "v")
        pg.set(0, np.arange(n), "v", v & 0x7F if kv == I8 else np.minimum(v & 0x7F, 0x7E))  # (no cancelling)
        q = _case(rng, pg, F32, [new], nh)
        out = run_attention8(native, pg, q, F32, new, [new], nh, 0.1)
        scale = float(np.float32(0.1))
        ref = attention8_reference(pg, q, F32, new, [new], nh, scale)
        for r, (y, tol) in enumerate(ref):
            # (products below f32's subnormals vanish: sums are kept in units of 2^38)
            assert (np.abs(out[r].astype(np.float64) - y) <= tol + 2.0 ** -149 * 2.0 ** 38 * n).all() and np.isfinite(out[r]).all()


@pytest.mark.parametrize("new", [1, 6, 40])
@pytest.mark.parametrize("size,scale,ke", [(1.0, -0.125, 120), (1.0, 0.0, 120), (1e30, 1e-31, 120), (1e-30, 1e29, 122),
                                           (3e38, 1e-38, 100), (1e-42, 1e30, 160), (100.0, 3.0, 124), (1.0, 2.0 ** -100, 200)])
def test_queries_and_scales_of_any_size(native, new, size, scale, ke):
    rng = np.random.default_rng(new)
    nh, n_kv, hd, lens = 4, 2, 64, [90, 200]
    pg = Pages8(rng, lens, 16, n_kv, hd, I8)
    for s, n in enumerate(lens):
        pg.ke[pg.table[s, :-(-n // 16)]] = ke
    q = np.clip(rng.normal(0, 0.4, (2 * new, nh * hd)), -1, 1) * size
    q = q.astype(np.float32)
    scale = float(np.float32(scale))
    out = run_attention8(native, pg, q, F32, new, [new, new], nh, scale)
    assert np.isfinite(out).all()
    check_attention8(out, attention8_reference(pg, q, F32, new, [new, new], nh, scale), F32)


@pytest.mark.parametrize("qt", [F32, BF16])
@pytest.mark.parametrize("m", [5, 40])
@pytest.mark.parametrize("where", ["k exponent", "v exponent", "k byte", "v byte"])
def test_nan_reaches_the_rows_that_see_it(native, qt, m, where):
    """NaN in the newest tokens: of a block's exponent from the block's first position on, of an e4m3 byte from its own;
    earlier rows and other sequences are as they would be without it."""
    rng = np.random.default_rng(m)
    nh, n_kv, hd, n = 8, 2, 128, 133
    pg = Pages8(rng, [n, n], 16, n_kv, hd, E4M3)
    pos = n - 3
    if "exponent" in where:
        pg.exps(where[0])[pg.table[0, pos // 16], 0, 0] = 255
        first_bad = pos // 16 * 16
    else:
        b = pg.raw(0, [pos], where[0])
        b[0, 0, 7] = 0x7F if qt == F32 else 0xFF
        pg.set(0, [pos], where[0], b)
        first_bad = pos
    q = _case(rng, pg, qt, [m, m], nh)
    out = value(run_attention8(native, pg, q, qt, m, [m, m], nh, 0.1), qt)
    ref = attention8_reference(pg, q, qt, m, [m, m], nh, float(np.float32(0.1)), one_term=qt != F32 and m > 8)
    clean = 0
    for r, (y, tol) in enumerate(ref):
        t = n - m + r
        got, want = out[r].reshape(nh, hd), y.reshape(nh, hd)
        near = np.abs(out[r] - y) <= tol + HALF_STEP[qt] * (np.abs(y) + tol)
        if r >= m or t < first_bad:
            assert near.all(), r
            clean += r < m
            continue
        hit = np.zeros((nh, hd), bool)
        hit[:nh // n_kv] = True
        if where == "v byte":
            hit[:, np.arange(hd) != 7] = False
        assert np.isnan(got[hit]).all() and near.reshape(nh, hd)[~hit].all(), (r, where)
    assert clean > 0 or where != "v byte"


@pytest.mark.parametrize("qt,new", [(F32, [2, 3, 1, 2, 1]), (F16, [40, 30, 9, 2, 33])])
def test_attention_with_bad_pages_and_lengths(native, qt, new):
    rng = np.random.default_rng(12)
    nh, n_kv, hd, lens = 8, 2, 64, [150, 70, 100, 5, 40]
    pg = Pages8(rng, lens, 16, n_kv, hd, E4M3)
    pg.table[0, 3] = pg.n_pages            # positions 48 .. 63 of sequence 0 count as masked
    pg.table[4, :] = 0xFFFFFFFF            # nothing left: zeros
    pg.lens[2] = pg.cap + 1                # left alone
    new = list(new)
    if max(new) == 3:
        new[3] = 2
    q = _case(rng, pg, qt, new, nh)
    out = run_attention8(native, pg, q, qt, max(new), new, nh, 0.125)
    assert pg.status() == 3
    host = Pages8(rng, [150, 70, 1, 5, 1], 16, n_kv, hd, E4M3, fill=False)
    for name in ("k", "v", "ke", "ve", "ps", "stride", "n_pages"):
        setattr(host, name, getattr(pg, name))
    host.table = pg.table.copy()
    host.table[0, 3] = host.table[0, 2]    # (a page to read; masked below)
    host.lens = np.array([150, 70, 1, 5, 1], np.uint32)
    live = [new[0], new[1], 0, min(new[3], 5), 0]
    ref = attention8_reference(host, q, qt, max(new), live, nh, 0.125, bad={(0, p) for p in range(48, 64)},
                               one_term=qt != F32 and max(new) > 8)
    rows = max(new)
    for r in range(rows * 2, rows * 3):
        assert (out[r] == 7).all()
    assert (out[rows * 4:rows * 4 + new[4]] == 0).all()
    ref[rows * 4:rows * 4 + new[4]] = [None] * new[4]
    out[rows * 4:rows * 4 + new[4]] = 7
    check_attention8(out, ref, qt)


LONG = [
    # nh, n_kv, hd, lens, new, page, q type, kv type, positions that the table has room for
    (8, 2, 128, [9000, 300, 5000], [1, 1, 1], 64, F32, I8, None),
    (32, 8, 128, [1500] * 20, [4] * 20, 32, BF16, E4M3, None),
    (8, 8, 64, [700, 20, 3000], [1, 1, 1], 128, F16, I8, 1 << 19),      # past the caches
    (4, 1, 256, [2500], [2], 16, F32, E4M3, 1 << 20),
    (16, 2, 128, [3000, 50], [1, 1], 16, F32, I8, 1 << 20),
    (4, 1, 128, [2600], [600], 16, F16, E4M3, None),
    (8, 2, 64, [1500, 900], [500, 700], 64, F32, I8, None),
    (2, 1, 256, [1200], [300], 16, BF16, I8, None),
    (3, 1, 128, [1400], [300], 4096, F32, E4M3, 1 << 18),               # large f32 prompts, by the table's room
    (3, 1, 128, [1400], [300], 4096, F16, E4M3, 1 << 18),               # and 16-bit ones
    (4, 2, 128, [900, 1, 2000, 0, 130], [128, 1, 257, 0, 130], 64, BF16, I8, 1 << 18),
    (1, 1, 128, [70000], [130], 16, F16, I8, 1 << 20),
    (2, 2, 128, [64 * i % 700 + 1 for i in range(90)], [min(64 * i % 700 + 1, i % 70) for i in range(90)], 16, BF16, I8, None),
]


@pytest.mark.parametrize("nh,n_kv,hd,lens,new,ps,qt,kv,room", LONG)
def test_attention_over_many_tiles(native, nh, n_kv, hd, lens, new, ps, qt, kv, room):
    rng = np.random.default_rng(nh + hd + len(lens))
    pg = Pages8(rng, lens, ps, n_kv, hd, kv)
    if room:
        pg.table = np.pad(pg.table, ((0, 0), (0, room // ps - pg.stride)))
        pg.stride = room // ps
    q = _case(rng, pg, qt, new, nh)
    scale = float(np.float32(1 / math.sqrt(hd)))
    first = run_attention8(native, pg, q, qt, max(new), new, nh, scale)
    ref = attention8_reference(pg, q, qt, max(new), new, nh, scale, one_term=qt != F32 and max(new) > 8)
    check_attention8(first, ref, qt)
    again = run_attention8(native, pg, q, qt, max(new), new, nh, scale, upload=False)
    assert (first == again).all()          # the same call, the same bits


def test_workspace_holds_for_smaller_calls(native):
    """The bytes for calls of at most some sizes are enough for all smaller ones."""
    rng = np.random.default_rng(5)
    size = native.camelid_hip_paged8_attention_workspace
    for _ in range(300):
        n_kv, g, hd = int(rng.choice([1, 2, 8])), int(rng.integers(1, 20)), int(rng.choice([64, 128, 256]))
        n, new, stride = int(rng.integers(1, 30)), int(2 ** rng.uniform(0, 11)), int(2 ** rng.uniform(0, 11))
        most = size(n, new, n_kv * g, n_kv, hd, 16, stride)
        for _ in range(5):
            assert size(int(rng.integers(1, n + 1)), int(rng.integers(1, new + 1)), n_kv * g, n_kv, hd, 16,
                        int(rng.integers(1, stride + 1))) <= most


def _graph(native, call):
    stream, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    _hip(native, "hipStreamCreate", C.byref(stream))
    _hip(native, "hipStreamBeginCapture", stream, 1)
    call(stream)
    _hip(native, "hipStreamEndCapture", stream, C.byref(graph))
    _hip(native, "hipGraphInstantiate", C.byref(run), graph, None, None, C.c_size_t(0))
    return stream, graph, run


def _graph_gone(native, stream, graph, run):
    _hip(native, "hipGraphExecDestroy", run)
    _hip(native, "hipGraphDestroy", graph)
    _hip(native, "hipStreamDestroy", stream)


@pytest.mark.parametrize("nh,n_kv,hd,new,qt,kv", [(24, 8, 128, 8, F32, I8), (4, 4, 256, 1, BF16, E4M3), (8, 2, 128, 60, F16, I8),
                                                  (16, 2, 64, 100, F32, E4M3)])
def test_attention8_replays_in_a_graph_over_a_growing_cache(native, nh, n_kv, hd, new, qt, kv):
    rng = np.random.default_rng(61)
    n, cap = 3, 1024
    pg = Pages8(rng, [cap] * n, 16, n_kv, hd, kv, extra_stride=0)
    pg.upload()
    b = attention8_buffers(native, pg, _case(rng, pg, qt, [new] * n, nh), new, [new] * n, nh)
    call = lambda stream: call_attention8(native, pg, b, qt, new, nh, 0.1, nh * hd, nh * hd, stream)  # noqa: E731
    held = _graph(native, call)
    for lens in ([new] * n, [new, 300, 133], [cap, new, 513], [1000, 1001, 1002], [new] * n):
        pg.dl.upload(np.array(lens, np.uint32))
        _ok(native.camelid_hip_synchronize())
        call(None)
        want = b["out"].download(b["out0"].dtype, b["out0"].size)
        b["out"].upload(b["out0"])
        _hip(native, "hipGraphLaunch", held[2], held[0])
        _hip(native, "hipStreamSynchronize", held[0])
        assert (b["out"].download(b["out0"].dtype, b["out0"].size) == want).all(), lens
    assert pg.status() == 0
    _graph_gone(native, *held)


def test_two_batches_on_two_streams(native):
    rng = np.random.default_rng(63)
    jobs = []
    for nh, n_kv, lens, new, kv in ((32, 8, [1500] * 12, 5, I8), (8, 2, [700, 90], 80, E4M3)):
        pg = Pages8(rng, lens, 32, n_kv, 128, kv)
        pg.upload()
        stream = C.c_void_p()
        _hip(native, "hipStreamCreate", C.byref(stream))
        jobs.append((pg, attention8_buffers(native, pg, _case(rng, pg, F32, [new] * len(lens), nh), new, [new] * len(lens), nh),
                     nh, new, stream))

    def call(job, stream):
        call_attention8(native, job[0], job[1], F32, job[3], job[2], 0.1, job[2] * 128, job[2] * 128, stream)

    def read(job):
        return job[1]["out"].download(np.uint32, job[1]["out0"].size)

    want = []
    for job in jobs:
        call(job, None)
        _ok(native.camelid_hip_synchronize())
        want.append(read(job))
    for _ in range(8):
        for job in jobs:
            call(job, job[4])
    for job, w in zip(jobs, want):
        _hip(native, "hipStreamSynchronize", job[4])
        assert (read(job) == w).all()
        _hip(native, "hipStreamDestroy", job[4])


def test_a_cache_past_two_to_the_32_bytes(native):
    """The same calls over a small pool and over the far end of one whose offsets pass 32 bits: the same bits."""
    rng = np.random.default_rng(62)
    n, n_kv, nh, hd, ps, new = 2, 8, 16, 128, 4096, 150
    page = n_kv * hd * ps
    far = (1 << 32) // page + 1
    table = np.array([[3], [1]], np.uint32)
    rows = rng.normal(0, 1, (n * new, (nh + 2 * n_kv) * hd)).astype(np.float32)
    angle = rng.uniform(0, 7, (n * new, hd // 2))
    dq, dc, dn = _dev(rows), _dev(np.cos(angle).astype(np.float32)), _dev(np.sin(angle).astype(np.float32))
    results = []
    for offset in (0, far):
        pages = offset + 6
        kc, vc = _buf(pages * page), _buf(pages * page)
        ke, ve = _buf(pages * n_kv * ps // 16), _buf(pages * n_kv * ps // 16)
        dt, dl, stat = _dev(table + np.uint32(offset)), _dev(np.zeros(n, np.uint32)), _dev(np.zeros(1, np.uint32))
        q_out, out = _buf(n * new * nh * hd * 4), _dev(np.zeros((n * new, nh * hd), np.float32))
        for at, dim in ((new, hd), (2 * new, hd - 32), (3 * new, hd)):
            dl.upload(np.full(n, at, np.uint32))
            _ok(native.camelid_hip_paged8_rope_kv(dq.ptr, n, new, None, nh, n_kv, hd, dim, 1, dc.ptr, dn.ptr, None, None, 1e-5,
                                                  q_out.ptr, F32, kc.ptr, vc.ptr, ke.ptr, ve.ptr, E4M3, pages, ps, dt.ptr, 1,
                                                  dl.ptr, stat.ptr, None))
            _ok(native.camelid_hip_synchronize())
        # both sequences' pages copied within the pool, and read there
        pairs = _dev((np.array([[3, 4], [1, 5]]) + offset).astype(np.uint32))
        where = (C.c_void_p * 4)(kc.ptr.value, vc.ptr.value, ke.ptr.value, ve.ptr.value)
        per = (C.c_size_t * 4)(page, page, n_kv * ps // 16, n_kv * ps // 16)
        _ok(native.camelid_hip_pages_copy(where, per, 4, pages, pairs.ptr, 2, None, stat.ptr, None))
        dt.upload((np.array([[4], [5]]) + offset).astype(np.uint32))
        got = []
        for m in (2, new):
            size = native.camelid_hip_paged8_attention_workspace(n, m, nh, n_kv, hd, ps, 1)
            ws = _buf(size)
            _ok(native.camelid_hip_paged8_attention(q_out.ptr, F32, nh * hd, n, m, None, nh, n_kv, hd, kc.ptr, vc.ptr, ke.ptr,
                                                    ve.ptr, E4M3, pages, ps, dt.ptr, 1, dl.ptr, 0.09, out.ptr, nh * hd, ws.ptr,
                                                    size, stat.ptr, None))
            got.append(out.download(np.uint32, n * m * nh * hd))
        rk, rv = (_dev(np.zeros((n, n_kv, 3 * new, hd), np.uint16)) for _ in range(2))
        _ok(native.camelid_hip_paged8_read(kc.ptr, vc.ptr, ke.ptr, ve.ptr, E4M3, pages, ps, n_kv, hd, dt.ptr, 1, dl.ptr, n, rk.ptr,
                                           rv.ptr, F16, 3 * new, stat.ptr, None))
        got += [x.download(np.uint16, n * n_kv * 3 * new * hd) for x in (rk, rv)]
        assert stat.download(np.uint32, 1)[0] == 0
        assert np.isfinite(got[0].view(np.float32)).all() and got[0].view(np.float32).std() > 0.01
        results.append(got)
        for b in (kc, vc, ke, ve):
            b.free()
    for near, off in zip(*results):
        assert (near == off).all()


def test_a_serving_loop(native):
    """Prompts, then forks and rounds of reserve, copy, store, attend, adjust and verify over one pool, every call
    against its definition on what the calls before it left."""
    import copy
    rng = np.random.default_rng(41)
    nh, n_kv, hd, ps, k, vocab, n, stride, pages = 8, 2, 64, 16, 3, 300, 4, 9, 40
    kv = I8
    book = Book(n, stride, pages, ps)
    pg = Pages8(rng, [stride * ps] * n, ps, n_kv, hd, kv, spare=0, extra_stride=0, fill=False)
    pg.n_pages = pages
    for name, shape in (("k", (pages, n_kv, hd * ps)), ("v", (pages, n_kv, hd * ps)), ("ke", (pages, n_kv, 1)),
                        ("ve", (pages, n_kv, 1))):
        setattr(pg, name, np.full(shape, 255 if "e" in name else 0x80, np.uint8))
    proj = rng.normal(0, 0.3, (nh * hd, vocab))
    lens, texts = [0] * n, [[] for _ in range(n)]

    def reserve(first, grown):
        from test_gpu_pages import OnDevice
        dev = OnDevice(native, book)
        got, count, granted = dev.reserve(first, grown, 8)
        pairs, g, status = reserve_reference(book, first, grown, 8)
        have = dev.back()
        assert dev.status() == status == 0 and (granted == g).all() and count == len(pairs)
        assert (have.table == book.table).all() and (have.refs == book.refs).all()
        if pairs:
            pg.upload()
            where = (C.c_void_p * 4)(*[x.ptr.value for x in (pg.dk, pg.dv, pg.dke, pg.dve)])
            per = (C.c_size_t * 4)(n_kv * hd * ps, n_kv * hd * ps, n_kv, n_kv)
            was = copy.deepcopy({name: getattr(pg, name) for name in ("k", "v", "ke", "ve")})
            dp, dc = _dev(got), _dev(np.array([count], np.uint32))
            _ok(native.camelid_hip_pages_copy(where, per, 4, pages, dp.ptr, 8, dc.ptr, None, None))
            pg.download()
            for name, old in was.items():
                for _, a, b in pairs:
                    old[b] = old[a]
                assert (getattr(pg, name) == old).all()
        pg.table = book.table.copy()
        return len(pairs)

    def store(new, n_new):
        qkv = rng.normal(0, 1.2, (n * n_new, (nh + 2 * n_kv) * hd)).astype(np.float32)
        ang = rng.uniform(-3, 3, (n * n_new, hd // 2))
        cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
        pg.lens = np.array(lens, np.uint32)
        was = copy.deepcopy({name: getattr(pg, name) for name in ("k", "v", "ke", "ve")})
        q, _ = run_store(native, pg, qkv, n_new, new, nh, hd, False, cos, sin, None, None, 0.0, F32)
        y, _ = rope_reference(qkv, cos, sin, nh, n_kv, hd, hd, False, None, None, 0.0)
        before = copy.copy(pg)
        for name, old in was.items():
            setattr(before, name, old)
        for s in range(n):
            if new[s]:
                r = slice(s * n_new, s * n_new + new[s])
                check_stored(pg, before, s, lens[s] - new[s], "k", y[r, nh:nh + n_kv], False)
                check_stored(pg, before, s, lens[s] - new[s], "v", qkv[r].reshape(new[s], -1, hd)[:, nh + n_kv:].astype(np.float64), True)
        for name in was:
            assert (getattr(pg, name) == getattr(before, name)).all()
        return q

    copied = 0
    prompt = [40, 21, 0, 0]
    reserve(None, prompt)
    lens = list(prompt)
    texts = [list(rng.integers(0, vocab, x)) for x in prompt]
    q = store(prompt, max(prompt))
    out = run_attention8(native, pg, q, F32, max(prompt), prompt, nh, 0.125)
    check_attention8(out, attention8_reference(pg, q, F32, max(prompt), prompt, nh, 0.125), F32)
    # rows 2 and 3 go on from rows 0 and 1
    from test_gpu_pages import OnDevice
    dev = OnDevice(native, book)
    pairs = [_dev(np.array(x, np.uint32)) for x in ([0, 1], [2, 3], lens)]
    _ok(native.camelid_hip_pages_fork(dev.t.ptr, stride, dev.h.ptr, n, pairs[0].ptr, pairs[1].ptr, 2, pairs[2].ptr, ps,
                                      dev.r.ptr, pages, dev.st.ptr, None))
    book = dev.back()
    assert dev.status() == 0 and (book.counts() == book.refs).all()
    lens[2:], texts[2:] = lens[:2], [list(t) for t in texts[:2]]
    pg.table = book.table.copy()
    for step in range(12):
        new = [k + 1 - (s + step) % 2 for s in range(n)]         # the last token and its drafts
        grown = [a + b for a, b in zip(lens, new)]
        copied += reserve(lens, grown)
        lens = grown
        q = store(new, k + 1)
        out = run_attention8(native, pg, q, F32, k + 1, new, nh, 0.125)
        check_attention8(out, attention8_reference(pg, q, F32, k + 1, new, nh, 0.125), F32)
        real = np.arange(k + 1)[None] < np.array(new)[:, None]
        target = np.float32(np.where(real.reshape(-1, 1), out.astype(np.float64), 0.0) @ proj).reshape(n, k + 1, vocab)
        tokens = target[:, :k].argmax(-1).astype(np.uint32)
        tokens[:, 1] = rng.integers(0, vocab, n)
        dl = np.array(new, np.uint32) - 1
        # penalties over the text, a grammar without the even tokens for one sequence
        known = max(len(t) for t in texts)
        history = np.array([t + [0] * (known - len(t)) for t in texts], np.uint32)
        hl, prompts = np.array([len(t) for t in texts], np.uint32), np.array([40, 21, 40, 21], np.uint32)
        rep, freq, pres = (np.full(n, x, np.float32) for x in (1.2, 0.1, 0.2))
        mask = np.full((n, k + 1, 10), 0xFFFFFFFF, np.uint32)
        mask[1] = 0xAAAAAAAA
        keep = [_dev(x) for x in (target, history, hl, prompts, tokens, dl, rep, freq, pres, mask)]
        _ok(native.camelid_hip_adjust_logits(keep[0].ptr, vocab, keep[0].ptr, vocab, F32, n, k + 1, vocab, keep[1].ptr, known,
                                             keep[2].ptr, keep[3].ptr, keep[4].ptr, keep[5].ptr, keep[6].ptr, keep[7].ptr,
                                             keep[8].ptr, None, None, 0, None, keep[9].ptr, 10, None))
        want = logits_reference(target, history, hl, prompts, tokens, dl, rep, freq, pres, None, None, None, mask)
        target = keep[0].download(np.float32, target.size).reshape(target.shape)
        assert (target.view(np.uint32) == want.view(np.uint32)).all()
        u = rng.random((n, k + 1)).astype(np.float32)
        got = run_verify(native, target.astype(np.float64), None, tokens, dl, [0.8] * n, u, F32)
        check_verify(got, verify_reference(target.astype(np.float64), None, tokens, dl, [0.8] * n, u))
        assert got[1][1][int(got[0][1])] % 2 == 1
        for s in range(n):                                       # the rejected drafts leave the cache
            a = int(got[0][s])
            lens[s] -= new[s] - 1 - a
            texts[s] += [int(x) for x in got[1][s][:a + 1]]
        if step == 8:                                            # one sequence ends, another's row is let go
            lens[0] = 0
            texts[0] = []
            reserve(None, lens)
            lens[0] = 0
    assert copied >= 3 and (book.counts() == book.refs).all()
