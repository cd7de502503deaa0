"""A server's whole step over the 8-bit cache captured once and replayed over batches that grow, against the same calls
made one by one on a twin; buffers at the least alignment that the calls accept.  All bits are the same."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_pages import Book
from test_gpu_serving import BF16, F32, _buf, _dev, _hip, _ok
from test_gpu_serving8 import E4M3, I8
from test_gpu_serving8_ranges import _graph, _graph_gone

pytestmark = pytest.mark.gpu


class Step:
    """reserve, copy, store, attention and logits of one batch, all lengths and counts on the device."""

    def __init__(self, native, book, n_new, kv, nh=4, n_kv=2, hd=64, vocab=500):
        self.native, self.book, self.n_new, self.kv = native, book, n_new, kv
        self.nh, self.n_kv, self.hd, self.vocab = nh, n_kv, hd, vocab
        n, pages, ps = book.n, book.pages, book.ps
        self.room = 2 * n
        zeros = lambda *shape: _dev(np.zeros(shape, np.uint8))  # noqa: E731
        self.per = [n_kv * hd * ps] * 2 + [n_kv * ps // 16] * 2
        self.cache = [zeros(pages * size) for size in self.per]
        words = lambda x: _dev(np.ascontiguousarray(x, np.uint32))  # noqa: E731
        self.table, self.held, self.refs = words(book.table), words(book.held), words(book.refs)
        self.lens, self.first, self.new = (words(np.zeros(n)) for _ in range(3))
        self.pairs, self.count, self.granted, self.stat = (words(np.zeros(k)) for k in (2 * self.room, 1, n, 1))
        rows = n * n_new
        self.qkv = _dev(np.zeros((rows, (nh + 2 * n_kv) * hd), np.float32))
        self.cos, self.sin = (_dev(np.zeros((rows, hd // 2), np.float32)) for _ in range(2))
        self.q, self.out = (_dev(np.zeros((rows, nh * hd), np.uint16)) for _ in range(2))
        self.logits, self.adjusted = (_dev(np.zeros((rows, vocab), np.float32)) for _ in range(2))
        self.history, self.drafts = words(np.zeros((n, 64))), words(np.zeros((n, max(n_new - 1, 1))))
        self.last = words(np.zeros(n))
        self.factor = _dev(np.full(n, 1.25, np.float32))
        self.ws_size = [native.camelid_hip_pages_reserve_workspace(n, pages),
                        native.camelid_hip_paged8_attention_workspace(n, n_new, nh, n_kv, hd, ps, book.stride)]
        self.ws = [_buf(size) for size in self.ws_size]

    def feed(self, first, new, inputs):
        self.first.upload(np.array(first, np.uint32))
        self.new.upload(np.array(new, np.uint32))
        self.last.upload(np.array([max(m, 1) - 1 for m in new], np.uint32))
        self.lens.upload(np.array([a + b for a, b in zip(first, new)], np.uint32))
        for name, x in inputs.items():
            getattr(self, name).upload(x)
        _ok(self.native.camelid_hip_synchronize())

    def __call__(self, stream):
        nat, b, n = self.native, self.book, self.book.n
        _ok(nat.camelid_hip_pages_reserve(self.table.ptr, b.stride, self.held.ptr, n, self.first.ptr, self.lens.ptr, b.ps,
                                          self.refs.ptr, b.pages, self.pairs.ptr, self.room, self.count.ptr, self.granted.ptr,
                                          self.ws[0].ptr, self.ws_size[0], self.stat.ptr, stream))
        where, per = (C.c_void_p * 4)(*[x.ptr.value for x in self.cache]), (C.c_size_t * 4)(*self.per)
        _ok(nat.camelid_hip_pages_copy(where, per, 4, b.pages, self.pairs.ptr, self.room, self.count.ptr, self.stat.ptr, stream))
        cache = [x.ptr for x in self.cache]
        _ok(nat.camelid_hip_paged8_rope_kv(self.qkv.ptr, n, self.n_new, self.new.ptr, self.nh, self.n_kv, self.hd, self.hd, 1,
                                           self.cos.ptr, self.sin.ptr, None, None, 1e-5, self.q.ptr, BF16, *cache, self.kv,
                                           b.pages, b.ps, self.table.ptr, b.stride, self.lens.ptr, self.stat.ptr, stream))
        _ok(nat.camelid_hip_paged8_attention(self.q.ptr, BF16, self.nh * self.hd, n, self.n_new, self.new.ptr, self.nh, self.n_kv,
                                             self.hd, *cache, self.kv, b.pages, b.ps, self.table.ptr, b.stride, self.lens.ptr,
                                             0.125, self.out.ptr, self.nh * self.hd, self.ws[1].ptr, self.ws_size[1],
                                             self.stat.ptr, stream))
        if self.n_new <= 32:
            _ok(nat.camelid_hip_adjust_logits(self.logits.ptr, self.vocab, self.adjusted.ptr, self.vocab, F32, n, self.n_new,
                                              self.vocab, self.history.ptr, 64, self.lens.ptr, None, self.drafts.ptr,
                                              self.last.ptr, self.factor.ptr, self.factor.ptr, None, None, None, 0, None, None, 0,
                                              stream))

    def results(self):
        n = self.book.n
        got = dict(table=self.table, held=self.held, refs=self.refs, count=self.count, granted=self.granted, stat=self.stat)
        sizes = dict(table=n * self.book.stride, held=n, refs=self.book.pages, count=1, granted=n, stat=1)
        got = {name: x.download(np.uint32, sizes[name]) for name, x in got.items()}
        for i, x in enumerate(self.cache):
            got["cache%d" % i] = x.download(np.uint8, self.book.pages * self.per[i])
        rows = n * self.n_new
        got["out"] = self.out.download(np.uint16, rows * self.nh * self.hd)
        got["adjusted"] = self.adjusted.download(np.uint32, rows * self.vocab)
        return got


@pytest.mark.parametrize("n,stride,pages,ps,n_new,kv", [(6, 30, 120, 16, 4, I8), (6, 20, 9000, 32, 1, E4M3),
                                                       (3, 20, 60, 32, 70, E4M3), (5, 6000, 300, 16, 3, I8)])
def test_a_whole_step_replays_in_a_graph(native, n, stride, pages, ps, n_new, kv):
    rng = np.random.default_rng(n + pages + n_new)
    book = Book(n, stride, pages, ps)
    at = [int(x) for x in rng.integers(1, 3 * ps, n)]
    book.fill(rng, at)
    book.table[1, :book.held[0]] = book.table[0, :book.held[0]]    # row 1 begins as row 0 does
    book.held[1], at[1] = book.held[0], at[0]
    book.refs = book.counts()
    eager, replayed = Step(native, book, n_new, kv), Step(native, book, n_new, kv)
    held = _graph(native, replayed)
    copies = 0
    for step in range(6):
        rows = n * n_new
        new = [int(x) for x in rng.integers(0, n_new + 1, n)]
        if step == 0:
            new = [n_new] * n
        if step == 3:
            at[-1], new[-1] = 0, 0                               # a sequence ends
        angle = rng.uniform(-3, 3, (rows, 32))
        inputs = dict(qkv=rng.normal(0, 1.3, (rows, 8 * 64)).astype(np.float32), cos=np.cos(angle).astype(np.float32),
                      sin=np.sin(angle).astype(np.float32), logits=rng.normal(0, 2, (rows, 500)).astype(np.float32),
                      history=rng.integers(0, 500, (n, 64)).astype(np.uint32),
                      drafts=rng.integers(0, 500, (n, max(n_new - 1, 1))).astype(np.uint32))
        for one in (eager, replayed):
            one.feed(at, new, inputs)
        eager(None)
        want = eager.results()
        _hip(native, "hipGraphLaunch", held[2], held[0])
        _hip(native, "hipStreamSynchronize", held[0])
        got = replayed.results()
        for name, x in want.items():
            assert (got[name] == x).all(), (step, name)
        assert want["stat"][0] == 0 and want["granted"].all()
        assert np.isfinite((want["out"].astype(np.uint32) << 16).view(np.float32)).all()
        copies += int(want["count"][0])
        now = book.copy()
        now.table, now.held, now.refs = want["table"].reshape(n, stride), want["held"], want["refs"]
        assert (now.counts() == now.refs).all()
        at = [a + b for a, b in zip(at, new)]
    assert copies >= 1
    _graph_gone(native, *held)


@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("kv", [I8, E4M3])
def test_tables_and_exponents_at_their_least_alignment(native, kv, split):
    """cos, sin and the norms 4 bytes, exponents one byte off a granule: the same bits."""
    rng = np.random.default_rng(5)
    n, n_new, nh, n_kv, hd, ps, pages = 2, 20, 8, 2, 128, 16, 8
    rows = rng.normal(0, 1, (n * n_new, (nh + 2 * n_kv) * hd)).astype(np.float32)
    angle = rng.uniform(-3, 3, n * n_new * hd // 2)
    small = [np.cos(angle), np.sin(angle), rng.normal(1, 0.2, hd), rng.normal(1, 0.2, hd)]
    table, lens, dq = _dev(np.array([[5, 0], [2, 7]], np.uint32)), _dev(np.array([20, 31], np.uint32)), _dev(rows)
    results = []
    for off in (0, 1):
        keep = [_dev(np.concatenate([np.zeros(off), x]).astype(np.float32)) for x in small]
        cos, sin, qn, kn = [C.c_void_p(x.ptr.value + 4 * off) for x in keep]
        kc, vc = (_dev(np.zeros(pages * n_kv * hd * ps, np.uint8)) for _ in range(2))
        exps = [_dev(np.full(pages * n_kv + 1, 100, np.uint8)) for _ in range(2)]
        ke, ve = [C.c_void_p(x.ptr.value + off) for x in exps]
        q, out, stat = _dev(np.zeros((n * n_new, nh * hd), np.float32)), _dev(np.zeros((n * n_new, nh * hd), np.float32)), \
            _dev(np.zeros(1, np.uint32))
        _ok(native.camelid_hip_paged8_rope_kv(dq.ptr, n, n_new, None, nh, n_kv, hd, hd, split, cos, sin, qn, kn, 1e-5, q.ptr, F32,
                                              kc.ptr, vc.ptr, ke, ve, kv, pages, ps, table.ptr, 2, lens.ptr, stat.ptr, None))
        got = [x.download(np.uint8, pages * n_kv * hd * ps) for x in (kc, vc)]
        got += [x.download(np.uint8, pages * n_kv + 1)[off:off + pages * n_kv] for x in exps]
        for m in (1, n_new):
            size = native.camelid_hip_paged8_attention_workspace(n, m, nh, n_kv, hd, ps, 2)
            ws = _buf(size)
            _ok(native.camelid_hip_paged8_attention(q.ptr, F32, nh * hd, n, m, None, nh, n_kv, hd, kc.ptr, vc.ptr, ke, ve, kv,
                                                    pages, ps, table.ptr, 2, lens.ptr, 0.09, out.ptr, nh * hd, ws.ptr, size,
                                                    stat.ptr, None))
            got.append(out.download(np.uint32, n * m * nh * hd))
        k_out, v_out = (_dev(np.zeros((n, n_kv, 31, hd), np.float32)) for _ in range(2))
        _ok(native.camelid_hip_paged8_read(kc.ptr, vc.ptr, ke, ve, kv, pages, ps, n_kv, hd, table.ptr, 2, lens.ptr, n, k_out.ptr,
                                           v_out.ptr, F32, 31, stat.ptr, None))
        got += [x.download(np.uint32, n * n_kv * 31 * hd) for x in (k_out, v_out)]
        assert stat.download(np.uint32, 1)[0] == 0
        results.append(got)
    for near, far in zip(*results):
        assert (near == far).all()
