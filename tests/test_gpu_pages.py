"""Who holds which page, on the GPU: reserve, fork, compact and copy against a plain sequential evaluation of their
definitions.  All results are whole numbers or copies: exact."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_serving import _dev, _ok

pytestmark = pytest.mark.gpu

BAD_PAGE, BAD_LENGTH, NO_PAGE, BAD_FORK = 1, 2, 4, 8


def _u32(x):
    return np.ascontiguousarray(x, np.uint32)


class Book:
    """table, held, refs as the calls keep them."""

    def __init__(self, n, stride, pages, ps):
        self.n, self.stride, self.pages, self.ps = n, stride, pages, ps
        self.table = np.full((n, stride), 0xDEAD0000, np.uint32)
        self.held = np.zeros(n, np.uint32)
        self.refs = np.zeros(pages, np.uint32)

    def fill(self, rng, lens, order=None):
        """Rows of pages of their own in random order."""
        order = rng.permutation(self.pages) if order is None else order
        at = 0
        for s, x in enumerate(lens):
            k = -(-int(x) // self.ps)
            self.table[s, :k] = order[at:at + k]
            self.refs[order[at:at + k]] += 1
            self.held[s] = k
            at += k

    def copy(self):
        b = Book(self.n, self.stride, self.pages, self.ps)
        b.table, b.held, b.refs = self.table.copy(), self.held.copy(), self.refs.copy()
        return b

    def counts(self):
        """refs by counting the entries."""
        c = np.zeros(self.pages, np.uint32)
        for s in range(self.n):
            np.add.at(c, self.table[s, :self.held[s]], 1)
        return c


def reserve_reference(b, first, lens, max_pairs):
    """(pairs, granted, status) of camelid_hip_pages_reserve, b brought up to date."""
    n, status = b.n, 0
    want = [-(-int(x) // b.ps) for x in lens]
    good = []
    for s in range(n):
        if b.held[s] > b.stride or want[s] > b.stride:
            status |= BAD_LENGTH
            good.append(False)
        elif (b.table[s, :b.held[s]] >= b.pages).any():
            status |= BAD_PAGE
            good.append(False)
        else:
            good.append(True)
    for s in range(n):
        if good[s]:
            for j in range(want[s], int(b.held[s])):
                b.refs[b.table[s, j]] -= 1
            b.held[s] = min(int(b.held[s]), want[s])
    free = [int(p) for p in np.nonzero(b.refs == 0)[0]]
    need, cows = [], []
    for s in range(n):
        c = []
        if good[s] and first is not None and first[s] < lens[s]:
            c = [j for j in range(int(first[s]) // b.ps, int(b.held[s])) if b.refs[b.table[s, j]] > 1]
        cows.append(c)
        need.append(len(c) + want[s] - int(b.held[s]) if good[s] else 0)
    pairs, granted = [], np.zeros(n, np.uint32)
    drop, at, cow_at = [], 0, 0
    for s in range(n):
        at += need[s]
        cow_at += len(cows[s])
        if not good[s]:
            continue
        if need[s] and (at > len(free) or (cows[s] and cow_at > max_pairs)):
            status |= NO_PAGE
            continue
        granted[s] = 1
        mine = free[at - need[s]:at]
        for j in cows[s]:
            old, new = int(b.table[s, j]), mine.pop(0)
            pairs.append((cow_at - len(cows[s]) + cows[s].index(j), old, new))
            drop.append(old)
            b.table[s, j] = new
            b.refs[new] = 1
        for j in range(int(b.held[s]), want[s]):
            b.table[s, j] = mine.pop(0)
            b.refs[b.table[s, j]] = 1
        b.held[s] = max(int(b.held[s]), want[s])
    for p in drop:
        b.refs[p] -= 1
    return pairs, granted, status


class OnDevice:
    def __init__(self, native, b):
        self.native, self.b = native, b
        self.t, self.h, self.r, self.st = _dev(b.table), _dev(b.held), _dev(b.refs), _dev(_u32([0]))

    def back(self):
        b = self.b.copy()
        b.table = self.t.download(np.uint32, b.table.size).reshape(b.table.shape)
        b.held, b.refs = self.h.download(np.uint32, b.n), self.r.download(np.uint32, b.pages)
        return b

    def status(self):
        return int(self.st.download(np.uint32, 1)[0])

    def reserve(self, first, lens, max_pairs, stream=None, keep=None):
        b = self.b
        f = _dev(_u32(first)) if first is not None else None
        ln, pairs = _dev(_u32(lens)), _dev(np.full((max_pairs + 1, 2), 0xABABABAB, np.uint32))
        count, granted = _dev(_u32([99])), _dev(np.full(b.n, 99, np.uint32))
        size = self.native.camelid_hip_pages_reserve_workspace(b.n, b.pages)
        ws = _dev(np.full(size + 64, 0xEE, np.uint8))
        _ok(self.native.camelid_hip_pages_reserve(
            self.t.ptr, b.stride, self.h.ptr, b.n, f.ptr if f else None, ln.ptr, b.ps, self.r.ptr, b.pages, pairs.ptr,
            max_pairs, count.ptr, granted.ptr, ws.ptr, size, self.st.ptr, stream))
        got = pairs.download(np.uint32, 2 * (max_pairs + 1)).reshape(-1, 2)
        assert (got[max_pairs:] == 0xABABABAB).all() and (ws.download(np.uint8, size + 64)[size:] == 0xEE).all()
        return got, int(count.download(np.uint32, 1)[0]), granted.download(np.uint32, b.n)


def check_reserve(native, b, first, lens, max_pairs):
    dev = OnDevice(native, b)
    got, count, granted = dev.reserve(first, lens, max_pairs)
    want = b.copy()
    pairs, g, status = reserve_reference(want, first, lens, max_pairs)
    have = dev.back()
    assert dev.status() == status
    assert (granted == g).all()
    assert count == max([k + 1 for k, _, _ in pairs], default=0) == len(pairs)
    for k, old, new in pairs:
        assert tuple(got[k]) == (old, new)
    assert (have.table == want.table).all() and (have.held == want.held).all() and (have.refs == want.refs).all()
    return want


# (sequences, stride, pages, page size): by one workgroup, and by launches for each step
SIZES = [(1, 1, 1, 16), (7, 12, 100, 16), (64, 33, 2100, 8), (3, 5000, 8192, 16), (300, 50, 8192, 32),
         (1030, 3, 2000, 16), (40, 9, 9000, 64), (5, 7000, 20000, 16)]


@pytest.mark.parametrize("n,stride,pages,ps", SIZES)
def test_reserve_grows_shrinks_and_frees(native, n, stride, pages, ps):
    rng = np.random.default_rng(n + pages)
    b = Book(n, stride, pages, ps)
    most = min(stride, pages // n) * ps
    b.fill(rng, rng.integers(0, most + 1, n))
    for step in range(3):
        lens = rng.integers(0, most + 1, n)
        lens[rng.random(n) < 0.2] = 0
        b = check_reserve(native, b, None, lens, 4)
        assert (b.counts() == b.refs).all()


@pytest.mark.parametrize("n,stride,pages,ps", SIZES[1:])
def test_shared_pages_are_replaced_where_they_are_written(native, n, stride, pages, ps):
    rng = np.random.default_rng(n * 3 + pages)
    b = Book(n, stride, pages, ps)
    half = n // 2 + 1
    most = max(1, min(stride, pages // (3 * n)) * ps)
    lens = np.zeros(n, int)
    lens[:half] = rng.integers(1, most + 1, half)
    b.fill(rng, lens)
    for s in range(half, n):  # the rest share the beginnings of others
        k = int(rng.integers(0, b.held[s - half] + 1))
        b.table[s, :k] = b.table[s - half, :k]
        b.held[s] = k
        np.add.at(b.refs, b.table[s, :k], 1)
        lens[s] = max(0, k * ps - int(rng.integers(0, ps)))
    first = np.maximum(lens - rng.integers(0, 3 * ps, n), 0)
    first[::5] = lens[::5] + 4 * ps                      # nothing written
    grown = np.minimum(lens + rng.integers(0, 2 * ps, n), stride * ps)
    after = check_reserve(native, b, first, grown, 3 * n + 8)
    assert (after.counts() == after.refs).all()
    check_reserve(native, b, first, grown, 2)            # room for two pairs only


@pytest.mark.parametrize("pages", [60, 9000])
def test_reserve_without_enough_pages(native, pages):
    """The sequences behind the first one that cannot be served get nothing, needs of 0 are served."""
    rng = np.random.default_rng(pages)
    b = Book(8, 2000 if pages == 60 else 12000, pages, 16)  # (both kinds)
    b.fill(rng, [16 * (pages // 10), 32, 0, 0, 5, 0, 0, 1])
    left = int((b.refs == 0).sum())
    lens = [0, 32, 16 * (left // 2), 16 * left, 5, 40, 0, 1]   # (row 0 gives its pages back first)
    after = check_reserve(native, b, [0] * 8, lens, 4)
    assert (after.counts() == after.refs).all()


@pytest.mark.parametrize("pages", [200, 9000])
def test_reserve_leaves_bad_rows_alone(native, pages):
    rng = np.random.default_rng(1)
    b = Book(6, 4, pages, 16)
    b.fill(rng, [20, 33, 64, 10, 50, 0])
    b.table[1, 1] = pages                  # no page
    b.held[3] = 5                          # more than a row
    lens = [40, 10, 65, 30, 0, 20]         # the third longer than a row
    check_reserve(native, b, [0] * 6, lens, 8)


def test_forks(native):
    rng = np.random.default_rng(2)
    b = Book(12, 10, 80, 16)
    b.fill(rng, [100, 17, 160, 0, 0, 0, 0, 0, 0, 0, 48, 0])
    b.table[10, 2] = 80
    parents = [0, 0, 1, 2, 3, 2, 0, 12, 10, 4, 1]
    children = [3, 4, 5, 6, 7, 1, 8, 9, 9, 11, 8]
    lens = [33, 17, 160] + [0] * 9
    #       ok  -  ok ok -  -  -  -  -  -  -
    dev = OnDevice(native, b)
    pr, ch, ln = _dev(_u32(parents)), _dev(_u32(children)), _dev(_u32(lens))
    _ok(native.camelid_hip_pages_fork(dev.t.ptr, 10, dev.h.ptr, 12, pr.ptr, ch.ptr, len(parents), ln.ptr, 16, dev.r.ptr,
                                      80, dev.st.ptr, None))
    want, status = b.copy(), 0
    for i, (p, c) in enumerate(zip(parents, children)):
        if p >= 12 or p in children or children.count(c) > 1 or b.held[c]:
            status |= BAD_FORK
            continue
        k = min(int(b.held[p]), -(-lens[p] // 16))
        if (b.table[p, :k] >= 80).any():
            status |= BAD_PAGE
            continue
        want.table[c, :k] = b.table[p, :k]
        want.held[c] = k
        np.add.at(want.refs, want.table[c, :k], 1)
    have = dev.back()
    assert dev.status() == status == BAD_FORK
    assert (have.table == want.table).all() and (have.held == want.held).all() and (have.refs == want.refs).all()
    assert have.held[4] == 3 and have.held[6] == 10
    # all of the parent's pages without lens; many children of one parent
    b = Book(70, 4, 10, 8)
    b.fill(rng, [25] + [0] * 69)
    dev = OnDevice(native, b)
    pr, ch = _dev(_u32([0] * 69)), _dev(_u32(rng.permutation(np.arange(1, 70))))
    _ok(native.camelid_hip_pages_fork(dev.t.ptr, 4, dev.h.ptr, 70, pr.ptr, ch.ptr, 69, None, 8, dev.r.ptr, 10, None, None))
    have = dev.back()
    assert (have.table[:, :4] == b.table[0]).all() and (have.held == 4).all() and (have.refs[b.table[0]] == 70).all()


@pytest.mark.parametrize("n,stride,pages,used,most", [(1, 1, 1, 1, 4), (5, 40, 100, 40, 1000), (5, 40, 100, 40, 7),
                                                      (9, 700, 5000, 3000, 9999), (9, 700, 5000, 3000, 333),
                                                      (3, 30, 60, 0, 5), (4, 30, 64, 64, 5), (4, 4000, 12345, 9000, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(native, n, stride, pages, used, most, in_place):
    rng = np.random.default_rng(pages + used)
    b = Book(n, stride, pages, 16)
    share = rng.multinomial(used, np.ones(n) / n)
    share = np.minimum(share, stride)
    b.fill(rng, share * 16)
    for s in range(1, n):                                # some pages shared
        k = int(min(b.held[s - 1], stride - b.held[s], 3))
        b.table[s, b.held[s]:b.held[s] + k] = b.table[s - 1, :k]
        b.held[s] += k
        np.add.at(b.refs, b.table[s - 1, :k], 1)
    dev = OnDevice(native, b)
    to, ro = (dev.t, dev.r) if in_place else (_dev(np.zeros_like(b.table)), _dev(np.zeros_like(b.refs)))
    pairs, count, extent = _dev(np.full((most + 1, 2), 0xABABABAB, np.uint32)), _dev(_u32([9])), _dev(_u32([9]))
    size = native.camelid_hip_pages_compact_workspace(pages)
    ws = _dev(np.full(size + 64, 0xEE, np.uint8))
    _ok(native.camelid_hip_pages_compact(dev.t.ptr, stride, dev.h.ptr, n, dev.r.ptr, pages, to.ptr, ro.ptr, pairs.ptr, most,
                                         count.ptr, extent.ptr, ws.ptr, size, dev.st.ptr, None))
    live = np.nonzero(b.refs)[0]
    highs = [int(p) for p in live[::-1] if p >= len(live)]
    holes = [int(p) for p in np.nonzero(b.refs == 0)[0] if p < len(live)]
    moves = list(zip(highs, holes))[:most]
    got = pairs.download(np.uint32, 2 * (most + 1)).reshape(-1, 2)
    assert int(count.download(np.uint32, 1)[0]) == len(moves)
    assert [tuple(int(v) for v in x) for x in got[:len(moves)]] == moves and (got[len(moves):] == 0xABABABAB).all()
    table, refs = b.table.copy(), b.refs.copy()
    remap = dict(moves)
    for s in range(n):
        for j in range(int(b.held[s])):
            table[s, j] = remap.get(int(table[s, j]), table[s, j])
    for old, new in moves:
        refs[new], refs[old] = refs[old], 0
    assert (to.download(np.uint32, table.size).reshape(table.shape) == table).all()
    have = ro.download(np.uint32, pages)
    assert (have == refs).all()
    e = int(extent.download(np.uint32, 1)[0])
    assert (have[e:] == 0).all() and (e == 0 or have[e - 1] > 0)
    assert dev.status() == 0 and (ws.download(np.uint8, size + 64)[size:] == 0xEE).all()


@pytest.mark.parametrize("sizes", [[4096, 16, 1, 33], [65536] * 3, [8] * 300, [100, 48, 0, 7]])
def test_copy(native, sizes):
    rng = np.random.default_rng(len(sizes))
    pages, n = 50, 20
    data = [rng.integers(0, 256, (pages, size), dtype=np.uint8) for size in sizes]
    devs = [_dev(np.concatenate([d.reshape(-1), np.full(64, 0xEE, np.uint8)])) for d in data]
    order = rng.permutation(pages)
    pairs = order[:2 * n].reshape(n, 2).astype(np.uint32)
    pairs[3] = [50, 1]                                    # no page
    pairs[4] = [2, 0xFFFFFFFF]
    dp, st = _dev(pairs), _dev(_u32([0]))
    where = (C.c_void_p * len(sizes))(*[d.ptr.value for d in devs])
    per = (C.c_size_t * len(sizes))(*sizes)
    for count, room in ((n - 5, n), (n + 7, n), (None, n - 2), (0, n)):
        dc = _dev(_u32([count])) if count is not None else None
        _ok(native.camelid_hip_pages_copy(where, per, len(sizes), pages, dp.ptr, room, dc.ptr if dc else None, st.ptr, None))
        k = room if count is None else min(count, room)
        for i, (a, z) in enumerate(pairs[:k]):
            if i not in (3, 4):
                for d in data:
                    d[z] = d[a]
        for d, dev in zip(data, devs):
            got = dev.download(np.uint8, d.size + 64)
            assert (got[:d.size] == d.reshape(-1)).all() and (got[d.size:] == 0xEE).all()
    assert int(st.download(np.uint32, 1)[0]) == BAD_PAGE


def test_copy_of_large_pages_and_unaligned_buffers(native):
    rng = np.random.default_rng(9)
    size, pages = (1 << 22) + 16, 40                      # 168 MB: past the caches
    data = rng.integers(0, 256, pages * size, dtype=np.uint8)
    dev = _dev(data)
    pairs = _dev(_u32([[i, 39 - i] for i in range(15)]))
    where, per = (C.c_void_p * 1)(dev.ptr.value), (C.c_size_t * 1)(size)
    count = _dev(_u32([15]))
    _ok(native.camelid_hip_pages_copy(where, per, 1, pages, pairs.ptr, 40, count.ptr, None, None))
    data = data.reshape(pages, size)
    for i in range(15):
        data[39 - i] = data[i]
    assert (dev.download(np.uint8, data.size).reshape(data.shape) == data).all()
    where[0], per[0] = dev.ptr.value + 3, 1001            # odd addresses, odd sizes
    flat = data.reshape(-1)
    odd = _dev(_u32([[7, 400]]))
    _ok(native.camelid_hip_pages_copy(where, per, 1, 500, odd.ptr, 1, None, None, None))
    flat[3 + 400 * 1001:3 + 401 * 1001] = flat[3 + 7 * 1001:3 + 8 * 1001]
    assert (dev.download(np.uint8, flat.size) == flat).all()
