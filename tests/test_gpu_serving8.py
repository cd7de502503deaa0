"""Serving over a paged cache held in 8 bits on the GPU, each entry point against a plain evaluation of its
definition in 64 bits.

Tolerances.  u = 2^-24 is half an f32 step, e = finfo(type).eps / 2 half a step of a 16-bit output.
 * q rows: those of the 16-bit store's tests.
 * Stored bytes and exponents are exact: K is worked out in f64 (relative error below 2^-45 with the norm's
   sum), so a byte may differ only where the definition's value is within 2^-38 of a border between two bytes, an
   exponent only where the largest element is as close to a power of two's end.  V takes no arithmetic: exact.
 * Attention: a score is a sum of hd products, (hd + 8) u sum |q_d k_d| scale off at most, 2^-21 of it more where
   f32 queries go through pairs of f16; a weight is then exp(+-2 d) - 1 off relatively, 2^-21 more for its own
   rounding to a pair of f16 (2^-11 to one, for the 16-bit rows of prompts), 2^-20 for the exponential, whose
   argument of up to 16 is an f32 (2^-21 log(2)), and f16's smallest step, 2^-39 of the row's largest weight times its
   block's scale, against numbers of up to 448.  Sums run in chains of n / 32 + 64.  All against sum_p w_p |v_p|, plus
   e |result| for the final rounding."""
import ctypes as C
import math

import numpy as np
import pytest

from test_gpu_serving import (BF16, F16, F32, HALF_STEP, U, _dev, _ok, rope_reference, typed, value)

pytestmark = pytest.mark.gpu

I8, E4M3 = 3, 4
LARGEST = {I8: 127.0, E4M3: 448.0}
TOP_EXP = {I8: 121, E4M3: 119}
NAN_BYTE = {I8: 0x80, E4M3: 0x7F}  # what lies where nobody wrote (int8 has no NaN: its lowest number)


def _e4m3_values():
    b = np.arange(128)
    m, x = b & 7, b >> 3
    v = np.where(x > 0, (1 + m / 8.0) * 2.0 ** (x - 7.0), m / 8.0 * 2.0 ** -6)
    v[127] = np.nan
    return v


E4M3_VALUES = _e4m3_values()


def numbers(b, kv):
    """Bytes -> the numbers that they stand for without their block's scale."""
    if kv == I8:
        return b.view(np.int8).astype(np.float64)
    return np.where(b & 0x80, -1.0, 1.0) * E4M3_VALUES[b & 0x7F]


def rounded(x, kv):
    """Numbers -> bytes, to nearest even; and how far each is from a border between two of them, in steps."""
    x = np.clip(x, -LARGEST[kv], LARGEST[kv])
    if kv == I8:
        y = np.rint(x)
        return y.astype(np.int8).view(np.uint8), np.abs(np.abs(x - np.trunc(x)) - 0.5)
    a = np.abs(x)
    unit = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    y = np.rint(a / unit) * unit
    code = np.searchsorted(E4M3_VALUES[:127], y).astype(np.uint8)
    return np.where(np.signbit(x), code | 0x80, code).astype(np.uint8), np.abs(a / unit - np.trunc(a / unit) - 0.5)


def exponent(top, kv):
    """The smallest e with top <= LARGEST 2^e."""
    if not np.isfinite(top):
        return 128
    if top == 0:
        return -126
    e = math.frexp(top)[1] - 10
    while top > LARGEST[kv] * 2.0 ** e:
        e += 1
    return min(max(e, -126), TOP_EXP[kv])


class Pages8:
    """An 8-bit cache on the host: pages in random order, poison in everything nobody owns."""

    def __init__(self, rng, lens, ps, n_kv, hd, kv, spare=2, extra_stride=1, fill=True, size=1.0):
        self.ps, self.n_kv, self.hd, self.kv, self.n = ps, n_kv, hd, kv, len(lens)
        self.lens = np.array(lens, np.uint32)
        self.stride = max(1, -(-int(max(lens)) // ps)) + extra_stride
        self.n_pages = self.n * self.stride + spare
        self.table = rng.permutation(self.n_pages)[:self.n * self.stride].astype(np.uint32).reshape(self.n, self.stride)
        self.k = np.full((self.n_pages, n_kv, hd * ps), NAN_BYTE[kv], np.uint8)
        self.v = self.k.copy()
        self.ke = np.full((self.n_pages, n_kv, ps // 16), 255, np.uint8)
        self.ve = self.ke.copy()
        if fill:
            for s, n in enumerate(lens):
                if n:
                    self.put(rng, s, n, size)

    def put(self, rng, s, n, size=1.0, spread=2):
        """Random rows at positions [0, n) of sequence s: numbers of a model's distribution, scales around `size`."""
        near = 127 + int(round(math.log2(size))) - (5 if self.kv == I8 else 7)
        for name in ("k", "v"):
            x = rng.normal(0, 36 if self.kv == I8 else 110, (n, self.n_kv, self.hd))
            self.set(s, np.arange(n), name, rounded(x, self.kv)[0])
            e = rng.integers(near - spread, near + spread + 1, (self.n_kv, -(-n // 16)))
            for b in range(e.shape[1]):
                self.exps(name)[self.table[s, 16 * b // self.ps], :, 16 * b % self.ps // 16] = e[:, b]

    def exps(self, name):
        return self.ke if name == "k" else self.ve

    def cells(self, s, pos, name):
        pos = np.asarray(pos)
        page = self.table[s][pos // self.ps].astype(np.int64)[:, None, None]
        o = (pos % self.ps)[:, None, None]
        h, d = np.arange(self.n_kv)[:, None], np.arange(self.hd)[None]
        base = (page * self.n_kv + h) * (self.hd * self.ps)
        return base + ((d // 16 * self.ps + o) * 16 + d % 16 if name == "k" else (o // 16 * self.hd + d) * 16 + o % 16)

    def set(self, s, pos, name, b):
        (self.k if name == "k" else self.v).reshape(-1)[self.cells(s, pos, name)] = b

    def raw(self, s, pos, name):
        return (self.k if name == "k" else self.v).reshape(-1)[self.cells(s, pos, name)]

    def exp_bytes(self, s, pos, name):
        """[positions][n_kv]"""
        pos = np.asarray(pos)
        return self.exps(name)[self.table[s][pos // self.ps], :, pos % self.ps // 16]

    def get(self, s, pos, name):
        """Values in 64 bits [positions][n_kv][hd]."""
        e = self.exp_bytes(s, pos, name).astype(np.float64)
        scale = np.where(e == 255, np.nan, 2.0 ** (e - 127))
        return numbers(self.raw(s, pos, name), self.kv) * scale[..., None]

    @property
    def cap(self):
        return self.stride * self.ps

    def upload(self):
        self.dk, self.dv, self.dke, self.dve = (_dev(x) for x in (self.k, self.v, self.ke, self.ve))
        self.dt, self.dl, self.dstat = _dev(self.table), _dev(self.lens), _dev(np.zeros(1, np.uint32))

    def download(self):
        for name, dev in (("k", self.dk), ("v", self.dv), ("ke", self.dke), ("ve", self.dve)):
            old = getattr(self, name)
            setattr(self, name, dev.download(np.uint8, old.size).reshape(old.shape))

    def status(self):
        return int(self.dstat.download(np.uint32, 1)[0])


# --------------------------------------------------------------------------------------- RoPE + store
def run_store(native, pg, qkv, n_new, new, nh, rope_dim, split, cos, sin, qn, kn, eps, qt):
    pg.upload()
    q0 = np.full((pg.n * n_new, nh * pg.hd), 7, np.float32 if qt == F32 else np.uint16)
    dq = _dev(q0)
    dn = [_dev(w) if w is not None else None for w in (qn, kn)]
    bufs = _dev(qkv), _dev(cos), _dev(sin), _dev(np.array(new, np.uint32))
    _ok(native.camelid_hip_paged8_rope_kv(
        bufs[0].ptr, pg.n, n_new, bufs[3].ptr, nh, pg.n_kv, pg.hd, rope_dim, int(split), bufs[1].ptr, bufs[2].ptr,
        dn[0].ptr if dn[0] else None, dn[1].ptr if dn[1] else None, eps, dq.ptr, qt, pg.dk.ptr, pg.dv.ptr, pg.dke.ptr,
        pg.dve.ptr, pg.kv, pg.n_pages, pg.ps, pg.dt.ptr, pg.stride, pg.dl.ptr, pg.dstat.ptr, None))
    q = dq.download(q0.dtype, q0.size).reshape(q0.shape)
    pg.download()
    return q, q0


def check_stored(pg, was, s, first, name, rows, exact):
    """The cache of sequence s against rows [new][n_kv][hd] stored from `first` on over what `was` held; what `was`
    holds is brought up to date, so that everything else can be compared as a whole."""
    kv, end, near = pg.kv, first + len(rows), 0.0 if exact else 2.0 ** -38
    for begin in range(first // 16 * 16, end, 16):
        lo, hi = max(begin, first), min(begin + 16, end)
        old = np.arange(begin, lo)
        for h in range(pg.n_kv):
            top = np.abs(rows[lo - first:hi - first, h]).max() if np.isfinite(rows[lo - first:hi - first, h]).all() else np.inf
            e = exponent(top, kv)
            e_was = int(was.exp_bytes(s, [begin], name)[0, h]) - 127
            if lo > begin:
                e = max(e, e_was)
            got = int(pg.exp_bytes(s, [begin], name)[0, h]) - 127
            if e != got:
                m = math.frexp(top / LARGEST[kv])[0]
                assert abs(got - e) == 1 and min(abs(m - 0.5), abs(m - 1.0)) <= near, (s, name, begin, h, e, got)
            if got == 128:
                continue
            want, border = rounded(rows[lo - first:hi - first, h] * 2.0 ** -got, kv)
            have = pg.raw(s, np.arange(lo, hi), name)[:, h]
            # (-0 and 0 are the same number)
            same = (want == have) | ((want & 0x7F == 0) & (have & 0x7F == 0) & (kv == E4M3))
            assert (same | (border <= near)).all(), (s, name, begin, h)
            if len(old):
                keep = was.raw(s, old, name)[:, h]
                if got != e_was:
                    keep = rounded(numbers(keep, kv) * 2.0 ** (e_was - got), kv)[0]
                have = pg.raw(s, old, name)[:, h]
                assert ((keep == have) | ((keep & 0x7F == 0) & (have & 0x7F == 0) & (kv == E4M3))).all(), (s, name, begin, h)
    span = np.arange(first // 16 * 16, end)
    was.set(s, span, name, pg.raw(s, span, name))
    for begin in range(first // 16 * 16, end, 16):
        page, b = pg.table[s, begin // pg.ps], begin % pg.ps // 16
        was.exps(name)[page, :, b] = pg.exps(name)[page, :, b]


STORE_CASES = [
    # nh, n_kv, hd, rope_dim, split, norm, lens, new, page, q type, kv type
    (32, 4, 64, 64, False, False, [128], [1], 16, F32, I8),
    (8, 8, 128, 128, True, True, [1, 17, 16, 300, 0], [1, 5, 0, 3, 0], 32, BF16, E4M3),
    (24, 8, 128, 128, False, True, [70, 33], [70, 1], 16, F16, I8),
    (4, 2, 256, 256, True, True, [40, 17], [13, 17], 256, F32, E4M3),
    (6, 3, 64, 64, False, False, [31, 32, 33, 47], [15, 16, 2, 31], 16, BF16, I8),
    (3, 1, 256, 256, False, False, [100], [99], 64, F16, I8),
    (5, 5, 128, 128, False, True, [70, 20], [64, 4], 4096, F32, E4M3),
    (24, 8, 128, 96, False, True, [70, 33], [70, 1], 16, F16, I8),
    (2, 1, 64, 0, False, True, [21], [3], 16, F32, E4M3),
    (16, 2, 64, 32, True, False, [65, 1, 64], [64, 1, 33], 64, BF16, E4M3),
]


@pytest.mark.parametrize("nh,n_kv,hd,rope_dim,split,norm,lens,new,ps,qt,kv", STORE_CASES)
def test_store_against_64_bits(native, nh, n_kv, hd, rope_dim, split, norm, lens, new, ps, qt, kv):
    import copy
    rng = np.random.default_rng(hd + nh + ps)
    pg = Pages8(rng, lens, ps, n_kv, hd, kv, fill=False)
    for s, (n, m) in enumerate(zip(lens, new)):
        if n > m:
            pg.put(rng, s, n - m, spread=4)
    n_new, rows = max(new), len(lens) * max(new)
    qkv = (rng.normal(0, 1.5, (rows, (nh + 2 * n_kv) * hd)) * 2.0 ** rng.integers(-3, 4, (rows, 1))).astype(np.float32)
    ang = rng.uniform(-4, 4, (rows, max(rope_dim // 2, 1)))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    if not rope_dim:
        cos, sin = np.zeros((rows, 0), np.float32), np.zeros((rows, 0), np.float32)
    qn, kn = (rng.normal(1, 0.2, hd).astype(np.float32) for _ in range(2)) if norm else (None, None)
    was = copy.deepcopy(pg)
    eps = float(np.float32(1e-5))
    q, q0 = run_store(native, pg, qkv, n_new, new, nh, rope_dim, split, cos, sin, qn, kn, eps, qt)
    assert pg.status() == 0
    y, err = rope_reference(qkv, cos, sin, nh, n_kv, hd, rope_dim, split, qn, kn, eps)
    for s, m in enumerate(new):
        r = slice(s * n_new, s * n_new + m)
        want, tol = y[r, :nh].reshape(m, nh * hd), err[r, :nh].reshape(m, nh * hd)
        assert (np.abs(value(q[r], qt) - want) <= tol + HALF_STEP[qt] * (np.abs(want) + tol) + 2.0 ** -25).all()
        assert (q[s * n_new + m:(s + 1) * n_new] == q0[s * n_new + m:(s + 1) * n_new]).all()
        if m:
            check_stored(pg, was, s, lens[s] - m, "k", y[r, nh:nh + n_kv], False)
            check_stored(pg, was, s, lens[s] - m, "v", qkv[r].reshape(m, -1, hd)[:, nh + n_kv:].astype(np.float64), True)
    for name in ("k", "v", "ke", "ve"):
        assert (getattr(pg, name) == getattr(was, name)).all(), name


@pytest.mark.parametrize("hd,norm,split,rope_dim", [(64, False, False, 64), (128, True, True, 128), (128, True, False, 64)])
def test_store_gives_the_16_bit_stores_q_rows(native, hd, norm, split, rope_dim):
    from test_gpu_serving import Pages, run_rope
    rng = np.random.default_rng(4)
    nh, n_kv, lens, new = 8, 2, [40, 21], [7, 21]
    qkv = rng.normal(0, 2, (2 * 21, (nh + 2 * n_kv) * hd)).astype(np.float32)
    ang = rng.uniform(-4, 4, (42, rope_dim // 2))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    qn, kn = (rng.normal(1, 0.2, hd).astype(np.float32) for _ in range(2)) if norm else (None, None)
    pg = Pages(rng, lens, 16, n_kv, hd, F16)
    want, _ = run_rope(native, pg, qkv, 21, new, nh, rope_dim, split, cos, sin, qn, kn, 1e-6, F32)
    p8 = Pages8(rng, lens, 16, n_kv, hd, I8)
    got, _ = run_store(native, p8, qkv, 21, new, nh, rope_dim, split, cos, sin, qn, kn, 1e-6, F32)
    assert (got.view(np.uint32) == want.view(np.uint32)).all()


@pytest.mark.parametrize("kv", [I8, E4M3])
def test_store_token_by_token(native, kv):
    """A block filled token by token has the exponents of one filled at once; e4m3 elements are the same
    numbers unless subnormal, int8 ones less than one step off."""
    rng = np.random.default_rng(6)
    nh, n_kv, hd, n = 2, 2, 64, 40
    x = (rng.normal(0, 1, (n, (nh + 2 * n_kv) * hd)) * 2.0 ** (np.arange(n)[:, None] / 3.0)).astype(np.float32)
    one, zero = np.ones((n, 32), np.float32), np.zeros((n, 32), np.float32)
    at_once = Pages8(rng, [n], 16, n_kv, hd, kv, fill=False)
    run_store(native, at_once, x, n, [n], nh, 64, False, one, zero, None, None, 0.0, F32)
    steps = Pages8(rng, [n], 16, n_kv, hd, kv, fill=False)
    for t in range(n):
        steps.lens = np.array([t + 1], np.uint32)
        run_store(native, steps, x[t:t + 1], 1, [1], nh, 64, False, one[:1], zero[:1], None, None, 0.0, F32)
    pos = np.arange(n)
    for name in ("k", "v"):
        e = at_once.exp_bytes(0, pos, name)
        assert (steps.exp_bytes(0, pos, name) == e).all() and len(set(e[:, 0])) == 3
        off = np.abs(steps.get(0, pos, name) - at_once.get(0, pos, name)) / 2.0 ** (e.astype(np.float64) - 127)[..., None]
        if kv == I8:
            assert off.max() <= 1.0
        else:  # a subnormal's step is 2^-9
            small = np.abs(numbers(at_once.raw(0, pos, name), kv)) < 2.0 ** -6
            assert (off[~small] == 0).all() and off.max() <= 2.0 ** -9


@pytest.mark.parametrize("kv", [I8, E4M3])
def test_store_of_odd_numbers(native, kv):
    """Zeros, subnormals, the ends of f32, ties; infinity and NaN take their block and no other with them."""
    import copy
    rng = np.random.default_rng(8)
    nh, n_kv, hd, n = 2, 2, 128, 160
    x = np.zeros((n, nh + 2 * n_kv, hd), np.float32)
    kinds = [0.0, 1e-45, 2.0 ** -130, 1e-30, 3.4028235e38, 1.9 * 2.0 ** 126, 1.0]
    for b, size in enumerate(kinds):
        x[16 * b:16 * b + 16] = (np.clip(rng.normal(0, 0.4, (16, nh + 2 * n_kv, hd)), -1, 1) * size).astype(np.float32)
        x[16 * b + 3, :, 5] = size
    ties = np.arange(-64, 64) + 0.5
    x[112:128] = ties                      # int8: half a step each
    x[113, :, 0] = 127.0
    x[128:144] = 1.0
    x[130, nh + 1, 7] = np.inf             # K of head 1
    x[131, nh + n_kv, 9] = np.nan          # V of head 0
    x[144:] = 2.0
    one, zero = np.ones((n, hd // 2), np.float32), np.zeros((n, hd // 2), np.float32)
    pg = Pages8(rng, [n], 32, n_kv, hd, kv, fill=False)
    was = copy.deepcopy(pg)
    x = x.reshape(n, -1)
    run_store(native, pg, x, n, [n], nh, hd, True, one, zero, None, None, 0.0, F32)
    y = x.reshape(n, -1, hd).astype(np.float64)
    with np.errstate(invalid="ignore"):
        check_stored(pg, was, 0, 0, "k", y[:, nh:nh + n_kv], True)
        check_stored(pg, was, 0, 0, "v", y[:, nh + n_kv:], True)
    bad_k, bad_v = np.isnan(pg.get(0, np.arange(n), "k")), np.isnan(pg.get(0, np.arange(n), "v"))
    assert bad_k[128:144, 1].all() and bad_v[128:144, 0].all()
    bad_k[128:144, 1] = bad_v[128:144, 0] = False
    assert not bad_k.any() and not bad_v.any()


def test_store_bad_pages_and_lengths(native):
    import copy
    rng = np.random.default_rng(5)
    nh, n_kv, hd, ps = 4, 2, 64, 16
    pg = Pages8(rng, [17, 30, 12, 3, 5], ps, n_kv, hd, I8)
    pg.lens = np.array([17, 30, 200, 3, 5], np.uint32)
    new = [2, 4, 1, 4, 2]
    pg.table[0, 1] = pg.n_pages          # position 16 of sequence 0; position 15 is in page 0
    pg.table[1, 0] = 0xFFFFFFFF          # not needed by positions 26 .. 29
    rows = 5 * 4
    qkv = rng.normal(0, 1, (rows, (nh + 2 * n_kv) * hd)).astype(np.float32)
    cos, sin = np.ones((rows, 32), np.float32), np.zeros((rows, 32), np.float32)
    was = copy.deepcopy(pg)
    q, q0 = run_store(native, pg, qkv, 4, new, nh, 64, False, cos, sin, None, None, 0.0, F32)
    assert pg.status() == 3
    assert (q[:2] == qkv[:2, :nh * hd]).all() and (q[4:8] == qkv[4:8, :nh * hd]).all()
    assert (q[8:16] == 7).all()          # a length past the table; more new tokens than positions
    x = qkv.reshape(rows, -1, hd).astype(np.float64)
    for s, first, r in ((0, 15, [0]), (1, 26, [4, 5, 6, 7]), (4, 3, [16, 17])):
        check_stored(pg, was, s, first, "k", x[r, nh:nh + n_kv], True)
        check_stored(pg, was, s, first, "v", x[r, nh + n_kv:], True)
    for name in ("k", "v", "ke", "ve"):
        assert (getattr(pg, name) == getattr(was, name)).all(), name


# ------------------------------------------------------------------------------------------- reading back
@pytest.mark.parametrize("hd,n_kv,ps,kv,t,n_out", [(64, 3, 16, I8, F32, 100), (128, 2, 64, E4M3, F16, 33),
                                                   (256, 1, 32, I8, BF16, 200), (128, 4, 16, E4M3, F32, 64)])
def test_read_exact(native, hd, n_kv, ps, kv, t, n_out):
    rng = np.random.default_rng(hd + n_out)
    lens = [90, 0, 17, 64, 1]
    pg = Pages8(rng, lens, ps, n_kv, hd, kv)
    pg.exps("v")[pg.table[2, 0], 0, 0] = 255    # NaN
    pg.exps("k")[pg.table[3, 0], 0, 0] = 0      # 2^-127
    pg.table[0, 80 // ps] = pg.n_pages + 5
    pg.upload()
    out0 = np.full((len(lens), n_kv, n_out, hd), 7, np.float32 if t == F32 else np.uint16)
    dk, dv = _dev(out0), _dev(out0)
    _ok(native.camelid_hip_paged8_read(pg.dk.ptr, pg.dv.ptr, pg.dke.ptr, pg.dve.ptr, kv, pg.n_pages, ps, n_kv, hd,
                                       pg.dt.ptr, pg.stride, pg.dl.ptr, len(lens), dk.ptr, dv.ptr, t, n_out,
                                       pg.dstat.ptr, None))
    assert pg.status() == (1 if n_out > 80 // ps * ps else 0)
    for name, dev in (("k", dk), ("v", dv)):
        got = dev.download(out0.dtype, out0.size).reshape(out0.shape)
        for s, n in enumerate(lens):
            n = min(n, n_out)
            good = np.array([p for p in range(n) if pg.table[s, p // ps] < pg.n_pages], int)
            want = pg.get(s, good, name).transpose(1, 0, 2)
            have = value(got[s][:, good], t)
            # up to 8 bits and a power of two: exact in every type (f16 down to 2^-24)
            near = np.abs(have - want) <= (2.0 ** -25 if t == F16 else 0)
            assert (near | (np.isnan(have) & np.isnan(want))).all(), (name, s)
            rest = np.setdiff1d(np.arange(n_out), good)
            assert (got[s][:, rest] == 7).all()


# ------------------------------------------------------------------------------------------- attention
def attention8_reference(pg, q, qt, n_new, new, nh, scale, bad=(), one_term=False):
    """(rows, bounds) in 64 bits; None for padding rows.  bad: (sequence, position) pairs that count as masked."""
    g, hd = nh // pg.n_kv, pg.hd
    out = [None] * len(q)
    for s, m in enumerate(new):
        n = int(pg.lens[s])
        if m == 0:
            continue
        pos = np.arange(n)
        k, v, ve = pg.get(s, pos, "k"), pg.get(s, pos, "v"), 2.0 ** (pg.exp_bytes(s, pos, "v").astype(np.float64) - 127)
        ok = np.array([(s, p) not in bad for p in range(n)])
        x = value(q[s * n_new:s * n_new + m], qt).reshape(m, nh, hd)
        rows, tols = np.zeros((m, nh, hd)), np.zeros((m, nh, hd))
        with np.errstate(invalid="ignore", over="ignore"):
            for t in range(m):
                see = np.nonzero(ok[:n - m + t + 1])[0]
                if not len(see):
                    continue
                for h in range(pg.n_kv):
                    xs, kk, vv = x[t, h * g:(h + 1) * g], k[see, h], v[see, h]
                    sc = xs @ kk.T * scale
                    d = (((hd + 8) * U + (2.0 ** -21 if qt == F32 else 0)) * abs(scale) *
                         (np.abs(xs) @ np.abs(kk).T).max(-1, keepdims=True))
                    p = np.exp(sc - sc.max(-1, keepdims=True))
                    p /= p.sum(-1, keepdims=True)
                    rel = np.expm1(2 * d) + (2.0 ** -11 if one_term else 2.0 ** -21) + 2.0 ** -20
                    chain = (len(see) / 32 + 64) * U
                    rows[t, h * g:(h + 1) * g] = p @ vv
                    least = 2.0 ** -38 * 448 * len(see) * (p * ve[see, h]).max(-1, keepdims=True)
                    tols[t, h * g:(h + 1) * g] = (rel + 2 * chain) * (p @ np.abs(vv)) + least
        for t in range(m):
            out[s * n_new + t] = (rows[t].reshape(-1), tols[t].reshape(-1))
    return out


def attention8_buffers(native, pg, q, n_new, new, nh, q_pad=0, out_pad=0):
    rows, width = pg.n * n_new, nh * pg.hd
    qp = np.full((rows, width + q_pad), 3 if q.dtype == np.float32 else 0x4000, q.dtype)
    qp[:, :width] = q
    out0 = np.full((rows, width + out_pad), 7, q.dtype)
    size = native.camelid_hip_paged8_attention_workspace(pg.n, n_new, nh, pg.n_kv, pg.hd, pg.ps, pg.stride)
    return dict(q=_dev(qp), out=_dev(out0), new=_dev(np.array(new, np.uint32)), ws=_dev(np.full(size + 64, 0xEE, np.uint8)),
                size=size, out0=out0)


def call_attention8(native, pg, b, qt, n_new, nh, scale, q_stride, out_stride, stream=None):
    _ok(native.camelid_hip_paged8_attention(
        b["q"].ptr, qt, q_stride, pg.n, n_new, b["new"].ptr, nh, pg.n_kv, pg.hd, pg.dk.ptr, pg.dv.ptr, pg.dke.ptr,
        pg.dve.ptr, pg.kv, pg.n_pages, pg.ps, pg.dt.ptr, pg.stride, pg.dl.ptr, scale, b["out"].ptr, out_stride,
        b["ws"].ptr, b["size"], pg.dstat.ptr, stream))


def run_attention8(native, pg, q, qt, n_new, new, nh, scale, q_pad=0, out_pad=0, upload=True):
    if upload:
        pg.upload()
    width = nh * pg.hd
    b = attention8_buffers(native, pg, q, n_new, new, nh, q_pad, out_pad)
    call_attention8(native, pg, b, qt, n_new, nh, scale, width + q_pad, width + out_pad)
    out = b["out"].download(b["out0"].dtype, b["out0"].size).reshape(b["out0"].shape)
    assert (out[:, width:] == 7).all()
    assert (b["ws"].download(np.uint8, b["size"] + 64)[b["size"]:] == 0xEE).all()
    return out[:, :width]


def check_attention8(out, ref, qt):
    for r, want in enumerate(ref):
        if want is None:
            assert (out[r] == 7).all(), r
            continue
        got, (y, tol) = value(out[r], qt), want
        near = np.abs(got - y) <= tol + HALF_STEP[qt] * (np.abs(y) + tol) + (2.0 ** -25 if qt == F16 else 0)
        assert (near | (np.isnan(got) & np.isnan(y))).all(), (r, np.nanmax(np.abs(got - y)), tol.max())


ATT8_CASES = [
    # nh, n_kv, hd, lens, new, page, q type, kv type
    (32, 4, 64, [127], [1], 16, F32, I8),
    (8, 8, 128, [1], [1], 16, F32, E4M3),
    (32, 8, 128, [1, 15, 16, 17, 0, 63, 64, 65, 257], [1, 1, 1, 1, 0, 1, 1, 1, 1], 16, F32, I8),
    (24, 8, 128, [5, 64, 300, 0], [5, 8, 1, 0], 32, F16, E4M3),
    (32, 8, 128, [1100, 7, 700], [5, 2, 3], 64, BF16, I8),
    (14, 2, 64, [8, 1025, 513], [8, 1, 7], 16, BF16, E4M3),
    (4, 1, 256, [90, 2049], [3, 1], 128, F32, E4M3),
    (6, 6, 256, [40, 555], [1, 8], 256, F16, I8),
    (64, 2, 64, [600, 77], [8, 1], 16, F16, I8),
    (40, 8, 128, [4100], [1], 16, BF16, E4M3),
    (32, 8, 128, [5003], [1], 4096, F32, I8),
    (71, 1, 64, [333, 12], [2, 8], 32, F32, E4M3),
    (4, 2, 64, [i * 37 % 400 for i in range(150)], [min(i * 37 % 400, i % 4) for i in range(150)], 16, F32, I8),
    (4, 2, 128, [40000], [1], 16, F32, I8),
    (1, 1, 128, [300], [1], 32, BF16, I8),
]


@pytest.mark.parametrize("nh,n_kv,hd,lens,new,ps,qt,kv", ATT8_CASES)
def test_attention8_against_64_bits(native, nh, n_kv, hd, lens, new, ps, qt, kv):
    rng = np.random.default_rng(nh * 7 + hd + len(lens))
    pg = Pages8(rng, lens, ps, n_kv, hd, kv)
    n_new = max(new)
    q = typed(rng.normal(0, 1.7, (len(lens) * n_new, nh * hd)), qt)
    scale = float(np.float32(1 / math.sqrt(hd)))
    out = run_attention8(native, pg, q, qt, n_new, new, nh, scale, q_pad=16, out_pad=8)
    assert pg.status() == 0
    check_attention8(out, attention8_reference(pg, q, qt, n_new, new, nh, scale), qt)


PROMPT_CASES = [
    # nh, n_kv, hd, lens, new, page, q type, kv type
    (8, 2, 128, [200], [200], 16, F32, I8),
    (8, 8, 128, [300, 0, 129, 1], [130, 0, 129, 1], 64, BF16, E4M3),
    (32, 4, 64, [75, 1300, 16], [75, 40, 3], 32, F16, I8),
    (6, 3, 64, [140, 700], [100, 69], 16, F32, E4M3),
    (4, 2, 256, [333, 90], [70, 90], 128, BF16, I8),
    (2, 1, 256, [150], [64], 256, F32, E4M3),
    (71, 1, 64, [60, 9], [2, 9], 32, F16, E4M3),
    (2, 2, 128, [60, 700, 30], [9, 64, 30], 32, BF16, E4M3),
    (4, 1, 128, [9000], [33], 16, F16, I8),
    (1, 1, 128, [4000], [130], 16, F32, I8),
]


@pytest.mark.parametrize("nh,n_kv,hd,lens,new,ps,qt,kv", PROMPT_CASES)
def test_prompts8_against_64_bits(native, nh, n_kv, hd, lens, new, ps, qt, kv):
    rng = np.random.default_rng(nh * 7 + hd + len(lens))
    pg = Pages8(rng, lens, ps, n_kv, hd, kv)
    n_new = max(new)
    q = typed(rng.normal(0, 1.7, (len(lens) * n_new, nh * hd)), qt)
    scale = float(np.float32(1 / math.sqrt(hd)))
    out = run_attention8(native, pg, q, qt, n_new, new, nh, scale, q_pad=16, out_pad=8)
    assert pg.status() == 0
    check_attention8(out, attention8_reference(pg, q, qt, n_new, new, nh, scale, one_term=qt != F32 and n_new > 8), qt)
