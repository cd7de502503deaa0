"""Batched serving over a paged cache on the GPU, each entry point against a plain evaluation of its
definition in 64 bits.

Tolerances.  u = 2^-24 is half an f32 step, e = finfo(type).eps / 2 half a step of a 16-bit output.
 * RoPE: two rounded products and one rounded sum: 3 u (|a c| + |b s|); behind an RMSNorm whose sum
   takes hd roundings, (hd + 8) u relative more.
 * Attention: a score is a sum of hd products, (hd + 8) u sum |q_d k_d| scale off at most, 2^-21 of it
   more where f32 queries go through pairs of 16-bit numbers (2^-22 each); a weight is then
   exp(+-2 d) - 1 off relatively (numerator and sum), 2^-16 more for its own rounding to a pair of 16-bit
   numbers in a 16-bit type (2^-21 for f32 outputs), and 2^-22 for the exponential.  Sums run in chains of
   n / 32 + 64 (32 positions a matrix instruction).  All against sum_p w_p |v_p|, plus e |result| for
   the final rounding and half the smallest f16 step.
 * Moves, indexes and tokens are exact.  Log-probabilities: f64, rounded once, 2 u relative."""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2
U = 2.0 ** -24
HALF_STEP = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}
NONE = 0xFFFFFFFF


def _dev(a):
    from camelid_amd.engine import DeviceBuffer
    return DeviceBuffer.from_array(np.ascontiguousarray(a))


def _buf(nbytes):
    from camelid_amd.engine import DeviceBuffer
    return DeviceBuffer(nbytes)


def _ok(rc):
    from camelid_amd._native import check
    check(rc)


def to16(x, t):
    """f32 values -> bits of the 16-bit type, to nearest even."""
    x = np.ascontiguousarray(x, np.float32)
    if t == F16:
        return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32).astype(np.uint64)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def from16(b, t):
    b = np.ascontiguousarray(b, np.uint16)
    if t == F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def typed(x, t):
    return np.ascontiguousarray(x, np.float32) if t == F32 else to16(x, t)


def value(b, t):
    return b.astype(np.float64) if t == F32 else from16(b, t)


class Pages:
    """A cache on the host: pages in random order, bits of everything nobody owns planted NaNs."""

    def __init__(self, rng, lens, ps, n_kv, hd, kv, spare=2, extra_stride=1, rows=None):
        self.ps, self.n_kv, self.hd, self.kv, self.n = ps, n_kv, hd, kv, len(lens)
        self.lens = np.array(lens, np.uint32)
        self.stride = max(1, -(-int(max(lens)) // ps)) + extra_stride
        self.n_pages = self.n * self.stride + spare
        self.table = rng.permutation(self.n_pages)[:self.n * self.stride].astype(np.uint32).reshape(self.n, self.stride)
        nan = {F16: 0x7E01, BF16: 0x7FC1}[kv]
        self.k = np.full((self.n_pages, n_kv, hd * ps), nan, np.uint16)
        self.v = np.full((self.n_pages, n_kv, hd * ps), nan, np.uint16)
        for s, n in enumerate(lens):
            if n:
                make = rows or (lambda *sh: rng.normal(0, 1, sh))
                self.set(s, np.arange(n), to16(make(n, n_kv, hd), kv), to16(make(n, n_kv, hd), kv))

    def cells(self, s, pos):
        pos = np.asarray(pos)
        page = self.table[s][pos // self.ps].astype(np.int64)[:, None, None]
        o = (pos % self.ps)[:, None, None]
        h, d = np.arange(self.n_kv)[:, None], np.arange(self.hd)[None]
        base = (page * self.n_kv + h) * (self.hd * self.ps)
        return base + (d // 8 * self.ps + o) * 8 + d % 8, base + (o // 8 * self.hd + d) * 8 + o % 8

    def set(self, s, pos, k, v):
        ik, iv = self.cells(s, pos)
        self.k.reshape(-1)[ik] = k
        self.v.reshape(-1)[iv] = v

    def get(self, s, pos):
        ik, iv = self.cells(s, pos)
        return self.k.reshape(-1)[ik], self.v.reshape(-1)[iv]

    @property
    def cap(self):
        return self.stride * self.ps

    def upload(self):
        self.dk, self.dv, self.dt, self.dl = _dev(self.k), _dev(self.v), _dev(self.table), _dev(self.lens)
        self.dstat = _dev(np.zeros(1, np.uint32))

    def download(self):
        self.k = self.dk.download(np.uint16, self.k.size).reshape(self.k.shape)
        self.v = self.dv.download(np.uint16, self.v.size).reshape(self.v.shape)

    def status(self):
        return int(self.dstat.download(np.uint32, 1)[0])


# --------------------------------------------------------------------------------------- RoPE + store
def rope_reference(qkv, cos, sin, nh, n_kv, hd, rope_dim, split, qn, kn, eps):
    """(q, k, v) rows in 64 bits and the bounds of their f32 evaluation."""
    x = qkv.astype(np.float64).reshape(len(qkv), nh + 2 * n_kv, hd)
    y, err = x.copy(), np.zeros_like(x)
    half = rope_dim // 2
    for a, b, w in ((0, nh, qn), (nh, nh + n_kv, kn)):
        z, rel = x[:, a:b], 0.0
        if w is not None:
            z = z / np.sqrt((z * z).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
            rel = (hd + 8) * U
        y[:, a:b], err[:, a:b] = z, rel * np.abs(z)
        lo, hi = (slice(0, half), slice(half, rope_dim)) if split else (slice(0, rope_dim, 2), slice(1, rope_dim, 2))
        c, s = cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
        p, q = z[..., lo], z[..., hi]
        out, e = y[:, a:b].copy(), err[:, a:b].copy()
        out[..., lo], out[..., hi] = p * c - q * s, p * s + q * c
        e[..., lo] = (3 * U + rel) * (np.abs(p * c) + np.abs(q * s))
        e[..., hi] = (3 * U + rel) * (np.abs(p * s) + np.abs(q * c))
        y[:, a:b], err[:, a:b] = out, e
    return y, err


def run_rope(native, pg, qkv, n_new, new, nh, rope_dim, split, cos, sin, qn, kn, eps, qt):
    pg.upload()
    rows = pg.n * n_new
    q0 = np.full((rows, nh * pg.hd), 7, np.float32 if qt == F32 else np.uint16)
    dq = _dev(q0)
    dn = [_dev(w) if w is not None else None for w in (qn, kn)]
    bufs = _dev(qkv), _dev(cos), _dev(sin), _dev(np.array(new, np.uint32))
    _ok(native.camelid_hip_paged_rope_kv(
        bufs[0].ptr, pg.n, n_new, bufs[3].ptr, nh, pg.n_kv, pg.hd, rope_dim, int(split), bufs[1].ptr, bufs[2].ptr,
        dn[0].ptr if dn[0] else None, dn[1].ptr if dn[1] else None, eps, dq.ptr, qt, pg.dk.ptr, pg.dv.ptr, pg.kv,
        pg.n_pages, pg.ps, pg.dt.ptr, pg.stride, pg.dl.ptr, pg.dstat.ptr, None))
    q = dq.download(q0.dtype, q0.size).reshape(q0.shape)
    pg.download()
    return q, q0


ROPE_CASES = [
    # nh, n_kv, hd, rope_dim, split, norm, lens, new, page, q type, kv type
    (32, 4, 64, 64, False, False, [128], [1], 16, F32, F16),
    (8, 8, 128, 128, True, True, [1, 9, 8, 300], [1, 5, 0, 3], 32, BF16, BF16),
    (24, 8, 128, 96, False, False, [70, 33], [70, 1], 8, F16, F16),
    (4, 2, 256, 256, True, True, [40, 17], [13, 17], 256, F32, BF16),
    (2, 1, 64, 0, False, True, [11], [3], 8, F32, F16),
    (16, 2, 64, 64, True, False, [65, 1, 64], [64, 1, 33], 64, BF16, BF16),
]


@pytest.mark.parametrize("nh,n_kv,hd,rope_dim,split,norm,lens,new,ps,qt,kv", ROPE_CASES)
def test_rope_kv_against_64_bits(native, nh, n_kv, hd, rope_dim, split, norm, lens, new, ps, qt, kv):
    rng = np.random.default_rng(hd + nh + ps)
    pg = Pages(rng, lens, ps, n_kv, hd, kv)
    n_new = max(new)
    rows = len(lens) * n_new
    qkv = rng.normal(0, 1.5, (rows, (nh + 2 * n_kv) * hd)).astype(np.float32)
    ang = rng.uniform(-4, 4, (rows, max(rope_dim // 2, 1)))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    if not rope_dim:
        cos, sin = np.zeros((rows, 0), np.float32), np.zeros((rows, 0), np.float32)
    qn, kn = (rng.normal(1, 0.2, hd).astype(np.float32) for _ in range(2)) if norm else (None, None)
    k0, v0 = pg.k.copy(), pg.v.copy()
    q, q0 = run_rope(native, pg, qkv, n_new, new, nh, rope_dim, split, cos, sin, qn, kn, 1e-5, qt)
    assert pg.status() == 0
    y, err = rope_reference(qkv, cos, sin, nh, n_kv, hd, rope_dim, split, qn, kn, 1e-5)
    for s, m in enumerate(new):
        r = slice(s * n_new, s * n_new + m)
        want, tol = y[r, :nh].reshape(m, nh * hd), err[r, :nh].reshape(m, nh * hd)
        assert (np.abs(value(q[r], qt) - want) <= tol + HALF_STEP[qt] * (np.abs(want) + tol) + 2.0 ** -25).all()
        assert (q[s * n_new + m:(s + 1) * n_new] == q0[s * n_new + m:(s + 1) * n_new]).all()
        pos = np.arange(lens[s] - m, lens[s])
        if m:
            gk, gv = pg.get(s, pos)
            want, tol = y[r, nh:nh + n_kv], err[r, nh:nh + n_kv]
            assert (np.abs(from16(gk, kv) - want) <= tol + HALF_STEP[kv] * (np.abs(want) + tol) + 2.0 ** -25).all()
            assert (gv == to16(qkv[r].reshape(m, -1, hd)[:, nh + n_kv:], kv)).all()
            ik, iv = pg.cells(s, pos)  # everything else keeps its bits
            k0.reshape(-1)[ik], v0.reshape(-1)[iv] = gk, gv
    assert (pg.k == k0).all() and (pg.v == v0).all()


@pytest.mark.parametrize("norm,split,hd", [(False, False, 64), (True, True, 128), (True, False, 128)])
def test_rope_kv_bits_equal_the_contiguous_store(native, norm, split, hd):
    """f32 q rows and an f16 cache hold camelid_hip_rope_kv's bits."""
    rng = np.random.default_rng(3)
    nh, n_kv, n, max_pos, pos = 8, 2, 5, 40, 30
    qkv = rng.normal(0, 2, (n, (nh + 2 * n_kv) * hd)).astype(np.float32)
    ang = rng.uniform(-4, 4, (n, hd // 2))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    qn, kn = (rng.normal(1, 0.2, hd).astype(np.float32) for _ in range(2)) if norm else (None, None)
    pg = Pages(rng, [pos + n], 16, n_kv, hd, F16)
    q, _ = run_rope(native, pg, qkv, n, [n], nh, hd, split, cos, sin, qn, kn, 1e-6, F32)
    kc, vc, dq = _dev(np.zeros(n_kv * hd * max_pos, np.uint16)), _dev(np.zeros(n_kv * hd * max_pos, np.uint16)), \
        _buf(nh * hd * 4)
    dn = [_dev(w) if norm else None for w in (qn, kn)]
    for t in range(n):
        row = _dev(qkv[t]), _dev(cos[t]), _dev(sin[t]), _dev(np.array([pos + t], np.uint32))
        _ok(native.camelid_hip_rope_kv(row[0].ptr, nh, n_kv, hd, hd, int(split), row[1].ptr, row[2].ptr,
                                       dn[0].ptr if norm else None, dn[1].ptr if norm else None, 1e-6, dq.ptr, kc.ptr,
                                       vc.ptr, 0, max_pos, row[3].ptr, None))
        assert (dq.download(np.uint32, nh * hd) == q[t].view(np.uint32)).all()
    k = kc.download(np.uint16, n_kv * hd * max_pos).reshape(n_kv, hd // 8, max_pos, 8)
    v = vc.download(np.uint16, n_kv * hd * max_pos).reshape(n_kv, max_pos // 8, hd, 8)
    gk, gv = pg.get(0, np.arange(pos, pos + n))
    assert (gk == k.transpose(2, 0, 1, 3).reshape(max_pos, n_kv, hd)[pos:pos + n]).all()
    assert (gv == v.transpose(1, 3, 0, 2).reshape(max_pos, n_kv, hd)[pos:pos + n]).all()


def test_rope_kv_bad_pages_and_lengths(native):
    """Errors only the device sees: reported, the rest of the call done, no other memory touched."""
    rng = np.random.default_rng(5)
    nh, n_kv, hd, ps = 4, 2, 64, 8
    lens, new = [9, 12, 200, 3, 5], [2, 4, 1, 4, 2]
    pg = Pages(rng, [9, 12, 12, 3, 5], ps, n_kv, hd, F16)
    pg.lens = np.array(lens, np.uint32)
    pg.table[0, 1] = pg.n_pages          # position 8 of sequence 0; position 7 is in page 0
    pg.table[1, 0] = 0xFFFFFFFF          # not needed by positions 8 .. 11
    rows = 5 * 4
    qkv = rng.normal(0, 1, (rows, (nh + 2 * n_kv) * hd)).astype(np.float32)
    cos, sin = np.ones((rows, 32), np.float32), np.zeros((rows, 32), np.float32)
    k0, v0 = pg.k.copy(), pg.v.copy()
    q, q0 = run_rope(native, pg, qkv, 4, new, nh, 64, False, cos, sin, None, None, 0.0, F32)
    assert pg.status() == 3
    x = qkv.reshape(rows, -1, hd)
    assert (q[:2] == qkv[:2, :nh * hd]).all() and (q[4:8] == qkv[4:8, :nh * hd]).all()
    assert (q[8:16] == 7).all()          # a length past the table; more new tokens than positions
    for s, pos, r in ((0, [7], [0]), (1, [8, 9, 10, 11], [4, 5, 6, 7]), (4, [3, 4], [16, 17])):
        gk, gv = pg.get(s, pos)
        assert (gk == to16(x[r, nh:nh + n_kv], F16)).all() and (gv == to16(x[r, nh + n_kv:], F16)).all()
        ik, iv = pg.cells(s, pos)
        k0.reshape(-1)[ik], v0.reshape(-1)[iv] = gk, gv
    assert (pg.k == k0).all() and (pg.v == v0).all()


# ------------------------------------------------------------------------------------------- attention
def attention_reference(pg, q, qt, n_new, new, nh, scale, weights, bad=()):
    """(rows, bounds, weights, their bounds) in 64 bits; None for padding rows.  bad: (sequence,
    position) pairs that count as masked."""
    g, hd = nh // pg.n_kv, pg.hd
    out = [None] * len(q)
    w = None if weights is None else weights.astype(np.float64)
    werr = None if weights is None else np.zeros_like(w)
    pair = 2.0 ** -21 if qt == F32 else 2.0 ** -16
    for s, m in enumerate(new):
        n = int(pg.lens[s])
        if m == 0:
            continue
        if w is not None:
            w[s, :, n - m:n] = 0
        kb, vb = pg.get(s, np.arange(n))
        k, v = from16(kb, pg.kv), from16(vb, pg.kv)
        ok = np.array([(s, p) not in bad for p in range(n)])
        for t in range(m):
            c = n - m + t + 1
            x = value(q[s * n_new + t], qt).reshape(nh, hd)
            rows, tols = np.zeros((nh, hd)), np.zeros((nh, hd))
            for h in range(pg.n_kv):
                see = np.nonzero(ok[:c])[0]
                if not len(see):
                    continue
                xs = x[h * g:(h + 1) * g]
                with np.errstate(invalid="ignore", over="ignore"):
                    kk, vv = k[see, h], v[see, h]
                    sc = xs @ kk.T * scale
                    d = (((hd + 8) * U + (2.0 ** -21 if qt == F32 else 0)) * abs(scale) *
                         (np.abs(xs) @ np.abs(kk).T).max(-1, keepdims=True))
                    p = np.exp(sc - sc.max(-1, keepdims=True))
                    p /= p.sum(-1, keepdims=True)
                    rel = np.expm1(2 * d) + pair + 2.0 ** -22
                    chain = (len(see) / 32 + 64) * U
                    rows[h * g:(h + 1) * g] = p @ vv
                    tols[h * g:(h + 1) * g] = (rel + 2 * chain) * (p @ np.abs(vv))
                if w is not None:
                    w[s, h, see] += p.sum(0)
                    werr[s, h, see] += ((rel + chain) * p).sum(0)
            out[s * n_new + t] = (rows.reshape(-1), tols.reshape(-1))
    if w is not None:
        werr += 16 * U * np.abs(w)
    return out, w, werr


def run_attention(native, pg, q, qt, n_new, new, nh, scale, weights=None, q_pad=0, out_pad=0, upload=True):
    if upload:
        pg.upload()
    rows, width = pg.n * n_new, nh * pg.hd
    qp = np.full((rows, width + q_pad), 3 if qt == F32 else 0x4000, q.dtype)
    qp[:, :width] = q
    out0 = np.full((rows, width + out_pad), 7, q.dtype)
    dq, do, dn = _dev(qp), _dev(out0), _dev(np.array(new, np.uint32))
    dw = _dev(weights) if weights is not None else None
    size = native.camelid_hip_paged_attention_workspace(pg.n, n_new, nh, pg.n_kv, pg.hd, pg.ps, pg.stride,
                                                        int(weights is not None))
    ws = _dev(np.full(size + 64, 0xEE, np.uint8))
    _ok(native.camelid_hip_paged_attention(
        dq.ptr, qt, width + q_pad, pg.n, n_new, dn.ptr, nh, pg.n_kv, pg.hd, pg.dk.ptr, pg.dv.ptr, pg.kv, pg.n_pages,
        pg.ps, pg.dt.ptr, pg.stride, pg.dl.ptr, scale, do.ptr, width + out_pad, dw.ptr if dw else None, ws.ptr, size,
        pg.dstat.ptr, None))
    out = do.download(out0.dtype, out0.size).reshape(out0.shape)
    assert (out[:, width:] == 7).all()
    assert (ws.download(np.uint8, size + 64)[size:] == 0xEE).all()
    got_w = dw.download(np.float32, weights.size).reshape(weights.shape) if dw else None
    return out[:, :width], got_w


def check_attention(out, got_w, ref, weights, pg, n_new, new, qt):
    rows, w, werr = ref
    for r, want in enumerate(rows):
        if want is None:
            assert (out[r] == 7).all(), r
            continue
        got = value(out[r], qt)
        y, tol = want
        near = np.abs(got - y) <= tol + HALF_STEP[qt] * (np.abs(y) + tol) + 2.0 ** -25
        assert near.all(), (r, np.abs(got - y).max(), tol.max())
    if w is not None:
        for s in range(pg.n):
            n = int(pg.lens[s])
            assert (np.abs(got_w[s, :, :n] - w[s, :, :n]) <= werr[s, :, :n] + 1e-30).all(), s
            assert (got_w[s, :, n:].view(np.uint32) == weights[s, :, n:].view(np.uint32)).all()


ATT_CASES = [
    # nh, n_kv, hd, lens, new, page, q type, kv type, weights
    (32, 4, 64, [127], [1], 16, F32, F16, False),
    (8, 8, 128, [1], [1], 8, F32, F16, True),
    (32, 8, 128, [1, 31, 32, 33, 0, 257], [1, 1, 1, 1, 0, 1], 8, F32, BF16, True),
    (24, 8, 128, [5, 64, 300, 0], [5, 8, 1, 0], 32, F16, F16, True),
    (32, 8, 128, [1100, 7, 700], [5, 2, 3], 64, F32, F16, True),
    (14, 2, 64, [8, 1025, 513], [8, 1, 7], 16, BF16, BF16, True),
    (4, 1, 256, [90, 2049], [3, 1], 128, F32, F16, False),
    (6, 6, 256, [40, 555], [1, 8], 256, F32, BF16, True),
    (64, 2, 64, [600, 77], [8, 1], 16, F16, F16, False),
    (40, 8, 128, [4100], [1], 16, BF16, BF16, False),
    (32, 8, 128, [5003], [1], 4096, F32, F16, False),
    (71, 1, 64, [333, 12], [2, 8], 32, F32, F16, True),
    (4, 2, 64, [i * 37 % 400 for i in range(150)], [min(i * 37 % 400, i % 4) for i in range(150)], 16, F32, F16, True),
]


@pytest.mark.parametrize("nh,n_kv,hd,lens,new,ps,qt,kv,keep_w", ATT_CASES)
def test_attention_against_64_bits(native, nh, n_kv, hd, lens, new, ps, qt, kv, keep_w):
    rng = np.random.default_rng(nh * 7 + hd + len(lens))
    pg = Pages(rng, lens, ps, n_kv, hd, kv)
    n_new = max(new)
    q = typed(rng.normal(0, 1.7, (len(lens) * n_new, nh * hd)), qt)
    weights = rng.uniform(0, 2, (len(lens), n_kv, pg.cap)).astype(np.float32) if keep_w else None
    scale = 1 / math.sqrt(hd)
    out, got_w = run_attention(native, pg, q, qt, n_new, new, nh, scale, weights, q_pad=16, out_pad=8)
    assert pg.status() == 0
    ref = attention_reference(pg, q, qt, n_new, new, nh, float(np.float32(scale)), weights)
    check_attention(out, got_w, ref, weights, pg, n_new, new, qt)


@pytest.mark.parametrize("qt,kv", [(F32, F16), (BF16, BF16)])
def test_attention_extreme_values(native, qt, kv):
    """Scores far apart, far from zero and tiny; a uniform row; values at the type's ends."""
    rng = np.random.default_rng(9)
    nh, n_kv, hd, lens = 8, 2, 64, [70, 400, 33, 64, 300]
    big = 3e4 if kv == F16 else 1e30
    pg = Pages(rng, lens, 16, n_kv, hd, kv)
    for s, (ks, vs) in enumerate([(30.0, 1.0), (0.0, 1.0), (1e-4, 1e-4), (1.0, big), (5.0, 1.0)]):
        n = lens[s]
        pg.set(s, np.arange(n), to16(rng.normal(0, 1, (n, n_kv, hd)) * ks, kv),
               to16(rng.uniform(-1, 1, (n, n_kv, hd)) * vs, kv))
    q = rng.normal(0, 1, (5, nh * hd))
    q[4] = -np.abs(q[4]) * 4
    kb, vb = pg.get(4, np.arange(300))
    pg.set(4, np.arange(300), to16(np.abs(from16(kb, kv)), kv), vb)  # every score far below zero
    q = typed(q, qt)
    weights = np.zeros((5, n_kv, pg.cap), np.float32)
    out, got_w = run_attention(native, pg, q, qt, 1, [1] * 5, nh, 0.125, weights)
    check_attention(out, got_w, attention_reference(pg, q, qt, 1, [1] * 5, nh, 0.125, weights), weights, pg, 1, [1] * 5,
                    qt)


@pytest.mark.parametrize("qt,kv", [(F32, F16), (F16, F16), (F32, BF16)])
def test_attention_of_tokens_before_a_bad_one(native, qt, kv):
    """Infinities and NaN at a draft's position reach that draft's row and the later ones only."""
    rng = np.random.default_rng(10)
    nh, n_kv, hd, n, m = 8, 2, 128, 45, 5
    inf, nan = (0x7C00, 0x7E00) if kv == F16 else (0x7F80, 0x7FC0)
    for bits_k, bits_v in ((0x3C00, inf), (0x3C00, nan), (nan, 0x3C00), (nan, nan)):
        pg = Pages(rng, [n, n], 8, n_kv, hd, kv)
        kb, vb = pg.get(0, [n - 3])
        kb[0, :, 5], vb[0, :, 7] = bits_k if bits_k != 0x3C00 else kb[0, :, 5], \
            bits_v if bits_v != 0x3C00 else vb[0, :, 7]
        pg.set(0, [n - 3], kb, vb)
        q = typed(rng.normal(0, 1, (2 * m, nh * hd)), qt)
        w = np.zeros((2, n_kv, pg.cap), np.float32)
        out, got_w = run_attention(native, pg, q, qt, m, [m, m], nh, 0.1, w)
        ref, _, _ = attention_reference(pg, q, qt, m, [m, m], nh, float(np.float32(0.1)), None)
        got = value(out, qt)
        for r in list(range(2)) + list(range(m, 2 * m)):  # rows before the bad position; the other sequence
            y, tol = ref[r]
            assert (np.abs(got[r] - y) <= tol + HALF_STEP[qt] * (np.abs(y) + tol) + 2.0 ** -25).all(), r
        for r in range(2, m):
            rows = got[r].reshape(nh, hd)
            if bits_k == nan:
                assert np.isnan(rows).all()
            else:
                assert not np.isfinite(rows[:, 7]).any() and np.isfinite(np.delete(rows, 7, 1)).all()
        assert np.isfinite(got_w[1]).all()


def test_attention_infinite_scores(native):
    """-inf scores weigh nothing beside finite ones, wherever the split falls; a row of nothing else,
    and a +inf score, are NaN as in the formula."""
    rng = np.random.default_rng(12)
    nh, n_kv, hd, lens = 2, 1, 64, [3000, 40, 900]
    pg = Pages(rng, lens, 16, n_kv, hd, BF16)
    big = np.float32(3e38)
    for s, rows in ((0, np.r_[0:2990]), (1, np.r_[0:40]), (2, np.r_[500:501])):
        kb, vb = pg.get(s, rows)
        kb[:, 0, :] = to16(np.full((len(rows), hd), big if s == 2 else -big), BF16)
        pg.set(s, rows, kb, vb)
    q = np.full((3, nh * hd), 2.0, np.float32)
    out, _ = run_attention(native, pg, q, F32, 1, [1] * 3, nh, 1.0)
    kb, vb = pg.get(0, np.arange(2990, 3000))
    sc = 2.0 * from16(kb[:, 0], BF16).sum(-1)
    p = np.exp(sc - sc.max())
    p /= p.sum()
    want = p @ from16(vb[:, 0], BF16)
    assert np.abs(out[0].reshape(2, hd) - want).max() < 1e-4
    assert np.isnan(out[1]).all() and np.isnan(out[2]).all()


def test_attention_bad_pages_and_lengths(native):
    rng = np.random.default_rng(13)
    nh, n_kv, hd, ps = 4, 2, 64, 8
    pg = Pages(rng, [30, 8, 20, 20, 9], ps, n_kv, hd, F16)
    table = pg.table.copy()
    ref_pg = Pages(rng, [30, 8, 20, 20, 9], ps, n_kv, hd, F16)
    ref_pg.__dict__.update({k: v for k, v in pg.__dict__.items()})
    q = typed(rng.normal(0, 1, (10, nh * hd)), F32)
    new = [2, 1, 2, 2, 2]
    w0 = np.zeros((5, n_kv, pg.cap), np.float32)
    bad = {(0, p) for p in range(8, 16)} | {(1, p) for p in range(8)}
    ref = attention_reference(pg, q, F32, 2, new, nh, 0.125, w0, bad)
    pg.table = table.copy()
    pg.table[0, 1], pg.table[1, 0] = pg.n_pages, 0xFFFFFFFF
    pg.lens = np.array([30, 8, pg.cap + 1, 1, 9], np.uint32)
    out, got_w = run_attention(native, pg, q, F32, 2, new, nh, 0.125, w0)
    assert pg.status() == 3
    assert (out[4:8] == 7).all() and (got_w[2:4] == 0).all()   # those sequences are left alone
    assert (out[2] == 0).all()                                 # no position left to attend to
    for r in (0, 1, 8, 9):
        y, tol = ref[0][r]
        assert (np.abs(out[r] - y) <= tol + 2.0 ** -25).all()
    for s in (0, 4):
        assert (np.abs(got_w[s] - ref[1][s]) <= ref[2][s] + 1e-30).all()


def test_attention_same_bits_twice_and_padded_batch(native):
    """The same call gives the same bits, also where a padding sequence stands beside the real ones."""
    rng = np.random.default_rng(14)
    nh, n_kv, hd = 32, 8, 128
    pg = Pages(rng, [900, 0, 4000, 17], 32, n_kv, hd, F16)
    q = typed(rng.normal(0, 1, (8, nh * hd)), F32)
    w = np.zeros((4, n_kv, pg.cap), np.float32)
    a, wa = run_attention(native, pg, q, F32, 2, [2, 0, 1, 2], nh, 0.1, w)
    b, wb = run_attention(native, pg, q, F32, 2, [2, 0, 1, 2], nh, 0.1, w)
    assert (a.view(np.uint32) == b.view(np.uint32)).all() and (wa.view(np.uint32) == wb.view(np.uint32)).all()


def test_attention_agrees_with_the_contiguous_decode(native):
    """One sequence: the same rows as camelid_hip_attention_decode, whose sums run in another order."""
    rng = np.random.default_rng(15)
    nh, n_kv, hd, n = 32, 8, 128, 700
    pg = Pages(rng, [n], 32, n_kv, hd, F16)
    q = typed(rng.normal(0, 1, (1, nh * hd)), F32)
    out, _ = run_attention(native, pg, q, F32, 1, [1], nh, float(1 / np.sqrt(np.float32(hd))))
    cap = (n + 7) // 8 * 8
    k, v = np.zeros((cap, n_kv, hd), np.uint16), np.zeros((cap, n_kv, hd), np.uint16)
    k[:n], v[:n] = pg.get(0, np.arange(n))
    kc = _dev(k.reshape(cap, n_kv, hd // 8, 8).transpose(1, 2, 0, 3))
    vc = _dev(v.reshape(cap // 8, 8, n_kv, hd).transpose(2, 0, 3, 1))
    dq, pos, o, xq, xs = _dev(q), _dev(np.array([n - 1], np.uint32)), _buf(nh * hd * 4), _buf(nh * hd), _buf(nh * hd)
    _ok(native.camelid_hip_attention_decode(dq.ptr, kc.ptr, vc.ptr, 0, nh, n_kv, hd, cap, pos.ptr,
                                            float(1 / np.sqrt(np.float32(hd))), o.ptr, xq.ptr, xs.ptr, None))
    (y, tol), = attention_reference(pg, q, F32, 1, [1], nh, float(1 / np.sqrt(np.float32(hd))), None)[0]
    # (that kernel's chains are n positions long)
    assert (np.abs(out[0] - o.download(np.float32, nh * hd)) <= 2 * tol + n * U * 4).all()


# -------------------------------------------------------------------------------------------- eviction
def evict_reference(pg, weights, keep, recent):
    """Pages and weights after the eviction, lens_out, kept."""
    k, v, w = pg.k.copy(), pg.v.copy(), weights.copy()
    kept = np.full((pg.n, pg.n_kv, keep), NONE, np.uint32)
    lens = np.minimum(pg.lens, keep)
    for s, n in enumerate(pg.lens.astype(int)):
        if n <= keep:
            kept[s, :, :n] = np.arange(n)
            continue
        kb, vb = pg.get(s, np.arange(n))
        nk, nv = np.empty((keep,) + kb.shape[1:], np.uint16), np.empty((keep,) + kb.shape[1:], np.uint16)
        for h in range(pg.n_kv):
            x = weights[s, h, :n - recent].astype(np.float64)
            order = sorted(range(n - recent), key=lambda p: (0 if x[p] == x[p] else 1, -x[p] if x[p] == x[p] else 0, p))
            at = np.array(sorted(order[:keep - recent]) + list(range(n - recent, n)), np.int64)
            kept[s, h] = at
            nk[:, h], nv[:, h] = kb[at, h], vb[at, h]
            w[s, h, :keep] = weights[s, h, at]
        ik, iv = pg.cells(s, np.arange(keep))
        k.reshape(-1)[ik], v.reshape(-1)[iv] = nk, nv
    return k, v, w, lens, kept


def run_evict(native, pg, weights, keep, recent, want_kept=True, alias=False):
    pg.upload()
    dw = _dev(weights)
    do = pg.dl if alias else _dev(np.full(pg.n, 99, np.uint32))
    dk = _dev(np.full(pg.n * pg.n_kv * keep, NONE, np.uint32)) if want_kept else None
    size = native.camelid_hip_paged_evict_workspace(pg.n, pg.n_kv, pg.ps, pg.stride, keep)
    ws = _dev(np.full(size + 64, 0xEE, np.uint8))
    _ok(native.camelid_hip_paged_evict(pg.dk.ptr, pg.dv.ptr, pg.n_pages, pg.ps, pg.n_kv, pg.hd, pg.dt.ptr, pg.stride,
                                       pg.dl.ptr, pg.n, dw.ptr, keep, recent, do.ptr, dk.ptr if dk else None, ws.ptr,
                                       size, pg.dstat.ptr, None))
    pg.download()
    assert (ws.download(np.uint8, size + 64)[size:] == 0xEE).all()
    return (dw.download(np.float32, weights.size).reshape(weights.shape), do.download(np.uint32, pg.n),
            dk.download(np.uint32, pg.n * pg.n_kv * keep).reshape(pg.n, pg.n_kv, keep) if dk else None)


def heavy(rng, *shape):
    return rng.lognormal(-2, 2, shape).astype(np.float32)


def tied(rng, *shape):
    return rng.integers(0, 4, shape).astype(np.float32)


def strange(rng, *shape):
    x = rng.normal(0, 1, shape).astype(np.float32)
    x[rng.random(shape) < 0.1] = np.nan
    x[rng.random(shape) < 0.1] = -0.0
    x[rng.random(shape) < 0.1] = 0.0
    x[rng.random(shape) < 0.05] = np.inf
    x[rng.random(shape) < 0.05] = -np.inf
    x[rng.random(shape) < 0.1] = np.float32(1e-41)
    return x


EVICT_CASES = [
    # n_kv, hd, lens, page, keep, recent, weights
    (4, 64, [100], 16, 64, 16, heavy),
    (8, 128, [65, 64, 63, 0, 200], 8, 64, 0, tied),
    (2, 128, [70, 300, 1], 32, 1, 0, heavy),
    (2, 64, [70, 300, 2], 32, 1, 1, heavy),
    (2, 256, [1500, 1029], 64, 1027, 1027, strange),
    (1, 64, [5000, 2048, 2049], 16, 2047, 100, strange),
    (3, 128, [777], 256, 333, 332, tied),
    (2, 64, [20000, 9], 128, 3001, 17, heavy),
    (2, 64, [40], 8, 1000, 10, heavy),
    (8, 128, [1088] * 3, 32, 1024, 256, heavy),
    (8, 128, [3000, 2500], 32, 2100, 50, strange),
    (8, 128, [78, 11, 60, 33] * 20, 8, 22, 9, heavy),
    (4, 64, [400, 512, 1, 0, 257], 64, 130, 0, strange),
    (8, 256, [300, 512], 128, 256, 255, tied),
    (2, 256, [40, 17], 8, 3, 1, strange),
]


@pytest.mark.parametrize("n_kv,hd,lens,ps,keep,recent,make", EVICT_CASES)
def test_evict_exact(native, n_kv, hd, lens, ps, keep, recent, make):
    rng = np.random.default_rng(keep + hd)
    bits = lambda *sh: rng.integers(-2000, 2000, sh).astype(np.float32)  # noqa: E731
    pg = Pages(rng, lens, ps, n_kv, hd, F16, rows=bits)
    weights = make(rng, len(lens), n_kv, pg.cap)
    k, v, w, lo, kept = evict_reference(pg, weights, keep, recent)
    got_w, got_lens, got_kept = run_evict(native, pg, weights, keep, recent, alias=keep % 2 == 1)
    assert pg.status() == 0
    assert (got_lens == lo).all() and (got_kept == kept).all()
    assert (got_w.view(np.uint32) == w.view(np.uint32)).all()
    assert (pg.k == k).all() and (pg.v == v).all()


def test_evict_without_kept_and_bad_input(native):
    rng = np.random.default_rng(21)
    pg = Pages(rng, [100, 90, 80, 60], 8, 2, 64, BF16)
    weights = heavy(rng, 4, 2, pg.cap)
    k, v, w, lo, _ = evict_reference(pg, weights, 32, 8)
    k0, v0 = pg.k.copy(), pg.v.copy()
    good = pg.table.copy()
    pg.table[1, 9] = pg.n_pages + 5   # among the 90 positions: the sequence stays as it is
    pg.table[3, 8] = 0xFFFFFFFF       # behind the 60 positions: never looked at
    pg.lens[2] = pg.cap + 1
    got_w, got_lens, _ = run_evict(native, pg, weights, 32, 8, want_kept=False)
    assert pg.status() == 3
    assert got_lens.tolist() == [32, 90, pg.cap + 1, 32]
    for s in (1, 2):
        w[s] = weights[s]
        pages = good[s]
        k[pages], v[pages] = k0[pages], v0[pages]
    assert (got_w.view(np.uint32) == w.view(np.uint32)).all()
    assert (pg.k == k).all() and (pg.v == v).all()


# ---------------------------------------------------------------------------------------- verification
def softmax64(x, t):
    z = (x - x.max()) / t
    e = np.where(np.isneginf(x), 0.0, np.exp(z))
    return e / e.sum()


def verify_reference(target, draft, tokens, lens, temps, u):
    """accepted, tokens, log-probabilities, one draft after the other in 64 bits."""
    n, k1, vocab = target.shape
    acc, out, lps = np.zeros(n, np.uint32), np.full((n, k1), NONE, np.uint32), np.zeros((n, k1))
    for s in range(n):
        temp = float(np.float32(temps[s])) if temps[s] > 0 else 0.0  # the f32 number the call gets
        m = min(int(lens[s]), k1 - 1)
        for t in range(m + 1):
            x = target[s, t]
            bad = np.isnan(x).any() or np.isposinf(x).any() or np.isneginf(x).all()
            if t < m and draft is not None and temp:
                y = draft[s, t]
                bad = bad or np.isnan(y).any() or np.isposinf(y).any() or np.isneginf(y).all()
            if bad:
                lps[s, t] = np.nan
                break
            with np.errstate(divide="ignore"):
                told = np.log(softmax64(x, temp or 1.0))
            p = softmax64(x, temp) if temp else np.eye(1, vocab, int(x.argmax()))[0]
            rest = p
            if t < m:
                d = int(tokens[s, t])
                q = np.zeros(vocab)
                if draft is not None and temp:
                    q = softmax64(draft[s, t], temp)
                elif d < vocab:
                    q[d] = 1.0
                if d < vocab and float(u[s, t]) * q[d] < p[d]:
                    out[s, t], lps[s, t] = d, told[d]
                    acc[s] += 1
                    continue
                rest = np.maximum(p - q, 0)
                if not rest.sum() > 0:
                    rest = p
            c = np.cumsum(rest)
            pick = int(np.searchsorted(c, float(u[s, -1]) * c[-1], side="right"))
            out[s, t] = pick = min(pick, int(np.nonzero(rest)[0].max()))
            lps[s, t] = told[pick]
            break
    return acc, out, lps


def run_verify(native, target, draft, tokens, lens, temps, u, lt, logprobs=True, null_lens=False):
    n, k1, vocab = target.shape
    bufs = [_dev(x) for x in (typed(target, lt), np.array(tokens, np.uint32), np.array(lens, np.uint32),
                              np.array(temps, np.float32), np.array(u, np.float32))]
    dd = _dev(typed(draft, lt)) if draft is not None else None
    acc, out = _dev(np.full(n, 77, np.uint32)), _dev(np.full(n * k1, 77, np.uint32))
    lp = _dev(np.full(n * k1, 77, np.float32)) if logprobs else None
    size = native.camelid_hip_verify_drafts_workspace(n, k1 - 1, vocab)
    ws = _dev(np.full(size + 64, 0xEE, np.uint8))
    _ok(native.camelid_hip_verify_drafts(bufs[0].ptr, dd.ptr if dd else None, lt, bufs[1].ptr,
                                         None if null_lens else bufs[2].ptr, n, k1 - 1, vocab, bufs[3].ptr,
                                         bufs[4].ptr, acc.ptr, out.ptr, lp.ptr if lp else None, ws.ptr, size, None))
    got = acc.download(np.uint32, n), out.download(np.uint32, n * k1).reshape(n, k1)
    assert (ws.download(np.uint8, size + 64)[size:] == 0xEE).all()
    return got + (lp.download(np.float32, n * k1).reshape(n, k1) if lp else None,)


def check_verify(got, want):
    assert (got[0] == want[0]).all(), (got[0], want[0])
    assert (got[1] == want[1]).all(), (got[1], want[1])
    if got[2] is not None:
        assert (np.isnan(got[2]) == np.isnan(want[2])).all()
        ok = np.isfinite(want[2])
        # (a log-probability near 0 is a difference of numbers near 1: 1e-14 of its own)
        assert (np.abs(got[2] - want[2])[ok] <= 2 * U * np.abs(want[2])[ok] + 1e-12).all()


VERIFY_CASES = [
    # seqs, drafts, vocab, draft logits, type
    (1, 4, 32000, False, F32), (5, 3, 1000, True, F32), (7, 0, 4097, False, F16), (3, 7, 151936, True, BF16),
    (2, 1, 1, True, F32), (4, 5, 63, False, BF16), (9, 2, 8191, True, F16), (2, 31, 500, True, F32),
    (3, 4, 128256, False, F32), (2, 1, 700001, True, F16), (1, 2, 600000, False, BF16),
]


@pytest.mark.parametrize("n,k,vocab,has_draft,lt", VERIFY_CASES)
def test_verify_against_64_bits(native, n, k, vocab, has_draft, lt):
    rng = np.random.default_rng(n * 100 + k)
    target = rng.normal(0, 2.5, (n, k + 1, vocab))
    draft = target[:, :k] + rng.normal(0, 0.7, (n, k, vocab)) if has_draft else None
    target = value(typed(target, lt), lt).reshape(target.shape)
    tokens = rng.integers(0, vocab, (n, k))
    if draft is not None:
        draft = value(typed(draft, lt), lt).reshape(draft.shape)
        for s in range(n):
            for t in range(k):
                tokens[s, t] = rng.choice(vocab, p=softmax64(draft[s, t], 0.9))
    else:
        best = target[:, :k].argmax(-1)
        tokens = np.where(rng.random((n, k)) < 0.8, best, tokens)
        np.put_along_axis(target[:, :k], best[..., None], 30.0, -1)
    temps = np.array([0.0 if s % 4 == 3 else 0.5 + 0.3 * (s % 3) for s in range(n)], np.float32)
    lens = np.array([k if s == 0 else (s * 3) % (k + 2) for s in range(n)])  # some past n_draft
    u = rng.random((n, k + 1)).astype(np.float32)
    want = verify_reference(target, draft, tokens, lens, temps, u)
    check_verify(run_verify(native, target, draft, tokens, lens, temps, u, lt), want)
    full = verify_reference(target, draft, tokens, [k] * n, temps, u)
    check_verify(run_verify(native, target, draft, tokens, lens, temps, u, lt, logprobs=False, null_lens=True), full)


def test_verify_borders(native):
    """Numbers on a border of the prefix sums, exact in binary: C_i > u S is strict."""
    n, vocab = 12, 8
    target = np.zeros((n, 1, vocab))                  # p_i = 1/8 exactly
    u = (np.arange(n) / 12 * 8 // 1 / 8).astype(np.float32).reshape(n, 1)
    u[-1] = np.float32(1 - 2.0 ** -24)
    u[0] = 0.0
    want = verify_reference(target, None, np.zeros((n, 0), int), [0] * n, [1.0] * n, u)
    assert (want[1][:, 0] == np.minimum((u[:, 0] * 8).astype(int), 7)).all()
    check_verify(run_verify(native, target, None, np.zeros((n, 0), int), [0] * n, [1.0] * n, u, F32), want)
    # acceptance: u q < p is strict too.  q certain, p_x = 1/8
    target = np.zeros((3, 2, vocab))
    u = np.array([[0.125, 0.5], [np.nextafter(np.float32(0.125), np.float32(0)), 0.5], [0.0, 0.0]], np.float32)
    got = run_verify(native, target, None, np.array([[3], [3], [3]]), [1] * 3, [1.0] * 3, u, F32)
    check_verify(got, verify_reference(target, None, np.array([[3], [3], [3]]), [1] * 3, [1.0] * 3, u))
    assert got[0].tolist() == [0, 1, 1] and got[1][0, 0] != 3


def test_verify_masked_and_missing_distributions(native):
    """-inf logits are never drawn; rows without a distribution end their sequence; equal rows."""
    rng = np.random.default_rng(31)
    n, k, vocab = 9, 2, 5000
    target = rng.normal(0, 2, (n, k + 1, vocab))
    target[:, :, ::2] = -np.inf
    target = value(typed(target, F32), F32)
    draft = target[:, :k].copy()
    draft[0] = value(typed(rng.normal(0, 2, (k, vocab)), F32), F32)       # may name masked tokens
    tokens = rng.integers(0, vocab, (n, k))
    target[1, 0, 77] = np.nan
    target[2, 1, 1] = np.inf
    tokens[2, 0] = int(target[2, 0].argmax())
    target[3, 2] = -np.inf
    tokens[3] = target[3, :2].argmax(-1)
    draft[4, 0, 9] = np.nan
    tokens[5, 0] = vocab                                                  # no such token
    tokens[6] = [4, 6]                                                    # masked drafts, certain or not
    target[7, 0] = -np.inf
    target[7, 0, vocab - 1] = -5.0                                        # one token left
    temps = np.array([1.0, 0.7, 0.0, 0.0, 1.0, 1.0, 1.0, 1.3, -1.0], np.float32)
    u = np.full((n, k + 1), 0.9, np.float32)
    u[7, 2] = 0.0
    for d in (draft, None):
        want = verify_reference(target, d, tokens, [k] * n, temps, u)
        check_verify(run_verify(native, target, d, tokens, [k] * n, temps, u, F32), want)
    assert want[1][1, 0] == NONE and want[1][2, 1] == NONE and want[1][3, 2] == NONE


@pytest.mark.parametrize("has_draft", [False, True])
def test_verify_extreme_temperatures(native, has_draft):
    """From temperatures so low that only the largest logit is left (and its equals), past the f32 step of
    the logits, to ones so high that every token that is not masked is as likely as any other."""
    rng = np.random.default_rng(35)
    temps = np.array([1e-40, 1e-30, 1e-12, 1e-7, 1e-5, 1e-3, 50.0, 1e6, 1e34, 1e36, 3e38, np.inf], np.float32)
    n, k, vocab = len(temps), 2, 3000
    target = rng.normal(0, 4, (n, k + 1, vocab)) + 1000.0 * rng.choice([-1, 0, 1], (n, 1, 1))
    target[:, :, 5::7] = -np.inf
    target[:, 1, 100:103] = target[:, 1].max(-1, keepdims=True) + 1.0    # three equal best ones
    target = value(typed(target, F32), F32)
    draft = value(typed(target[:, :k] + rng.normal(0, 1, (n, k, vocab)), F32), F32) if has_draft else None
    tokens = target[:, :k].argmax(-1)
    u = rng.random((n, k + 1)).astype(np.float32)
    with np.errstate(all="ignore"):
        want = verify_reference(target, draft, tokens, [k] * n, temps, u)
    check_verify(run_verify(native, target, draft, tokens, [k] * n, temps, u, F32), want)


def test_verify_logits_near_the_largest(native):
    """Sums of a row's logits are beyond f32 (and beside -inf nearly NaN); every row has a distribution."""
    rng = np.random.default_rng(36)
    n, k, vocab = 4, 1, 5000
    target = np.full((n, k + 1, vocab), -np.inf)
    target[:, :, :600] = 3e38
    target[1:, :, 300:900] = rng.uniform(1e38, 3.4e38, (n - 1, k + 1, 600))
    target[2, :, 1000:] = -3.4e38
    target = value(typed(target, F32), F32)
    temps = np.array([1.0, 3e37, 1e38, 0.0], np.float32)
    u = rng.random((n, k + 1)).astype(np.float32)
    tokens = target[:, :k].argmax(-1)
    want = verify_reference(target, None, tokens, [k] * n, temps, u)
    check_verify(run_verify(native, target, None, tokens, [k] * n, temps, u, F32), want)


def test_verify_frequencies(native):
    """What comes out of one draft and its correction is distributed as the target: 20000 sequences of
    one small vocabulary, each token's count within 6 standard deviations."""
    rng = np.random.default_rng(33)
    n, vocab = 20000, 12
    t1, d1 = rng.normal(0, 1, vocab), rng.normal(0, 1, vocab)
    target = np.broadcast_to(t1, (n, 2, vocab))
    draft = np.broadcast_to(d1, (n, 1, vocab))
    p = softmax64(t1.astype(np.float32).astype(np.float64), 1.0)
    q = softmax64(d1.astype(np.float32).astype(np.float64), 1.0)
    tokens = rng.choice(vocab, (n, 1), p=q)
    u = rng.random((n, 2)).astype(np.float32)
    _, out, _ = run_verify(native, target, draft, tokens, [1] * n, [1.0] * n, u, F32)
    count = np.bincount(out[:, 0], minlength=vocab)
    assert (np.abs(count - n * p) <= 6 * np.sqrt(n * p * (1 - p))).all()


# ------------------------------------------------------------------------------------ a run of them
def test_a_serving_loop(native):
    """Prompt, then rounds of draft, store, attend, verify and evict over one cache: every call against
    64 bits, on what the calls before it left on the device."""
    rng = np.random.default_rng(41)
    nh, n_kv, hd, ps, k, vocab, keep, recent = 8, 2, 64, 16, 3, 300, 48, 16
    n, g = 3, 4
    pg = Pages(rng, [96] * n, ps, n_kv, hd, F16)
    prompt = [40, 17, 30]
    where = np.zeros(n, int)                                   # each sequence's next position in the text
    weights = np.zeros((n, n_kv, pg.cap), np.float32)
    proj = rng.normal(0, 0.3, (nh * hd, vocab))

    def store(lens, new, n_new):
        qkv = rng.normal(0, 1.2, (n * n_new, (nh + 2 * n_kv) * hd)).astype(np.float32)
        pos = np.array([[where[s] + t for t in range(n_new)] for s in range(n)]).reshape(-1, 1)
        ang = pos * 10000.0 ** (-np.arange(hd // 2) * 2.0 / hd)
        cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
        pg.lens = np.array(lens, np.uint32)
        q, _ = run_rope(native, pg, qkv, n_new, new, nh, hd, False, cos, sin, None, None, 0.0, F32)
        y, err = rope_reference(qkv, cos, sin, nh, n_kv, hd, hd, False, None, None, 0.0)
        for s in range(n):
            gk, gv = pg.get(s, np.arange(lens[s] - new[s], lens[s]))
            r = slice(s * n_new, s * n_new + new[s])
            assert (np.abs(from16(gk, F16) - y[r, nh:nh + n_kv]) <= err[r, nh:nh + n_kv] +
                    2.0 ** -11 * np.abs(y[r, nh:nh + n_kv]) + 2.0 ** -24).all()
        return q

    store(prompt, prompt, max(prompt))
    where += prompt
    lens = list(prompt)
    evictions = 0
    for step in range(14):
        new = [k + 1 - (s + step) % 2 for s in range(n)]       # the last token and its drafts
        lens = [a + b for a, b in zip(lens, new)]
        q = store(lens, new, k + 1)
        out, got_w = run_attention(native, pg, q, F32, k + 1, new, nh, 0.125, weights)
        check_attention(out, got_w, attention_reference(pg, q, F32, k + 1, new, nh, 0.125, weights), weights, pg, k + 1,
                        new, F32)
        weights = got_w
        target = np.float32(np.where(np.arange(n * (k + 1))[:, None] % (k + 1) < np.repeat(new, k + 1)[:, None],
                                     out.astype(np.float64), 0.0) @ proj).reshape(n, k + 1, vocab)
        target = target.astype(np.float64)
        tokens = target[:, :k].argmax(-1)
        tokens[:, 1] = rng.integers(0, vocab, n)
        u = rng.random((n, k + 1)).astype(np.float32)
        dl = np.array(new) - 1
        got = run_verify(native, target, None, tokens, dl, [0.8] * n, u, F32)
        check_verify(got, verify_reference(target, None, tokens, dl, [0.8] * n, u))
        for s in range(n):                                     # the rejected drafts leave the cache
            lens[s] -= new[s] - 1 - int(got[0][s])
            where[s] += 1 + int(got[0][s])
        pg.lens = np.array(lens, np.uint32)
        want = evict_reference(pg, weights, keep, recent)
        evictions += int((pg.lens > keep).sum())
        weights, lo, _ = run_evict(native, pg, weights, keep, recent)
        assert (pg.k == want[0]).all() and (pg.v == want[1]).all() and (lo == want[3]).all()
        assert (weights.view(np.uint32) == want[2].view(np.uint32)).all()
        lens = [int(x) for x in lo]
    assert evictions > 10 and pg.status() == 0


class Batch:
    """Inputs and outputs of all four calls on the device, and the calls."""

    NH, HD, N, NEW, VOCAB, KEEP = 32, 128, 4, 2, 3001, 600
    OUT = {"q": np.float32, "out": np.float32, "w": np.float32, "kept": np.uint32, "lens_out": np.uint32,
           "acc": np.uint32, "tok": np.uint32, "lp": np.float32, "stat": np.uint32, "k": np.uint16, "v": np.uint16}

    def __init__(self, native, seed):
        self.native = native
        self.host = self.make(seed)
        self.buf = {k: _dev(x) for k, x in self.host.items()}
        c = self
        sizes = (native.camelid_hip_paged_attention_workspace(c.N, c.NEW, c.NH, 8, c.HD, 32, 40, 1),
                 native.camelid_hip_paged_evict_workspace(c.N, 8, 32, 40, c.KEEP),
                 native.camelid_hip_verify_drafts_workspace(c.N, c.NEW - 1, c.VOCAB))
        self.ws = [(_buf(x), x) for x in sizes]

    def make(self, seed):
        rng = np.random.default_rng(seed)
        n, new, nh, hd, vocab = self.N, self.NEW, self.NH, self.HD, self.VOCAB
        pg = Pages(rng, rng.integers(700, 1200, n), 32, 8, hd, F16, extra_stride=0)
        table = np.zeros((n, 40), np.uint32)
        table[:, :pg.stride] = pg.table
        k, v = (np.zeros((170, 8, hd * 32), np.uint16) for _ in range(2))
        k[:pg.n_pages], v[:pg.n_pages] = pg.k, pg.v
        rows, f = n * new, np.float32
        return {"k": k, "v": v, "table": table, "lens": pg.lens,
                "qkv": rng.normal(0, 1, (rows, (nh + 16) * hd)).astype(f),
                "cos": rng.uniform(-1, 1, (rows, hd // 2)).astype(f),
                "sin": rng.uniform(-1, 1, (rows, hd // 2)).astype(f),
                "w": rng.uniform(0, 1, (n, 8, 40 * 32)).astype(f),
                "target": rng.normal(0, 3, (n, new, vocab)).astype(f),
                "tokens": rng.integers(0, vocab, (n, new - 1)).astype(np.uint32), "temp": np.ones(n, f),
                "u": rng.random((n, new)).astype(f), "q": np.zeros((rows, nh * hd), f),
                "out": np.zeros((rows, nh * hd), f), "acc": np.zeros(n, np.uint32),
                "tok": np.zeros((n, new), np.uint32), "lp": np.zeros((n, new), f), "lens_out": np.zeros(n, np.uint32),
                "kept": np.zeros((n, 8, self.KEEP), np.uint32), "stat": np.zeros(1, np.uint32)}

    def fill(self, seed):
        for k, x in self.make(seed).items():
            self.buf[k].upload(x)

    def calls(self, stream):
        lib, p, ws = self.native, {k: b.ptr for k, b in self.buf.items()}, [(b.ptr, x) for b, x in self.ws]
        n, new, nh, hd = self.N, self.NEW, self.NH, self.HD
        _ok(lib.camelid_hip_paged_rope_kv(p["qkv"], n, new, None, nh, 8, hd, hd, 0, p["cos"], p["sin"], None, None, 0.0,
                                          p["q"], F32, p["k"], p["v"], F16, 170, 32, p["table"], 40, p["lens"],
                                          p["stat"], stream))
        _ok(lib.camelid_hip_paged_attention(p["q"], F32, nh * hd, n, new, None, nh, 8, hd, p["k"], p["v"], F16, 170, 32,
                                            p["table"], 40, p["lens"], 0.09, p["out"], nh * hd, p["w"], *ws[0],
                                            p["stat"], stream))
        _ok(lib.camelid_hip_paged_evict(p["k"], p["v"], 170, 32, 8, hd, p["table"], 40, p["lens"], n, p["w"],
                                        self.KEEP, 100, p["lens_out"], p["kept"], *ws[1], p["stat"], stream))
        _ok(lib.camelid_hip_verify_drafts(p["target"], None, F32, p["tokens"], None, n, new - 1, self.VOCAB,
                                          p["temp"], p["u"], p["acc"], p["tok"], p["lp"], *ws[2], stream))

    def results(self):
        return {k: self.buf[k].download(t, self.host[k].size).view(f"u{np.dtype(t).itemsize}")
                for k, t in self.OUT.items()}


def _hip(native, name, *args):
    """A HIP runtime call, through the library that the native code is linked with."""
    fn = getattr(native, name)
    fn.restype = C.c_int
    rc = fn(*args)
    assert rc == 0, (name, rc)


def _same(got, want, what):
    for k in want:
        assert (got[k] == want[k]).all(), (what, k)


def test_calls_replay_in_a_graph_and_run_on_other_streams(native):
    """All four calls captured into one graph and replayed over changing inputs, against the same calls
    made eagerly; two streams at once with workspaces of their own."""
    wants = []
    for seed in range(4):
        b = Batch(native, seed)
        b.calls(None)
        wants.append(b.results())
        assert wants[-1]["stat"][0] == 0 and wants[-1]["kept"].any() and wants[-1]["lp"].any()
    live = Batch(native, 0)
    stream, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    _hip(native, "hipStreamCreate", C.byref(stream))
    _hip(native, "hipStreamBeginCapture", stream, 1)
    live.calls(stream)
    _hip(native, "hipStreamEndCapture", stream, C.byref(graph))
    _hip(native, "hipGraphInstantiate", C.byref(run), graph, None, None, C.c_size_t(0))
    for seed in (1, 0, 3, 2, 1):
        live.fill(seed)
        _ok(native.camelid_hip_synchronize())
        _hip(native, "hipGraphLaunch", run, stream)
        _hip(native, "hipStreamSynchronize", stream)
        _same(live.results(), wants[seed], seed)
    _hip(native, "hipGraphExecDestroy", run)
    _hip(native, "hipGraphDestroy", graph)
    other = C.c_void_p()
    _hip(native, "hipStreamCreate", C.byref(other))
    both = [Batch(native, 2), Batch(native, 3)]
    _ok(native.camelid_hip_synchronize())
    both[0].calls(stream)
    both[1].calls(other)
    for st, b, seed in zip((stream, other), both, (2, 3)):
        _hip(native, "hipStreamSynchronize", st)
        _same(b.results(), wants[seed], seed)
        _hip(native, "hipStreamDestroy", st)


# ------------------------------------------------------------------------------- the engine's own path
@pytest.mark.parametrize("prefill", ["batched", "token"])
def test_verify_sampled_draws_from_the_engine_logits(native, monkeypatch, prefill):
    """Drafts verified by sampling on the engine: exactly what the definition gives on the logits that
    single-token steps return (the forward is bit-identical to them)."""
    from camelid_amd.model import ResidentSession, SyntheticModel, prompt_tokens, rope_tables, tiny_config
    monkeypatch.setenv("CAMELID_HIP_PREFILL", prefill)
    cfg = tiny_config(prompt_len=20)
    model = SyntheticModel.generate(cfg)
    prompt = prompt_tokens(cfg)
    rng = np.random.default_rng(51)
    sess = ResidentSession(model, 40)
    eng, base = sess.engine, len(prompt) - 1
    sess.prefill(prompt[:-1])
    for k in (1, 2, 5, 8):
        for temp in (0.0, 0.7, 1.3):
            for with_draft in (False, True):
                eng.set_filled(base)
                drafts = [int(t) for t in rng.integers(0, cfg.vocab, k - 1)]
                rows, step = [], [int(prompt[-1])] + drafts
                for i in range(k):
                    greedy = sess.step(step[i], base + i, logits=True)
                    rows.append(eng.last_logits.astype(np.float64))
                    if i < k - 1 and rng.random() < 0.6:  # some drafts right
                        step[i + 1] = int(greedy)
                drafts = step[1:]
                target = np.array(rows)[None]
                dl = (target[:, :k - 1] + rng.normal(0, 0.5, (1, k - 1, cfg.vocab))).astype(np.float32) \
                    if with_draft and k > 1 else None
                u = rng.random(k, dtype=np.float32)
                eng.set_filled(base)
                cos, sin = rope_tables(cfg, base, k)
                toks, lps = eng.verify_sampled(model.embed(step), cos, sin, base, cfg.scale(), drafts, u, temp,
                                               None if dl is None else dl[0])
                want = verify_reference(target, None if dl is None else dl.astype(np.float64), np.array([drafts], np.int64)
                                        .reshape(1, k - 1), [k - 1], [temp], u[None])
                n = int(want[0][0]) + 1
                assert [int(t) for t in toks] == want[1][0, :n].tolist(), (k, temp, with_draft)
                assert (np.abs(lps - want[2][0, :n]) <= 2 * U * np.abs(want[2][0, :n]) + 1e-12).all()
    # the session's sampled generation: greedy at 0 with and without looked-up drafts; runs at 1
    sess.engine.set_filled(0)
    greedy = sess.generate(prompt, 12)
    assert sess.generate_sampled(prompt, 12, 0.0, np.random.default_rng(1)) == greedy
    text = list(prompt[:8]) * 2 + list(prompt[:3])
    want = sess.generate(text, 12)
    assert sess.generate_sampled(text, 12, 0.0, np.random.default_rng(1), max_draft=5) == want
    assert len(sess.generate_sampled(text, 12, 1.0, np.random.default_rng(2), max_draft=5)) == 12
    sess.close()


def test_verify_sampled_refusals(native):
    from camelid_amd._native import HipError
    from camelid_amd.model import ResidentSession, SyntheticModel, prompt_tokens, rope_tables, tiny_config
    cfg = tiny_config(prompt_len=8)
    model = SyntheticModel.generate(cfg)
    sess = ResidentSession(model, 16)
    prompt = prompt_tokens(cfg)
    sess.prefill(prompt[:-1])
    base = len(prompt) - 1

    def call(k=2, drafts=(3,), u=(0.5, 0.5), temp=1.0, pos=base):
        cos, sin = rope_tables(cfg, pos, k)
        return sess.engine.verify_sampled(model.embed([1] * k), cos, sin, pos, cfg.scale(), list(drafts), list(u), temp)

    for change, match in ((dict(u=(0.5, 1.0)), "uniforms"), (dict(u=(float("nan"), 0.1)), "uniforms"),
                          (dict(temp=-1.0), "temperature"), (dict(temp=float("inf")), "temperature"),
                          (dict(drafts=(cfg.vocab,)), "draft token"), (dict(pos=base + 1), "base_position"),
                          (dict(k=9, drafts=[1] * 8, u=[0.1] * 9), "k out of")):
        with pytest.raises(HipError, match=match):
            call(**change)
    with pytest.raises(ValueError, match="draft_tokens"):
        call(drafts=(1, 2))
    with pytest.raises(ValueError, match="uniforms"):
        call(u=(0.5,))
    assert len(call()[0]) in (1, 2)  # nothing above has hurt the engine
    sess.close()


@pytest.mark.parametrize("nh,n_kv,hd,new", [(32, 8, 128, 5), (16, 4, 256, 2), (64, 2, 64, 8)])
def test_attention_with_large_workgroups_replays_in_a_graph(native, nh, n_kv, hd, new):
    """Kernels that need more LDS than 64 KB, captured as their first call and replayed over a cache that
    grows between the replays, against eager calls."""
    rng = np.random.default_rng(61)
    n, ps, cap = 3, 16, 1024
    pg = Pages(rng, [cap] * n, ps, n_kv, hd, F16, extra_stride=0)
    pg.upload()
    q = _dev(rng.normal(0, 1, (n * new, nh * hd)).astype(np.float32))
    size = native.camelid_hip_paged_attention_workspace(n, new, nh, n_kv, hd, ps, pg.stride, 0)
    ws, out = _buf(size), _dev(np.zeros((n * new, nh * hd), np.float32))

    def call(stream):
        _ok(native.camelid_hip_paged_attention(q.ptr, F32, nh * hd, n, new, None, nh, n_kv, hd, pg.dk.ptr, pg.dv.ptr, F16,
                                               pg.n_pages, ps, pg.dt.ptr, pg.stride, pg.dl.ptr, 0.1, out.ptr, nh * hd,
                                               None, ws.ptr, size, pg.dstat.ptr, stream))

    stream, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    _hip(native, "hipStreamCreate", C.byref(stream))
    _hip(native, "hipStreamBeginCapture", stream, 1)
    call(stream)
    _hip(native, "hipStreamEndCapture", stream, C.byref(graph))
    _hip(native, "hipGraphInstantiate", C.byref(run), graph, None, None, C.c_size_t(0))
    for lens in ([new] * n, [8, 300, 33], [cap, 9, 513], [1000, 1001, 1002]):
        pg.dl.upload(np.array(lens, np.uint32))
        _ok(native.camelid_hip_synchronize())
        call(None)
        want = out.download(np.uint32, n * new * nh * hd)
        out.upload(np.zeros((n * new, nh * hd), np.float32))
        _hip(native, "hipGraphLaunch", run, stream)
        _hip(native, "hipStreamSynchronize", stream)
        assert (out.download(np.uint32, n * new * nh * hd) == want).all(), lens
    assert pg.status() == 0
    _hip(native, "hipGraphExecDestroy", run)
    _hip(native, "hipGraphDestroy", graph)
    _hip(native, "hipStreamDestroy", stream)


def test_a_cache_past_two_to_the_32_elements(native):
    """The same calls over a small pool and over the far end of one whose offsets pass 32 bits (in elements
    and in bytes): the same bits everywhere."""
    rng = np.random.default_rng(62)
    n, n_kv, nh, hd, ps, new = 2, 8, 16, 128, 4096, 100
    page = n_kv * hd * ps
    far = (1 << 32) // page + 1
    table = np.array([[3, 0], [1, 2]], np.uint32)
    prompts = rng.normal(0, 1, (n * new, (nh + 2 * n_kv) * hd)).astype(np.float32)
    angle = rng.uniform(0, 7, (n * new, hd // 2))
    dq, dc, dn = _dev(prompts), _dev(np.cos(angle).astype(np.float32)), _dev(np.sin(angle).astype(np.float32))
    drafts = _dev(rng.normal(0, 1, (n * 2, nh * hd)).astype(np.float32))
    results = []
    for offset in (0, far):
        pages = offset + 4
        kc, vc = _buf(pages * page * 2), _buf(pages * page * 2)
        dt, dl, stat = _dev(table + np.uint32(offset)), _dev(np.full(n, new, np.uint32)), _dev(np.zeros(1, np.uint32))
        q_out, out = _buf(n * new * nh * hd * 4), _dev(np.zeros((n * 2, nh * hd), np.float32))
        weights = _dev(np.zeros((n, n_kv, 2 * ps), np.float32))
        # a prompt over the end of each first page, in three calls; half of them by the path for part of a head
        at = ps - 130
        for rope_dim in (hd, hd - 32, hd):
            at += new
            dl.upload(np.full(n, at, np.uint32))
            _ok(native.camelid_hip_paged_rope_kv(dq.ptr, n, new, None, nh, n_kv, hd, rope_dim, 1, dc.ptr, dn.ptr, None, None,
                                                 1e-5, q_out.ptr, F32, kc.ptr, vc.ptr, F16, pages, ps, dt.ptr, 2, dl.ptr,
                                                 stat.ptr, None))
            _ok(native.camelid_hip_synchronize())
        # the positions before them: none; their pages hold whatever the allocation held, so only the newest
        # tokens' own pages count: a second table whose sequences begin at the second page
        dt2 = _dev((table[:, 1:] + np.uint32(offset)).astype(np.uint32))
        held = at - ps
        dl.upload(np.full(n, held, np.uint32))
        size = native.camelid_hip_paged_attention_workspace(n, 2, nh, n_kv, hd, ps, 1, 1)
        ws = _buf(size)
        evict = native.camelid_hip_paged_evict_workspace(n, n_kv, ps, 1, 64)
        ws2, kept = _buf(evict), _dev(np.zeros((n, n_kv, 64), np.uint32))
        got = []
        for turn in range(2):
            _ok(native.camelid_hip_paged_attention(drafts.ptr, F32, nh * hd, n, 2, None, nh, n_kv, hd, kc.ptr, vc.ptr, F16,
                                                   pages, ps, dt2.ptr, 1, dl.ptr, 0.09, out.ptr, nh * hd, weights.ptr,
                                                   ws.ptr, size, stat.ptr, None))
            got.append(out.download(np.uint32, n * 2 * nh * hd))
            if turn == 0:
                _ok(native.camelid_hip_paged_evict(kc.ptr, vc.ptr, pages, ps, n_kv, hd, dt2.ptr, 1, dl.ptr, n, weights.ptr,
                                                   64, 16, dl.ptr, kept.ptr, ws2.ptr, evict, stat.ptr, None))
                _ok(native.camelid_hip_synchronize())
                assert dl.download(np.uint32, n).tolist() == [64, 64]
                got.append(kept.download(np.uint32, n * n_kv * 64))
        assert stat.download(np.uint32, 1)[0] == 0
        assert np.isfinite(got[0].view(np.float32)).all() and got[0].view(np.float32).std() > 0.01
        results.append(got)
        for b in (kc, vc):
            b.free()
    for near, off in zip(*results):
        assert (near == off).all()


def test_attention_on_two_streams_at_once(native):
    """Two batches in flight on two streams, each with a workspace of its own, as one after the other."""
    rng = np.random.default_rng(63)
    jobs = []
    for nh, n_kv, lens, new in ((32, 8, [1500] * 12, 5), (32, 2, [6000, 1, 40], 1)):
        pg = Pages(rng, lens, 32, n_kv, 128, F16)
        pg.upload()
        n = len(lens)
        size = native.camelid_hip_paged_attention_workspace(n, new, nh, n_kv, 128, 32, pg.stride, 0)
        q = _dev(rng.normal(0, 1, (n * new, nh * 128)).astype(np.float32))
        pg.dl.upload(np.maximum(pg.lens, new).astype(np.uint32))
        stream = C.c_void_p()
        _hip(native, "hipStreamCreate", C.byref(stream))
        jobs.append((pg, q, n, new, nh, n_kv, _buf(size), size, _buf(n * new * nh * 128 * 4), stream))

    def call(job, stream):
        pg, q, n, new, nh, n_kv, ws, size, out, _ = job
        _ok(native.camelid_hip_paged_attention(q.ptr, F32, nh * 128, n, new, None, nh, n_kv, 128, pg.dk.ptr, pg.dv.ptr, F16,
                                               pg.n_pages, 32, pg.dt.ptr, pg.stride, pg.dl.ptr, 0.1, out.ptr, nh * 128,
                                               None, ws.ptr, size, pg.dstat.ptr, stream))

    def read(job):
        return job[8].download(np.uint32, job[2] * job[3] * job[4] * 128)

    want = []
    for job in jobs:
        call(job, None)
        _ok(native.camelid_hip_synchronize())
        want.append(read(job))
    for _ in range(8):
        for job in jobs:
            call(job, job[9])
    for job, w in zip(jobs, want):
        _hip(native, "hipStreamSynchronize", job[9])
        assert (read(job) == w).all()
    for job in jobs:
        _hip(native, "hipStreamDestroy", job[9])
