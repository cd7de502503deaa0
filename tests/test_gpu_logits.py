"""Penalties, biases and masks on logits on the GPU, against their definition step by step in f32: the same bits."""
import numpy as np
import pytest

from test_gpu_serving import BF16, F16, F32, _dev, _ok, from16, to16, typed

pytestmark = pytest.mark.gpu


def reference(x, history, lens, prompts, drafts, dl, rep, freq, pres, bt, bv, bl, mask):
    """x [n][rows][vocab] f32 values of the logits; rows behind dl[s] as they were."""
    n, rows, vocab = x.shape
    y = x.copy()
    for s in range(n):
        text = [] if history is None else list(history[s, :lens[s]])
        cut = 0 if prompts is None else int(prompts[s])
        for t in range(min(int(dl[s]), rows - 1) + 1):
            more = [] if drafts is None else list(drafts[s, :t])
            seen, count = np.zeros(vocab, bool), np.zeros(vocab, np.int64)
            for i, v in enumerate(text + more):
                if v < vocab:
                    seen[v] = True
                    if i >= cut or i >= len(text):
                        count[v] += 1
            z = y[s, t]
            with np.errstate(invalid="ignore", over="ignore"):
                if rep is not None:
                    z = np.where(seen, np.where(z > 0, z / rep[s], z * rep[s]), z)
                if freq is not None:
                    z = np.where(count > 0, z - freq[s] * count.astype(np.float32), z)
                if pres is not None:
                    z = np.where(count > 0, z - pres[s], z)
                if bt is not None:
                    last = {int(v): k for k, v in enumerate(bt[s, :bl[s]])}
                    for v, k in last.items():
                        if v < vocab:
                            z[v] = z[v] + bv[s, k]
            if mask is not None:
                bits = np.unpackbits(mask[s, t].view(np.uint8), bitorder="little")[:vocab]
                z = np.where(bits == 1, z, -np.float32(np.inf))
            y[s, t] = z.astype(np.float32)
    return y


def run(native, x, lt, in_pad, out_pad, in_place, vocab, history, lens, prompts, drafts, dl, rep, freq, pres, bt, bv, bl,
        mask):
    n, rows = x.shape[:2]
    src = np.full((n, rows, vocab + in_pad), 5, x.dtype)
    src[..., :vocab] = x
    di = _dev(src)
    out0 = src if in_place else np.full((n, rows, vocab + out_pad), 7, x.dtype)
    do = di if in_place else _dev(out0)
    keep = [None if a is None else _dev(np.ascontiguousarray(a)) for a in
            (history, lens, prompts, drafts, dl, rep, freq, pres, bt, bv, bl, mask)]
    h, hl, pl, dr, d, r, f, p, b, v, c, m = [a.ptr if a else None for a in keep]
    _ok(native.camelid_hip_adjust_logits(
        di.ptr, vocab + in_pad, do.ptr, vocab + (in_pad if in_place else out_pad), lt, n, rows, vocab, h,
        0 if history is None else history.shape[1], hl, pl, dr, d, r, f, p, b, v, 0 if bt is None else bt.shape[1], c, m,
        0 if mask is None else mask.shape[2], None))
    got = do.download(out0.dtype, out0.size).reshape(out0.shape)
    assert (got[..., vocab:] == out0[..., vocab:]).all()
    return got[..., :vocab], out0[..., :vocab]


def f32_of(b, t):
    return b.astype(np.float32) if t == F32 else from16(b, t).astype(np.float32)


CASES = [
    # n, rows, vocab, history, biases, mask, in place, type, input and output padding, drafts
    (1, 1, 32000, 300, 0, False, True, F32, 0, 0, False),
    (3, 4, 4097, 50, 7, True, False, BF16, 7, 1, True),
    (2, 8, 1, 9, 2, True, False, F32, 0, 0, True),
    (5, 2, 151936, 5000, 300, True, False, F16, 0, 0, True),
    (2, 3, 8192, 20000, 40, False, True, BF16, 0, 0, True),
    (4, 1, 1000, 64, 1000, False, False, F32, 3, 5, False),
    (2, 5, 4095, 33, 16, True, True, F16, 1, 1, True),
    (1, 32, 777, 0, 0, True, False, BF16, 0, 8, True),
    (3, 7, 50257, 700, 2000, False, False, F32, 0, 0, True),
    (2, 2, 10000, 1000, 16384, True, False, F32, 0, 0, True),
]


@pytest.mark.parametrize("n,rows,vocab,known,biases,masked,in_place,lt,in_pad,out_pad,has_drafts", CASES)
def test_adjusted_logits(native, n, rows, vocab, known, biases, masked, in_place, lt, in_pad, out_pad, has_drafts):
    rng = np.random.default_rng(vocab + known)
    x = typed(rng.normal(0, 3, (n, rows, vocab)), lt)
    tokens = lambda *sh: (rng.random(sh) ** 3 * (vocab + vocab // 50 + 1)).astype(np.uint32)  # noqa: E731 (some >= vocab)
    history = tokens(n, known) if known else None
    lens = rng.integers(0, known + 1, n).astype(np.uint32)
    lens[0] = known
    prompts = rng.integers(0, known + 2, n).astype(np.uint32)
    drafts = tokens(n, rows - 1) if has_drafts and rows > 1 else None
    dl = rng.integers(0, rows, n).astype(np.uint32)
    dl[0] = rows - 1
    rep, freq, pres = (rng.uniform(lo, hi, n).astype(np.float32) for lo, hi in ((0.8, 1.5), (-0.5, 1), (-1, 1)))
    bt = bv = bl = None
    if biases:
        bt, bv = tokens(n, biases), rng.normal(0, 4, (n, biases)).astype(np.float32)
        bl = rng.integers(0, biases + 1, n).astype(np.uint32)
        bl[0] = biases
    mask = rng.integers(0, 1 << 32, (n, rows, (vocab + 31) // 32 + 1), dtype=np.uint32) if masked else None
    if masked and rows > 1:
        mask[0, 0] = 0                      # a grammar that leaves nothing
        mask[-1, -1] = 0xFFFFFFFF
    got, before = run(native, x, lt, in_pad, out_pad, in_place, vocab, history, lens, prompts, drafts, dl, rep, freq, pres,
                      bt, bv, bl, mask)
    want = typed(reference(f32_of(x, lt), history, lens, prompts, drafts, dl, rep, freq, pres, bt, bv, bl, mask), lt)
    for s in range(n):
        k = int(dl[s]) + 1
        same = got[s, :k].view(np.uint16 if lt != F32 else np.uint32) == want[s, :k].view(np.uint16 if lt != F32 else np.uint32)
        assert same.all(), (s, np.argwhere(~same)[:3])
        assert (got[s, k:] == before[s, k:]).all()


@pytest.mark.parametrize("masked", [False, True])
def test_values_that_are_not_numbers(native, masked):
    """Infinities, NaN and zeros; -infinity stays, a masked NaN does not."""
    inf = np.float32(np.inf)
    x = np.zeros((1, 1, 64), np.float32)
    x[0, 0, :8] = [inf, -inf, np.nan, -0.0, 0.0, 1e-45, 3e38, -3e38]
    x[0, 0, 32:40] = x[0, 0, :8]
    history = np.array([list(range(8)) * 2], np.uint32)
    one = lambda v: np.array([v], np.float32)  # noqa: E731
    mask = np.array([[[0xFFFFFFFF, 0]]], np.uint32) if masked else None
    args = (history, np.array([16], np.uint32), None, None, np.array([0], np.uint32), one(1.5), one(0.25), one(0.5), None,
            None, None, mask)
    got, _ = run(native, x, F32, 0, 0, False, 64, *args)
    want = reference(x, *args)
    assert ((got.view(np.uint32) == want.view(np.uint32)) | (np.isnan(got) & np.isnan(want))).all()
    if masked:
        assert (got[0, 0, 32:] == -inf).all()


def test_absent_arguments_and_zero_lengths(native):
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, (2, 3, 500)).astype(np.float32)
    none = (None,) * 12
    got, _ = run(native, x, F32, 0, 0, False, 500, *none)
    assert (got == x).all()
    history = rng.integers(0, 500, (2, 20)).astype(np.uint32)
    huge = np.array([4000000000, 0], np.uint32)           # counts as the stride
    rep = np.array([1.25, 1.25], np.float32)
    got, _ = run(native, x, F32, 0, 0, True, 500, history, huge, None, None, None, rep, None, None, None, None, None, None)
    want = reference(x, history, [20, 0], None, None, [2, 2], rep, None, None, None, None, None, None)
    assert (got.view(np.uint32) == want.view(np.uint32)).all()
    # lens beyond the rows count as all of them
    got, _ = run(native, x, F32, 0, 0, False, 500, history, None, None, None, np.array([9, 1], np.uint32), rep, None, None,
                 None, None, None, None)
    want = reference(x, history, [20, 20], None, None, [2, 1], rep, None, None, None, None, None, None)
    assert (got[0] == want[0]).all() and (got[1, :2] == want[1, :2]).all() and (got[1, 2] == 7).all()
