"""Rows in 8-bit floating point, their scores and score rows as distributions (comet_fp8_*, comet_logprobs_*) against plain restatements in 64 bits.

Tolerances. Quantised values, rows read back and ids are compared exactly. A score is a sum of K exact products formed in float32: each of the K additions
is off by at most one step (2^-23) of a partial sum that never exceeds sum |q r|, so by K * 2^-23 * sum |q r| in all, plus half a step of the output type.
A log-probability is d - log S with d = (s - max) * scale: two roundings of d and one of the difference (2^-23 (|d| + |lp|)), and log S, whose S is off
relatively by the additions a thread makes one after the other (16 per chunk of 4096 columns, 2^-24 each, and eight joins), by the exponent's rounding
(3 * 2^-24 |t| weighted by p: the mean of |d| is at most H + log S) and by the exponential's last place: together 2^-23 (16 n / 8192 + 16 + |d| + |lp| + 3 (H + log S)).
The entropy adds log S and a mean of |d| with the same relative error; logsum the rounding of max * scale."""
import threading

import numpy as np
import pytest

import fp8_ref as ref
from comet_amd import CometError, Fp8Rows, LogProbs

pytestmark = pytest.mark.gpu
DTYPES = ["f32", "f16", "bf16"]


class Dev:
    """device arrays of one test"""

    def __init__(self, ctx):
        self.ctx, self.ptrs = ctx, []

    def put(self, a):
        a = np.ascontiguousarray(a)
        p = self.ctx.alloc(max(a.nbytes, 16))
        self.ptrs.append(p)
        if a.nbytes:
            self.ctx.upload(p, a)
        return p

    def new(self, shape, dtype, fill=0x5A):
        return self.put(np.full(int(np.prod(shape)) * np.dtype(dtype).itemsize, fill, np.uint8))

    def get(self, p, shape, dtype):
        self.ctx.sync()
        return self.ctx.download(p, shape, dtype) if int(np.prod(shape)) else np.empty(shape, dtype)

    def close(self):
        self.ctx.sync()
        for p in self.ptrs:
            self.ctx.free(p)


@pytest.fixture
def dev(ctx):
    d = Dev(ctx)
    yield d
    d.close()


def rows_of(seed, n, dim):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, dim)) * np.exp(rng.standard_normal(dim))
    return (x / np.maximum(np.linalg.norm(x, axis=1, keepdims=True), 1e-30)).astype(np.float32)


def write(dev, store, x, dtype="f32", pad=0, slots=None, first=0, offset=0):
    """x (float32 values) as a device matrix of stride dim + pad that starts `offset` elements into its allocation"""
    n, dim = x.shape
    buf = np.full(offset + n * (dim + pad), 77, ref.NP[dtype])
    buf[offset:].reshape(n, dim + pad)[:, :dim] = ref.encode(x, dtype)
    p = dev.put(buf) + offset * buf.itemsize
    store.write_dev(p, n, dtype, ld=dim + pad, slots=dev.put(np.asarray(slots, np.int64)) if slots is not None else 0, first=first)


def read(dev, store, n, dtype="f32", pad=0, slots=None, first=0, offset=0):
    dim, es = store.dim, np.dtype(ref.NP[dtype]).itemsize
    size = offset + n * (dim + pad)
    p = dev.new((size,), ref.NP[dtype])
    store.read_dev(p + offset * es, n, dtype, ld=dim + pad, slots=dev.put(np.asarray(slots, np.int64)) if slots is not None else 0, first=first)
    raw = dev.get(p, (size,), ref.NP[dtype])
    untouched = np.full(1, 0x5A5A5A5A, np.uint32).view(np.uint8)[:es].copy().view(ref.NP[dtype])[0]
    out = raw[offset:].reshape(n, dim + pad)
    bits = {2: np.uint16, 4: np.uint32}[es]
    assert (raw[:offset].view(bits) == untouched.view(bits)).all() and (np.ascontiguousarray(out[:, dim:]).view(bits) == untouched.view(bits)).all()
    return ref.decode(out[:, :dim], dtype)


def same(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return a.shape == b.shape and bool(((a == b) | (np.isnan(a) & np.isnan(b))).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,dim,pad,offset", [(1, 1, 0, 0), (3, 5, 2, 1), (7, 127, 0, 0), (9, 128, 1, 0), (130, 129, 0, 1), (65, 300, 7, 3), (33, 768, 0, 0), (5, 1000, 5, 1), (2, 4111, 0, 0)])
def test_write_then_read(ctx, dev, dtype, n, dim, pad, offset):
    x = ref.decode(ref.encode(rows_of(n + dim, n, dim), dtype), dtype)
    store = Fp8Rows(ctx, n + 3, dim)
    write(dev, store, x, dtype, pad, first=2, offset=offset)
    want = ref.held(x)
    for out in DTYPES:
        got = read(dev, store, n, out, pad, first=2, offset=offset)
        assert same(got, ref.decode(ref.encode(want.astype(np.float32), out), out)), out
    assert same(read(dev, store, 2), np.zeros((2, dim))) and same(read(dev, store, 1, first=n + 2), np.zeros((1, dim)))
    store.close()


def test_values_where_the_format_can_go_wrong(ctx, dev):
    """zeros, infinities and NaN in a block, its largest value at and next to 448 * 2^e, ties, subnormals, the ends of float32"""
    dim = 256
    base = rows_of(1, 24, dim)
    x = base.copy()
    x[0] = 0
    x[1] = -0.0
    x[2, 3], x[2, 200] = np.nan, np.inf
    x[3] = -np.inf
    x[4] = np.nan
    for i, a in enumerate([448.0, np.nextafter(np.float32(448), np.float32(1e9)), np.nextafter(np.float32(448), np.float32(0)), 1.75, np.nextafter(np.float32(1.75), np.float32(9)), 2.0 ** -120]):
        x[5 + i] = 0.01 * a * base[5 + i]
        x[5 + i, 7] = a
    k = np.arange(dim)
    x[11] = np.where(k % 128 == 0, 448, 16 + (k % 64) * 0.25)          # between the numbers of a step of 1 and of 2: exact ties among them
    x[12] = np.where(k % 128 == 0, 448, (k % 128 - 64) * 2.0 ** -10)   # half steps of the codes below 2^-6
    x[13] = 3.4028235e38
    x[13, ::3] = 1.0
    x[14] = 1e-38 * np.sign(base[14])
    x[15] = 1e-44
    x[16] = np.where(k < 128, 1e-42, 1e-30) * base[16]
    x[17, 5] = 3e38
    store = Fp8Rows(ctx, 24, dim)
    write(dev, store, x)
    # the nearest code to the largest float32 stands for 2^128 (its block's e is 120: 255.99 rounds to 256), which float32 holds as infinity
    with np.errstate(over="ignore"):
        assert same(read(dev, store, 24), ref.held(x).astype(np.float32))
    assert np.signbit(read(dev, store, 2)[1]).all()
    store.close()


@pytest.mark.parametrize("dtype,pad,offset", [("f32", 0, 0), ("f32", 3, 1), ("f16", 1, 0), ("bf16", 0, 0), ("bf16", 5, 3)])
@pytest.mark.parametrize("dim", [1, 7, 16, 17, 32, 33, 40, 63, 64, 65, 100, 128])
def test_rows_of_up_to_one_block(ctx, dev, dtype, pad, offset, dim):
    """narrow rows share a wave: consecutive slots, few rows and many rows to given slots, some named twice, some outside"""
    rng = np.random.default_rng(dim)
    capacity = 700
    R = Fp8Rows(ctx, capacity, dim)
    held = np.zeros((capacity, dim))
    for n, given in ((333, False), (50, True), (600, True)):
        x = ref.decode(ref.encode((rng.standard_normal((n, dim)) * np.exp(4 * rng.standard_normal((n, 1)))).astype(np.float32), dtype), dtype)
        slots = rng.integers(-2, capacity + 2, n) if given else np.arange(100, 100 + n)
        write(dev, R, x, dtype, pad, slots if given else None, 0 if given else 100, offset)
        h = ref.held(x)
        for i, at in enumerate(slots):
            if 0 <= at < capacity:
                held[at] = h[i]
        want = ref.decode(ref.encode(held.astype(np.float32), dtype), dtype)
        assert same(read(dev, R, capacity, dtype, pad, None, 0, offset), want)
        assert same(read(dev, R, n, dtype, pad, slots, 0, offset), np.where(((slots >= 0) & (slots < capacity))[:, None], want[np.clip(slots, 0, capacity - 1)], 0.0))
    one = np.ones((3, dim), np.float32)                     # what lies behind the rows' width adds nothing to a product
    Q = Fp8Rows(ctx, 3, dim)
    write(dev, Q, one)
    got, want, mag = scores(dev, Q, 3, R, capacity), held.sum(axis=1), np.abs(held).sum(axis=1)
    assert ((np.abs(got - want) <= dim * 2.0 ** -23 * mag) | (np.isnan(got) & np.isnan(want))).all()       # float16 rows hold infinities: NaN
    Q.close(); R.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [2, 64, 65, 1000, 5000])
def test_slots_repeated_and_outside(ctx, dev, n, dtype):
    """of rows with one slot the last stays; rows with a slot outside the store are skipped; every other slot keeps what it held"""
    dim, cap = 200, 400
    rng = np.random.default_rng(n)
    x0, x1, x2 = (ref.decode(ref.encode(rows_of(n + i, r, dim), dtype), dtype) for i, r in enumerate((cap, n, n)))
    store = Fp8Rows(ctx, cap, dim)
    write(dev, store, x0, dtype)
    want = ref.held(x0)
    for x in (x1, x2):          # twice: what the first call leaves behind serves the second
        slots = rng.integers(-2, cap + 2, n)
        slots[0], slots[-1] = 7, 7
        slots[n // 2] = 2 ** 40
        write(dev, store, x, dtype, slots=slots)
        h = ref.held(x)
        for i, s in enumerate(slots):
            if 0 <= s < cap:
                want[s] = h[i]
    assert same(read(dev, store, cap), want)
    at = rng.integers(-3, cap + 3, 777)
    at[5] = -2 ** 62
    ok = (at >= 0) & (at < cap)
    assert same(read(dev, store, 777, slots=at), np.where(ok[:, None], want[np.clip(at, 0, cap - 1)], 0.0))
    store.close()


def scores(dev, q, m, r, n, dtype="f32", pad=0, q_first=0, first=0, offset=0):
    es = np.dtype(ref.NP[dtype]).itemsize
    size = offset + m * (n + pad) + 8
    p = dev.new((size,), ref.NP[dtype])
    r.scores_dev(q, m, p + offset * es, dtype, ld=n + pad, q_first=q_first, first=first, n=n)
    raw = dev.get(p, (size,), ref.NP[dtype])
    out = raw[offset:offset + m * (n + pad)].reshape(m, n + pad)
    bits = {2: np.uint16, 4: np.uint32}[es]
    fill = {2: 0x5A5A, 4: 0x5A5A5A5A}[es]
    for part in (raw[:offset], np.ascontiguousarray(out[:, n:]), raw[offset + m * (n + pad):]):
        assert (part.view(bits) == fill).all()
    return ref.decode(out[:, :n], dtype)


@pytest.mark.parametrize("dtype,pad,offset", [("f32", 0, 0), ("f16", 3, 1), ("bf16", 1, 0)])
@pytest.mark.parametrize("m,n,dim", [(1, 1, 1), (1, 1000, 128), (2, 17, 129), (15, 255, 300), (16, 256, 768), (17, 257, 640), (33, 300, 513), (64, 511, 384), (65, 700, 1000), (100, 129, 2048),
                                     (129, 1025, 96), (255, 260, 1537), (256, 512, 768), (300, 2111, 200), (513, 777, 1100)])
def test_scores_against_64_bits(ctx, dev, m, n, dim, dtype, pad, offset):
    q, r = rows_of(m, m, dim), rows_of(n + 1, n, dim)
    Q, R = Fp8Rows(ctx, m + 2, dim), Fp8Rows(ctx, n + 5, dim)
    write(dev, Q, q, first=1); write(dev, R, r, first=4)
    hq, hr = ref.held(q), ref.held(r)
    want, mag = hq @ hr.T, np.abs(hq) @ np.abs(hr).T
    got = scores(dev, Q, m, R, n, dtype, pad, q_first=1, first=4, offset=offset)
    tol = dim * 2.0 ** -23 * mag + ref.EPS[dtype] * np.abs(want) * 1.01 + (2.0 ** -25 if dtype == "f16" else 0)     # 2^-25: half the step of subnormal fp16
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])
    Q.close(); R.close()


@pytest.mark.parametrize("m,n,dim", [(1, 500, 257), (16, 300, 1000), (48, 333, 128), (200, 600, 900), (257, 1030, 640)])
def test_scores_of_whole_numbers_are_exact(ctx, dev, m, n, dim):
    """numbers of up to three bits times the blocks' powers of two: every sum is a whole number below 2^24, whatever the order"""
    rng = np.random.default_rng(dim)
    q, r = rng.integers(-7, 8, (m, dim)).astype(np.float32), rng.integers(-7, 8, (n, dim)).astype(np.float32)
    q[0], r[-1] = 0, 0
    for c in range(0, dim, 256):       # every other block four times as large
        q[:, c:c + 128] *= 4
    Q, R = Fp8Rows(ctx, m, dim), Fp8Rows(ctx, n, dim)
    write(dev, Q, q); write(dev, R, r)
    assert same(scores(dev, Q, m, R, n), q.astype(np.float64) @ r.astype(np.float64).T)
    Q.close(); R.close()


@pytest.mark.parametrize("m,n,dim", [(4, 30001, 300), (5, 100003, 100), (20, 80001, 200), (130, 70001, 130), (300, 40003, 100), (520, 33000, 300), (256, 66000, 20)])
def test_scores_over_many_tiles(ctx, dev, m, n, dim):
    """more tiles than run at once, of one block and of a few: a workgroup's next tile arrives while it finishes the last"""
    rng = np.random.default_rng(n)
    q, r = rng.integers(-7, 8, (m, dim)).astype(np.float32), rng.integers(-7, 8, (n, dim)).astype(np.float32)
    Q, R = Fp8Rows(ctx, m, dim), Fp8Rows(ctx, n, dim)
    write(dev, Q, q); write(dev, R, r)
    assert same(scores(dev, Q, m, R, n), q.astype(np.float64) @ r.astype(np.float64).T)
    assert same(scores(dev, Q, m, R, n - 5, "bf16", pad=3, first=2), ref.from_bf16_bits(ref.to_bf16_bits(q @ r[2:n - 3].T)))
    Q.close(); R.close()


def test_a_pair_has_one_score(ctx, dev):
    """the score of a query and a row does not depend on what they are multiplied with: few queries, tiles of every shape, any window"""
    n, dim, m = 9000, 700, 600
    q, r = rows_of(31, m, dim), rows_of(32, n, dim)
    Q, R = Fp8Rows(ctx, m, dim), Fp8Rows(ctx, n, dim)
    write(dev, Q, q); write(dev, R, r)
    whole = scores(dev, Q, m, R, n)
    for q0, mm, r0, nn in ((0, 1, 0, n), (17, 3, 5, 777), (100, 5, 11, 4001), (33, 64, 1, 300), (1, 599, 8000, 1000), (300, 129, 257, 8000)):
        assert same(scores(dev, Q, mm, R, nn, q_first=q0, first=r0), whole[q0:q0 + mm, r0:r0 + nn])
    Q.close(); R.close()


@pytest.mark.parametrize("m", [1, 40, 300])
def test_scores_of_non_finite_and_far_apart_rows(ctx, dev, m):
    """a NaN stays in its row's and its query's scores; blocks at both ends of the scales' range keep their products"""
    n, dim = 400, 384
    q, r = rows_of(3, m, dim), rows_of(4, n, dim)
    r[5, 9] = np.nan
    r[300, 380] = np.inf
    q[m - 1, 130] = -np.inf
    r[7, :128] *= 2.0 ** 100
    r[8, :128], r[8, 128:] = r[8, :128] * 2.0 ** -100, 0
    r[9] = 0
    Q, R = Fp8Rows(ctx, m, dim), Fp8Rows(ctx, n, dim)
    write(dev, Q, q); write(dev, R, r)
    got = scores(dev, Q, m, R, n)
    hq, hr = ref.held(q), ref.held(r)
    with np.errstate(invalid="ignore"):
        want, mag = hq @ hr.T, np.abs(hq) @ np.abs(hr).T
    assert (np.isnan(got) == np.isnan(want)).all() and np.isnan(got[:, [5, 300]]).all() and np.isnan(got[m - 1]).all()
    ok = ~np.isnan(want)
    assert (np.abs(got - want)[ok] <= (dim * 2.0 ** -23 * mag + 2.0 ** -140)[ok]).all()
    Q.close(); R.close()


def test_rows_and_scores_behind_four_gibibytes(ctx, dev):
    dim, cap = 1024, (1 << 22) + 1000           # 4 GiB of codes and a little more
    n, m = 900, 70
    x = rows_of(11, n, dim)
    store = Fp8Rows(ctx, cap, dim)
    write(dev, store, x, first=cap - n)
    write(dev, store, x[:5], slots=[cap - n - 1, 3, cap - n - 7, 1 << 22, 0])
    h = ref.held(x)
    assert same(read(dev, store, n, first=cap - n), h)
    assert same(read(dev, store, 4, slots=[3, cap - n - 7, cap - n - 2, 1 << 22]), np.stack([h[1], h[2], 0 * h[0], h[3]]))
    Q = Fp8Rows(ctx, m, dim)
    q = rows_of(12, m, dim)
    write(dev, Q, q)
    hq = ref.held(q)
    for mm in (3, m):
        got = scores(dev, Q, mm, store, n, first=cap - n)
        assert (np.abs(got - hq[:mm] @ h.T) <= dim * 2.0 ** -23 * (np.abs(hq[:mm]) @ np.abs(h).T)).all()
    Q.close(); store.close()


# ---- log-probabilities -------------------------------------------------------------------------------------------------
def run_logprobs(ctx, dev, s, dtype, n, pad, counts, scale, targets, k, plan=None, offset=0):
    m = s.shape[0]
    buf = np.full(offset + m * (n + pad), 0, ref.NP[dtype])
    buf[offset:].reshape(m, n + pad)[:, :n] = ref.encode(s, dtype)
    buf[offset:].reshape(m, n + pad)[:, n:] = ref.encode(np.float32(np.nan), dtype)      # never read
    p = dev.put(buf) + offset * buf.itemsize
    T = 0 if targets is None else targets.shape[1]
    o = {"logsum": (m,), "entropy": (m,), "logprobs": (m, T), "ids": (m, k), "top": (m, k)}
    ptr = {a: dev.new(sh, np.float32) for a, sh in o.items()}
    own = plan or LogProbs(ctx, m, n, k)
    own.run_dev(p, dtype, m, n, ld=n + pad, scale=scale, counts=dev.put(np.asarray(counts, np.int32)) if counts is not None else 0,
                targets=dev.put(np.asarray(targets, np.int32)) if T else 0, n_targets=T, k=k, out_logprobs=ptr["logprobs"] if T else 0, out_logsum=ptr["logsum"],
                out_entropy=ptr["entropy"], out_ids=ptr["ids"] if k else 0, out_top_logprobs=ptr["top"] if k else 0)
    got = {a: dev.get(ptr[a], sh, np.int32 if a == "ids" else np.float32) for a, sh in o.items()}
    if plan is None:
        own.close()
    return got


def close(got, want, tol):
    with np.errstate(invalid="ignore", over="ignore"):
        got, want = got.astype(np.float64), np.asarray(want, np.float64)
        want = np.where(np.isinf(want.astype(np.float32)), want.astype(np.float32), want)       # beyond float32: its infinity
        ok = (np.abs(got - want) <= tol) | (got == want) | (np.isnan(got) & np.isnan(want))
    assert ok.all(), (np.argwhere(~ok)[:4], got[~ok][:4], want[~ok][:4])


def check_logprobs(got, s, n, counts, scale, targets, k):
    L, H, lp, ids, tl = ref.logprobs(s, n, counts, scale, targets, k)
    assert (got["ids"] == ids).all(), np.argwhere(got["ids"] != ids)[:4]
    with np.errstate(invalid="ignore", over="ignore"):
        top = np.where(np.isfinite(L), np.nanmax(np.where(np.isfinite(s[:, :n] * np.float64(scale)), s[:, :n] * np.float64(scale), -np.inf), axis=1, initial=-np.inf), 0.0)
        top = np.where(np.isfinite(top), top, 0.0)
        log_s = np.where(np.isfinite(L), np.maximum(L - top, 0), 0.0)
        if counts is not None:           # the maximum above may lie behind the count: bound log S by the number of columns instead
            log_s = np.full(len(L), np.log(max(n, 2)))
        base = 16 * n / 8192 + 16 + 3 * (np.where(np.isfinite(H), H, 0) + log_s)
        unit = 2.0 ** -23
        close(got["logprobs"], lp, unit * (base[:, None] + 2 * np.abs(np.where(np.isfinite(lp), lp, 0)) + log_s[:, None]))
        close(got["top"], tl, unit * (base[:, None] + 2 * np.abs(np.where(np.isfinite(tl), tl, 0)) + log_s[:, None]))
        close(got["logsum"], L, unit * (base + 2 * np.abs(top) + np.abs(np.where(np.isfinite(L), L, 0))))
        close(got["entropy"], H, unit * (base * (1 + np.where(np.isfinite(H), H, 0))))


def score_rows(seed, m, n, kind="normal"):
    rng = np.random.default_rng(seed)
    s = rng.standard_normal((m, n)).astype(np.float32)
    if kind == "ties":
        s = np.round(s * 2) / 2
    if kind == "equal":
        s[:] = -0.75
    if kind in ("ascending", "descending"):
        s = np.sort(s, axis=1)[:, ::1 if kind == "ascending" else -1]
    if kind == "zeros":
        s = np.where(s > 0, np.float32(0.0), np.float32(-0.0))
    if kind == "one thread":       # the best of a chunk all belong to the columns of one thread
        s[:, ::1024] += 50
        s[:, 1::1024] += 40
    return np.ascontiguousarray(s)


@pytest.mark.parametrize("dtype,pad,offset", [("f32", 0, 0), ("f16", 1, 1), ("bf16", 5, 3)])
@pytest.mark.parametrize("m,n,k,scale", [(1, 1, 1, 1.0), (2, 5, 10, -1.0), (1, 255, 0, 0.5), (3, 257, 128, 20.0), (5, 4096, 1, 1.0), (1, 8191, 10, -4.0), (2, 8192, 100, 3.0), (300, 2049, 33, 1.0),
                                         (1, 8193, 128, 1.0), (2, 40001, 100, 20.0), (1100, 9001, 5, -1.0), (1, 300007, 128, 2.0), (7, 100003, 64, 1.0)])
def test_logprobs_against_64_bits(ctx, dev, m, n, k, scale, dtype, pad, offset):
    s = ref.decode(ref.encode(score_rows(m + n, m, n), dtype), dtype)
    targets = np.random.default_rng(n).integers(-1, n + 1, (m, 3)).astype(np.int32)
    targets[0] = [0, n - 1, n]
    got = run_logprobs(ctx, dev, s, dtype, n, pad, None, scale, targets, k, offset=offset)
    check_logprobs(got, s, n, None, scale, targets, k)


@pytest.mark.parametrize("kind", ["ties", "equal", "ascending", "descending", "zeros", "one thread"])
@pytest.mark.parametrize("m,n,k,scale", [(2, 30000, 128, 1.0), (2, 30000, 17, -2.0), (1, 70000, 100, 1.0), (1100, 9000, 128, 1.0)])
def test_logprobs_of_rows_in_awkward_orders(ctx, dev, m, n, k, scale, kind):
    s = score_rows(m + n, m, n, kind)
    check_logprobs(run_logprobs(ctx, dev, s, "f32", n, 0, None, scale, None, k), s, n, None, scale, None, k)


@pytest.mark.parametrize("kind", ["normal", "ties", "ascending", "descending", "equal"])
@pytest.mark.parametrize("m,k", [(1, 128), (2, 1), (3, 30)])
def test_logprobs_of_rows_in_hundreds_of_splits(ctx, dev, m, k, kind):
    """the best columns of all splits, or of one split alone, are found however few turns the joining takes"""
    n = 1000003
    s = score_rows(m + k, m, n, kind)
    check_logprobs(run_logprobs(ctx, dev, s, "f32", n, 0, None, 1.5, None, k), s, n, None, 1.5, None, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [1, 20, 32, 33, 100, 128])
def test_logprobs_of_rows_that_end_early_in_a_chunk(ctx, dev, dtype, k):
    """rows whose last columns are more candidates than are held at once and lie in few threads"""
    counts = np.array([513, 514, 600, 640, 641, 800, 1023, 1025, 2000, 4096 + 513, 4096 + 600, 8192 + 639, 0, 512], np.int32)
    n = int(counts.max())
    for kind in ("normal", "ascending", "ties"):
        s = ref.decode(ref.encode(score_rows(n + k, len(counts), n, kind), dtype), dtype)
        check_logprobs(run_logprobs(ctx, dev, s, dtype, n, 1, counts, 2.0, None, k), s, n, counts, 2.0, None, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1.0, -3.0])
@pytest.mark.parametrize("n", [200, 20000])
def test_logprobs_of_masked_ragged_and_non_finite_rows(ctx, dev, dtype, scale, n):
    m, k = 24, 40
    s = ref.decode(ref.encode(score_rows(n, m, n), dtype), dtype)
    mask = np.float32(-np.inf if scale > 0 else np.inf)
    low = {"f32": np.float32(3.4028235e38), "f16": np.float32(65504.0), "bf16": ref.from_bf16_bits(np.uint16(0x7F7F))}[dtype] * (-1 if scale > 0 else 1)
    counts = np.random.default_rng(n).integers(0, n + 1, m).astype(np.int32)
    counts[:8] = [0, 1, n, n, n, n + 50, -7, 2]
    s[2] = mask                           # nothing left
    s[3, : n - 1] = mask                  # one entry left, the last
    s[4, 1::2] = mask
    s[5] = low                            # masks of the type's lowest value: a row of them is uniform
    s[8, 3:] = low
    counts[8:14] = n
    s[9, 7] = np.nan
    s[10, n - 1] = -mask                  # the scaled score is +inf
    s[11] = np.nan
    s[12, : n // 2] = mask; s[12, n // 2:] = low
    s[13] = mask; s[13, 5] = np.nan
    counts[14] = n // 2; s[14, n // 2:] = np.nan       # behind the count: not part of the row
    targets = np.random.default_rng(1).integers(-1, n + 1, (m, 2)).astype(np.int32)
    targets[:, 0] = 1
    got = run_logprobs(ctx, dev, s, dtype, n, 3, counts, scale, targets, k)
    check_logprobs(got, s, n, counts, scale, targets, k)
    assert got["logsum"][0] == -np.inf and got["entropy"][0] == 0 and (got["ids"][[0, 2, 6]] == -1).all() and (got["logprobs"][[0, 2, 6]] == -np.inf).all()


def test_logprobs_of_no_columns_and_no_rows(ctx, dev):
    got = run_logprobs(ctx, dev, np.empty((3, 0), np.float32), "f32", 0, 4, None, 1.0, np.zeros((3, 1), np.int32), 2)
    assert (got["logsum"] == -np.inf).all() and (got["entropy"] == 0).all() and (got["ids"] == -1).all() and (got["logprobs"] == -np.inf).all() and (got["top"] == -np.inf).all()
    LogProbs(ctx, 0, 10, 1).run_dev(0, "f32", 0, 10, out_logsum=0, out_entropy=0, k=1)


def test_logprobs_plan_serves_smaller_calls(ctx, dev):
    plan = LogProbs(ctx, 64, 60000, 50)
    for m, n, k in [(64, 60000, 50), (1, 60000, 3), (2, 50001, 50), (63, 9000, 0), (5, 10, 10), (64, 60000, 50)]:
        s = score_rows(m, m, n)
        check_logprobs(run_logprobs(ctx, dev, s, "f32", n, 0, None, 2.0, None, k, plan=plan), s, n, None, 2.0, None, k)
    plan.close()


# ---- together ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,n,dim,k,scale", [(1, 500, 64, 10, 8.0), (20, 9000, 300, 100, 20.0), (70, 20000, 128, 5, -3.0)])
def test_write_score_rank_and_read_back_as_one_run(ctx, dev, B, n, dim, k, scale):
    """the store's rows written, queries scored against a window of them, the best slots read back; the same through the host call"""
    cap, first = n + 40, 17
    x, q = rows_of(n, n, dim), rows_of(B, B, dim)
    slots = np.random.default_rng(n).permutation(n) + first
    R, Q = Fp8Rows(ctx, cap, dim), Fp8Rows(ctx, B, dim)
    write(dev, R, x, slots=slots); write(dev, Q, q)
    s = scores(dev, Q, B, R, n, first=first)
    got = run_logprobs(ctx, dev, s, "f32", n, 0, None, scale, None, k)
    check_logprobs(got, s, n, None, scale, None, k)
    best = got["ids"][0].astype(np.int64) + first
    at = np.argsort(slots)                      # slot first + j holds row at[j]
    assert same(read(dev, R, k, slots=best), ref.held(x)[at[got["ids"][0]]])
    r = R.search(q, k, scale, first=first, n=n)
    assert (r.slots == got["ids"] + first).all() and (r.logprobs == got["top"]).all() and (r.logsum == got["logsum"]).all() and (r.entropy == got["entropy"]).all()
    # the host forms of write and read leave and give the same
    H = Fp8Rows(ctx, cap, dim)
    H.write(x, slots)
    assert same(H.read(np.arange(cap)), read(dev, R, cap))
    for o in (R, Q, H):
        o.close()


def test_search_of_narrow_rows_behind_one_of_wide_rows(ctx):
    """the queries' padding is zero whatever an earlier call left in the workspace"""
    wide = Fp8Rows(ctx, 300, 128)
    wide.write(rows_of(60, 300, 128), np.arange(300))
    narrow = Fp8Rows(ctx, 500, 20)
    x, q = rows_of(61, 500, 20), rows_of(62, 9, 20)
    narrow.write(x, np.arange(500))
    hq, hx = ref.held(q), ref.held(x)
    s = hq @ hx.T
    for turn in range(3):
        wide.search(np.full((200, 128), 3.0, np.float32), 10, 1.0)
        r = narrow.search(q, 1, 50.0)
        best = s.argmax(axis=1)
        assert (r.slots[:, 0] == best).all()
        want = (50 * (s - s.max(axis=1, keepdims=True)))
        # 20 additions of products below 1 move a score by 20 * 2^-23 at most, times the scale
        assert (np.abs(r.logprobs[:, 0] + np.log(np.exp(want).sum(axis=1))) <= 50 * 2 * 20 * 2.0 ** -23 + 64 * 2.0 ** -23).all()
    wide.close(); narrow.close()


def test_search_of_many_queries_runs_in_pieces(ctx):
    n, dim, B, k = 1_200_000, 16, 500, 3        # 2.4 GB of scores: three pieces
    x, q = rows_of(5, n, dim), rows_of(6, B, dim)
    R = Fp8Rows(ctx, n, dim)
    R.write(x, np.arange(n))
    r = R.search(q, k, 10.0)
    one = [R.search(q[i], k, 10.0) for i in (0, 222, 223, 447, 499)]
    for i, o in zip((0, 222, 223, 447, 499), one):
        assert (r.slots[i] == o.slots[0]).all() and abs(r.logsum[i] - o.logsum[0]) < 2 * 2.0 ** -23 * (16 * n / 8192 + 60)
    R.close()


def test_searches_from_several_threads(ctx):
    x, q = rows_of(8, 3000, 96), rows_of(9, 4, 96)
    R = Fp8Rows(ctx, 3000, 96)
    R.write(x, np.arange(3000))
    want = R.search(q, 7, 5.0)
    bad = []

    def work():
        for _ in range(10):
            r = R.search(q, 7, 5.0)
            if not ((r.slots == want.slots).all() and (r.logprobs == want.logprobs).all()):
                bad.append(1)
    t = [threading.Thread(target=work) for _ in range(4)]
    [i.start() for i in t]; [i.join() for i in t]
    assert not bad
    R.close()


# ---- calls of more than one launch ---------------------------------------------------------------------------------
def test_writes_and_reads_of_more_rows_than_one_launch_takes(ctx, dev):
    n, capacity = (1 << 22) + 70, 1000
    rng = np.random.default_rng(5)
    x, slots = rng.standard_normal((n, 1)).astype(np.float32), rng.integers(-1, capacity, n)
    slots[5], slots[(1 << 22) + 3] = 7, 7                     # one slot in both launches
    R = Fp8Rows(ctx, capacity, 1)
    write(dev, R, x, slots=slots)
    last = np.full(capacity + 1, -1)
    last[slots] = np.arange(n)                                # numpy keeps the last of equal indices
    want = ref.held(x[last[:capacity]])
    assert same(R.read(np.arange(capacity)), want)
    n = (1 << 24) + 300
    slots = rng.integers(-1, capacity + 1, n)
    got = read(dev, R, n, "f16", slots=slots)[:, 0]
    want = np.append(want[:, 0].astype(np.float16).astype(np.float64), [0.0, 0.0])
    assert (got == want[np.where((slots < 0) | (slots >= capacity), capacity, slots)]).all()
    R.close()


def test_scores_of_more_queries_and_rows_than_one_launch_takes(ctx, dev):
    rng = np.random.default_rng(6)
    q, r = rng.integers(-7, 8, ((1 << 16) + 9, 3)).astype(np.float32), rng.integers(-7, 8, (6, 3)).astype(np.float32)
    Q, R = Fp8Rows(ctx, len(q), 3), Fp8Rows(ctx, 6, 3)
    write(dev, Q, q); write(dev, R, r)
    assert same(scores(dev, Q, len(q), R, 6, pad=1), q.astype(np.float64) @ r.astype(np.float64).T)
    Q.close(); R.close()
    n, m = (1 << 24) + 40, 5
    q, r = rng.integers(-7, 8, (m, 1)).astype(np.float32), rng.integers(-7, 8, (n, 1)).astype(np.float32)
    Q, R = Fp8Rows(ctx, m, 1), Fp8Rows(ctx, n, 1)
    write(dev, Q, q); write(dev, R, r)
    for mm in (3, m):                                         # both kernels
        out = dev.new((mm, n), np.float32)
        R.scores_dev(Q, mm, out)
        got = dev.get(out, (mm, n), np.float32)
        for a, b in ((0, 500), ((1 << 24) - 300, n)):
            assert (got[:, a:b] == q[:mm] * r[a:b, 0]).all()
    Q.close(); R.close()


def test_logprobs_of_more_rows_than_one_launch_takes(ctx, dev):
    m, n = (1 << 22) + 9, 3
    s = score_rows(9, m, n)
    counts = np.random.default_rng(1).integers(0, n + 1, m).astype(np.int32)
    got = run_logprobs(ctx, dev, s, "f32", n, 0, counts, -2.0, None, 1)
    for a, b in ((0, 300), ((1 << 22) - 100, m)):
        check_logprobs({x: v[a:b] for x, v in got.items()}, s[a:b], n, counts[a:b], -2.0, None, 1)


# ---- refusals ----------------------------------------------------------------------------------------------------------
def test_refusals(ctx, dev):
    for cap, dim in ((0, 8), (-1, 8), (8, 0), (8, -4), (1 << 40, 8), (1, (1 << 20) + 1)):
        with pytest.raises(CometError):
            Fp8Rows(ctx, cap, dim)
    R, S = Fp8Rows(ctx, 50, 100), Fp8Rows(ctx, 50, 101)
    x = dev.new((50, 128), np.float32)
    bad = [lambda: R.write_dev(x, 51), lambda: R.write_dev(x, 1, first=50), lambda: R.write_dev(x, 1, first=-1), lambda: R.write_dev(x, 2, ld=99), lambda: R.write_dev(0, 1),
           lambda: R.write_dev(x + 1, 1), lambda: R.write_dev(x + 2, 1), lambda: R.write_dev(x, -1), lambda: R.write_dev(x, 2, ld=2 ** 62), lambda: R.write_dev(x, 1, slots=x + 4),
           lambda: R.read_dev(x, 51), lambda: R.read_dev(x, 1, ld=1), lambda: R.read_dev(0, 1), lambda: R.read_dev(x + 1, 1, "bf16"), lambda: R.read_dev(x, -1, slots=x),
           lambda: R.scores_dev(S, 1, x), lambda: R.scores_dev(R, 51, x), lambda: R.scores_dev(R, 1, x, first=1, n=50), lambda: R.scores_dev(R, -1, x), lambda: R.scores_dev(R, 2, x, ld=49),
           lambda: R.scores_dev(R, 2, 0), lambda: R.scores_dev(R, 1, x, q_first=2 ** 62), lambda: R.write(np.zeros((2, 100)), [0, 50]), lambda: R.read([-1]),
           lambda: R.search(np.zeros(100), 3, 0.0), lambda: R.search(np.zeros(100), 3, float("nan")), lambda: R.search(np.zeros(100), 129), lambda: R.search(np.zeros(100), -1),
           lambda: R.search(np.zeros(100), 1, n=51)]
    for f in bad:
        with pytest.raises(CometError) as e:
            f()
        assert str(e.value)
    for f in (lambda: R.write_dev(x, 1, "f64"), lambda: R.write(np.zeros((2, 99)), [0, 1]), lambda: R.write(np.zeros((2, 100)), [0]), lambda: R.search(np.zeros((1, 7)), 1)):
        with pytest.raises(ValueError):
            f()
    assert same(R.read(np.arange(50)), np.zeros((50, 100)))           # nothing of the refused writes arrived
    R.write_dev(x, 0); R.read_dev(0, 0); R.scores_dev(R, 0, 0); R.scores_dev(R, 3, 0, n=0)
    o = dev.new((64,), np.float32)
    big = LogProbs(ctx, 4, 20000, 10)
    ok = dict(out_logsum=o, out_entropy=o, k=0)
    small, wide = LogProbs(ctx, 4, 100, 10), dev.new((40000,), np.float32)
    for f in (lambda: LogProbs(ctx, 1, 10, 129), lambda: LogProbs(ctx, 1, 2 ** 30 + 1, 1), lambda: LogProbs(ctx, -1, 1, 1), lambda: big.run_dev(x, "f32", 1, 10, scale=0.0, **ok),
              lambda: big.run_dev(x, "f32", 1, 10, scale=float("inf"), **ok), lambda: big.run_dev(x, "f32", 1, 10, scale=1e38, **ok), lambda: big.run_dev(x, "f32", 2, 10, ld=9, **ok), lambda: big.run_dev(0, "f32", 2, 10, **ok),
              lambda: big.run_dev(x, "f32", 1, 10, out_logsum=0, out_entropy=o), lambda: big.run_dev(x, "f32", 1, 10, n_targets=1, **ok),
              lambda: big.run_dev(x, "f32", 1, 10, out_logsum=o, out_entropy=o, k=1), lambda: big.run_dev(x, "f32", 1, 10, n_targets=-1, **ok),
              lambda: small.run_dev(wide, "f32", 1, 40000, **ok), lambda: big.run_dev(x, "f32", 1, 10, out_logsum=o, out_entropy=o, k=-1)):
        with pytest.raises(CometError):
            f()
    for p in (R, S, big, small):
        p.close()


# ---- streams and graphs ------------------------------------------------------------------------------------------------
def test_on_a_stream_of_the_callers(ctx):
    torch = pytest.importorskip("torch")
    n, dim, m, k = 5000, 256, 20, 10
    x, q = rows_of(21, n, dim), rows_of(22, m, dim)
    s = torch.cuda.Stream()
    R, Q, plan = Fp8Rows(ctx, n, dim), Fp8Rows(ctx, m, dim), LogProbs(ctx, m, n, k)
    with torch.cuda.stream(s):
        st = s.cuda_stream
        a = torch.randn(2048, 2048, device="cuda")
        for _ in range(20):                     # work that the calls have to come behind
            a = a @ a * 1e-3
        dx, dq = torch.from_numpy(x).cuda(non_blocking=False) + 0 * a[0, 0].nan_to_num(), torch.from_numpy(q).cuda()
        out = torch.full((m, n), 9.0, device="cuda")
        ids, tl = torch.empty(m, k, dtype=torch.int32, device="cuda"), torch.empty(m, k, device="cuda")
        ls, en = torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
        R.write_dev(dx.data_ptr(), n, stream=st); Q.write_dev(dq.data_ptr(), m, stream=st)
        R.scores_dev(Q, m, out.data_ptr(), stream=st)
        plan.run_dev(out.data_ptr(), "f32", m, n, out_logsum=ls.data_ptr(), out_entropy=en.data_ptr(), k=k, out_ids=ids.data_ptr(), out_top_logprobs=tl.data_ptr(), stream=st)
        back = out.clone()
    s.synchronize()
    hq, hr = ref.held(q), ref.held(x)
    assert (np.abs(back.cpu().numpy() - hq @ hr.T) <= dim * 2.0 ** -23 * (np.abs(hq) @ np.abs(hr).T)).all()
    check_logprobs({"ids": ids.cpu().numpy(), "top": tl.cpu().numpy(), "logsum": ls.cpu().numpy(), "entropy": en.cpu().numpy(), "logprobs": np.empty((m, 0), np.float32)},
                   back.cpu().numpy(), n, None, 1.0, None, k)
    for p in (R, Q, plan):
        p.close()


def test_captured_into_graphs_and_replayed(ctx):
    """two graphs of the whole run, each with a store and a plan of its own, replayed in turn with eager calls and synchronisations between"""
    torch = pytest.importorskip("torch")
    n, dim, m, k = 30000, 200, 7, 20
    runs = []
    for g in range(2):
        r = {"R": Fp8Rows(ctx, n, dim), "Q": Fp8Rows(ctx, m, dim), "plan": LogProbs(ctx, m, n, k), "x": torch.empty(300, dim, device="cuda"), "q": torch.empty(m, dim, device="cuda"),
             "slots": torch.empty(300, dtype=torch.int64, device="cuda"), "out": torch.empty(m, n, device="cuda"), "ids": torch.empty(m, k, dtype=torch.int32, device="cuda"),
             "tl": torch.empty(m, k, device="cuda"), "ls": torch.empty(m, device="cuda"), "en": torch.empty(m, device="cuda"), "back": torch.empty(300, dim, device="cuda")}
        x = rows_of(30 + g, n, dim)
        r["R"].write(x, np.arange(n))
        r["host"] = ref.held(x)
        runs.append(r)

    def once(r, st):
        r["R"].write_dev(r["x"].data_ptr(), 300, slots=r["slots"].data_ptr(), stream=st)
        r["R"].read_dev(r["back"].data_ptr(), 300, slots=r["slots"].data_ptr(), stream=st)
        r["Q"].write_dev(r["q"].data_ptr(), m, stream=st)
        r["R"].scores_dev(r["Q"], m, r["out"].data_ptr(), stream=st)
        r["plan"].run_dev(r["out"].data_ptr(), "f32", m, n, scale=9.0, out_logsum=r["ls"].data_ptr(), out_entropy=r["en"].data_ptr(), k=k, out_ids=r["ids"].data_ptr(),
                          out_top_logprobs=r["tl"].data_ptr(), stream=st)

    def feed(r, seed):
        rng = np.random.default_rng(seed)
        x, q, slots = rows_of(seed, 300, dim), rows_of(seed + 1, m, dim), rng.integers(-1, n, 300)
        slots[10:20] = slots[0]
        r["x"].copy_(torch.from_numpy(x)); r["q"].copy_(torch.from_numpy(q)); r["slots"].copy_(torch.from_numpy(slots))
        h = ref.held(x)
        for i, s in enumerate(slots):
            if s >= 0:
                r["host"][s] = h[i]
        r["hq"], r["hs"] = ref.held(q), slots

    def check(r):
        torch.cuda.synchronize()
        want, mag = r["hq"] @ r["host"].T, np.abs(r["hq"]) @ np.abs(r["host"]).T
        out = r["out"].cpu().numpy()
        assert (np.abs(out - want) <= dim * 2.0 ** -23 * mag).all()
        assert same(r["back"].cpu().numpy(), np.where(r["hs"][:, None] >= 0, r["host"][np.maximum(r["hs"], 0)], 0.0))
        check_logprobs({"ids": r["ids"].cpu().numpy(), "top": r["tl"].cpu().numpy(), "logsum": r["ls"].cpu().numpy(), "entropy": r["en"].cpu().numpy(),
                        "logprobs": np.empty((m, 0), np.float32)}, out, n, None, 9.0, None, k)

    for g, r in enumerate(runs):
        feed(r, 100 + g)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            once(r, side.cuda_stream)
        side.synchronize()
        check(r)
        r["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(r["graph"]):
            once(r, torch.cuda.current_stream().cuda_stream)
    for turn in range(4):
        for g, r in enumerate(runs):
            feed(r, 200 + 10 * turn + g)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for st, r in zip(streams, runs):         # both at once
            with torch.cuda.stream(st):
                r["graph"].replay()
        for r in runs:
            check(r)
        for g, r in enumerate(runs):             # the program's own eager work between the replays
            feed(r, 300 + 10 * turn + g)
            once(r, torch.cuda.current_stream().cuda_stream)
            check(r)
    for r in runs:
        del r["graph"]
        for p in ("R", "Q", "plan"):
            r[p].close()


def test_orders_before_asynchronous_searches_on_lane_zero(ctx):
    """rows read back on lane 0 are the queries of an asynchronous search that may start on any lane"""
    from comet_amd import L2_SQUARED, FlatIndex
    n, dim, B, k = 4000, 64, 32, 5
    x = rows_of(50, n, dim)
    R = Fp8Rows(ctx, n, dim)
    R.write(x, np.arange(n))
    flat = FlatIndex(ctx, dim, L2_SQUARED)
    h = ref.held(x).astype(np.float32)
    flat.add_batch(np.arange(1, n + 1, dtype=np.uint32), h)
    q, ids, sc, ct = (ctx.alloc(b) for b in (B * dim * 4, B * k * 4, B * k * 4, B * 4))
    for turn in range(8):
        R.read_dev(q, B, first=turn * B)
        t = flat.search_batch_dev_async(q, B, k, ids, sc, ct, k)
        flat.search_wait(t)
        assert (ctx.download(ids, (B, k), np.uint32)[:, 0] == np.arange(turn * B, turn * B + B) + 1).all()
    for p in (q, ids, sc, ct):
        ctx.free(p)
    R.close()
