"""Forms of the 8-bit row store's calls at the ends of their ranges: the widest rows, many targets, split rows without best columns, windows with slots that
were never written or hold NaN. References and tolerances are those of test_fp8_gpu."""
import numpy as np
import pytest

import fp8_ref as ref
from comet_amd import Fp8Rows
from test_fp8_gpu import DTYPES, Dev, check_logprobs, read, rows_of, run_logprobs, same, score_rows, scores, write

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(ctx):
    d = Dev(ctx)
    yield d
    d.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [(1 << 17) + 77, 1 << 20])
def test_the_widest_rows(ctx, dev, dim, dtype):
    """rows of up to 8192 blocks: every group of lanes walks several of them; scores of ones and minus ones are whole numbers below 2^24"""
    rng = np.random.default_rng(dim)
    x = ref.decode(ref.encode((rng.standard_normal((3, dim)) * np.exp(3 * rng.standard_normal((1, dim)))).astype(np.float32), dtype), dtype)
    R = Fp8Rows(ctx, 9, dim)
    write(dev, R, x, dtype, slots=[7, 2, 7])
    h = ref.held(x)
    want = np.zeros((9, dim))
    want[7], want[2] = h[2], h[1]
    assert same(read(dev, R, 9, "f32"), want)
    s = rng.integers(0, 2, (9, dim)).astype(np.float32) * 2 - 1
    write(dev, R, s, dtype)
    for m in (2, 9):                 # both kernels
        assert same(scores(dev, R, m, R, 9), s[:m].astype(np.float64) @ s.astype(np.float64).T)
    R.close()


@pytest.mark.parametrize("n_targets", [255, 256, 257, 600])
@pytest.mark.parametrize("m,n,k", [(5, 3000, 10), (3, 60000, 0), (2, 60000, 128), (1030, 5000, 3)])
def test_more_targets_than_threads(ctx, dev, m, n, k, n_targets):
    """a thread takes more than one target: of one workgroup a row, of several joined, behind ragged counts and outside the row"""
    s = score_rows(n + m, m, n)
    rng = np.random.default_rng(n_targets)
    targets = rng.integers(-3, n + 3, (m, n_targets)).astype(np.int32)
    targets[:, -1], targets[:, 0] = 0, n - 1
    targets[0, -3:] = [np.iinfo(np.int32).min, np.iinfo(np.int32).max, 1]
    counts = rng.integers(0, n + 1, m).astype(np.int32)
    counts[0] = n
    for c in (None, counts):
        check_logprobs(run_logprobs(ctx, dev, s, "f32", n, 0, c, 1.5, targets, k), s, n, c, 1.5, targets, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n", [(1, 16385), (3, 100003), (300, 20011), (1, 1000003)])
def test_split_rows_without_best_columns(ctx, dev, m, n, dtype):
    s = ref.decode(ref.encode(score_rows(m + n, m, n), dtype), dtype)
    s[:, 1::3] = np.inf              # masked for a negative scale
    targets = np.random.default_rng(n).integers(0, n, (m, 2)).astype(np.int32)
    counts = np.random.default_rng(m).integers(0, n + 1, m).astype(np.int32)
    for c in (None, counts):
        check_logprobs(run_logprobs(ctx, dev, s, dtype, n, 1, c, -3.0, targets, 0), s, n, c, -3.0, targets, 0)


def test_search_over_slots_that_were_never_written(ctx):
    """such a slot is a row of zeros: its score is 0, it is part of the distribution and stands in front of rows with negative scores"""
    n, dim, B, k, scale = 400, 96, 3, 128, 6.0
    x, q = rows_of(70, n, dim), rows_of(71, B, dim)
    R = Fp8Rows(ctx, n + 50, dim)
    filled = np.arange(0, n, 2)
    R.write(x[filled], filled)
    h = np.zeros((n + 50, dim))
    h[filled] = ref.held(x[filled])
    r = R.search(q, k, scale)
    s = ref.held(q) @ h.T
    for b in range(B):
        order = np.argsort(-s[b], kind="stable")[:k]
        assert (np.sort(s[b][r.slots[b]]) <= np.sort(s[b][order]) + dim * 2.0 ** -22).all() and (r.slots[b] >= 0).all()
        if (s[b] > 1e-3).sum() <= k:
            assert set(np.flatnonzero(s[b] > 1e-3)) <= set(r.slots[b])
        z = scale * s[b]
        assert abs(r.logsum[b] - np.log(np.exp(z).sum())) <= scale * dim * 2.0 ** -22 + 64 * 2.0 ** -23
    # one row of NaN: every query's statistics are NaN, and it is never among the ids
    bad = np.full((1, dim), np.nan, np.float32)
    R.write(bad, [20])
    r = R.search(q, k, scale)
    assert np.isnan(r.logsum).all() and np.isnan(r.entropy).all() and np.isnan(r.logprobs).all() and not (r.slots == 20).any()
    # ... unless the window leaves it out
    r = R.search(q, k, scale, first=21)
    assert np.isfinite(r.logsum).all() and (r.slots >= 21).all()
    R.close()
