"""Forms of the 8-bit row store's calls at the ends of their ranges: the widest rows, many targets, split rows without best columns, windows with slots that
were never written or hold NaN. References and tolerances are those of test_fp8_gpu."""
import numpy as np
import pytest

import fp8_ref as ref
from comet_amd import Fp8Rows, LogProbs
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


def test_host_writes_and_reads_of_more_rows_than_one_piece(ctx):
    """uploads of 256 MiB at a time, the same slots in two of them: the last row stays (ones and minus ones are held exactly)"""
    dim, n = 1 << 20, 70                # 64 rows a piece
    rng = np.random.default_rng(9)
    x = rng.integers(0, 2, (n, dim), np.int8).astype(np.float32) * 2 - 1
    slots = np.arange(n) % 67           # rows 67, 68 and 69 over rows 0, 1 and 2
    R = Fp8Rows(ctx, 67, dim)
    R.write(x, slots)
    want = x[:67].copy()
    want[:3] = x[67:]
    at = np.r_[np.arange(67), [0, 66, 1]]
    assert (R.read(at) == want[at]).all()
    R.close()


def test_strides_behind_32_bits(ctx):
    """two rows 2^31 + 3 elements apart, of each matrix that the calls take"""
    torch = pytest.importorskip("torch")
    ld, dim, n, k = (1 << 31) + 3, 300, 5000, 10
    x, q = rows_of(80, n, dim), rows_of(81, 2, dim)
    st = torch.cuda.current_stream().cuda_stream
    buf = torch.zeros(ld + n + 7, dtype=torch.bfloat16, device="cuda")
    R, Q, plan = Fp8Rows(ctx, n, dim), Fp8Rows(ctx, 2, dim), LogProbs(ctx, 2, n, k)
    R.write(x, np.arange(n))
    qb = torch.from_numpy(q).to(torch.bfloat16)
    for i in range(2):
        buf[i * ld:i * ld + dim] = qb[i].cuda()
    Q.write_dev(buf.data_ptr(), 2, "bf16", ld=ld, stream=st)
    hq, h = ref.held(qb.float().numpy()), ref.held(x)
    buf.zero_()
    Q.read_dev(buf.data_ptr(), 2, "bf16", ld=ld, stream=st)
    got = torch.stack([buf[:dim], buf[ld:ld + dim]]).float().cpu().numpy()
    assert same(got, hq) and buf[dim:ld].any().item() is False       # (bfloat16 holds the values exactly)
    R.scores_dev(Q, 2, buf.data_ptr(), "bf16", ld=ld, stream=st)
    s = torch.stack([buf[:n], buf[ld:ld + n]]).float().cpu().numpy()
    want, mag = hq @ h.T, np.abs(hq) @ np.abs(h).T
    assert (np.abs(s - want) <= dim * 2.0 ** -23 * mag + ref.EPS["bf16"] * np.abs(want) * 1.01).all()
    ls, en, tl = (torch.empty(2, *sh, device="cuda") for sh in ((), (), (k,)))
    ids = torch.empty(2, k, dtype=torch.int32, device="cuda")
    plan.run_dev(buf.data_ptr(), "bf16", 2, n, ld=ld, scale=5.0, out_logsum=ls.data_ptr(), out_entropy=en.data_ptr(), k=k, out_ids=ids.data_ptr(), out_top_logprobs=tl.data_ptr(), stream=st)
    check_logprobs({"ids": ids.cpu().numpy(), "top": tl.cpu().numpy(), "logsum": ls.cpu().numpy(), "entropy": en.cpu().numpy(), "logprobs": np.empty((2, 0), np.float32)}, s, n, None, 5.0, None, k)
    for p in (R, Q, plan):
        p.close()


def test_the_longest_score_row(ctx):
    """2^30 columns: all of score 0 but one at the front and the last"""
    torch = pytest.importorskip("torch")
    n, k = 1 << 30, 4
    st = torch.cuda.current_stream().cuda_stream
    s = torch.zeros(n, dtype=torch.float16, device="cuda")
    s[12345], s[n - 1] = 2.0, 3.0
    plan = LogProbs(ctx, 1, n, k)
    ls, en, tl, lp = (torch.empty(i, device="cuda") for i in (1, 1, k, 3))
    ids, targets = torch.empty(k, dtype=torch.int32, device="cuda"), torch.tensor([n - 1, 12345, n - 2], dtype=torch.int32, device="cuda")
    plan.run_dev(s.data_ptr(), "f16", 1, n, scale=4.0, targets=targets.data_ptr(), n_targets=3, out_logprobs=lp.data_ptr(), out_logsum=ls.data_ptr(), out_entropy=en.data_ptr(), k=k,
                 out_ids=ids.data_ptr(), out_top_logprobs=tl.data_ptr(), stream=st)
    z = np.array([12.0, 8.0, 0.0])
    logsum = np.log(np.exp(z) @ np.array([1.0, 1.0, n - 2.0]))
    p = np.exp(z - logsum)
    # a thread adds up whole numbers (exp(0) times the columns), the larger terms are joined with a rounding each: some tens of steps of 2^-24 in S, and those of z and log S
    tol = 64 * 2.0 ** -23 * (1 + abs(logsum))
    assert ids.tolist() == [n - 1, 12345, 0, 1]
    assert abs(ls.item() - logsum) <= tol and abs(en.item() + (p * (z - logsum)) @ np.array([1.0, 1.0, n - 2.0])) <= tol
    assert np.abs(tl.cpu().numpy() - (z - logsum)[[0, 1, 2, 2]]).max() <= tol and np.abs(lp.cpu().numpy() - (z - logsum)).max() <= tol
    plan.close()


def test_scores_of_more_than_2_31_elements(ctx, dev):
    torch = pytest.importorskip("torch")
    m, n, dim = 256, 8_500_001, 3
    rng = np.random.default_rng(10)
    q, r = rng.integers(-7, 8, (m, dim)).astype(np.float32), rng.integers(-7, 8, (n, dim)).astype(np.float32)
    Q, R = Fp8Rows(ctx, m, dim), Fp8Rows(ctx, n, dim)
    write(dev, Q, q); write(dev, R, r)
    ctx.sync()
    out = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    R.scores_dev(Q, m, out.data_ptr(), "bf16", stream=torch.cuda.current_stream().cuda_stream)
    dq, dr = torch.from_numpy(q).cuda(), torch.from_numpy(r).cuda()
    for i in (0, 1, 252, 253, 254, 255):
        assert torch.equal(out[i].float(), (dr @ dq[i]).to(torch.bfloat16).float()), i         # whole numbers below 2^8: exact
    Q.close(); R.close()
