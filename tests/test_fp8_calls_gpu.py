"""The 8-bit row store's calls among others: behind a call that failed, beside a call that holds the context, in front of searches on other lanes."""
import threading

import numpy as np
import pytest

import fp8_ref as ref
from comet_amd import L2_SQUARED, CometError, FlatIndex, Fp8Rows, LogProbs
from test_fp8_gpu import Dev, check_logprobs, read, rows_of, same, write

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(ctx):
    d = Dev(ctx)
    yield d
    d.close()


def test_a_store_that_does_not_fit_leaves_no_error_behind(ctx, dev):
    """the allocation's error is reported once, by the call that met it"""
    x = rows_of(1, 100, 64)
    R = Fp8Rows(ctx, 100, 64)
    for _ in range(2):
        with pytest.raises(CometError, match="out of memory"):
            Fp8Rows(ctx, 1 << 36, 16)          # 8 TiB of codes
        write(dev, R, x, slots=np.arange(100))
        assert same(read(dev, R, 100), ref.held(x))
    R.close()


def test_an_error_of_another_call_does_not_stop_these(ctx, dev):
    """an error left in the runtime by the caller's own HIP call: the row store's calls check their own launches, and a write to slots arrives whole, as do later ones"""
    n, dim = 300, 200
    x, y = rows_of(2, n, dim), rows_of(3, n, dim)
    R = Fp8Rows(ctx, n, dim)
    assert ctx.lib.hipSetDevice(10 ** 6) != 0         # refused: the process has no such device
    write(dev, R, x[::-1], slots=np.arange(n)[::-1])
    assert same(read(dev, R, n), ref.held(x))
    write(dev, R, y[:70], slots=np.arange(70))        # rows of lower numbers than the first call's in the same slots
    assert same(read(dev, R, n), ref.held(np.concatenate([y[:70], x[70:]])))
    ctx.lib.hipGetLastError()
    R.close()


@pytest.mark.parametrize("stream", [0, None])
def test_calls_on_device_arrays_do_not_stand_behind_a_call_that_holds_the_context(ctx, dev, stream):
    """a thread that streams an index out holds the context for as long as its writer takes; another thread's calls on device arrays return meanwhile,
    on a stream of its own and on lane 0"""
    n, dim, m, k = 3000, 100, 5, 7
    x, q = rows_of(4, n, dim), rows_of(5, m, dim)
    flat = FlatIndex(ctx, 8, L2_SQUARED)
    flat.add_batch(np.arange(1, 11, dtype=np.uint32), rows_of(6, 10, 8))
    R, Q, plan = Fp8Rows(ctx, n, dim), Fp8Rows(ctx, m, dim), LogProbs(ctx, m, n, k)
    px, pq, out, back = dev.put(x), dev.put(q), dev.new((m, n), np.float32), dev.new((n, dim), np.float32)
    ls, en, ids, tl = dev.new((m,), np.float32), dev.new((m,), np.float32), dev.new((m, k), np.int32), dev.new((m, k), np.float32)
    returned, failed = threading.Event(), []

    def calls():
        try:
            R.write_dev(px, n, stream=stream)
            Q.write_dev(pq, m, stream=stream)
            R.read_dev(back, n, stream=stream)
            R.scores_dev(Q, m, out, stream=stream)
            plan.run_dev(out, "f32", m, n, scale=3.0, out_logsum=ls, out_entropy=en, k=k, out_ids=ids, out_top_logprobs=tl, stream=stream)
            returned.set()
        except BaseException as e:
            failed.append(e)

    class Writer:
        seen = None

        def write(self, b):
            if self.seen is None:
                t = threading.Thread(target=calls)
                t.start()
                self.seen = returned.wait(20)
                self.thread = t
            return len(b)
    w = Writer()
    flat.write_to(w)
    w.thread.join()
    assert not failed and w.seen
    if stream == 0:
        torch = pytest.importorskip("torch")
        torch.cuda.synchronize()
    h, hq = ref.held(x), ref.held(q)
    assert same(dev.get(back, (n, dim), np.float32), h)
    s = dev.get(out, (m, n), np.float32)
    assert (np.abs(s - hq @ h.T) <= dim * 2.0 ** -23 * (np.abs(hq) @ np.abs(h).T)).all()
    check_logprobs({"ids": dev.get(ids, (m, k), np.int32), "top": dev.get(tl, (m, k), np.float32), "logsum": dev.get(ls, (m,), np.float32), "entropy": dev.get(en, (m,), np.float32),
                    "logprobs": np.empty((m, 0), np.float32)}, s, n, None, 3.0, None, k)
    for p in (R, Q, plan):
        p.close()


def test_asynchronous_searches_start_behind_a_long_queue_on_lane_zero(ctx, dev):
    """queries read back on lane 0 behind a millisecond of products: a search on another lane that did not wait would find the previous turn's"""
    n, dim, B, k = 4000, 64, 32, 5
    x = rows_of(50, n, dim)
    R, big, Q = Fp8Rows(ctx, n, dim), Fp8Rows(ctx, 200000, 768), Fp8Rows(ctx, 256, 768)
    R.write(x, np.arange(n))
    flat = FlatIndex(ctx, dim, L2_SQUARED)
    flat.add_batch(np.arange(1, n + 1, dtype=np.uint32), ref.held(x).astype(np.float32))
    q, ids, sc, ct = dev.new((B, dim), np.float32, 0), dev.new((B, k), np.uint32), dev.new((B, k), np.float32), dev.new((B,), np.int32)
    out = dev.new((256, 200000), np.float32)
    for turn in range(12):
        for _ in range(12):
            big.scores_dev(Q, 256, out)
        R.read_dev(q, B, first=turn * B)
        t = flat.search_batch_dev_async(q, B, k, ids, sc, ct, k)
        flat.search_wait(t)
        assert (ctx.download(ids, (B, k), np.uint32)[:, 0] == np.arange(turn * B, turn * B + B) + 1).all()
    for p in (R, big, Q):
        p.close()
