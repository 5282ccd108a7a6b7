"""The 8-bit row store's calls among others: behind a call that failed, beside a call that holds the context, in front of searches on other lanes."""
import numpy as np
import pytest

import fp8_ref as ref
from comet_amd import CometError, Fp8Rows
from test_fp8_gpu import Dev, read, rows_of, same, write

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
