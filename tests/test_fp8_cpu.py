"""What the 8-bit row store's entry points refuse before they touch a device, and the plain restatements the GPU tests compare with."""
import ctypes as C
import re
from pathlib import Path

import numpy as np
import pytest

import fp8_ref as ref
from comet_amd import _lib


def test_null_handles_are_refused():
    lib = _lib.load()
    h, z = C.c_void_p(), C.c_size_t()
    assert lib.comet_fp8_create(None, 8, 8, C.byref(h)) == _lib.ERR_INVALID_ARG and not h.value and b"context" in lib.comet_last_error()
    assert lib.comet_fp8_destroy(None) == _lib.OK
    assert lib.comet_fp8_capacity(None) == 0 and lib.comet_fp8_dim(None) == 0
    assert lib.comet_fp8_write_dev(None, None, 0, None, 0, 0, 0, None) == _lib.ERR_INVALID_ARG and b"rows must not be null" in lib.comet_last_error()
    assert lib.comet_fp8_read_dev(None, None, 0, None, 0, 0, 0, None) == _lib.ERR_INVALID_ARG
    assert lib.comet_fp8_scores_dev(None, 0, 0, None, 0, 0, None, 0, 0, None) == _lib.ERR_INVALID_ARG
    assert lib.comet_fp8_write(None, None, None, 0) == _lib.ERR_INVALID_ARG
    assert lib.comet_fp8_read(None, None, 0, None) == _lib.ERR_INVALID_ARG
    assert lib.comet_fp8_search(None, 0, 0, None, 0, 1.0, 0, None, None, None, None) == _lib.ERR_INVALID_ARG
    assert lib.comet_logprobs_dev(None, None, 0, 0, 0, 0, None, 1.0, None, 0, 0, None, None, None, None, None, None, 0, None) == _lib.ERR_INVALID_ARG
    assert lib.comet_logprobs_work_bytes(1, 1, 1, None) == _lib.ERR_INVALID_ARG
    for m, n, k in ((-1, 1, 1), (1, -1, 1), (1, (1 << 30) + 1, 1), (1, 1, -1), (1, 1, 129)):
        assert lib.comet_logprobs_work_bytes(m, n, k, C.byref(z)) == _lib.ERR_INVALID_ARG, (m, n, k)


def test_numbers_beyond_32_bits_are_refused_before_they_are_cut():
    from types import SimpleNamespace

    from comet_amd import Fp8Rows, LogProbs
    ctx = SimpleNamespace(lib=_lib.load(), h=None, stream=0)
    for f in (lambda: Fp8Rows(ctx, 8, (1 << 32) + 8), lambda: LogProbs(ctx, 1, 10, (1 << 32) + 1)):
        with pytest.raises(ValueError, match="32 bits"):
            f()
    p = LogProbs(ctx, 1, 10, 1)
    for kw in (dict(k=1 << 32), dict(n_targets=(1 << 32) + 1)):
        with pytest.raises(ValueError, match="32 bits"):
            p.run_dev(16, "f32", 1, 10, out_logsum=16, out_entropy=16, **kw)


def test_workspace_of_a_large_call_serves_smaller_ones():
    lib = _lib.load()

    def need(m, n, k):
        z = C.c_size_t()
        assert lib.comet_logprobs_work_bytes(m, n, k, C.byref(z)) == 0
        return z.value
    rng = np.random.default_rng(0)
    for _ in range(500):
        m, n, k = int(rng.integers(1, 5000)), int(rng.integers(1, 1 << 21)), int(rng.integers(0, 129))
        a, b, c = int(rng.integers(1, m + 1)), int(rng.integers(1, n + 1)), int(rng.integers(0, k + 1))
        assert need(a, b, c) <= need(m, n, k), ((a, b, c), (m, n, k))
    assert need(1, 1000, 128) == 0 and need(0, 1 << 30, 128) == 0


@pytest.mark.parametrize("seed", range(4))
def test_reference_codes_are_the_nearest(seed):
    """the plain quantiser against torch's own e4m3 conversion on scaled values, and its error bound"""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((40, 300)) * np.exp(3 * rng.standard_normal((40, 300)))).astype(np.float32)
    h = ref.held(x)
    for c in range(0, 300, 128):
        b, hb = x[:, c:c + 128].astype(np.float64), h[:, c:c + 128]
        A = np.abs(b).max(axis=1)
        e = np.array([min(i for i in range(-126, 121) if a * 2.0 ** -i <= 448) for a in A])
        u = 2.0 ** e[:, None]
        t = torch.from_numpy((b / u).astype(np.float32)).to(torch.float8_e4m3fn).to(torch.float64).numpy()
        assert (hb == t * u).all()
        assert (np.abs(hb - b) <= np.maximum(np.abs(b) * 2.0 ** -4, 2.0 ** -10 * u)).all()


def test_reference_bf16_round_trip():
    u = np.arange(0, 65536, dtype=np.uint32).astype(np.uint16)
    f = ref.from_bf16_bits(u)
    ok = ~np.isnan(f)
    assert (ref.to_bf16_bits(f)[ok] == u[ok]).all()


def test_asm_names_the_registers_it_takes():
    """a load into LDS takes its address from M0: an operand of the asm statement, never written behind the compiler's back"""
    seen = 0
    for f in sorted((Path(__file__).resolve().parent.parent / "comet_amd" / "csrc" / "fp8").glob("*.h*")):
        for stmt in re.findall(r"asm volatile\((.*?)\);", f.read_text(), re.S):
            code, _, operands = stmt.partition("::")
            assert not re.search(r"\bm0\b", code), (f.name, stmt)
            if "_lds_" in code:
                assert '"{m0}"' in operands, (f.name, stmt)
                seen += 1
    assert seen


def test_buffers_are_read_before_they_are_handed_over():
    """in front of each bare barrier the wave waits for its LDS reads: what is filled behind the barrier is filled by asm statements that the compiler does not see"""
    text = (Path(__file__).resolve().parent.parent / "comet_amd" / "csrc" / "fp8" / "scores.hip").read_text()
    waits = re.findall(r"void (\w+)\(\) \{ asm volatile\(\"s_waitcnt vmcnt\(%0\) lgkmcnt\(0\)\"", text)
    assert len(waits) == 1
    for before in text.split("__builtin_amdgcn_s_barrier()")[:-1]:
        lines = [line.strip() for line in before.rstrip().splitlines() if not line.strip().startswith("//")][-4:]
        assert sum(waits[0] + "<" in line for line in lines) == 2, lines         # both branches


def test_numbers_beyond_64_bits_are_refused_before_they_are_cut():
    from types import SimpleNamespace

    from comet_amd import Fp8Rows, LogProbs
    ctx = SimpleNamespace(lib=_lib.load(), h=None, stream=0)
    R, big = Fp8Rows.__new__(Fp8Rows), 1 << 64
    R.ctx, R.lib, R.h, R.capacity, R.dim = ctx, ctx.lib, None, 8, 8
    plan = LogProbs(ctx, 1, 10, 1)
    for f in (lambda: Fp8Rows(ctx, big + 8, 8), lambda: R.write_dev(16, big + 1), lambda: R.write_dev(16, 1, first=big), lambda: R.write_dev(16, 1, ld=big + 8),
              lambda: R.read_dev(16, big + 1), lambda: R.read_dev(16, 1, first=-big), lambda: R.read_dev(16, 1, ld=big + 8), lambda: R.scores_dev(R, big + 1, 16, n=8),
              lambda: R.scores_dev(R, 1, 16, n=big + 8), lambda: R.scores_dev(R, 1, 16, first=big, n=8), lambda: R.scores_dev(R, 1, 16, q_first=big, n=8),
              lambda: R.scores_dev(R, 1, 16, n=8, ld=big + 8), lambda: R.search(np.zeros(8), 1, first=big), lambda: R.search(np.zeros(8), 1, n=big + 1), lambda: LogProbs(ctx, big + 1, 10, 1),
              lambda: LogProbs(ctx, 1, big + 10, 1), lambda: plan.run_dev(16, "f32", big + 1, 10, out_logsum=16, out_entropy=16),
              lambda: plan.run_dev(16, "f32", 1, big + 10, out_logsum=16, out_entropy=16), lambda: plan.run_dev(16, "f32", 1, 10, ld=big + 10, out_logsum=16, out_entropy=16)):
        with pytest.raises(ValueError, match="64 bits"):
            f()
