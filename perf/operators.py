"""The 8-bit row store's operators as measurable cases: rows quantised as they are written and read back, the product of
queries with stored rows, and the log-probabilities / entropy / best columns of score rows.

``own`` False: the operators written out in elementary torch operations, in 32 bits. ``own`` True: the calls a program makes
of this package. Both work on what ``prepare`` returns; ``exact`` is the operators' definition in 64 bits.

A block is 128 consecutive values of a row (the last one padded with zeros). With A the largest finite magnitude of a block,
its exponent e is the least integer with A * 2^-e <= 448, clamped to [-126, 120]; a value is held as the e4m3 number nearest
to x * 2^-e (ties to even, non-finite values as NaN) and stands for that number times 2^e.
"""
import math
import os

import torch

own = False

BLOCK = 128
E_MIN, E_MAX = -126, 120
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one document joins a store: the latency of a single write and of reading it back
        {"name": "write-one", "op": "write", "n": 1, "dim": 384, "capacity": 65536, "dtype": "f32", "pad": 0, "out": "f32"},
        # some thousand re-embedded documents, odd width, rows of a wider buffer, scattered over the store, a few of them padding
        {"name": "write-scattered", "op": "write", "n": 3001, "dim": 300, "capacity": 100000, "dtype": "bf16", "pad": 7, "out": "bf16"},
        # bulk ingest of a corpus, 128 Ki rows a call
        {"name": "write-bulk", "op": "write", "n": 131072, "dim": 768, "capacity": 262144, "dtype": "f32", "pad": 0, "out": "bf16"},
        # the ten best rows of one query, for a reranker
        {"name": "read-ten", "op": "read", "n": 10, "dim": 128, "capacity": 10000, "out": "f32", "pad": 0},
        # the hundred best rows of each of 256 queries
        {"name": "read-batch", "op": "read", "n": 25600, "dim": 768, "capacity": 1000000, "out": "f32", "pad": 0},
        # one query against a small store: latency
        {"name": "scores-small", "op": "scores", "m": 1, "n": 10000, "dim": 128, "dtype": "f32", "out": "f32"},
        # one query against a million rows: the stream of the rows
        {"name": "scores-one", "op": "scores", "m": 1, "n": 1000000, "dim": 768, "dtype": "f32", "out": "f32"},
        # a batch of 256 queries against a million rows
        {"name": "scores-batch", "op": "scores", "m": 256, "n": 1000000, "dim": 768, "dtype": "f32", "out": "f32"},
        # documents against documents (near duplicates), wide embeddings, odd counts: bound by arithmetic
        {"name": "scores-cross", "op": "scores", "m": 2047, "n": 30011, "dim": 2000, "dtype": "bf16", "out": "bf16"},
        # the distribution of one query over a small store
        {"name": "logprobs-one", "op": "logprobs", "m": 1, "n": 10000, "dtype": "f32", "k": 10, "targets": 1, "scale": 20.0, "ragged": False, "pad": 0},
        # a batch of 256 queries over a million rows, the hundred best of each
        {"name": "logprobs-batch", "op": "logprobs", "m": 256, "n": 1000000, "dtype": "f32", "k": 100, "targets": 4, "scale": 20.0, "ragged": False, "pad": 0},
        # distances (smaller is better) over candidate lists of uneven length, some empty, some wholly masked
        {"name": "logprobs-ragged", "op": "logprobs", "m": 1000, "n": 30011, "dtype": "bf16", "k": 20, "targets": 2, "scale": -4.0, "ragged": True, "pad": 5},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "scores", "scores", "logprobs", "logprobs"])
    dtype, out = rng.choice(list(DTYPES)), rng.choice(list(DTYPES))
    pad = rng.choice([0, 0, 1, 3, 8])
    if op in ("write", "read"):
        dim = _log_uniform(rng, 16, 2048)
        n = _log_uniform(rng, 1, 100_000_000 // dim if op == "write" else 30_000_000 // dim)
        case = {"op": op, "n": n, "dim": dim, "capacity": max(n, _log_uniform(rng, 1000, 800_000_000 // dim)), "out": out, "pad": pad}
        if op == "write":
            case["dtype"] = dtype
        return case
    if op == "scores":
        dim = _log_uniform(rng, 16, 2048)
        n = _log_uniform(rng, 1, min(1_000_000, 768_000_000 // dim))
        m = _log_uniform(rng, 1, max(1, min(2048, 256_000_000 // n, 190_000_000_000 // (n * dim))))
        return {"op": op, "m": m, "n": n, "dim": dim, "dtype": dtype, "out": out}
    n = _log_uniform(rng, 1, 1_000_000)
    m = _log_uniform(rng, 1, max(1, min(2048, 200_000_000 // n)))
    return {"op": op, "m": m, "n": n, "dtype": dtype, "k": rng.choice([0, 1, 10, 33, 100, 128]), "targets": rng.choice([0, 1, 4]),
            "scale": rng.choice([1.0, 20.0, 100.0, -4.0]), "ragged": rng.random() < 0.5, "pad": pad}


def work(case):
    if case["op"] in ("write", "read"):
        n, dim = case["n"], case["dim"]
        nb = -(-dim // BLOCK)
        held = n * (nb * BLOCK + nb)
        if case["op"] == "read":
            return {"bytes": held + 8 * n + n * dim * SIZE[case["out"]], "flops": n * dim}
        return {"bytes": n * dim * SIZE[case["dtype"]] + 2 * held + 8 * n + n * dim * SIZE[case["out"]], "flops": 4 * n * dim}
    m, n = case["m"], case["n"]
    if case["op"] == "scores":
        dim = case["dim"]
        nb = -(-dim // BLOCK)
        return {"bytes": m * dim * SIZE[case["dtype"]] + n * (nb * BLOCK + nb) + m * n * SIZE[case["out"]], "flops": 2 * m * n * dim}
    cols = m * n // 2 if case["ragged"] else m * n   # ragged rows hold half of the columns on average
    return {"bytes": cols * SIZE[case["dtype"]] + m * (8 * case["k"] + 8 * case["targets"] + 12), "flops": 6 * cols}


# ---- the inputs --------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _embeddings(n, dim, dtype, pad, g):
    """Rows as an embedding model gives them: unit length, some dimensions much larger than others; a view of a buffer whose rows are dim + pad wide."""
    x = torch.empty(n, dim + pad, dtype=DTYPES[dtype], device="cuda")
    weight = torch.exp(torch.randn(dim, device="cuda", generator=g))
    step = max(1, (1 << 27) // max(1, dim))
    for i in range(0, n, step):
        r = torch.randn(min(step, n - i), dim, device="cuda", generator=g) * weight
        x[i:i + step, :dim] = (r / r.norm(dim=1, keepdim=True).clamp_min(1e-30)).to(x.dtype)
    x[:, dim:] = 7.0
    return x[:, :dim]


def _slots(n, capacity, g, holes):
    if n * 2 <= capacity:       # distinct by construction: a random start and an odd stride over the store's power-of-two part
        p = 1 << (capacity.bit_length() - 1)
        a = torch.randint(0, p, (2,), device="cuda", generator=g)
        s = (torch.arange(n, device="cuda") * (a[0] * 2 + 1) + a[1]) % p
    else:
        s = torch.arange(n, device="cuda") + int(torch.randint(0, capacity - n + 1, (1,), device="cuda", generator=g))
    if holes and n > 16:
        s = torch.where(torch.rand(n, device="cuda", generator=g) < 0.02, torch.full_like(s, -1), s)
    return s.contiguous()


def _score_rows(case, g):
    """Score rows as a search leaves them: a bulk near zero, a few close rows, 2 % filtered out; distances for a negative scale."""
    m, n, dt = case["m"], case["n"], DTYPES[case["dtype"]]
    buf = torch.empty(m, n + case["pad"], dtype=dt, device="cuda")
    masked = math.inf if case["scale"] < 0 else -math.inf
    step = max(1, (1 << 26) // n)
    for i in range(0, m, step):
        r = torch.randn(min(step, m - i), n, device="cuda", generator=g)
        r = 0.08 * r + 0.004 * r * r * r
        if case["scale"] < 0:
            r = 2.0 - 2.0 * r
        drop = torch.rand(r.shape, device="cuda", generator=g) < 0.02
        buf[i:i + step, :n] = r.masked_fill(drop, masked).to(dt)
    counts = None
    if case["ragged"]:
        counts = torch.randint(0, n + 1, (m,), device="cuda", generator=g).to(torch.int32)
        if m > 2:
            counts[m // 2] = 0
            buf[m - 1, :n] = masked
    buf[:, n:] = 9.0
    targets = torch.randint(0, n, (m, case["targets"]), device="cuda", generator=g).to(torch.int32) if case["targets"] else None
    return buf[:, :n], counts, targets


_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        os.environ.setdefault("COMET_STREAM_PRIORITY", "normal")   # torch's own streams share the GPU
        import comet_amd
        _ctx = comet_amd.Context(torch.cuda.current_device())
    return _ctx


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("write", "read"):
        n, dim, cap = case["n"], case["dim"], case["capacity"]
        s["slots"] = _slots(n, cap, g, holes=True)
        if op == "write":
            s["x"] = _embeddings(n, dim, case["dtype"], case["pad"], g)
            stored = None
        else:
            stored = _embeddings(cap, dim, "bf16", 0, g)
        s["store"] = _store(cap, dim, stored)
        s["out"] = torch.empty(n, dim + case["pad"], dtype=DTYPES[case["out"]], device="cuda")[:, :dim]
    elif op == "scores":
        s["q"] = _embeddings(case["m"], case["dim"], case["dtype"], 0, g)
        s["store"] = _store(case["n"], case["dim"], _embeddings(case["n"], case["dim"], "bf16", 0, g))
        if own:
            s["queries"] = _store(case["m"], case["dim"], None)
            s["out"] = torch.empty(case["m"], case["n"], dtype=DTYPES[case["out"]], device="cuda")
    else:
        s["scores"], s["counts"], s["targets"] = _score_rows(case, g)
        if own:
            import comet_amd
            m, k, t = case["m"], case["k"], case["targets"]
            s["plan"] = comet_amd.LogProbs(_context(), m, case["n"], k)
            f = lambda *shape: torch.empty(*shape, dtype=torch.float32, device="cuda")  # noqa: E731
            s["logsum"], s["entropy"], s["top_logprobs"], s["logprobs"] = f(m), f(m), f(m, k), f(m, t)
            s["top"] = torch.empty(m, k, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    case = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] in ("write", "read"):
        if case["op"] == "write":
            s["store"].write_dev(s["x"].data_ptr(), case["n"], case["dtype"], ld=s["x"].stride(0), slots=s["slots"].data_ptr(), stream=stream)
        s["store"].read_dev(s["out"].data_ptr(), case["n"], case["out"], ld=s["out"].stride(0), slots=s["slots"].data_ptr(), stream=stream)
        return s["out"]
    if case["op"] == "scores":
        s["queries"].write_dev(s["q"].data_ptr(), case["m"], case["dtype"], ld=s["q"].stride(0), stream=stream)
        s["store"].scores_dev(s["queries"], case["m"], s["out"].data_ptr(), case["out"], ld=case["n"], stream=stream)
        return s["out"]
    s["plan"].run_dev(s["scores"].data_ptr(), case["dtype"], case["m"], case["n"], ld=s["scores"].stride(0), scale=case["scale"], counts=_ptr(s["counts"]),
                      targets=_ptr(s["targets"]), n_targets=case["targets"], k=case["k"], out_logprobs=_ptr(s["logprobs"]), out_logsum=_ptr(s["logsum"]),
                      out_entropy=_ptr(s["entropy"]), out_ids=_ptr(s["top"]), out_top_logprobs=_ptr(s["top_logprobs"]), stream=stream)
    return _named(case, s["logsum"], s["entropy"], s["logprobs"], s["top"], s["top_logprobs"])


def _named(case, logsum, entropy, logprobs, top, top_logprobs):
    out = {"logsum": logsum, "entropy": entropy}
    if case["targets"]:
        out["logprobs"] = logprobs
    if case["k"]:
        out["top"], out["top_logprobs"] = top, top_logprobs
    return out


def _power_of_two(e):
    """2^e in float32 for integer e in [-126, 127], exactly."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantise(x):
    """codes (float8_e4m3fn, rows padded to whole blocks) and exponents (int32) of float rows"""
    x = x.float()
    n, dim = x.shape
    nb = -(-dim // BLOCK)
    x = torch.nn.functional.pad(x, (0, nb * BLOCK - dim)).view(n, nb, BLOCK)
    finite = x.abs() < math.inf
    mant, ex = torch.frexp(torch.where(finite, x, 0.0).abs().amax(dim=2))
    e = (ex - torch.where(mant <= 0.875, 9, 8)).clamp(E_MIN, E_MAX).to(torch.int32)
    y = torch.where(finite, x * _power_of_two(-e)[:, :, None], math.nan)
    return y.to(torch.float8_e4m3fn).view(n, nb * BLOCK), e


def _dequantise(codes, e, dim):
    n, nb = e.shape
    return (codes.float().view(n, nb, BLOCK) * _power_of_two(e)[:, :, None]).view(n, nb * BLOCK)[:, :dim]


def _store(capacity, dim, rows):
    if own:
        import comet_amd
        store = comet_amd.Fp8Rows(_context(), capacity, dim)
        if rows is not None:
            store.write_dev(rows.data_ptr(), capacity, "bf16", ld=rows.stride(0), stream=torch.cuda.current_stream().cuda_stream)
        return store
    nb = -(-dim // BLOCK)
    codes = torch.zeros(capacity, nb * BLOCK, dtype=torch.uint8, device="cuda")
    e = torch.zeros(capacity, nb, dtype=torch.int32, device="cuda")
    if rows is not None:
        step = max(1, (1 << 27) // dim)
        for i in range(0, capacity, step):
            c, ee = _quantise(rows[i:i + step])
            codes[i:i + step], e[i:i + step] = c.view(torch.uint8), ee
    return codes, e


def _run_plain(s):
    case = s["case"]
    if case["op"] in ("write", "read"):
        codes, e = s["store"]
        held = s["slots"] >= 0
        at = s["slots"].clamp_min(0)
        if case["op"] == "write":
            c, ee = _quantise(s["x"])
            keep, to = held.nonzero()[:, 0], s["slots"][held]
            codes[to], e[to] = c.view(torch.uint8)[keep], ee[keep]
        v = _dequantise(codes[at].view(torch.float8_e4m3fn), e[at], case["dim"])
        return torch.where(held[:, None], v, 0.0).to(DTYPES[case["out"]])
    if case["op"] == "scores":
        codes, e = s["store"]
        a = _dequantise(*_quantise(s["q"]), case["dim"])
        out = torch.empty(case["m"], case["n"], dtype=DTYPES[case["out"]], device="cuda")
        step = max(1, (1 << 28) // case["dim"])
        for i in range(0, case["n"], step):
            out[:, i:i + step] = (a @ _dequantise(codes[i:i + step].view(torch.float8_e4m3fn), e[i:i + step], case["dim"]).t()).to(out.dtype)
        return out
    m, n, k, scale = case["m"], case["n"], case["k"], case["scale"]
    parts = []
    step = max(1, (1 << 26) // n)
    for i in range(0, m, step):
        x = s["scores"][i:i + step].float()
        cols = torch.arange(n, device="cuda")
        if s["counts"] is not None:
            x = torch.where(cols < s["counts"][i:i + step, None], x, math.inf if scale < 0 else -math.inf)
        z = x * scale
        top = z.amax(dim=1, keepdim=True)
        empty = top == -math.inf
        d = torch.where(empty, -math.inf, z - torch.where(empty, 0.0, top))
        p = d.exp()
        total = p.sum(dim=1, keepdim=True)
        logs = total.log()
        logsum = torch.where(empty, -math.inf, top + logs)
        entropy = torch.where(empty, 0.0, logs + torch.where(p > 0, -d * p, 0.0).sum(dim=1, keepdim=True) / total)
        lp = torch.where(empty, -math.inf, d - logs)
        ids = torch.empty(len(x), 0, dtype=torch.int32, device="cuda")
        if k:
            v, ids = torch.sort(x if scale > 0 else -x, dim=1, descending=True, stable=True)
            v, ids = v[:, :k], ids[:, :k]
            ids = torch.where(v == -math.inf, -1, ids)
        got = torch.where(ids >= 0, lp.gather(1, ids.clamp_min(0).long()), -math.inf)
        if k > n:
            ids = torch.nn.functional.pad(ids, (0, k - n), value=-1)
            got = torch.nn.functional.pad(got, (0, k - n), value=-math.inf)
        given = lp.gather(1, s["targets"][i:i + step].long()) if case["targets"] else lp[:, :0]
        parts.append((logsum[:, 0], entropy[:, 0], given, ids.to(torch.int32), got))
    return _named(case, *(torch.cat(p) for p in zip(*parts)))


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def _held_values(x):
    """the numbers that the 8-bit codes of these rows stand for, from the definition"""
    x = x.double()
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], BLOCK):
        b = x[:, c:c + BLOCK]
        good = torch.isfinite(b)
        a = torch.where(good, b.abs(), 0.0).amax(dim=1)
        e = torch.ceil(torch.log2(a / 448.0)).clamp(-400, 400)       # corrected below where the logarithm rounds across an integer
        e = torch.where(a * torch.exp2(-e) > 448.0, e + 1, e)
        e = torch.where(a * torch.exp2(1 - e) <= 448.0, e - 1, e)
        u = torch.exp2(torch.where(a > 0, e, 0.0).clamp(E_MIN, E_MAX))[:, None]
        y = torch.where(good, b, 0.0) / u
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
        out[:, c:c + BLOCK] = torch.where(good, torch.round(y / step) * step * u, math.nan)
    return out


def exact(case, seed):
    g = _generator(seed)
    if case["op"] in ("write", "read"):
        slots = _slots(case["n"], case["capacity"], g, holes=True)
        if case["op"] == "write":
            x = _embeddings(case["n"], case["dim"], case["dtype"], case["pad"], g)
        else:
            x = _embeddings(case["capacity"], case["dim"], "bf16", 0, g)[slots.clamp_min(0)]
        return torch.where(slots[:, None] >= 0, _held_values(x), 0.0)
    if case["op"] == "scores":
        a = _held_values(_embeddings(case["m"], case["dim"], case["dtype"], 0, g))
        r = _embeddings(case["n"], case["dim"], "bf16", 0, g)
        out = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
        step = max(1, (1 << 26) // case["dim"])
        for i in range(0, case["n"], step):
            out[:, i:i + step] = a @ _held_values(r[i:i + step]).t()
        return out
    scores, counts, targets = _score_rows(case, g)
    m, n, k, scale = case["m"], case["n"], case["k"], case["scale"]
    logsum, entropy = torch.empty(m, dtype=torch.float64, device="cuda"), torch.empty(m, dtype=torch.float64, device="cuda")
    given = torch.full((m, case["targets"]), -math.inf, dtype=torch.float64, device="cuda")
    ids = torch.full((m, k), -1, dtype=torch.int32, device="cuda")
    got = torch.full((m, k), -math.inf, dtype=torch.float64, device="cuda")
    lengths = [n] * m if counts is None else counts.tolist()
    for i, c in enumerate(lengths):
        z = scores[i, :c].double() * scale
        real = (z > -math.inf).nonzero()[:, 0]
        if not len(real):
            logsum[i], entropy[i] = -math.inf, 0.0
            continue
        logsum[i] = torch.logsumexp(z, 0)
        lp = z - logsum[i]
        entropy[i] = -(lp[real].exp() * lp[real]).sum()
        if targets is not None:
            t = targets[i].long()
            given[i] = torch.where(t < c, lp[t.clamp_max(c - 1)], -math.inf)
        if k:
            order = real[torch.sort(z[real], descending=True, stable=True).indices[:k]]
            ids[i, :len(order)] = order.to(torch.int32)
            got[i, :len(order)] = lp[order]
    return _named(case, logsum, entropy, given, ids, got)
