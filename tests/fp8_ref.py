"""Plain numpy restatements, in 64 bits, of the 8-bit row store's operators (include/comet_gpu.h: comet_fp8_*, comet_logprobs_*)."""
import numpy as np

BLOCK = 128
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}       # half a step, relative


def to_bf16_bits(x):
    """float32 -> bfloat16 bits, to nearest even; NaN stays NaN"""
    b = np.asarray(x, np.float32).view(np.uint32)
    r = (b.astype(np.uint64) + 0x7FFF + ((b >> 16) & 1)) >> 16
    return np.where(np.isnan(np.asarray(x, np.float32)), 0x7FC0, r).astype(np.uint16)


def from_bf16_bits(u):
    return (np.asarray(u, np.uint16).astype(np.uint32) << 16).view(np.float32)


def encode(x, dtype):
    """float32 array -> the array whose bytes go to the device"""
    with np.errstate(over="ignore"):
        return {"f32": lambda: np.asarray(x, np.float32), "f16": lambda: np.asarray(x, np.float32).astype(np.float16), "bf16": lambda: to_bf16_bits(x)}[dtype]()


def decode(a, dtype):
    """device bytes -> float32 values"""
    return from_bf16_bits(a) if dtype == "bf16" else np.asarray(a).astype(np.float32)


NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


def held(x):
    """the numbers the codes of these rows stand for (float64)"""
    x = np.asarray(x, np.float64)
    out = np.empty_like(x)
    for c in range(0, x.shape[1], BLOCK):
        b = x[:, c:c + BLOCK]
        fin = np.isfinite(b)
        A = np.where(fin, np.abs(b), 0.0).max(axis=1, initial=0.0)
        f, p = np.frexp(A)                                   # A = f * 2^p, f in [0.5, 1): 448 = 0.875 * 2^9
        e = np.maximum(np.where(A == 0, -126, p - 9 + (f > 0.875)), -126).astype(np.int64)
        u = np.ldexp(1.0, e)[:, None]
        y = np.where(fin, b, 0.0) / u
        _, q = np.frexp(np.maximum(np.abs(y), 2.0 ** -6))
        step = np.ldexp(1.0, q - 1 - 3)
        out[:, c:c + BLOCK] = np.where(fin, np.rint(y / step) * step * u, np.nan)
    return out


def logprobs(scores, n, counts, scale, targets, k):
    """scores: float32 values (m x >= n). Returns logsum, entropy, logprobs, ids, top_logprobs in float64 / int."""
    m = scores.shape[0]
    T = 0 if targets is None else targets.shape[1]
    L, H = np.empty(m), np.empty(m)
    lp, ids, tl = np.full((m, T), -np.inf), np.full((m, k), -1, np.int64), np.full((m, k), -np.inf)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        for i in range(m):
            c = n if counts is None else int(np.clip(counts[i], 0, n))
            z = scores[i, :c].astype(np.float64) * scale
            order = np.argsort(-np.where(np.isnan(z), -np.inf, z), kind="stable")
            order = order[z[order] > -np.inf][:k]
            ids[i, :len(order)] = order
            real = z[z > -np.inf]
            if np.isnan(z).any() or (z == np.inf).any():
                L[i] = H[i] = np.nan
                full = np.full(c, np.nan)
            elif not len(real):
                L[i], H[i], full = -np.inf, 0.0, np.full(c, -np.inf)
            else:
                M = real.max()
                log_s = np.log(np.exp(real - M).sum())
                L[i] = M + log_s
                full = (z - M) - log_s              # not z - L: a row of the type's lowest value has an L that swallows log S
                lr = (real - M) - log_s
                H[i] = -(np.exp(lr) * lr).sum()
            tl[i, :len(order)] = full[order]
            for t in range(T):
                if 0 <= targets[i, t] < c:
                    lp[i, t] = full[targets[i, t]]
    return L, H, lp, ids, tl
