"""64-bit definitions of the scoring operators, in numpy."""
import numpy as np

BLOCK = 128


def e4m3_round(y):
    """Nearest e4m3 value (half to even) of |y| <= 448: 3 mantissa bits, normal from 2^-6."""
    y = np.asarray(y, np.float64)
    mag = np.maximum(np.abs(y), 2.0 ** -6)
    step = 2.0 ** (np.floor(np.log2(mag)) - 3)
    return np.rint(y / step) * step


def fp8_exponents(x):
    """Per block: the least e >= -127 with max|finite x| <= 448 * 2^e; 0 for zeros."""
    x = np.asarray(x, np.float64)
    n, dim = x.shape
    nb = -(-dim // BLOCK)
    out = np.zeros((n, nb), np.int64)
    for b in range(nb):
        part = np.abs(x[:, b * BLOCK:(b + 1) * BLOCK])
        top = np.where(np.isfinite(part), part, 0.0).max(1)
        for i, t in enumerate(top):
            if t > 0:
                e = -127
                m, ex = np.frexp(t / 448.0)  # t / 448 rounds: settled by comparing
                e = int(ex) - 1
                while t > 448.0 * 2.0 ** e:
                    e += 1
                while t <= 448.0 * 2.0 ** (e - 1):
                    e -= 1
                out[i, b] = max(e, -127)
    return out


def fp8_values(x):
    """What FP8 rows of x stand for (NaN for what is not finite), and the exponents."""
    x = np.asarray(x, np.float64)
    e = fp8_exponents(x)
    scale = 2.0 ** np.repeat(e, BLOCK, axis=1)[:, : x.shape[1]]
    with np.errstate(invalid="ignore"):
        v = e4m3_round(np.where(np.isfinite(x), x, 0.0) / scale) * scale
    return np.where(np.isfinite(x), v, np.nan), e


def score_bound(q, v, alpha, bias, out_eps, exact):
    """How far a score may be off: the operands are exact in the products, each
    of at most dim additions in f32 is off by at most 2^-23 of the sum of
    magnitudes (truncation counted), alpha and bias add one f32 rounding, and
    the type of the scores half a step; 1e-37 covers scores near f32's underflow."""
    mags = np.abs(q) @ np.abs(v).T
    off = abs(alpha) * (q.shape[1] + 1) * 2.0 ** -23 * mags + 2.0 ** -23 * np.abs(exact)
    if bias is not None:
        off = off + 2.0 ** -23 * np.abs(bias)[None, :]
    return off + out_eps / 2 * (np.abs(exact) + off) + 1e-37


def top_k(rows, k, largest):
    """values, ids, counts by a stable sort: NaN last, equal values by the lower index."""
    nq = len(rows)
    vals, ids, counts = np.zeros((nq, k)), np.zeros((nq, k), np.int64), np.zeros(nq, np.int64)
    for i, r in enumerate(rows):
        r = np.asarray(r, np.float64) + 0.0
        key = np.where(np.isnan(r), np.inf, -r if largest else r)
        # +inf scores sort with NaN by value alone: NaN after them
        order = np.lexsort((np.arange(r.size), np.isnan(r), key))[:k]
        counts[i] = order.size
        vals[i, : order.size] = r[order]
        ids[i, : order.size] = order
    return vals, ids, counts


def group_starts(qo, vo, nq, n):
    """Where each query's scores start, from the definition, for query offsets
    that never fall: groups whose offsets fall or leave the rows have no scores."""
    at, starts = 0, np.zeros(nq + 1, np.int64)
    for g in range(len(qo) - 1):
        a, b, c, d = (int(x) for x in (qo[g], qo[g + 1], vo[g], vo[g + 1]))
        width = d - c if 0 <= a and b <= nq and 0 <= c <= d <= n else 0
        for i in range(max(a, 0), min(b, nq)):
            starts[i] = at + (i - a) * width
        at += (b - a) * width
        starts[max(min(b, nq), 0):] = at
    return starts
