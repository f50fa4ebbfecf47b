"""64-bit definitions of the operators on 4-bit rows and of adjusted scores, in numpy."""
import numpy as np

BLOCK, UNIT = 128, 32
NAN_WORD = 0x7FC00000


def step_and_offset(lo, hi):
    """(step, z) of a group of values from lo to hi."""
    need = max((hi - lo) / 15.0, max(hi, -lo) / 127.0)
    if need == 0.0:
        return 0.0, 0
    e = max(np.frexp(need)[1], -125)
    step = np.ldexp(np.ceil(np.ldexp(need, 16 - e)), e - 16)
    return step, int(np.rint(lo / step))


def encode(x, group):
    """Codes [n, dim], scale words [n, groups] (uint32) and the values that they stand for."""
    x = np.asarray(x, np.float64)
    n, dim = x.shape
    ng = -(-dim // group)
    codes, words, vals = np.zeros((n, dim), np.int64), np.zeros((n, ng), np.uint32), np.zeros((n, dim))
    for i in range(n):
        for g in range(ng):
            at = slice(g * group, min(dim, (g + 1) * group))
            p = x[i, at]
            if not np.isfinite(p).all():
                words[i, g], vals[i, at] = NAN_WORD, np.nan
                continue
            step, z = step_and_offset(p.min(), p.max())
            words[i, g] = np.float32(step).view(np.uint32) | np.uint32(z & 255)
            if step:
                codes[i, at] = np.minimum(np.rint(p / step) - z, 15)
                vals[i, at] = (codes[i, at] + z) * step
    return codes, words, vals


def held_codes(dim):
    """For each value of a row: the byte that holds its code, and the bits to shift it by."""
    units = -(-dim // UNIT)
    at, shift = np.zeros(dim, np.int64), np.zeros(dim, np.int64)
    for d in range(dim):
        block, unit, quarter, k = d // BLOCK, d % BLOCK // UNIT, d % UNIT // 8, d % 8
        u = min(4, units - 4 * block)
        at[d] = 4 * (16 * block + u * quarter + unit) + k // 2
        shift[d] = 4 * (k % 2)
    return at, shift


def unpack(codes, dim):
    at, shift = held_codes(dim)
    return (np.asarray(codes, np.int64)[:, at] >> shift) & 15


def values(codes, words, dim, group):
    """What rows stand for, from their bytes and words."""
    w = np.asarray(words).astype(np.int64) & 0xFFFFFFFF
    z = ((w & 255) ^ 128) - 128
    step = (w & 0xFFFFFF00).astype(np.uint32).view(np.float32).astype(np.float64)
    c = unpack(codes, dim)
    g = np.arange(dim) // group
    return (c + z[:, g]) * step[:, g]


def score_bound(q, codes, words, dim, group, alpha, bias, out_eps, exact, f32_queries):
    """How far a score may be off. Against a group either sum (c - 8) q and
    (z + 8) * sum q or sum (c + z) q are summed in f32 from products that are exact
    (|c + z| <= |c - 8| + |z + 8|, so the first form bounds both): at most 2 * group
    additions (two parts of each f32 value), each off by 2^-23 of the magnitudes so
    far (truncation counted), and the groups of a row by as many additions more as
    there are groups, with three roundings each. f32 queries keep 22 bits (off by
    2^-23), and every query loses what is below 2^-34 of its largest value. alpha
    and bias add an f32 rounding each, the type of the scores half a step; 1e-37
    covers scores near f32's underflow."""
    w = np.asarray(words).astype(np.int64) & 0xFFFFFFFF
    z = ((w & 255) ^ 128) - 128
    step = (w & 0xFFFFFF00).astype(np.uint32).view(np.float32).astype(np.float64)
    g = np.arange(dim) // group
    mag = (np.abs(unpack(codes, dim) - 8) + np.abs(z[:, g] + 8)) * np.abs(step[:, g])  # of a product's parts, before they cancel
    mags = np.abs(q) @ mag.T
    adds = 2 * min(group, dim) + 3 * (-(-dim // group)) + 4
    off = adds * 2.0 ** -23 * mags + (2.0 ** -23 * mags if f32_queries else 0.0)
    off = off + 2.0 ** -34 * np.abs(q).max(1, keepdims=True) * mag.sum(1)[None, :]
    off = abs(alpha) * off + 2.0 ** -23 * np.abs(exact)
    if bias is not None:
        off = off + 2.0 ** -23 * np.abs(bias)[None, :]
    return off + out_eps / 2 * (np.abs(exact) + off) + 1e-37


def adjust(x, largest, bias=None, allow=None, allow_rows=None, seen=None, starts=None, repetition=1.0, presence=0.0,
           frequency=0.0):
    """Adjusted scores in f32, each operation rounded (not yet rounded to the scores' type)."""
    f = np.float32
    x = np.array(x, f)
    nq, n = x.shape
    per = lambda v: np.broadcast_to(np.asarray(v, f), (nq,))  # noqa: E731
    rep, pre, freq = per(repetition), per(presence), per(frequency)
    with np.errstate(all="ignore"):
        for i in range(nq):
            if starts is not None and 0 <= starts[i] <= starts[i + 1] <= len(seen):
                ids, count = np.unique(seen[starts[i]:starts[i + 1]], return_counts=True)
                for j, c in zip(ids, count):
                    if 0 <= j < n:
                        less = f(pre[i] + f(freq[i] * f(c)))
                        s = x[i, j]
                        s = f(s / rep[i]) if (s > 0) == largest else f(s * rep[i])
                        x[i, j] = f(s - less) if largest else f(s + less)
            if bias is not None:
                x[i] = x[i] + (bias if bias.ndim == 1 else bias[i])
            if allow is not None:
                a = 0 if len(allow) == 1 and allow_rows is None else i if allow_rows is None else allow_rows[i]
                if a >= 0:
                    keep = np.zeros(n, bool)
                    if a < len(allow):
                        j = np.arange(n)
                        keep = (allow[a][j // 32].astype(np.int64) >> (j % 32) & 1).astype(bool)
                    x[i, ~keep] = -np.inf if largest else np.inf
    return x
