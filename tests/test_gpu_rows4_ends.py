"""4-bit rows, scores against them and adjusted scores at the ends: of f32's range, of sizes, of what a call allows."""
import ctypes as C

import numpy as np
import pytest

import rows4_util as U

pytestmark = pytest.mark.gpu

GROUPS = (32, 64, 128)


def _torch():
    import torch

    return torch


@pytest.fixture(scope="module")
def S(raven_lib):
    from raven_b200 import scoring

    return scoring


def _gpu(x, t="float32"):
    torch = _torch()
    return torch.from_numpy(np.ascontiguousarray(x)).cuda().to(getattr(torch, t))


def _np(t):
    return t.double().cpu().numpy()


def _words(rows):
    return rows.scales.cpu().numpy().view(np.uint32)


def _check(got, q, rows, alpha=1.0, bias=None):
    """f32 scores against the definition in 64 bits; rows4_util.score_bound says how far off they may be. Scores whose
    exact value f32 holds with that bound to spare have to be finite."""
    codes, words = rows.codes.cpu().numpy(), _words(rows)
    v = U.values(codes, words, rows.dim, rows.group)
    exact = alpha * (q @ v.T) + (0.0 if bias is None else bias[None, :])
    lim = U.score_bound(q, codes, words, rows.dim, rows.group, alpha, bias, 2.0 ** -23, exact, True)
    got = _np(got)
    held = np.abs(exact) + lim < np.finfo(np.float32).max
    assert np.isfinite(got[held]).all()
    off = np.abs(got[held] - exact[held])
    assert np.all(off <= lim[held]), (off / lim[held]).max()
    return held


# Few queries, wide ones of 32, 64 and 96 columns; rows that are one slice of all of them, and rows of several.
@pytest.mark.parametrize("dim", [1, 64, 200, 1000, 8200, 20_000])
@pytest.mark.parametrize("nq", [1, 6, 12, 30, 45])
def test_scores_of_the_largest_values(S, nq, dim):
    """Rows of up to f32's largest values against small queries, or with a small alpha: the scores are ordinary ones."""
    r = np.random.default_rng(nq * dim)
    x = 3.4e38 * np.where(np.arange(40)[:, None] % 2 == 0, 1.0, r.uniform(-1, 1, (40, dim)))
    x[::5] *= r.choice([-1.0, 1.0], (8, dim))
    x[1::5] *= 1e-3
    u = r.uniform(0.5, 1.0, (nq, dim)) * r.choice([-1.0, 1.0], (nq, 1))
    for group in GROUPS if dim < 8000 else (GROUPS[nq % 3],):
        rows = S.Int4Rows.encode(_gpu(x), group)
        for size, alpha in ((1e-38, 1.0), (1e-3 / dim, 1.0), (1.0, 1e-30), (1e10, -1e-42), (1e-30, 1e-10), (1e-36, 1e30)):
            q = _gpu(u * size)
            bias = _gpu(r.normal(size=40)) if alpha == 1.0 else None
            got = S.scores(q, rows, alpha=alpha, bias=bias)
            assert _check(got, _np(q), rows, float(np.float32(alpha)), None if bias is None else _np(bias)).all()


@pytest.mark.parametrize("dim", [64, 512, 20_032])
@pytest.mark.parametrize("nq", [1, 12, 45])
def test_scores_of_the_largest_values_that_cancel(S, nq, dim):
    """The first half of a row against the second: sums pass f32's largest value on the way, most scores do not. (Of the
    longest rows against a query of 1 the bound alone passes it: 1900 roundings of 2^-23 of magnitudes of 6e42.)"""
    half = dim // 2
    x = np.full((9, dim), 3e38)
    x[:, half:] *= -np.linspace(0.0, 1.0, 9)[:, None]
    rows = S.Int4Rows.encode(_gpu(x), 32)
    q = _gpu(np.repeat(2.0 ** -np.arange(float(nq))[:, None], dim, 1))
    _check(S.scores(q, rows), _np(q), rows)


def test_scores_tell_what_is_too_large(S):
    """Past f32's largest value a score is infinite, with its sign."""
    torch = _torch()
    rows = S.Int4Rows.encode(torch.full((3, 96), 3e38, device="cuda"))
    for nq in (1, 12, 45):
        q = torch.ones(nq, 96, device="cuda")
        assert bool((S.scores(q, rows) == float("inf")).all())
        assert bool((S.scores(q, rows, alpha=-1.0) == -float("inf")).all())


@pytest.mark.parametrize("dim", [1, 128, 5000, 65_536])
def test_scores_of_the_smallest_steps(S, dim):
    """Steps of 16 significant bits are exact down to 2^-118, and lose what is below 2^-134 from there on. One value of
    a query is not 0, so a score is one product: off by that loss, and by half of what the last bit of a sum stands
    for, 2^-149 * 2^28 / 2^10 / 2 = 2^-132 of the query's largest value (2^28 the sum's scale, 2^10 the query's in the
    longest rows, 2^14 in short ones)."""
    torch = _torch()
    r = np.random.default_rng(dim)
    n = 4096
    exp = np.repeat(np.arange(-127, -95), n // 32)
    step = (2 ** 15 + r.integers(0, 2 ** 15, n)) * 2.0 ** (exp - 15)
    c, z = r.integers(0, 16, n), r.integers(-127, 113, n)
    for group in GROUPS:
        rows = S.Int4Rows.empty(n, dim, "cuda", group)
        rows.codes.zero_(), rows.scales.zero_()
        at, shift = U.held_codes(dim)
        last = dim - 1  # a value of the last group
        rows.codes[:, int(at[last])] = _gpu((c << shift[last]).astype(np.uint8), "uint8")
        word = step.astype(np.float32).view(np.uint32) & np.uint32(0xFFFFFF00) | (z & 255).astype(np.uint32)
        rows.scales[:, last // group] = _gpu(word.view(np.int32), "int32")
        held = (word & np.uint32(0xFFFFFF00)).view(np.float32).astype(np.float64)  # below 2^-126 fewer bits are left
        want = (c + z) * held
        assert np.array_equal(_np(rows.decode()[:, last]), want)
        lost = np.abs(c + z) * np.where(held >= 2.0 ** -118, 0.0, 2.0 ** -134)
        for nq in (1, 12, 45):
            for size in (1.0, 2.0 ** 40):
                q = torch.zeros(nq, dim, device="cuda")
                q[:, last] = size
                got = _np(S.scores(q, rows)) / size
                assert np.all(np.abs(got - want) <= lost + 2.0 ** (-132 if dim > 4096 else -136) + 2.0 ** -149)


def test_adjust_output_over_its_arguments(S):
    from raven_b200._lib import RavenError

    torch = _torch()
    x, b = torch.randn(4, 100, device="cuda"), torch.randn(4, 100, device="cuda")
    words = torch.zeros(4, 100, dtype=torch.int32, device="cuda")
    for call in (lambda: S.adjust(x, bias=b, out=b), lambda: S.adjust(x, bias=b[1], out=b),
                 lambda: S.adjust(x, allow=words, out=words.view(torch.float32)),
                 lambda: S.adjust(x, presence=b.view(-1)[8:12], out=b), lambda: S.adjust(x, bias=x[0], out=x)):
        with pytest.raises(RavenError, match="overlaps"):
            call()
    wide = torch.randn(4, 200, device="cuda")
    want = x + wide[:, 100:]
    assert S.adjust(x, bias=wide[:, 100:], out=wide[:, :100]).equal(want)  # beside one another: no memory is shared


@pytest.mark.parametrize("t", ["float32", "float16", "bfloat16"])
def test_adjust_columns_of_one_matrix(S, t):
    """Scores and output side by side, in either order, starting anywhere."""
    torch = _torch()
    for nq, n, first, gap in ((5, 100, 0, 0), (3, 9001, 3, 1), (7, 63, 5, 0)):
        room = torch.randn(nq, 2 * n + first + gap + 2, device="cuda").to(getattr(torch, t))
        a, b = slice(first, first + n), slice(first + n + gap, first + 2 * n + gap)
        bias = torch.randn(n, device="cuda")
        for src, dst in ((a, b), (b, a)):
            buf = room.clone()
            want = room.clone()
            want[:, dst] = S.adjust(room[:, src].contiguous(), bias=bias)
            S.adjust(buf[:, src], bias=bias, out=buf[:, dst])
            assert torch.equal(buf, want)


class _Scratch:
    """The most that the device's default pool, which scratch comes from, has given out at once."""

    HIGH = 8  # CU_MEMPOOL_ATTR_USED_MEM_HIGH

    def __init__(self):
        self.cuda, self.pool = C.CDLL("libcuda.so.1"), C.c_void_p()
        assert self.cuda.cuDeviceGetDefaultMemPool(C.byref(self.pool), _torch().cuda.current_device()) == 0
        _torch().cuda.synchronize()
        assert self.cuda.cuMemPoolSetAttribute(self.pool, self.HIGH, C.byref(C.c_uint64(0))) == 0

    def high(self):
        _torch().cuda.synchronize()
        most = C.c_uint64(0)
        assert self.cuda.cuMemPoolGetAttribute(self.pool, self.HIGH, C.byref(most)) == 0
        return most.value


def _repeated(S, n, dim, g):
    """(x, rows): n rows of dim values, the 32 of x again and again, whole numbers of -7..8 exactly."""
    torch = _torch()
    x = torch.randint(-7, 8, (n, 32), generator=g, device="cuda").float()
    x[:, 0], x[:, 1] = -7, 8
    short = S.Int4Rows.encode(x, 32)
    codes = torch.empty(n, dim // 2, dtype=torch.uint8, device="cuda")
    # a block holds the words of its four units side by side by quarter
    codes.view(torch.int32).copy_(short.codes.view(torch.int32).repeat_interleave(4, 1).repeat(1, dim // 128))
    return x, S.Int4Rows(codes, short.scales[:, :1].repeat(1, dim // 32).contiguous(), dim, 32)


@pytest.mark.parametrize("nq,n,dim,t", [(40_003, 300, 16_384, "float16"),     # many long queries, few rows, in slices
                                        (300_001, 20, 1024, "float32"),       # queries laid out, no slices
                                        (64, 340_007, 16_384, "float16")])    # one chunk of queries: halves of the rows
def test_scores_in_little_scratch(S, nq, n, dim, t):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(1)
    x, rows = _repeated(S, n, dim, g)
    q = torch.randint(-2, 3, (nq, dim), generator=g, device="cuda", dtype=torch.int8).to(getattr(torch, t))
    bias = torch.arange(n, device="cuda") % 100 + 0.0
    want = torch.cat([p.view(len(p), dim // 32, 32).sum(1, dtype=torch.float32) for p in q.split(5000)]) @ x.T + bias
    scratch = _Scratch()
    got = S.scores(q, rows, bias=bias)
    assert scratch.high() <= (1 << 30) + (1 << 20)  # the pool rounds up
    assert torch.equal(got, want)


def test_adjust_histories_past_32_bits(S):
    """2^32 ids of one query are more than are counted; many histories may have as many together."""
    from raven_b200 import _lib as L

    torch = _torch()
    torch.cuda.empty_cache()
    many = (1 << 32) + 3
    seen = torch.full((many + 40,), 5, dtype=torch.int32, device="cuda")
    seen[many:] = torch.arange(40, dtype=torch.int32, device="cuda") // 2
    x = torch.zeros(3, 100, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, many, many + 10, many + 40], device="cuda")
    got = S.adjust(x, seen=seen, seen_starts=starts, presence=1.0, frequency=0.5, status=status)
    want = torch.zeros(3, 100, device="cuda")
    want[1, :5], want[2, 5:20] = -2.0, -2.0
    assert torch.equal(got, want) and int(status) == L.RAVEN_S_OFFSETS


@pytest.mark.parametrize("t", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("largest", [True, False])
def test_adjust_infinities_are_not_the_largest_values(S, t, largest):
    """Infinities, the type's largest and lowest values and NaN, seen or not, hidden or not, with biases of each kind: each
    stays what it is, and what passes the largest value (or, in 16 bits, half a step above it) becomes an infinity."""
    torch = _torch()
    dt = getattr(torch, t)
    top, f32 = torch.finfo(dt).max, float(torch.finfo(torch.float32).max)
    half = top * (1 + torch.finfo(dt).eps / 4)  # in f32: half a step above the largest value, which rounds to infinity
    vals = [np.inf, -np.inf, np.nan, top, -top, 0.0, -0.0, 1.0, -1.0, top / 2, -top / 2, 1e-45, -1e-45]
    biases = [0.0, np.inf, -np.inf, np.nan, 1.0, half - top, top - half, top, -top, f32, -f32]
    x, bias = np.meshgrid(np.float64(vals), np.float64(biases))
    x, bias = np.tile(x.reshape(-1), 30), np.tile(bias.reshape(-1), 30).astype(np.float32)
    nq, n = 3, len(x)
    scores = torch.from_numpy(np.tile(x, (nq, 1))).to(dt).cuda()
    r = np.random.default_rng(0)
    starts = np.array([0, 0, n, n + 2 * n])
    seen = np.concatenate([np.arange(n), r.integers(0, n, 2 * n)]).astype(np.int32)
    allow = r.integers(-2 ** 31, 2 ** 31, (2, -(-n // 32))).astype(np.int32)
    rows = np.array([0, -1, 1], np.int32)
    with np.errstate(all="ignore"):
        for b in (None, bias):
            for rep, pre, freq in ((1.5, 0.5, 0.25), (0.5, top, 0.0), (1.0, -top, 0.0)):
                got = S.adjust(scores, bias=None if b is None else _gpu(b), allow=_gpu(allow, "int32"),
                               allow_rows=_gpu(rows, "int32"), seen=_gpu(seen, "int32"), seen_starts=_gpu(starts, "int64"),
                               repetition=rep, presence=pre, frequency=freq, largest=largest).cpu()
                want = torch.from_numpy(U.adjust(scores.float().cpu().numpy(), largest, b, allow, rows, seen, starts, rep, pre,
                                                 freq)).to(dt)
                assert torch.equal(got.isnan(), want.isnan())
                assert torch.equal(got[~got.isnan()], want[~want.isnan()])
                assert got.isinf().any() and (got.abs() == top).any()


@pytest.mark.parametrize("t", ["float32", "float16", "bfloat16"])
def test_adjust_hides_with_infinities(S, t):
    """A hidden score is infinite whatever it was, not the type's lowest value, at any start and end of a row."""
    torch = _torch()
    dt = getattr(torch, t)
    for n, first in ((1, 0), (37, 3), (1000, 1), (9000, 5)):
        room = torch.full((3, n + 8), torch.finfo(dt).min, dtype=dt, device="cuda")
        x = room[:, first:first + n]
        x[1] = torch.finfo(dt).max
        x[2] = float("nan")
        bits = torch.randint(-2 ** 31, 2 ** 31, (1, -(-n // 32)), device="cuda").int()
        keep = (bits[0, torch.arange(n, device="cuda") // 32] >> (torch.arange(n, device="cuda") % 32).int() & 1).bool()
        for largest in (True, False):
            got = S.adjust(x, allow=bits, largest=largest)
            worst = torch.tensor(float("-inf" if largest else "inf"), dtype=dt, device="cuda")
            want = torch.where(keep, x, worst)
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[:2], want[:2])
            assert bool((got[2][~keep] == worst).all())
