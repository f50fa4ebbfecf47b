"""4-bit rows, scores against them and adjusted scores on the GPU against 64-bit
definitions (rows4_util.py), and a run of them together."""
import numpy as np
import pytest

import rows4_util as U
import scoring_util

pytestmark = pytest.mark.gpu

TYPES = ("f32", "f16", "bf16")
GROUPS = (32, 64, 128)


def _torch():
    import torch

    return torch


def _dt(name):
    torch = _torch()
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


@pytest.fixture(scope="module")
def S(raven_lib):
    from raven_b200 import scoring

    return scoring


def _data(n, dim, seed, spread=6.0):
    """Rows whose groups of 32 differ in size by up to 2^spread either way, some of one sign, some far from 0."""
    r = np.random.default_rng(seed)
    ng = -(-dim // 32)
    x = r.normal(size=(n, ng, 32))
    kind = r.integers(0, 4, (n, ng, 1))
    x = np.where(kind == 1, np.abs(x), np.where(kind == 2, x + 20.0, np.where(kind == 3, -np.abs(x) - 1.0, x)))
    return (x * 2.0 ** r.uniform(-spread, spread, (n, ng, 1))).reshape(n, -1)[:, :dim]


def _gpu(x, t="f32"):
    torch = _torch()
    return torch.from_numpy(np.ascontiguousarray(x)).cuda().to(_dt(t))


def _np(t):
    return t.double().cpu().numpy()


def _words(rows):
    return rows.scales.cpu().numpy().view(np.uint32)


# ---- rows ---------------------------------------------------------------------

SHAPES = [(1, 1), (3, 16), (2, 31), (5, 32), (4, 33), (7, 100), (33, 128), (5, 129), (9, 255), (20, 515), (300, 96), (2, 1500)]


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,dim", SHAPES)
def test_encode_decode(S, t, group, n, dim):
    x = _gpu(_data(n, dim, n * 1000 + dim), t)
    rows = S.Int4Rows.encode(x, group)
    codes, words, vals = U.encode(_np(x), group)
    held, ng = rows.codes.cpu().numpy(), words.shape[1]
    np.testing.assert_array_equal(_words(rows)[:, :ng], words)
    assert np.all(_words(rows)[:, ng:] == 0)
    np.testing.assert_array_equal(U.unpack(held, dim), codes)
    wide = 32 * -(-dim // 32)
    assert np.all(U.unpack(held, wide)[:, dim:] == 0)
    np.testing.assert_array_equal(_np(rows.decode()), vals)
    for out in ("f16", "bf16"):
        want = _torch().from_numpy(vals).to(_dt(out))
        assert _torch().equal(rows.decode(dtype=_dt(out)).cpu(), want)


def test_encode_special_values(S):
    big, tiny = np.finfo(np.float32).max, 1e-42
    x = np.zeros((10, 260))
    x[1, 3] = tiny
    x[2, 130], x[2, 131] = big, -big
    x[3, :] = 7.25                        # all the same, far from 0
    x[4, 0], x[4, 1] = np.inf, 3.0
    x[5, 200], x[5, 201] = np.nan, -7.0
    x[6, 259] = -np.inf
    x[7, :] = 17.0 * 2.0 ** -np.arange(260.0)
    x[8, :] = 200.0 + np.arange(260) % 16
    x[9, :] = -big
    for group in GROUPS:
        rows = S.Int4Rows.encode(_gpu(x), group)
        codes, words, vals = U.encode(x.astype(np.float32), group)
        np.testing.assert_array_equal(_words(rows)[:, : words.shape[1]], words)
        np.testing.assert_array_equal(U.unpack(rows.codes.cpu().numpy(), 260), codes)
        with np.errstate(over="ignore"):  # a step rounded up can take the largest value past f32's
            np.testing.assert_array_equal(rows.decode().cpu().numpy(), vals.astype(np.float32))


@pytest.mark.parametrize("seed", range(4))
def test_encode_at_every_border(S, seed):
    """Values on the border between two codes and the f32 next to it on either side."""
    r = np.random.default_rng(seed)
    n = 300
    step = (r.integers(1 << 15, 1 << 16, n) * 2.0 ** r.integers(-30, 10, n)).astype(np.float32)
    z = r.integers(-112, 113, n)
    x = np.zeros((n, 64), np.float32)
    half = (np.arange(15) + 0.5)[None, :] + z[:, None]
    at = (half * step[:, None].astype(np.float64)).astype(np.float32)
    x[:, :15], x[:, 15:30], x[:, 30:45] = at, np.nextafter(at, np.float32(np.inf)), np.nextafter(at, np.float32(-np.inf))
    x[:, 45], x[:, 46] = z * step, (z + 15) * step
    x[:, 47:] = x[:, 45:46]
    rows = S.Int4Rows.encode(_torch().from_numpy(x).cuda(), 64)
    codes, words, vals = U.encode(x, 64)
    np.testing.assert_array_equal(_words(rows), np.pad(words, ((0, 0), (0, 1))))
    np.testing.assert_array_equal(U.unpack(rows.codes.cpu().numpy(), 64), codes)
    np.testing.assert_array_equal(_np(rows.decode()), vals)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("group", GROUPS)
def test_strided_rows_and_room(S, t, group):
    torch = _torch()
    big = _gpu(_data(40, 333, 5), t)
    x = big[3:33:2, 5:205]  # pitch 666, rows that do not start on 16 bytes
    _, _, vals = U.encode(_np(x), group)
    per = 128 // group
    codes = torch.full((15, 160), 9, dtype=torch.uint8, device="cuda")
    scales = torch.full((15, 4 * per), 9, dtype=torch.int32, device="cuda")
    out = S.Int4Rows(codes, scales, 200, group)
    assert S.Int4Rows.encode(x, group, out=out) is out
    np.testing.assert_array_equal(_np(out.decode()), vals)
    assert bool((codes[:, 112:] == 9).all()) and bool((scales[:, 2 * per:] == 9).all())
    # values into a matrix with room beside them, starting anywhere
    for out_t in TYPES:
        room = torch.full((15, 230), 5.0, dtype=_dt(out_t), device="cuda")
        for first in (0, 1, 8):
            room.fill_(5.0)
            got = out.decode(out=room[:, first:first + 200])
            assert torch.equal(got.cpu(), torch.from_numpy(vals).to(_dt(out_t)))
            assert bool((room[:, :first] == 5).all()) and bool((room[:, first + 200:] == 5).all())
    part = out.rows(4, 7)
    np.testing.assert_array_equal(_np(part.decode()), vals[4:11])


@pytest.mark.parametrize("dim", [7, 16, 100, 128, 130, 256])
@pytest.mark.parametrize("group", GROUPS)
def test_of_index(S, raven_lib, dim, group):
    from raven_b200.index import DeviceIndex, Graph

    base = np.random.default_rng(dim).normal(size=(300, dim)).astype(np.float32)
    g = Graph.build(base, r=8, l=16, alpha=1.2, nav_m=4, directional=True, seed=7)
    rows = S.Int4Rows.of_index(DeviceIndex(g, base, sq4=True), group)
    want = S.Int4Rows.encode(_gpu(base), group)
    assert bool((rows.codes == want.codes).all()) and bool((rows.scales == want.scales).all())


# ---- writing into slots, reading by id --------------------------------------------


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,dim,group", [(1, 1, 128, 64), (5, 9, 100, 32), (64, 1000, 129, 128), (700, 900, 96, 64),
                                           (4096, 5000, 64, 32), (4097, 5000, 33, 64), (9000, 20_000, 40, 128)])
def test_write_and_read_slots(S, t, m, n, dim, group):
    torch = _torch()
    r = np.random.default_rng(m + dim)
    rows = S.Int4Rows.encode(_gpu(r.normal(size=(n, dim))), group)
    before = (rows.codes.clone(), rows.scales.clone())
    x = _gpu(r.normal(size=(m, dim)) * 3.0, t)
    # some left out, some slots more than once
    slots = r.permutation(n)[:m].astype(np.int32)
    slots[r.random(m) < 0.1] = -1
    twice = r.random(m) < 0.2
    slots[twice] = slots[r.integers(0, m, int(twice.sum()))]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert rows.write(x, torch.from_numpy(slots).cuda(), status=status) is rows
    fresh = S.Int4Rows.encode(x, group)
    codes, scales = before[0].cpu().numpy(), before[1].cpu().numpy()
    fc, fs = fresh.codes.cpu().numpy(), fresh.scales.cpu().numpy()
    for i, s in enumerate(slots):  # in order: the last one is held
        if s >= 0:
            codes[s], scales[s] = fc[i], fs[i]
    np.testing.assert_array_equal(rows.codes.cpu().numpy(), codes)
    np.testing.assert_array_equal(rows.scales.cpu().numpy(), scales)
    ids = r.integers(-2, n, 2 * m + 3).astype(np.int32)
    got = rows.decode(torch.from_numpy(ids).cuda(), status=status)
    want = U.values(codes, scales.view(np.uint32), dim, group)[np.maximum(ids, 0)] * (ids >= 0)[:, None]
    np.testing.assert_array_equal(_np(got), want)
    assert int(status) == 0


def test_all_rows_in_one_slot(S):
    torch = _torch()
    for m in (2, 256, 3000, 4096, 5000, 40_000):
        rows = S.Int4Rows.encode(torch.zeros(3, 100, device="cuda"), 32)
        x = torch.randn(m, 100, device="cuda")
        rows.write(x, torch.ones(m, dtype=torch.int32, device="cuda"))
        want = S.Int4Rows.encode(x[-1:], 32).decode()
        got = rows.decode()
        assert torch.equal(got[1], want[0]) and bool((got[::2] == 0).all())


@pytest.mark.parametrize("m", [20, 5000])
def test_slots_and_ids_that_are_not_there(S, m):
    torch = _torch()
    n, dim = 50, 70
    rows = S.Int4Rows.encode(torch.randn(n, dim, device="cuda"))
    want = rows.decode()
    x = torch.randn(m, dim, device="cuda")
    slots = torch.full((m,), n, dtype=torch.int32, device="cuda")
    slots[1], slots[2], slots[3] = 2 ** 31 - 1, -(2 ** 31), 7
    S.take_status()
    rows.write(x, slots)
    assert S.take_status() == 8 and S.take_status() == 0
    want[7] = S.Int4Rows.encode(x[3:4]).decode()[0]
    assert torch.equal(rows.decode(), want)
    ids = torch.tensor([3, n, -1, n - 1, 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32, device="cuda")
    got = rows.decode(ids)
    assert S.take_status() == 8
    assert torch.equal(got[0], want[3]) and torch.equal(got[3], want[n - 1]) and bool((got[[1, 2, 4, 5]] == 0).all())
    rows.decode(ids[[0, 2, 3, 5]])
    rows.write(x[:4], ids[[0, 2, 3, 5]])
    assert S.take_status() == 0
    own = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows.decode(ids, status=own)
    assert int(own) == 8 and S.take_status() == 0


def test_nothing_to_write_or_read(S):
    torch = _torch()
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    rows = S.Int4Rows.encode(torch.randn(5, 40, device="cuda"))
    rows.write(torch.empty(0, 40, device="cuda"), none)
    assert rows.decode(none).shape == (0, 40)
    empty = S.Int4Rows.encode(torch.empty(0, 40, device="cuda"))
    assert len(empty) == 0 and empty.decode().shape == (0, 40)
    # no rows at all: every id is one that is not there
    S.take_status()
    assert bool((empty.decode(torch.tensor([0, 3, -1], dtype=torch.int32, device="cuda")) == 0).all())
    assert S.take_status() == 8
    empty.write(torch.randn(2, 40, device="cuda"), torch.tensor([0, -1], dtype=torch.int32, device="cuda"))
    assert S.take_status() == 8


def test_rows_past_32_bits_of_bytes(S):
    torch = _torch()
    n, dim = 5000, 96
    codes = torch.zeros(n, 1 << 20, dtype=torch.uint8, device="cuda")  # rows 1 MB apart: 5 GB
    rows = S.Int4Rows(codes, torch.zeros(n, 4, dtype=torch.int32, device="cuda"), dim, 32)
    x = torch.randn(40, dim, device="cuda")
    slots = torch.arange(n - 40, n, dtype=torch.int32, device="cuda")
    rows.write(x, slots)
    want = S.Int4Rows.encode(x, 32)
    assert torch.equal(rows.decode(slots), want.decode())
    q = torch.randn(3, dim, device="cuda")
    assert torch.equal(S.scores(q, rows)[:, -40:], S.scores(q, want))


# ---- scores -----------------------------------------------------------------------


def _check(got, q, rows, t, alpha=1.0, bias=None, f32_queries=True):
    codes, words = rows.codes.cpu().numpy(), _words(rows)
    v = U.values(codes, words, rows.dim, rows.group)
    exact = alpha * (q @ v.T) + (0.0 if bias is None else bias[None, :])
    eps, most = _torch().finfo(_dt(t)).eps, _torch().finfo(_dt(t)).max
    lim = U.score_bound(q, codes, words, rows.dim, rows.group, alpha, bias, eps, exact, f32_queries)
    got = _np(got)
    assert got.shape == lim.shape
    # rounding to the type gives an infinity from half a step above its largest value on (f16: 65504 + 16);
    # the bound says on which side of it the f32 sum lies, or that it may be either
    over = np.isinf(got)
    assert np.all(np.sign(got[over]) == np.sign(exact[over])) and np.all(np.abs(exact[over]) + lim[over] >= most)
    assert np.all(over | (np.abs(exact) - lim <= most))
    off = np.abs(np.where(over, exact, got) - exact)
    assert np.all(off <= lim), (off / lim).max()


SCORES = [(1, 1, 1), (1, 7, 32), (2, 33, 96), (3, 65, 100), (5, 130, 128), (7, 100, 129), (8, 257, 200), (9, 300, 256),
          (16, 100, 384), (17, 500, 515), (31, 130, 1000), (33, 1000, 64), (64, 333, 130), (65, 200, 96), (130, 90, 300),
          (1, 5000, 128), (4, 3, 4096), (2, 40, 5000), (20, 70, 1), (40, 300, 20), (70, 129, 33), (96, 128, 128), (25, 1, 500)]


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("qt,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("nq,n,dim", SCORES)
def test_scores(S, nq, n, dim, qt, out, group):
    q = _gpu(_data(nq, dim, nq + dim, 3.0), qt)
    rows = S.Int4Rows.encode(_gpu(_data(n, dim, n, 3.0)), group)
    _check(S.scores(q, rows, dtype=_dt(out)), _np(q), rows, out, f32_queries=qt == "f32")


def test_scores_alpha_bias_pitch(S):
    torch = _torch()
    q, x = _gpu(_data(19, 300, 1, 1.0)), _gpu(_data(77, 300, 2, 1.0))
    rows = S.Int4Rows.encode(x, 64)
    bias = torch.randn(77, device="cuda")
    b = _np(bias)
    for t in TYPES:
        for pitch, first in ((77, 0), (80, 0), (96, 3), (101, 1)):
            room = torch.full((19, pitch + 4), 5.0, dtype=_dt(t), device="cuda")[:, first:]
            out = room[:, :77]
            assert S.scores(q, rows, alpha=-2.0, bias=bias, dtype=_dt(t), out=out) is out
            _check(out, _np(q), rows, t, alpha=-2.0, bias=b)
            assert bool((room[:, 77:] == 5).all())
    # queries at any pitch, starting anywhere
    wide = _gpu(_data(19, 337, 3, 1.0), "bf16")[:, 5:305]
    _check(S.scores(wide, rows), _np(wide), rows, "f32", f32_queries=False)
    one = _gpu(_data(300, 3, 3, 1.0))[:, 1]
    _check(S.scores(one.reshape(300, 1).T.contiguous(), rows), _np(one)[None], rows, "f32")


@pytest.mark.parametrize("nq", [3, 12, 40])
def test_scores_any_alpha(S, nq):
    """alpha and a query's scale, apart and together at the ends of f32's range."""
    torch = _torch()
    rows = S.Int4Rows.encode(_gpu(_data(50, 100, 1, 1.0)), 32)
    q = _data(nq, 100, 2, 1.0)
    for alpha, scale in ((0.0, 1.0), (-3.0, 1.0), (1e30, 1e-25), (1e-30, 1e25), (1e38, 1e-38), (1e-38, 1e30), (1e-42, 1e20), (3e38, 1e-44)):
        x = _gpu(q * scale)
        got, a = S.scores(x, rows, alpha=alpha), float(np.float32(alpha))
        _check(got, _np(x), rows, "f32", alpha=a)
    for alpha in (float("inf"), float("nan")):
        assert not bool(torch.isfinite(S.scores(_gpu(q), rows, alpha=alpha)).any())


def test_scores_of_wide_ranges(S):
    """Values and steps of very different size; the largest and smallest of f32."""
    torch = _torch()
    r = np.random.default_rng(0)
    x = r.normal(size=(70, 200)) * 2.0 ** r.uniform(-60, 60, (70, 1))
    q = r.normal(size=(9, 200)) * 2.0 ** np.array([-100, -60, -20, -3, 0, 3, 20, 40, 60.0])[:, None]
    q[3, ::7] *= 2.0 ** -20
    for group in GROUPS:
        rows = S.Int4Rows.encode(_gpu(x), group)
        _check(S.scores(_gpu(q), rows), _np(_gpu(q)), rows, "f32")
    rows = S.Int4Rows.encode(torch.ones(40, 64, device="cuda"))
    for big in (1e38, 1e-38, 1e-44):
        q = torch.full((2, 64), big, device="cuda")
        q[:, 1:] = 0
        _check(S.scores(q, rows), _np(q), rows, "f32")
    half = torch.full((2, 64), 65504.0, device="cuda", dtype=torch.float16)
    half[1] = 2.0 ** -24
    _check(S.scores(half, rows), _np(half), rows, "f32", f32_queries=False)
    assert bool((S.scores(torch.zeros(3, 64, device="cuda"), rows) == 0).all())


@pytest.mark.parametrize("nq", [1, 6, 40])
def test_scores_not_finite_stay_apart(S, nq):
    torch = _torch()
    x = _data(60, 300, 1, 1.0)
    x[7, 299], x[8, 0], x[59, 130] = np.nan, np.inf, -np.inf
    q = _gpu(_data(nq, 300, 2, 1.0))
    for group in GROUPS:
        rows = S.Int4Rows.encode(_gpu(x), group)
        got = S.scores(q, rows)
        bad = torch.zeros(60, dtype=torch.bool, device="cuda")
        bad[[7, 8, 59]] = True
        assert bool(got[:, bad].isnan().all()) and not bool(got[:, ~bad].isnan().any())
    good = S.Int4Rows.encode(_gpu(_data(60, 300, 1, 1.0)))
    want = S.scores(q, good)
    for what in (float("nan"), float("inf"), -float("inf")):
        for t in TYPES:
            p = q.to(_dt(t))
            clean = S.scores(p, good)
            p[0, 299] = what
            got = S.scores(p, good)
            assert bool(got[0].isnan().all()) and torch.equal(got[1:], clean[1:])
    assert want.shape == (nq, 60)


def test_scores_bytes_past_the_values_do_not_matter(S):
    torch = _torch()
    for dim in (1, 33, 100, 130, 300):
        for group in GROUPS:
            q = _gpu(_data(5, dim, 1, 1.0))
            rows = S.Int4Rows.encode(_gpu(_data(40, dim, 2, 1.0)), group)
            want, vals = S.scores(q, rows), rows.decode()
            codes, scales = rows.codes.clone().cpu().numpy(), rows.scales.clone()
            ng, wide = -(-dim // group), 32 * -(-dim // 32)
            at, shift = U.held_codes(wide)
            for d in range(dim, wide):
                codes[:, at[d]] |= np.uint8(15 << shift[d])
            scales[:, ng:] = U.NAN_WORD
            dirty = S.Int4Rows(torch.from_numpy(codes).cuda(), scales, dim, group)
            assert torch.equal(S.scores(q, dirty), want) and torch.equal(dirty.decode(), vals)


def test_scores_every_code_and_offset(S):
    """One value a row, all codes with all offsets, steps of either sign."""
    torch = _torch()
    c = np.repeat(np.arange(16), 256)
    z = np.tile(np.arange(-128, 128), 16)
    step = np.where(np.arange(4096) % 3 == 0, -0.75, 0.75).astype(np.float32)
    codes = torch.zeros(4096, 16, dtype=torch.uint8, device="cuda")
    codes[:, 0] = torch.from_numpy(c.astype(np.uint8)).cuda()
    word = (step.view(np.uint32) | (z & 255).astype(np.uint32)).view(np.int32)
    rows = S.Int4Rows(codes, torch.from_numpy(word.reshape(-1, 1)).cuda(), 1, 128)
    want = (c + z) * step.astype(np.float64)
    np.testing.assert_array_equal(_np(rows.decode())[:, 0], want)
    for nq in (1, 6, 12, 20, 40):
        for t in TYPES:
            got = _np(S.scores(torch.full((nq, 1), 2.0, device="cuda", dtype=_dt(t)), rows))
            np.testing.assert_array_equal(got, np.broadcast_to(2 * want, got.shape))


def test_scores_empty(S):
    torch = _torch()
    rows = S.Int4Rows.encode(torch.randn(5, 40, device="cuda"))
    assert S.scores(torch.empty(0, 40, device="cuda"), rows).shape == (0, 5)
    none = S.Int4Rows.empty(0, 40, "cuda")
    assert S.scores(torch.randn(3, 40, device="cuda"), none).shape == (3, 0)


def test_scores_exactly(S):
    """Small whole numbers: every sum is exact, whatever its order."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(3)
    for nq, n, dim, group in ((1, 70_001, 128, 64), (3, 9999, 1000, 32), (8, 20_000, 96, 128), (33, 5003, 256, 64),
                              (70, 3001, 4096, 128), (64, 40_000, 128, 32)):
        x = torch.randint(-7, 8, (n, dim), generator=g, device="cuda").float()
        # the group's range is made 15 steps of 1
        x[:, ::32], x[:, 1::32] = -7, 8
        rows = S.Int4Rows.encode(x, group)
        assert torch.equal(rows.decode(), x)
        for t in TYPES:
            q = torch.randint(-2, 3, (nq, dim), generator=g, device="cuda").to(_dt(t))
            want = (q.double() @ x.double().T).float()
            assert torch.equal(S.scores(q, rows), want)


@pytest.mark.parametrize("dim", [8200, 20_000, 65_535, 65_536])
@pytest.mark.parametrize("group", GROUPS)
def test_scores_of_long_rows_exactly(S, dim, group):
    """Rows too long to hold all queries for: slices, whose sums a second kernel adds up. Small whole numbers."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randint(-7, 8, (300, dim), generator=g, device="cuda").float()
    x[:, ::32], x[:, 1::32] = -7, 8
    rows = S.Int4Rows.encode(x, group)
    assert torch.equal(rows.decode(), x)
    bias = torch.arange(300, device="cuda").float()
    for nq in (1, 7, 12, 20, 40, 70):
        for t, out in (("f32", "f32"), ("f16", "f32"), ("bf16", "bf16")):
            q = torch.randint(-2, 3, (nq, dim), generator=g, device="cuda").to(_dt(t))
            want = (q.double() @ x.double().T).float()
            assert torch.equal(S.scores(q, rows, dtype=_dt(out)), want.to(_dt(out)))
        assert torch.equal(S.scores(q, rows, alpha=-2.0, bias=bias), -2.0 * want + bias)


def test_scores_of_slices_in_pieces(S):
    """Sums of slices that would take more than 1 GB of scratch: the rows are taken in halves."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(1)
    n, dim = 30_011, 16_384
    x = torch.randint(-7, 8, (n, 32), generator=g, device="cuda").float()
    x[:, 0], x[:, 1] = -7, 8
    short = S.Int4Rows.encode(x, 32)
    codes = short.codes.repeat(1, 1).new_empty((n, dim // 2))
    # the same 32 values 512 times: a block holds its four units' words side by side by quarter
    w = short.codes.view(torch.int32)  # [n, 4]: a word for each quarter
    codes.view(torch.int32).copy_(w.repeat_interleave(4, 1).repeat(1, dim // 128))
    rows = S.Int4Rows(codes, short.scales[:, :1].repeat(1, dim // 32).contiguous(), dim, 32)
    assert torch.equal(rows.decode(torch.tensor([0, n - 1], dtype=torch.int32, device="cuda")), x[[0, n - 1]].repeat(1, dim // 32))
    q = torch.randint(-2, 3, (1500, dim), generator=g, device="cuda").half()
    bias = torch.arange(n, device="cuda") % 100 + 0.0
    got = S.scores(q, rows, bias=bias)
    want = q.float().view(1500, dim // 32, 32).sum(1) @ x.T + bias
    assert torch.equal(got, want)


def test_scores_past_2_31(S):
    torch = _torch()
    nq, n = 70_000, 33_000
    q = torch.randint(-3, 4, (nq, 16), device="cuda").half()
    x = torch.randint(-7, 8, (n, 16), device="cuda").float()
    x[:, 0], x[:, 1] = -7, 8
    out = S.scores(q, S.Int4Rows.encode(x), dtype=torch.float16)
    assert torch.equal(out[-300:].float(), q[-300:].float() @ x.T)  # whole numbers: exact
    assert torch.equal(out[:200].float(), q[:200].float() @ x.T)


# ---- adjusted scores ----------------------------------------------------------------


def _histories(r, nq, n, most):
    length = (r.random(nq) ** 2 * (most + 1)).astype(np.int64)
    starts = np.concatenate([[0], np.cumsum(length)])
    return (r.random(int(starts[-1])) ** 3 * n).astype(np.int32), starts


def _adjust(S, x, t, largest, **k):
    torch = _torch()
    to = lambda v: torch.from_numpy(np.ascontiguousarray(v)).cuda() if isinstance(v, np.ndarray) else v  # noqa: E731
    names = {"starts": "seen_starts"}
    got = S.adjust(x, largest=largest, **{names.get(a, a): to(b) for a, b in k.items()})
    want = torch.from_numpy(U.adjust(x.float().cpu().numpy(), largest, **k)).to(_dt(t))
    assert got.dtype == x.dtype and torch.equal(got.cpu().nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))
    return got


ADJUST = [(1, 1), (1, 31), (3, 32), (2, 33), (5, 1000), (7, 4095), (4, 4096), (3, 4097), (6, 9001), (2, 40_000), (40, 777)]


@pytest.mark.parametrize("largest", [True, False])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nq,n", ADJUST)
def test_adjust(S, t, nq, n, largest):
    r = np.random.default_rng(nq * 100_000 + n)
    x = _gpu(r.normal(size=(nq, n)) * 3, t)
    seen, starts = _histories(r, nq, n, 3 * n if n < 5000 else 2000)
    f = lambda lo, hi: r.uniform(lo, hi, nq).astype(np.float32)  # noqa: E731
    bits = lambda m: r.integers(-2 ** 31, 2 ** 31, (m, -(-n // 32))).astype(np.int32)  # noqa: E731
    filters = bits(3)
    filters[2] = 0
    which = r.integers(-1, 3, nq).astype(np.int32)
    bias = r.normal(size=n).astype(np.float32)
    pen = dict(seen=seen, starts=starts, repetition=f(0.7, 1.6), presence=f(-1, 1), frequency=f(-0.2, 0.5))
    _adjust(S, x, t, largest)
    _adjust(S, x, t, largest, **pen)
    _adjust(S, x, t, largest, seen=seen, starts=starts, repetition=1.3, presence=0.5, frequency=0.25)
    _adjust(S, x, t, largest, bias=bias)
    _adjust(S, x, t, largest, bias=r.normal(size=(nq, n)).astype(np.float32))
    _adjust(S, x, t, largest, allow=filters, allow_rows=which)
    _adjust(S, x, t, largest, allow=bits(1))
    _adjust(S, x, t, largest, allow=bits(nq))
    _adjust(S, x, t, largest, bias=bias, allow=filters, allow_rows=which, **pen)


@pytest.mark.parametrize("t", TYPES)
def test_adjust_pitch_place_and_room(S, t):
    """Any pitch and start, written elsewhere or in place; nothing beside the scores is touched."""
    torch = _torch()
    r = np.random.default_rng(3)
    for n, pitch, first, out_pitch, out_first in ((500, 500, 0, 512, 0), (500, 520, 8, 500, 0), (501, 503, 1, 509, 3),
                                                  (9001, 9001, 0, 9008, 5), (64, 80, 3, 80, 3), (8200, 8200, 0, 8200, 0)):
        nq = 6
        src = _gpu(r.normal(size=(nq, pitch + 8)), t)
        x = src[:, first:first + n]
        seen, starts = _histories(r, nq, n, 400)
        k = dict(seen=torch.from_numpy(seen).cuda(), seen_starts=torch.from_numpy(starts).cuda(), repetition=1.5,
                 presence=0.25, frequency=0.5, bias=torch.randn(n + 3, device="cuda")[3:],
                 allow=torch.randint(-2 ** 31, 2 ** 31, (2, -(-n // 32) + 3), device="cuda").int()[:, 3:],
                 allow_rows=torch.tensor([0, 1, -1, 0, 1, 1], dtype=torch.int32, device="cuda"))
        want = S.adjust(x.contiguous(), **k)
        ref = U.adjust(x.float().cpu().numpy(), True, k["bias"].cpu().numpy(), k["allow"].cpu().numpy(),
                       k["allow_rows"].cpu().numpy(), seen, starts, 1.5, 0.25, 0.5)
        assert torch.equal(want.cpu(), torch.from_numpy(ref).to(_dt(t)))
        room = torch.full((nq, out_pitch + 8), 5.0, dtype=_dt(t), device="cuda")
        out = room[:, out_first:out_first + n]
        assert S.adjust(x, out=out, **k) is out
        assert torch.equal(out, want) and bool((room[:, :out_first] == 5).all()) and bool((room[:, out_first + n:] == 5).all())
        keep = src.clone()
        S.adjust(x, out=x, **k)
        assert torch.equal(x, want)
        assert torch.equal(src[:, :first], keep[:, :first]) and torch.equal(src[:, first + n:], keep[:, first + n:])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("largest", [True, False])
def test_adjust_values_that_are_not_finite(S, t, largest):
    """Infinities and NaN pass through, except where a filter hides them; the type's lowest value, overflow."""
    torch = _torch()
    low = torch.finfo(_dt(t)).min
    base = [float("inf"), -float("inf"), float("nan"), low, -low, 0.0, -0.0, 1.0, -1.0, 3.0]
    x = torch.tensor([base * 10, base * 10], device="cuda").to(_dt(t))
    n = 100
    allow = np.zeros((1, 4), np.int32)
    allow[0, :2] = -1
    seen = np.concatenate([np.arange(20, 100), np.arange(0, 100)]).astype(np.int32)
    starts = np.array([0, 80, 180])
    bias = np.zeros(n, np.float32)
    bias[40:50], bias[50:60] = np.inf, np.nan
    got = _adjust(S, x, t, largest, allow=allow, seen=seen, starts=starts, repetition=2.0, presence=1.0, frequency=1.0,
                  bias=bias)
    hidden = -float("inf") if largest else float("inf")
    assert bool((got[:, 64:] == hidden).all())
    _adjust(S, x, t, largest, seen=seen, starts=starts, repetition=0.5, presence=float("inf"), frequency=-1.0)


def test_adjust_long_and_repeated_histories(S):
    torch = _torch()
    r = np.random.default_rng(8)
    n = 20_011
    seen = np.concatenate([np.full(100_000, 17), r.integers(0, n, 50_000), np.full(70_000, n - 1), [-1] * 50,
                           np.arange(n)]).astype(np.int32)
    starts = np.array([0, 100_000, 150_000, 150_000, 220_050, len(seen)])
    for t in TYPES:
        x = _gpu(r.normal(size=(5, n)), t)
        _adjust(S, x, t, True, seen=seen, starts=starts, repetition=1.1, presence=0.1, frequency=2.0 ** -10)
    assert S.take_status() == 0
    del torch


def test_adjust_bad_histories_and_filters(S):
    torch = _torch()
    x = torch.randn(5, 100, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    i64 = lambda *v: torch.tensor(v, device="cuda")  # noqa: E731
    S.take_status()
    seen = i32(3, 100, 4, -1, 2 ** 31 - 1, -(2 ** 31), 5)
    got = S.adjust(x, seen=seen, seen_starts=i64(0, 2, 3, 5, 6, 7), presence=1.0)
    assert S.take_status() == 8
    want = x.clone()
    want[0, 3] -= 1
    want[1, 4] -= 1
    want[4, 5] -= 1
    assert torch.equal(got, want)
    big = 2 ** 62
    for starts, good in ((i64(0, 2, 1, 3, 4, 7), (0, 2, 3, 4)), (i64(-1, 1, 1, 1, 1, 1), (1, 2, 3, 4)), (i64(0, 0, 0, 0, 0, 8), ()),
                         (i64(-big, big, -big, big, 0, 1), (4,)), (i64(9, 9, 9, 9, 9, 9), ())):
        S.take_status()
        got = S.adjust(x, seen=seen, seen_starts=starts, presence=1.0)
        assert S.take_status() & 1
        ref = U.adjust(x.cpu().numpy(), True, seen=seen.cpu().numpy(), starts=starts.cpu().numpy(), presence=1.0)
        assert torch.equal(got.cpu(), torch.from_numpy(ref))
    allow = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    status = i32(0)
    got = S.adjust(x, allow=allow, allow_rows=i32(0, 2, -7, 2 ** 31 - 1, 1), status=status)
    assert int(status) == 8 and S.take_status() == 0
    assert torch.equal(got[[0, 2, 4]], x[[0, 2, 4]]) and bool((got[[1, 3]] == -float("inf")).all())
    # no history at all; starts that leave it
    assert torch.equal(S.adjust(x, seen=i32()[:0], seen_starts=i64(0, 0, 0, 0, 0, 0), presence=1.0), x)
    assert S.take_status() == 0
    assert torch.equal(S.adjust(x, seen=i32()[:0], seen_starts=i64(0, 0, 1, 1, 1, 1), presence=1.0), x)
    assert S.take_status() == 1


def test_adjust_past_2_31(S):
    torch = _torch()
    nq, n = 70_000, 33_001
    x = torch.zeros(nq, n, dtype=torch.float16, device="cuda")
    seen = torch.tensor([33_000, 5], dtype=torch.int32, device="cuda")
    starts = torch.zeros(nq + 1, dtype=torch.int64, device="cuda")
    starts[-1] = 2
    out = S.adjust(x, seen=seen, seen_starts=starts, presence=2.0, bias=torch.arange(n, device="cuda") % 7 + 0.0, out=x)
    want = (torch.arange(n, device="cuda") % 7).half()
    assert torch.equal(out[-2], want)
    want[[5, 33_000]] -= 2
    assert torch.equal(out[-1], want)


def test_adjust_empty(S):
    torch = _torch()
    assert S.adjust(torch.empty(0, 40, device="cuda"), bias=torch.zeros(40, device="cuda")).shape == (0, 40)
    assert S.adjust(torch.empty(3, 0, device="cuda"), presence=1.0).shape == (3, 0)


# ---- together -----------------------------------------------------------------------


@pytest.mark.parametrize("t", TYPES)
def test_search_of_a_changing_collection(S, t):
    """A collection in 4 bits is changed in place, scored, filtered, searched, and
    the candidates are read back and ranked, twice."""
    torch = _torch()
    r = np.random.default_rng(5)
    n, dim, nq, k = 3000, 96, 12, 20
    x = r.normal(size=(n, dim)).astype(np.float32)
    rows = S.Int4Rows.encode(_gpu(x), 32)
    held = U.encode(x, 32)[2]
    filters = r.integers(-2 ** 31, 2 ** 31, (2, -(-n // 32))).astype(np.int32)
    which = np.array([0, 1, -1] * 4, np.int32)
    seen, starts = _histories(r, nq, n, 300)
    for turn in range(2):
        fresh = _gpu(r.normal(size=(500, dim)), t)
        slots = r.permutation(n)[:500].astype(np.int32)
        rows.write(fresh, torch.from_numpy(slots).cuda())
        held[slots] = U.encode(_np(fresh), 32)[2]
        q = _gpu(r.normal(size=(nq, dim)), t)
        s = S.scores(q, rows)
        a = S.adjust(s, allow=torch.from_numpy(filters).cuda(), allow_rows=torch.from_numpy(which).cuda(),
                     seen=torch.from_numpy(seen).cuda(), seen_starts=torch.from_numpy(starts).cuda(), presence=1.0,
                     frequency=0.5)
        vals, ids, counts = S.top_k(a, k)
        near = rows.decode(ids.reshape(-1)).view(nq, k, dim)
        ranked = (near * q.float()[:, None]).sum(2)
        want = U.adjust(s.cpu().numpy(), True, None, filters, which, seen, starts, 1.0, 1.0, 0.5)
        wv, wi, wc = scoring_util.top_k(want, k, True)
        np.testing.assert_array_equal(ids.cpu().numpy(), wi)
        np.testing.assert_array_equal(_np(vals), wv)
        np.testing.assert_array_equal(_np(near), held[wi])
        exact = np.einsum("qkd,qd->qk", held[wi], _np(q))
        assert np.abs(_np(ranked) - exact).max() <= dim * 2.0 ** -22 * np.abs(held).max() * np.abs(_np(q)).max()
        bound = U.score_bound(_np(q), rows.codes.cpu().numpy(), _words(rows), dim, 32, 1.0, None, 2.0 ** -23, _np(q) @ held.T, True)
        assert np.all(np.abs(_np(s) - _np(q) @ held.T) <= bound)


def _pass(S, rows, x, slots, q, seen, starts, allow):
    rows.write(x, slots)
    s = S.adjust(S.scores(q, rows), seen=seen, seen_starts=starts, presence=0.5, allow=allow)
    vals, ids, _ = S.top_k(s, 9)
    return vals, ids, rows.decode(ids.reshape(-1), dtype=_torch().float16)


def _inputs(seed, m=5000, n=6000, dim=200, nq=20):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    starts = torch.arange(nq + 1, device="cuda") * 50
    return dict(x=r(m, dim), slots=torch.randint(-1, n, (m,), generator=g, device="cuda").int(), q=r(nq, dim),
                seen=torch.randint(0, n, (nq * 50,), generator=g, device="cuda").int(), starts=starts,
                allow=torch.randint(-2 ** 31, 2 ** 31, (nq, -(-n // 32)), generator=g, device="cuda").int())


def test_streams_and_graphs(S):
    """Passes on two streams at once, and captured passes replayed on new inputs, give what eager calls give."""
    torch = _torch()
    for m in (300, 5000):
        ins = [_inputs(i, m) for i in range(4)]
        stores = [S.Int4Rows.encode(torch.zeros(6000, 200, device="cuda")) for _ in range(4)]
        want = []
        for i, rows in zip(ins, stores):
            want.append(_pass(S, rows, **i))
            torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(4)]
        for _ in range(5):
            got = []
            for st, rows, i in zip(streams, stores, ins):
                with torch.cuda.stream(st):
                    got.append(_pass(S, rows, **i))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
        graphs = []
        for j in range(2):
            buf = {k: v.clone() for k, v in ins[j].items()}
            rows = S.Int4Rows.encode(torch.zeros(6000, 200, device="cuda"))
            torch.cuda.synchronize()
            graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            with torch.cuda.graph(graph, stream=side):
                out = _pass(S, rows, **buf)
            graphs.append((graph, buf, rows, out))
        for turn in range(3):
            for j, (graph, buf, rows, _) in enumerate(graphs):
                with torch.cuda.stream(streams[j]):
                    rows.codes.zero_()
                    rows.scales.zero_()
                    for k, v in ins[(turn + j) % 4].items():
                        buf[k].copy_(v)
                    graph.replay()
            torch.cuda.synchronize()
            for j, (_, _, _, out) in enumerate(graphs):
                assert all(torch.equal(x, y) for x, y in zip(out, want[(turn + j) % 4]))


def test_first_call_inside_a_capture(raven_lib):
    """A process whose first calls of the library are captured."""
    import os
    import subprocess
    import sys

    code = """
import torch
from raven_b200 import scoring as S
x, q = torch.randn(5000, 96, device="cuda"), torch.randn(64, 96, device="cuda")
slots = torch.randperm(5000, device="cuda").int()
rows = S.Int4Rows.empty(5000, 96, "cuda")
seen, starts = torch.arange(640, device="cuda").int(), torch.arange(65, device="cuda") * 10
def f():
    rows.write(x, slots)
    s = S.adjust(S.scores(q, rows), seen=seen, seen_starts=starts, presence=1.0)
    return S.scores(q[:3], rows), s, rows.decode(slots)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = f()
for _ in range(3):
    x.normal_(); q.normal_()
    graph.replay()
    torch.cuda.synchronize()
    kept = [t.clone() for t in got]
    want = f()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, want))
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_two_threads(S):
    import threading

    torch = _torch()
    ins = [_inputs(30 + i) for i in range(2)]
    stores = [S.Int4Rows.encode(torch.zeros(6000, 200, device="cuda")) for _ in range(2)]
    want = [_pass(S, rows, **i) for rows, i in zip(stores, ins)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = _pass(S, stores[i], **ins[i])
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


def test_same_results_every_time(S):
    torch = _torch()
    i = _inputs(1)
    rows = S.Int4Rows.encode(torch.zeros(6000, 200, device="cuda"))
    first = [t.clone() for t in _pass(S, rows, **i)] + [S.scores(i["q"][:2], rows)]
    for _ in range(4):
        again = [*_pass(S, rows, **i), S.scores(i["q"][:2], rows)]
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_rows_keep_no_old_memory(S):
    torch = _torch()
    x = torch.randn(50, 64, device="cuda")
    rows = S.Int4Rows.encode(x)
    want = rows.decode()
    new = rows.codes.clone()
    rows.codes.set_(new)
    assert torch.equal(rows.decode(), want) and rows._rows.data == new.data_ptr()


def test_refusals(S):
    torch = _torch()
    x, rows = torch.randn(4, 64, device="cuda"), S.Int4Rows.encode(torch.randn(9, 64, device="cuda"))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    slots = i32(0, 1, 2, 3)
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="cuda")  # noqa: E731
    w = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    calls = [
        lambda: S.Int4Rows.encode(x, 48),
        lambda: S.Int4Rows.encode(x.double()),
        lambda: S.Int4Rows.encode(x.cpu()),
        lambda: S.Int4Rows.encode(x, out=rows),
        lambda: S.Int4Rows.encode(x, 32, out=rows.rows(0, 4)),
        lambda: S.Int4Rows.encode(torch.randn(4, 0, device="cuda")),
        lambda: S.Int4Rows.empty(-1, 64, "cuda"),
        lambda: S.Int4Rows(u8(4, 16), w(4, 2), 64, 64),
        lambda: S.Int4Rows(u8(4, 32), w(4, 1), 64, 64),
        lambda: S.Int4Rows(u8(4, 32), w(5, 2), 64, 64),
        lambda: S.Int4Rows(u8(4, 32).cpu(), w(4, 2).cpu(), 64, 64),
        lambda: S.Int4Rows(w(4, 32), w(4, 2), 64, 64),
        lambda: S.Int4Rows(u8(4, 64)[:, ::2], w(4, 2), 64, 64),
        lambda: S.Int4Rows(u8(4, 32), w(4, 2), 0, 64),
        lambda: rows.write(x[:, :63], slots),
        lambda: rows.write(x, slots[:3]),
        lambda: rows.write(x, slots.long()),
        lambda: rows.write(x, slots.cpu()),
        lambda: rows.write(x, torch.stack([slots, slots], 1)[:, 0]),
        lambda: rows.write(x.cpu(), slots),
        lambda: rows.decode(slots.long()),
        lambda: rows.decode(dtype=torch.float64),
        lambda: rows.decode(out=torch.empty(8, 64, device="cuda")),
        lambda: rows.decode(slots, out=torch.empty(64, 4, device="cuda").T),
        lambda: rows.decode(status=w(2)),
        lambda: rows.rows(5, 5),
        lambda: S.scores(x[:, :32], rows),
        lambda: S.scores(rows, rows),
        lambda: S.scores(S.Fp8Rows.encode(x), rows),
        lambda: S.scores(x, rows, dtype=torch.int32),
        lambda: S.scores(x, rows, bias=torch.zeros(8, device="cuda")),
        lambda: S.scores(x, rows, out=torch.empty(4, 8, device="cuda")),
        lambda: S.group_scores(x, torch.tensor([0, 4], device="cuda"), rows, torch.tensor([0, 9], device="cuda"), total=36),
    ]
    s = torch.randn(4, 100, device="cuda")
    starts = torch.tensor([0, 1, 2, 3, 4], device="cuda")
    calls += [
        lambda: S.adjust(s.cpu()),
        lambda: S.adjust(s.double()),
        lambda: S.adjust(s[0]),
        lambda: S.adjust(s.T),
        lambda: S.adjust(s, bias=torch.zeros(99, device="cuda")),
        lambda: S.adjust(s, bias=torch.zeros(100, device="cuda").half()),
        lambda: S.adjust(s, bias=torch.zeros(100)),
        lambda: S.adjust(s, bias=torch.zeros(100, 4, device="cuda").T),
        lambda: S.adjust(s, allow=w(3)),
        lambda: S.adjust(s, allow=w(2, 4)),
        lambda: S.adjust(s, allow=w(0, 4), allow_rows=slots),
        lambda: S.adjust(s, allow=w(2, 4).long(), allow_rows=slots),
        lambda: S.adjust(s, allow=w(2, 4), allow_rows=slots[:3]),
        lambda: S.adjust(s, allow_rows=slots),
        lambda: S.adjust(s, seen=slots),
        lambda: S.adjust(s, seen_starts=starts),
        lambda: S.adjust(s, seen=slots, seen_starts=starts[:4]),
        lambda: S.adjust(s, seen=slots.long(), seen_starts=starts),
        lambda: S.adjust(s, seen=slots, seen_starts=starts.int()),
        lambda: S.adjust(s, repetition=0.0),
        lambda: S.adjust(s, repetition=float("nan")),
        lambda: S.adjust(s, presence=torch.zeros(3, device="cuda")),
        lambda: S.adjust(s, presence=torch.zeros(4, device="cuda").half()),
        lambda: S.adjust(s, presence=torch.zeros(4)),
        lambda: S.adjust(s, out=torch.empty(4, 99, device="cuda")),
        lambda: S.adjust(s, out=torch.empty(4, 100, device="cuda").half()),
        lambda: S.adjust(s, status=w(1).long()),
    ]
    for k, call in enumerate(calls):
        with pytest.raises((ValueError, TypeError)):
            call()
            print(k)
    # refused by the library
    from raven_b200._lib import RavenError

    long = torch.empty(4 * 100 + 50, device="cuda")
    a, b = long[:400].view(4, 100), long[50:].view(4, 100)
    for call in (lambda: S.adjust(a, out=b), lambda: S.adjust(b, out=a),
                 lambda: S.adjust(long[:400:1].view(4, 100)[:, :50], out=long[10:410].view(4, 100)[:, :50]),
                 lambda: S.Int4Rows(u8(4 * 40).view(4, 40)[:, :32], w(4, 2), 64, 64).decode(),
                 lambda: S.Int4Rows(u8(4 * 32 + 8)[8:].view(4, 32), w(4, 2), 64, 64).decode(),
                 lambda: S.Int4Rows(u8(4, 32), w(9)[1:].view(4, 2), 64, 64).decode(),
                 lambda: S.Int4Rows(u8(4, 32), w(12).view(4, 3)[:, :2], 64, 64).decode()):
        with pytest.raises((RavenError, ValueError)):
            call()
