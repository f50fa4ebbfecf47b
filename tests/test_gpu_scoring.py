"""Scoring operators on the GPU against 64-bit definitions (scoring_util.py):
FP8 rows, dense and grouped scores, top-k of rows, and a run of them together."""
import numpy as np
import pytest

import scoring_util as U

pytestmark = pytest.mark.gpu

TYPES = ("f32", "f16", "bf16")


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
    """Rows whose blocks differ in size by up to 2^spread either way."""
    r = np.random.default_rng(seed)
    x = r.normal(size=(n, dim))
    nb = -(-dim // U.BLOCK)
    return x * np.repeat(2.0 ** r.uniform(-spread, spread, (n, nb)), U.BLOCK, axis=1)[:, :dim]


def _gpu(x, t="f32"):
    torch = _torch()
    return torch.from_numpy(np.ascontiguousarray(x)).cuda().to(_dt(t))


def _np(t):
    return t.double().cpu().numpy()


# ---- FP8 rows -----------------------------------------------------------------


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,dim", [(1, 1), (3, 16), (7, 100), (33, 128), (5, 129), (20, 515), (300, 96), (2, 1500)])
def test_fp8_encode_decode(S, t, n, dim):
    x = _gpu(_data(n, dim, n * 1000 + dim), t)
    rows = S.Fp8Rows.encode(x)
    want, e = U.fp8_values(_np(x))
    nb = e.shape[1]
    exps = rows.exps.cpu().numpy().astype(np.int64)
    np.testing.assert_array_equal(exps[:, :nb] - 127, e)
    assert np.all(exps[:, nb:] == 127)
    assert np.all(rows.codes.cpu().numpy()[:, dim:] == 0)
    np.testing.assert_array_equal(_np(rows.decode()), want)


def test_fp8_encode_special_values(S):
    x = np.zeros((8, 260))
    x[1, 3] = 1e-42                       # an f32 subnormal: the least exponent
    x[2, 130] = np.finfo(np.float32).max  # the largest exponent
    x[3, :5] = [448.0, -448.0, 464.0, 1.0, 2.0 ** -9]
    x[4, 0], x[4, 1], x[4, 2] = np.inf, 3.0, -np.inf
    x[5, 200], x[5, 201] = np.nan, -7.0
    x[6, :] = np.nan
    x[7, :] = 17.0 * 2.0 ** -np.arange(260.0)  # ties and values below e4m3's normal range
    rows = S.Fp8Rows.encode(_gpu(x))
    want, e = U.fp8_values(x.astype(np.float32))
    np.testing.assert_array_equal(rows.exps.cpu().numpy()[:, :3].astype(np.int64) - 127, e)
    with np.errstate(over="ignore"):  # f32's largest value rounds to 2^128, which f32 cannot hold
        np.testing.assert_array_equal(rows.decode().cpu().numpy(), want.astype(np.float32))


def test_fp8_encode_ties_to_even(S):
    # 448 fixes the scale at 1; halves between neighbours go to the even code
    x = np.zeros((1, 128))
    x[0, :6] = [448.0, 17.0, 19.0, 25.0, 27.0, -17.0]
    got = _np(S.Fp8Rows.encode(_gpu(x)).decode())[0, :6]
    np.testing.assert_array_equal(got, [448.0, 16.0, 20.0, 24.0, 28.0, -16.0])


@pytest.mark.parametrize("t", TYPES)
def test_fp8_encode_strided_rows_and_reuse(S, t):
    torch = _torch()
    big = _gpu(_data(40, 333, 5), t)
    x = big[3:33:2, 5:205]  # pitch 666, rows that do not start on 16 bytes
    want, _ = U.fp8_values(_np(x))
    out = S.Fp8Rows(torch.full((15, 256), 9, dtype=torch.uint8, device="cuda"),
                    torch.full((15, 8), 9, dtype=torch.uint8, device="cuda"), 200)
    assert S.Fp8Rows.encode(x, out=out) is out
    np.testing.assert_array_equal(_np(out.decode()), want)
    assert bool((out.codes[:, 208:] == 9).all()) and bool((out.exps[:, 4:] == 9).all())


def test_fp8_of_index(S, small_case):
    from raven_b200.index import DeviceIndex

    base, _, g = small_case
    rows = S.Fp8Rows.of_index(DeviceIndex(g, base, sq4=True))
    want = S.Fp8Rows.encode(_gpu(base))
    assert bool((rows.codes == want.codes).all()) and bool((rows.exps == want.exps).all())


# ---- dense scores ---------------------------------------------------------------


def _check(got, q, v, t, alpha=1.0, bias=None):
    exact = alpha * (q @ v.T) + (0.0 if bias is None else bias[None, :])
    eps = _torch().finfo(_dt(t)).eps
    off = np.abs(_np(got) - exact)
    lim = U.score_bound(q, v, alpha, bias, eps, exact)
    assert off.shape == lim.shape
    assert np.all(off <= lim), (off / lim).max()


SHAPES = [(1, 1, 1), (1, 1000, 128), (3, 77, 100), (16, 128, 96), (17, 129, 130), (33, 1000, 512), (64, 300, 640),
          (100, 257, 33), (130, 500, 1000), (200, 640, 129), (257, 20000, 64), (500, 311, 2050), (1, 64, 8192)]


@pytest.mark.parametrize("nq,n,dim", SHAPES)
@pytest.mark.parametrize("qt,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_scores_fp8(S, nq, n, dim, qt, out):
    # bounded spread: f16 scores stay finite
    q, v = _gpu(_data(nq, dim, 1, 2.0), qt), _gpu(_data(n, dim, 2, 2.0) / dim)
    rows = S.Fp8Rows.encode(v)
    got = S.scores(q, rows, dtype=_dt(out))
    qv, _ = U.fp8_values(_np(q))
    _check(got, qv, _np(rows.decode()), out)
    assert bool((S.scores(S.Fp8Rows.encode(q), rows, dtype=_dt(out)) == got).all())


def test_scores_fp8_far_scales(S):
    """Blocks of very different size: every exponent reaches its own block, row and query."""
    q, v = _gpu(_data(140, 1400, 3, 20.0)), _gpu(_data(270, 1400, 4, 20.0))
    rows = S.Fp8Rows.encode(v)
    qv, _ = U.fp8_values(_np(q))
    _check(S.scores(q, rows), qv, _np(rows.decode()), "f32")


@pytest.mark.parametrize("nq,n,dim", SHAPES)
@pytest.mark.parametrize("t,out", [("f16", "f32"), ("bf16", "bf16")])
def test_scores_16bit(S, nq, n, dim, t, out):
    q, v = S.aligned_rows(_gpu(_data(nq, dim, 5, 1.0), t)), S.aligned_rows(_gpu(_data(n, dim, 6, 1.0), t))
    _check(S.scores(q, v, dtype=_dt(out)), _np(q), _np(v), out)


def test_scores_alpha_bias_pitch(S):
    torch = _torch()
    q, v = _data(70, 200, 7, 1.0), _data(333, 200, 8, 1.0)
    rows = S.Fp8Rows.encode(_gpu(v))
    vv, (qv, _) = _np(rows.decode()), U.fp8_values(_gpu(q).cpu().numpy())
    norms = (rows.decode() ** 2).sum(1)
    room = torch.full((70, 400), 7.0, device="cuda")
    got = S.scores(_gpu(q), rows, alpha=-2.0, bias=norms, out=room[:, 11:344])
    _check(got, qv, vv, "f32", -2.0, _np(norms))
    assert bool((room[:, :11] == 7.0).all()) and bool((room[:, 344:] == 7.0).all())


def test_scores_not_finite_rows_stay_apart(S):
    """A row or query with NaN or infinities only spoils its own scores."""
    q, v = _data(40, 150, 9, 1.0), _data(200, 150, 10, 1.0)
    clean = S.scores(_gpu(q), S.Fp8Rows.encode(_gpu(v)))
    q[7, 3], v[131, 140], v[5, 0] = np.nan, np.inf, np.nan
    got = S.scores(_gpu(q), S.Fp8Rows.encode(_gpu(v)))
    bad = np.zeros((40, 200), bool)
    bad[7], bad[:, 131], bad[:, 5] = True, True, True
    got, clean = _np(got), _np(clean)
    assert np.all(np.isnan(got[bad]))
    # the blocks that hold what is not finite have another scale; no other score moves
    np.testing.assert_array_equal(got[~bad], clean[~bad])


def test_scores_empty(S):
    torch = _torch()
    rows = S.Fp8Rows.encode(_gpu(_data(5, 64, 1)))
    assert S.scores(torch.empty(0, 64, device="cuda"), rows).shape == (0, 5)
    assert S.scores(torch.zeros(3, 64, device="cuda"), rows.rows(2, 0)).shape == (3, 0)
    assert S.Fp8Rows.encode(torch.empty(0, 64, device="cuda")).decode().shape == (0, 64)


def test_scores_large_offsets(S):
    """Scores past 2^31 elements."""
    torch = _torch()
    nq, n = 70_000, 33_000
    q = torch.randint(-3, 4, (nq, 16), device="cuda").half()
    v = torch.randint(-3, 4, (n, 16), device="cuda").half()
    out = S.scores(q, v, dtype=torch.float16)
    want = q[-300:].float() @ v.float().T  # whole numbers: exact
    assert bool((out[-300:].float() == want).all())
    assert bool((out[:200].float() == q[:200].float() @ v.float().T).all())


# ---- grouped scores ---------------------------------------------------------------


def _groups(seed, groups, nq, n, even=False):
    r = np.random.default_rng(seed)

    def cut(total):
        w = r.random(groups) ** 3 * (r.random(groups) > 0.2)
        w[0] += 1e-3
        c = np.rint(np.cumsum(w) / w.sum() * total).astype(np.int64)
        c[-1] = total
        return np.concatenate([[0], c])

    return cut(nq), np.arange(groups + 1) * (n // groups) if even else cut(n)


def _grouped(S, t, out, groups, nq, n, dim, seed, even=False, alpha=1.0, with_bias=False):
    torch = _torch()
    qo, vo = _groups(seed, groups, nq, n, even)
    q, v = _data(nq, dim, seed + 1, 1.0), _data(n, dim, seed + 2, 1.0)
    bias = np.random.default_rng(seed).normal(size=n).astype(np.float32) if with_bias else None
    if t == "fp8":
        qd, rows = _gpu(q, "bf16"), S.Fp8Rows.encode(_gpu(v))
        qv, vv = U.fp8_values(_np(qd))[0], _np(rows.decode())
    else:
        qd, rows = S.aligned_rows(_gpu(q, t)), S.aligned_rows(_gpu(v, t))
        qv, vv = _np(qd), _np(rows)
    total = int(((qo[1:] - qo[:-1]) * (vo[1:] - vo[:-1])).sum())
    room = torch.full((total + 100,), 5.0, dtype=_dt(out), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = S.group_scores(qd, torch.from_numpy(qo).cuda(), rows, torch.from_numpy(vo).cuda(), total=total, out=room,
                         dtype=_dt(out), alpha=alpha, bias=None if bias is None else _gpu(bias), status=status)
    assert int(status) == 0
    assert bool((room[total:] == 5.0).all())
    at = 0
    for g in range(groups):
        m, c = int(qo[g + 1] - qo[g]), int(vo[g + 1] - vo[g])
        if m * c:
            _check(got[at:at + m * c].view(m, c), qv[qo[g]:qo[g + 1]], vv[vo[g]:vo[g + 1]], out, alpha,
                   None if bias is None else bias[vo[g]:vo[g + 1]].astype(np.float64))
        at += m * c
    assert at == total
    starts = S.group_rows(torch.from_numpy(qo).cuda(), torch.from_numpy(vo).cuda(), nq, n).cpu().numpy()
    width = np.zeros(nq, np.int64)
    for g in range(groups):
        width[qo[g]:qo[g + 1]] = vo[g + 1] - vo[g]
    np.testing.assert_array_equal(starts, np.concatenate([[0], np.cumsum(width)]))


@pytest.mark.parametrize("t,out", [("f16", "f32"), ("bf16", "bf16"), ("fp8", "f32"), ("fp8", "f16")])
@pytest.mark.parametrize("groups,nq,n,dim,even", [(1, 5, 7, 8, False), (3, 40, 700, 128, False),
                                                  (40, 300, 3000, 72, False), (70, 200, 7000, 520, True),
                                                  (300, 1000, 2000, 40, False), (5, 900, 1500, 136, False),
                                                  (2, 3, 4, 1000, False)])
def test_group_scores(S, t, out, groups, nq, n, dim, even):
    _grouped(S, t, out, groups, nq, n, dim, groups + nq, even)


def test_group_scores_alpha_bias(S):
    _grouped(S, "fp8", "f32", 9, 80, 900, 200, 3, alpha=-2.0, with_bias=True)
    _grouped(S, "bf16", "f32", 9, 80, 900, 200, 4, alpha=0.5, with_bias=True)


def test_group_scores_rows_outside_groups(S):
    """Offsets need not cover the rows: what lies outside has no scores, and an
    unreached NaN row spoils none."""
    torch = _torch()
    q, v = _gpu(_data(50, 64, 1, 1.0), "f16"), _gpu(_data(90, 64, 2, 1.0), "f16")
    q[:4], q[30:], v[:10], v[60:] = float("nan"), float("nan"), float("nan"), float("nan")
    qo, vo = torch.tensor([4, 4, 30], device="cuda"), torch.tensor([10, 20, 60], device="cuda")
    got = S.group_scores(q, qo, v, vo, total=26 * 40)
    _check(got.view(26, 40), _np(q)[4:30], _np(v)[20:60], "f32")
    starts = S.group_rows(qo, vo, 50, 90).cpu().numpy()
    np.testing.assert_array_equal(starts, [0] * 4 + list(range(0, 26 * 40, 40)) + [26 * 40] * 21)


def test_group_scores_bad_offsets_and_small_outputs(S):
    """Offsets that fall or leave the rows count as empty groups; scores past the
    output are not written; both set the status."""
    torch = _torch()
    q, v = _gpu(_data(20, 64, 1, 1.0), "bf16"), _gpu(_data(30, 64, 2, 1.0), "bf16")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for qo, vo in (([0, 10, 5], [0, 10, 20]), ([0, 10, 20], [0, 10, 31]), ([-1, 10, 20], [0, 0, 30]),
                   ([0, 10, 20], [0, 1 << 62, 30])):
        status.zero_()
        room = torch.full((700,), 5.0, device="cuda")
        S.group_scores(q, torch.tensor(qo, device="cuda"), v, torch.tensor(vo, device="cuda"), out=room, status=status)
        assert int(status) & 1
        status.zero_()
        S.group_rows(torch.tensor(qo, device="cuda"), torch.tensor(vo, device="cuda"), 20, 30, status=status)
        assert int(status) & 1
    status.zero_()
    room = torch.full((700,), 5.0, device="cuda")
    qo, vo = torch.tensor([0, 20], device="cuda"), torch.tensor([0, 30], device="cuda")
    S.group_scores(q, qo, v, vo, out=room[:100], status=status)  # three queries' scores fit
    assert int(status) == 2
    _check(room[:90].view(3, 30), _np(q)[:3], _np(v), "f32")
    assert bool((room[90:] == 5.0).all())


# ---- top-k --------------------------------------------------------------------------


def _top(S, rows, k, largest, t, ragged):
    torch = _torch()
    if ragged:
        flat = np.concatenate([np.asarray(r, np.float64) for r in rows]) if rows else np.zeros(0)
        x = _gpu(flat, t)
        starts = np.concatenate([[0], np.cumsum([len(r) for r in rows])]).astype(np.int64)
        vals, ids, counts = S.top_k(x, k, largest=largest, row_starts=torch.from_numpy(starts).cuda())
        held = _np(x)
        rows = [held[a:b] for a, b in zip(starts[:-1], starts[1:])]
    else:
        x = _gpu(np.asarray(rows), t)
        vals, ids, counts = S.top_k(x, k, largest=largest)
        rows = list(_np(x))
    wv, wi, wc = U.top_k(rows, k, largest)
    np.testing.assert_array_equal(counts.cpu().numpy(), wc)
    np.testing.assert_array_equal(_np(vals), wv)
    np.testing.assert_array_equal(ids.cpu().numpy(), wi)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("largest", [True, False])
@pytest.mark.parametrize("nq,n,k", [(1, 1, 1), (3, 5, 8), (9, 100, 10), (40, 1000, 33), (5, 1025, 256), (2, 5000, 1),
                                    (7, 9001, 100), (700, 3000, 10), (1, 300_001, 10), (2, 100_003, 256),
                                    (600, 5003, 256)])
def test_top_k(S, t, largest, nq, n, k):
    r = np.random.default_rng(nq + n + k)
    _top(S, r.normal(size=(nq, n)), k, largest, t, False)


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few", "special", "nan"])
@pytest.mark.parametrize("n,k", [(40, 50), (700, 20), (9000, 64), (40_000, 256)])
def test_top_k_hard_rows(S, kind, n, k):
    r = np.random.default_rng(n)
    x = {"equal": np.full((3, n), 2.5), "rising": np.tile(np.arange(n) / 1000.0, (3, 1)),
         "falling": np.tile(-np.arange(n) / 1000.0, (3, 1)), "few": r.integers(0, 3, (3, n)).astype(float),
         "special": r.choice([0.0, -0.0, np.inf, -np.inf, np.nan, 1.0, -1.0], (3, n)),
         "nan": np.full((3, n), np.nan)}[kind]
    for largest in (True, False):
        _top(S, x, k, largest, "f32", False)
        _top(S, x, k, largest, "bf16", False)


@pytest.mark.parametrize("t", TYPES)
def test_top_k_ragged(S, t):
    r = np.random.default_rng(4)
    for lens in ([0], [0, 3, 0, 1, 17], list(r.integers(0, 60, 300)), [50_000, 0, 1, 20_011], list(r.integers(0, 9000, 40))):
        _top(S, [r.normal(size=n) for n in lens], 16, True, t, True)
        _top(S, [r.integers(0, 9, n).astype(float) for n in lens], 100, False, t, True)


def test_top_k_pitch_and_bad_starts(S):
    torch = _torch()
    x = torch.randn(9, 3000, device="cuda")
    for part in (x[:, 1:2001], x[1::3, 7:1500], x[:, :1]):
        got = S.top_k(part, 5)
        want = U.top_k(list(_np(part)), 5, True)
        np.testing.assert_array_equal(got[1].cpu().numpy(), want[1])
    # starts that fall or leave the scores: those rows are cut to what is there
    flat = torch.arange(100.0, device="cuda")
    vals, ids, counts = S.top_k(flat, 3, row_starts=torch.tensor([-5, 10, 5, 90, 1 << 60], device="cuda"))
    assert counts.tolist() == [0, 0, 3, 3] and vals[2].tolist() == [89.0, 88.0, 87.0] and vals[3].tolist() == [99.0, 98.0, 97.0]


# ---- together ------------------------------------------------------------------------


def test_partitioned_search(S):
    """Queries go to their best partition by the centroids' scores, are scored
    against its rows, and keep the best ten: the run a program makes."""
    torch = _torch()
    parts, n, nq, dim, k = 30, 6000, 200, 128, 10
    x, q = _data(n, dim, 1, 0.5), _gpu(_data(nq, dim, 2, 0.5))
    vo = _groups(5, parts, 0, n)[1]
    cent = _gpu(np.stack([x[a:b].mean(0) if b > a else np.full(dim, -1e3) for a, b in zip(vo[:-1], vo[1:])]))
    rows = S.Fp8Rows.encode(_gpu(x))
    _, best, _ = S.top_k(S.scores(q, S.Fp8Rows.encode(cent)), 1)
    order = torch.argsort(best[:, 0].long(), stable=True)
    qo = torch.searchsorted(best[order, 0].long(), torch.arange(parts + 1, device="cuda"))
    vod = torch.from_numpy(vo).cuda()
    starts = S.group_rows(qo, vod, nq, n)
    packed = S.group_scores(q[order], qo, rows, vod, total=int(starts[-1]))
    vals, ids, counts = S.top_k(packed, k, row_starts=starts)
    # the same from the whole matrix of scores
    full = S.scores(q[order], rows)
    b = best[order, 0].long().tolist()
    for i in range(nq):
        lo, hi = int(vo[b[i]]), int(vo[b[i] + 1])
        assert bool((packed[int(starts[i]):int(starts[i + 1])] == full[i, lo:hi]).all())
    wv, wi, wc = U.top_k([_np(full[i, int(vo[b[i]]):int(vo[b[i] + 1])]) for i in range(nq)], k, True)
    np.testing.assert_array_equal(counts.cpu().numpy(), wc)
    np.testing.assert_array_equal(ids.cpu().numpy(), wi)
    np.testing.assert_array_equal(_np(vals), wv)


def test_nearest_by_scores_matches_exact_knn(S, small_case):
    """alpha = -2 with squared norms as bias, then the smallest ten, finds the
    exact kNN of the rows that the FP8 codes stand for."""
    torch = _torch()
    from raven_b200.index import DeviceIndex

    base, q, g = small_case
    rows = S.Fp8Rows.of_index(DeviceIndex(g, base, sq4=True))
    v = rows.decode().double()
    qv = S.Fp8Rows.encode(_gpu(q)).decode().double()
    sc = S.scores(_gpu(q), rows, alpha=-2.0, bias=(v ** 2).sum(1).float())
    vals, ids, _ = S.top_k(sc, 10, largest=False)
    d = torch.cdist(qv, v) ** 2 - (qv ** 2).sum(1, keepdim=True)
    want = torch.sort(d, dim=1).values[:, :10]
    # scores of at most 2^22 in f32: 128 additions and the bias are off by at most 130 * 2^-23 * 2^22
    assert float((vals.double() - want).abs().max()) <= 65.0 + 1e-3
    exact_at = d.gather(1, ids.long())
    assert float((vals.double() - exact_at).abs().max()) <= 65.0 + 1e-3


def test_streams_and_graphs(S):
    """Two streams at once, and two captured graphs replayed on new inputs, give
    what eager calls give."""
    torch = _torch()
    rows = S.Fp8Rows.encode(_gpu(_data(5000, 256, 1, 1.0)))
    qs = [_gpu(_data(300, 256, 10 + i, 1.0)) for i in range(4)]
    want = [S.top_k(S.scores(q, rows), 20) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for _ in range(5):
        got = []
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(S.top_k(S.scores(q, rows), 20))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(bool((x == y).all()) for x, y in zip(a, b))
    long = _gpu(np.random.default_rng(0).normal(size=(2, 200_000)))
    want_long = S.top_k(long, 50)
    graphs = []
    for q in qs[:2]:
        buf = torch.empty_like(q)
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            r = S.top_k(S.scores(buf, rows), 20)
            r_long = S.top_k(long, 50)
        graphs.append((graph, buf, r, r_long))
    for turn in range(3):
        for (graph, buf, _, _), s, i in zip(graphs, streams, (turn % 4, (turn + 1) % 4)):
            with torch.cuda.stream(s):
                buf.copy_(qs[i])
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, r, r_long), i in zip(graphs, (turn % 4, (turn + 1) % 4)):
            assert all(bool((x == y).all()) for x, y in zip(r, want[i]))
            assert all(bool((x == y).all()) for x, y in zip(r_long, want_long))


def test_same_results_every_time(S):
    torch = _torch()
    q, rows = _gpu(_data(90, 700, 1, 1.0)), S.Fp8Rows.encode(_gpu(_data(3000, 700, 2, 1.0)))
    a = [S.scores(q, rows) for _ in range(5)]
    x = torch.randint(0, 50, (300, 20_000), device="cuda").float()
    b = [S.top_k(x, 40) for _ in range(5)]
    for y in a[1:]:
        assert bool((y == a[0]).all())
    for y in b[1:]:
        assert all(bool((u == w).all()) for u, w in zip(y, b[0]))


def test_refusals(S):
    torch = _torch()
    f = lambda *s, t="f32": torch.zeros(*s, device="cuda", dtype=_dt(t))  # noqa: E731
    rows = S.Fp8Rows.encode(f(10, 64))
    off = torch.tensor([0, 5], device="cuda")
    for call in (
        lambda: S.scores(f(3, 32), rows),                                  # dim
        lambda: S.scores(f(3, 64), f(4, 64)),                              # float32 vectors
        lambda: S.scores(f(3, 64, t="f16"), f(4, 64, t="bf16")),           # two types
        lambda: S.scores(rows, f(4, 64, t="bf16")),                        # FP8 queries, 16-bit vectors
        lambda: S.scores(f(3, 60, t="f16"), f(4, 60, t="f16")),            # pitch of 120 bytes
        lambda: S.scores(f(3, 64, t="f16"), f(4, 72, t="f16")[:, 1:65]),   # not on 16 bytes
        lambda: S.scores(f(3, 64), rows, bias=f(9)),
        lambda: S.scores(f(3, 64), rows, out=f(3, 9)),
        lambda: S.scores(f(3, 64), rows, dtype=torch.float64),
        lambda: S.scores(f(3, 64).cpu(), rows),
        lambda: S.scores(f(3, 64), rows, status=torch.zeros(1, dtype=torch.int64, device="cuda")),
        lambda: S.scores(f(64, 3).T, rows),
        lambda: S.group_scores(f(3, 64), off, rows, off),                  # no size
        lambda: S.group_scores(f(3, 64), off.int(), rows, off, total=1),
        lambda: S.group_scores(f(3, 64), off, rows, torch.tensor([0, 1, 2], device="cuda"), total=1),
        lambda: S.group_scores(f(3, 64), off, rows, off, total=20, out=f(10)),
        lambda: S.Fp8Rows.encode(f(10, 64), out=rows.rows(0, 9)),
        lambda: S.Fp8Rows(rows.codes[:, :48], rows.exps, 64),
        lambda: rows.rows(5, 6),
        lambda: S.top_k(f(4, 4).T, 2),
        lambda: S.top_k(f(16), 2),
        lambda: S.top_k(f(4, 4).int(), 2),
    ):
        with pytest.raises(ValueError):
            call()
    from raven_b200 import RavenError

    for call in (lambda: S.top_k(f(4, 4), 0), lambda: S.top_k(f(4, 4), 257),
                 lambda: S.Fp8Rows.encode(f(2, 65537))):
        with pytest.raises(RavenError):
            call()


# ---- each layout and team, at the sizes where the choice between them changes ---------


def _check_on_gpu(got, q, v, t, alpha=1.0, bias=None):
    """_check with the 64-bit products on the GPU, for large outputs."""
    torch = _torch()
    for at in range(0, q.shape[0], 64):
        a = q[at:at + 64].double()
        exact = alpha * (a @ v.double().T) + (0.0 if bias is None else bias.double())
        mags = a.abs() @ v.double().abs().T
        off = abs(alpha) * (q.shape[1] + 1) * 2.0 ** -23 * mags + 2.0 ** -23 * exact.abs()
        if bias is not None:
            off = off + 2.0 ** -23 * bias.double().abs()
        lim = off + torch.finfo(_dt(t)).eps / 2 * (exact.abs() + off) + 1e-37
        assert bool(((got[at:at + 64].double() - exact).abs() <= lim).all())


LAYOUTS = [(300, 30_011, 40), (300, 30_016, 40), (130, 20_007, 300), (129, 33_001, 128), (65, 25_003, 17),
           (70, 400_003, 16), (70, 400_000, 16), (66, 800_001, 16), (40, 50_001, 900), (33, 150_001, 16),
           (32, 9_001, 128), (4, 20_001, 1024), (4, 20_001, 1025), (1, 300_001, 100), (2000, 1_503, 96), (1000, 209, 64)]


@pytest.mark.parametrize("nq,n,dim", LAYOUTS)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fp8", [True, False])
def test_scores_layouts(S, nq, n, dim, t, fp8):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(nq + n + dim)
    q = torch.randn(nq, dim, generator=g, device="cuda").half()
    v = torch.randn(n, dim, generator=g, device="cuda").half()
    bias = torch.randn(n, generator=g, device="cuda")
    if fp8:
        rows, qv = S.Fp8Rows.encode(v), S.Fp8Rows.encode(q).decode()
        vv = rows.decode()
    else:
        q, rows = S.aligned_rows(q), S.aligned_rows(v)
        qv, vv = q, rows
    # scores that start anywhere: a pitch and a start of their own, and the bytes around them untouched
    for room, left in ((n, 0), (n + 13, 5)):
        big = torch.full((nq, room), 9.0, dtype=_dt(t), device="cuda")
        out = big[:, left:left + n]
        with_bias = left > 0
        S.scores(q, rows, dtype=_dt(t), out=out, alpha=0.5 if with_bias else 1.0, bias=bias if with_bias else None)
        _check_on_gpu(out, qv, vv, t, 0.5 if with_bias else 1.0, bias if with_bias else None)
        assert bool((big[:, :left] == 9.0).all()) and bool((big[:, left + n:] == 9.0).all())


@pytest.mark.parametrize("t,out", [("fp8", "bf16"), ("fp8", "f32"), ("bf16", "f16"), ("f16", "f32")])
def test_group_scores_large_groups(S, t, out):
    """Groups of more than 64 queries on average: the layout by pairs, with packed
    scores that start anywhere."""
    _grouped(S, t, out, 4, 700, 1500, 136, 11)
    _grouped(S, t, out, 3, 400, 901, 72, 12, alpha=-1.5, with_bias=True)


def test_group_scores_capacity_by_pairs(S):
    torch = _torch()
    q, v = _gpu(_data(200, 64, 1, 1.0), "bf16"), _gpu(_data(301, 64, 2, 1.0), "bf16")
    qo, vo = torch.tensor([0, 200], device="cuda"), torch.tensor([0, 301], device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for fit in (0, 1, 57, 199):
        status.zero_()
        room = torch.full((200 * 301,), 5.0, device="cuda")
        S.group_scores(q, qo, v, vo, out=room[:fit * 301 + 100], status=status)
        assert int(status) == 2
        if fit:
            _check(room[:fit * 301].view(fit, 301), _np(q)[:fit], _np(v), "f32")
        assert bool((room[fit * 301 + 100:] == 5.0).all())


def test_fp8_bytes_past_the_values_do_not_matter(S):
    """Code bytes past dim and exponent bytes past the last block are not read as values."""
    torch = _torch()
    for nq, n, dim in ((3, 300, 200), (40, 300, 200), (200, 1000, 520)):
        rows, q = S.Fp8Rows.encode(_gpu(_data(n, dim, 1, 1.0))), S.Fp8Rows.encode(_gpu(_data(nq, dim, 2, 1.0)))
        want = S.scores(q, rows)
        for r in (rows, q):
            r.codes[:, dim:] = 0x7F  # NaN
            r.exps[:, -(-dim // 128):] = 255
        assert bool((S.scores(q, rows) == want).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nq,n,k", [(1300, 1500, 100), (1300, 1500, 40), (1300, 2100, 256), (2500, 1200, 20),
                                    (2500, 1100, 33), (1, 70_000, 200), (3, 4097, 129), (5000, 30, 30), (5000, 900, 200)])
def test_top_k_teams(S, t, nq, n, k):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(n + k)
    for x in (torch.randn(nq, n, generator=g, device="cuda"),
              torch.randint(0, 40, (nq, n), generator=g, device="cuda").float()):
        x[0], x[-1, : n // 2] = float("nan"), float("nan")
        x[nq // 2, ::3], x[nq // 2, 1::3] = float("inf"), float("-inf")
        x = x.to(_dt(t))
        for largest in (True, False):
            vals, ids, counts = S.top_k(x, k, largest=largest)
            # by a stable sort of the values with NaN behind the worst infinity
            key = torch.where(x.isnan(), torch.full_like(x, float("nan")), x).float()
            order = torch.sort(torch.where(key.isnan(), torch.full_like(key, float("inf")), -key if largest else key),
                               dim=1, stable=True)
            idx = order.indices
            # NaN after infinities of the same place: a second stable sort by whether it is NaN
            idx = idx.gather(1, torch.sort(key.gather(1, idx).isnan().to(torch.int8), dim=1, stable=True).indices)
            c = min(k, n)
            assert bool((counts == c).all())
            assert bool((ids[:, :c].long() == idx[:, :c]).all())
            want = x.gather(1, idx[:, :c])
            assert bool(((vals[:, :c] == want) | (vals[:, :c].isnan() & want.isnan())).all())
            assert bool((ids[:, c:] == 0).all()) and bool((vals[:, c:] == 0).all())


def test_group_scores_without_room_tell(S):
    torch = _torch()
    q, v = _gpu(_data(20, 64, 1, 1.0), "bf16"), _gpu(_data(30, 64, 2, 1.0), "bf16")
    qo, vo = torch.tensor([0, 20], device="cuda"), torch.tensor([0, 30], device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    S.group_scores(q, qo, v, vo, total=0, status=status)
    assert int(status) == 2
    status.zero_()
    S.group_scores(q, torch.zeros_like(qo), v, vo, total=0, status=status)  # no scores: nothing is missing
    assert int(status) == 0


def test_inputs_written_just_before(S):
    """Every operator on what the one before it has just written, in one stream
    without a wait, the buffers the same each time and their contents not."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = S.Fp8Rows.empty(3000, 200, "cuda")
    out, back = torch.empty(70, 3000, device="cuda"), torch.empty(70, 200, device="cuda")
    x, q = torch.empty(3000, 200, device="cuda"), torch.empty(70, 200, device="cuda")
    got, inputs = [], []
    for i in range(12):
        x.normal_(generator=g)
        q.normal_(generator=g)
        S.Fp8Rows.encode(x, out=rows)
        S.scores(q, rows, out=out)
        vals, ids, _ = S.top_k(out, 7)
        again = S.Fp8Rows.encode(out)  # scores as rows: reads what the product wrote
        got.append((vals, ids, S.scores(again, again), S.top_k(S.scores(q[:3], rows), 5)[1]))
        inputs.append((x.clone(), q.clone()))
    torch.cuda.synchronize()
    for (vals, ids, self_scores, few), (x, q) in zip(got, inputs):
        rows = S.Fp8Rows.encode(x)
        torch.cuda.synchronize()
        out = S.scores(q, rows)
        torch.cuda.synchronize()
        want = S.top_k(out, 7)
        again = S.Fp8Rows.encode(out)
        torch.cuda.synchronize()
        assert bool((vals == want[0]).all()) and bool((ids == want[1]).all())
        assert bool((self_scores == S.scores(again, again)).all())
        few_out = S.scores(q[:3], rows)
        torch.cuda.synchronize()
        assert bool((few == S.top_k(few_out, 5)[1]).all())


def test_first_call_inside_a_capture(raven_lib):
    """A process whose first calls of the library are captured."""
    import subprocess
    import sys

    code = """
import torch
from raven_b200 import scoring as S
x, q = torch.randn(5000, 96, device="cuda"), torch.randn(64, 96, device="cuda")
long = torch.randn(2, 100_000, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = S.top_k(S.scores(q, S.Fp8Rows.encode(x)), 9)
    got_long = S.top_k(long, 9)
for _ in range(3):
    x.normal_(); q.normal_(); long.normal_()
    graph.replay()
    want, want_long = S.top_k(S.scores(q, S.Fp8Rows.encode(x)), 9), S.top_k(long, 9)
    torch.cuda.synchronize()
    assert all(bool((a == b).all()) for a, b in zip(got, want)) and all(bool((a == b).all()) for a, b in zip(got_long, want_long))
print("captured")
"""
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_two_threads(S):
    """Calls from two threads, each on a stream of its own."""
    import threading

    torch = _torch()
    rows = S.Fp8Rows.encode(_gpu(_data(4000, 160, 1, 1.0)))
    qs = [_gpu(_data(100, 160, 20 + i, 1.0)) for i in range(2)]
    want = [S.top_k(S.scores(q, rows), 12) for q in qs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(40):
                got = S.top_k(S.scores(qs[i], rows), 12)
            torch.cuda.current_stream().synchronize()
            if not all(bool((a == b).all()) for a, b in zip(got, want[i])):
                bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


@pytest.mark.parametrize("t,groups,nq,n,even", [("bf16", 1600, 3000, 20000, False), ("fp8", 1900, 1000, 9000, False),
                                                ("f16", 2000, 2000, 20000, True)])
def test_group_scores_many_groups(S, t, groups, nq, n, even):
    _grouped(S, t, "f32", groups, nq, n, 72, 5, even, alpha=0.5, with_bias=True)


@pytest.mark.parametrize("groups,most_q,most_v,empty", [(1536, 9, 300, 0.3), (1537, 9, 300, 0.3), (5000, 300, 40, 0.2),
                                                        (150_000, 4, 20, 0.5), (150_000, 2, 9, 0.999), (40_000, 1, 3, 1.0)])
def test_many_groups_exactly(S, groups, most_q, most_v, empty):
    """Small integers, whose products and sums are exact: every score as it is."""
    torch = _torch()
    r = np.random.default_rng(groups + most_q)
    m, c = r.integers(0, most_q + 1, groups), r.integers(0, most_v + 1, groups)
    m[r.random(groups) < empty] = 0
    m[groups // 3: groups // 2] = 0  # chunks without a score
    c[r.random(groups) < 0.1] = 0
    qo, vo = np.concatenate([[0], np.cumsum(m)]), np.concatenate([[0], np.cumsum(c)])
    nq, n, total = int(qo[-1]) + 3, int(vo[-1]) + 5, int((m * c).sum())
    g = torch.Generator(device="cuda").manual_seed(groups)
    q = torch.randint(-3, 4, (nq, 40), device="cuda", generator=g).half()
    v = torch.randint(-3, 4, (n, 40), device="cuda", generator=g).half()
    tq, tv = torch.from_numpy(qo).cuda(), torch.from_numpy(vo).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    starts = S.group_rows(tq, tv, nq, n, status=status)
    room = torch.full((total + 64,), 5.0, device="cuda")
    S.group_scores(q, tq, v, tv, out=room, status=status)
    assert int(status) == 0
    want = np.concatenate([[0], np.cumsum(np.repeat(c, m)), [total] * 3])
    np.testing.assert_array_equal(starts.cpu().numpy(), want)
    at = torch.arange(total, device="cuda")
    query = torch.searchsorted(starts, at, right=True) - 1
    group = torch.searchsorted(tq, query, right=True) - 1
    row = tv[group] + at - starts[query]
    for a in range(0, total, 1 << 20):
        b = slice(a, min(total, a + (1 << 20)))
        assert bool((room[b] == (q[query[b]].float() * v[row[b]].float()).sum(1)).all())
    assert bool((room[total:] == 5.0).all())


def test_many_groups_bad_offsets(S):
    """A bad group among many sets the status, wherever it is, and has no scores."""
    torch = _torch()
    groups = 4000
    q, v = _gpu(_data(groups, 64, 1, 1.0), "bf16"), _gpu(_data(groups, 64, 2, 1.0), "bf16")
    o = np.arange(groups + 1)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for at, value in ((0, -1), (1700, groups + 1), (groups, groups + 1), (2500, 7)):
        bad = o.copy()
        bad[at] = value
        good, tb = torch.from_numpy(o).cuda(), torch.from_numpy(bad).cuda()
        ok = (bad[:-1] >= 0) & (bad[1:] >= bad[:-1]) & (bad[1:] <= groups)
        width = (bad[1:] - bad[:-1])[ok]
        status.zero_()
        room = torch.full((2 * groups,), 5.0, device="cuda")
        S.group_scores(q, good, v, tb, out=room, status=status)
        assert int(status) & 1
        status.zero_()
        starts = S.group_rows(good, tb, groups, groups, status=status)
        assert int(status) & 1 and int(starts[-1]) == int(width.sum())
        rows = np.concatenate([bad[g] + np.arange(bad[g + 1] - bad[g]) for g in np.flatnonzero(ok)])
        want = (_np(q)[np.repeat(np.flatnonzero(ok), width)] * _np(v)[rows]).sum(1)
        size = (np.abs(_np(q))[np.repeat(np.flatnonzero(ok), width)] * np.abs(_np(v)[rows])).sum(1)
        # 64 products, exact in f32, summed with at most one rounding or truncation each
        assert np.all(np.abs(_np(room[:len(want)]) - want) <= 64 * 2.0 ** -23 * size)
        assert bool((room[len(want):] == 5.0).all())


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("largest", [True, False])
@pytest.mark.parametrize("k", [10, 40, 100, 256])
def test_top_k_every_16_bit_value(S, t, largest, k):
    """Rows of all values of a type, infinities, NaN and both zeros among them,
    and rows of those nearest to zero, several of each."""
    torch = _torch()
    r = np.random.default_rng(k)
    every = torch.from_numpy(np.arange(65536).astype(np.uint16).view(np.int16)).view(_dt(t)).double().numpy()
    _top(S, np.stack([r.permutation(every) for _ in range(3)]), k, largest, t, False)
    small = np.concatenate([every[:40], every[0x8000:0x8000 + 40]])
    _top(S, np.stack([r.choice(small, 4000) for _ in range(1300)]), k, largest, t, False)


def test_many_groups_captured(S):
    """Offsets that change between replays of one captured run over many groups."""
    torch = _torch()
    groups, nq, n = 10_000, 12_000, 30_000
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randint(-3, 4, (nq, 64), device="cuda", generator=g).bfloat16()
    v = torch.randint(-3, 4, (n, 64), device="cuda", generator=g).bfloat16()

    def offsets(total):
        cuts = torch.randint(0, total + 1, (groups - 1,), device="cuda", generator=g).sort().values
        return torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), total)])

    qo, vo = offsets(nq), offsets(n)
    out = torch.empty(400_000, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        S.group_scores(q, qo, v, vo, out=out, status=status)
        starts = S.group_rows(qo, vo, nq, n)
    for _ in range(3):
        qo.copy_(offsets(nq))
        vo.copy_(offsets(n))
        graph.replay()
        want = S.group_rows(qo, vo, nq, n)
        total = int(want[-1])
        assert total <= out.numel() and int(status) == 0
        assert bool((starts == want).all())
        at = torch.arange(total, device="cuda")
        query = torch.searchsorted(want, at, right=True) - 1
        row = vo[torch.searchsorted(qo, query, right=True) - 1] + at - want[query]
        assert bool((out[:total] == (q[query].float() * v[row].float()).sum(1)).all())


# ---- rows beside malformed groups -----------------------------------------------------


def _poisoned_starts(S, qo, vo, nq, n):
    """The row starts written over memory that holds something else, and the status."""
    torch = _torch()
    from raven_b200 import _lib as L

    out = torch.full((nq + 1,), -12345, dtype=torch.int64, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    tq, tv = torch.from_numpy(np.asarray(qo, np.int64)).cuda(), torch.from_numpy(np.asarray(vo, np.int64)).cuda()
    L.check(L.load().raven_group_rows_device(tq.data_ptr(), tv.data_ptr(), len(qo) - 1, nq, n, out.data_ptr(),
                                             status.data_ptr(), torch.cuda.current_stream().cuda_stream))
    return out, int(status)


@pytest.mark.parametrize("qo,vo", [([0, 10, 20], [0, 30, 20]), ([0, 10, 25], [0, 10, 20]), ([-5, 4, 20], [0, 10, 20]),
                                   ([0, 5, 5, 12, 20], [0, 31, 8, 8, 30]), ([0, 7, 20], [-1, 4, 1 << 62]),
                                   ([21, 30, 40], [0, 4, 5]), ([-9, -3, -1], [0, 4, 5]),
                                   ([3, 9, 14], [4, 2, 9]), ([-(1 << 60), 20, 1 << 62], [0, 30, 30]),
                                   ([0, 1 << 62, (1 << 62) + 20], [0, 10, 30]),
                                   ([-(1 << 63), -(1 << 63) + 20, (1 << 63) - 1], [0, 10, 30])])
def test_group_rows_beside_malformed_groups(S, qo, vo):
    """Every start is written, and the queries of sound groups have the rows of theirs."""
    torch = _torch()
    starts, status = _poisoned_starts(S, qo, vo, 20, 30)
    np.testing.assert_array_equal(starts.cpu().numpy(), U.group_starts(qo, vo, 20, 30))
    assert status == int(any(a > b or a < 0 or b > lim for o, lim in ((qo, 20), (vo, 30)) for a, b in zip(o[:-1], o[1:])))
    # the neighbours' best scores are those of their own group's vectors
    q, v = _gpu(_data(20, 64, 1, 1.0), "bf16"), _gpu(_data(30, 64, 2, 1.0), "bf16")
    packed = S.group_scores(q, torch.tensor(qo, device="cuda"), v, torch.tensor(vo, device="cuda"), total=int(starts[-1]))
    vals, ids, counts = S.top_k(packed, 4, row_starts=starts)
    full = S.scores(q, v)
    for g in range(len(qo) - 1):
        sound = 0 <= qo[g] <= qo[g + 1] <= 20 and 0 <= vo[g] <= vo[g + 1] <= 30
        for i in range(max(qo[g], 0), min(qo[g + 1], 20)):
            part = _np(full[i, vo[g]:vo[g + 1]]) if sound else np.zeros(0)
            wv, wi, wc = U.top_k([part], 4, True)
            assert int(counts[i]) == wc[0]
            np.testing.assert_array_equal(ids[i].cpu().numpy(), wi[0])
            np.testing.assert_array_equal(_np(vals[i]), wv[0])


@pytest.mark.parametrize("groups", [700, 8192, 9000, 20_000])
def test_group_rows_beside_malformed_groups_among_many(S, groups):
    r = np.random.default_rng(groups)
    for _ in range(3):
        qo = np.concatenate([[0], np.cumsum(r.integers(0, 5, groups))])
        vo = np.concatenate([[0], np.cumsum(r.integers(0, 40, groups))])
        nq, n = int(qo[-1]) - 3, int(vo[-1]) - 30  # the last groups leave the rows
        vo[r.integers(1, groups, 20)] = r.integers(-5, n + 5, 20)
        starts, status = _poisoned_starts(S, qo, vo, nq, n)
        assert status == 1
        np.testing.assert_array_equal(starts.cpu().numpy(), U.group_starts(qo, vo, nq, n))


@pytest.mark.parametrize("groups", [3, 40, 900, 9000, 20_000])
def test_group_rows_where_query_offsets_fall(S, groups):
    """Several groups cover a query: its place is in one of them, the same every
    time, starts rise, and none is left as it was."""
    r = np.random.default_rng(groups)
    nq, n = 500, 50
    for turn in range(6):
        qo = r.integers(-20, nq + 20, groups + 1)
        qo[: groups // 2] = np.sort(qo[: groups // 2])
        vo = np.sort(r.integers(0, n + 1, groups + 1))
        starts, status = _poisoned_starts(S, qo, vo, nq, n)
        got = starts.cpu().numpy()
        for _ in range(3):
            np.testing.assert_array_equal(_poisoned_starts(S, qo, vo, nq, n)[0].cpu().numpy(), got)
        assert status == int(np.any(qo[1:] < qo[:-1]) or qo.min() < 0 or qo.max() > nq)
        assert got[0] >= 0 and np.all(np.diff(got) >= 0)
        sound = (qo[:-1] >= 0) & (qo[1:] >= qo[:-1]) & (qo[1:] <= nq)
        size = np.where(sound, (qo[1:] - qo[:-1]) * (vo[1:] - vo[:-1]), 0)
        base = np.concatenate([[0], np.cumsum(size)])
        assert got[nq] == base[-1]
        for i in range(nq):
            may = {0} if i < qo[0] else set()
            may |= {int(base[-1])} if i >= qo[-1] else set()
            for g in np.flatnonzero((qo[:-1] <= i) & (i < qo[1:])):
                may.add(int(base[g] + ((i - qo[g]) * (vo[g + 1] - vo[g]) if sound[g] else 0)))
            assert int(got[i]) in may


@pytest.mark.parametrize("capacity", [35, (1 << 63) - 1, 1 << 63, (1 << 64) - 1])
def test_group_scores_any_capacity(S, capacity):
    """A caller who knows that the output is large enough may give any capacity."""
    torch = _torch()
    from raven_b200 import _lib as L

    q, v = _gpu(_data(5, 64, 1, 1.0), "f16"), _gpu(_data(7, 64, 2, 1.0), "f16")
    qo, vo = torch.tensor([0, 5], device="cuda"), torch.tensor([0, 7], device="cuda")
    out, status = torch.full((36,), 9.0, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    rows = [L.Rows(x.data_ptr(), None, len(x), 64, 0, L.RAVEN_TYPE_F16) for x in (q, v)]
    L.check(L.load().raven_group_scores_device(rows[0], qo.data_ptr(), rows[1], vo.data_ptr(), 1, 64, 1.0, None,
                                               out.data_ptr(), L.RAVEN_TYPE_F32, capacity, status.data_ptr(),
                                               torch.cuda.current_stream().cuda_stream))
    assert int(status) == 0 and float(out[35]) == 9.0
    assert bool((out[:35].view(5, 7) == S.scores(q, v)).all())


@pytest.mark.parametrize("groups", [1501, 3001])
def test_group_scores_end_at_the_capacity(S, groups):
    """Offsets that fall again and again, so that hundreds of groups cover all
    rows: the work is that of the groups that reach into the output, not of all."""
    torch = _torch()
    nq = n = 60_000
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randint(-3, 4, (nq, 64), device="cuda", generator=g).half()
    v = torch.randint(-3, 4, (n, 64), device="cuda", generator=g).half()
    fit = 9 * n + 50
    out = torch.full((fit + 100,), 5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(offsets, want_status):
        o = torch.tensor(offsets, device="cuda")
        for timed in (False, True):
            out.fill_(5.0)
            status.zero_()
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            S.group_scores(q, o, v, o, out=out[:fit], status=status)
            b.record()
            b.synchronize()
        assert int(status) == want_status
        assert bool((out[:9 * n].view(9, n) == q[:9].float() @ v.float().T).all()) and bool((out[fit:] == 5.0).all())
        return a.elapsed_time(b)

    one = run([0, nq], 2)
    many = run([0, nq] * ((groups + 1) // 2), 3)
    assert many <= 50 * one + 5.0, (one, many)  # (groups + 1) / 2 times one if all were computed
    # a bad group far behind the output's end is still told of
    assert run([0, nq] + [nq] * (groups - 2) + [nq + 1], 3) <= 50 * one + 5.0


def test_status_of_calls_without_one(S):
    """What goes wrong in calls without a status is kept until it is taken."""
    torch = _torch()
    q, v = _gpu(_data(20, 64, 1, 1.0), "bf16"), _gpu(_data(30, 64, 2, 1.0), "bf16")
    o = lambda *x: torch.tensor(x, device="cuda")  # noqa: E731
    S.take_status()
    S.scores(q, v)
    S.group_scores(q, o(0, 20), v, o(0, 30), total=600)
    S.group_rows(o(0, 20), o(0, 30), 20, 30)
    assert S.take_status() == 0
    S.group_scores(q, o(0, 20), v, o(0, 30), total=599)
    S.group_scores(q, o(0, 20), v, o(0, 30), total=600)  # does not clear it
    assert S.take_status("cuda:0") == 2 and S.take_status() == 0
    S.group_scores(q, o(0, 20), v, o(0, 30), total=0)  # asks for nothing
    assert S.take_status() == 0
    S.group_scores(q, o(0, 10, 5), v, o(0, 10, 20), total=600)
    assert S.take_status() == 1
    S.group_rows(o(0, 20), o(0, 31), 20, 30)
    assert S.take_status() == 1
    falls = torch.arange(3002, device="cuda").flip(0)  # many groups
    S.group_scores(q, falls, v, falls, total=600)
    assert S.take_status() == 1
    # a call with a status of its own says nothing here
    own = torch.zeros(1, dtype=torch.int32, device="cuda")
    S.group_scores(q, o(0, 20), v, o(0, 31), total=600, status=own)
    assert int(own) == 1 and S.take_status() == 0
    # in a captured run
    qo, vo = o(0, 20), o(0, 30)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        S.group_scores(q, qo, v, vo, total=600)
    graph.replay()
    assert S.take_status() == 0
    vo[1] = 31
    graph.replay()
    assert S.take_status() == 1
    with pytest.raises(ValueError):
        S.take_status("cpu")


@pytest.mark.parametrize("nq", [2, 40, 200])
def test_fp8_every_scale(S, nq):
    """The least, the largest and the NaN exponent byte mean the same to the
    products and to decode, block by block."""
    torch = _torch()
    q, v = S.Fp8Rows.empty(nq, 256, "cuda"), S.Fp8Rows.empty(300, 256, "cuda")
    q.codes.fill_(0x38)  # 1
    v.codes.fill_(0x38)
    q.exps.fill_(127)
    v.exps.fill_(127)
    for a, b in ((254, 0), (0, 254), (254, 1), (0, 127), (127, 0), (120, 134), (255, 0), (0, 255), (127, 255)):
        q.exps[:, 0], v.exps[:, 0] = 127, 127
        q.exps[1, 0], v.exps[131, 0] = a, b
        assert bool((q.decode()[1, :128] == 2.0 ** (a - 127)).all()) != (a == 255)
        assert bool(v.decode()[131, :128].isnan().all()) == (b == 255)
        want = q.decode().double() @ v.decode().double().T  # what is far below the largest vanishes
        got = S.scores(q, v)
        assert bool(((got.double() == want.float().double()) | (got.isnan() & want.isnan())).all()), (a, b)


def test_fp8_rows_keep_no_old_memory(S):
    """Rows follow their tensors, which cannot be exchanged for others."""
    torch = _torch()
    a, b = S.Fp8Rows.encode(_gpu(_data(50, 200, 1, 1.0))), S.Fp8Rows.encode(_gpu(_data(80, 200, 2, 1.0)))
    q = _gpu(_data(9, 200, 3, 1.0))
    want = S.scores(q, b)
    for name, value in (("codes", b.codes), ("exps", b.exps), ("dim", 100)):
        with pytest.raises(AttributeError):
            setattr(a, name, value)
    a.codes.set_(b.codes.clone())
    with pytest.raises(ValueError):  # 80 rows of codes, 50 of exponents
        S.scores(q, a)
    a.exps.set_(b.exps.clone())
    assert len(a) == 80 and bool((S.scores(q, a) == want).all()) and bool((a.decode() == b.decode()).all())
    assert bool((S.scores(a.rows(3, 5), a) == S.scores(b.rows(3, 5), b)).all())
    x = _gpu(_data(80, 200, 4, 1.0))
    S.Fp8Rows.encode(x, out=a)
    assert bool((a.decode() == S.Fp8Rows.encode(x).decode()).all()) and bool((S.scores(q, b) == want).all())


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_one_row_has_no_pitch(S, t):
    """A single row may come with any strides: nothing is a pitch away from it."""
    torch = _torch()
    x, q = _gpu(_data(3, 100, 1, 1.0), t), _gpu(_data(4, 100, 2, 1.0), t)
    want = S.scores(q, S.aligned_rows(x))
    for row in (x[:1], x[0].as_strided((1, 100), (1 << 45, 1)), x[0].as_strided((1, 100), (3, 1))):
        assert bool((S.scores(q, row) == want[:, :1]).all())
        assert bool((S.scores(row, S.aligned_rows(q))[0] == S.scores(x, S.aligned_rows(q))[0]).all())
        assert bool((S.Fp8Rows.encode(row).decode() == S.Fp8Rows.encode(x).decode()[:1]).all())
    rows = S.Fp8Rows.encode(x)
    codes, exps = rows.codes[:1, :112].as_strided((1, 112), (1 << 45, 1)), rows.exps[:1].as_strided((1, 4), (5, 1))
    one = S.Fp8Rows(codes, exps, 100)
    assert bool((S.scores(q, one) == S.scores(q, rows)[:, :1]).all()) and bool((one.decode() == rows.decode()[:1]).all())
    out = torch.empty(700, device="cuda").as_strided((1, 4), (1 << 45, 1))
    assert bool((S.scores(x[:1], S.aligned_rows(q), out=out) == S.scores(x, S.aligned_rows(q))[:1]).all())
    vals, ids, _ = S.top_k(torch.arange(9.0, device="cuda").as_strided((1, 9), (1 << 45, 1)), 2)
    assert ids.tolist() == [[8, 7]] and vals.tolist() == [[8.0, 7.0]]


def test_sizes_past_32_bits_are_refused(S):
    """Sizes that the library takes as 32 bits are not cut to their low ones."""
    torch = _torch()
    from raven_b200 import RavenError

    x = torch.randn(2, 9, device="cuda")
    off = torch.tensor([0, 2], device="cuda")
    for k in ((1 << 32) + 3, (1 << 64) + 3, 3 - (1 << 32), -1, 257, 1 << 31):
        with pytest.raises(RavenError):
            S.top_k(x, k)
        with pytest.raises(RavenError):
            S.top_k(x[:0], k)
    for n in ((1 << 32) + 2, (1 << 64) + 2):
        with pytest.raises(RavenError):
            S.group_rows(off, off, 2, n)
    # a row of 2^32 + 16 codes, which are never read
    codes = torch.empty((1, (1 << 32) + 16), dtype=torch.uint8, device="cuda")
    rows = S.Fp8Rows(codes, torch.empty((1, (1 << 25) + 4), dtype=torch.uint8, device="cuda"), (1 << 32) + 16)
    with pytest.raises(RavenError):
        S.scores(rows, rows)
    with pytest.raises(RavenError):
        S.group_scores(rows, off, rows, off, total=4)
    wide = codes[:, : (1 << 32) + 16].view(torch.float16)  # 2^31 + 8 values
    with pytest.raises(RavenError):
        S.Fp8Rows.encode(wide)


@pytest.mark.parametrize("nq,n,rows", [(100, 10_001, 80), (100, 10_000, 80), (128, 7_008, 96), (70, 32_001, 208), (300, 3_001, 80)])
def test_scores_take_a_cta_per_tile(S, nq, n, rows):
    """Up to the number of SMs there are as many CTAs as tiles of 128 queries and
    `rows` rows; where scores start between sectors a tile keeps 16 rows less."""
    torch = _torch()
    driver = pytest.importorskip("cuda.bindings.driver")
    q, v = _gpu(_data(nq, 64, 1, 1.0), "f16"), _gpu(_data(n, 64, 2, 1.0), "f16")
    t = torch.float32 if rows in (80, 208) else torch.bfloat16  # 16-bit scores that start on sectors: whole tiles
    room = torch.empty(nq, -(-n // 16) * 16 + (1 if rows in (80, 208) else 0), dtype=t, device="cuda")
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        S.scores(q, v, dtype=t, out=room[:, :n])
    _, _, count = driver.cuGraphGetNodes(driver.CUgraph(graph.raw_cuda_graph()), 0)
    _, nodes, _ = driver.cuGraphGetNodes(driver.CUgraph(graph.raw_cuda_graph()), count)
    grids = [driver.cuGraphKernelNodeGetParams(x)[1].gridDimX for x in nodes[:count]]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert grids == [min(sms, -(-n // rows) * -(-nq // 128))]
    graph.replay()
    _check(room[:, :n], _np(q), _np(v), "f32" if t == torch.float32 else "bf16")


# ---- long rows, exactly ----------------------------------------------------------------


@pytest.mark.parametrize("dim", [1000, 4095, 8192, 8200, 65_535, 65_536])
@pytest.mark.parametrize("nq,n", [(1, 300), (2, 500), (40, 300), (70, 300), (130, 1000)])
@pytest.mark.parametrize("t", ["f16", "bf16", "fp8", "fp8 from f32"])
def test_scores_of_long_rows_exactly(S, nq, n, dim, t):
    """Whole numbers of at most 3 in magnitude, with a scale of its own for each
    block: products and sums (of at most 9 * 65536 * 4 < 2^24 in units of the
    least product) are exact in f32 and the codes are exact, so a value that is
    dropped, doubled or given another block's scale shows in every score."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(dim + nq)
    blocks = -(-dim // 128)

    def make(rows):
        x = torch.randint(1, 4, (rows, dim), device="cuda", generator=g).float()
        x *= torch.randint(0, 2, (rows, dim), device="cuda", generator=g) * 2 - 1
        scale = torch.randint(0, 2, (rows, blocks), device="cuda", generator=g).float().exp2()
        return x * scale.repeat_interleave(128, 1)[:, :dim]

    q, v = make(nq), make(n)
    if t.startswith("fp8"):
        rows, ops = S.Fp8Rows.encode(v), (q if t != "fp8" else S.Fp8Rows.encode(q))
        assert bool((rows.decode() == v).all())
    else:
        rows, ops = S.aligned_rows(v.to(_dt(t))), S.aligned_rows(q.to(_dt(t)))
    want = q.double() @ v.double().T
    assert bool((S.scores(ops, rows).double() == want).all())
    room = torch.empty(nq, n + 3, device="cuda")  # scores between sectors
    assert bool((S.scores(ops, rows, out=room[:, 1:n + 1]).double() == want).all())
    # the same in two groups
    a, b = nq // 2, n // 3
    qo, vo = torch.tensor([0, a, nq], device="cuda"), torch.tensor([0, b, n], device="cuda")
    got = S.group_scores(ops, qo, rows, vo, total=a * b + (nq - a) * (n - b))
    assert bool((got[:a * b].view(a, b).double() == want[:a, :b]).all())
    assert bool((got[a * b:].view(nq - a, n - b).double() == want[a:, b:]).all())


@pytest.mark.parametrize("dim", [7, 16, 100, 130, 256])
def test_fp8_of_index_of_any_dimension(S, raven_lib, dim):
    """The index holds its vectors in an order of its own; their FP8 rows are in the caller's."""
    from raven_b200.index import DeviceIndex, Graph

    base = _data(300, dim, dim, 2.0).astype(np.float32)
    g = Graph.build(base, r=16, l=32, alpha=1.2, seed=1)
    rows = S.Fp8Rows.of_index(DeviceIndex(g, base))
    want = S.Fp8Rows.encode(_gpu(base))
    assert len(rows) == 300 and rows.dim == dim
    assert bool((rows.codes == want.codes).all()) and bool((rows.exps == want.exps).all())


def test_fp8_decode_every_code_and_scale(S):
    """All 256 codes under all 256 exponent bytes, rounded to f32 where a value is
    below its normal range."""
    torch = _torch()
    rows = S.Fp8Rows.empty(256, 256, "cuda")
    rows.codes.copy_(torch.arange(256, device="cuda").to(torch.uint8).expand(256, 256))
    rows.exps.copy_(torch.arange(256, device="cuda").to(torch.uint8)[:, None].expand(256, 4))
    c = np.arange(256)
    mag = np.where((c & 127) >> 3 == 0, (c & 7) * 2.0 ** -9, (8 + (c & 7)) * 2.0 ** (((c & 127) >> 3) - 10.0))
    value = np.where((c & 127) == 127, np.nan, np.where(c > 127, -mag, mag))
    scale = np.where(c == 255, np.nan, 2.0 ** (c - 127.0))
    with np.errstate(over="ignore"):
        want = (scale[:, None] * value[None, :]).astype(np.float32)
    got = rows.decode().cpu().numpy()
    np.testing.assert_array_equal(got, want)
    assert np.array_equal(np.signbit(got[:255, :127]), np.signbit(want[:255, :127]))


@pytest.mark.parametrize("groups", [2, 60, 9000, 20_000])
def test_group_rows_of_wild_offsets(S, groups):
    """Offsets near the ends of 64 bits, in any order: every start is written, none beside them."""
    r = np.random.default_rng(groups)
    nq, n = 300, 50
    ends = np.array([-(1 << 63), -(1 << 63) + 1, -(1 << 62), -1, 0, 7, 299, 300, 301, (1 << 31) + 5, (1 << 32) + 9, 1 << 62,
                     (1 << 63) - 2, (1 << 63) - 1], np.int64)
    for turn in range(8):
        qo, vo = r.choice(ends, groups + 1), r.choice(ends, groups + 1)
        if turn % 2:
            qo.sort()
        if turn < 4:
            vo = np.sort(r.integers(0, n + 1, groups + 1))
        starts, _ = _poisoned_starts(S, qo, vo, nq, n)
        got = starts.cpu().numpy()
        assert got[0] >= 0 and np.all(np.diff(got) >= 0)
        if turn % 2:
            np.testing.assert_array_equal(got, U.group_starts(qo, vo, nq, n))


@pytest.mark.parametrize("groups", [2, 60, 1536, 9000])
def test_group_scores_of_wild_offsets(S, groups):
    """Sound groups among offsets near the ends of 64 bits have their scores, and
    nothing is written past the output."""
    torch = _torch()
    r = np.random.default_rng(groups)
    g = torch.Generator(device="cuda").manual_seed(groups)
    q = torch.randint(-3, 4, (300, 64), device="cuda", generator=g).half()
    v = torch.randint(-3, 4, (50, 64), device="cuda", generator=g).half()
    full = (q.float() @ v.float().T).cpu().numpy()
    ends = np.array([-(1 << 63), -1, 0, 7, 9, 20, 50, 299, 300, 301, (1 << 31) + 5, 1 << 62, (1 << 63) - 1], np.int64)
    cap = 40_000
    for turn in range(4):
        qo, vo = r.choice(ends, groups + 1), r.choice(ends, groups + 1)
        want = []
        for i in range(groups):
            a, b, c, d = (int(x) for x in (qo[i], qo[i + 1], vo[i], vo[i + 1]))
            if 0 <= a <= b <= 300 and 0 <= c <= d <= 50:
                want.append(full[a:b, c:d].ravel())
        want = np.concatenate(want) if want else np.zeros(0, np.float32)
        room = torch.full((cap + 100,), 5.0, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        S.group_scores(q, torch.from_numpy(qo).cuda(), v, torch.from_numpy(vo).cuda(), out=room[:cap], status=status)
        got = room.cpu().numpy()
        assert np.all(got[cap:] == 5.0)
        assert int(status) == (1 if groups > 2 or np.any(qo[1:] < qo[:-1]) or np.any(vo[1:] < vo[:-1]) or
                               qo.min() < 0 or qo.max() > 300 or vo.min() < 0 or vo.max() > 50 else 0) + 2 * (len(want) > cap)
        if len(want) <= cap:
            np.testing.assert_array_equal(got[:len(want)], want)
            assert np.all(got[len(want):] == 5.0)
        else:
            np.testing.assert_array_equal(got[:cap - 50], want[:cap - 50])  # all but a query that does not fit
