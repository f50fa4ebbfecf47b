"""What an output of scores, or of adjusted ones, may share memory with, decided before any device work (no GPU
needed)."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def adjust(raven_lib):
    from raven_b200 import _lib as L

    def call(x=1 << 30, type=0, nq=4, n=100, ld=100, out=1 << 20, ld_out=100, status=None, **k):
        """Whether the call is refused for what overlaps (without a GPU the others fail later, for that)."""
        by = L.Adjustments(**k)
        by.repetition_all = 1.0
        rc = raven_lib.raven_adjust_scores_device(x, type, nq, n, ld, by, 1, out, ld_out, status, None)
        refused = rc == L.RAVEN_EINVAL and b"overlaps" in raven_lib.raven_last_error()
        assert refused or rc == L.RAVEN_ECUDA, (rc, raven_lib.raven_last_error())
        return refused

    import torch

    if torch.cuda.is_available():
        pytest.skip("made-up addresses: calls that are not refused must not run")
    return call


def test_output_over_what_scores_are_adjusted_by(adjust):
    out, end = 1 << 20, (1 << 20) + 1600  # 4 x 100 f32
    bias = dict(ld_bias=100)
    assert adjust(bias=out, **bias) and adjust(bias=out + 1596, **bias) and adjust(bias=out - 1596, **bias)
    assert not adjust(bias=end, **bias) and not adjust(bias=out - 1600, **bias)
    assert adjust(bias=out + 16) and adjust(bias=out - 396) and not adjust(bias=out - 400)  # one row for all
    assert adjust(bias=out, type=1, **bias)  # bytes, not values
    assert adjust(allow=out + 4, allow_count=1, ld_allow=4)
    assert adjust(allow=out - 48 - 12, allow_count=4, ld_allow=4) and not adjust(allow=out - 64, allow_count=4, ld_allow=4)
    filters = dict(allow=1 << 25, allow_count=4, ld_allow=4)
    assert adjust(allow_rows=out + 8, **filters) and not adjust(allow_rows=end, **filters)
    seen = dict(seen=1 << 25, seen_starts=1 << 26, seen_total=50)
    assert adjust(**dict(seen, seen=out - 196)) and not adjust(**dict(seen, seen=out - 200))
    assert adjust(**dict(seen, seen_starts=out - 32)) and not adjust(**dict(seen, seen_starts=out - 40))
    for name in ("repetition", "presence", "frequency"):
        assert adjust(**{name: out - 12}) and not adjust(**{name: out - 16}) and not adjust(**{name: end})
    assert adjust(status=out) and not adjust(status=end)


def _shares(a, rows_a, b, rows_b, pitch, wide_a, wide_b):
    """By every byte."""
    at = lambda p, rows, wide: (p + pitch * np.arange(rows)[:, None] + np.arange(wide)).ravel()  # noqa: E731
    return np.intersect1d(at(a, rows_a, wide_a), at(b, rows_b, wide_b)).size > 0


def test_rows_beside_one_another_by_every_byte(adjust):
    """Biases of the output's pitch, and single rows, wherever they start."""
    r = np.random.default_rng(0)
    out = 1 << 20
    seen = [0, 0]
    for _ in range(3000):
        nq, n = int(r.integers(1, 5)), int(r.integers(1, 7))
        ld = n if nq == 1 else n + int(r.integers(0, 9))
        shift = 4 * int(r.integers(-5 * ld - 2, 5 * ld + 2))
        one = nq > 1 and bool(r.integers(0, 2))
        want = _shares(out, nq, out + shift, 1 if one else nq, 4 * ld, 4 * n, 4 * n)
        assert adjust(nq=nq, n=n, ld=ld, ld_out=ld, bias=out + shift, ld_bias=0 if one or nq == 1 else ld) == want
        seen[want] += 1
    assert min(seen) > 500


def test_output_beside_its_scores_by_every_byte(adjust):
    """Columns of one matrix may be scores and output; where pitches differ the whole of both is apart."""
    r = np.random.default_rng(1)
    out, seen = 1 << 20, [0, 0]
    for _ in range(4000):
        nq, n, size = int(r.integers(1, 5)), int(r.integers(1, 7)), (4, 2)[int(r.integers(0, 2))]
        ld = n if nq == 1 else n + int(r.integers(0, 9))
        shift = size * int(r.integers(-5 * ld - 2, 5 * ld + 2))
        want = shift != 0 and _shares(out, nq, out + shift, nq, size * ld, size * n, size * n)
        assert adjust(x=out + shift, type=int(size == 2), nq=nq, n=n, ld=ld, ld_out=ld) == want
        seen[want] += 1
    assert min(seen) > 500
    assert adjust(x=out + 400, ld=201, ld_out=200) and not adjust(x=out + 400, ld=200, ld_out=200)
    assert adjust(ld=1 << 40, nq=(1 << 31) - 1, x=4096, out=1 << 60, ld_out=100)  # sizes past 64 bits


def test_scores_over_what_they_are_made_of(adjust, raven_lib):
    from raven_b200 import _lib as L

    def refused(out, q=1 << 30, bias=None, codes=1 << 28, words=1 << 29, nq=4, n=8, dim=128, ld_q=128, ld=8, type=0, out_type=0):
        rc = raven_lib.raven_scores_device(L.Rows(q, None, nq, ld_q, 0, type), L.Rows(codes, words, n, 64, 2, 5), dim, 1.0, bias,
                                           out, out_type, ld, None, None)
        no = rc == L.RAVEN_EINVAL and b"overlaps" in raven_lib.raven_last_error()
        assert no or rc == L.RAVEN_ECUDA, (rc, raven_lib.raven_last_error())
        return no

    at = 1 << 20
    assert refused(at, q=at) and refused(at, q=at + 124) and not refused(at, q=at + 128)
    assert not refused(at, q=at - 2048) and refused(at, q=at - 2044)
    assert refused(at, q=at, n=128, ld=128) and refused(at, q=at + 128, n=32, ld=128)
    assert not refused(at + 512, q=at, n=8, ld=136, ld_q=136) and refused(at + 508, q=at, n=8, ld=136, ld_q=136)  # columns
    assert refused(at, bias=at + 4) and not refused(at, bias=at - 32)
    assert refused(at, codes=at + 64) and not refused(at, codes=at + 128) and refused(at, codes=at - 448 - 48)
    assert refused(at, words=at + 120) and not refused(at, words=at + 128) and not refused(at, words=at - 64)
    assert refused(at + 62, out_type=1, bias=at + 124) and not refused(at + 62, out_type=1, bias=at + 128)
    assert not refused(at, nq=1, q=at + 32, ld=1 << 40)  # one row, at any pitch


def test_rows_over_what_they_are_made_of(adjust, raven_lib):
    from raven_b200 import _lib as L

    def said(rc):
        no = rc == L.RAVEN_EINVAL and b"overlaps" in raven_lib.raven_last_error()
        assert no or rc == L.RAVEN_ECUDA, (rc, raven_lib.raven_last_error())
        return no

    at, far = 1 << 20, 1 << 30

    def write(x=far, slots=None, codes=at, words=1 << 25, m=4, dim=128, ld=128, rows=8, pitch=64, type=0):
        return said(raven_lib.raven_int4_write_device(x, type, m, dim, ld, slots, L.Rows(codes, words, rows, pitch, 2, 5), None,
                                                      None))

    slots = dict(slots=1 << 28)
    assert write(x=at) and write(x=at + 252) and not write(x=at + 256)  # the rows that are written: the first 4
    assert write(x=at + 508, **slots) and not write(x=at + 512, **slots)
    assert not write(x=at - 2048) and write(x=at - 2044)
    assert write(x=at, pitch=512) and not write(x=at + 64, pitch=576, ld=144) and write(x=at + 60, pitch=576, ld=144)
    assert write(words=far + 8) and write(words=far + 2040) and not write(words=far + 2048) and not write(words=far - 64)
    assert write(slots=at + 8) and not write(slots=at - 16) and write(slots=(1 << 25) + 60) and not write(slots=(1 << 25) + 64)
    assert write(x=at - 1020, type=1) and not write(x=at - 1024, type=1)

    def read(out=far, ids=None, codes=at, words=1 << 25, m=4, dim=128, ld=128, rows=8, type=0):
        return said(raven_lib.raven_int4_read_device(L.Rows(codes, words, rows, 64, 2, 5), dim, ids, m, out, type, ld, None, None))

    assert read(out=at) and read(out=at + 252) and not read(out=at + 256) and not read(out=at - 2048) and read(out=at - 2044)
    assert read(out=at + 508, ids=1 << 28) and not read(out=at + 512, ids=1 << 28)
    assert read(out=(1 << 25) + 60, ids=1 << 28) and not read(out=(1 << 25) + 64, ids=1 << 28) and not read(out=(1 << 25) + 32) and read(ids=far + 16) and not read(ids=far + 2048)
