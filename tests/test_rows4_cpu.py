"""Refusals of the operators on 4-bit rows and of adjusted scores, which come
before any device work, and the 64-bit definitions the GPU tests use (no GPU needed)."""
import ctypes as C

import numpy as np
import pytest

import rows4_util as U


def _rows(data=4096, exps=4096, rows=8, ld=64, ld_exps=2, type=5):
    from raven_b200 import _lib as L

    return L.Rows(data, exps, rows, ld, ld_exps, type)


BAD_ROWS = [dict(type=3), dict(type=0), dict(type=7), dict(rows=1 << 31), dict(data=None), dict(exps=None), dict(data=4104),
            dict(ld=72), dict(ld=48), dict(exps=4100), dict(ld_exps=3), dict(ld_exps=0), dict(type=4, ld_exps=2),
            dict(type=4, exps=4104)]


def test_write_refusals(raven_lib):
    from raven_b200 import _lib as L

    def write(x=4096, type=0, m=4, dim=128, ld=128, slots=None, out=None, status=None, **k):
        out = _rows(**k) if out is None else out
        return raven_lib.raven_int4_write_device(x, type, m, dim, ld, slots, out, status, None)

    for bad in BAD_ROWS:
        kind = L.RAVEN_ELIMIT if bad.get("rows") == 1 << 31 else L.RAVEN_EINVAL
        bad = dict(bad)
        rows = _rows(**bad)
        assert raven_lib.raven_int4_write_device(4096, 0, 4, 128, 128, None, rows, None, None) == kind, bad
    assert raven_lib.raven_int4_write_device(4096, 0, 4, 128, 128, None, None, None, None) == L.RAVEN_EINVAL
    assert write(type=3) == L.RAVEN_EINVAL and write(type=5) == L.RAVEN_EINVAL
    assert write(x=None) == L.RAVEN_EINVAL and write(x=4098) == L.RAVEN_EINVAL and write(ld=127) == L.RAVEN_EINVAL
    assert write(dim=0) == L.RAVEN_ELIMIT and write(dim=65537) == L.RAVEN_ELIMIT
    assert write(m=9) == L.RAVEN_EINVAL                        # more rows than there are, without slots
    assert write(m=1 << 31) == L.RAVEN_ELIMIT and write(m=(1 << 30) + 1, slots=4096) == L.RAVEN_ELIMIT
    assert write(slots=4098) == L.RAVEN_EINVAL and write(status=4097) == L.RAVEN_EINVAL
    assert write(m=0) == 0 and write(m=0, x=None) == 0


def test_read_refusals(raven_lib):
    from raven_b200 import _lib as L

    def read(rows=None, dim=128, ids=None, m=4, out=4096, type=0, ld=128, status=None):
        return raven_lib.raven_int4_read_device(_rows() if rows is None else rows, dim, ids, m, out, type, ld, status, None)

    for bad in BAD_ROWS:
        kind = L.RAVEN_ELIMIT if bad.get("rows") == 1 << 31 else L.RAVEN_EINVAL
        assert read(_rows(**bad)) == kind, bad
    assert read(out=None) == L.RAVEN_EINVAL and read(out=4098) == L.RAVEN_EINVAL and read(type=3) == L.RAVEN_EINVAL
    assert read(ld=127) == L.RAVEN_EINVAL and read(dim=0) == L.RAVEN_ELIMIT and read(m=9) == L.RAVEN_EINVAL
    assert read(m=1 << 31, ids=4096) == L.RAVEN_ELIMIT and read(ids=4098) == L.RAVEN_EINVAL
    assert read(status=4098) == L.RAVEN_EINVAL and read(m=0) == 0
    assert raven_lib.raven_index_int4_device(None, _rows(), None) == L.RAVEN_EINVAL


def test_scores_refusals(raven_lib):
    from raven_b200 import _lib as L

    def scores(q=None, v=None, dim=128, bias=None, out=4096, type=0, ld=8, status=None):
        q = L.Rows(4096, None, 4, 128, 0, 0) if q is None else q
        v = _rows() if v is None else v
        return raven_lib.raven_scores_device(q, v, dim, 1.0, bias, out, type, ld, status, None)

    for bad in BAD_ROWS[3:]:
        kind = L.RAVEN_ELIMIT if bad.get("rows") == 1 << 31 else L.RAVEN_EINVAL
        assert scores(v=_rows(**bad)) == kind, bad
    for q in (L.Rows(4096, 4096, 4, 128, 4, 3), _rows(), L.Rows(None, None, 4, 128, 0, 0), L.Rows(4098, None, 4, 128, 0, 0),
              L.Rows(4096, None, 4, 127, 0, 0), L.Rows(4097, None, 4, 128, 0, 1)):
        assert scores(q=q) == L.RAVEN_EINVAL
    assert scores(q=L.Rows(4096, None, 1 << 31, 128, 0, 0)) == L.RAVEN_ELIMIT
    assert raven_lib.raven_scores_device(None, _rows(), 128, 1.0, None, 4096, 0, 8, None, None) == L.RAVEN_EINVAL
    assert scores(dim=0) == L.RAVEN_ELIMIT and scores(out=None) == L.RAVEN_EINVAL and scores(out=4098) == L.RAVEN_EINVAL
    assert scores(type=3) == L.RAVEN_EINVAL and scores(ld=7) == L.RAVEN_EINVAL
    assert scores(bias=4098) == L.RAVEN_EINVAL and scores(status=4098) == L.RAVEN_EINVAL
    assert scores(q=L.Rows(None, None, 0, 128, 0, 0)) == 0 and scores(v=_rows(rows=0)) == 0
    group = raven_lib.raven_group_scores_device(L.Rows(4096, None, 4, 128, 0, 0), 4096, _rows(), 4096, 1, 128, 1.0, None, 4096,
                                                0, 32, None, None)
    assert group == L.RAVEN_EINVAL and b"grouped" in raven_lib.raven_last_error()


def test_adjust_refusals(raven_lib):
    from raven_b200 import _lib as L

    def adjust(x=4096, type=0, nq=4, n=100, ld=100, out=1 << 20, ld_out=100, status=None, null=False, **k):
        by = L.Adjustments(**k)
        by.repetition_all = 1.0
        return raven_lib.raven_adjust_scores_device(x, type, nq, n, ld, None if null else by, 1, out, ld_out, status, None)

    E = L.RAVEN_EINVAL
    assert adjust(null=True) == E and adjust(type=3) == E and adjust(x=None) == E and adjust(out=None) == E
    assert adjust(nq=1 << 31) == L.RAVEN_ELIMIT and adjust(n=1 << 31, ld=1 << 31, ld_out=1 << 31) == L.RAVEN_ELIMIT
    assert adjust(ld=99) == E and adjust(ld_out=99) == E and adjust(x=4098) == E and adjust(out=4098) == E
    assert adjust(ld=1 << 62) == L.RAVEN_ELIMIT and adjust(ld_out=1 << 62) == L.RAVEN_ELIMIT
    assert adjust(out=4096 + 400) == E and adjust(x=4096 + 400, out=4096) == E and adjust(out=4096, ld_out=101) == E
    assert adjust(bias=4098) == E and adjust(bias=4096, ld_bias=99) == E
    assert adjust(allow=4096, allow_count=0, ld_allow=4) == E and adjust(allow=4096, allow_count=4, ld_allow=3) == E
    assert adjust(allow=4096, allow_count=2, ld_allow=4) == E and adjust(allow=4098, allow_count=1, ld_allow=4) == E
    assert adjust(allow=4096, allow_count=2, ld_allow=4, allow_rows=4098) == E
    assert adjust(seen=4096, seen_total=3) == E and adjust(seen_starts=4096, seen_total=3) == E
    assert adjust(seen=4096, seen_total=3, seen_starts=4100) == E
    assert adjust(repetition=4098) == E and adjust(presence=4098) == E and adjust(frequency=4098) == E
    assert adjust(status=4098) == E
    assert adjust(nq=0) == 0 and adjust(n=0) == 0


def test_structs_match_header(tmp_path):
    import os
    import shutil
    import subprocess

    from raven_b200 import _lib as L

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "a.c"
    fields = [f for f, _ in L.Adjustments._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "raven_gpu.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu ", offsetof(raven_adjustments, {f}));\n' for f in fields)
                   + '  printf("%zu %d %d %d %d", sizeof(raven_adjustments), RAVEN_TYPE_INT4_32, RAVEN_TYPE_INT4_64, '
                   'RAVEN_TYPE_INT4_128, RAVEN_S_IDS);\n  return 0;\n}\n')
    exe = tmp_path / "a"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(L.Adjustments, f).offset for f in fields] + [
        C.sizeof(L.Adjustments), L.RAVEN_TYPE_INT4_32, L.RAVEN_TYPE_INT4_64, L.RAVEN_TYPE_INT4_128, L.RAVEN_S_IDS]


def test_python_refuses_host_tensors(raven_lib):
    import torch

    from raven_b200 import scoring

    x = torch.zeros(4, 64)
    for call in (lambda: scoring.Int4Rows.encode(x), lambda: scoring.adjust(x),
                 lambda: scoring.Int4Rows(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.int32), 64)):
        with pytest.raises(ValueError):
            call()


def test_definitions():
    from fractions import Fraction

    r = np.random.default_rng(0)
    x = r.normal(size=(40, 70)) * 2.0 ** r.uniform(-8, 8, (40, 1))
    x[3], x[4, :32], x[5, 32:64] = 0.0, 5.5, np.arange(32) - 4.0
    x = x.astype(np.float32)
    for group in (32, 64, 128):
        codes, words, vals = U.encode(x, group)
        for i in range(40):
            for g in range(words.shape[1]):
                p = x[i, g * group:(g + 1) * group]
                lo, hi = Fraction(float(p.min())), Fraction(float(p.max()))
                need = max((hi - lo) / 15, max(hi, -lo) / 127)
                step = Fraction(float(np.uint32(words[i, g] & 0xFFFFFF00).view(np.float32)))
                z = int((int(words[i, g]) & 255) ^ 128) - 128
                assert step >= need and (step == 0 or step * (1 - Fraction(1, 1 << 15)) < need)
                assert -127 <= z <= 127
                for k, v in enumerate(p):
                    got = (int(codes[i, g * group + k]) + z) * step
                    assert got == Fraction(float(vals[i, g * group + k]))
                    assert abs(got - Fraction(float(v))) <= step / 2
    # a row as it is held, and back
    at, shift = U.held_codes(300)
    assert len({(a, s) for a, s in zip(at, shift)}) == 300 and at.max() < 160
    held = np.zeros((2, 160), np.uint8)
    c = r.integers(0, 16, (2, 300))
    for d in range(300):
        held[:, at[d]] |= (c[:, d] << shift[d]).astype(np.uint8)
    np.testing.assert_array_equal(U.unpack(held, 300), c)
    # adjusted scores by hand
    got = U.adjust([[2.0, -2.0, 1.0, 3.0]], True, np.float32([0, 0, 1, 0]), np.array([[0b0111]], np.int32), None,
                   np.array([0, 1, 1]), np.array([0, 3]), 2.0, 0.5, 0.25)
    assert got.tolist() == [[1.0 - 0.75, -4.0 - 1.0, 2.0, -np.inf]]
    got = U.adjust([[2.0, -2.0, 1.0]], False, None, None, None, np.array([0, 1, 1]), np.array([0, 3]), 2.0, 0.5, 0.25)
    assert got.tolist() == [[4.0 + 0.75, -1.0 + 1.0, 1.0]]
