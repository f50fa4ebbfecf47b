"""Refusals of the scoring entry points, which come before any device work, and
the 64-bit definitions the GPU tests use (no GPU needed)."""
import ctypes as C

import numpy as np
import pytest

import scoring_util as U


def _rows(L, data=4096, exps=4096, rows=8, ld=128, ld_exps=4, type=3):
    return L.Rows(data, exps, rows, ld, ld_exps, type)


def _call(raven_lib, q, v, dim=128, out=4096, out_type=0, ld=8):
    return raven_lib.raven_scores_device(q, v, dim, 1.0, None, out, out_type, ld, None, None)


def test_scores_refusals(raven_lib):
    from raven_b200 import _lib as L

    ok = lambda **k: _rows(L, **k)  # noqa: E731
    EINVAL, ELIMIT = L.RAVEN_EINVAL, L.RAVEN_ELIMIT
    assert _call(raven_lib, ok(), ok(), dim=0) == ELIMIT
    assert _call(raven_lib, ok(), ok(), dim=65537) == ELIMIT
    assert _call(raven_lib, ok(rows=1 << 31), ok()) == ELIMIT
    assert _call(raven_lib, None, ok()) == EINVAL
    assert _call(raven_lib, ok(type=7), ok()) == EINVAL
    assert _call(raven_lib, ok(), ok(type=0)) == EINVAL            # f32 vectors
    assert _call(raven_lib, ok(type=3), ok(type=1)) == EINVAL      # FP8 queries, f16 vectors
    assert _call(raven_lib, ok(type=2), ok(type=1)) == EINVAL
    assert _call(raven_lib, ok(), ok(data=4100)) == EINVAL         # codes off 16 bytes
    assert _call(raven_lib, ok(), ok(ld=132)) == EINVAL
    assert _call(raven_lib, ok(), ok(ld=112)) == EINVAL
    assert _call(raven_lib, ok(), ok(ld_exps=6)) == EINVAL
    assert _call(raven_lib, ok(), ok(exps=None)) == EINVAL
    assert _call(raven_lib, ok(), ok(exps=4098)) == EINVAL
    assert _call(raven_lib, ok(), ok(ld=1024, ld_exps=4), dim=600) == EINVAL  # five blocks need eight bytes
    assert _call(raven_lib, ok(), ok(data=None)) == EINVAL
    assert _call(raven_lib, ok(type=1, data=4098), ok(type=1)) == EINVAL
    assert _call(raven_lib, ok(type=1, ld=132), ok(type=1)) == EINVAL
    assert _call(raven_lib, ok(type=0, data=4097), ok()) == EINVAL
    assert _call(raven_lib, ok(), ok(), out=None) == EINVAL
    assert _call(raven_lib, ok(), ok(), out=4098) == EINVAL
    assert _call(raven_lib, ok(), ok(), out_type=3) == EINVAL
    assert _call(raven_lib, ok(), ok(), ld=7) == EINVAL
    assert b"pitch" in raven_lib.raven_last_error()
    # nothing to do is no error
    assert _call(raven_lib, ok(rows=0), ok()) == 0
    assert _call(raven_lib, ok(), ok(rows=0)) == 0
    group = lambda qo, vo, groups, cap: raven_lib.raven_group_scores_device(  # noqa: E731
        ok(), qo, ok(), vo, groups, 128, 1.0, None, 4096, 0, cap, None, None)
    assert group(None, 4096, 1, 10) == EINVAL
    assert group(4096, 4100, 1, 10) == EINVAL
    assert group(4096, 4096, 0, 10) == 0
    assert group(4096, 4096, 3, 0) == 0
    assert group(4096, 4096, 1 << 31, 10) == L.RAVEN_ELIMIT
    for bias, status in ((4098, None), (None, 4097)):
        assert raven_lib.raven_scores_device(ok(), ok(), 128, 1.0, bias, 4096, 0, 8, status, None) == EINVAL


def test_encode_decode_refusals(raven_lib):
    from raven_b200 import _lib as L

    def enc(x=4096, type=0, n=4, dim=100, ld=100, codes=4096, ldc=112, exps=4096, lde=4):
        return raven_lib.raven_fp8_encode_device(x, type, n, dim, ld, codes, ldc, exps, lde, None)

    assert enc(type=3) == L.RAVEN_EINVAL and enc(x=None) == L.RAVEN_EINVAL and enc(ld=99) == L.RAVEN_EINVAL
    assert enc(x=4098) == L.RAVEN_EINVAL and enc(ldc=96) == L.RAVEN_EINVAL and enc(ldc=113) == L.RAVEN_EINVAL
    assert enc(codes=None) == L.RAVEN_EINVAL and enc(exps=4097) == L.RAVEN_EINVAL and enc(lde=2) == L.RAVEN_EINVAL
    assert enc(dim=0) == L.RAVEN_ELIMIT and enc(n=1 << 31) == L.RAVEN_ELIMIT and enc(n=0) == 0

    def dec(out=4096, ld=100, codes=4096):
        return raven_lib.raven_fp8_decode_device(codes, 112, 4096, 4, 4, 100, out, ld, None)

    assert dec(out=None) == L.RAVEN_EINVAL and dec(ld=99) == L.RAVEN_EINVAL and dec(codes=4104) == L.RAVEN_EINVAL
    assert raven_lib.raven_index_fp8_device(None, 4096, 112, 4096, 4, None) == L.RAVEN_EINVAL


def test_topk_and_group_rows_refusals(raven_lib):
    from raven_b200 import _lib as L

    def top(x=4096, type=0, nq=2, n=10, ld=10, starts=None, k=3, vals=4096, ids=4096, counts=None):
        return raven_lib.raven_topk_rows_device(x, type, nq, n, ld, starts, k, 1, vals, ids, counts, None)

    assert top(k=0) == L.RAVEN_ELIMIT and top(k=257) == L.RAVEN_ELIMIT
    assert top(n=1 << 31, ld=1 << 31) == L.RAVEN_ELIMIT and top(nq=1 << 31) == L.RAVEN_ELIMIT
    assert top(type=3) == L.RAVEN_EINVAL and top(x=None) == L.RAVEN_EINVAL and top(ld=9) == L.RAVEN_EINVAL
    assert top(x=4098) == L.RAVEN_EINVAL and top(starts=4100) == L.RAVEN_EINVAL and top(vals=None) == L.RAVEN_EINVAL
    assert top(ids=None) == L.RAVEN_EINVAL and top(ids=4097) == L.RAVEN_EINVAL and top(nq=0) == 0

    def rows(qo=4096, vo=4096, groups=2, nq=5, n=5, out=4096):
        return raven_lib.raven_group_rows_device(qo, vo, groups, nq, n, out, None, None)

    assert rows(groups=1 << 31) == L.RAVEN_ELIMIT
    assert raven_lib.raven_group_rows_device(4096, 4096, 2, 5, 5, 4096, 4098, None) == L.RAVEN_EINVAL
    assert rows(qo=None) == L.RAVEN_EINVAL and rows(groups=0) == L.RAVEN_EINVAL and rows(out=4100) == L.RAVEN_EINVAL
    assert rows(nq=1 << 31) == L.RAVEN_ELIMIT


def test_rows_struct_matches_header(tmp_path):
    import os
    import shutil
    import subprocess

    from raven_b200 import _lib as L

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "rows.c"
    fields = [f for f, _ in L.Rows._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "raven_gpu.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu ", offsetof(raven_rows, {f}));\n' for f in fields)
                   + '  printf("%zu %d %d %d %d", sizeof(raven_rows), RAVEN_TYPE_F32, RAVEN_TYPE_F16, RAVEN_TYPE_BF16, '
                   'RAVEN_TYPE_FP8);\n  return 0;\n}\n')
    exe = tmp_path / "rows"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(L.Rows, f).offset for f in fields] + [C.sizeof(L.Rows), L.RAVEN_TYPE_F32, L.RAVEN_TYPE_F16,
                                                                 L.RAVEN_TYPE_BF16, L.RAVEN_TYPE_FP8]


def test_python_refuses_host_tensors(raven_lib):
    import torch

    from raven_b200 import scoring

    x = torch.zeros(4, 64)
    for call in (lambda: scoring.Fp8Rows.encode(x), lambda: scoring.scores(x, x.half()),
                 lambda: scoring.top_k(x, 2), lambda: scoring.aligned_rows(x),
                 lambda: scoring.Fp8Rows(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 64)):
        with pytest.raises(ValueError):
            call()


def test_definitions():
    torch = pytest.importorskip("torch")
    r = np.random.default_rng(0)
    y = np.concatenate([r.uniform(-448, 448, 2000), r.uniform(-0.1, 0.1, 2000), [17.0, 19.0, 448.0, 2.0 ** -10, 0.0]])
    want = torch.tensor(y, dtype=torch.float64).float().to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(U.e4m3_round(y.astype(np.float32)), want)
    assert U.fp8_exponents(np.array([[448.0], [449.0], [0.0], [224.0], [1e-42]])).ravel().tolist() == [0, 1, 0, -1, -127]
    vals, ids, counts = U.top_k([[1.0, np.nan, 1.0, np.inf], []], 3, True)
    assert ids.tolist() == [[3, 0, 2], [0, 0, 0]] and counts.tolist() == [3, 0]


def test_status_refusals(raven_lib):
    from raven_b200 import _lib as L

    assert raven_lib.raven_scoring_status_device(None, None) == L.RAVEN_EINVAL
    assert raven_lib.raven_scoring_status_device(4098, None) == L.RAVEN_EINVAL
