"""Exhaustive scores beside the graph search, on torch tensors of one GPU.

* `Fp8Rows`      — embedding rows as e4m3 codes with one power-of-two scale per
                   128 values (a quarter of f32, like the SQ8 codes, but with a
                   scale for each block of each row): encode / decode / of_index.
* `scores`       — every query against every row (FP8, f16 or bf16 rows).
* `group_scores` — the queries of each group against the rows of that group,
                   groups of any size: partitions (tenants, lists) of a
                   collection, or one projection per group.
* `group_rows`   — where each query's scores start in grouped scores.
* `top_k`        — the best k of each row of scores, dense or packed.
* `take_status`  — what went wrong on a device in calls without a status.

    rows = Fp8Rows.encode(X)                              # or Fp8Rows.of_index(searcher.device_index)
    near = scores(Q, rows, alpha=-2.0, bias=(rows.decode() ** 2).sum(1))
    dist, ids, _ = top_k(near, 10, largest=False)         # squared distances less |q|^2

Everything runs in libraven_gpu.so on the current stream of the tensors'
device and returns without waiting; nothing is differentiable. The reference
has no counterpart: it scores every vector only in its tests
(test_pybinding.py:16-18), by numpy.
"""
from __future__ import annotations

import ctypes as C
import operator
from typing import Optional, Tuple, Union

import torch

from . import _lib as L

BLOCK = 128  # values under one scale

_TYPES = {torch.float32: L.RAVEN_TYPE_F32, torch.float16: L.RAVEN_TYPE_F16, torch.bfloat16: L.RAVEN_TYPE_BF16}


def _up(x: int, m: int) -> int:
    return -(-x // m) * m


def _u32(x: int) -> int:
    """x as the library's 32-bit arguments take it: what they cannot hold stays out of every limit."""
    return x if 0 <= x < 1 << 32 else (1 << 32) - 1


def _matrix(x, name: str) -> int:
    """The row pitch of a matrix on a GPU with each row's values side by side."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError(f"{name} must be a 2-D tensor")
    if not x.is_cuda:
        raise ValueError(f"{name} must be on a GPU")
    if x.dtype not in _TYPES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, not {x.dtype}")
    (n, dim), (pitch, step) = x.shape, x.stride()
    if dim == 0:
        raise ValueError(f"{name} has rows of no values")
    # one row, or rows of one value, may come with any strides
    if (step != 1 and dim > 1) or (pitch < dim and n > 1):
        raise ValueError(f"{name} must hold each row's values side by side and its rows one after another")
    return pitch if n > 1 else _up(dim, 8)


def _pitch(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else max(x.stride(0), x.shape[1])


def _on(device: int, *tensors) -> None:
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise ValueError(f"all tensors must be on cuda:{device}, got one on {t.device}")


_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _call(device: int, fn, *args) -> None:
    """The library call with `device` current, on its current stream."""
    if torch.cuda.current_device() == device:
        rc = fn(*args, _stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream(device))
    if rc:
        L.check(rc)


def aligned_rows(x: torch.Tensor) -> torch.Tensor:
    """The rows of `x` as `scores` takes 16-bit rows: starting on 16 bytes, 16
    bytes times a whole number apart. A copy where `x` is not laid out so."""
    pitch, step = _matrix(x, "rows"), 16 // x.element_size()
    if x.data_ptr() % 16 == 0 and pitch % step == 0:
        return x
    out = x.new_empty(x.shape[0], _up(x.shape[1], step))[:, : x.shape[1]]
    out.copy_(x)
    return out


class Fp8Rows:
    """Rows held as FP8: `codes` uint8 [n, roundup(dim, 16)] (e4m3) and `exps`
    uint8 [n, roundup(ceil(dim / 128), 4)]; a value is its code times
    2^(exps - 127) of its block of 128, and NaN where that byte is 255. Their
    contents may change, the two tensors stay: other ones make other rows."""

    def __init__(self, codes: torch.Tensor, exps: torch.Tensor, dim: int):
        self._hold(codes, exps, dim)

    def _hold(self, codes: torch.Tensor, exps: torch.Tensor, dim: int) -> None:
        if dim < 1:
            raise ValueError("dim must be at least 1")
        if codes.dim() != 2 or exps.dim() != 2 or codes.dtype != torch.uint8 or exps.dtype != torch.uint8 or \
                not codes.is_cuda:
            raise ValueError("codes and exps must be 2-D uint8 tensors on a GPU")
        (n, wide), (pitch, step) = codes.shape, codes.stride()
        (en, ewide), (epitch, estep) = exps.shape, exps.stride()
        if step != 1 or estep != 1:
            raise ValueError("codes and exps must hold each row's bytes side by side")
        if wide < -(-dim // 16) * 16 or ewide < -(-dim // 512) * 4:
            raise ValueError(f"dim {dim} needs {_up(dim, 16)} columns of codes and {_up(-(-dim // BLOCK), 4)} of exps, "
                             f"got {wide} and {ewide}")
        self.device_index = codes.get_device()
        if en != n or exps.get_device() != self.device_index:
            raise ValueError("codes and exps must have the same rows and device")
        if n == 1:  # one row may come with any pitch
            pitch, epitch = _up(dim, 16), _up(-(-dim // BLOCK), 4)
        self._codes, self._exps, self._dim = codes, exps, dim
        self._n, self._at, self._exps_at = n, codes.data_ptr(), exps.data_ptr()
        self._held = L.Rows(self._at, self._exps_at, n, pitch, epitch, L.RAVEN_TYPE_FP8)

    @property
    def _rows(self) -> L.Rows:
        """The rows as the library takes them, where the tensors are now (resize_ and set_ move them)."""
        if self._codes.data_ptr() != self._at or self._exps.data_ptr() != self._exps_at:
            self._hold(self._codes, self._exps, self._dim)
        return self._held

    @property
    def codes(self) -> torch.Tensor:
        return self._codes

    @property
    def exps(self) -> torch.Tensor:
        return self._exps

    @property
    def dim(self) -> int:
        return self._dim

    @property
    def device(self) -> torch.device:
        return self._codes.device

    def __len__(self) -> int:
        return self._rows.rows

    @staticmethod
    def empty(n: int, dim: int, device) -> "Fp8Rows":
        """Room for n rows, uninitialised."""
        if dim < 1 or n < 0:
            raise ValueError("n must not be negative and dim at least 1")
        return Fp8Rows(torch.empty(n, _up(dim, 16), dtype=torch.uint8, device=device),
                       torch.empty(n, _up(-(-dim // BLOCK), 4), dtype=torch.uint8, device=device), dim)

    @staticmethod
    def encode(x: torch.Tensor, out: Optional["Fp8Rows"] = None) -> "Fp8Rows":
        """The rows of a float32, float16 or bfloat16 matrix, rounded to nearest
        even. The scale of a block is the least power of two that brings its
        values to at most 448; infinities and NaN become NaN. `out`: rows to
        write instead of new ones (len(x) of them)."""
        pitch = _matrix(x, "x")
        (n, dim), device = x.shape, x.get_device()
        if out is None:
            out = Fp8Rows.empty(n, dim, x.device)
        elif len(out) != n or out.dim != dim:
            raise ValueError(f"out holds {len(out)} rows of {out.dim}, expected {n} of {dim}")
        if out.device_index != device:
            raise ValueError(f"out must be on cuda:{device}")
        r = out._rows
        _call(device, L.load().raven_fp8_encode_device, x.data_ptr(), _TYPES[x.dtype], n, _u32(dim), pitch, r.data, r.ld,
              r.exps, r.ld_exps)
        return out

    @staticmethod
    def of_index(index) -> "Fp8Rows":
        """FP8 rows of the vectors of a `DeviceIndex`, on its GPU."""
        out = Fp8Rows.empty(index.n, index.dim, torch.device("cuda", index.device))
        r = out._rows
        _call(index.device, L.load().raven_index_fp8_device, index._h, r.data, r.ld, r.exps, r.ld_exps)
        return out

    def decode(self) -> torch.Tensor:
        """The values, float32 [n, dim] (exact)."""
        out = torch.empty(len(self), self.dim, dtype=torch.float32, device=self.device)
        r = self._rows
        _call(self.device_index, L.load().raven_fp8_decode_device, r.data, r.ld, r.exps, r.ld_exps, len(self),
              _u32(self.dim), out.data_ptr(), self.dim)
        return out

    def rows(self, first: int, count: int) -> "Fp8Rows":
        """Rows [first, first + count), without a copy."""
        if first < 0 or count < 0 or first + count > len(self):
            raise ValueError(f"rows [{first}, {first + count}) of {len(self)}")
        return Fp8Rows(self.codes[first:first + count], self.exps[first:first + count], self.dim)


Rows = Union[torch.Tensor, Fp8Rows]


def _operands(queries: Rows, vectors: Rows, dtype: torch.dtype, bias: Optional[torch.Tensor]):
    """(device, dim, nq, n, queries, vectors) as the library takes them, and what must stay alive until the call."""
    fp8 = isinstance(vectors, Fp8Rows)
    if fp8:
        device, dim, v = vectors.device_index, vectors._dim, vectors._rows
        n = vectors._n
    else:
        pitch = _matrix(vectors, "vectors")
        if vectors.dtype == torch.float32:
            raise ValueError("vectors must be Fp8Rows, float16 or bfloat16 (Fp8Rows.encode holds float32 rows as FP8)")
        (n, dim), device, at = vectors.shape, vectors.get_device(), vectors.data_ptr()
        if at % 16 or pitch % 8:
            raise ValueError("16-bit vectors must start on 16 bytes, a multiple of 8 values apart "
                             "(aligned_rows makes them so)")
        v = L.Rows(at, None, n, pitch, 0, _TYPES[vectors.dtype])
    if isinstance(queries, Fp8Rows):
        if not fp8:
            raise ValueError("FP8 queries need FP8 vectors")
        qdim, q, qdevice = queries._dim, queries._rows, queries.device_index
        nq = queries._n
    else:
        pitch = _matrix(queries, "queries")
        if not fp8:
            if queries.dtype != vectors.dtype:
                raise ValueError(f"queries must have the vectors' type {vectors.dtype}, got {queries.dtype}")
            if pitch % 8 or queries.data_ptr() % 16:
                queries = aligned_rows(queries)
                pitch = _pitch(queries)
        (nq, qdim), qdevice = queries.shape, queries.get_device()
        q = L.Rows(queries.data_ptr(), None, nq, pitch, 0, _TYPES[queries.dtype])
    if qdim != dim:
        raise ValueError(f"dim mismatch: expected {dim}, got {qdim}")
    if qdevice != device:
        raise ValueError(f"queries and vectors must be on one GPU, got cuda:{qdevice} and cuda:{device}")
    if dtype not in _TYPES:
        raise ValueError(f"scores must be float32, float16 or bfloat16, not {dtype}")
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous float32 tensor of {n} values")
        _on(device, bias)
    return device, dim, nq, n, q, v, queries


def _status(status: Optional[torch.Tensor], device: int) -> Optional[int]:
    if status is None:
        return None
    if status.dtype != torch.int32 or status.numel() != 1:
        raise ValueError("status must be an int32 tensor of one value")
    _on(device, status)
    return status.data_ptr()


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def scores(queries: Rows, vectors: Rows, *, alpha: float = 1.0, bias: Optional[torch.Tensor] = None,
           dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None,
           status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """alpha * <query, vector> + bias[vector] for every pair, [nq, n] of `dtype`:
    summed in float32 on the tensor cores, rounded once. Float queries against
    FP8 rows are encoded first. alpha = -2 with the vectors' squared norms as
    bias ranks like squared distances. `out`: a matrix of `dtype` to write (any
    row pitch). `status`: an int32 that gets RAVEN_S_* bits; without it
    `take_status` tells whether the scores are valid."""
    device, dim, nq, n, q, v, keep = _operands(queries, vectors, dtype, bias)
    pitch = n
    if out is None:
        out = (vectors._codes if isinstance(vectors, Fp8Rows) else vectors).new_empty((nq, n), dtype=dtype)
    else:
        if out.shape != (nq, n) or out.dtype != dtype or (n > 1 and out.stride(1) != 1) or (nq > 1 and out.stride(0) < n):
            raise ValueError(f"out must be a {dtype} matrix of {nq} x {n}, each row's values side by side")
        _on(device, out)
        pitch = _pitch(out)
    _call(device, L.load().raven_scores_device, q, v, _u32(dim), float(alpha), _ptr(bias), out.data_ptr(), _TYPES[dtype], pitch,
          _status(status, device))
    return out


def _offsets(name: str, t: torch.Tensor, device: int) -> int:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int64 or t.dim() != 1 or t.numel() < 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D int64 tensor")
    _on(device, t)
    return t.numel() - 1


def group_scores(queries: Rows, query_offsets: torch.Tensor, vectors: Rows, vector_offsets: torch.Tensor, *,
                 total: Optional[int] = None, alpha: float = 1.0, bias: Optional[torch.Tensor] = None,
                 dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Scores of the queries [query_offsets[g], query_offsets[g + 1]) against the
    vectors [vector_offsets[g], vector_offsets[g + 1]) for each group g, packed:
    groups in order, their queries in order, for each the scores of its group's
    vectors. Offsets are int64 tensors on the GPU, rising; either side of a group
    may be empty.

    `total` is the number of scores (the program that made the groups knows it:
    the sum of queries times vectors; the last of `group_rows`), or `out` a 1-D
    tensor with room for them. Nothing is written past it: queries whose scores
    all fit have them, and `status` gets RAVEN_S_CAPACITY. Groups whose offsets fall
    or leave the rows have no scores, and it gets RAVEN_S_OFFSETS; without a
    `status`, `take_status` tells of both."""
    device, dim, nq, n, q, v, keep = _operands(queries, vectors, dtype, bias)
    groups = _offsets("query_offsets", query_offsets, device)
    if _offsets("vector_offsets", vector_offsets, device) != groups:
        raise ValueError("query_offsets and vector_offsets must have the same length")
    if out is None:
        if total is None:
            raise ValueError("total or out is needed: the number of scores is known on the GPU only")
        out = torch.empty(total, dtype=dtype, device=vectors.device)
    elif out.dim() != 1 or out.dtype != dtype or not out.is_contiguous() or (total is not None and out.numel() < total):
        raise ValueError(f"out must be a contiguous 1-D {dtype} tensor with room for the scores")
    else:
        _on(device, out)
    _call(device, L.load().raven_group_scores_device, q, query_offsets.data_ptr(), v, vector_offsets.data_ptr(),
          _u32(groups), _u32(dim), float(alpha), _ptr(bias), out.data_ptr(), _TYPES[dtype], out.numel(), _status(status, device))
    return out


def group_rows(query_offsets: torch.Tensor, vector_offsets: torch.Tensor, nq: int, n: int,
               status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int64 [nq + 1]: where each query's scores start in the output of
    `group_scores`, and its size; the row_starts of `top_k`. Queries of no group,
    or of one whose offsets fall or leave the rows, have rows of no scores."""
    device = query_offsets.get_device()
    groups = _offsets("query_offsets", query_offsets, device)
    if _offsets("vector_offsets", vector_offsets, device) != groups:
        raise ValueError("query_offsets and vector_offsets must have the same length")
    if not query_offsets.is_cuda:
        raise ValueError("query_offsets must be on a GPU")
    if groups == 0 or nq < 0 or n < 0:
        raise ValueError("there must be at least one group, and nq and n must not be negative")
    out = torch.empty(nq + 1, dtype=torch.int64, device=query_offsets.device)
    _call(device, L.load().raven_group_rows_device, query_offsets.data_ptr(), vector_offsets.data_ptr(), _u32(groups), nq,
          _u32(n), out.data_ptr(), _status(status, device))
    return out


def take_status(device=None) -> int:
    """The RAVEN_S_* bits that calls without a `status` have set on a GPU (the
    current one) since they were last taken: 0 when all went well. Waits for the
    current stream; calls on others may add theirs later."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError("device must be a GPU")
    bits = torch.zeros(1, dtype=torch.int32, device=device)
    _call(bits.get_device(), L.load().raven_scoring_status_device, bits.data_ptr())
    return int(bits)


def top_k(scores: torch.Tensor, k: int, *, largest: bool = True,
          row_starts: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(values [nq, k], ids [nq, k] int32, counts [nq] int32) of the best k
    (1..256) of each row, best first, equal scores by the lower index, NaN after
    every number. Rows are those of a matrix, or with `row_starts` (int64, nq + 1
    values) pieces of a packed 1-D tensor; ids count within the row (in rows of
    2^31 scores and more, which only packed ones can be, their bits are unsigned;
    scores from 2^32 - 1 on are not looked at). Slots past a row's count (rows of
    fewer than k) are 0."""
    if not isinstance(scores, torch.Tensor) or not scores.is_cuda or scores.dtype not in _TYPES:
        raise ValueError("scores must be a float32, float16 or bfloat16 tensor on a GPU")
    index, device, k = scores.get_device(), scores.device, operator.index(k)
    if row_starts is None:
        if scores.dim() != 2:
            raise ValueError("scores must be a matrix, or packed with row_starts")
        (nq, n), (ld, step), starts = scores.shape, scores.stride(), None
        if (n > 1 and step != 1) or (nq > 1 and ld < n):
            raise ValueError("scores must hold each row's values side by side and its rows one after another")
        ld = max(ld, n)
    else:
        if scores.dim() != 1 or not scores.is_contiguous():
            raise ValueError("packed scores must be a contiguous 1-D tensor")
        nq, n, ld, starts = _offsets("row_starts", row_starts, index), scores.numel(), 0, row_starts.data_ptr()
    wide = k if 0 < k <= L.RAVEN_MAX_TOP_K else 0  # other k are refused before anything is written
    vals = scores.new_empty((nq, wide))
    ids = torch.empty((nq, wide), dtype=torch.int32, device=device)
    counts = torch.empty(nq, dtype=torch.int32, device=device)
    _call(index, L.load().raven_topk_rows_device, scores.data_ptr(), _TYPES[scores.dtype], nq, n, ld, starts, _u32(k),
          int(largest), vals.data_ptr(), ids.data_ptr(), counts.data_ptr())
    return vals, ids, counts
