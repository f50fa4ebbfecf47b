"""Cases of the 4-bit rows and of what is done to scores before the best are
taken: rows held as 4-bit codes with a scale for each group of values, written
into a collection in place and read back by id; the scores of a few queries
against such rows; and scores put right for what a query has seen, a bias and
the rows it may see.

`run` computes a case in its plain form (elementary torch operations, 32 bits,
64 where a code lies next to a border) or, with `own` true, through
raven_b200.scoring. `exact` computes the same in 64 bits from the definitions.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one query against a 100k collection of 128-dim descriptors: latency of a lookup
        dict(name="int4-1x100k-d128", op="int4", nq=1, n=100_000, dim=128, group=128, query="f32", out="f32"),
        # one query against the 1M collection: reading the codes
        dict(name="int4-1x1m-d128", op="int4", nq=1, n=1_000_000, dim=128, group=64, query="f32", out="f32"),
        # a small serving batch over text embeddings
        dict(name="int4-8x65536-d1024", op="int4", nq=8, n=65_536, dim=1024, group=128, query="bf16", out="f32"),
        # a few queries against few long rows: a projection of one token of each request
        dict(name="int4-3x20011-d4096", op="int4", nq=3, n=20_011, dim=4096, group=32, query="f16", out="f16"),
        # an odd batch against 96-dim rows, 16-bit scores
        dict(name="int4-33x250007-d96", op="int4", nq=33, n=250_007, dim=96, group=32, query="f32", out="bf16"),
        # the largest batch before tensor-core rows pay: reading codes and writing scores
        dict(name="int4-64x1m-d128", op="int4", nq=64, n=1_000_000, dim=128, group=64, query="f16", out="f32"),
        # a batch of changed descriptors goes into the collection and is read back
        dict(name="rows-64-of-100k-d128", op="rows", m=64, n=100_000, reads=64, dim=128, group=64, type="f32", out="f32"),
        # rows that have just been embedded are written; candidates of a batch of queries are read for ranking
        dict(name="rows-30000-of-100k-d768", op="rows", m=30_000, n=100_000, reads=40_000, dim=768, group=128, type="f16",
             out="f16"),
        # a whole collection goes in and comes back
        dict(name="rows-1m-of-1m-d128", op="rows", m=1_000_000, n=1_000_000, reads=1_000_000, dim=128, group=32,
             type="f32", out="bf16"),
        # one user's scores over a 100k collection: seen rows count less, a filter of the user's own
        dict(name="adjust-1x100k", op="adjust", nq=1, n=100_000, masks=1, seen=500, bias=True, type="f32", largest=True),
        # a batch of 16-bit scores over an odd collection, filters shared by tenants, long histories
        dict(name="adjust-256x250007", op="adjust", nq=256, n=250_007, masks=20, seen=4000, bias=True, type="bf16",
             largest=True),
        # squared distances of a batch against the 1M collection
        dict(name="adjust-64x1m", op="adjust", nq=64, n=1_000_000, masks=64, seen=200, bias=False, type="f32",
             largest=False),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["int4", "rows", "adjust"])
    if op == "int4":
        while True:
            c = dict(op=op, nq=_spread(rng, 1, 64), n=_spread(rng, 1000, 1_000_000), dim=_spread(rng, 32, 4096),
                     group=rng.choice([32, 64, 128]), query=rng.choice(["f32", "f16", "bf16"]),
                     out=rng.choice(["f32", "f16", "bf16"]))
            if c["n"] * c["dim"] <= 1 << 27 and c["nq"] * c["n"] <= 1 << 25:
                return c
    if op == "rows":
        while True:
            n = _spread(rng, 64, 1_000_000)
            c = dict(op=op, m=min(n, _spread(rng, 1, 1_000_000)), n=n, reads=_spread(rng, 1, 1_000_000),
                     dim=_spread(rng, 32, 4096), group=rng.choice([32, 64, 128]), type=rng.choice(["f32", "f16", "bf16"]),
                     out=rng.choice(["f32", "f16", "bf16"]))
            if n * c["dim"] <= 1 << 27 and c["m"] * c["dim"] <= 1 << 26 and c["m"] <= c["reads"] and c["reads"] * c["dim"] <= 1 << 26:
                return c
    while True:
        c = dict(op=op, nq=_spread(rng, 1, 2000), n=_spread(rng, 1000, 1_000_000), masks=_spread(rng, 1, 64),
                 seen=_spread(rng, 1, 8000), bias=rng.random() < 0.5, type=rng.choice(["f32", "f16", "bf16"]),
                 largest=rng.random() < 0.7)
        if c["nq"] * c["n"] <= 1 << 26:
            return c


# ---- inputs -----------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _rows(g, n, dim):
    """Embedding rows: points around shared centres; 128-dim and shorter ones
    are descriptors (integers in 0..255, a third of them zero), longer ones
    have unit length and a few outlying values."""
    centres = torch.randn(64, dim, generator=g, device=DEV)
    at = torch.randint(0, 64, (n,), generator=g, device=DEV)
    x = centres[at].add_(torch.randn(n, dim, generator=g, device=DEV))
    if dim <= 128:
        return x.mul_(40.0).clamp_(0.0, 255.0).round_()
    x[:, :: max(1, dim // 5)] *= 6.0
    return x.div_(x.norm(dim=1, keepdim=True))


def _units(dim):
    return -(-dim // 32)


def _words_wide(dim, group):
    """Scale words of a row as it is held: whole blocks of 128 values."""
    return -(-dim // 128) * (128 // group)


def _order(dim, device):
    """Where the eight values 8i..8i+7 of a row are held, by i: word number.
    A block of 128 values is 16 words, a shorter last one (u units of 32 values)
    4u; the words of a quarter of each unit stand side by side."""
    units = _units(dim)
    i = torch.arange(4 * units, device=device)
    block, unit, quarter = i // 16, i // 4 % 4, i % 4
    wide = (units - 4 * block).clamp(max=4)
    return 16 * block + wide * quarter + unit


def _pow2(e):
    """2^e in 64 bits, -1022 <= e <= 1023."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _over(x, by):
    """x / by, the quotient itself rounded: by a plain number torch multiplies with its reciprocal."""
    return x / torch.full((), float(by), dtype=x.dtype, device=x.device)


def _encode(x, group):
    """Codes and scale words of rows. The step of a group is the least with 16
    significant bits that covers its range in 15 steps and its magnitude in 127;
    a value is held as the nearest multiple of it."""
    n, dim = x.shape
    ng = -(-dim // group)
    p = torch.zeros(n, ng * group, dtype=torch.float64, device=x.device)
    p[:, :dim] = x
    p = p.view(n, ng, group)
    there = (torch.arange(ng * group, device=x.device) < dim).view(ng, group)
    lo = torch.where(there, p, torch.full_like(p, math.inf)).amin(2)
    hi = torch.where(there, p, torch.full_like(p, -math.inf)).amax(2)
    need = torch.maximum(_over(hi - lo, 15), _over(torch.maximum(hi, -lo), 127))
    e = torch.frexp(need)[1].clamp(min=-125)
    step = torch.ceil(need * _pow2(16 - e)) * _pow2(e - 16)
    by = torch.where(step > 0, step, torch.ones_like(step))
    z = torch.round(lo / by)
    c = (torch.round(p / by[:, :, None]) - z[:, :, None]).clamp_(0, 15).int()
    c = torch.where(there, c, torch.zeros_like(c)).view(n, ng * group)
    wide = 32 * _units(dim)
    c = torch.nn.functional.pad(c, (0, max(0, wide - ng * group)))[:, :wide].reshape(n, wide // 8, 8)
    word = c[:, :, 7]
    for k in range(6, -1, -1):
        word = (word << 4) | c[:, :, k]
    codes = torch.empty_like(word)
    codes[:, _order(dim, x.device)] = word
    scales = torch.zeros(n, _words_wide(dim, group), dtype=torch.int32, device=x.device)
    scales[:, :ng] = step.float().view(torch.int32) | (z.int() & 255)
    return codes.view(torch.uint8), scales


def _decode(codes, scales, dim, group):
    word = codes.view(torch.int32)[:, _order(dim, codes.device)]
    shift = 4 * torch.arange(8, device=codes.device, dtype=torch.int32)
    c = ((word[:, :, None] >> shift) & 15).view(codes.shape[0], -1)[:, :dim]
    z = ((scales << 24) >> 24).repeat_interleave(group, 1)[:, :dim]
    step = (scales & -256).view(torch.float32).repeat_interleave(group, 1)[:, :dim]
    return (c + z).float() * step


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "int4":
        s["q"] = _rows(g, case["nq"], case["dim"]).to(TYPES[case["query"]])
        s["codes"], s["scales"] = _encode(_rows(g, case["n"], case["dim"]), case["group"])
    elif case["op"] == "rows":
        n, m, reads = case["n"], case["m"], case["reads"]
        s["codes"], s["scales"] = _encode(_rows(g, n, case["dim"]), case["group"])
        s["x"] = _rows(g, m, case["dim"]).to(TYPES[case["type"]])
        s["slots"] = torch.randperm(n, generator=g, device=DEV)[:m].int()
        # every row that the pass changes is read back, among others
        more = torch.randint(0, n, (reads - m,), generator=g, device=DEV).int()
        s["ids"] = torch.cat([s["slots"], more])[torch.randperm(reads, generator=g, device=DEV)]
    else:
        nq, n = case["nq"], case["n"]
        x = torch.randn(nq, n, generator=g, device=DEV)
        s["x"] = (x.mul_(3.0) if case["largest"] else x.mul_(900.0).add_(3000.0).round_()).to(TYPES[case["type"]])
        # histories of uneven length, popular rows more often, some more than once
        length = (torch.rand(nq, generator=g, device=DEV).pow_(2.0) * (2 * case["seen"] + 1)).long()
        s["starts"] = torch.cat([length.new_zeros(1), length.cumsum(0)])
        total = int(s["starts"][-1])
        s["seen"] = (torch.rand(total, generator=g, device=DEV, dtype=torch.float64).pow_(3.0) * n).int().clamp_(max=n - 1)
        s["owner"] = torch.repeat_interleave(torch.arange(nq, device=DEV), length)  # of the plain form
        s["repetition"] = 1.0 + 0.5 * torch.rand(nq, generator=g, device=DEV)
        s["presence"] = torch.rand(nq, generator=g, device=DEV)
        s["frequency"] = 0.5 * torch.rand(nq, generator=g, device=DEV)
        # filters: half of the words leave most rows, the others few; the last filter of several leaves none
        bits = torch.randint(-(1 << 31), 1 << 31, (3, case["masks"], -(-n // 32)), generator=g, device=DEV).int()
        s["allow"] = torch.where(bits[2] < 0, bits[0] | bits[1], bits[0] & bits[1])
        if case["masks"] > 2:
            s["allow"][-1] = 0
        # the filter of each query; -1: it may see all
        s["allow_rows"] = torch.randint(-1, case["masks"], (nq,), generator=g, device=DEV).int()
        s["bias"] = torch.randn(n, generator=g, device=DEV) if case["bias"] else None
    return s


# ---- one pass ---------------------------------------------------------------


def _run_own(s):
    from raven_b200 import scoring

    if s["op"] == "int4":
        return scoring.scores(s["q"], scoring.Int4Rows(s["codes"], s["scales"], s["dim"], s["group"]), dtype=TYPES[s["out"]])
    if s["op"] == "rows":
        rows = scoring.Int4Rows(s["codes"], s["scales"], s["dim"], s["group"])
        rows.write(s["x"], s["slots"])
        return rows.decode(s["ids"], dtype=TYPES[s["out"]])
    return scoring.adjust(s["x"], bias=s["bias"], allow=s["allow"], allow_rows=s["allow_rows"], seen=s["seen"],
                          seen_starts=s["starts"], repetition=s["repetition"], presence=s["presence"],
                          frequency=s["frequency"], largest=s["largest"])


def _run_plain(s):
    if s["op"] == "int4":
        v = _decode(s["codes"], s["scales"], s["dim"], s["group"])
        return (s["q"].float() @ v.T).to(TYPES[s["out"]])
    if s["op"] == "rows":
        codes, scales = _encode(s["x"], s["group"])
        to, ids = s["slots"].long(), s["ids"].long()
        s["codes"][to], s["scales"][to] = codes, scales
        return _decode(s["codes"][ids], s["scales"][ids], s["dim"], s["group"]).to(TYPES[s["out"]])
    x = s["x"].float()
    nq, n = x.shape
    count = torch.bincount(s["owner"] * n + s["seen"], minlength=nq * n).view(nq, n)
    r = s["repetition"][:, None]
    less = s["presence"][:, None] + s["frequency"][:, None] * count
    if s["largest"]:
        y = torch.where(x > 0, x / r, x * r) - less
    else:
        y = torch.where(x > 0, x * r, x / r) + less
    x = torch.where(count > 0, y, x)
    if s["bias"] is not None:
        x = x + s["bias"]
    j = torch.arange(n, device=DEV)
    rows = s["allow_rows"].long()
    mine = s["allow"][rows.clamp(min=0)]
    allowed = ((mine[:, j // 32] >> (j % 32).int()) & 1).bool() | (rows < 0)[:, None]
    return torch.where(allowed, x, torch.full_like(x, -math.inf if s["largest"] else math.inf)).to(s["x"].dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without --------------------------------------------


def _held(case):
    """Bytes of a row as it is held."""
    return case["dim"] / 2 + 4 * -(-case["dim"] // case["group"])


def work(case):
    if case["op"] == "int4":
        nq, n, dim = case["nq"], case["n"], case["dim"]
        return {"bytes": nq * dim * SIZE[case["query"]] + n * _held(case) + nq * n * SIZE[case["out"]],
                "flops": 2.0 * nq * n * dim}
    if case["op"] == "rows":
        m, reads, dim = case["m"], case["reads"], case["dim"]
        return {"bytes": m * (dim * SIZE[case["type"]] + 4 + _held(case)) +
                reads * (dim * SIZE[case["out"]] + 4 + _held(case)), "flops": 0.0}
    nq, n = case["nq"], case["n"]
    seen = nq * case["seen"] * 2 / 3
    used = min(nq, case["masks"])
    return {"bytes": nq * (2.0 * n * SIZE[case["type"]] + 24) + 4 * seen + used * n / 8 + (4 * n if case["bias"] else 0),
            "flops": 0.0}


# ---- the definitions in 64 bits -----------------------------------------------


def _values(codes, scales, dim, group):
    """The values that rows stand for, one by one from their bytes: value d of a
    row is nibble d % 8 of the word that holds the eight values from 8 (d // 8) on."""
    out = torch.empty(codes.shape[0], dim, dtype=torch.float64, device=codes.device)
    units = (dim + 31) // 32
    for first in range(0, dim, 8):
        block = first // 128
        across = min(4, units - 4 * block)
        at = 64 * block + 4 * (across * (first % 32 // 8) + first % 128 // 32)
        w = scales[:, first // group].long() & 0xFFFFFFFF
        z = ((w & 255) ^ 128) - 128
        exponent, significand = (w >> 23) & 255, ((w & 0x7FFF00) | torch.where(((w >> 23) & 255) > 0, 1 << 23, 0)).double()
        step = significand * _pow2(exponent.clamp(min=1) - 150)
        for d in range(first, min(dim, first + 8)):
            byte = codes[:, at + d % 8 // 2].long()
            out[:, d] = ((byte >> (4 * (d % 2)) & 15) + z).double() * step
    return out


def _nearest(x, group):
    """What rows of x are held as, from the definition."""
    x = x.double()
    out = torch.empty_like(x)
    for first in range(0, x.shape[1], group):
        part = x[:, first:first + group]
        lo, hi = part.min(1, keepdim=True).values, part.max(1, keepdim=True).values
        need = torch.maximum(_over(hi - lo, 15), _over(part.abs().max(1, keepdim=True).values, 127))
        unit = _pow2(torch.floor(torch.log2(need.clamp(min=2.0 ** -126))) - 15)
        unit = torch.where(need >= unit * 65536, unit * 2, torch.where(need < unit * 32768, unit / 2, unit))  # log2 rounds
        unit = unit.clamp(min=2.0 ** -141)
        step = torch.ceil(need / unit) * unit
        some = torch.where(step > 0, step, torch.ones_like(step))
        low = torch.round(lo / some)
        out[:, first:first + group] = torch.minimum(torch.round(part / some), low + 15) * step
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "int4":
        return s["q"].double() @ _values(s["codes"], s["scales"], case["dim"], case["group"]).T
    if case["op"] == "rows":
        held = _values(s["codes"], s["scales"], case["dim"], case["group"])
        held[s["slots"].long()] = _nearest(s["x"], case["group"])
        return held[s["ids"].long()]
    nq, n = case["nq"], case["n"]
    out = torch.empty(nq, n, dtype=torch.float64, device=DEV)
    starts, rows = s["starts"].tolist(), s["allow_rows"].tolist()
    worse = -1.0 if case["largest"] else 1.0
    bit = torch.arange(32, device=DEV)
    for i in range(nq):
        x = s["x"][i].double()
        ids, times = torch.unique(s["seen"][starts[i]:starts[i + 1]].long(), return_counts=True)
        y, r = x[ids], s["repetition"][i].double()
        grows = (y > 0) != case["largest"]
        y = torch.where(grows, y * r, y / r)
        x[ids] = y + worse * (s["presence"][i].double() + s["frequency"][i].double() * times)
        if s["bias"] is not None:
            x += s["bias"].double()
        if rows[i] >= 0:
            keep = ((s["allow"][rows[i]].long()[:, None] >> bit) & 1).reshape(-1)[:n].bool()
            x[~keep] = worse * math.inf
        out[i] = x
    return out
