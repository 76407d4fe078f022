"""Performance cases of the 4-bit KV cache: writing it, reading it back, and decode attention over it.

Format of a row, one (sequence, KV head, token) vector of D elements.  A group of g consecutive elements has two fp16
numbers, a minimum m and a step s, and each element a code n of 4 bits that stands for m + n s:

    lo, hi = min and max of the group, clamped to +-65504
    m = fp16(lo)                                    (to nearest, ties to even)
    s = fp16(max(0, fp32(fp32(hi - m) / 15)))       (towards zero)
    n = round(fp32(fp32(x - m) / s)), at most 15, at least 0; 0 where s = 0

A group that holds a NaN or an infinity has NaN for s and m, and codes 0.  Element 8 p + i is in bits 4 i .. 4 i + 3 of
32-bit word p.  Inside each block of min(D, 128) elements word p stands at place (p % 4) * (block / 32) + p // 4; a row of
16 elements has its two words in order.  The row of s and m is [s0, m0, s1, m1, ...].

Kinds of case:

* ``write``: new tokens quantised into a cache, contiguous or paged, then read back as the values that they stand for, as
  a prompt in chunks does before its attention.
* ``read``: a cached prefix read back for the next chunk of a prompt.
* ``contig``: one decode step's attention over a contiguous cache.
* ``paged``: the same over a paged pool.

A drawn case moves at most the bytes of the largest listed one of its kind.
"""

from __future__ import annotations

import importlib
import math
import random
from types import SimpleNamespace

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
LARGEST = {"write": 0.344e9, "read": 0.415e9, "contig": 0.296e9, "paged": 1.165e9}
MAX_FLOPS = 2.9e10
VECTOR = 0.05e9         # fp32 queries, head_dim below 64, pages that are no whole tiles: calls of small and medium size
F16_MAX = 65504.0


def _sia():
    return importlib.import_module("simple-inference-autoresearch_amd")


# ---------------------------------------------------------------------- cases


def _write(dtype, B, H, D, g, T, page, lo, hi, lens=0):
    return {"kind": "write", "dtype": dtype, "B": B, "H": H, "D": D, "g": g, "T": T, "page": page, "lo": lo, "hi": hi,
            "lens": lens}


def _read(dtype, B, H, D, g, T, page):
    return {"kind": "read", "dtype": dtype, "B": B, "H": H, "D": D, "g": g, "T": T, "page": page}


def _decode(kind, dtype, B, heads, D, g, page, dist, lo, hi, lens=0):
    return {"kind": kind, "dtype": dtype, "B": B, "Hq": heads[0], "H": heads[1], "D": D, "g": g, "page": page,
            "dist": dist, "lo": lo, "hi": hi, "lens": lens}


def listed():
    cases = {
        # the smallest call: one decode step's new token of every request of a serving batch
        "write_step_b32": _write("bf16", 32, 8, 128, 64, 1, 16, 100, 4000, 1),
        # one user's prompt of ordinary, odd length into a contiguous cache, small groups
        "write_prompt_1500": _write("bf16", 1, 8, 128, 32, 1500, 0, 0, 0),
        # a batch of long fp16 prompts of a head_dim-64 model into a paged pool
        "write_prompts_8k_d64": _write("fp16", 4, 16, 64, 64, 8192, 16, 0, 0),
        # the next turn of a conversation: its prefix of ordinary length read back
        "read_prefix_1000": _read("bf16", 1, 8, 128, 64, 1000, 0),
        # the prefixes of a batch of a head_dim-256 model, from pages of 32 tokens
        "read_prefix_b16_d256": _read("bf16", 16, 4, 256, 128, 5000, 32),
        # interactive generation: one sequence over a cache of ordinary length
        "contig_b1_1000": _decode("contig", "bf16", 1, (32, 8), 128, 64, 0, "equal", 1000, 1000),
        # a batch of a head_dim-256 model at a long context
        "contig_b32_8k_d256": _decode("contig", "bf16", 32, (16, 4), 256, 64, 0, "equal", 8000, 8000),
        # an fp32 query, as an accuracy evaluation runs it, one request empty
        "contig_fp32_b4": _decode("contig", "fp32", 4, (32, 8), 64, 32, 0, "uniform", 0, 512, 3),
        # a full decode batch at one long context: the headline shape of the benchmark
        "paged_b64_8k": _decode("paged", "bf16", 64, (32, 8), 128, 64, 16, "equal", 8192, 8192),
        # a large serving batch with the lengths of live traffic, small groups
        "paged_b256_lognormal": _decode("paged", "bf16", 256, (64, 8), 128, 32, 16, "lognormal", 128, 32768, 4),
        # ragged fp16 requests of a head_dim-64 model with one KV head per query head, one of them empty
        "paged_fp16_b16_d64": _decode("paged", "fp16", 16, (16, 16), 64, 32, 16, "uniform", 0, 4096, 1),
        # a pool whose pages are no whole tiles of 16 tokens
        "paged_b4_page24": _decode("paged", "bf16", 4, (12, 4), 128, 128, 24, "uniform", 40, 2000, 2),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    """A whole number between lo and hi, spread evenly over the logarithm."""
    return max(int(lo), min(int(hi), round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _vector(c) -> bool:
    return c["dtype"] == "fp32" or c["D"] < 64 or (c["page"] not in (0, 16, 32, 64))


def draw(rng):
    while True:
        c = _draw(rng)
        most = LARGEST[c["kind"]]
        if c["kind"] in ("contig", "paged") and _vector(c):
            most = min(most, VECTOR)
        w = work(c)
        if w["bytes"] <= most and w["flops"] <= MAX_FLOPS and _state_bytes(c) <= 4e9:
            return c


def _draw(rng):
    kind = rng.choice(["write", "read", "contig", "paged", "paged"])
    D = rng.choice([16, 32, 64, 64, 128, 128, 128, 256])
    g = min(D, rng.choice([32, 64, 64, 128]))
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    page = rng.choice([16, 16, 32, 64, 24, 8])
    H = rng.choice([1, 2, 4, 8, 8, 16])
    lens = rng.randrange(1 << 20)
    if kind == "write":
        page = rng.choice([0, page])
        lo = _log(rng, 1, 4096) - 1
        return _write(dtype, _log(rng, 1, 64), H, D, g, rng.choice([1, _log(rng, 2, 8192)]), page, lo,
                      lo + rng.randint(0, 2000), lens)
    if kind == "read":
        return _read(rng.choice(["bf16", "fp16", "fp32"]), _log(rng, 1, 64), H, D, g, _log(rng, 1, 16384),
                     rng.choice([0, page]))
    heads = rng.choice([(32, 8), (64, 8), (16, 4), (12, 4), (16, 16), (8, 2), (5, 1), (40, 2)])
    dist = rng.choice(["equal", "uniform", "lognormal"])
    lo = _log(rng, 1, 8192)
    hi = lo if dist == "equal" else min(32768, lo * rng.randint(2, 16))
    if dist == "uniform" and rng.random() < 0.3:
        lo = 0
    return _decode(kind, dtype, _log(rng, 1, 256 if kind == "paged" else 32), heads, D, g, page if kind == "paged" else 0,
                   dist, lo, hi, lens)


def _row_bytes(c) -> float:
    return c["D"] / 2 + 4 * c["D"] / c["g"]


def _state_bytes(c) -> float:
    if c["kind"] in ("write", "read"):
        return 2.0 * c["B"] * c["H"] * (c["T"] * c["D"] * 4 + (c["T"] + c.get("hi", 0)) * _row_bytes(c))
    return 2.0 * c["B"] * c["H"] * c["hi"] * _row_bytes(c)


def _lengths(c):
    """Context length of every sequence, or the first position of a write (a fixed function of the case)."""
    B, lo, hi = c["B"], c["lo"], c["hi"]
    g = torch.Generator().manual_seed(c["lens"])
    dist = c.get("dist", "uniform")
    if dist == "equal" or lo == hi:
        return [lo] * B
    if dist == "uniform":
        n = torch.randint(max(lo, 1), hi + 1, (B,), generator=g).tolist()
        if lo == 0 and B > 1:
            n[B // 2] = 0
        return n
    # log-normal around the geometric middle of [lo, hi]: most requests near it, a few close to hi
    z = torch.randn(B, generator=g, dtype=torch.float64)
    mid = 0.5 * (math.log(lo) + math.log(hi))
    sigma = (math.log(hi) - math.log(lo)) / 5.5
    return [int(x) for x in torch.exp(mid + sigma * z).round().clamp(lo, hi).tolist()]


def work(case):
    c = case
    if c["kind"] in ("write", "read"):
        rows = 2.0 * c["B"] * c["H"] * c["T"]
        es = 4 if c["dtype"] == "fp32" else 2
        # a write reads its source and writes the rows; its values are read back from them and written out
        passes = 2 if c["kind"] == "write" else 1
        return {"bytes": passes * rows * (c["D"] * es + _row_bytes(c)), "flops": rows * c["D"] * 4.0 * passes}
    tokens = float(sum(_lengths(c)))
    es = 4 if c["dtype"] == "fp32" else 2
    kv = tokens * c["H"] * 2 * _row_bytes(c)
    return {"bytes": kv + 2.0 * c["B"] * c["Hq"] * c["D"] * es, "flops": 4.0 * tokens * c["Hq"] * c["D"]}


# --------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _values(g, rows, D):
    """fp32 rows as a projection leaves them: normal, with channels of different spread and offset."""
    spread = torch.exp(0.4 * torch.randn(D, generator=g, device="cuda"))
    offset = 0.5 * torch.randn(D, generator=g, device="cuda")
    return torch.randn(rows, D, generator=g, device="cuda") * spread + offset


def _tensor(g, shape, dtype):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1, shape[-1])
    step = max(1, (1 << 26) // shape[-1])
    for i in range(0, flat.shape[0], step):
        flat[i:i + step] = _values(g, min(step, flat.shape[0] - i), shape[-1])
    return out


def _cache(g, shape, group):
    """Codes and parameters of a cache (..., D) that holds such rows."""
    D = shape[-1]
    codes = torch.empty(shape[:-1] + (D // 2,), dtype=torch.uint8, device="cuda")
    params = torch.empty(shape[:-1] + (2 * D // group,), dtype=torch.float16, device="cuda")
    c, p = codes.view(-1, D // 2), params.view(-1, 2 * D // group)
    step = max(1, (1 << 25) // D)
    for i in range(0, c.shape[0], step):
        c[i:i + step], p[i:i + step] = _quantise(_values(g, min(step, c.shape[0] - i), D), group)
    return codes, params


def _table(pages, seed):
    """Block table of requests with these page counts: their pages anywhere in the pool."""
    P = max(1, sum(pages))
    perm = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    bt = torch.zeros(len(pages), max(1, max(pages)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        bt[b, :n] = perm[at:at + n]
        at += n
    return bt.cuda(), P


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    B, H, D, group, page = c["B"], c["H"], c["D"], c["g"], c["page"]
    s = SimpleNamespace(case=c, bt=None, start=None)
    if c["kind"] == "write":
        T, dtype = c["T"], DTYPES[c["dtype"]]
        first = _lengths(c)
        cap = max(first) + T
        # token-major, as the projection leaves them
        s.k, s.v = (_tensor(g, (B, T, H, D), dtype).transpose(1, 2) for _ in range(2))
        if page:
            s.bt, P = _table([-(-(n + T) // page) for n in first], int(seed))
            shape = (P, H, page)
        else:
            shape = (B, H, cap)
        s.start = torch.tensor(first, dtype=torch.int32, device="cuda")
        s.kc, s.vc = (torch.zeros(shape + (D // 2,), dtype=torch.uint8, device="cuda") for _ in range(2))
        s.ks, s.vs = (torch.zeros(shape + (2 * D // group,), dtype=torch.float16, device="cuda") for _ in range(2))
        return s
    ctx = [c["T"]] * B if c["kind"] == "read" else _lengths(c)
    if page:
        s.bt, P = _table([-(-n // page) for n in ctx], int(seed))
        shape = (P, H, page, D)
    else:
        shape = (B, H, max(1, max(ctx)), D)
    s.kc, s.ks = _cache(g, shape, group)
    s.vc, s.vs = _cache(g, shape, group)
    if c["kind"] != "read":
        s.ctx = ctx
        s.q = torch.randn(B, c["Hq"], 1, D, generator=g, device="cuda").to(DTYPES[c["dtype"]])
        s.kv_len = torch.tensor(ctx[:1] if c["dist"] == "equal" else ctx, dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------- the operators' plain form


def _word_places(D):
    """Place of word p (elements 8 p .. 8 p + 7) in a row of codes, for every p."""
    if D == 16:
        return [0, 1]
    block = min(D, 128)
    n = block // 8
    return [(w // n) * n + (w % n % 4) * (block // 32) + w % n // 4 for w in range(D // 8)]


def _quantise(x, group):
    """Rows (n, D) of fp32 values -> codes (n, D / 2) uint8, parameters (n, 2 D / group) fp16."""
    n, D = x.shape
    x = x.view(n, D // group, group)
    bad = ~torch.isfinite(x).all(dim=-1)
    xc = x.clamp(-F16_MAX, F16_MAX)
    lo, hi = xc.amin(dim=-1), xc.amax(dim=-1)
    m = lo.half()
    step = ((hi - m.float()).double() / 15).float().clamp_min(0.0)     # (a quotient in 64 bits rounds to fp32's own)
    s = step.half()
    s = torch.where(s.float() > step, (s.view(torch.int16) - 1).view(torch.float16), s)
    sf = s.float()[..., None]
    t = (xc - m.float()[..., None]).double() / sf.double()
    code = torch.where(sf > 0, t.float().round().clamp(0, 15), torch.zeros_like(xc))
    code = torch.where(bad[..., None], torch.zeros_like(code), code).to(torch.uint8).view(n, D // 8, 8)
    nan = torch.full_like(m, float("nan"))
    params = torch.stack([torch.where(bad, nan, s), torch.where(bad, nan, m)], dim=-1).view(n, 2 * D // group)
    words = torch.empty_like(code)
    words[:, _word_places(D)] = code
    words = words.view(n, D // 2, 2)
    return words[..., 0] | (words[..., 1] << 4), params


def _values_of(codes, params):
    """The fp32 values that codes (..., D / 2) and parameters (..., 2 D / g) stand for."""
    D = codes.shape[-1] * 2
    lead = codes.shape[:-1]
    n = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(lead + (D // 8, 8))[..., _word_places(D), :]
    p = params.float().view(lead + (params.shape[-1] // 2, 2))
    n = n.reshape(lead + (p.shape[-2], -1)).float()
    return (p[..., 1:] + n * p[..., :1]).reshape(lead + (D,))


def _slots(s, positions):
    """Index pair (first, third dimension of the cache) of positions (B, T)."""
    c = s.case
    if s.bt is None:
        return torch.arange(c["B"], device="cuda")[:, None].expand_as(positions), positions
    return s.bt.gather(1, positions // c["page"]).long(), positions % c["page"]


def _plain_write(s):
    c = s.case
    B, H, T, D = c["B"], c["H"], c["T"], c["D"]
    a, b = _slots(s, s.start.long()[:, None] + torch.arange(T, device="cuda"))
    out = []
    for x, codes, params in ((s.k, s.kc, s.ks), (s.v, s.vc, s.vs)):
        xt = x.transpose(1, 2).reshape(B * T * H, D).float()
        qc, qp = _quantise(xt, c["g"])
        codes[a, :, b] = qc.view(B, T, H, -1)
        params[a, :, b] = qp.view(B, T, H, -1)
        out.append(_values_of(codes[a, :, b], params[a, :, b]).transpose(1, 2).to(x.dtype))
    return tuple(out)


def _plain_read(s):
    c = s.case
    a, b = _slots(s, torch.arange(c["T"], device="cuda").expand(c["B"], -1))
    return tuple(_values_of(codes[a, :, b], params[a, :, b]).transpose(1, 2).to(DTYPES[c["dtype"]])
                 for codes, params in ((s.kc, s.ks), (s.vc, s.vs)))


def _sequence(s, codes, params, b, n):
    """Codes and parameters (H, n, ...) of the first n tokens of sequence b."""
    if s.bt is None:
        return codes[b, :, :n], params[b, :, :n]
    pages = s.bt[b, :-(-n // s.case["page"])].long()
    return tuple(t[pages].transpose(0, 1).flatten(1, 2)[:, :n] for t in (codes, params))


def _plain_decode(s):
    c = s.case
    B, Hq, H, D = c["B"], c["Hq"], c["H"], c["D"]
    out = torch.zeros(B, 1, Hq, D, dtype=torch.float32, device="cuda")
    for b, n in enumerate(s.ctx):
        if n == 0:
            continue
        k = _values_of(*_sequence(s, s.kc, s.ks, b, n))
        v = _values_of(*_sequence(s, s.vc, s.vs, b, n))
        q = s.q[b, :, 0].float().view(H, Hq // H, D)
        score = torch.matmul(q, k.transpose(1, 2).contiguous()) * D ** -0.5
        p = torch.exp(score - score.amax(dim=-1, keepdim=True))
        out[b, 0] = (torch.matmul(p, v) / p.sum(dim=-1, keepdim=True)).view(Hq, D)
    return out.to(s.q.dtype)


def run(state):
    s = state
    kind = s.case["kind"]
    if not own:
        return {"write": _plain_write, "read": _plain_read}.get(kind, _plain_decode)(s)
    sia, c = _sia(), s.case
    if kind == "write":
        sia.kv_write(s.k, s.v, s.kc, s.vc, s.ks, s.vs, block_table=s.bt, start_pos=s.start, page_size=c["page"])
        return sia.kv_read(s.kc, s.vc, c["T"], s.ks, s.vs, block_table=s.bt, start_pos=s.start, page_size=c["page"],
                           dtype=s.k.dtype)
    if kind == "read":
        return sia.kv_read(s.kc, s.vc, c["T"], s.ks, s.vs, block_table=s.bt, page_size=c["page"], dtype=DTYPES[c["dtype"]])
    if kind == "contig":
        return sia.attention_flash_decode_int4(s.q, s.kc, s.vc, s.ks, s.vs, s.kv_len)
    return sia.paged_gqa_int4_flash_decode(s.q, s.kc, s.vc, s.ks, s.vs, s.bt, s.kv_len, c["page"])


# --------------------------------------------------- the definition, in 64 bits


def _exact_values(codes, params):
    """Values m + n s in 64 bits: nibble i of stored word w belongs to element 8 p + i, p the word whose place is w."""
    D = codes.shape[-1] * 2
    place = _word_places(D)
    at = [4 * place[e // 8] + (e % 8) // 2 for e in range(D)]
    shift = torch.tensor([4 * (e % 2) for e in range(D)], dtype=torch.uint8, device=codes.device)
    n = ((codes[..., at] >> shift) & 15).double()
    group = 2 * D // params.shape[-1]
    which = [e // group for e in range(D)]
    p = params.double()
    return p[..., 1::2][..., which] + n * p[..., 0::2][..., which]


def _exact_round(x, group):
    """What rows x (..., D) in 64 bits are held as."""
    shape = x.shape
    x = x.reshape(-1, group)
    finite = torch.isfinite(x).all(dim=1)
    x = x.clamp(-F16_MAX, F16_MAX)
    m = x.min(dim=1).values.half().double()
    step = ((x.max(dim=1).values - m).float().double() / 15).float().double().clamp_min(0.0)
    e = torch.frexp(step).exponent.clamp_min(-13).double() - 11       # the spacing of fp16 at the step is 2^e
    s = torch.floor(step * torch.exp2(-e)) * torch.exp2(e)
    t = ((x - m[:, None]).float().double() / torch.where(s > 0, s, torch.ones_like(s))[:, None]).float().double()
    y = m[:, None] + torch.where((s > 0)[:, None], torch.round(t).clamp(0, 15), torch.zeros_like(t)) * s[:, None]
    y[~finite] = float("nan")
    return y.reshape(shape)


def exact(case, seed):
    s = prepare(case, seed)
    c = s.case
    if c["kind"] == "write":
        return tuple(torch.cat([_exact_round(x[b:b + 1].double(), c["g"]) for b in range(c["B"])]) for x in (s.k, s.v))
    if c["kind"] == "read":
        out = []
        for codes, params in ((s.kc, s.ks), (s.vc, s.vs)):
            out.append(torch.stack([_exact_values(*_sequence(s, codes, params, b, c["T"])) for b in range(c["B"])]))
        return tuple(out)
    B, Hq, H, D = c["B"], c["Hq"], c["H"], c["D"]
    out = torch.zeros(B, 1, Hq, D, dtype=torch.float64, device="cuda")
    per = Hq // H
    for b, n in enumerate(s.ctx):
        if n == 0:
            continue
        ck, pk = _sequence(s, s.kc, s.ks, b, n)
        cv, pv = _sequence(s, s.vc, s.vs, b, n)
        for h in range(H):
            k, v = _exact_values(ck[h], pk[h]), _exact_values(cv[h], pv[h])
            q = s.q[b, h * per:(h + 1) * per, 0].double()
            w = torch.softmax(torch.mm(k, q.t().contiguous()) / math.sqrt(D), dim=0)
            out[b, 0, h * per:(h + 1) * per] = torch.mm(w.t().contiguous(), v)
    return out
