"""Performance cases of attention with a score function, for prompts and single tokens, and of rotary positions from frequencies.

A query at position p of its row sees key j, in the sequence b and the query head h, with the score

    s = sm_scale q . k        (sm_scale = 1 / sqrt(D))
    s = c tanh(s / c)         where the scores are capped by c
    s = s - slope_h |p - j|   where they get a bias that depends on distance

where  start_b <= j < len_b,  p and j lie in the same document (no boundary x with min(p, j) < x <= max(p, j)),
|p - j| < W where there is a window, and, in a causal call, j <= p or j < prefix_b.  The output is the softmax of the
visible scores times V, and zero for a query that sees no key.

Rotary positions turn the pairs of the first R elements of a head, (i, i + R/2) or (2 i, 2 i + 1), by the angle
position x frequency_i and stretch them by a factor; the elements from R on stay as they are.

Kinds of case:

* ``prompt``: the attention of prompts, or of chunks of prompts behind a cached prefix (query i at position Tk - Tq + i).
* ``step``: the attention of one decode step over a contiguous cache or a paged pool, 16-bit, fp32 or int8 with a scale
  per token and head (query at position len_b - 1).
* ``rope``: q and k of a prompt or a decode step rotated.

A drawn case costs at most what the largest listed one of its kind does.
"""

from __future__ import annotations

import importlib
import math
import random
from types import SimpleNamespace

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
PROMPT_FLOPS = {"bf16": 1.38e11, "fp16": 1.38e11, "fp32": 4.0e9}
STEP_BYTES = 0.56e9
VECTOR_BYTES = 0.04e9      # fp32, head_dim below 64, pages that are no whole tiles: calls of small and medium size
ROPE_BYTES = 0.17e9


def _sia():
    return importlib.import_module("simple-inference-autoresearch_amd")


# ---------------------------------------------------------------------- cases


def _prompt(dtype, B, heads, D, Tq, Tk, causal=True, cap=0.0, alibi=False, window=0, docs=0, prefix=0, pad=0, lens=0):
    return {"kind": "prompt", "dtype": dtype, "B": B, "Hq": heads[0], "H": heads[1], "D": D, "Tq": Tq, "Tk": Tk,
            "causal": causal, "cap": cap, "alibi": alibi, "window": window, "docs": docs, "prefix": prefix, "pad": pad,
            "lens": lens}


def _step(dtype, cache, B, heads, D, page, dist, lo, hi, cap=0.0, alibi=False, window=0, start=False, lens=0):
    return {"kind": "step", "dtype": dtype, "cache": cache, "B": B, "Hq": heads[0], "H": heads[1], "D": D, "page": page,
            "dist": dist, "lo": lo, "hi": hi, "cap": cap, "alibi": alibi, "window": window, "start": start, "lens": lens}


def _rope(dtype, B, T, heads, D, R, pairs, scaling, first, docs=0, lens=0):
    return {"kind": "rope", "dtype": dtype, "B": B, "T": T, "Hq": heads[0], "H": heads[1], "D": D, "R": R, "pairs": pairs,
            "scaling": scaling, "first": first, "docs": docs, "lens": lens}


def listed():
    cases = {
        # a batch of prompts of a model with capped scores: the headline shape of the prefill benchmark
        "prompt_capped_b4_2048": _prompt("bf16", 4, (32, 8), 128, 2048, 2048, cap=50.0),
        # a long prompt in a layer with a sliding window, head_dim 256
        "prompt_window_8k_d256": _prompt("bf16", 1, (16, 4), 256, 8192, 8192, window=1024),
        # two ordinary fp16 prompts of odd length with a bias by distance, one KV head per query head
        "prompt_alibi_b2_1000": _prompt("fp16", 2, (16, 16), 64, 1000, 1000, alibi=True),
        # documents packed into one row, as evaluation and scoring of a corpus run them
        "prompt_documents_16k": _prompt("bf16", 1, (32, 8), 128, 16384, 16384, docs=24, lens=1),
        # a right-padded batch of ragged requests whose prefixes see each other in both directions
        "prompt_prefix_b8_700": _prompt("fp16", 8, (12, 4), 128, 700, 700, prefix=400, pad=500, lens=2),
        # an fp32 chunk behind a cached prefix, as an accuracy evaluation runs it, capped and in a window
        "prompt_fp32_b1_333": _prompt("fp32", 1, (32, 8), 64, 333, 1000, cap=30.0, window=500),
        # interactive generation: one sequence over a cache of ordinary length, capped scores
        "step_b1_1000": _step("bf16", "same", 1, (32, 8), 128, 0, "equal", 1000, 1000, cap=50.0),
        # a full decode batch over int8 pools in a layer with a sliding window and capped scores
        "step_paged_int8_b64_8k": _step("bf16", "int8", 64, (32, 8), 128, 16, "equal", 8192, 8192, cap=50.0, window=4096),
        # ragged fp16 requests with a bias by distance, one of them empty
        "step_paged_alibi_b16": _step("fp16", "same", 16, (16, 16), 64, 16, "uniform", 0, 4096, alibi=True, lens=3),
        # a left-padded batch at a long context, head_dim 256
        "step_padded_b32_d256": _step("bf16", "same", 32, (16, 4), 256, 0, "equal", 8000, 8000, start=True, lens=4),
        # one decode step's tokens of a serving batch, half of each head rotated
        "rope_step_b64": _rope("bf16", 64, 1, (32, 8), 128, 64, "half", "none", 5000),
        # a long prompt at scaled frequencies, interleaved pairs
        "rope_prompt_8k": _rope("bf16", 1, 8192, (32, 8), 128, 128, "interleaved", "yarn", 100000),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    """A whole number between lo and hi, spread evenly over the logarithm."""
    return max(int(lo), min(int(hi), round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if c["kind"] == "prompt" and w["flops"] <= PROMPT_FLOPS[c["dtype"]] and c["B"] * c["Hq"] * c["Tk"] <= 1 << 20:
            return c
        if c["kind"] == "rope" and w["bytes"] <= ROPE_BYTES:
            return c
        vector = c["dtype"] == "fp32" or c["D"] < 64 or c.get("page") not in (0, 16, 32, 64)
        if c["kind"] == "step" and _state_bytes(c) <= (VECTOR_BYTES if vector else 2 * STEP_BYTES) and w["bytes"] <= STEP_BYTES:
            return c


def _draw(rng):
    kind = rng.choice(["prompt", "prompt", "step", "step", "rope"])
    heads = rng.choice([(32, 8), (64, 8), (16, 4), (12, 4), (16, 16), (8, 2), (5, 1), (40, 2)])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    lens = rng.randrange(1 << 20)
    shape = rng.choice(["cap", "alibi", "window", "cap window", "alibi window", "cap alibi"])
    more = {"cap": rng.choice([20.0, 30.0, 50.0]) if "cap" in shape else 0.0, "alibi": "alibi" in shape,
            "window": _log(rng, 1, 4096) if "window" in shape else 0, "lens": lens}
    if kind == "prompt":
        Tq = _log(rng, 1, 8192)
        Tk = Tq if rng.random() < 0.6 else Tq + _log(rng, 1, 8192)
        which = rng.choice(["", "docs", "prefix", "pad"])
        return _prompt(dtype, _log(rng, 1, 16), heads, rng.choice([16, 32, 64, 64, 128, 128, 128, 256]), Tq, Tk,
                       causal=rng.random() < 0.8, docs=_log(rng, 2, 64) if which == "docs" else 0,
                       prefix=rng.randint(1, Tk) if which == "prefix" else 0,
                       pad=rng.randint(0, Tk) if which in ("prefix", "pad") else 0, **more)
    if kind == "step":
        page = rng.choice([0, 0, 16, 16, 32, 64, 24, 8])
        dist = rng.choice(["equal", "uniform", "lognormal"])
        lo = _log(rng, 1, 8192)
        hi = lo if dist == "equal" else min(32768, lo * rng.randint(2, 16))
        if dist == "uniform" and rng.random() < 0.3:
            lo = 0
        return _step(dtype, rng.choice(["same", "same", "int8"]), _log(rng, 1, 256 if page else 32), heads,
                     rng.choice([16, 32, 64, 64, 128, 128, 128, 256]), page, dist, lo, hi, start=rng.random() < 0.3, **more)
    D = rng.choice([64, 128, 128, 256])
    T = rng.choice([1, _log(rng, 2, 8192)])
    return _rope(dtype, _log(rng, 1, 64), T, heads, D, rng.choice([D, D // 2, D // 4, 32, 24]), rng.choice(["half", "interleaved"]),
                 rng.choice(["none", "linear", "ntk", "yarn"]), _log(rng, 1, 1000000) - 1, docs=rng.choice([0, 3]) if T > 8 else 0,
                 lens=lens)


def _state_bytes(c) -> float:
    return 2.0 * c["B"] * c["H"] * c["hi"] * c["D"] * (1 if c["cache"] == "int8" else 4 if c["dtype"] == "fp32" else 2)


def _lengths(c):
    """Context length of every sequence of a decode step (a fixed function of the case)."""
    B, lo, hi = c["B"], c["lo"], c["hi"]
    g = torch.Generator().manual_seed(c["lens"])
    if c["dist"] == "equal" or lo == hi:
        return [lo] * B
    if c["dist"] == "uniform":
        n = torch.randint(max(lo, 1), hi + 1, (B,), generator=g).tolist()
        if lo == 0 and B > 1:
            n[B // 2] = 0
        return n
    # log-normal around the geometric middle of [lo, hi]: most requests near it, a few close to hi
    z = torch.randn(B, generator=g, dtype=torch.float64)
    mid = 0.5 * (math.log(lo) + math.log(hi))
    sigma = (math.log(hi) - math.log(lo)) / 5.5
    return [int(x) for x in torch.exp(mid + sigma * z).round().clamp(lo, hi).tolist()]


def _starts(c):
    """First visible token of every sequence of a decode step: the padding in front of it, up to half of the row."""
    if not c["start"]:
        return [0] * c["B"]
    g = torch.Generator().manual_seed(c["lens"] + 1)
    return (torch.tensor(_lengths(c)) * 0.5 * torch.rand(c["B"], generator=g)).long().tolist()


def _cuts(c, T):
    """Boundaries 0 .. T of c["docs"] documents of log-normal length."""
    g = torch.Generator().manual_seed(c["lens"])
    w = torch.exp(0.8 * torch.randn(c["docs"], generator=g, dtype=torch.float64)).cumsum(0)
    return [0] + [int(x) for x in (w / w[-1] * T).round().tolist()]


def _rows(c):
    """(start, length, prefix) of every sequence of a prompt: padded on the right, in every third row on the left."""
    g = torch.Generator().manual_seed(c["lens"] + 2)
    out = []
    for b in range(c["B"]):
        n = c["Tk"] - int(torch.randint(0, c["pad"] + 1, (1,), generator=g)) if c["pad"] else c["Tk"]
        n = max(1, n)
        prefix = int(torch.randint(0, c["prefix"] + 1, (1,), generator=g)) if c["prefix"] else 0
        out.append((c["Tk"] - n, c["Tk"], prefix) if c["pad"] and b % 3 == 2 else (0, n, prefix))
    return out


def _pairs(c) -> float:
    """Visible (query, key) pairs of one query head, over the batch."""
    off, total = c["Tk"] - c["Tq"], 0.0
    p = torch.arange(off, c["Tk"])
    dlo, dhi = torch.zeros_like(p), torch.full_like(p, c["Tk"])
    if c["docs"]:
        cuts = torch.tensor(_cuts(c, c["Tk"])).unique()
        at = torch.searchsorted(cuts, p, right=True)
        dlo, dhi = cuts[at - 1], cuts[at.clamp(max=len(cuts) - 1)]
    for start, n, prefix in _rows(c):
        lo, hi = dlo.clamp(min=start), dhi.clamp(max=n)
        if c["causal"]:
            hi = torch.minimum(hi, (p + 1).clamp(min=prefix))
        if c["window"]:
            lo, hi = torch.maximum(lo, p - c["window"] + 1), torch.minimum(hi, p + c["window"])
        total += float((hi - lo).clamp(min=0).sum())
    return total


def work(case):
    c = case
    es = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "prompt":
        return {"bytes": 2.0 * c["B"] * c["D"] * es * (c["Hq"] * c["Tq"] + c["H"] * c["Tk"]),
                "flops": 4.0 * c["D"] * c["Hq"] * _pairs(c)}
    if c["kind"] == "rope":
        n = float(c["B"]) * c["T"] * (c["Hq"] + c["H"])
        return {"bytes": 2.0 * n * c["D"] * es, "flops": 3.0 * n * c["R"]}
    tokens = 0.0
    for n, s in zip(_lengths(c), _starts(c)):
        tokens += max(0, n - max(s, n - c["window"] if c["window"] else 0))
    row = c["D"] + (2 if c["page"] == 0 else 4) if c["cache"] == "int8" else c["D"] * es
    return {"bytes": 2.0 * tokens * c["H"] * row + 2.0 * c["B"] * c["Hq"] * c["D"] * es,
            "flops": 4.0 * tokens * c["Hq"] * c["D"]}


# --------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _values(g, rows, D, dtype):
    """Rows as a projection leaves them: normal, with channels of different spread and offset."""
    spread = torch.exp(0.4 * torch.randn(D, generator=g, device="cuda"))
    offset = 0.3 * torch.randn(D, generator=g, device="cuda")
    out = torch.empty(rows, D, dtype=dtype, device="cuda")
    step = max(1, (1 << 26) // D)
    for i in range(0, rows, step):
        n = min(step, rows - i)
        out[i:i + n] = torch.randn(n, D, generator=g, device="cuda") * spread + offset
    return out


def _cache(g, shape, c):
    """K or V rows of a cache and the scales of an int8 one: fp16 in a contiguous cache, fp32 in pools."""
    D = shape[-1]
    n = math.prod(shape[:-1])
    if c["cache"] == "same":
        return _values(g, n, D, DTYPES[c["dtype"]]).view(shape), None
    codes = torch.empty(n, D, dtype=torch.int8, device="cuda")
    scale = torch.empty(n, dtype=torch.float32 if c["page"] else torch.float16, device="cuda")
    step = max(1, (1 << 25) // D)
    for i in range(0, n, step):
        x = _values(g, min(step, n - i), D, torch.float32)
        s = (x.abs().amax(dim=-1) / 127).to(scale.dtype)
        scale[i:i + step] = s
        codes[i:i + step] = (x / s.float()[:, None]).round().clamp(-127, 127).to(torch.int8)
    return codes.view(shape), scale.view(shape[:-1])


def _slopes(c):
    n = c["Hq"]
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / n) for h in range(n)], device="cuda") if c["alibi"] else None


def _frequencies(c):
    """Frequencies of the pairs, fp64, and the factor, at 8 times the context that a model of 8192 positions had."""
    R, theta, factor, L = c["R"], 10000.0, 8.0, 8192
    i = torch.arange(R // 2, dtype=torch.float64)
    scale = 1.0
    if c["scaling"] == "ntk" and R > 2:
        theta *= factor ** (R / (R - 2))
    f = theta ** (-2.0 * i / R)
    if c["scaling"] == "linear":
        f = f / factor
    if c["scaling"] == "yarn":
        low, high = (R * math.log(L / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), R // 2 - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        scale = 0.1 * math.log(factor) + 1.0
    return f, scale


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    B, Hq, H, D, dtype = c["B"], c["Hq"], c["H"], c["D"], DTYPES[c["dtype"]]
    s = SimpleNamespace(case=c)
    if c["kind"] == "rope":
        T = c["T"]
        # q and k as the fused projection leaves them, V behind them
        qkv = _values(g, B * T * (Hq + 2 * H), D, dtype).view(B, T, Hq + 2 * H, D)
        s.q, s.k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + H]
        pos = torch.arange(T).expand(B, T)
        if c["docs"]:
            cuts = torch.tensor(_cuts(c, T)).unique()
            pos = pos - cuts[torch.searchsorted(cuts, pos.contiguous(), right=True) - 1]
        else:
            pos = pos + c["first"] + torch.arange(B)[:, None] * 17
        s.pos = pos.to(torch.int32).contiguous().cuda()
        f, s.scale = _frequencies(c)
        s.freq = f.cuda()
        return s
    s.slopes = _slopes(c)
    if c["kind"] == "prompt":
        Tq, Tk = c["Tq"], c["Tk"]
        # token-major, as the projection leaves them; larger queries, so that the cap counts
        s.q = (_values(g, B * Tq * Hq, D, torch.float32) * 2).to(dtype).view(B, Tq, Hq, D).transpose(1, 2)
        s.k, s.v = (_values(g, B * Tk * H, D, dtype).view(B, Tk, H, D).transpose(1, 2) for _ in range(2))
        rows = _rows(c)
        s.start, s.len, s.prefix = (torch.tensor([r[i] for r in rows], dtype=torch.int32, device="cuda") for i in range(3))
        s.cuts = _cuts(c, Tk) if c["docs"] else [0, Tk]
        s.boundaries = torch.tensor(s.cuts, dtype=torch.int32, device="cuda") if c["docs"] else None
        return s
    s.ctx, page = _lengths(c), c["page"]
    s.bt = None
    if page:
        pages = [-(-n // page) for n in s.ctx]
        P = max(1, sum(pages))
        perm = torch.randperm(P, generator=torch.Generator().manual_seed(int(seed))).to(torch.int32)
        bt, at = torch.zeros(B, max(1, max(pages)), dtype=torch.int32), 0
        for b, n in enumerate(pages):
            bt[b, :n] = perm[at:at + n]
            at += n
        s.bt, shape = bt.cuda(), (P, H, page, D)
    else:
        shape = (B, H, max(1, max(s.ctx)), D)
    s.k, s.ks = _cache(g, shape, c)
    s.v, s.vs = _cache(g, shape, c)
    s.q = (torch.randn(B, Hq, 1, D, generator=g, device="cuda") * 2).to(dtype)
    s.kv_len = torch.tensor(s.ctx[:1] if c["dist"] == "equal" else s.ctx, dtype=torch.int32, device="cuda")
    s.first = _starts(c)
    s.start = torch.tensor(s.first, dtype=torch.int32, device="cuda") if c["start"] else None
    return s


# ------------------------------------------------------- the operators' plain form


def _attend(q, k, v, p, j, c, slopes, visible):
    """Queries (H, G, Tq, D) at positions p over keys (H, Tk, D) at positions j, all fp32 -> (H, G, Tq, D)."""
    H, G, Tq, D = q.shape
    score = torch.matmul(q.reshape(H, G * Tq, D), k.transpose(1, 2).contiguous()).mul_(D ** -0.5)
    if c["cap"]:
        score.div_(c["cap"]).tanh_().mul_(c["cap"])
    score = score.view(H, G, Tq, -1)
    if slopes is not None:
        score -= slopes.view(H, G, 1, 1) * (p[:, None] - j).abs().float()
    score.masked_fill_(~visible, float("-inf"))
    top = score.amax(dim=-1, keepdim=True)
    w = score.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = w.sum(dim=-1, keepdim=True)
    out = torch.matmul(w.view(H, G * Tq, -1), v).view(H, G, Tq, D)
    return out / torch.where(total == 0, torch.ones_like(total), total)


def _plain_prompt(s):
    c = s.case
    B, Hq, H, D, Tq, Tk = (c[x] for x in ("B", "Hq", "H", "D", "Tq", "Tk"))
    off, W = Tk - Tq, c["window"]
    out = torch.empty(B, Tq, Hq, D, dtype=s.q.dtype, device="cuda")
    rows = max(1, min(Tq, (1 << 28) // (Hq * Tk)))                    # queries at a time
    for b in range(B):
        q, k, v = s.q[b].float().view(H, Hq // H, Tq, D), s.k[b].float(), s.v[b].float()
        for a, e in zip(s.cuts, s.cuts[1:]):                          # (one document at a time)
            for i in range(max(a - off, 0), e - off, rows):
                n = min(rows, e - off - i)
                x = max(a, off + i - W + 1) if W else a
                y = min(e, off + i + n - 1 + W) if W else e
                if c["causal"] and not c["prefix"]:
                    y = min(y, off + i + n)
                p, j = torch.arange(off + i, off + i + n, device="cuda"), torch.arange(x, y, device="cuda")
                vis = (j >= s.start[b]) & (j < s.len[b])
                vis = vis.expand(n, -1)
                if c["causal"]:
                    vis = vis & ((j <= p[:, None]) | (j < s.prefix[b]))
                if W:
                    vis = vis & ((j - p[:, None]).abs() < W)
                o = _attend(q[:, :, i:i + n], k[:, x:y].contiguous(), v[:, x:y].contiguous(), p, j, c, s.slopes, vis)
                out[b, i:i + n] = o.permute(2, 0, 1, 3).reshape(n, Hq, D).to(out.dtype)
    return out


def _sequence(s, x, b, n):
    """Rows (H, n, ...) of the first n tokens of sequence b of a cache or pool, or of its scales."""
    if x is None:
        return None
    if s.bt is None:
        return x[b, :, :n]
    pages = s.bt[b, :-(-n // s.case["page"])].long()
    return x[pages].transpose(0, 1).flatten(1, 2)[:, :n]


def _plain_step(s):
    c = s.case
    B, Hq, H, D = c["B"], c["Hq"], c["H"], c["D"]
    out = torch.zeros(B, 1, Hq, D, dtype=torch.float32, device="cuda")
    for b, n in enumerate(s.ctx):
        lo = max(s.first[b], n - c["window"] if c["window"] else 0)
        if n <= lo:
            continue
        k, v = (_sequence(s, x, b, n)[:, lo:].float() for x in (s.k, s.v))
        if s.ks is not None:
            k, v = k * _sequence(s, s.ks, b, n)[:, lo:, None].float(), v * _sequence(s, s.vs, b, n)[:, lo:, None].float()
        p, j = torch.full((1,), n - 1, device="cuda"), torch.arange(lo, n, device="cuda")
        q = s.q[b, :, 0].float().view(H, Hq // H, 1, D)
        out[b, 0] = _attend(q, k.contiguous(), v.contiguous(), p, j, c, s.slopes, torch.ones_like(j, dtype=torch.bool)).view(Hq, D)
    return out.to(s.q.dtype)


def _plain_rope(s):
    c = s.case
    R = c["R"]
    angle = s.pos.double()[..., None] * s.freq
    cos, sin = ((s.scale * f).float()[:, :, None] for f in (angle.cos(), angle.sin()))
    out = []
    for x in (s.q, s.k):
        x = x.float()
        a, b = (x[..., :R // 2], x[..., R // 2:R]) if c["pairs"] == "half" else (x[..., 0:R:2], x[..., 1:R:2])
        turned = (a * cos - b * sin, b * cos + a * sin)
        head = torch.cat(turned, dim=-1) if c["pairs"] == "half" else torch.stack(turned, dim=-1).flatten(-2)
        out.append(torch.cat([head, x[..., R:]], dim=-1).to(s.q.dtype))
    return tuple(out)


def run(state):
    s = state
    c = s.case
    if not own:
        return {"prompt": _plain_prompt, "step": _plain_step, "rope": _plain_rope}[c["kind"]](s)
    sia = _sia()
    if c["kind"] == "rope":
        return sia.rope_scaled(s.q, s.k, s.pos, s.freq, rotary_dim=c["R"], interleaved=c["pairs"] == "interleaved",
                               scale=s.scale)
    shape = {"softcap": c["cap"] or None, "alibi_slopes": s.slopes, "window": c["window"] or None}
    if c["kind"] == "prompt":
        padded = bool(c["pad"])
        return sia.scored_attention_flash(s.q, s.k, s.v, causal=c["causal"], cu_seqlens=s.boundaries,
                                          prefix_len=s.prefix if c["prefix"] else None,
                                          kv_start=s.start if padded else None, kv_len=s.len if padded else None,
                                          out_token_major=True, **shape)
    if s.bt is None:
        return sia.scored_attention_flash_decode(s.q, s.k, s.v, s.kv_len, s.ks, s.vs, kv_start=s.start, **shape)
    return sia.paged_scored_attention_flash_decode(s.q, s.k, s.v, s.bt, s.kv_len, c["page"], s.ks, s.vs,
                                                   kv_start=s.start, **shape)


# --------------------------------------------------- the definition, in 64 bits


def _exact_scores(qk, c, slope, p, j):
    x = qk / math.sqrt(c["D"])
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    if c["alibi"]:
        x = x - slope * (p[:, None] - j[None, :]).abs().double()
    return x


def _exact_prompt(s):
    c = s.case
    off = c["Tk"] - c["Tq"]
    out = torch.zeros(c["B"], c["Tq"], c["Hq"], c["D"], dtype=torch.float64, device="cuda")
    rows = _rows(c)
    for b in range(c["B"]):
        start, n, prefix = rows[b]
        for a, e in zip(s.cuts, s.cuts[1:]):
            step = 2048
            for first in range(max(a, off), e, step):
                p = torch.arange(first, min(e, first + step), device="cuda")
                j = torch.arange(a, e, device="cuda")
                hidden = (j[None, :] < start) | (j[None, :] >= n)
                if c["causal"]:
                    hidden = hidden | ((j[None, :] > p[:, None]) & (j[None, :] >= prefix))
                if c["window"]:
                    d = j[None, :] - p[:, None]
                    hidden = hidden | (d <= -c["window"]) | (d >= c["window"])
                hidden = hidden.expand(len(p), len(j))
                for h in range(c["Hq"]):
                    kv = h // (c["Hq"] // c["H"])
                    k, v = s.k[b, kv, a:e].double(), s.v[b, kv, a:e].double()
                    x = torch.mm(s.q[b, h, first - off:first - off + len(p)].double(), k.t().contiguous())
                    x = _exact_scores(x, c, 2.0 ** (-8.0 * (h + 1) / c["Hq"]), p, j).masked_fill(hidden, float("-inf"))
                    w = torch.softmax(x, dim=-1).masked_fill(hidden.all(dim=-1, keepdim=True), 0.0)
                    out[b, first - off:first - off + len(p), h] = torch.mm(w, v)
    return out


def _exact_step(s):
    c = s.case
    out = torch.zeros(c["B"], 1, c["Hq"], c["D"], dtype=torch.float64, device="cuda")
    per = c["Hq"] // c["H"]
    for b, n in enumerate(s.ctx):
        first = s.first[b]
        if c["window"]:
            first = max(first, n - c["window"])
        if first >= n:
            continue
        k, v, ks, vs = (_sequence(s, x, b, n) for x in (s.k, s.v, s.ks, s.vs))
        p, j = torch.tensor([n - 1], device="cuda"), torch.arange(first, n, device="cuda")
        for h in range(c["Hq"]):
            kh, vh = k[h // per, first:].double(), v[h // per, first:].double()
            if ks is not None:
                kh, vh = kh * ks[h // per, first:, None].double(), vh * vs[h // per, first:, None].double()
            x = torch.mm(s.q[b, h].double(), kh.t().contiguous())
            w = torch.softmax(_exact_scores(x, c, 2.0 ** (-8.0 * (h + 1) / c["Hq"]), p, j), dim=-1)
            out[b, 0, h] = torch.mm(w, vh)[0]
    return out


def _exact_rope(s):
    c = s.case
    R = c["R"]
    turn = torch.polar(torch.full((1,), s.scale, dtype=torch.float64, device="cuda"),
                       s.pos.double()[:, :, None, None] * s.freq)
    out = []
    for x in (s.q, s.k):
        y = x.double().clone()
        pair = y[..., :R].unflatten(-1, (2, R // 2)).transpose(-1, -2) if c["pairs"] == "half" else y[..., :R].unflatten(-1, (R // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        y[..., :R] = (z.transpose(-1, -2) if c["pairs"] == "half" else z).flatten(-2)
        out.append(y)
    return tuple(out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"prompt": _exact_prompt, "step": _exact_step, "rope": _exact_rope}[s.case["kind"]](s)
