"""The operators around a decoder layer's attention, and how their speed is judged.

* ``norm_rope``: RMS norm of every query and key head and the rotation by position in one pass (``train``: with its
  pullback, gradients of the inputs and of both weight vectors).
* ``cache``: keys and values of new tokens quantised into an 8-bit cache (one scale per page of tokens and head) and
  read back.
* ``attend``: attention of new queries over such a cache.

``run`` computes them in elementary torch operations in 32 bits (64 for the angles), or, where ``own`` is set, through
the public entry points of ``nnlib_jl_b200``.  Arrays are column-major like everything of this framework: an ``(E, L, B)``
array is the permuted view of a contiguous ``(B, L, E)`` one.  Activations are N(0, 1), weights 1 + N(0, 0.1).
"""
import math

import numpy as np
import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_TOP = {"int8": 127.0, "e4m3": 448.0}
_EPS = 1e-6
_TINY = 2.0 ** -126          # a smaller scale is none: the block's codes are zero


def _norm(dtype, d, H, Hk, L, B, rot, neighbours, far, train):
    """H query and Hk key heads of d features, L tokens of B sequences, the first of them at a position up to ``far``;
    the first ``rot`` features are rotated, as pairs of neighbours or of the two halves."""
    return {"op": "norm_rope", "dtype": dtype, "d": d, "H": H, "Hk": Hk, "L": L, "B": B, "rot": rot,
            "neighbours": neighbours, "far": far, "train": train}


def _cache(dtype, code, d, Hk, L, B, page, past, paged):
    """L new tokens of each of B sequences behind up to ``past`` tokens; paged: pages in any order, through a table."""
    return {"op": "cache", "dtype": dtype, "code": code, "d": d, "Hk": Hk, "L": L, "B": B, "page": page,
            "past": past, "paged": paged}


def _attend(dtype, code, d, H, Hk, Lq, Lkv, B, page, ragged, paged):
    """The last Lq tokens of B sequences of Lkv tokens (ragged: from half of that to all of it) attend, causally, to
    their sequence."""
    return {"op": "attend", "dtype": dtype, "code": code, "d": d, "H": H, "Hk": Hk, "Lq": Lq, "Lkv": Lkv,
            "B": B, "page": page, "ragged": ragged, "paged": paged}


def listed():
    return [
        # one generated token of eight sequences far into their context, grouped heads: latency
        {"name": "rope_token"} | _norm("bf16", 128, 32, 8, 1, 8, 128, False, 100000, False),
        # the prompt of eight sequences
        {"name": "rope_prefill"} | _norm("bf16", 128, 32, 8, 4096, 8, 128, False, 0, False),
        # a training step of the decoder layer that perf/cases.py trains
        {"name": "rope_train"} | _norm("bf16", 128, 32, 32, 4096, 8, 128, False, 0, True),
        # a small model's step: lengths and head size of no roundness, half of a head's features rotated, as neighbours
        {"name": "rope_train_ragged"} | _norm("f16", 80, 8, 8, 1000, 6, 40, True, 0, True),
        # a generated token of 64 sequences into pages that are partly full
        {"name": "cache_token"} | _cache("bf16", "int8", 128, 8, 1, 64, 64, 4096, True),
        # the prompt of eight sequences, from an empty cache
        {"name": "cache_prefill"} | _cache("bf16", "int8", 128, 8, 4096, 8, 64, 0, False),
        # the next part of a prompt, ending inside a page, floating-point codes
        {"name": "cache_chunk_ragged"} | _cache("f16", "e4m3", 80, 8, 777, 6, 32, 1000, True),
        # one generated token against a short history, the smallest model's heads
        {"name": "decode_small"} | _attend("f16", "int8", 64, 12, 12, 1, 500, 1, 16, False, False),
        # one generated token of eight sequences of up to 8k tokens
        {"name": "decode_8k"} | _attend("bf16", "e4m3", 128, 32, 8, 1, 8192, 8, 64, True, True),
        # the same against very long histories: the largest read
        {"name": "decode_131k"} | _attend("bf16", "int8", 128, 32, 8, 1, 131072, 4, 64, True, True),
        # a part of a prompt of some sequences that are already long
        {"name": "chunk_16k"} | _attend("f16", "e4m3", 128, 32, 8, 512, 16384, 4, 64, True, True),
        # a second prompt as long as the first: the most arithmetic
        {"name": "prefill_8k"} | _attend("bf16", "int8", 128, 32, 8, 4096, 8192, 4, 128, False, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    d = rng.choice([32, 48, 64, 64, 80, 96, 112, 128, 128, 128])
    Hk = _log(rng, 1, 12)
    G = rng.choice([1, 1, 2, 3, 4, 5, 8])
    op = rng.choice(["norm_rope", "cache", "attend", "attend"])
    if op == "norm_rope":
        L, B = _log(rng, 1, 8192), _log(rng, 1, 16)
        while L * B * Hk * (G + 1) * d > 4096 * 8 * 64 * 128:
            L = (L + 1) // 2
        rot = rng.choice([d, d, d // 2])
        return _norm(dtype, d, Hk * G, Hk, L, B, rot - rot % 2, rng.random() < 0.3,
                     rng.choice([0, 1000, 500000]), rng.random() < 0.5)
    page = rng.choice([16, 32, 64, 64, 128])
    code = rng.choice(["int8", "e4m3"])
    paged = rng.random() < 0.6
    if op == "cache":
        L, B = rng.choice([1, _log(rng, 1, 8192)]), _log(rng, 1, 64)
        while L * B * Hk * d > 4096 * 8 * 8 * 128:
            L = (L + 1) // 2
        return _cache(dtype, code, d, Hk, L, B, page, rng.choice([0, 100, 2000]), paged)
    Lkv, B = _log(rng, 64, 131072), _log(rng, 1, 16)
    while Lkv * B * Hk * d > 131072 * 4 * 8 * 128:
        Lkv = (Lkv + 1) // 2
    Lq = min(Lkv // 2, rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 2, 4096)]))
    while Lq * Lkv * B * Hk * G * d > 4096 * 6144 * 4 * 32 * 128 // (8 if dtype == "f32" else 1):
        Lq = (Lq + 1) // 2
    return _attend(dtype, code, d, Hk * G, Hk, Lq, Lkv, B, page, rng.random() < 0.6, paged)


# ---------------------------------------------------------------------------------------------------- inputs
def _array(gen, E, L, B, dtype):
    """(E, L, B), column-major."""
    t = torch.empty((B, L, E), device="cuda", dtype=torch.float32).normal_(generator=gen)
    return t.to(dtype).permute(2, 1, 0)


def _scale(amax, code):
    """The scale of a block: its largest magnitude becomes Int8's 127, or is the first power of two that brings it to
    E4M3's 448 or less (a floating-point code then rounds like its value, whatever the scale)."""
    if code == "int8":
        s = amax / 127.0
    else:
        m, e = torch.frexp(amax)                                           # 448 = 0.875 * 2^9
        s = torch.ldexp(torch.ones_like(amax), e - 9 + (m > 0.875).int())
    return torch.where(s * amax.sign() < _TINY, 0.0, s)


def _codes(x, scale, code):
    """Codes of x under scale (which broadcasts), as numbers: x / scale to the nearest code."""
    inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    t = (x * inv).clamp(-_TOP[code], _TOP[code])
    return t.round() if code == "int8" else t.to(torch.float8_e4m3fn).float()


def _filled(gen, d, Hk, page, pages, code):
    """A pool of full pages: codes (Hk d, page, pages) and scales (Hk, pages)."""
    x = torch.empty((pages, page, Hk, d), device="cuda", dtype=torch.bfloat16).normal_(generator=gen)
    scale = _scale(x.abs().amax((1, 3)).float(), code)
    c = torch.empty((pages, page, Hk, d), device="cuda", dtype=_CODE[code])
    step = max(1, (1 << 26) // (page * Hk * d))
    for at in range(0, pages, step):
        c[at:at + step] = _codes(x[at:at + step].float(), scale[at:at + step, None, :, None], code).to(_CODE[code])
    return c.view(pages, page, Hk * d).permute(2, 1, 0), scale.t()


def _table(gen, B, N, paged):
    """(N, B) page numbers; pages in any order among some that are not used."""
    if not paged:
        return None
    return torch.randperm(B * N + 8, device="cuda", generator=gen)[:B * N].to(torch.int32).view(B, N).t()


def _lengths(case):
    """Tokens of each sequence; they are the case's own, so that its work is."""
    Lkv, B = case["Lkv"], case["B"]
    return [Lkv - (Lkv // 2 * b) // B if case["ragged"] else Lkv for b in range(B)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, d, Hk, B = _DTYPE[case["dtype"]], case["d"], case["Hk"], case["B"]
    s = {"case": case}
    if case["op"] == "norm_rope":
        L, H = case["L"], case["H"]
        s["q"], s["k"] = _array(gen, H * d, L, B, dtype), _array(gen, Hk * d, L, B, dtype)
        s["gq"], s["gk"] = ((1 + 0.1 * torch.randn(d, device="cuda", generator=gen)).to(dtype) for _ in range(2))
        pair = torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64)
        s["freqs"] = 10000.0 ** (-2.0 * pair / case["rot"])
        s["start"] = torch.randint(0, case["far"] + 1, (B,), device="cuda", generator=gen).to(torch.int32)
        if case["train"]:
            s["dq"], s["dk"] = _array(gen, H * d, L, B, dtype), _array(gen, Hk * d, L, B, dtype)
        return s
    page, code = case["page"], case["code"]
    most = case["past"] + case["L"] if case["op"] == "cache" else case["Lkv"]
    N = -(-most // page)
    pool = B * N + (8 if case["paged"] else 0)
    s["table"] = _table(gen, B, N, case["paged"])
    s["ck"], s["sk"] = _filled(gen, d, Hk, page, pool, code)
    s["cv"], s["sv"] = _filled(gen, d, Hk, page, pool, code)
    if case["op"] == "cache":
        s["k"], s["v"] = _array(gen, Hk * d, case["L"], B, dtype), _array(gen, Hk * d, case["L"], B, dtype)
        s["start"] = torch.randint(0, case["past"] + 1, (B,), device="cuda", generator=gen).to(torch.int32)
    else:
        s["q"] = _array(gen, case["H"] * d, case["Lq"], B, dtype)
        s["lens"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _angles(s, L):
    """cos and sin, (B, L, 1, pairs): the angles of far positions need 64 bits."""
    pos = s["start"].double()[:, None] + torch.arange(L, device="cuda")
    a = pos[:, :, None, None] * s["freqs"]
    return a.cos().float(), a.sin().float()


def _rotate(x, cos, sin, case, back=False):
    """Rotates the pairs of the first ``rot`` features of x (..., d); back: by the opposite angle."""
    rot = case["rot"]
    head, rest = x[..., :rot], x[..., rot:]
    if case["neighbours"]:
        a, b = head[..., 0::2], head[..., 1::2]
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
    if back:
        sin = -sin
    u, v = a * cos - b * sin, a * sin + b * cos
    both = torch.stack((u, v), -1).flatten(-2) if case["neighbours"] else torch.cat((u, v), -1)
    return torch.cat((both, rest), -1)


def _heads(t, d):
    """(E, L, B) as (B, L, heads, d) in 32 bits."""
    t = t.permute(2, 1, 0)
    return t.reshape(t.shape[0], t.shape[1], -1, d).float()


def _columns(t, dtype):
    """(B, L, heads, d) as (E, L, B)."""
    return t.reshape(t.shape[0], t.shape[1], -1).to(dtype).permute(2, 1, 0)


def _plain_norm_rope(s, case):
    dtype, d = s["q"].dtype, case["d"]
    cos, sin = _angles(s, case["L"])

    def forward(x, g):
        x = _heads(x, d)
        r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)
        return _columns(_rotate(x * r * g.float(), cos, sin, case), dtype)

    def backward(x, g, dy):
        x, u = _heads(x, d), _rotate(_heads(dy, d), cos, sin, case, back=True)
        r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)
        n = x * r
        w = u * g.float()
        dx = r * (w - n * (w * n).mean(-1, keepdim=True))
        return _columns(dx, dtype), (u * n).sum((0, 1, 2)).to(dtype)

    y = forward(s["q"], s["gq"]), forward(s["k"], s["gk"])
    if not case["train"]:
        return y
    dq, dgq = backward(s["q"], s["gq"], s["dq"])
    dk, dgk = backward(s["k"], s["gk"], s["dk"])
    return (*y, dq, dk, dgq, dgk)


def _pages_of(s, case, n):
    """Page numbers (B, n) of local pages 0 .. n - 1."""
    if s["table"] is not None:
        return s["table"].t().long()[:, :n]
    per = s["ck"].shape[2] // case["B"]
    return torch.arange(case["B"], device="cuda")[:, None] * per + torch.arange(n, device="cuda")


def _plain_write(s, case, codes, scales, x):
    """Quantises x (E, L, B) into the pool and gives back what the pool then holds of it, in x's type."""
    d, T, L, B, code, Hk = (case[n] for n in ("d", "page", "L", "B", "code", "Hk"))
    pool = codes.permute(2, 1, 0).view(-1, T, Hk, d)
    raw = pool.view(torch.uint8)                                           # 8-bit floats are indexed as bytes
    per_page = scales.t()                                                  # (pages, Hk), the caller's memory
    new = _heads(x, d)                                                     # (B, L, Hk, d)
    start = s["start"].long()
    pos = start[:, None] + torch.arange(L, device="cuda")                  # (B, L)
    n = (L - 1) // T + 2                                                   # pages that L tokens can touch
    local = pos // T - (start // T)[:, None]                               # (B, L), 0 .. n - 1
    page = _pages_of(s, case, per_page.shape[0]).gather(1, pos // T)       # (B, L)
    amax = torch.zeros((B, n, Hk), device="cuda").scatter_reduce(
        1, local[:, :, None].expand(-1, -1, Hk), new.abs().amax(-1), "amax")
    first = page[:, 0]                                                     # the page that may hold older tokens
    fill = start % T
    old = torch.where((fill > 0)[:, None], per_page[first], 0.0)           # (B, Hk)
    scale = _scale(amax, code)
    scale[:, 0] = torch.maximum(scale[:, 0], old)
    grown = torch.where(scale[:, 0] > 0, old / scale[:, 0], 0.0)           # (B, Hk)
    held = raw[first].view(pool.dtype).float()
    older = held * grown[:, None, :, None]
    older = older.round() if code == "int8" else older.to(_CODE[code]).float()
    keep = (torch.arange(T, device="cuda") < fill[:, None])[:, :, None, None]
    raw[first] = torch.where(keep, older, held).to(pool.dtype).view(torch.uint8)
    per_token = scale.gather(1, local[:, :, None].expand(-1, -1, Hk))      # (B, L, Hk)
    per_page[page] = per_token
    got = _codes(new, per_token[..., None], code)
    raw[page, pos % T] = got.to(pool.dtype).view(torch.uint8)
    return _columns(got * per_token[..., None], x.dtype)


def _plain_cache(s, case):
    k = _plain_write(s, case, s["ck"], s["sk"], s["k"])
    v = _plain_write(s, case, s["cv"], s["sv"], s["v"])
    return k, v, s["sk"], s["sv"]


def _plain_attend(s, case):
    d, T, Hk, Lq, B = (case[n] for n in ("d", "page", "Hk", "Lq", "B"))
    G, N = case["H"] // Hk, -(-case["Lkv"] // T)
    page = _pages_of(s, case, N)

    def values(codes, scales):                                             # (B, Hk, N T, d)
        raw = codes.permute(2, 1, 0).view(torch.uint8).view(-1, T, Hk, d)
        c = raw[page].view(codes.dtype).float()                            # (B, N, T, Hk, d)
        c *= scales.t()[page][:, :, None, :, None]
        return c.view(B, N * T, Hk, d).transpose(1, 2)

    q = _heads(s["q"], d).view(B, Lq, Hk, G, d).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Lq, d)
    t = torch.matmul(q * (1.0 / math.sqrt(d)), values(s["ck"], s["sk"]).transpose(2, 3)).view(B, Hk, G, Lq, N * T)
    lens = s["lens"].long()[:, None, None]
    last = lens - Lq + torch.arange(Lq, device="cuda")[:, None]            # (B, Lq, 1): the last key a query sees
    hidden = torch.arange(N * T, device="cuda") > last                     # (B, Lq, keys)
    t.masked_fill_(hidden[:, None, None], -math.inf)
    t -= t.amax(-1, keepdim=True)
    t.exp_()
    t /= t.sum(-1, keepdim=True)
    x = torch.matmul(t.view(B, Hk, G * Lq, N * T), values(s["cv"], s["sv"]))
    x = x.view(B, Hk, G, Lq, d).permute(0, 3, 1, 2, 4)                     # (B, Lq, Hk, G, d)
    return _columns(x, s["q"].dtype)


def _own(s, case):
    import nnlib_jl_b200 as nb
    if case["op"] == "norm_rope":
        args = (s["q"], s["k"], s["gq"], s["gk"], s["freqs"])
        how = {"nheads": case["H"], "start": s["start"], "interleaved": case["neighbours"], "eps": _EPS}
        if not case["train"]:
            return nb.qk_norm_rope(*args, **how)
        qn, kn, back = nb.qk_norm_rope_pullback(*args, **how)
        return (qn, kn, *back(s["dq"], s["dk"]))
    c = nb.QuantizedCache.from_arrays(s["ck"], s["cv"], s["sk"], s["sv"])
    if case["op"] == "attend":
        return nb.cached_attention(s["q"], c, s["lens"], nheads=case["H"], table=s["table"])
    nb.cache_write_(c, s["k"], s["v"], start=s["start"], table=s["table"])
    k, v = nb.cache_read(c, case["L"], start=s["start"], table=s["table"], dtype=s["k"].dtype)
    return k, v, c.k_scale, c.v_scale


def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return {"norm_rope": _plain_norm_rope, "cache": _plain_cache, "attend": _plain_attend}[case["op"]](s, case)


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    z, d, Hk, B = _BYTES[case["dtype"]], case["d"], case["Hk"], case["B"]
    if case["op"] == "norm_rope":
        n = (case["H"] + Hk) * d * case["L"] * B
        # forward: in and out; pullback: in, gradient in, gradient out
        return {"bytes": n * z * (5 if case["train"] else 2), "flops": n * (25.0 if case["train"] else 8.0)}
    if case["op"] == "cache":
        # new tokens in, codes out, codes in, read back out; a scale for each page and head
        n = 2 * Hk * d * case["L"] * B
        return {"bytes": n * (2 * z + 2) + 2 * 4 * Hk * B * -(-case["L"] // case["page"]), "flops": 6.0 * n}
    lens, Lq = _lengths(case), case["Lq"]
    pairs = sum(Lq * (m - Lq) + Lq * (Lq + 1) // 2 for m in lens) * case["H"]
    kv = sum(2 * Hk * d * m + 2 * 4 * Hk * -(-m // case["page"]) for m in lens)
    return {"bytes": kv + 2 * z * case["H"] * d * Lq * B, "flops": 4.0 * d * pairs}


# ---------------------------------------------------------------------------------------------------- 64 bits
def _exact_norm_rope(s, case):
    """From the definition, per token: y = R n, n = x g / sqrt(mean x^2 + eps), R as complex numbers of modulus 1; the
    gradient as the derivative along x of <dy, y>."""
    d, rot, L, B = case["d"], case["rot"], case["L"], case["B"]
    pos = s["start"].double().view(B, 1) + torch.arange(L, device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), (pos[..., None] * s["freqs"])).unsqueeze(2)
    first = torch.arange(0, rot, 2, device="cuda") if case["neighbours"] else torch.arange(rot // 2, device="cuda")
    second = first + (1 if case["neighbours"] else rot // 2)

    def turned(n, by):
        z = torch.complex(n[..., first], n[..., second]) * by
        out = n.clone()
        out[..., first], out[..., second] = z.real, z.imag
        return out

    got, grads, weights = [], [], []
    for x, g, dy in ((s["q"], s["gq"], s.get("dq")), (s["k"], s["gk"], s.get("dk"))):
        ys, dxs, dg = [], [], torch.zeros(d, device="cuda", dtype=torch.float64)
        for b in range(B):                                                 # one sequence at a time: memory
            xb = x[:, :, b].t().double().view(L, -1, d)
            size = torch.sqrt(torch.einsum("lhd,lhd->lh", xb, xb) / d + _EPS)[..., None]
            ys.append(turned(xb / size * g.double(), turn[b]))
            if dy is not None:
                u = turned(dy[:, :, b].t().double().view(L, -1, d), turn[b].conj())
                dg += torch.einsum("lhd,lhd->d", u, xb / size)
                w = u * g.double()
                dxs.append(w / size - xb * torch.einsum("lhd,lhd->lh", w, xb)[..., None] / (d * size ** 3))
        got.append(torch.stack(ys).reshape(B, L, -1).permute(2, 1, 0))
        if dy is not None:
            grads.append(torch.stack(dxs).reshape(B, L, -1).permute(2, 1, 0))
            weights.append(dg)
    return (*got, *grads, *weights)


def _exact_cache(s, case):
    """Page by page, the way the definition reads."""
    d, T, L, B, code, Hk = (case[n] for n in ("d", "page", "L", "B", "code", "Hk"))
    per = s["ck"].shape[2] // B
    starts = s["start"].tolist()
    table = s["table"].t().tolist() if s["table"] is not None else [list(range(b * per, (b + 1) * per)) for b in range(B)]
    out = []
    for x, scales in ((s["k"], s["sk"]), (s["v"], s["sv"])):
        x64 = x.double().permute(2, 1, 0).reshape(B, L, Hk, d)
        after, back = scales.double().clone(), torch.empty_like(x64)
        for b in range(B):
            at = 0
            while at < L:
                here = starts[b] + at
                n = min(L - at, T - here % T)
                page = table[b][here // T]
                block = x64[b, at:at + n]                                  # (n, Hk, d)
                scale = block.abs().amax((0, 2)) / _TOP[code]
                if code == "e4m3":
                    scale = torch.exp2(torch.ceil(torch.log2(scale)))
                if here % T:
                    scale = torch.maximum(scale, after[:, page])
                after[:, page] = scale
                c = block / scale[None, :, None]
                c = torch.round(c) if code == "int8" else c.float().to(torch.float8_e4m3fn).double()
                back[b, at:at + n] = c * scale[None, :, None]
                at += n
        out.append((back.reshape(B, L, -1).permute(2, 1, 0), after))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_attend(s, case):
    """Sequence by sequence and head by head over the tokens that are there, a share of the queries at a time."""
    d, T, Hk, Lq, B = (case[n] for n in ("d", "page", "Hk", "Lq", "B"))
    G = case["H"] // Hk
    per = s["ck"].shape[2] // B
    out = torch.empty((B, Lq, case["H"], d), device="cuda", dtype=torch.float64)
    for b, m in enumerate(s["lens"].tolist()):
        need = -(-m // T)
        pages = s["table"][:need, b].long() if s["table"] is not None else torch.arange(b * per, b * per + need, device="cuda")
        for h in range(Hk):
            def side(codes, scales):
                c = codes.permute(2, 1, 0).view(torch.uint8)[pages, :, h * d:(h + 1) * d].contiguous()
                return (c.view(codes.dtype).double() * scales[h, pages].double()[:, None, None]).reshape(need * T, d)[:m]
            K, V = side(s["ck"], s["sk"]), side(s["cv"], s["sv"])
            step = max(1, (1 << 27) // (G * m))
            for i in range(0, Lq, step):
                n = min(step, Lq - i)
                q = s["q"][h * G * d:(h + 1) * G * d, i:i + n, b].t().double().reshape(n * G, d)
                logits = (q @ K.t() / math.sqrt(d)).view(n, G, m)
                seen = torch.arange(m, device="cuda") <= (m - Lq + i + torch.arange(n, device="cuda"))[:, None]
                p = torch.softmax(logits.masked_fill(~seen[:, None], -np.inf), -1)
                out[b, i:i + n, h * G:(h + 1) * G] = (p.view(n * G, m) @ V).view(n, G, d)
    return out.reshape(B, Lq, -1).permute(2, 1, 0)


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm_rope": _exact_norm_rope, "cache": _exact_cache, "attend": _exact_attend}[case["op"]](s, case)
