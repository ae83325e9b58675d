"""Products of ragged groups of columns, and how their speed is judged.

* ``route``: each token's ``k`` best of ``G`` experts, their softmax weights, and the tokens' order by expert (``train``: with the
  gradient of the logits).
* ``experts``: the product of each expert's matrix and the columns of its tokens (``train``: with both gradients).
* ``combine``: each token's weighted sum of its experts' columns (``train``: with the gradients of columns and weights).
* ``adapters``: one matrix for all columns and a low-rank pair of matrices for each request's own (``train``: with the
  gradients of the columns and of the pairs).

``run`` computes them in elementary torch operations in 32 bits, groups padded to the largest one and multiplied as a batch, or,
where ``own`` is set, through the public entry points of ``nnlib_jl_b200``.  Arrays are column-major like everything of this
framework: an ``(E, N)`` array is the transposed view of a contiguous ``(N, E)`` one.  Activations are N(0, 1), matrices
N(0, 1 / columns), router logits N(0, 1) with an expert's own popularity added.
"""
import math
import zlib

import numpy as np
import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _route(dtype, G, k, N, live, bias, normalize, train):
    """N tokens, of which the first ``live`` take part; ``bias`` is added for the choice alone; the weights are those of the
    chosen (normalize) or of all experts."""
    return {"op": "route", "dtype": dtype, "G": G, "k": k, "N": N, "live": live, "bias": bias, "normalize": normalize, "train": train}


def _experts(dtype, G, k, N, live, M, K, turned, train):
    """G matrices (M, K), stored as they are or ``turned``: as (K, M)."""
    return {"op": "experts", "dtype": dtype, "G": G, "k": k, "N": N, "live": live, "M": M, "K": K, "turned": turned, "train": train}


def _combine(dtype, G, k, N, live, E, train):
    return {"op": "combine", "dtype": dtype, "G": G, "k": k, "N": N, "live": live, "E": E, "train": train}


def _adapters(dtype, R, L, ragged, M, K, r, n, train):
    """R requests of L tokens (ragged: from L down to half of it) in one run of columns, n pairs of rank r."""
    return {"op": "adapters", "dtype": dtype, "R": R, "L": L, "ragged": ragged, "M": M, "K": K, "r": r, "n": n, "train": train}


def listed():
    return [
        # one generated token of up to 64 sequences, some of which have ended: latency
        {"name": "route_token"} | _route("f32", 128, 8, 64, 50, False, True, False),
        # the prompts of eight sequences, many experts, 16-bit logits (of which many are equal)
        {"name": "route_prefill"} | _route("bf16", 256, 8, 32768, 32768, True, True, False),
        # a small model's training step
        {"name": "route_train_ragged"} | _route("f32", 60, 4, 10007, 10007, False, False, True),
        # a generated token of 32 sequences: nearly every expert has a token or a few
        {"name": "experts_token"} | _experts("bf16", 128, 8, 32, 32, 1536, 2048, True, False),
        # the prompt of eight sequences, few large experts: the most arithmetic
        {"name": "experts_prefill"} | _experts("bf16", 8, 2, 8192, 8192, 14336, 4096, False, False),
        # a training step, middling experts
        {"name": "experts_train"} | _experts("f16", 32, 4, 4096, 4096, 1408, 2048, True, True),
        # a small training step with sizes of no roundness, the last tokens padding
        {"name": "experts_train_ragged"} | _experts("f32", 5, 2, 600, 555, 333, 200, False, True),
        # the prompt of eight sequences of experts_prefill, back in the tokens' order
        {"name": "combine_prefill"} | _combine("bf16", 8, 2, 8192, 8192, 4096, False),
        # a training step, many small experts
        {"name": "combine_train"} | _combine("f16", 64, 6, 4096, 4096, 2048, True),
        # one generated token of 64 requests, nearly all with a pair of their own
        {"name": "adapters_token"} | _adapters("bf16", 64, 1, False, 4096, 4096, 16, 64, False),
        # the prompts of eight requests
        {"name": "adapters_prefill"} | _adapters("bf16", 8, 1024, True, 4096, 4096, 64, 8, False),
        # a training step of four pairs
        {"name": "adapters_train"} | _adapters("f16", 4, 2048, False, 2048, 2048, 32, 4, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _size(rng, lo, hi):
    """A number of features: odd now and then, mostly a multiple of 8."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.15 else max(8, n - n % 8)


def draw(rng):
    op = rng.choice(["route", "experts", "experts", "combine", "adapters", "adapters"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    train = rng.random() < 0.4
    if op == "adapters":
        R, M, K = _log(rng, 1, 64), _size(rng, 64, 8192), _size(rng, 64, 8192)
        L = rng.choice([1, _log(rng, 2, 4096)])
        top = 8192 * 4096 * 4096 // (8 if dtype == "f32" else 1) // (2 if train else 1)
        while R * L * M * K > top and L > 1:
            L = (L + 1) // 2
        return _adapters(dtype, R, L, rng.random() < 0.6, M, K, rng.choice([4, 8, 16, 16, 32, 64, 128]), _log(rng, 1, 64), train)
    G = _log(rng, 2, 256)
    k = min(G, rng.choice([1, 2, 2, 4, 6, 8]))
    N = _log(rng, 1, 32768)
    if op == "route":
        return _route(dtype, G, k, N, N - rng.choice([0, 0, N // 5]), rng.random() < 0.4, rng.random() < 0.6, train)
    if op == "combine":
        E = _size(rng, 64, 8192)
        while N * k * E > 8192 * 8 * 4096:
            N = (N + 1) // 2
        return _combine(dtype, G, k, N, N - rng.choice([0, 0, N // 5]), E, train)
    M, K = _size(rng, 64, 14336), _size(rng, 64, 8192)
    while G * M * K > 128 * 1536 * 2048:
        G = (G + 1) // 2
    k = min(k, G)
    top = 16384 * 14336 * 4096 // (16 if dtype == "f32" else 1) // (3 if train else 1)
    while N * k * M * K > top:
        N = (N + 1) // 2
    return _experts(dtype, G, k, N, N - rng.choice([0, 0, N // 5]), M, K, rng.random() < 0.5, train)


# ---------------------------------------------------------------------------------------------------- inputs
def _array(gen, E, N, dtype, scale=1.0):
    """(E, N), column-major."""
    t = torch.empty((N, E), device="cuda", dtype=dtype if dtype != torch.float16 else torch.float32)
    return t.normal_(0.0, scale, generator=gen).to(dtype).t()


def _matrices(gen, M, K, G, dtype, turned=False):
    """(M, K, G) matrices, column-major, or the transposes of column-major (K, M, G) ones."""
    t = torch.empty((G, M, K) if turned else (G, K, M), device="cuda", dtype=dtype)
    t.normal_(0.0, 1.0 / math.sqrt(K), generator=gen)
    return t.permute(1, 2, 0) if turned else t.permute(2, 1, 0)


def _chosen(case):
    """Experts of each token (N, k) in falling order, the case's own, so that its work is; of the first ``live`` alone."""
    rng = np.random.RandomState(zlib.crc32(repr(sorted((a, b) for a, b in case.items() if a != "name")).encode()) % (1 << 31))
    G, k, live = case["G"], case["k"], case["live"]
    logits = rng.standard_normal((live, G)).astype(np.float32) + 0.5 * rng.standard_normal(G).astype(np.float32)
    return np.argsort(-logits, 1, kind="stable")[:, :k], logits


def _most(case):
    """Tokens of the busiest expert."""
    return max(1, int(np.bincount(_chosen(case)[0].reshape(-1), minlength=case["G"]).max(initial=0)))


def _order(experts, G, k):
    """offsets (G + 1), columns (k N), position (N, k) of experts (N, k), which are G for a token that takes no part."""
    flat = experts.reshape(-1)
    order = flat.sort(stable=True).indices
    count = torch.zeros(G + 1, dtype=torch.int64, device=flat.device).scatter_add_(0, flat, torch.ones_like(flat))
    ends = count.cumsum(0)
    offsets = torch.cat((torch.zeros_like(ends[:1]), ends[:-1]))
    place = torch.arange(flat.numel(), device=flat.device)
    columns = torch.where(place < offsets[G], order // k, -1)
    position = torch.empty_like(place).scatter_(0, order, place).view(-1, k)
    position = torch.where(experts < G, position, -1)
    return offsets.to(torch.int32), columns.to(torch.int32), position.to(torch.int32)


def _routing(gen, case, s):
    """What route gives for the case's own choice, its tokens in an order of the seed's."""
    N, k, G, live = case["N"], case["k"], case["G"], case["live"]
    top, _ = _chosen(case)
    perm = torch.randperm(live, device="cuda", generator=gen)
    experts = torch.full((N, k), G, device="cuda", dtype=torch.int64)
    experts[:live] = torch.from_numpy(top).cuda()[perm]
    s["offsets"], s["columns"], position = _order(experts, G, k)
    s["position"] = position.t()
    weights = torch.softmax(torch.randn((N, k), device="cuda", generator=gen), 1)
    s["weights"] = torch.where(experts < G, weights, 0.0).t()
    s["experts"] = torch.where(experts < G, experts, -1).to(torch.int32).t()


def _lens(case):
    R, L = case["R"], case["L"]
    return [L - (L // 2 * b) // R if case["ragged"] else L for b in range(R)]


def _ids(case, seed):
    """The pair of each request; every eighth has none."""
    return [-1 if b % 8 == 7 else (7 * b + seed) % case["n"] for b in range(case["R"])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op = _DTYPE[case["dtype"]], case["op"]
    s = {"case": case}
    if op == "route":
        N, G, k = case["N"], case["G"], case["k"]
        favour = 0.5 * torch.randn(G, device="cuda", generator=gen)
        s["logits"] = (torch.randn((N, G), device="cuda", generator=gen) + favour).to(dtype).t()
        s["bias"] = 0.1 * torch.randn(G, device="cuda", generator=gen) if case["bias"] else None
        s["mask"] = torch.arange(N, device="cuda") < case["live"] if case["live"] < N else None
        if case["train"]:
            s["dweights"] = torch.randn((N, k), device="cuda", generator=gen).t()
    elif op == "experts":
        N, G, k, M, K = (case[n] for n in ("N", "G", "k", "M", "K"))
        _routing(gen, case, s)
        s["A"] = _matrices(gen, M, K, G, dtype, case["turned"])
        s["X"] = _array(gen, K, N, dtype)
        s["most"] = _most(case)
        if case["train"]:
            s["dY"] = _array(gen, M, N * k, dtype)
    elif op == "combine":
        N, k, E = case["N"], case["k"], case["E"]
        _routing(gen, case, s)
        s["Y"] = _array(gen, E, N * k, dtype)
        if case["train"]:
            s["dy"] = _array(gen, E, N, dtype)
    else:
        M, K, r, n = (case[x] for x in ("M", "K", "r", "n"))
        lens = _lens(case)
        s["W"] = _matrices(gen, M, K, 1, dtype)[:, :, 0]
        s["A"], s["B"] = _matrices(gen, r, K, n, dtype), _matrices(gen, M, r, n, dtype)
        s["X"] = _array(gen, K, sum(lens), dtype)
        s["offsets"] = torch.tensor(np.concatenate(([0], np.cumsum(lens))), device="cuda", dtype=torch.int32)
        s["ids"] = torch.tensor(_ids(case, seed), device="cuda", dtype=torch.int32)
        s["scale"] = 0.5 + torch.rand(n, device="cuda", generator=gen)
        s["most"] = max(lens)
        if case["train"]:
            s["dY"] = _array(gen, M, sum(lens), dtype)
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _columns(t, dtype):
    """(N, E) as (E, N) in dtype."""
    return t.to(dtype).t()


def _plain_route(s, case):
    x, k, G = s["logits"].t().float(), case["k"], case["G"]                # (N, G)
    key = x if s["bias"] is None else x + s["bias"]
    top = key.sort(dim=1, descending=True, stable=True).indices[:, :k]     # the lowest index first among equals
    chosen = x.gather(1, top)
    if case["normalize"]:
        e = (chosen - chosen.amax(1, keepdim=True)).exp()
        w = e / e.sum(1, keepdim=True)
    else:
        e = (x - x.amax(1, keepdim=True)).exp()
        p = e / e.sum(1, keepdim=True)
        w = p.gather(1, top)
    live = None if s["mask"] is None else s["mask"][:, None]
    experts, weights = top, w
    if live is not None:
        experts, weights = torch.where(live, top, G), torch.where(live, w, 0.0)
    offsets, columns, position = _order(experts, G, k)
    out = (weights.t(), torch.where(experts < G, experts, -1).to(torch.int32).t(), offsets, columns, position.t())
    if not case["train"]:
        return out
    dw = s["dweights"].t()
    if live is not None:
        dw = torch.where(live, dw, 0.0)
    mean = (weights * dw).sum(1, keepdim=True)
    if case["normalize"]:
        dx = torch.zeros_like(x).scatter_(1, top, weights * (dw - mean))
    else:
        dx = p * (torch.zeros_like(x).scatter_(1, top, dw) - mean)
    return (*out, _columns(dx, s["logits"].dtype))


def _rows_of(s, n):
    """Padded groups: rows (groups, most) of the sorted order, which of them are there, and the group of each of n rows."""
    o = s["offsets"].long()
    row = o[:-1, None] + torch.arange(s["most"], device=o.device)
    there = row < o[1:, None]
    place = torch.arange(n, device=o.device)
    group = torch.searchsorted(o[1:].contiguous(), place, right=True)
    return torch.where(there, row, 0), there[..., None], group.clamp(max=o.numel() - 2), place


def _padded(rows, there, x):
    """Rows of x (n, E), in 32 bits, as (groups, most, E) with zeros behind a group's end."""
    return torch.where(there, x[rows].float(), 0.0)


def _unpadded(s, out, group, place):
    """(groups, most, E) as (n, E), zeros behind the last group."""
    o = s["offsets"].long()
    local = (place - o[group]).clamp(0, out.shape[1] - 1)
    return torch.where((place < o[-1])[:, None], out[group, local], 0.0)


def _gathered(x, position):
    """Sum of the rows of x that position (N, k) names, -1 for none: (N, k, E) before the sum."""
    return torch.where((position >= 0)[..., None], x[position.clamp(min=0).long()], 0.0)


def _plain_experts(s, case):
    dtype, k = s["X"].dtype, case["k"]
    rows, there, group, place = _rows_of(s, case["N"] * k)
    A = s["A"].permute(2, 0, 1).float()                                    # (G, M, K)
    x = _padded(s["columns"].long().clamp(min=0)[rows], there, s["X"].t())
    y = _unpadded(s, torch.matmul(x, A.transpose(1, 2)), group, place)
    if not case["train"]:
        return _columns(y, dtype)
    y = _columns(y, dtype)
    dy = _padded(rows, there, s["dY"].t())
    dA = torch.matmul(dy.transpose(1, 2), x).to(dtype).permute(1, 2, 0)
    dx = _unpadded(s, torch.matmul(dy, A), group, place)
    return y, dA, _columns(_gathered(dx, s["position"].t()).sum(1), dtype)


def _plain_combine(s, case):
    dtype, w = s["Y"].dtype, s["weights"].t()
    parts = _gathered(s["Y"].t().float(), s["position"].t())
    y = _columns((w[..., None] * parts).sum(1), dtype)
    if not case["train"]:
        return y
    dy = s["dy"].t().float()
    dw = (parts * dy[:, None]).sum(2)
    token = s["columns"].long().clamp(min=0)
    mine = s["position"].t()[token] == torch.arange(token.numel(), device=token.device)[:, None]
    share = torch.where(mine, w[token], 0.0).sum(1)
    share = torch.where(s["columns"] >= 0, share, 0.0)
    return y, _columns(share[:, None] * dy[token], dtype), dw.t()


def _plain_adapters(s, case):
    dtype, N = s["X"].dtype, s["X"].shape[1]
    rows, there, group, place = _rows_of(s, N)
    ids = s["ids"].long()
    use = (ids >= 0)[:, None, None]
    ids = ids.clamp(min=0)
    A, B = s["A"].permute(2, 1, 0)[ids].float(), s["B"].permute(2, 1, 0)[ids].float()      # (R, K, r), (R, r, M)
    scale = torch.where(use, s["scale"][ids][:, None, None], 0.0)
    x = _padded(rows, there, s["X"].t())
    t = scale * torch.matmul(x, A)
    W = s["W"].t().float()                                                                 # (K, M)
    y = torch.matmul(s["X"].t().float(), W) + _unpadded(s, torch.matmul(t, B), group, place)
    if not case["train"]:
        return _columns(y, dtype)
    dy = _padded(rows, there, s["dY"].t())
    dt = scale * torch.matmul(dy, B.transpose(1, 2))
    dx = torch.matmul(s["dY"].t().float(), W.t()) + _unpadded(s, torch.matmul(dt, A.transpose(1, 2)), group, place)
    of_A = torch.zeros((case["n"], *A.shape[1:]), device=x.device).index_add_(0, ids, torch.matmul(x.transpose(1, 2), dt))
    of_B = torch.zeros((case["n"], *B.shape[1:]), device=x.device).index_add_(0, ids, torch.matmul(t.transpose(1, 2), dy))
    return _columns(y, dtype), _columns(dx, dtype), of_A.to(dtype).permute(2, 1, 0), of_B.to(dtype).permute(2, 1, 0)


def _own(s, case):
    import nnlib_jl_b200 as nb
    op = case["op"]
    if op == "route":
        how = {"bias": s["bias"], "mask": s["mask"], "normalize": case["normalize"]}
        if not case["train"]:
            r = nb.route_topk(s["logits"], case["k"], **how)
            return r.weights, r.experts, r.offsets, r.columns, r.position
        r, back = nb.route_topk_pullback(s["logits"], case["k"], **how)
        return r.weights, r.experts, r.offsets, r.columns, r.position, back(s["dweights"])
    if op == "adapters":
        args, how = (s["W"], s["X"], s["A"], s["B"], s["ids"]), {"offsets": s["offsets"], "scale": s["scale"]}
        if not case["train"]:
            return nb.adapter_mul(*args, **how)
        y, back = nb.adapter_mul_pullback(*args, **how)
        return (y, *back(s["dY"]))
    r = nb.Routing(s["weights"], s["experts"], s["offsets"], s["columns"], s["position"])
    if op == "combine":
        if not case["train"]:
            return nb.combine(s["Y"], r)
        y, back = nb.combine_pullback(s["Y"], r)
        return (y, *back(s["dy"]))
    if not case["train"]:
        return nb.grouped_mul(s["A"], s["X"], r)
    y, back = nb.grouped_mul_pullback(s["A"], s["X"], r)
    return (y, *back(s["dY"]))


def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return {"route": _plain_route, "experts": _plain_experts, "combine": _plain_combine, "adapters": _plain_adapters}[case["op"]](s, case)


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    z, op, train = _BYTES[case["dtype"]], case["op"], case["train"]
    if op == "adapters":
        N, M, K, r = sum(_lens(case)), case["M"], case["K"], case["r"]
        pairs = len({i for i in _ids(case, 0) if i >= 0}) * r * (M + K)
        low = sum(n for n, i in zip(_lens(case), _ids(case, 0)) if i >= 0) * r * (M + K)
        # columns, matrix and pairs in, columns out; training: the cotangent in, gradients of columns and of all pairs out
        data = M * K + pairs + N * (K + M) + (N * (M + K) + case["n"] * r * (M + K) if train else 0)
        return {"bytes": z * data, "flops": (2 if train else 1) * 2.0 * N * M * K + (4 if train else 1) * 2.0 * low}
    N, G, k, live = case["N"], case["G"], case["k"], case["live"]
    if op == "route":
        index = N * k * 12 + N * k * 4 + 4 * (G + 1)
        return {"bytes": N * G * z * (2 if train else 1) + index + (4 * N * k if train else 0), "flops": 4.0 * N * G * (2 if train else 1)}
    if op == "combine":
        E, rows = case["E"], live * k
        # the tokens' columns in, their sums out; training: the cotangent in, the columns' gradient (of all rows) out
        return {"bytes": z * E * (rows + N) + 8 * N * k + (z * E * (N + N * k) + 8 * N * k if train else 0),
                "flops": 2.0 * rows * E * (3 if train else 1)}
    M, K, rows = case["M"], case["K"], live * k
    used = len(np.unique(_chosen(case)[0]))
    data = used * M * K + live * K + N * k * M
    if train:
        data += rows * M + G * M * K + N * K
    return {"bytes": z * data + 4 * (N * k + G + 1), "flops": 2.0 * rows * M * K * (3 if train else 1)}


# ---------------------------------------------------------------------------------------------------- 64 bits
def _exact_route(s, case):
    """Token by token's definition as one softmax over what may be chosen; the gradient as the Jacobian's product."""
    x, k = s["logits"].double().t(), case["k"]
    score = s["logits"].float().t()
    score = score if s["bias"] is None else score + s["bias"]
    order = torch.argsort(-score, dim=1, stable=True)[:, :k]
    among = torch.zeros_like(x, dtype=torch.bool).scatter_(1, order, True)
    logits = x.masked_fill(~among, -math.inf) if case["normalize"] else x
    p = torch.softmax(logits, 1)
    w = p.gather(1, order)
    if s["mask"] is not None:
        w = w * s["mask"][:, None]
    if not case["train"]:
        return w.t(), None, None, None, None
    d = torch.zeros_like(x).scatter_(1, order, s["dweights"].double().t())
    if s["mask"] is not None:
        d = d * s["mask"][:, None]
    inner = torch.einsum("ng,ng->n", p, d)[:, None]
    return w.t(), None, None, None, None, (p * d - p * inner).t()


def _exact_experts(s, case):
    """Expert by expert over its own tokens."""
    k, N, M, K = case["k"], case["N"], case["M"], case["K"]
    ends, token = s["offsets"].tolist(), s["columns"].long()
    y = torch.zeros((N * k, M), device="cuda", dtype=torch.float64)
    dx, dA = torch.zeros((N, K), device="cuda", dtype=torch.float64), []
    for g in range(case["G"]):
        mine = slice(ends[g], ends[g + 1])
        a, x = s["A"][:, :, g].double(), s["X"][:, token[mine]].double()
        y[mine] = (a @ x).t()
        if case["train"]:
            dy = s["dY"][:, mine].double()
            dA.append(dy @ x.t())
            dx.index_add_(0, token[mine], dy.t() @ a)
    return (y.t(), torch.stack(dA, 2), dx.t()) if case["train"] else y.t()


def _exact_combine(s, case):
    """Row by row of the sorted order, added to its token; a row's weight is that of the place that names it."""
    N, E, k = case["N"], case["E"], case["k"]
    Y = s["Y"].double().t()
    place = s["position"].t().reshape(-1).long()
    slot = torch.full((N * k,), -1, device="cuda", dtype=torch.int64)
    named = place >= 0
    slot[place[named]] = torch.arange(N * k, device="cuda")[named]
    rows = (slot >= 0).nonzero()[:, 0]
    token, w = slot[rows] // k, s["weights"].t().reshape(-1).double()[slot[rows]][:, None]
    y = torch.zeros((N, E), device="cuda", dtype=torch.float64).index_add_(0, token, w * Y[rows])
    if not case["train"]:
        return y.t()
    dy = s["dy"].double().t()[token]
    dY = torch.zeros_like(Y)
    dY[rows] = w * dy
    dw = torch.zeros(N * k, device="cuda", dtype=torch.float64)
    dw[slot[rows]] = torch.einsum("re,re->r", dy, Y[rows])
    return y.t(), dY.t(), dw.view(N, k).t()


def _exact_adapters(s, case):
    """Request by request: the matrix that its columns see is W + scale B A."""
    W, ends, ids = s["W"].double(), s["offsets"].tolist(), s["ids"].tolist()
    y, dx = [], []
    dA, dB = (torch.zeros(t.shape, device="cuda", dtype=torch.float64) for t in (s["A"], s["B"]))
    for b, i in enumerate(ids):
        x = s["X"][:, ends[b]:ends[b + 1]].double()
        A, B = s["A"][:, :, i].double(), s["B"][:, :, i].double()
        c = float(s["scale"][i]) if i >= 0 else 0.0
        seen = W + c * (B @ A)
        y.append(seen @ x)
        if case["train"]:
            dy = s["dY"][:, ends[b]:ends[b + 1]].double()
            dx.append(seen.t() @ dy)
            if i >= 0:
                outer = c * (dy @ x.t())                                   # the gradient of B A
                dA[:, :, i] += B.t() @ outer
                dB[:, :, i] += outer @ A.t()
    y = torch.cat(y, 1)
    return (y, torch.cat(dx, 1), dA, dB) if case["train"] else y


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "experts": _exact_experts, "combine": _exact_combine, "adapters": _exact_adapters}[case["op"]](s, case)
