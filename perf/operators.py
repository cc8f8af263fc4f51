"""The operators around the projections of a decoding step, as cases that can be timed and checked.

``tables``: the pages, slots and positions of a step's new tokens from the requests' lengths (``_C_ops.page_step``).
``append``: rotary positions on one or several axes for queries and keys, keys and values written into the paged
cache (``_C_ops.rotary_append``).  ``attention``: one new token per request over the paged cache
(``_C_ops.paged_attention``).  ``adapters``: low-rank adapters of many requests beside a shared projection
(``_C_ops.low_rank_add``).

``own`` chooses between the framework's kernels and the plain forms: elementary torch operations in 32 bits, rounded
once at the end.  Head layouts are those of the benchmark's projections (4096 -> 12288 is 32 + 2 x 32 heads of 128,
8192 -> 10240 is 64 + 2 x 8) and generic ragged ones.
"""
import math

import torch

own = False

DEV = "cuda"
F32, F64, I32, I64 = torch.float32, torch.float64, torch.int32, torch.int64
TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _tables(name, B, L, page, fresh):
    return {"name": name, "op": "tables", "B": B, "L": L, "page": page, "fresh": fresh}


def _append(name, T, Hq, Hkv, D, R, page, dtype, *, axes=1, interleaved=False, pad=0):
    return {"name": name, "op": "append", "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "R": R, "page": page, "dtype": dtype,
            "axes": axes, "interleaved": interleaved, "pad": pad}


def _attention(name, B, L, Hq, Hkv, D, page, dtype, *, ragged=True, window=0, lse=False):
    return {"name": name, "op": "attention", "B": B, "L": L, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype,
            "ragged": ragged, "window": window, "lse": lse}


def _adapters(name, T, K, N, E, R, dtype, *, used=0, mixed=False, runs=False):
    return {"name": name, "op": "adapters", "T": T, "K": K, "N": N, "E": E, "R": R, "dtype": dtype, "used": used or min(T, E),
            "mixed": mixed, "runs": runs}


def listed():
    return [
        # every request of a large decoding batch gets one more token: latency alone
        _tables("tables_decode_b256", 256, 4000, 16, 1),
        # a step that takes in prompts beside decoding requests, pages of no power of two
        _tables("tables_prompts_b61", 61, 9000, 24, 1500),
        # one token of each of 64 requests, fused QKV projection with 8 KV heads
        _append("append_decode_t64", 64, 64, 8, 128, 128, 16, "float16", pad=3),
        # prompts with images: three axes, every query head with a KV head of its own
        _append("append_prompt_3axes_t4096", 4096, 32, 32, 128, 128, 64, "bfloat16", axes=3),
        # one request at 1000 tokens: the smallest call a decoder makes
        _attention("attention_b1_l1000", 1, 1000, 32, 32, 128, 16, "float16", ragged=False),
        # an ordinary batch with lengths from nothing to 4096
        _attention("attention_b32_l4096", 32, 4096, 64, 8, 128, 16, "float16"),
        # odd sizes: five query heads a KV head, heads of 80, odd pages, a window
        _attention("attention_odd_window_b7", 7, 5555, 20, 4, 80, 24, "bfloat16", window=1000, lse=True),
        # two requests over a very long cache: the largest call
        _attention("attention_b2_l131072", 2, 131072, 64, 8, 128, 64, "bfloat16", ragged=False),
        # one request's adapter beside a QKV projection
        _adapters("adapters_decode_t1", 1, 4096, 12288, 8, 16, "float16"),
        # a decoding batch over twenty adapters of different ranks, some requests without one
        _adapters("adapters_decode_t64", 64, 8192, 10240, 32, 64, "float16", used=20, mixed=True),
        # an odd batch beside a projection of odd sizes
        _adapters("adapters_ragged_t77", 77, 2912, 1003, 12, 8, "bfloat16", used=12),
        # prompts of several requests, each with an adapter: the activations are what has to be moved
        _adapters("adapters_prompt_t4096", 4096, 4096, 12288, 16, 32, "bfloat16", used=6, runs=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "append", "attention", "attention", "attention", "adapters", "adapters", "adapters"])
    dtype = rng.choice(["float16", "bfloat16"])
    page = rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 128])
    Hkv = rng.choice([1, 2, 4, 5, 8, 8, 32])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 12, 16, 24])
    D = rng.choice([64, 64, 80, 96, 112, 128, 128, 128, 192, 256])
    if op == "tables":
        c = _tables("", _log_int(rng, 1, 1500), _log_int(rng, 1, 20000), page, rng.choice([1, _log_int(rng, 2, 1500)]))
    elif op == "append":
        if Hkv == 32:
            group = 1
        R = rng.choice([D, D, D // 2])
        c = _append("", _log_int(rng, 1, 4096), Hkv * group, Hkv, D, R, page, dtype, axes=rng.choice([1, 1, 2, 3]),
                    interleaved=rng.random() < 0.3, pad=rng.choice([0, 0, 1, 5]))
    elif op == "attention":
        if Hkv == 32:
            group = rng.choice([1, 2])
        B = _log_int(rng, 1, 200)
        most = 2 * 131072 * 8 * 128 // (B * Hkv * D)             # the padded cache of the largest listed call
        L = _log_int(rng, 1, max(1, min(131072, most // max(1, group // 8))))
        c = _attention("", B, L, Hkv * group, Hkv, D, page, dtype, ragged=rng.random() < 0.7,
                       window=rng.choice([0, 0, 0, 127, 1024]), lse=rng.random() < 0.3)
    else:
        K = 32 * _log_int(rng, 8, 448)
        N = _log_int(rng, 100, 22016)
        T = min(_log_int(rng, 1, 4096), max(1, 4096 * (4096 + 12288) // (K + N)))
        E = rng.choice([1, 2, 3, 8, 16, 32])
        R = rng.choice([8, 8, 16, 16, 16, 24, 32, 64, 128])
        c = _adapters("", T, K, N, E, R, dtype, used=min(T, rng.randint(1, E)), mixed=rng.random() < 0.3, runs=rng.random() < 0.5)
    del c["name"]
    return c


# ---- sizes that follow from a case ----------------------------------------------------------------------------------
def _lengths(case):
    """Cached tokens of the requests, the same multiset for every seed: log-spread up to L, with an empty one."""
    B, L = case["B"], case["L"]
    if case["op"] == "attention" and not case["ragged"]:
        return [L] * B
    got = [max(1, round(L ** ((i + 1) / B))) for i in range(B)]
    return [0] + got[1:] if B >= 4 else got


def _fresh(case):
    """New tokens of the requests: one each, or (more than one) prompts for every third request and nothing for every eleventh."""
    n = case["fresh"]
    return [1 if n == 1 else 0 if i % 11 == 10 else n - i % 7 if i % 3 == 0 and n > 7 else 1 for i in range(case["B"])]


def _ranks(case):
    """Ranks of the adapters that are in use: all R, or from R / 8 (eight at least) to R."""
    R = case["R"]
    return [max(8, R >> (i % 4)) // 8 * 8 if case["mixed"] else R for i in range(case["E"])]


def _sections(case):
    half, n = case["R"] // 2, case["axes"]
    return [half - half // n * (n - 1)] + [half // n] * (n - 1)


def work(case):
    if case["op"] == "tables":
        P = case["page"]
        pairs = list(zip(_lengths(case), _fresh(case)))
        T, new = sum(f for _, f in pairs), sum(-(-(c + f) // P) + -c // P for c, f in pairs)
        return {"bytes": 16 * case["B"] + 8 * new + 16 * T, "flops": 0}
    if case["op"] == "append":
        T, D, heads = case["T"], case["D"], case["Hq"] + 2 * case["Hkv"]
        return {"bytes": 4 * T * D * heads + T * (8 + 4 * case["axes"] + 4 * case["R"]),
                "flops": 3 * T * case["R"] * (case["Hq"] + case["Hkv"])}
    if case["op"] == "attention":
        keys = sum(min(n, case["window"] or n) for n in _lengths(case))
        return {"bytes": 4 * keys * case["Hkv"] * case["D"] + 4 * case["B"] * case["Hq"] * case["D"] + 4 * keys // case["page"],
                "flops": 4 * keys * case["Hq"] * case["D"]}
    T, K, N = case["T"], case["K"], case["N"]
    ranks = _ranks(case)[:case["used"]]
    return {"bytes": 2 * T * (K + 2 * N) + 2 * sum(ranks) * (K + N) + 4 * T, "flops": 2 * T * (K + N) * sum(ranks) // len(ranks)}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _shuffled(values, g):
    v = torch.tensor(values, dtype=I32, device=DEV)
    return v[torch.randperm(len(values), generator=g, device=DEV)]


def _pool(lengths, page, extra, width, g):
    """Block table [B, width] of pages in no order, -1 where a request has none; the pages that are left."""
    B, have = lengths.numel(), (lengths + page - 1) // page
    perm = torch.randperm(int(have.sum()) + extra, generator=g, device=DEV).to(I32)
    col = torch.arange(width, device=DEV)
    at = (have.cumsum(0) - have).unsqueeze(1) + col
    return torch.where(col < have.unsqueeze(1), perm[at.clamp(max=perm.numel() - 1)], -1).to(I32), perm[int(have.sum()):].contiguous()


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] == "tables":
        P, B = case["page"], case["B"]
        at = torch.randperm(B, generator=g, device=DEV)
        cached, fresh = (torch.tensor(v(case), dtype=I32, device=DEV)[at] for v in (_lengths, _fresh))
        total = int(fresh.sum())
        width = -(-(case["L"] + case["fresh"]) // P) + 3
        s["cached"], s["fresh"] = cached, fresh
        s["table"], s["free"] = _pool(cached, P, total + 40, width, g)
        s["available"] = torch.tensor([s["free"].numel() - 7], dtype=I32, device=DEV)
        s["tokens"] = total + 5                    # a step of fixed size: some places stay empty
        # lengths, starts, slots, positions, requests, counts: kept by the program from step to step
        s["step"] = tuple(torch.empty(n, dtype=I64 if i == 2 else I32, device=DEV)
                          for i, n in enumerate((B, B + 1, total + 5, total + 5, total + 5, 3)))
        return s
    dtype = TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype).mul_(std)

    if case["op"] == "append":
        T, Hq, Hkv, D, R, P = (case[k] for k in ("T", "Hq", "Hkv", "D", "R", "page"))
        qkv = normal(T, (Hq + 2 * Hkv) * D)        # as the fused projection leaves them
        s["q"] = qkv[:, :Hq * D].view(T, Hq, D)
        s["k"] = qkv[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
        s["v"] = qkv[:, (Hq + Hkv) * D:].view(T, Hkv, D)
        pages = -(-(T + 100) // P)
        s["k_cache"], s["v_cache"] = normal(pages, P, Hkv, D), normal(pages, P, Hkv, D)
        slots = torch.randperm(pages * P, generator=g, device=DEV)[:T]
        pad = min(case["pad"], T - 1)
        if pad:
            slots[T - pad:] = -1
        s["slots"] = slots
        span = 8192
        inv = 10000.0 ** (-torch.arange(0, R // 2, dtype=F64, device=DEV) * 2 / R)
        angle = torch.arange(span, dtype=F64, device=DEV).unsqueeze(1) * inv
        s["table"] = torch.cat((angle.cos(), angle.sin()), dim=1).to(F32)
        shape = (T,) if case["axes"] == 1 else (case["axes"], T)
        s["positions"] = torch.randint(0, span, shape, generator=g, device=DEV, dtype=I32)
        s["sections"] = _sections(case)
        return s
    if case["op"] == "attention":
        B, Hq, Hkv, D, P = (case[k] for k in ("B", "Hq", "Hkv", "D", "page"))
        s["lengths"] = _shuffled(_lengths(case), g)
        width = -(-case["L"] // P)
        s["table"], left = _pool(s["lengths"], P, 3, width, g)
        pages = int(((s["lengths"] + P - 1) // P).sum()) + 3
        s["q"] = normal(B, Hq, D, std=2.0)
        s["k_cache"], s["v_cache"] = normal(pages, P, Hkv, D), normal(pages, P, Hkv, D)
        s["scale"] = D ** -0.5
        s["lse"] = torch.empty(B, Hq, device=DEV) if case["lse"] else None
        return s
    T, K, N, E, R = (case[k] for k in ("T", "K", "N", "E", "R"))
    s["x"], s["y"] = normal(T, K), normal(T, N)
    s["down"], s["up"] = normal(E, R, K, std=K ** -0.5), normal(E, N, R, std=0.5 * R ** -0.5)
    ranks = torch.tensor(_ranks(case), dtype=I32, device=DEV)
    s["ranks"] = ranks if case["mixed"] else None
    unused = torch.arange(R, device=DEV) >= ranks.unsqueeze(1)
    s["down"].masked_fill_(unused.unsqueeze(2), 0)
    s["up"].masked_fill_(unused.unsqueeze(1), 0)
    s["scales"] = torch.rand(E, generator=g, device=DEV) + 0.5
    # adapters of the tokens: in runs (prompts) or in no order, each in use at least once, some tokens without one
    at = torch.arange(T, device=DEV)
    ids = at * case["used"] // T if case["runs"] else at % case["used"]
    if not case["runs"]:
        ids = torch.where((at % 13 == 12) & (at >= case["used"]), -1, ids)[torch.randperm(T, generator=g, device=DEV)]
    s["ids"] = ids.to(I32)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def _plain_tables(s):
    P, T, table, free = s["case"]["page"], s["tokens"], s["table"], s["free"]
    c, f = s["cached"].clamp(min=0).long(), s["fresh"].clamp(min=0).long()
    B, W = table.shape
    have, want = (c + P - 1) // P, (c + f + P - 1) // P
    ends, pages = f.cumsum(0), (want - have).cumsum(0)
    starts, pages0 = ends - f, pages - (want - have)
    n = s["available"].clamp(0, free.numel()).long()

    def page(i):
        return torch.where((i >= 0) & (i < n), free[(n - 1 - i).clamp(0, free.numel() - 1)], -1)

    t = torch.arange(T, device=DEV)
    valid = t < ends[-1]
    b = torch.searchsorted(ends, t, right=True).clamp(max=B - 1)
    pos = c[b] + t - starts[b]
    col = pos // P
    pg = torch.where(col < have[b], table[b, col.clamp(max=W - 1)], page(pages0[b] + col - have[b])).long()
    slots = torch.where(valid & (col < W) & (pg >= 0), pg * P + pos % P, -1)
    j = torch.arange(W, device=DEV)
    new = page(pages0.unsqueeze(1) + j - have.unsqueeze(1))
    put = (j >= have.unsqueeze(1)) & (j < want.unsqueeze(1)) & (new >= 0)
    table.copy_(torch.where(put, new, table))
    counts = torch.stack((ends[-1], pages[-1], (n[0] - pages[-1]).clamp(min=0))).to(I32)
    return {"lengths": (c + f).to(I32), "starts": torch.cat((starts, ends[-1:])).to(I32), "slots": slots,
            "positions": torch.where(valid, pos, -1).to(I32), "requests": torch.where(valid, b, -1).to(I32), "counts": counts, "table": table}


def _rotate(x, cos, sin, R, interleaved):
    x = x.float()
    r, rest = x[..., :R], x[..., R:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :R // 2], r[..., R // 2:])
    lo, hi = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((lo, hi), dim=-1).flatten(-2) if interleaved else torch.cat((lo, hi), dim=-1)
    return torch.cat((r, rest), dim=-1)


def _plain_append(s):
    case, T = s["case"], s["case"]["T"]
    R, dtype = case["R"], TYPES[case["dtype"]]
    axis = torch.repeat_interleave(torch.arange(case["axes"], device=DEV), torch.tensor(s["sections"], device=DEV), output_size=R // 2)
    p = s["positions"].view(case["axes"], T)[axis].T.long()                              # [T, R / 2]
    i = torch.arange(R // 2, device=DEV)
    cos, sin = s["table"][p, i].unsqueeze(1), s["table"][p, R // 2 + i].unsqueeze(1)
    q = _rotate(s["q"], cos, sin, R, case["interleaved"]).to(dtype)
    k = _rotate(s["k"], cos, sin, R, case["interleaved"]).to(dtype)
    kept = s["slots"] >= 0
    at = s["slots"][kept]
    s["k_cache"].view(-1, case["Hkv"], case["D"])[at] = k[kept]
    s["v_cache"].view(-1, case["Hkv"], case["D"])[at] = s["v"][kept]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    case, q = s["case"], s["q"]
    B, Hq, Hkv, D = (case[k] for k in ("B", "Hq", "Hkv", "D"))
    pages = s["table"].clamp(min=0).long()
    k = s["k_cache"][pages].view(B, -1, Hkv, D).permute(0, 2, 3, 1).float()              # [B, Hkv, D, W * page]
    j = torch.arange(k.shape[-1], device=DEV)
    n = s["lengths"].view(B, 1)
    seen = (j < n) & (j >= n - case["window"]) if case["window"] else j < n
    seen = seen.view(B, 1, 1, -1)
    score = torch.matmul(q.float().view(B, Hkv, Hq // Hkv, D), k) * s["scale"]
    del k
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = torch.where(seen, torch.exp(score - top), 0)
    total = p.sum(dim=-1, keepdim=True)
    v = s["v_cache"][pages].view(B, -1, Hkv, D).permute(0, 2, 1, 3).float()
    out = torch.matmul(p, v)
    out = torch.where(total > 0, out / total, 0).view(B, Hq, D).to(q.dtype)
    if not case["lse"]:
        return out
    return out, torch.where(total > 0, top + torch.log(total), -torch.inf).view(B, Hq)


def _plain_adapters(s):
    T, E, R = s["case"]["T"], s["case"]["E"], s["case"]["R"]
    mine = (s["ids"].view(T, 1) == torch.arange(E, device=DEV)) * s["scales"]            # [T, E]
    v = torch.matmul(s["x"].float(), s["down"].float().view(E * R, -1).T).view(T, E, R) * mine.unsqueeze(2)
    d = torch.matmul(v.view(T, E * R), s["up"].float().transpose(1, 2).reshape(E * R, -1))
    return (s["y"].float() + d).to(s["y"].dtype)


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"tables": _plain_tables, "append": _plain_append, "attention": _plain_attention, "adapters": _plain_adapters}[case["op"]](s)
    from libortho_b200 import _C_ops
    if case["op"] == "tables":
        r = _C_ops.page_step(s["cached"], s["fresh"], s["table"], s["free"], s["available"], case["page"], s["tokens"], out=s["step"])
        return {"lengths": r.lengths, "starts": r.starts, "slots": r.slots, "positions": r.positions, "requests": r.requests,
                "counts": r.counts, "table": s["table"]}
    if case["op"] == "append":
        q = _C_ops.rotary_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["positions"], s["table"],
                                 sections=s["sections"], interleaved=case["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["op"] == "attention":
        out = _C_ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], scale=s["scale"],
                                     window=case["window"], lse=s["lse"])
        return (out, s["lse"]) if case["lse"] else out
    return _C_ops.low_rank_add(s["x"], s["y"], s["down"], s["up"], s["ids"], scales=s["scales"], ranks=s["ranks"])


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _exact_append(s):
    case = s["case"]
    T, R, D = case["T"], case["R"], case["D"]
    half, bounds = R // 2, [0]
    for n in s["sections"]:
        bounds.append(bounds[-1] + n)
    cos, sin = torch.empty(T, 1, half, dtype=F64, device=DEV), torch.empty(T, 1, half, dtype=F64, device=DEV)
    for a in range(case["axes"]):
        rows = s["table"].double()[s["positions"].view(case["axes"], T)[a].long()]
        lo, hi = bounds[a], bounds[a + 1]
        cos[:, 0, lo:hi], sin[:, 0, lo:hi] = rows[:, lo:hi], rows[:, half + lo:half + hi]
    first = torch.arange(half, device=DEV) * 2 if case["interleaved"] else torch.arange(half, device=DEV)
    second = first + (1 if case["interleaved"] else half)
    turned = []
    for x in (s["q"].double(), s["k"].double()):
        y = x.clone()
        y[..., first] = x[..., first] * cos - x[..., second] * sin
        y[..., second] = x[..., first] * sin + x[..., second] * cos
        turned.append(y)
    P = case["page"]
    caches = [s["k_cache"].double(), s["v_cache"].double()]
    keep = (s["slots"] >= 0).nonzero()[:, 0]
    page, place = s["slots"][keep] // P, s["slots"][keep] % P
    caches[0][page, place], caches[1][page, place] = turned[1][keep], s["v"].double()[keep]
    return {"q": turned[0], "k_cache": caches[0], "v_cache": caches[1]}


def _exact_attention(s):
    case = s["case"]
    B, Hq, Hkv, D, P = (case[k] for k in ("B", "Hq", "Hkv", "D", "page"))
    out = torch.zeros(B, Hq, D, dtype=F64, device=DEV)
    lse = torch.full((B, Hq), -math.inf, dtype=F64, device=DEV)
    for b, n in enumerate(s["lengths"].tolist()):
        lo = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        pages = s["table"][b, lo // P:-(-n // P)].long()
        cut = slice(lo - lo // P * P, n - lo // P * P)
        for h in range(Hkv):
            heads = slice(h * Hq // Hkv, (h + 1) * Hq // Hkv)
            k, v = (c[pages, :, h].reshape(-1, D)[cut].double() for c in (s["k_cache"], s["v_cache"]))
            score = (k @ s["q"][b, heads].double().T) * s["scale"]                       # [keys, group]
            lse[b, heads] = torch.logsumexp(score, dim=0)
            out[b, heads] = torch.softmax(score, dim=0).T @ v
    return (out, lse) if case["lse"] else out


def _exact_adapters(s):
    out = s["y"].double()
    for e in range(s["case"]["E"]):
        rows = (s["ids"] == e).nonzero()[:, 0]
        if rows.numel():
            out[rows] += float(s["scales"][e]) * (s["x"][rows].double() @ s["down"][e].double().T @ s["up"][e].double().T)
    return out


def exact(case, seed):
    if case["op"] == "tables":                     # whole numbers only
        return None
    return {"append": _exact_append, "attention": _exact_attention, "adapters": _exact_adapters}[case["op"]](prepare(case, seed))
