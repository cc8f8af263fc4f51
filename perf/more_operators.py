"""The operators of a paged key-value cache held in 4 bits, as cases that can be timed and checked.

``append``: rotary positions for queries and keys, keys and values quantised as they are written
(``_C_ops.rotary_append_quantised``), then the cache read back.  ``read``: cached tokens read back to 16 bits
(``_C_ops.read_quantised``), as a prompt's next chunk needs its prefix.  ``attention``: one new token per request over the
cache (``_C_ops.paged_attention_quantised``).

A group of elements (a whole head, or 64 elements of one) of a token is held as 4-bit codes with a scale and a zero in the model's type:
``value = zero + scale * code``; ``zero`` is the group's least value and ``scale`` a 15th of its range, both rounded to the type,
``code = rint((x - zero) / scale)`` within 0 to 15.  Two codes a byte, the even element in the low half.

``own`` chooses between the framework's kernels and the plain forms: elementary torch operations in 32 bits (codes: in 64, they are
values next to a border), rounded once at the end.  Head layouts are those of the benchmark's projections
(8192 -> 10240 is 64 + 2 x 8 heads of 128, 4096 -> 12288 is 32 + 2 x 32) and generic ragged ones.
"""
import math

import torch

own = False

DEV = "cuda"
F32, F64, I32, I64, U8 = torch.float32, torch.float64, torch.int32, torch.int64, torch.uint8
TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _append(name, T, Hq, Hkv, D, R, page, dtype, *, groups=1, axes=1, interleaved=False, pad=0):
    return {"name": name, "op": "append", "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "R": R, "page": page, "dtype": dtype,
            "groups": groups, "axes": axes, "interleaved": interleaved, "pad": pad}


def _read(name, T, Hkv, D, page, dtype, *, groups=1):
    return {"name": name, "op": "read", "T": T, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype, "groups": groups}


def _attention(name, B, L, Hq, Hkv, D, page, dtype, *, groups=1, ragged=True, window=0, lse=False):
    return {"name": name, "op": "attention", "B": B, "L": L, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype,
            "groups": groups, "ragged": ragged, "window": window, "lse": lse}


def listed():
    return [
        # one token of each of 64 requests behind a fused QKV projection with 8 KV heads, some places without a token
        _append("append_decode_t64", 64, 64, 8, 128, 128, 16, "float16", pad=3),
        # odd heads of which a part turns, pairs side by side, pages of no power of two
        _append("append_ragged_t77", 77, 20, 4, 80, 48, 24, "bfloat16", interleaved=True),
        # prompts with images: three axes, a scale for every 64 elements, every query head with a KV head of its own
        _append("append_prompt_3axes_t4096", 4096, 32, 32, 128, 128, 64, "bfloat16", groups=2, axes=3),
        # the prefix of a short conversation for its next chunk
        _read("read_prefix_t1003", 1003, 8, 128, 16, "float16"),
        # a document's prefix
        _read("read_document_t65536", 65536, 8, 128, 64, "bfloat16", groups=2),
        # one request at 1000 tokens: the smallest call a decoder makes
        _attention("attention_b1_l1000", 1, 1000, 32, 32, 128, 16, "float16", ragged=False),
        # an ordinary batch with lengths from nothing to 4096
        _attention("attention_b32_l4096", 32, 4096, 64, 8, 128, 16, "float16"),
        # odd sizes: five query heads a KV head, heads of 80, odd pages, a window
        _attention("attention_odd_window_b7", 7, 5555, 20, 4, 80, 24, "bfloat16", window=1000, lse=True),
        # a large batch with a scale for every 64 elements
        _attention("attention_groups_b100_l8000", 100, 8000, 32, 8, 128, 32, "bfloat16", groups=2, lse=True),
        # wide heads, many queries a KV head
        _attention("attention_wide_b16_l10000", 16, 10000, 32, 2, 256, 16, "bfloat16"),
        # two requests over a very long cache: the largest call
        _attention("attention_b2_l131072", 2, 131072, 64, 8, 128, 64, "float16", ragged=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "read", "attention", "attention", "attention", "attention"])
    dtype = rng.choice(["float16", "bfloat16"])
    page = rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 128])
    Hkv = rng.choice([1, 2, 4, 5, 8, 8, 32])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 12, 16, 24])
    D = rng.choice([64, 64, 72, 80, 96, 112, 128, 128, 128, 192, 256])
    groups = rng.choice([1, D // 64]) if D % 64 == 0 else 1
    if op == "append":
        if Hkv == 32:
            group = 1
        most = max(8, 4096 * 96 * 128 // ((group + 2) * Hkv * D))
        c = _append("", _log_int(rng, 1, min(4096, most)), Hkv * group, Hkv, D, rng.choice([D, D, D // 16 * 8]), page, dtype, groups=groups,
                    axes=rng.choice([1, 1, 2, 3]), interleaved=rng.random() < 0.3, pad=rng.choice([0, 0, 1, 5]))
    elif op == "read":
        c = _read("", _log_int(rng, 1, 65536 * 8 * 128 // (Hkv * D)), Hkv, D, page, dtype, groups=groups)
    else:
        if Hkv == 32:
            group = rng.choice([1, 2])
        B = _log_int(rng, 1, 200)
        most = 2 * 131072 * 8 * 128 // (B * Hkv * D)             # the padded cache of the largest listed call
        L = _log_int(rng, 1, max(1, min(131072, most // max(1, group // 8))))
        c = _attention("", B, L, Hkv * group, Hkv, D, page, dtype, groups=groups, ragged=rng.random() < 0.7,
                       window=rng.choice([0, 0, 0, 127, 1024]), lse=rng.random() < 0.3)
    del c["name"]
    return c


# ---- sizes that follow from a case ----------------------------------------------------------------------------------
def _lengths(case):
    """Cached tokens of the requests, the same multiset for every seed: log-spread up to L, with an empty one."""
    B, L = case["B"], case["L"]
    if not case["ragged"]:
        return [L] * B
    got = [max(1, round(L ** ((i + 1) / B))) for i in range(B)]
    return [0] + got[1:] if B >= 4 else got


def _sections(case):
    half, n = case["R"] // 2, case["axes"]
    return [half - half // n * (n - 1)] + [half // n] * (n - 1)


def _pages(case):
    return -(-(case["T"] + 100) // case["page"])


def work(case):
    Hkv, D = case["Hkv"], case["D"]
    held = Hkv * (D + 8 * case["groups"])                        # a token's keys and values with their scales and zeros
    if case["op"] == "append":
        T, n = case["T"], _pages(case) * case["page"]
        return {"bytes": 4 * T * D * case["Hq"] + 4 * T * D * Hkv + T * (8 + 4 * case["axes"] + 4 * case["R"]) + T * held + n * (held + 4 * Hkv * D + 8),
                "flops": 3 * T * case["R"] * (case["Hq"] + Hkv) + 8 * (T + n) * Hkv * D}
    if case["op"] == "read":
        return {"bytes": case["T"] * (8 + held + 4 * Hkv * D), "flops": 4 * case["T"] * Hkv * D}
    keys = sum(min(n, case["window"] or n) for n in _lengths(case))
    return {"bytes": keys * held + 4 * case["B"] * case["Hq"] * D + 4 * keys // case["page"], "flops": 4 * keys * case["Hq"] * D}


# ---- the format, in plain operations ----------------------------------------------------------------------------------
def _round(x, dtype):
    """64 bits to 16, rounded once (by way of 32 bits, rounded to odd)."""
    f = x.float()
    bits = f.view(I32) - (f.double().abs() > x.abs()).to(I32)
    return (bits | (f.double() != x).to(I32)).view(F32).to(dtype)


def _quantise(x, groups, dtype):
    """x [..., D] in 64 bits -> codes [..., D / 2], scales and zeros [..., groups, 2]."""
    g = x.view(*x.shape[:-1], groups, -1)
    lo, hi = g.amin(dim=-1), g.amax(dim=-1)
    held = torch.stack((_round((hi - lo) / 15, dtype), _round(lo, dtype)), dim=-1)
    scale, zero = held.double().unsqueeze(-2).unbind(-1)
    code = torch.where(scale > 0, ((g - zero) / scale).round().clamp(0, 15), 0).to(U8).view(x.shape)
    return code[..., 0::2] | code[..., 1::2] << 4, held


def _values(codes, held):
    """Codes [..., D / 2] with scales and zeros [..., groups, 2] -> values [..., D] in 32 bits."""
    c = torch.stack((codes & 15, codes >> 4), dim=-1).float()
    c = c.view(*codes.shape[:-1], held.shape[-2], -1)
    held = held.float()
    return (c * held[..., :1] + held[..., 1:]).flatten(-2)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _cache(pages, case, dtype, g):
    """Codes and scales of keys and values of normal tokens; a key's channels differ in size as they do in a model.
    A page lies head by head."""
    P, H, D, G = case["page"], case["Hkv"], case["D"], case["groups"]
    got = []
    for channels in (True, False):
        codes = torch.empty(pages, H, P, D // 2, dtype=U8, device=DEV)
        held = torch.empty(pages, H, P, G, 2, dtype=dtype, device=DEV)
        size = torch.randn(H, 1, D, generator=g, device=DEV).mul_(0.5).exp_() if channels else 1.0
        step = max(1, (1 << 26) // (P * H * D))
        for i in range(0, pages, step):
            x = (torch.randn(min(step, pages - i), H, P, D, generator=g, device=DEV) * size).view(-1, H, P, G, D // G)
            lo, hi = x.amin(dim=-1), x.amax(dim=-1)
            h = torch.stack(((hi - lo) / 15, lo), dim=-1).to(dtype)
            scale, zero = h.float().unsqueeze(-2).unbind(-1)
            c = ((x - zero) / scale).round_().clamp_(0, 15).to(U8).view(-1, H, P, D)
            codes[i:i + step] = c[..., 0::2] | c[..., 1::2] << 4
            held[i:i + step] = h
        got.append((codes.transpose(1, 2), held.transpose(1, 2)))
    return got


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    dtype = TYPES[case["dtype"]]
    Hkv, D, P = case["Hkv"], case["D"], case["page"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype).mul_(std)

    if case["op"] == "attention":
        B, Hq = case["B"], case["Hq"]
        lengths = torch.tensor(_lengths(case), dtype=I32, device=DEV)
        s["lengths"] = lengths = lengths[torch.randperm(B, generator=g, device=DEV)]
        have = (lengths + P - 1) // P
        pages = int(have.sum()) + 3
        perm = torch.randperm(pages, generator=g, device=DEV).to(I32)
        col = torch.arange(-(-case["L"] // P), device=DEV)
        at = (have.cumsum(0) - have).unsqueeze(1) + col
        s["table"] = torch.where(col < have.unsqueeze(1), perm[at.clamp(max=pages - 1)], -1).to(I32)
        s["q"] = normal(B, Hq, D, std=1.5)
        s["scale"] = D ** -0.5
        s["lse"] = torch.empty(B, Hq, device=DEV) if case["lse"] else None
        (s["k_cache"], s["k_scales"]), (s["v_cache"], s["v_scales"]) = _cache(pages, case, dtype, g)
        return s
    T, pages = case["T"], _pages(case)
    (s["k_cache"], s["k_scales"]), (s["v_cache"], s["v_scales"]) = _cache(pages, case, dtype, g)
    if case["op"] == "read":
        slots = torch.arange(T, device=DEV)
        s["slots"] = torch.randperm(pages, generator=g, device=DEV)[slots // P] * P + slots % P     # a request's pages, in no order
        return s
    Hq, R = case["Hq"], case["R"]
    qkv = normal(T, (Hq + 2 * Hkv) * D)            # as the fused projection leaves them
    s["q"] = qkv[:, :Hq * D].view(T, Hq, D)
    s["k"] = qkv[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
    s["v"] = qkv[:, (Hq + Hkv) * D:].view(T, Hkv, D)
    slots = torch.randperm(pages * P, generator=g, device=DEV)[:T]
    pad = min(case["pad"], T - 1)
    if pad:
        slots[T - pad:] = -1
    s["slots"], s["all"] = slots, torch.arange(pages * P, device=DEV)
    span = 8192
    inv = 10000.0 ** (-torch.arange(0, R // 2, dtype=F64, device=DEV) * 2 / R)
    angle = torch.arange(span, dtype=F64, device=DEV).unsqueeze(1) * inv
    s["table"] = torch.cat((angle.cos(), angle.sin()), dim=1).to(F32)
    s["positions"] = torch.randint(0, span, (T,) if case["axes"] == 1 else (case["axes"], T), generator=g, device=DEV, dtype=I32)
    s["sections"] = _sections(case)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def _rotate(x, cos, sin, R, interleaved):
    r, rest = x[..., :R], x[..., R:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :R // 2], r[..., R // 2:])
    lo, hi = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((lo, hi), dim=-1).flatten(-2) if interleaved else torch.cat((lo, hi), dim=-1)
    return torch.cat((r, rest), dim=-1)


def _plain_append(s):
    case, T = s["case"], s["case"]["T"]
    R, P, G, dtype = case["R"], case["page"], case["groups"], TYPES[case["dtype"]]
    axis = torch.repeat_interleave(torch.arange(case["axes"], device=DEV), torch.tensor(s["sections"], device=DEV), output_size=R // 2)
    p = s["positions"].view(case["axes"], T)[axis].T.long()                              # [T, R / 2]
    i = torch.arange(R // 2, device=DEV)
    cos, sin = s["table"][p, i].unsqueeze(1), s["table"][p, R // 2 + i].unsqueeze(1)
    q = _rotate(s["q"].float(), cos, sin, R, case["interleaved"]).to(dtype)
    k = _rotate(s["k"].double(), cos.double(), sin.double(), R, case["interleaved"])
    kept = s["slots"] >= 0
    page, place = s["slots"][kept] // P, s["slots"][kept] % P
    s["k_cache"][page, place], s["k_scales"][page, place] = _quantise(k[kept], G, dtype)
    s["v_cache"][page, place], s["v_scales"][page, place] = _quantise(s["v"].double()[kept], G, dtype)
    k, v = _plain_read(s, s["all"])
    return {"q": q, "k": k, "v": v}


def _plain_read(s, slots):
    P, dtype = s["case"]["page"], TYPES[s["case"]["dtype"]]
    page, place = slots // P, slots % P
    return (_values(s["k_cache"][page, place], s["k_scales"][page, place]).to(dtype),
            _values(s["v_cache"][page, place], s["v_scales"][page, place]).to(dtype))


def _plain_attention(s):
    case, q = s["case"], s["q"]
    B, Hq, Hkv, D = (case[k] for k in ("B", "Hq", "Hkv", "D"))
    pages = s["table"].clamp(min=0).long()
    k = _values(s["k_cache"][pages], s["k_scales"][pages]).view(B, -1, Hkv, D).permute(0, 2, 3, 1)      # [B, Hkv, D, W * page]
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
    v = _values(s["v_cache"][pages], s["v_scales"][pages]).view(B, -1, Hkv, D).permute(0, 2, 1, 3)
    out = torch.matmul(p, v)
    out = torch.where(total > 0, out / total, 0).view(B, Hq, D).to(q.dtype)
    if not case["lse"]:
        return out
    return out, torch.where(total > 0, top + torch.log(total), -torch.inf).view(B, Hq)


def run(state):
    s, case = state, state["case"]
    if not own:
        if case["op"] == "read":
            k, v = _plain_read(s, s["slots"])
            return {"k": k, "v": v}
        return _plain_append(s) if case["op"] == "append" else _plain_attention(s)
    from libortho_b200 import _C_ops
    cache = s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"]
    if case["op"] == "attention":
        out = _C_ops.paged_attention_quantised(s["q"], *cache, s["table"], s["lengths"], scale=s["scale"], window=case["window"], lse=s["lse"])
        return (out, s["lse"]) if case["lse"] else out
    if case["op"] == "read":
        k, v = _C_ops.read_quantised(*cache, s["slots"])
        return {"k": k, "v": v}
    q = _C_ops.rotary_append_quantised(s["q"], s["k"], s["v"], *cache, s["slots"], s["positions"], s["table"],
                                       sections=s["sections"], interleaved=case["interleaved"])
    k, v = _C_ops.read_quantised(*cache, s["all"])
    return {"q": q, "k": k, "v": v}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _nearest(x, dtype):
    """The value of a 16-bit type next to x, ties to even, in 64 bits."""
    digits, least = (11, -13) if dtype == torch.float16 else (8, -125)
    e = torch.frexp(x)[1].clamp(min=least) - digits
    return torch.ldexp(torch.round(torch.ldexp(x, -e)), e)


def _held_of(codes, held):
    """What a cache holds, in 64 bits, [pages, page, heads, D]."""
    out = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=F64, device=DEV)
    out[..., 0::2], out[..., 1::2] = codes % 16, codes // 16
    width = out.shape[-1] // held.shape[-2]
    for g in range(held.shape[-2]):
        part = out[..., g * width:(g + 1) * width]
        part.mul_(held[..., g, :1].double()).add_(held[..., g, 1:].double())
    return out


def _put(x, G, dtype):
    """What the cache stands for once x [..., D] in 64 bits has been written to it."""
    out = torch.empty_like(x)
    width = x.shape[-1] // G
    for g in range(G):
        part = x[..., g * width:(g + 1) * width]
        lo = part.min(dim=-1, keepdim=True)[0]
        scale, zero = _nearest((part.max(dim=-1, keepdim=True)[0] - lo) / 15, dtype), _nearest(lo, dtype)
        code = torch.round((part - zero) / torch.where(scale > 0, scale, 1)).clamp(0, 15) * (scale > 0)
        out[..., g * width:(g + 1) * width] = code * scale + zero
    return out


def _exact_append(s):
    case = s["case"]
    T, R, P = case["T"], case["R"], case["page"]
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
    k, v = _held_of(s["k_cache"], s["k_scales"]), _held_of(s["v_cache"], s["v_scales"])
    keep = (s["slots"] >= 0).nonzero()[:, 0]
    page, place = s["slots"][keep] // P, s["slots"][keep] % P
    k[page, place] = _put(turned[1][keep], case["groups"], TYPES[case["dtype"]])
    v[page, place] = _put(s["v"].double()[keep], case["groups"], TYPES[case["dtype"]])
    return {"q": turned[0], "k": k.reshape(-1, *k.shape[2:]), "v": v.reshape(-1, *v.shape[2:])}


def _exact_read(s):
    P = s["case"]["page"]
    page, place = s["slots"] // P, s["slots"] % P
    return {"k": _held_of(s["k_cache"][page, place], s["k_scales"][page, place]),
            "v": _held_of(s["v_cache"][page, place], s["v_scales"][page, place])}


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
            k, v = (_held_of(s[c + "_cache"][pages, :, h], s[c + "_scales"][pages, :, h]).reshape(-1, D)[cut] for c in "kv")
            score = (k @ s["q"][b, heads].double().T) * s["scale"]                       # [keys, group]
            lse[b, heads] = torch.logsumexp(score, dim=0)
            out[b, heads] = torch.softmax(score, dim=0).T @ v
    return (out, lse) if case["lse"] else out


def exact(case, seed):
    return {"append": _exact_append, "read": _exact_read, "attention": _exact_attention}[case["op"]](prepare(case, seed))
