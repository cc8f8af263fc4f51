"""Plain forms in 64 bits of a paged cache held in 4 bits, and the bounds within which the kernels have to agree."""
import torch

from plain_ops import E32

DIGITS = {torch.float16: (11, -13), torch.bfloat16: (8, -125)}      # significant bits, exponent of the smallest normal number (frexp's)


def nearest(x, dtype):
    """x in 64 bits rounded to the type once, ties to even, in 64 bits; infinity where it leaves the type."""
    digits, least = DIGITS[dtype]
    e = torch.frexp(x)[1].clamp(min=least) - digits
    y = torch.ldexp(torch.round(torch.ldexp(x, -e)), e)
    return torch.where(y.abs() > torch.finfo(dtype).max, torch.copysign(torch.full_like(y, torch.inf), y), y)


def quantise(x, groups, dtype):
    """x [..., D] in 64 bits -> codes 0 .. 15 [..., D] int64, scales and zeros [..., groups] in 64 bits (scale NaN: no number)."""
    g = x.reshape(*x.shape[:-1], groups, x.shape[-1] // groups)
    sound = torch.isfinite(nearest(torch.nan_to_num(g, nan=torch.inf, posinf=torch.inf, neginf=-torch.inf), dtype)).all(-1)
    lo, hi = torch.nan_to_num(g).amin(-1), torch.nan_to_num(g).amax(-1)
    zero, scale = nearest(lo, dtype), nearest((hi - lo) / 15, dtype)
    # where zero + 15 scale would leave the type: the next smaller scale
    e = torch.frexp(scale)[1] - DIGITS[dtype][0]
    scale = torch.where(torch.isinf(nearest(zero + 15 * scale, dtype)), scale - torch.ldexp(torch.ones_like(scale), e), scale)
    z, s = zero.unsqueeze(-1), scale.unsqueeze(-1)
    code = torch.where(s > 0, torch.round((torch.nan_to_num(g) - z) / torch.where(s > 0, s, 1.0)).clamp(0, 15), 0.0)
    code = torch.where(sound.unsqueeze(-1), code, 0.0)
    return code.long().reshape(x.shape), torch.where(sound, scale, torch.nan), zero


def codes_of(cache):
    """Codes [..., D] of a cache's bytes [..., D / 2]."""
    return torch.stack((cache & 15, cache >> 4), -1).flatten(-2).long()


def held(cache, scales):
    """What codes and scales stand for, in 64 bits [..., D]."""
    c = codes_of(cache).double()
    c = c.view(*c.shape[:-1], scales.shape[-2], c.shape[-1] // scales.shape[-2])
    return (c * scales[..., :1].double() + scales[..., 1:].double()).flatten(-2)


def attention(q, k_cache, v_cache, k_scales, v_scales, table, lengths, scale, window=0, rows=None):
    """(out, lse, bound of out before its rounding, bound of lse).  A score is made of D products of a query and 64 + code <= 79, a scale, and a sum of queries times zero - 64 scales:
    D + 16 roundings of at most 2^-24 of these terms' sizes.  Weights are off by that, and by 2^-18 for the exponential, the two parts and the sums over keys of a warp; the outputs'
    products are of at most 8 scales, and of zero + 8 scales.  BF16 outputs are made of one part, FP16: a weight times a scale is off by half its last place more, 2^-12."""
    part = 2.0 ** -12 if q.dtype == torch.bfloat16 else 0.0
    B, H, D = q.shape
    P, heads, G = k_cache.shape[1], k_cache.shape[2], k_scales.shape[3]
    out = torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, H), -torch.inf, dtype=torch.float64, device=q.device)
    bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(B):
        row = b if rows is None else int(rows[b])
        n = min(max(int(lengths[b]), 0), table.shape[1] * P) if 0 <= row < table.shape[0] else 0
        keys = torch.arange(max(0, n - window) if window else 0, n, device=q.device)
        pages = table[row, keys // P].long() if n else keys
        ok = (pages >= 0) & (pages < k_cache.shape[0])
        keys, pages = keys[ok], pages[ok]
        if not len(keys):
            continue
        for g in range(heads):
            hs = slice(g * (H // heads), (g + 1) * (H // heads))
            at = (pages, keys % P, g)
            k, v = held(k_cache[at], k_scales[at]), held(v_cache[at], v_scales[at])
            ks, vs = k_scales[at].double(), v_scales[at].double()                        # [keys, G, 2]
            x = q[b, hs].double()
            s = (k @ x.T) * scale                                                        # [keys, heads]
            each = (143 * ks[..., 0] + ks[..., 1].abs()).repeat_interleave(D // G, -1)   # 79 and 64 scales, and the zero
            off = (each @ x.abs().T).amax(0) * abs(scale) * (D + 16) * E32 + 2.0 ** -18
            sizes = (8 * vs[..., 0] + (vs[..., 1] + 8 * vs[..., 0]).abs()).repeat_interleave(D // G, -1)
            p = torch.softmax(s, 0)
            out[b, hs], lse[b, hs] = p.T @ v, torch.logsumexp(s, 0)
            bound[b, hs] = (2 * off.unsqueeze(1) + len(keys) * E32 + part) * (p.T @ sizes)
            lse_bound[b, hs] = off + (len(keys) + 8) * E32 + 4 * E32 * lse[b, hs].abs()
    return out, lse, bound, lse_bound
