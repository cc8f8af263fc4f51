"""Plain forms in 64 bits of the operators around the projections, one loop per request, head or token, and the bounds within
which a kernel that computes in FP32 and rounds once has to agree."""
import torch

# largest relative error of one rounding: 11 and 8 significant bits
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38}     # half the spacing of the smallest values
E32 = 2.0 ** -24


def within(got, want, bound, what=""):
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} against {tuple(want.shape)}"
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"{what}: off by {float((got - want).abs().max()):.3g}, {float(over.max()):.3g} over the bound"


def page_step(cached, fresh, table, free, available, P, T):
    """(step as lists, table) with Python's whole numbers."""
    table = [list(r) for r in table]
    W = len(table[0]) if table else 0
    n = min(max(available, 0), len(free))
    lengths, starts, slots, positions, requests = [], [0], [], [], []
    pages = 0
    for b, (c, f) in enumerate(zip(cached, fresh)):
        c, f = max(c, 0), max(f, 0)
        have, want = min(-(-c // P), W), min(-(-(c + f) // P), W)
        new = {}
        for col in range(have, want):
            new[col] = free[n - 1 - pages] if pages < n else -1
            table[b][col] = max(new[col], -1)
            pages += 1
        for pos in range(c, min(c + f, c + T - len(slots))):        # (what has a place)
            col = pos // P
            page = -1 if col >= W else new.get(col, table[b][col] if col < have else -1)
            slots.append(page * P + pos % P if page >= 0 else -1)
            positions.append(min(pos, 2 ** 31 - 1))
            requests.append(b)
        lengths.append(min(c + f, 2 ** 31 - 1))
        starts.append(starts[-1] + f)
    counts = [starts[-1], pages, max(n - pages, 0)]
    pad = max(0, T - len(slots))
    return lengths, starts, slots + [-1] * pad, positions + [-1] * pad, requests + [-1] * pad, counts, table


def rotate(x, positions, table, sections, interleaved):
    """x [T, H, D] in 64 bits turned, and the bound of an FP32 rotation (three roundings of products no larger than |a| + |b|)."""
    x = x.double().clone()
    bound = torch.zeros_like(x)
    half = table.shape[1] // 2
    i = 0
    for axis, n in enumerate(sections):
        for _ in range(n):
            p = positions[axis].long()
            inside = (p >= 0) & (p < table.shape[0])
            row = table[p.clamp(0, max(0, table.shape[0] - 1))] if table.shape[0] else torch.zeros(len(p), 2 * half, device=x.device)
            c = torch.where(inside, row[:, i].double(), 1.0).unsqueeze(1)
            s = torch.where(inside, row[:, half + i].double(), 0.0).unsqueeze(1)
            ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
            a, b = x[:, :, ia].clone(), x[:, :, ib].clone()
            x[:, :, ia], x[:, :, ib] = a * c - b * s, b * c + a * s
            bound[:, :, ia] = bound[:, :, ib] = 3 * E32 * (a.abs() + b.abs())
            i += 1
    return x, bound


def attention(q, k_cache, v_cache, table, lengths, scale, window=0, rows=None):
    """(out, lse, bound of out before its rounding, bound of lse).  A score that sums D products in FP32 is off by at most
    (D + 8) 2^-24 scale sum |q k|; with the exponential and the two-part probabilities a weight is off by that and 2^-14."""
    B, H, D = q.shape
    P, heads = k_cache.shape[1], k_cache.shape[2]
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
        for h in range(H):
            g = h // (H // heads)
            k, v = k_cache[pages, keys % P, g].double(), v_cache[pages, keys % P, g].double()
            s = (k @ q[b, h].double()) * scale
            off = float((k.abs() @ q[b, h].double().abs()).max()) * abs(scale) * (D + 8) * E32 + 2.0 ** -14
            p = torch.softmax(s, 0)
            out[b, h], lse[b, h] = p @ v, torch.logsumexp(s, 0)
            bound[b, h] = 2 * off * (p @ v.abs()) + len(keys) * E32 * (p @ v.abs())
            lse_bound[b, h] = off + (len(keys) + 8) * E32 + 4 * E32 * lse[b, h].abs()
    return out, lse, bound, lse_bound


def low_rank(x, y, down, up, ids, scales=None, ranks=None):
    """(out, bound before its rounding): both sums in FP32, the inner one in steps of 16 products, its result in two 16-bit parts."""
    out, bound = y.double().clone(), torch.zeros_like(y, dtype=torch.float64)
    K = x.shape[1]
    for t, e in enumerate(ids.tolist()):
        if not 0 <= e < down.shape[0]:
            continue
        r = down.shape[1] if ranks is None else min(-(-max(int(ranks[e]), 0) // 8) * 8, down.shape[1])
        s = 1.0 if scales is None else float(scales[e])
        a, b = down[e, :r].double(), up[e, :, :r].double() * s
        v = a @ x[t].double()
        out[t] += b @ v
        each = (K / 16 + 32) * E32 * (a.abs() @ x[t].double().abs()) + 2.0 ** -15 * v.abs().max() if r else v
        bound[t] = b.abs() @ each + 40 * E32 * (b.abs() @ v.abs() + y[t].double().abs())
    return out, bound


def rounded(want, bound, dtype):
    """The bound of a result that is rounded to `dtype` once."""
    return bound + U[dtype] * (want.abs() + bound) + TINY[dtype]
