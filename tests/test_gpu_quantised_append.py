"""Keys and values quantised to 4 bits as they are written, and read back: codes and scales as in exact arithmetic."""
import math

import pytest
import torch

import plain_ops
import quantised_ops
from libortho_b200 import _C_ops, rotary_table

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16
NAN = float("nan")


def make(T, Hq, Hkv, D, pages, P, dtype, groups=1, seed=0, layout="hpd", std=1.0, shift=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    qkv = (torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=DEV) * std + shift).to(dtype)
    q, k, v = qkv.split((Hq, Hkv, Hkv), dim=1)
    bytes_ = lambda *s: torch.randint(0, 256, s, generator=g, device=DEV, dtype=torch.uint8)        # noqa: E731
    held = lambda *s: torch.rand(*s, generator=g, device=DEV).to(dtype)                             # noqa: E731
    if layout == "hpd":                                                      # a page's tokens of one head together
        cache = [bytes_(pages, Hkv, P, D // 2).transpose(1, 2) for _ in range(2)] + [held(pages, Hkv, P, groups, 2).transpose(1, 2) for _ in range(2)]
    elif layout == "phd":
        cache = [bytes_(pages, P, Hkv, D // 2) for _ in range(2)] + [held(pages, P, Hkv, groups, 2) for _ in range(2)]
    else:                                                                    # keys and values of a page together, rows of an odd number of words
        both, rest = bytes_(pages, 2, P, Hkv, D // 2 + 4), held(pages, 2, P, Hkv, groups, 2)
        cache = [both[:, 0, ..., :D // 2], both[:, 1, ..., :D // 2], rest[:, 0], rest[:, 1]]
    slots = torch.randperm(pages * P, generator=g, device=DEV)[:T]
    return q, k, v, cache, slots


def check(q, k, v, cache, slots, positions=None, table=None, sections=None, interleaved=False, out=None):
    pages, P, Hkv, D = cache[0].shape[0], cache[0].shape[1], k.shape[1], k.shape[2]
    dtype, groups = k.dtype, cache[2].shape[3]
    keys = k.double()
    if table is not None:
        pos = positions.view(1, -1) if positions.dim() == 1 else positions
        keys = plain_ops.rotate(k, pos, table, sections or [table.shape[1] // 2], interleaved)[0]
    kept = (slots >= 0) & (slots < pages * P)
    at = slots[kept] // P, slots[kept] % P
    want = []
    for i, x in enumerate((keys, v.double())):
        codes, held = quantised_ops.codes_of(cache[i]), cache[2 + i].double().clone()
        c, s, z = quantised_ops.quantise(x[kept], groups, dtype)
        codes[at], held[at] = c, torch.stack((s, torch.where(torch.isnan(s), 0.0, z)), -1)
        want.append((codes, held))
    got = _C_ops.rotary_append_quantised(q, k, v, *cache, slots, positions, table, sections=sections, interleaved=interleaved, out=out)
    for i, name in enumerate(("keys", "values")):
        codes, held = want[i]
        assert torch.equal(torch.nan_to_num(cache[2 + i].double(), nan=-1.0), torch.nan_to_num(held, nan=-1.0)), name + ": scales"
        assert torch.equal(quantised_ops.codes_of(cache[i]), codes), name + ": codes"
    if q is None:
        assert got is None
    else:                                        # queries: what the operator without codes gives, bit for bit
        none = [torch.zeros(1, 1, Hkv, D, dtype=dtype, device=DEV) for _ in range(2)]
        assert torch.equal(got, _C_ops.rotary_append(q, k, v, *none, torch.full_like(slots, -1), positions, table, sections=sections, interleaved=interleaved))
    return got


def check_read(cache, slots, out=None):
    pages, P = cache[0].shape[:2]
    dtype = cache[2].dtype
    inside = (slots >= 0) & (slots < pages * P)
    page, place = torch.where(inside, slots // P, 0), torch.where(inside, slots % P, 0)
    got = _C_ops.read_quantised(*cache, slots, out=out)
    for i in range(2):
        want = quantised_ops.nearest(quantised_ops.held(cache[i][page, place], cache[2 + i][page, place]), dtype)
        want = torch.where(inside.view(-1, 1, 1), want, 0.0)
        assert got[i].dtype == dtype and torch.equal(torch.nan_to_num(got[i].double(), nan=7e9), torch.nan_to_num(want, nan=7e9)), "kv"[i]
    return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,Hq,Hkv,D,R,P,groups,layout", [
    (1, 8, 2, 128, 128, 16, 1, "hpd"), (1, 1, 1, 8, 8, 1, 1, "phd"), (5, 4, 4, 64, 64, 1, 1, "phd"), (33, 5, 1, 80, 40, 24, 1, "both"), (64, 64, 8, 128, 64, 16, 2, "hpd"),
    (1300, 3, 3, 96, 96, 5, 1, "phd"), (9, 7, 1, 72, 24, 16, 1, "both"), (40, 2, 2, 256, 256, 8, 4, "hpd"), (41, 2, 2, 256, 200, 8, 1, "both"),
    (39, 2, 1, 192, 192, 7, 3, "phd"), (7, 3, 2, 112, 56, 16, 1, "hpd"), (6, 2, 2, 24, 16, 3, 1, "phd"), (700, 1, 5, 128, 32, 64, 2, "both")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_shapes(T, Hq, Hkv, D, R, P, groups, layout, dtype, interleaved):
    q, k, v, cache, slots = make(T, Hq, Hkv, D, T // P + 3, P, dtype, groups, seed=T, layout=layout)
    positions = torch.randint(0, 500, (T,), dtype=torch.int32, device=DEV)
    check(q, k, v, cache, slots, positions, rotary_table(500, R, device=DEV), interleaved=interleaved)
    check_read(cache, torch.randperm(cache[0].shape[0] * P, device=DEV))


@pytest.mark.parametrize("D", [8, 16, 32, 40, 48, 56, 88, 104, 120, 136, 160, 200, 248])
def test_head_dims(D):
    for dtype in (F16, BF16):
        q, k, v, cache, slots = make(21, 3, 2, D, 6, 5, dtype, seed=D)
        check(q, k, v, cache, slots, torch.arange(21, dtype=torch.int32, device=DEV), rotary_table(30, D // 8 * 8, device=DEV))
        check(None, k, v, cache, slots)
        check_read(cache, slots)


@pytest.mark.parametrize("sections", [(16, 24, 24), (22, 21, 21), (64, 0, 0), (10, 20, 30, 4)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(sections, interleaved):
    T = 50
    q, k, v, cache, slots = make(T, 6, 2, 128, 9, 8, BF16, 2)
    positions = torch.randint(0, 300, (len(sections), T + 3), dtype=torch.int32, device=DEV)[:, 1:T + 1]
    check(q, k, v, cache, slots, positions, rotary_table(300, 128, device=DEV), sections=list(sections), interleaved=interleaved)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("groups", [1, 2])
def test_many_values_next_to_borders(dtype, groups):
    """Two million keys: some thousand lie within FP32's error of the border between two codes, some groups' scales or zeros between two numbers.  Values on a coarse grid meet ties."""
    for seed, std, shift in ((1, 1.0, 0.0), (2, 0.01, 5.0), (3, 100.0, -30.0)):
        q, k, v, cache, slots = make(1000, 1, 16, 128, 70, 16, dtype, groups, seed=seed, std=std, shift=shift)
        v.copy_((v.float() / std * 16).round() * std / 16)
        k[::2] = (k[::2].float() / std * 4).round() * std / 4
        check(q, k, v, cache, slots, torch.randint(0, 5000, (1000,), dtype=torch.int32, device=DEV), rotary_table(5000, 128, device=DEV))
        check(None, k, v, cache, slots)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_ranges(dtype):
    """Groups of one value, of zeros, of almost one value, at the ends of the type, and without a number."""
    T, top = 16, torch.finfo(dtype).max
    q, k, v, cache, slots = make(T, 1, 2, 128, 3, 8, dtype, 2)
    for x in (k, v):
        x[0] = 0
        x[1] = 3.25
        x[2] = -7.0
        x[2, :, 5] = -6.99609375 if dtype == F16 else -6.96875               # the next number
        x[3, 0, :64], x[3, 0, 0] = top, -top
        x[4, 0, 3], x[4, 1, 70] = math.inf, -math.inf
        x[5, 0, 9] = NAN
        x[6] = top
        x[7], x[7, :, 1] = -top, top
        x[8] = x[8] * 1e-6
        x[9, 0, 64:] = 0
        x[10, :, ::2], x[10, :, 1::2] = 15.0, 0.0                            # every code at an end
        x[11] = (torch.arange(128, device=DEV) % 31 * 0.5).to(dtype)         # scale 1, every other value a tie
        x[12] = -0.0
    check(None, k, v, cache, slots)
    got = check_read(cache, slots)
    assert torch.isnan(got[0][4, 0, :64]).all() and torch.isfinite(got[0][4, 0, 64:]).all() and torch.isfinite(got[0][4, 1, :64]).all()
    assert torch.isnan(got[1][5, 0, :64]).all() and torch.isfinite(got[1][5, 1]).all()
    assert torch.isfinite(torch.cat((got[0][:4], got[0][6:]))).all() and (got[0][1] == 3.25).all() and (got[1][0] == 0).all()
    # turned: two groups of a head meet in each pair; nothing that overflows on the way is taken for a number
    k[3], k[6], k[7] = 1.0, 2.0, 3.0
    k[13, 1, 0], k[13, 1, 64] = top, top
    k[14] = 0
    positions = torch.arange(T, dtype=torch.int32, device=DEV) + 1
    check(q, k, v, cache, slots, positions, rotary_table(100, 128, device=DEV))


def test_slots_and_positions_out_of_range():
    T = 40
    q, k, v, cache, slots = make(T, 4, 2, 64, 6, 8, F16)
    slots[::3] = -1
    slots[1::6] = 48 + torch.arange(len(slots[1::6]), device=DEV)
    slots[4] = 2 ** 40
    positions = torch.arange(T, dtype=torch.int32, device=DEV) * 5 - 20           # below zero, and behind 100
    check(q, k, v, cache, slots, positions, rotary_table(100, 64, device=DEV))
    got = check_read(cache, slots)
    assert (got[0][::3] == 0).all() and (got[1][4] == 0).all()
    none = [c[:0] for c in cache]
    assert (check(q, k, v, none, slots, positions, rotary_table(100, 64, device=DEV)) != 0).any()
    assert all((x == 0).all() for x in _C_ops.read_quantised(*none, slots))
    assert check(q, k, v, cache, slots, positions, rotary_table(100, 64, device=DEV)[:0]).equal(q)     # an empty table turns nothing


def test_in_place_unaligned_and_single_parts():
    q, k, v, cache, slots = make(12, 4, 2, 64, 4, 8, F16)
    table, positions = rotary_table(64, 64, device=DEV), torch.arange(12, dtype=torch.int32, device=DEV)
    first = [c.clone() for c in cache]
    want = _C_ops.rotary_append_quantised(q, k, v, *first, slots, positions, table)
    mine = q.clone()
    assert _C_ops.rotary_append_quantised(mine, k, v, *cache, slots, positions, table, out=mine) is mine and torch.equal(mine, want)
    # one value off every 16-byte boundary, rows of an odd length; four values off
    for off in (1, 4):
        wide = [torch.zeros(12, x.shape[1], 69, dtype=F16, device=DEV)[:, :, off:off + 64] for x in (q, k, v)]
        again = [c.clone() for c in cache]
        for w, x in zip(wide, (q, k, v)):
            w.copy_(x)
        assert torch.equal(_C_ops.rotary_append_quantised(*wide, *again, slots, positions, table), want)
        assert all(torch.equal(a, b) for a, b in zip(again, first))
    four = torch.zeros(12, 4, 72, dtype=F16, device=DEV)[:, :, 4:68]
    assert torch.equal(_C_ops.rotary_append_quantised(q, k, v, *cache, slots, positions, table, out=four), want)
    check(None, k, v, cache, slots, positions, table)
    check(None, k, v, cache, slots, None, None)
    for x in (_C_ops.rotary_append_quantised(q[:0], k[:0], v[:0], *cache, slots[:0], positions[:0], table), *_C_ops.read_quantised(*cache, slots[:0])):
        assert x.shape[0] == 0


def test_read_into_views_and_large_counts():
    _, k, v, cache, slots = make(9, 1, 2, 64, 50, 8, BF16)
    wide = torch.full((400, 5, 72), 5.0, dtype=BF16, device=DEV)
    all_slots = torch.arange(400, device=DEV)
    out = wide[:, :2, :64], wide[:, 2:4, :64]
    got = check_read(cache, all_slots, out=out)
    assert got is out and (wide[:, 4] == 5).all() and (wide[:, :, 64:] == 5).all()
    check_read(cache, all_slots.repeat(30)[3:])                              # the same slots several times
    check_read(cache, torch.randint(-5, 410, (5000,), device=DEV)[::2])


def test_streams_and_capture():
    q, k, v, cache, slots = make(30, 4, 2, 128, 6, 8, F16, 2)
    table, positions = rotary_table(64, 128, device=DEV), torch.arange(30, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine = [c.clone() for c in cache]
        got = _C_ops.rotary_append_quantised(q, k, v, *mine, slots, positions, table)
        back = _C_ops.read_quantised(*mine, slots)
    torch.cuda.synchronize()
    want = check(q, k, v, cache, slots, positions, table)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(mine, cache))
    assert all(torch.equal(a, b) for a, b in zip(back, _C_ops.read_quantised(*cache, slots)))
    graph, x, at = torch.cuda.CUDAGraph(), [t.clone() for t in (q, k, v)], slots.clone()
    with torch.cuda.graph(graph):
        got = _C_ops.rotary_append_quantised(*x, *mine, at, positions, table)
        back = _C_ops.read_quantised(*mine, at)
    for t, y in zip(x, (q, k, v)):
        t.copy_(y * 2)
    at.copy_(slots.flip(0))
    graph.replay()
    want = check(q * 2, k * 2, v * 2, cache, slots.flip(0), positions, table)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(mine, cache))
    assert all(torch.equal(a, b) for a, b in zip(back, _C_ops.read_quantised(*cache, slots.flip(0))))


def test_refusals():
    q, k, v, cache, slots = make(12, 4, 2, 64, 4, 8, F16)
    names = ("k_cache", "v_cache", "k_scales", "v_scales")
    base = dict(q=q, k=k, v=v, **dict(zip(names, cache)), slots=slots, positions=torch.arange(12, dtype=torch.int32, device=DEV), table=rotary_table(64, 64, device=DEV))

    def refused(error, match, call=_C_ops.rotary_append_quantised, **change):
        args = {**base, **change}
        if call is _C_ops.read_quantised:
            args = {n: args[n] for n in (*names, "slots", "out") if n in args}
        with pytest.raises(error, match=match):
            call(**args)
    for call in (_C_ops.rotary_append_quantised, _C_ops.read_quantised):
        refused(RuntimeError, "CPU", call, k_cache=cache[0].cpu())
        refused(TypeError, "k_cache", call, k_cache=cache[0].to(torch.int8))
        refused(TypeError, "v_scales", call, v_scales=cache[3].float())
        refused(TypeError, "slots", call, slots=slots.int())
        refused(ValueError, "alike", call, v_cache=cache[1][:1])
        refused(ValueError, "alike", call, v_scales=cache[3][..., :1])
        refused(ValueError, "alike", call, k_scales=cache[2][:, :1], v_scales=cache[3][:, :1])
        refused(ValueError, "contiguous", call, k_cache=cache[0].transpose(2, 3).contiguous().transpose(2, 3))
        refused(ValueError, "contiguous", call, k_scales=cache[2].transpose(1, 4).contiguous().transpose(1, 4))
        refused(ValueError, "64 elements", call, k_scales=cache[2].repeat(1, 1, 1, 2, 1), v_scales=cache[3].repeat(1, 1, 1, 2, 1))
        refused(ValueError, "aligned", call, k_cache=torch.zeros(cache[0].numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(4, 8, 2, 32))
        refused(ValueError, "multiples of 4", call, k_cache=torch.zeros(4, 8, 2, 34, dtype=torch.uint8, device=DEV)[..., :32])
    small = [torch.zeros(4, 8, 2, 6, dtype=torch.uint8, device=DEV)] * 2 + list(cache[2:])
    refused(ValueError, "multiple of 8", _C_ops.read_quantised, **dict(zip(names, small)))
    refused(TypeError, "k must be", k=k.float())
    refused(TypeError, "v must be", v=v.to(BF16))
    refused(ValueError, "head_dim", k=k[..., :32], v=v[..., :32])
    refused(ValueError, "heads", v=v[:, :1])
    refused(ValueError, "multiple of 8", table=rotary_table(64, 12, device=DEV))
    refused(ValueError, "go together", table=None)
    refused(ValueError, "nothing to do", positions=None, table=None)
    refused(ValueError, "sections", sections=[3, 3])
    refused(ValueError, "out", out=q[:1])
    refused(ValueError, "aligned", out=torch.zeros(12, 4, 66, dtype=F16, device=DEV)[:, :, 1:65])
    refused(ValueError, "slots", slots=slots[:3])
    refused(ValueError, "expanded", v_scales=cache[3][:1].expand(4, -1, -1, -1, -1))
    refused(TypeError, "pair", _C_ops.read_quantised, out=q)
    one = torch.zeros(12, 2, 64, dtype=F16, device=DEV)
    refused(ValueError, "two tensors", _C_ops.read_quantised, out=(one, one))
    refused(ValueError, r"out\[1\]", _C_ops.read_quantised, out=(torch.zeros(12, 2, 64, dtype=F16, device=DEV), torch.zeros(12, 2, 65, dtype=F16, device=DEV)))
