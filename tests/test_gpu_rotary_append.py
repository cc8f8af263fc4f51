"""Rotary positions and the write into the paged cache against 64 bits."""
import pytest
import torch

import plain_ops
from libortho_b200 import _C_ops, rotary_table

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def make(T, Hq, Hkv, D, pages, P, dtype, seed=0, layout="phd", fused=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)          # noqa: E731
    if fused:
        qkv = r(T, (Hq + 2 * Hkv) * D).view(T, Hq + 2 * Hkv, D)
        q, k, v = qkv.split((Hq, Hkv, Hkv), dim=1)
    else:
        q, k, v = r(T, Hq, D), r(T, Hkv, D), r(T, Hkv, D)
    if layout == "phd":
        caches = [r(pages, P, Hkv, D) for _ in range(2)]
    elif layout == "hpd":                                                    # a page's tokens of one head together
        caches = [r(pages, Hkv, P, D).transpose(1, 2) for _ in range(2)]
    else:                                                                    # keys and values of a page together
        both = r(pages, 2, P, Hkv, D)
        caches = [both[:, 0], both[:, 1]]
    slots = torch.randperm(pages * P, generator=g, device=DEV)[:T]
    return q, k, v, caches, slots


def check(q, k, v, caches, slots, positions, table, sections=None, interleaved=False, out=None):
    P, pages, dtype = caches[0].shape[1], caches[0].shape[0], k.dtype
    pos = positions.view(1, -1) if positions is not None and positions.dim() == 1 else positions
    want, bounds = [], []
    for x in (q, k):
        if x is None or table is None:
            w, b = (None, None) if x is None else (x.double(), torch.zeros_like(x, dtype=torch.float64))
        else:
            w, b = plain_ops.rotate(x, pos, table, sections or [table.shape[1] // 2], interleaved)
            turned = torch.zeros_like(b)
            turned[..., :table.shape[1]] = 1
            b = torch.where(turned > 0, plain_ops.rounded(w, b, dtype), 0)
        want.append(w)
        bounds.append(b)
    expect = [c.double().clone() for c in caches]
    limit = torch.zeros_like(expect[0])
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * P:
            expect[0][s // P, s % P], expect[1][s // P, s % P] = want[1][t], v[t].double()
            limit[s // P, s % P] = bounds[1][t]
    got = _C_ops.rotary_append(q, k, v, *caches, slots, positions, table, sections=sections, interleaved=interleaved, out=out)
    if q is None:
        assert got is None
    else:
        assert got.shape == q.shape and got.dtype == dtype
        plain_ops.within(got, want[0], bounds[0], "q")
    plain_ops.within(caches[0], expect[0], limit, "k_cache")
    assert torch.equal(caches[1].double(), expect[1])
    return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,Hq,Hkv,D,R,P,layout", [
    (1, 8, 2, 128, 128, 16, "phd"), (5, 4, 4, 64, 64, 1, "hpd"), (33, 5, 1, 80, 40, 24, "both"), (64, 64, 8, 128, 64, 16, "hpd"),
    (700, 3, 3, 96, 96, 5, "phd"), (9, 7, 1, 72, 24, 16, "phd"), (6, 2, 2, 20, 12, 3, "phd"), (7, 2, 1, 7, 6, 2, "hpd"),
    (3, 1, 1, 768, 768, 4, "phd"), (3, 2, 1, 602, 602, 4, "phd"), (2, 300, 2, 16, 2, 4, "phd")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_shapes(T, Hq, Hkv, D, R, P, layout, dtype, interleaved):
    q, k, v, caches, slots = make(T, Hq, Hkv, D, T // P + 3, P, dtype, seed=T, layout=layout)
    table = rotary_table(500, R, device=DEV)
    positions = torch.randint(0, 500, (T,), dtype=torch.int32, device=DEV)
    check(q, k, v, caches, slots, positions, table, interleaved=interleaved)


@pytest.mark.parametrize("sections", [(16, 24, 24), (22, 21, 21), (64, 0, 0), (0, 1, 63), (10, 20, 30, 4), (31, 33)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(sections, interleaved):
    T = 50
    q, k, v, caches, slots = make(T, 6, 2, 128, 9, 8, BF16)
    positions = torch.randint(0, 300, (len(sections), T + 3), dtype=torch.int32, device=DEV)[:, 1:T + 1]
    check(q, k, v, caches, slots, positions, rotary_table(300, 128, device=DEV), sections=list(sections), interleaved=interleaved)


def test_slots_and_positions_out_of_range():
    T = 40
    q, k, v, caches, slots = make(T, 4, 2, 64, 6, 8, F16)
    slots[::3] = -1
    slots[1::6] = 48 + torch.arange(len(slots[1::6]), device=DEV)
    slots[4] = 2 ** 40
    positions = torch.arange(T, dtype=torch.int32, device=DEV) * 5 - 20           # below zero, and behind 100
    check(q, k, v, caches, slots, positions, rotary_table(100, 64, device=DEV))


def test_in_place_unaligned_and_single_parts():
    q, k, v, caches, slots = make(12, 4, 2, 64, 4, 8, F16)
    table, positions = rotary_table(64, 64, device=DEV), torch.arange(12, dtype=torch.int32, device=DEV)
    want = _C_ops.rotary_append(q, k, v, *(c.clone() for c in caches), slots, positions, table)
    mine = q.clone()
    assert _C_ops.rotary_append(mine, k, v, *caches, slots, positions, table, out=mine) is mine and torch.equal(mine, want)
    # one value off every 16-byte boundary, rows of an odd length
    wide = torch.zeros(12, 4, 67, dtype=F16, device=DEV)
    odd = wide[:, :, 1:65]
    odd.copy_(q)
    assert torch.equal(_C_ops.rotary_append(odd, k, v, *caches, slots, positions, table), want)
    out = torch.zeros_like(wide)[:, :, 3:67]
    assert torch.equal(_C_ops.rotary_append(odd, k, v, *caches, slots, positions, table, out=out), want)
    # keys and values alone, with and without positions; nothing at all
    check(None, k, v, caches, slots, positions, table)
    check(None, k, v, caches, slots, None, None)
    check(q[:0], k[:0], v[:0], caches, slots[:0], positions[:0], table)
    # NaN payloads and infinities of values pass as they are
    v = torch.full_like(v, float("nan"))
    v[0] = float("inf")
    _C_ops.rotary_append(None, k, v, *caches, slots, positions, table)
    rows = caches[1].reshape(-1, 2, 64)[slots]
    assert torch.equal(rows.view(torch.int16), v.contiguous().view(torch.int16))


def test_a_cache_beyond_32_bits():
    """The last page of a cache of more than 2^31 elements; attention reads it back."""
    pages = 2 ** 31 // (64 * 2 * 128) + 2
    k_cache, v_cache = (torch.empty(pages, 64, 2, 128, dtype=F16, device=DEV) for _ in range(2))
    q, k, v, _, _ = make(70, 4, 2, 128, 1, 64, F16)
    slots = torch.arange(70, device=DEV) + (pages - 2) * 64
    positions = torch.arange(70, dtype=torch.int32, device=DEV)
    table = rotary_table(70, 128, device=DEV)
    qr = _C_ops.rotary_append(q, k, v, k_cache, v_cache, slots, positions, table)
    assert torch.equal(v_cache.view(-1, 2, 128)[slots], v)
    small = [torch.zeros(2, 64, 2, 128, dtype=F16, device=DEV) for _ in range(2)]
    _C_ops.rotary_append(q, k, v, *small, slots - (pages - 2) * 64, positions, table)
    assert torch.equal(k_cache[pages - 2:].reshape(-1, 2, 128)[:70], small[0].view(-1, 2, 128)[:70])
    tables = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device=DEV)
    n = torch.tensor([70], dtype=torch.int32, device=DEV)
    far = _C_ops.paged_attention(qr[-1:], k_cache, v_cache, tables, n)
    near = _C_ops.paged_attention(qr[-1:], *small, tables - (pages - 2), n)
    assert torch.equal(far, near)


def test_streams_and_capture():
    q, k, v, caches, slots = make(20, 4, 2, 128, 4, 8, BF16)
    table, positions = rotary_table(64, 128, device=DEV), torch.arange(20, dtype=torch.int32, device=DEV)
    want = [_C_ops.rotary_append(q, k, v, *caches, slots, positions, table), *[c.clone() for c in caches]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        caches[0].zero_()
        got = _C_ops.rotary_append(q, k, v, *caches, slots, positions, table)
    side.synchronize()
    rows = lambda c: c.reshape(-1, 2, 128)[slots]                             # noqa: E731
    assert torch.equal(got, want[0]) and torch.equal(rows(caches[0]), rows(want[1]))
    graph, x = torch.cuda.CUDAGraph(), q.clone()
    with torch.cuda.graph(graph):
        got = _C_ops.rotary_append(x, k, v, *caches, slots, positions, table)
    x.copy_(q.flip(0))
    graph.replay()
    assert torch.equal(got, _C_ops.rotary_append(q.flip(0), k, v, *caches, slots, positions, table))


def test_refusals():
    q, k, v, (kc, vc), slots = make(6, 4, 2, 64, 3, 8, F16)
    table, pos = rotary_table(64, 64, device=DEV), torch.arange(6, dtype=torch.int32, device=DEV)
    base = dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, slots=slots, positions=pos, table=table)
    _C_ops.rotary_append(**base)

    def refused(error, match, **change):
        with pytest.raises(error, match=match):
            _C_ops.rotary_append(**{**base, **change})
    refused(RuntimeError, "CPU", k=k.cpu())
    refused(TypeError, "k must be", k=k.float())
    refused(TypeError, "q must be", q=q.to(BF16))
    refused(TypeError, "slots", slots=slots.int())
    refused(TypeError, "k_cache", k_cache=kc.to(BF16))
    refused(ValueError, "q must be", q=q[:5])
    refused(ValueError, "same heads", v=v[:, :1])
    refused(ValueError, "alike", v_cache=vc[:2])
    refused(ValueError, "heads and head_dim", k_cache=kc[..., :32], v_cache=vc[..., :32])
    refused(ValueError, "contiguous", k_cache=torch.zeros(3, 8, 64, 2, dtype=F16, device=DEV).transpose(2, 3))
    refused(ValueError, "go together", table=None)
    refused(ValueError, "nothing to do", positions=None, table=None)
    refused(ValueError, "axes", positions=torch.zeros(5, 6, dtype=torch.int32, device=DEV))
    refused(ValueError, "sections", positions=pos.repeat(2, 1))
    refused(ValueError, "sections", positions=pos.repeat(2, 1), sections=[16, 15])
    refused(ValueError, "section", positions=pos.repeat(2, 1), sections=[33, -1])
    refused(ValueError, "sections", positions=pos.repeat(2, 1), sections=[32])
    refused(ValueError, "table", table=rotary_table(64, 128, device=DEV))
    refused(TypeError, "table", table=table.half())
    refused(ValueError, "out", out=q[:3])
    refused(ValueError, "out is for q", q=None, out=q)
    refused(TypeError, "v must be a tensor", v=None)


@pytest.mark.parametrize("interleaved", [False, True])
def test_a_cache_without_pages_keeps_nothing_and_queries_are_turned(interleaved):
    for T, D in ((1, 64), (12, 64), (5, 20)):
        q, k, v, caches, slots = make(T, 4, 2, D, 4, 8, F16)
        table, positions = rotary_table(64, D, device=DEV), torch.arange(T, dtype=torch.int32, device=DEV) * 3
        want = _C_ops.rotary_append(q, k, v, *(c.clone() for c in caches), slots, positions, table, interleaved=interleaved)
        got = _C_ops.rotary_append(q, k, v, caches[0][:0], caches[1][:0], slots, positions, table, interleaved=interleaved)
        assert torch.equal(got, want)
        assert _C_ops.rotary_append(None, k, v, caches[0][:0], caches[1][:0], slots, positions, table) is None
