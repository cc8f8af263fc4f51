"""Attention of one token over a paged cache held in 4 bits against 64 bits."""
import math

import pytest
import torch

import plain_ops
import quantised_ops
from libortho_b200 import _C_ops, _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16
NAN = float("nan")


def make(lengths, Hq, Hkv, D, P, dtype, groups=1, seed=0, layout="hpd", std=1.0, spare=2, size=1.0):
    """Inputs whose unused places -- behind a length, pages of nobody, table entries behind the last page -- have scales of NaN or are nonsense."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // P) for n in lengths]
    W, total = max(need + [1]) + 1, sum(need) + spare
    perm = torch.randperm(total, generator=g, device=DEV).tolist()
    table, at = torch.full((len(lengths), W), 2 ** 30, dtype=torch.int32), 0
    cache = []
    for i in range(4):
        shape = {"hpd": (total, Hkv, P), "phd": (total, P, Hkv), "odd": (total, P, Hkv)}[layout]
        c = torch.randint(0, 256, (*shape, D // 2 + (4 if layout == "odd" else 0)), generator=g, device=DEV, dtype=torch.uint8)[..., :D // 2] if i < 2 \
            else torch.full((*shape, groups, 2), NAN, dtype=dtype, device=DEV)
        cache.append(c.transpose(1, 2) if layout == "hpd" else c)
    for b, n in enumerate(lengths):
        for j in range(need[b]):
            table[b, j] = perm[at]
            m = min(P, n - j * P)
            for i in (2, 3):
                scale = torch.rand(m, Hkv, groups, generator=g, device=DEV) * 0.2 + 0.2
                zero = -7.5 * scale + torch.randn(m, Hkv, groups, generator=g, device=DEV) * 0.3
                cache[i][perm[at], :m] = (torch.stack((scale, zero), -1) * size).to(dtype)
            at += 1
    q = (torch.randn(len(lengths), Hq, D, generator=g, device=DEV) * std).to(dtype)
    return q, *cache, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)


def check(q, *rest, scale=None, **kw):
    """rest: the cache's four tensors, the table, the lengths."""
    out, lse, bound, lse_bound = quantised_ops.attention(q, *rest, q.shape[2] ** -0.5 if scale is None else scale, **kw)
    got_lse = torch.full_like(lse, 7.0, dtype=torch.float32)
    got = _C_ops.paged_attention_quantised(q, *rest, scale=scale, lse=got_lse, **kw)
    assert got.shape == q.shape and got.dtype == q.dtype
    plain_ops.within(got, out, plain_ops.rounded(out, bound, q.dtype), "out")
    empty = torch.isinf(lse)
    assert torch.equal(torch.isinf(got_lse), empty) and (got_lse[empty] < 0).all() and (got[empty] == 0).all()
    plain_ops.within(got_lse[~empty], lse[~empty], lse_bound[~empty], "lse")
    assert torch.equal(got, _C_ops.paged_attention_quantised(q, *rest, scale=scale, **kw))              # the same bits again
    assert _lib.lib().ortho_b200_query_kernel_status() == 0
    return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 8), (8, 1), (10, 2), (18, 2), (24, 1), (33, 1), (32, 2), (71, 1)])
@pytest.mark.parametrize("D,groups", [(8, 1), (64, 1), (80, 1), (96, 1), (128, 1), (128, 2), (192, 1), (192, 3), (256, 1), (256, 4)])
def test_heads(Hq, Hkv, D, groups, dtype):
    check(*make([0, 1, 17, 300, 128], Hq, Hkv, D, 16, dtype, groups, seed=Hq + D))


@pytest.mark.parametrize("D", [16, 24, 32, 40, 48, 56, 72, 88, 104, 112, 120, 136, 160, 200, 224, 248])
def test_head_dims(D):
    check(*make([5, 130], 6, 2, D, 8, BF16, seed=D))
    check(*make([70], 17, 1, D, 8, F16, seed=D))


@pytest.mark.parametrize("P", [1, 2, 3, 5, 16, 24, 64, 100, 128, 4096])
@pytest.mark.parametrize("layout", ["hpd", "phd", "odd"])
def test_pages(P, layout):
    check(*make([0, 1, P, P + 1, max(1, P - 1), 2 * P, 333], 4, 2, 64, P, F16, seed=P, layout=layout))


@pytest.mark.parametrize("lengths", [[1], [15], [16], [17], [31], [32], [33], [127], [128], [129], [255], [256], [257], [1000], [5000], [0], [0, 0, 0], [0, 9, 0],
                                     list(range(40)), [4000, 1, 1, 1, 1, 1, 1], [3, 0, 2500, 0, 64, 128]])
def test_lengths(lengths):
    check(*make(lengths, 8, 2, 128, 16, BF16, 2, seed=sum(lengths)))
    check(*make(lengths, 4, 4, 64, 16, F16, seed=sum(lengths)))


@pytest.mark.parametrize("B,Hq,Hkv,L", [(300, 2, 1, 9), (64, 8, 8, 200), (1500, 1, 1, 3), (5000, 1, 1, 2)])
def test_many_requests(B, Hq, Hkv, L):
    lengths = [(i * 7919) % (L + 1) for i in range(B)]
    q, *rest, table, n = make(lengths, Hq, Hkv, 64, 8, F16, seed=B)
    got = _C_ops.paged_attention_quantised(q, *rest, table, n)
    pick = torch.arange(0, B, max(1, B // 60), device=DEV)
    out, lse, bound, _ = quantised_ops.attention(q[pick], *rest, table[pick], n[pick], 0.125)
    plain_ops.within(got[pick], out, plain_ops.rounded(out, bound, F16))
    assert (got[n == 0] == 0).all() and torch.isfinite(got).all()


def test_a_long_cache():
    """100,000 keys: outputs a hundredth of the values' size."""
    for Hq, Hkv, dtype, groups in ((8, 1, F16, 1), (3, 3, BF16, 2)):
        check(*make([100000, 33], Hq, Hkv, 128, 256, dtype, groups, std=0.1))


@pytest.mark.parametrize("window", [1, 2, 16, 127, 128, 129, 1000])
def test_windows(window):
    check(*make([0, 1, 50, 64, 101, 700], 6, 2, 64, 8, F16, seed=window), window=window)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 4.0])
def test_scales(scale):
    check(*make([1, 40, 333], 4, 2, 64, 16, F16), scale=scale)


def test_one_key_that_outweighs_the_rest_and_many_that_weigh_little():
    q, k, v, ks, vs, table, n = make([2000], 8, 1, 64, 16, F16)
    ks[table[0, 70], 3] *= 8
    check(q, k, v, ks, vs, table, n, scale=0.3)
    ks.mul_(0.01)
    check(q, k, v, ks, vs, table, n)


def test_scores_that_grow_and_fall():
    """The running maximum, and the largest scale of the values, change in every tile, or never after the first."""
    for order in (1, -1):
        for dtype in (F16, BF16):
            q, k, v, ks, vs, table, n = make([1500], 4, 1, 64, 16, dtype)
            ramp = torch.linspace(*(0, 6)[::order], 1500, device=DEV)
            for j in range(1500):
                at = table[0, j // 16], j % 16, 0
                ks[at] = (ks[at].float() * ramp[j]).to(dtype)
                vs[at] = (vs[at].float() * 2.0 ** ramp[j]).to(dtype)
            check(q, k, v, ks, vs, table, n)


def test_sizes():
    """Queries, keys and values far from one; values whose scale is zero."""
    for size in (2.0 ** -10, 2.0 ** 10):
        check(*make([300, 7], 4, 2, 64, 16, F16, size=size, std=1 / size, seed=5))
    for size in (2.0 ** -90, 2.0 ** 90):
        check(*make([300, 7], 4, 2, 64, 16, BF16, size=size, std=1 / size, seed=5))
    q, k, v, ks, vs, table, n = make([300, 7], 4, 2, 64, 16, BF16)
    vs[..., 0] = 0
    check(q, k, v, ks, vs, table, n)
    q[0] = 0
    q[1, 1, 1:] *= 2.0 ** -40
    check(q, k, v, ks, vs, table, n)


def test_rows_that_share_requests():
    """The tokens of two prompts and an empty place, each up to itself."""
    _, *rest, table, _ = make([37, 20], 8, 2, 64, 8, F16)
    rows = torch.tensor([0] * 37 + [1] * 20 + [-1, 2, 0], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([*range(1, 38), *range(1, 21), 0, 5, 0], dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    check(torch.randn(60, 8, 64, generator=g, device=DEV).to(F16), *rest, table, lengths, rows=rows)


def test_pages_outside_the_cache_are_left_out():
    q, k, v, ks, vs, table, n = make([50, 50, 50], 4, 2, 64, 8, F16)
    table[0, 2], table[1, :] = -1, 2 ** 31 - 1
    table[2, 0], table[2, 6] = k.shape[0], -5
    check(q, k, v, ks, vs, table, n)
    check(q, k, v, ks, vs, table, torch.tensor([2 ** 31 - 1, -4, 10 ** 6], dtype=torch.int32, device=DEV)[[1, 1, 1]])
    # a length behind the table ends with it
    q, k, v, ks, vs, table, n = make([48], 4, 2, 64, 8, F16)
    table = table[:, :6].contiguous()
    got = _C_ops.paged_attention_quantised(q, k, v, ks, vs, table, torch.full_like(n, 2 ** 31 - 1))
    assert torch.equal(got, _C_ops.paged_attention_quantised(q, k, v, ks, vs, table, n))


def test_what_is_no_number():
    """A group without a number makes what it meets NaN: a value's, its elements; a key's or a query's, its heads."""
    for dtype in (F16, BF16):
        q, k, v, ks, vs, table, n = make([100, 40], 4, 2, 128, 16, dtype, 2)
        clean = _C_ops.paged_attention_quantised(q, k, v, ks, vs, table, n)
        vs[table[0, 1], 5, 0, 1, 0] = NAN
        got = _C_ops.paged_attention_quantised(q, k, v, ks, vs, table, n)
        assert torch.isnan(got[0, :2, 64:]).all() and torch.equal(got[0, :2, :64], clean[0, :2, :64]) and torch.equal(got[0, 2:], clean[0, 2:])
        assert torch.equal(got[1], clean[1])
        vs[table[0, 1], 5, 0, 1, 0] = 0.25
        ks[table[0, 2], 3, 1, 0, 0] = NAN
        q[1, 0, 7] = NAN
        got = _C_ops.paged_attention_quantised(q, k, v, ks, vs, table, n)
        assert torch.isnan(got[0, 2:]).all() and torch.isfinite(got[0, :2]).all() and torch.isnan(got[1, 0]).all() and torch.isfinite(got[1, 1:]).all()
        q[1, 0, 7] = math.inf
        assert not torch.isfinite(_C_ops.paged_attention_quantised(q, k, v, ks, vs, table, n)[1, 0]).any()


def test_strides_outputs_streams_and_capture():
    q, *rest, table, n = make([100, 7, 0, 400], 8, 2, 64, 16, F16)
    call = lambda q, table, n, **kw: _C_ops.paged_attention_quantised(q, *rest, table, n, **kw)         # noqa: E731
    want = call(q, table, n)
    fused = torch.zeros(4, 12, 64, dtype=F16, device=DEV)
    fused[:, 2:10] = q
    assert torch.equal(call(fused[:, 2:10], table, n), want)
    odd = torch.zeros(4, 8, 67, dtype=F16, device=DEV)[:, :, 1:65]
    odd.copy_(q)
    assert torch.equal(call(odd, table, n), want)
    wide = torch.full((4, 9, 72), 5.0, dtype=F16, device=DEV)
    out = wide[:, 1:, :64]
    assert call(q, table, n, out=out) is out and torch.equal(out, want)
    assert (wide[:, 0] == 5).all() and (wide[:, :, 64:] == 5).all()
    same = q.clone()
    assert torch.equal(call(same, table, n, out=same), want)
    part = torch.zeros(4, table.shape[1] + 3, dtype=torch.int32, device=DEV)[:, 1:-2]
    part.copy_(table)
    assert torch.equal(call(q, part, n.repeat_interleave(2)[::2]), want)
    # the same cache in other places: rows that are no multiples of 16 bytes, token by token
    for pitch in (32, 36, 48):
        other = [torch.zeros(*c.shape[:3], pitch, dtype=torch.uint8, device=DEV)[..., :32].copy_(c) for c in rest[:2]] + [c.contiguous() for c in rest[2:]]
        assert torch.equal(_C_ops.paged_attention_quantised(q, *other, table, n), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [call(q, table, n) for _ in range(5)]
    mine = [call(q, table, n) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got + mine)
    graph, x, m = torch.cuda.CUDAGraph(), q.clone(), n.clone()
    with torch.cuda.graph(graph):
        got = call(x, table, m)
    x.copy_(q * 2)
    m.copy_(torch.tensor([33, 0, 0, 16], dtype=torch.int32))
    graph.replay()
    assert torch.equal(got, call(q * 2, table, m))
    assert call(q[:0], table[:0], n[:0]).shape == (0, 8, 64)
    assert (_C_ops.paged_attention_quantised(q, *(c[:0] for c in rest), table, n) == 0).all()


# ---- requests that pass through many CTAs and CTAs that pass through many requests, for every variant of the kernel
SHAPES = [(D, groups, G) for D, groups in ((64, 1), (96, 1), (112, 1), (128, 1), (128, 2)) for G in (3, 12, 24, 40)] \
    + [(D, groups, G) for D, groups in ((192, 1), (192, 3), (256, 1), (256, 4)) for G in (3, 12, 24)]


def widened(table, columns):
    """The same rows in a table of more columns, with nonsense behind."""
    wide = torch.full((table.shape[0], max(columns, table.shape[1])), 2 ** 30, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    return wide


def check_some(q, *rest, pick, **kw):
    cache, table, n = rest[:4], rest[4], rest[5]
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    got = _C_ops.paged_attention_quantised(q, *rest, lse=lse, **kw)
    assert torch.isfinite(got).all() and (got[n == 0] == 0).all() and torch.equal(torch.isinf(lse), (n == 0).view(-1, 1).expand_as(lse))
    want, want_lse, bound, lse_bound = quantised_ops.attention(q[pick], *cache, table[pick], n[pick], q.shape[2] ** -0.5, **kw)
    plain_ops.within(got[pick], want, plain_ops.rounded(want, bound, q.dtype), "out")
    seen = n[pick] > 0
    plain_ops.within(lse[pick][seen], want_lse[seen], lse_bound[seen], "lse")
    again = torch.zeros_like(lse)
    assert torch.equal(_C_ops.paged_attention_quantised(q, *rest, lse=again, **kw), got) and torch.equal(again, lse)
    assert _lib.lib().ortho_b200_query_kernel_status() == 0


def kinds(D, G):
    return F16 if (D // 8 + G) % 2 else BF16


@pytest.mark.parametrize("D,groups,G", SHAPES)
def test_a_request_over_many_ctas(D, groups, G):
    q, *cache, table, n = make([60011], 2 * G, 2, D, 256, kinds(D, G), groups, seed=D + G)
    check_some(q, *cache, widened(table, 800), n, pick=[0])
    check_some(q, *cache, widened(table, 800), n - 13000, pick=[0], window=9999)


@pytest.mark.parametrize("D,groups,G", SHAPES)
def test_many_requests_to_a_cta(D, groups, G):
    lengths = [0 if i % 7 == 3 else (i * 7919) % 200 for i in range(400)]
    lengths[17], lengths[390] = 3000, 1777
    q, *cache, table, n = make(lengths, 2 * G, 2, D, 64, kinds(D, G), groups, seed=D * G)
    check_some(q, *cache, widened(table, 96), n, pick=[0, 1, 2, 3, 16, 17, 18, 199, 200, 201, 389, 390, 391, 398, 399])


def test_ctas_of_a_cluster_that_start_and_end_at_different_times():
    """Few items of very different lengths, behind a kernel that leaves the CTAs' room bit by bit: the same bits every time."""
    args = make([1, 3000, 64, 0, 513, 65], 4, 2, 64, 16, F16)
    want = check(*args)
    x, y, down, up, ids = (torch.randn(64, 2048, device=DEV, dtype=F16), torch.randn(64, 2048, device=DEV, dtype=F16),
                           torch.randn(9, 16, 2048, device=DEV, dtype=F16), torch.randn(9, 2048, 16, device=DEV, dtype=F16),
                           torch.arange(64, device=DEV, dtype=torch.int32) % 9)
    got = []
    for _ in range(100):
        _C_ops.low_rank_add(x, y, down, up, ids)
        got.append(_C_ops.paged_attention_quantised(*args))
    assert all(torch.equal(g, want) for g in got)


def test_refusals():
    q, k, v, ks, vs, table, n = make([9, 9], 4, 2, 64, 8, F16)
    base = dict(q=q, k_cache=k, v_cache=v, k_scales=ks, v_scales=vs, block_table=table, lengths=n)

    def refused(error, match, **change):
        with pytest.raises(error, match=match):
            _C_ops.paged_attention_quantised(**{**base, **change})
    refused(RuntimeError, "CPU", q=q.cpu())
    refused(RuntimeError, "CPU", v_scales=vs.cpu())
    refused(TypeError, "q must be", q=q.float())
    refused(TypeError, "k_cache", k_cache=k.to(torch.int8))
    refused(TypeError, "k_scales", k_scales=ks.to(BF16))
    refused(TypeError, "k_scales", q=q.to(BF16))
    refused(TypeError, "block_table", block_table=table.long())
    refused(ValueError, "lengths", lengths=n[:1])
    refused(ValueError, "block_table", block_table=table[:1])
    refused(ValueError, "heads", q=q[:, :3])
    refused(ValueError, "head_dim", q=q[..., :32])
    refused(ValueError, "alike", v_cache=v[:1])
    refused(ValueError, "alike", k_scales=ks[:1], v_scales=vs[:1])
    refused(ValueError, "window", window=-1)
    refused(ValueError, "rows", rows=n[:1])
    refused(ValueError, "out", out=q[:1])
    refused(ValueError, "lse", lse=torch.zeros(2, 3, device=DEV))
    refused(TypeError, "q must be a tensor", q=None)
