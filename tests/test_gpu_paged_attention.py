"""Attention of one token over a paged cache against 64 bits."""
import math

import pytest
import torch

import plain_ops
from libortho_b200 import _C_ops, _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16
NAN = float("nan")


def make(lengths, Hq, Hkv, D, P, dtype, seed=0, layout="phd", std=1.0, spare=2):
    """Inputs whose unused places -- behind a length, pages of nobody, table entries behind the last page -- hold NaN or nonsense."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // P) for n in lengths]
    W, total = max(need + [1]) + 1, sum(need) + spare
    perm = torch.randperm(total, generator=g, device=DEV).tolist()
    table, at = torch.full((len(lengths), W), 2 ** 30, dtype=torch.int32), 0
    shape = {"phd": (total, P, Hkv, D), "hpd": (total, Hkv, P, D), "both": (total, 2, P, Hkv, D)}[layout]
    if layout == "both":
        both = torch.full(shape, NAN, dtype=dtype, device=DEV)
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = (torch.full(shape, NAN, dtype=dtype, device=DEV) for _ in range(2))
        if layout == "hpd":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
    for b, n in enumerate(lengths):
        for j in range(need[b]):
            table[b, j] = perm[at]
            m = min(P, n - j * P)
            for c in (k, v):
                c[perm[at], :m] = torch.randn(m, Hkv, D, generator=g, device=DEV).to(dtype)
            at += 1
    q = (torch.randn(len(lengths), Hq, D, generator=g, device=DEV) * std).to(dtype)
    return q, k, v, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)


def check(q, k, v, table, lengths, scale=None, **kw):
    out, lse, bound, lse_bound = plain_ops.attention(q, k, v, table, lengths, q.shape[2] ** -0.5 if scale is None else scale, **kw)
    got_lse = torch.full_like(lse, 7.0, dtype=torch.float32)
    got = _C_ops.paged_attention(q, k, v, table, lengths, scale=scale, lse=got_lse, **kw)
    assert got.shape == q.shape and got.dtype == q.dtype
    plain_ops.within(got, out, plain_ops.rounded(out, bound, q.dtype), "out")
    empty = torch.isinf(lse)
    assert torch.equal(torch.isinf(got_lse), empty) and (got_lse[empty] < 0).all() and (got[empty] == 0).all()
    plain_ops.within(got_lse[~empty], lse[~empty], lse_bound[~empty], "lse")
    assert torch.equal(got, _C_ops.paged_attention(q, k, v, table, lengths, scale=scale, **kw))          # the same bits again
    assert _lib.lib().ortho_b200_query_kernel_status() == 0
    return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 8), (8, 1), (10, 2), (18, 2), (24, 1), (33, 1), (32, 2), (71, 1)])
@pytest.mark.parametrize("D", [8, 64, 80, 128, 256])
def test_heads(Hq, Hkv, D, dtype):
    check(*make([0, 1, 17, 300, 64], Hq, Hkv, D, 16, dtype, seed=Hq + D))


@pytest.mark.parametrize("D", [16, 24, 32, 40, 48, 56, 72, 88, 96, 104, 112, 120, 136, 160, 192, 200, 224, 248])
def test_head_dims(D):
    check(*make([5, 130], 6, 2, D, 8, BF16, seed=D))
    check(*make([70], 17, 1, D, 8, F16, seed=D))


@pytest.mark.parametrize("P", [1, 2, 3, 5, 16, 24, 64, 100, 128, 4096])
@pytest.mark.parametrize("layout", ["phd", "hpd", "both"])
def test_pages(P, layout):
    check(*make([0, 1, P, P + 1, max(1, P - 1), 2 * P, 333], 4, 2, 64, P, F16, seed=P, layout=layout))


@pytest.mark.parametrize("lengths", [[1], [15], [16], [17], [63], [64], [65], [127], [128], [129], [1000], [5000], [0], [0, 0, 0], [0, 9, 0],
                                     list(range(40)), [4000, 1, 1, 1, 1, 1, 1], [3, 0, 2500, 0, 64, 128]])
def test_lengths(lengths):
    check(*make(lengths, 8, 2, 128, 16, BF16, seed=sum(lengths)))
    check(*make(lengths, 4, 4, 64, 16, F16, seed=sum(lengths)))


@pytest.mark.parametrize("B,Hq,Hkv,L", [(300, 2, 1, 9), (64, 8, 8, 200), (1500, 1, 1, 3), (5000, 1, 1, 2)])
def test_many_requests(B, Hq, Hkv, L):
    lengths = [(i * 7919) % (L + 1) for i in range(B)]
    q, k, v, table, n = make(lengths, Hq, Hkv, 64, 8, F16, seed=B)
    got, lse = _C_ops.paged_attention(q, k, v, table, n), None
    pick = torch.arange(0, B, max(1, B // 60), device=DEV)
    out, lse, bound, _ = plain_ops.attention(q[pick], k, v, table[pick], n[pick], 0.125)
    plain_ops.within(got[pick], out, plain_ops.rounded(out, bound, F16))
    assert (got[n == 0] == 0).all() and torch.isfinite(got).all()


def test_a_long_cache():
    """100,000 keys, far more splits than a CTA has threads."""
    for Hq, Hkv, dtype in ((8, 1, F16), (3, 3, BF16)):
        check(*make([100000, 33], Hq, Hkv, 64, 256, dtype))


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
        got.append(_C_ops.paged_attention(*args))
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 100, 1000])
def test_windows(window):
    check(*make([0, 1, 50, 64, 101, 700], 6, 2, 64, 8, F16, seed=window), window=window)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 4.0])
def test_scales(scale):
    check(*make([1, 40, 333], 4, 2, 64, 16, F16), scale=scale)


def test_one_key_that_outweighs_the_rest_and_many_that_weigh_little():
    q, k, v, table, n = make([2000], 8, 1, 64, 16, F16)
    k[table[0, 70], 3] = (q[0, 0] * 3).to(F16)                                # a score some 20 above the others
    check(q, k, v, table, n, scale=0.3)
    k.mul_(0.01)
    check(q, k, v, table, n)


def test_scores_that_grow_and_fall():
    """The running maximum changes in every tile, or never after the first."""
    for order in (1, -1):
        q, k, v, table, n = make([1500], 4, 1, 64, 16, BF16)
        ramp = torch.linspace(0, 6, 1500, device=DEV)[::1] if order > 0 else torch.linspace(6, 0, 1500, device=DEV)
        for j in range(1500):
            k[table[0, j // 16], j % 16, 0] = (q[0, 1].float() * ramp[j] / 8).to(BF16)
        check(q, k, v, table, n)


def test_rows_that_share_requests():
    """The tokens of two prompts and an empty place, each up to itself."""
    q, k, v, table, _ = make([37, 20], 8, 2, 64, 8, F16)
    rows = torch.tensor([0] * 37 + [1] * 20 + [-1, 2, 0], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([*range(1, 38), *range(1, 21), 0, 5, 0], dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    check(torch.randn(60, 8, 64, generator=g, device=DEV).to(F16), k, v, table, lengths, rows=rows)


def test_pages_outside_the_cache_are_left_out():
    q, k, v, table, n = make([50, 50, 50], 4, 2, 64, 8, F16)
    table[0, 2], table[1, :] = -1, 2 ** 31 - 1
    table[2, 0], table[2, 6] = k.shape[0], -5
    check(q, k, v, table, n)
    check(q, k, v, table, torch.tensor([2 ** 31 - 1, -4, 10 ** 6], dtype=torch.int32, device=DEV)[[1, 1, 1]])
    # a length behind the table ends with it
    q, k, v, table, n = make([48], 4, 2, 64, 8, F16)
    table = table[:, :6].contiguous()
    got = _C_ops.paged_attention(q, k, v, table, torch.full_like(n, 2 ** 31 - 1))
    assert torch.equal(got, _C_ops.paged_attention(q, k, v, table, n))


def test_infinite_values_and_keys():
    """What is visible acts as the formula says; what is not has no effect (NaN fills the unused places of every test here)."""
    for dtype in (F16, BF16):
        q, k, v, table, n = make([100], 2, 1, 64, 16, dtype)
        clean = _C_ops.paged_attention(q, k, v, table, n)
        v[table[0, 1], 5, 0, 7] = math.inf
        v[table[0, 3], 2, 0, 9] = NAN
        got = _C_ops.paged_attention(q, k, v, table, n)
        assert (got[0, :, 7] == math.inf).all() and torch.isnan(got[0, :, 9]).all()
        rest = [i for i in range(64) if i not in (7, 9)]
        assert torch.equal(got[:, :, rest], clean[:, :, rest])
        # a key with a score of minus infinity for head 0 (and NaN or infinity elsewhere is that head's own)
        q[0, 0], q[0, 1] = 1.0, 0.5
        k[table[0, 0], 0, 0, 0] = -math.inf
        got = _C_ops.paged_attention(q, k, v, table, n)
        other = k.clone()
        other[table[0, 0], 0] = -1000.0
        v[table[0, 1], 5, 0, 7] = v[table[0, 3], 2, 0, 9] = 0.0
        got = _C_ops.paged_attention(q, k, v, table, n)
        plain_ops.within(got, *(lambda o, lse, b, _: (o, plain_ops.rounded(o, b, dtype)))(*plain_ops.attention(q, other, v, table, n, 0.125)))


def test_strides_outputs_streams_and_capture():
    q, k, v, table, n = make([100, 7, 0, 400], 8, 2, 64, 16, F16)
    want = _C_ops.paged_attention(q, k, v, table, n)
    fused = torch.zeros(4, 12, 64, dtype=F16, device=DEV)
    fused[:, 2:10] = q
    assert torch.equal(_C_ops.paged_attention(fused[:, 2:10], k, v, table, n), want)
    odd = torch.zeros(4, 8, 67, dtype=F16, device=DEV)[:, :, 1:65]
    odd.copy_(q)
    assert torch.equal(_C_ops.paged_attention(odd, k, v, table, n), want)
    wide = torch.full((4, 9, 72), 5.0, dtype=F16, device=DEV)
    out = wide[:, 1:, :64]
    assert _C_ops.paged_attention(q, k, v, table, n, out=out) is out and torch.equal(out, want)
    assert (wide[:, 0] == 5).all() and (wide[:, :, 64:] == 5).all()
    same = q.clone()
    assert torch.equal(_C_ops.paged_attention(same, k, v, table, n, out=same), want)
    part = torch.zeros(4, table.shape[1] + 3, dtype=torch.int32, device=DEV)[:, 1:-2]
    part.copy_(table)
    assert torch.equal(_C_ops.paged_attention(q, k, v, part, n.repeat_interleave(2)[::2]), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [_C_ops.paged_attention(q, k, v, table, n) for _ in range(5)]
    mine = [_C_ops.paged_attention(q, k, v, table, n) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got + mine)
    graph, x, m = torch.cuda.CUDAGraph(), q.clone(), n.clone()
    with torch.cuda.graph(graph):
        got = _C_ops.paged_attention(x, k, v, table, m)
    x.copy_(q * 2)
    m.copy_(torch.tensor([33, 0, 0, 16], dtype=torch.int32))
    graph.replay()
    assert torch.equal(got, _C_ops.paged_attention(q * 2, k, v, table, m))
    assert _C_ops.paged_attention(q[:0], k, v, table[:0], n[:0]).shape == (0, 8, 64)
    none = _C_ops.paged_attention(q, k[:0], v[:0], table, n)
    assert (none == 0).all()


def test_parts_of_a_cache():
    """Two parts of a request, each against 64 bits, and the sums of exponentials of the parts against the whole's."""
    q, k, v, table, n = make([90], 4, 2, 64, 8, F16)
    whole, first, second = (torch.empty(1, 4, device=DEV) for _ in range(3))
    for t, m, lse in ((table, 90, whole), (table[:, :5].contiguous(), 40, first), (table[:, 5:].contiguous(), 50, second)):
        m = torch.full_like(n, m)
        got = check(q, k, v, t, m)
        assert torch.equal(_C_ops.paged_attention(q, k, v, t, m, lse=lse), got)
    top = torch.logaddexp(first.double(), second.double())
    plain_ops.within(whole, top, 1e-5 * top.abs() + 1e-5)


def test_refusals():
    q, k, v, table, n = make([9, 9], 4, 2, 64, 8, F16)
    base = dict(q=q, k_cache=k, v_cache=v, block_table=table, lengths=n)

    def refused(error, match, **change):
        with pytest.raises(error, match=match):
            _C_ops.paged_attention(**{**base, **change})
    refused(RuntimeError, "CPU", q=q.cpu())
    refused(RuntimeError, "CPU", lengths=n.cpu())
    refused(TypeError, "q must be", q=q.float())
    refused(TypeError, "k_cache", k_cache=k.to(BF16))
    refused(TypeError, "block_table", block_table=table.long())
    refused(TypeError, "lengths", lengths=n.long())
    refused(ValueError, "lengths", lengths=n[:1])
    refused(ValueError, "block_table", block_table=table[:1])
    refused(ValueError, "block_table", block_table=table.T.contiguous().T)
    refused(ValueError, "heads", q=q[:, :3])
    refused(ValueError, "head_dim", q=q[..., :32])
    refused(ValueError, "multiple of 8", q=q[..., :60], k_cache=k[..., :60], v_cache=v[..., :60])
    big = torch.zeros(1, 8, 1, 264, dtype=F16, device=DEV)
    refused(ValueError, "256", q=big[0, :2], k_cache=big, v_cache=big)
    refused(ValueError, "alike", v_cache=v[:1])
    refused(ValueError, "contiguous", k_cache=k.transpose(2, 3).contiguous().transpose(2, 3))
    shifted = torch.zeros(k.numel() + 1, dtype=F16, device=DEV)[1:].view(k.shape)
    refused(ValueError, "aligned", k_cache=shifted)
    refused(ValueError, "window", window=-1)
    refused(ValueError, "rows", rows=n[:1])
    refused(TypeError, "rows", rows=n.long())
    refused(ValueError, "out", out=q[:1])
    refused(ValueError, "lse", lse=torch.zeros(2, 3, device=DEV))
    refused(TypeError, "lse", lse=torch.zeros(2, 4, device=DEV, dtype=F16))
    refused(TypeError, "q must be a tensor", q=None)
