"""Attention over a cache held in 4 bits where sizes of scales lie far apart: from request to request, head to head and key to key.

The bound on a head's outputs: their own rounding, which is known, and what the kernel is off before it.  The two are independent, so that squares of norms add up.
FP16 weights have two parts, 2^-21: scores off by some 2^-18 and cuts of sums leave 2^-13 of the outputs' norm plenty of room.  BF16 weights have one, 2^-11 each, of what are
8 scales at most where outputs may be less: 2^-10."""
import pytest
import torch

import quantised_ops
from libortho_b200 import _C_ops
from test_gpu_quantised_attention import make, widened

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16
BEFORE = {F16: 2.0 ** -13, BF16: 2.0 ** -10}


def plain(q, *rest, **kw):
    return quantised_ops.attention(q, *rest, q.shape[2] ** -0.5, **kw)[0]


def near(got, want):
    assert torch.isfinite(got).all()
    rounding = (quantised_ops.nearest(want, got.dtype) - want).norm(dim=-1)
    most = (rounding ** 2 + (BEFORE[got.dtype] * want.norm(dim=-1)) ** 2).sqrt()
    off = (got.double() - want).norm(dim=-1)
    assert (off <= most).all(), f"{float((off / most).max()):.3g} times the bound"


def times(scales, pages, factor, head=slice(None)):
    scales[pages, :, head] = (scales[pages, :, head].double() * factor).to(scales.dtype)


@pytest.mark.parametrize("dtype,far", [(F16, 9), (BF16, 24), (BF16, 60)])
@pytest.mark.parametrize("D,groups,G", [(64, 1, 2), (96, 1, 12), (128, 1, 2), (128, 2, 8), (128, 1, 24), (192, 3, 8), (256, 1, 16)])
def test_requests_and_heads_beside_larger_ones(D, groups, G, dtype, far):
    """Values of every other request, and of every other head, 2^far times as large and as small: the same bits as where the neighbours are of one size with them."""
    lengths = [(i * 7919) % 200 + 1 for i in range(300)]
    q, k, v, ks, vs, table, n = make(lengths, 2 * G, 2, D, 64, dtype, groups, seed=D + G)
    table = widened(table, 96)
    pages = [table[b, :-(-m // 64)].long() for b, m in enumerate(lengths)]
    for b in range(300):
        times(vs, pages[b], 2.0 ** (-far if b % 2 else 0.0))
    want = _C_ops.paged_attention_quantised(q, k, v, ks, vs, table, n)
    for b in range(0, 300, 2):
        times(vs, pages[b], 2.0 ** far)
    got = _C_ops.paged_attention_quantised(q, k, v, ks, vs, table, n)
    assert torch.equal(got[1::2], want[1::2])
    pick = [0, 1, 2, 3, 150, 151, 298, 299]
    near(got[pick], plain(q[pick], k, v, ks, vs, table[pick], n[pick]))
    for b in range(300):
        times(vs, pages[b], 2.0 ** (far if b % 2 else -2 * far if b % 4 else -far), head=1)
        times(vs, pages[b], 2.0 ** (far if b % 2 else -far), head=0)
    got = _C_ops.paged_attention_quantised(q, k, v, ks, vs, table, n)
    near(got[pick], plain(q[pick], k, v, ks, vs, table[pick], n[pick]))


@pytest.mark.parametrize("dtype,far", [(F16, 20), (BF16, 24), (BF16, 50)])
@pytest.mark.parametrize("G", [4, 12, 24])
@pytest.mark.parametrize("at", [0, 77, 1999])
def test_a_key_of_large_scale_that_weighs_nothing(at, G, dtype, far):
    """One of 2000 keys has value scales 2^far times as large, and a score some 70 below the others'."""
    for width in (1, 900):                       # few items to a cluster, and the even cut
        q, k, v, ks, vs, table, n = make([2000], G, 1, 64, 16, dtype, seed=at)
        q.abs_()
        times(vs, table[0, :125].long(), 2.0 ** -9)
        page, place = table[0, at // 16].long(), at % 16
        vs[page, place] = (vs[page, place].double() * 2.0 ** far).to(dtype)
        ks[page, place, :, :, 1] -= 12.0
        near(_C_ops.paged_attention_quantised(q, k, v, ks, vs, widened(table, width), n), plain(q, k, v, ks, vs, table, n))


@pytest.mark.parametrize("dtype,far", [(F16, 8), (BF16, 40)])
@pytest.mark.parametrize("D,groups,G", [(64, 1, 4), (128, 2, 12), (64, 1, 24), (256, 1, 8)])
def test_scales_that_rise_and_fall_along_a_request(D, groups, G, dtype, far):
    """Value scales from 2^-far to 2^far, and back: with equal scores, and with scores that go the other way, so that all keys count alike."""
    for order in (1, -1):
        for against in (0.0, 1.0):
            q, k, v, ks, vs, table, n = make([1600], G, 1, D, 16, dtype, groups, seed=G)
            q = torch.full_like(q, D ** -0.5)
            ramp = torch.linspace(-order * far, order * far, 1600, device=DEV, dtype=torch.float64)
            held = table[0, :100].long()
            vs[held] = (vs[held].double() * (2.0 ** ramp).view(100, 16, 1, 1, 1)).to(dtype)
            # score = zero * D * D^-1/2 * D^-1/2 = zero: log 2 for a power of two
            ks[held] = 0
            ks[held, :, 0, :, 1] = (-against * 0.6931471805599453 * ramp).view(100, 16, 1).to(dtype)
            near(_C_ops.paged_attention_quantised(q, k, v, ks, vs, table, n), plain(q, k, v, ks, vs, table, n))


@pytest.mark.parametrize("D,groups,G", [(64, 1, 4), (128, 2, 4), (128, 1, 12), (96, 1, 24), (256, 1, 4)])
def test_sizes_near_the_ends_of_a_type(D, groups, G):
    """Keys of 2^112 with queries of 2^-112, and the other way round; values of 2^112 and 2^-90: beside ordinary requests, which give the same bits without them."""
    lengths = [300 if b % 3 else (b * 7919) % 200 + 1 for b in range(60)]
    q, k, v, ks, vs, table, n = make(lengths, 2 * G, 2, D, 64, BF16, groups, seed=D)
    table = widened(table, 96)
    want = _C_ops.paged_attention_quantised(q, k, v, ks, vs, table, n)
    for b in range(0, 60, 2):
        pages, far = table[b, :-(-lengths[b] // 64)].long(), 112 if b % 4 else -112
        times(ks, pages, 2.0 ** far)
        q[b] = (q[b].double() * 2.0 ** -far).to(BF16)
        times(vs, pages, 2.0 ** (112 if b % 8 < 4 else -90))
    got = _C_ops.paged_attention_quantised(q, k, v, ks, vs, table, n)
    assert torch.equal(got[1::2], want[1::2])
    pick = list(range(12)) + [56, 57, 58, 59]
    near(got[pick], plain(q[pick], k, v, ks, vs, table[pick], n[pick]))
