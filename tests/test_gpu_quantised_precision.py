"""Attention over a cache held in 4 bits: how many outputs are not the exact ones rounded once, and how far ``lse`` is off.

An output x = sigma * normal that is off by d sigma before it is rounded comes out otherwise where x lies that near a border between two numbers of the type.  Borders are some 2^-p |x| apart,
p = 10.5 (FP16) and 7.5 (BF16) on the average, so with y = E|normal| d 2^p this happens to about E|normal| y (log(1 / y) + 1) of the outputs (E|normal| = 0.8; the last term: |x| below y sigma).
Scores are off by some 3e-7 where they are about one, exponentials by 2^-22, weights by 2^-21, sums by the tensor core's cuts, 2^-25 of the largest product each, which count
in one direction: d = 2^-17 leaves room for what 100000 keys make of them."""
import math

import pytest
import torch

import plain_ops
import quantised_ops
from libortho_b200 import _C_ops
from test_gpu_quantised_attention import make, widened

DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def share(dtype, n, d=2.0 ** -17):
    """Most of n outputs that may be rounded otherwise: what is expected, and four times its spread."""
    y = 0.8 * d * 2 ** (10.5 if dtype == F16 else 7.5)
    f = 0.8 * y * (math.log(1 / y) + 1)
    return f + 4 * math.sqrt(f / n)


def otherwise(got, want):
    return float((got.double() != quantised_ops.nearest(want, got.dtype)).double().mean())


def lse_bound(q, ks, lse, keys):
    """A step of the tensor core (16 elements) cuts its terms and its sum 2^-23 below the largest of them: at most 15 sum |q| + 8 |sum q| of a query's group times a key's scale.  FP32 beyond."""
    D, G = q.shape[2], ks.shape[-2]
    x = q.double().view(*q.shape[:2], G, D // G)
    sizes = 15 * x.abs().sum(-1) + 8 * x.sum(-1).abs()
    most = ks[..., 0].double().nan_to_num(0).abs().max()
    return D / 16 * 2.0 ** -22 * sizes.sum(-1) * most * D ** -0.5 + (keys + 16) * plain_ops.E32 + 4 * plain_ops.E32 * lse.abs()


CASES = [([3 + i % 50 for i in range(64)], 8, 8, 128, 1, 1.0), ([3 + i % 50 for i in range(64)], 12, 1, 64, 1, 1.0), ([1000, 700, 333, 90], 16, 4, 128, 2, 1.0), ([1000, 700, 333, 90], 32, 1, 96, 1, 1.0),
         ([3000] * 4, 10, 5, 80, 1, 1.0), ([5000, 2500], 24, 2, 256, 4, 1.0), ([5000, 2500], 16, 8, 192, 1, 1.0), ([131072], 16, 2, 128, 1, 0.1), ([100000], 24, 1, 128, 2, 0.1), ([100000, 60000], 32, 1, 64, 1, 0.1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lengths,Hq,Hkv,D,groups,std", CASES)
def test_outputs_are_rounded_as_the_exact_ones(lengths, Hq, Hkv, D, groups, std, dtype):
    q, *cache, table, n = make(lengths, Hq, Hkv, D, 64, dtype, groups, seed=D + Hq, std=std)
    lse = torch.empty(q.shape[:2], device=DEV)
    want, want_lse, _, _ = quantised_ops.attention(q, *cache, table, n, D ** -0.5)
    for columns in (1, 40):                      # few items to a cluster; a table that is wider than the requests has them cut
        got = _C_ops.paged_attention_quantised(q, *cache, widened(table, columns), n, lse=lse)
        off = otherwise(got, want)
        assert off <= share(dtype, got.numel()), f"{off:.3g} of the outputs against {share(dtype, got.numel()):.3g}"
        plain_ops.within(lse, want_lse, lse_bound(q, cache[2], want_lse, max(lengths)), "lse")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Hq,Hkv,D,groups", [(8, 2, 64, 1), (24, 2, 96, 1), (8, 8, 128, 2), (48, 2, 128, 1), (16, 1, 256, 4)])
def test_a_key_alone_gives_its_value(Hq, Hkv, D, groups, dtype):
    """One key weighs one: zero + scale code, rounded once, with ties (one value in dozens) to even."""
    for B, columns in ((3, 1), (200, 40)):
        q, *cache, table, n = make([1] * B, Hq, Hkv, D, 16, dtype, groups, seed=D)
        got = _C_ops.paged_attention_quantised(q, *cache, widened(table, columns), n)
        want = quantised_ops.held(cache[1][table[:, 0].long(), 0], cache[3][table[:, 0].long(), 0]).repeat_interleave(Hq // Hkv, 1)
        assert torch.equal(got.double(), quantised_ops.nearest(want, dtype))


def test_the_bound_sees_weights_of_few_digits():
    """Weights rounded to 11 bits in the plain form: too many outputs are rounded otherwise."""
    g = torch.Generator().manual_seed(0)
    w, v = torch.rand(64, 300, generator=g, dtype=torch.float64) + 0.1, torch.randn(300, 128, generator=g, dtype=torch.float64)
    want = w @ v / w.sum(1, keepdim=True)
    for digits, dtype in ((11, BF16), (11, F16), (14, F16)):
        e = torch.frexp(w)[1] - digits
        got = (torch.ldexp(torch.round(torch.ldexp(w, -e)), e) @ v / w.sum(1, keepdim=True))
        assert otherwise(got.to(dtype), want) > share(dtype, got.numel()), (digits, dtype)
        assert otherwise(want.to(dtype), want) <= share(dtype, got.numel())
