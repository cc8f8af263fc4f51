"""Attention over a paged cache where the work is cut evenly over the CTAs: every head size with every number of query heads a unit,
requests that pass through many CTAs and CTAs that pass through many requests."""
import ctypes

import pytest
import torch

import plain_ops
from libortho_b200 import _C_ops, _lib
from test_gpu_paged_attention import BF16, DEV, F16, make

pytestmark = pytest.mark.gpu

# query heads for one key-value head: 8, 16 and 32 columns of a unit (32: head dims up to 128), and two units of 16 or 32
SHAPES = [(D, G) for D in (64, 72, 80, 96, 104, 112, 128) for G in (3, 8, 12, 16, 24, 32, 40)] + [(D, G) for D in (136, 192, 200, 256) for G in (3, 8, 12, 16, 24)]


def widened(table, columns):
    """The same rows in a table of more columns, with nonsense behind."""
    wide = torch.full((table.shape[0], max(columns, table.shape[1])), 2 ** 30, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    return wide


def is_cut(q, k, table):
    """Only the even cut needs a workspace."""
    d = _lib.PagedAttentionDesc()
    for name in "q k_cache v_cache out block_table lengths".split():
        setattr(d, name, 256)
    d.batch, d.q_heads, d.head_dim = q.shape
    d.pages, d.page_size, d.kv_heads = k.shape[:3]
    d.rows, d.width = table.shape
    d.type = 0 if q.dtype == F16 else 1
    return _lib.lib().ortho_b200_paged_attention_workspace_bytes(ctypes.byref(d)) > 0


def check(q, k, v, table, n, pick, **kw):
    assert is_cut(q, k, table)
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    got = _C_ops.paged_attention(q, k, v, table, n, lse=lse, **kw)
    assert torch.isfinite(got).all() and (got[n == 0] == 0).all() and torch.equal(torch.isinf(lse), (n == 0).view(-1, 1).expand_as(lse))
    want, want_lse, bound, lse_bound = plain_ops.attention(q[pick], k, v, table[pick], n[pick], q.shape[2] ** -0.5, **kw)
    plain_ops.within(got[pick], want, plain_ops.rounded(want, bound, q.dtype), "out")
    seen = n[pick] > 0
    plain_ops.within(lse[pick][seen], want_lse[seen], lse_bound[seen], "lse")
    again = torch.zeros_like(lse)
    assert torch.equal(_C_ops.paged_attention(q, k, v, table, n, lse=again, **kw), got) and torch.equal(again, lse)
    assert _lib.lib().ortho_b200_query_kernel_status() == 0


def kinds(D, G):
    return F16 if (D // 8 + G) % 2 else BF16


@pytest.mark.parametrize("D,G", SHAPES)
def test_a_request_over_many_ctas(D, G):
    """Some 470 units of 64 keys of each of two key-value heads: a few to every CTA, cut anywhere."""
    q, k, v, table, n = make([30011], 2 * G, 2, D, 256, kinds(D, G), seed=D + G)
    check(q, k, v, widened(table, 400), n, [0])
    check(q, k, v, widened(table, 400), n - 13000, [0], window=9999)


@pytest.mark.parametrize("D,G", SHAPES)
def test_many_requests_to_a_cta(D, G):
    """Some 400 requests, empty ones among them and two long ones: several short items to a CTA, and items that go on in the next one."""
    lengths = [0 if i % 7 == 3 else (i * 7919) % 200 for i in range(400)]
    lengths[17], lengths[390] = 3000, 1777
    q, k, v, table, n = make(lengths, 2 * G, 2, D, 64, kinds(D, G), seed=D * G)
    check(q, k, v, widened(table, 96), n, [0, 1, 2, 3, 16, 17, 18, 199, 200, 201, 389, 390, 391, 398, 399])
