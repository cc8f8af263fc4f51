"""Attention over a cache held in 4 bits: lengths behind the table together with pages outside the cache, and lengths below zero beside others."""
import pytest
import torch

import plain_ops
import quantised_ops
from libortho_b200 import _C_ops
from test_gpu_quantised_attention import make, widened

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[2 ** 31 - 1, -4, 10 ** 6], [-4, -2 ** 31, -1], [57, 2 ** 31 - 1, 0], [2 ** 31 - 1] * 3])
@pytest.mark.parametrize("columns,window", [(1, 0), (1, 13), (300, 0)])
def test_lengths_and_pages_outside(columns, window, lengths, dtype):
    """Columns behind a request's pages name pages far outside the cache; so do some between them.  Two requests have six places on their last page that hold no number: a length that
    takes these in gives none."""
    q, k, v, ks, vs, table, _ = make([50, 50, 56], 4, 2, 64, 8, dtype)
    table = widened(table, columns)
    table[0, 2], table[1, 0], table[2, 3] = -1, 2 ** 31 - 1, k.shape[0]
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want, want_lse, bound, lse_bound = quantised_ops.attention(q, k, v, ks, vs, table, n, 0.125, window=window)
    lse = torch.full_like(want_lse, 7.0, dtype=torch.float32)
    got = _C_ops.paged_attention_quantised(q, k, v, ks, vs, table, n, lse=lse, window=window)
    some = ~want.isnan()
    assert torch.equal(got.isnan(), ~some) and torch.equal(lse.isnan(), want_lse.isnan()) and torch.equal(lse.isinf(), want_lse.isinf())
    plain_ops.within(got[some], want[some], plain_ops.rounded(want, bound, dtype)[some], "out")
    seen = torch.isfinite(want_lse)
    plain_ops.within(lse[seen], want_lse[seen], lse_bound[seen], "lse")
    assert (got[want_lse.isinf()] == 0).all()
