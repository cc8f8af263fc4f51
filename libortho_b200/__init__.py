"""libortho_b200 -- the OrthoLinear forward for NVIDIA B200 (sm_100a).

The main operator: ``Y = X . dequant(W_base_int4)^T + alpha . X . W_ortho^T`` behind the reference's
``OrthoLinear`` / ``set_alpha`` API, executed by hand-written CUDA kernels reached through a
C ABI (``include/ortho_b200.h``).  Around it, the operators of a decoding step: page bookkeeping
and a paged key-value cache, in 16 or 4 bits (``PagePool``, ``PagedCache``, ``QuantisedCache``), rotary positions, attention of one new
token over the cache, low-rank adapters of many requests (``LowRankAdapters``), put together in
``PagedAttentionBlock``.  Importing the package does not load the CUDA library; the
first operator call does, and fails loudly if it has not been built.
"""
from .ortho_linear import OrthoLinear  # noqa: F401
from . import _C_ops  # noqa: F401
from ._C_ops import PageStep  # noqa: F401
from .adapters import LowRankAdapters  # noqa: F401
from .convert import set_alpha_all, swap_linear  # noqa: F401
from .paged import PagedAttentionBlock, PagedCache, PagePool, QuantisedCache, rotary_table  # noqa: F401

__all__ = ["OrthoLinear", "_C_ops", "swap_linear", "set_alpha_all", "LowRankAdapters", "PagedAttentionBlock", "PagedCache",
           "PagePool", "PageStep", "QuantisedCache", "rotary_table"]
__version__ = "0.1.0"
