"""A paged key-value cache and the attention part of a decoder block on it.

``PagePool`` keeps the requests' block table and the free pages on the GPU, ``PagedCache`` one layer's keys and values (``QuantisedCache``: in 4 bits),
``PagedAttentionBlock`` runs a step: fused QKV projection (``OrthoLinear``), adapters, rotary positions with the write into
the cache, attention, output projection, adapters.  One step serves requests that decode (one new token) and
requests that bring a prompt (several) alike.  The reference has no counterpart; its operator ends with the projection.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch
import torch.nn as nn

from . import _C_ops as _C
from ._C_ops import PageStep
from .adapters import LowRankAdapters
from .ortho_linear import OrthoLinear


def rotary_table(positions: int, rotary_dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """float32 [positions, rotary_dim]: cosines, then sines, of position * base^(-2 i / rotary_dim), computed in 64 bits (a float32 angle
    of a late position is off by up to 0.03 at 1 million)."""
    if positions < 0 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even")
    i = torch.arange(0, rotary_dim // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device).unsqueeze(1) * base ** (-2 * i / rotary_dim)
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


class PagePool:
    """Block table and free pages of up to ``requests`` requests, on the GPU; no call waits for it.  A request has at most ``max_pages`` pages
    (all, if not given); attention goes by that number when it divides its work, so it should be what the longest request needs.

    ``step(fresh, tokens)`` takes in ``fresh[b]`` new tokens of every request and returns the ``PageStep`` for all
    layers; ``release(which)`` gives the pages of finished requests back.  Pages that ran out show in ``PageStep.counts``
    (pages asked for against those left before) and as slots of -1: such tokens count in the request's length, but their keys are
    nowhere, then and later, and attention goes on without them.  ``incomplete()`` names the requests that this happened to, or that
    went past ``max_pages``; release them and bring their tokens again.  The pool's tensors stay where they are and change in
    place, so both may be captured and replayed; a ``PageStep`` is its own and keeps what it says."""

    def __init__(self, requests: int, pages: int, page_size: int, max_pages: Optional[int] = None, device=None):
        if requests < 1 or pages < 1 or page_size < 1:
            raise ValueError("need requests, pages and a page size")
        device = torch.device("cuda" if device is None else device)
        self.page_size = page_size
        self.block_table = torch.full((requests, max_pages or pages), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.available = torch.full((1,), pages, dtype=torch.int32, device=device)

    def step(self, fresh: torch.Tensor, tokens: int) -> PageStep:
        s = _C.page_step(self.lengths, fresh, self.block_table, self.free_pages, self.available, self.page_size, tokens)
        torch._foreach_copy_([self.lengths, self.available], [s.lengths, s.counts[2:]])    # (one launch)
        return s

    def incomplete(self) -> torch.Tensor:
        """bool [requests]: those of whose tokens some found no page."""
        columns = self.block_table.shape[1]
        need = (self.lengths.long().unsqueeze(1) + self.page_size - 1) // self.page_size
        lacks = (self.block_table < 0) & (torch.arange(columns, device=need.device) < need)
        return lacks.any(dim=1) | (need[:, 0] > columns)

    def release(self, which: torch.Tensor) -> None:
        """``which``: bool [requests].  Their pages go back to the pool, their lengths to zero."""
        mine = (self.block_table >= 0) & which.unsqueeze(1)
        pages = self.block_table.flatten()
        count = mine.flatten().cumsum(0, dtype=torch.int32)
        place = self.available + count - 1
        # entries that give nothing back aim behind the list
        room = torch.cat((self.free_pages, self.free_pages.new_empty(1)))
        room.scatter_(0, torch.where(mine.flatten(), place, self.free_pages.numel()).long(), pages)
        self.free_pages.copy_(room[:-1])
        self.available += count[-1:]
        self.block_table.masked_fill_(which.unsqueeze(1), -1)
        self.lengths.masked_fill_(which, 0)


class PagedCache:
    """Keys and values of one layer, ``pages`` pages of ``page_size`` tokens each."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, device=None, dtype=torch.float16):
        device = torch.device("cuda" if device is None else device)
        self.k = torch.zeros(pages, page_size, kv_heads, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)

    def append(self, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, positions: Optional[torch.Tensor] = None,
               table: Optional[torch.Tensor] = None, sections: Optional[Sequence[int]] = None, interleaved: bool = False) -> Optional[torch.Tensor]:
        """Turns queries and keys, writes keys and values to ``slots``; the turned queries (``_C_ops.rotary_append``)."""
        return _C.rotary_append(q, k, v, self.k, self.v, slots, positions, table, sections=sections, interleaved=interleaved)

    def attention(self, q: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, scale: Optional[float] = None, window: int = 0,
                  rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of one token per row (``_C_ops.paged_attention``)."""
        return _C.paged_attention(q, self.k, self.v, block_table, lengths, scale=scale, window=window, rows=rows)


class _Plain(PagedCache):
    """The methods of ``PagedCache`` on another object's ``k`` and ``v``."""

    def __init__(self, cache):
        self.k, self.v = cache.k, cache.v


class QuantisedCache:
    """Keys and values of one layer in 4 bits: what ``PagedCache`` holds, in a good quarter of its room.

    Each token's head, or every ``group`` = 64 elements of one, has a scale and a zero of its own.  ``read(slots)`` gives tokens back in ``dtype``.  A page lies head by
    head, so that attention reads whole lines of memory."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, group: Optional[int] = None, device=None, dtype=torch.float16):
        if head_dim < 8 or head_dim % 8 or head_dim > 256:
            raise ValueError("head_dim must be a multiple of 8 up to 256")
        if group not in (None, head_dim) and (group != 64 or head_dim % 64):
            raise ValueError("group must be 64, of a head_dim that is a multiple of it, or the whole head")
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError("scales are float16 or bfloat16")
        device = torch.device("cuda" if device is None else device)
        groups = head_dim // (group or head_dim)
        self.k, self.v = (torch.zeros(pages, kv_heads, page_size, head_dim // 2, dtype=torch.uint8, device=device).transpose(1, 2) for _ in range(2))
        self.k_scales, self.v_scales = (torch.zeros(pages, kv_heads, page_size, groups, 2, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))

    def append(self, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, positions: Optional[torch.Tensor] = None,
               table: Optional[torch.Tensor] = None, sections: Optional[Sequence[int]] = None, interleaved: bool = False) -> Optional[torch.Tensor]:
        """Turns queries and keys, quantises keys and values as it writes them to ``slots``; the turned queries (``_C_ops.rotary_append_quantised``)."""
        return _C.rotary_append_quantised(q, k, v, self.k, self.v, self.k_scales, self.v_scales, slots, positions, table, sections=sections, interleaved=interleaved)

    def attention(self, q: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, scale: Optional[float] = None, window: int = 0,
                  rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of one token per row (``_C_ops.paged_attention_quantised``)."""
        return _C.paged_attention_quantised(q, self.k, self.v, self.k_scales, self.v_scales, block_table, lengths, scale=scale, window=window, rows=rows)

    def read(self, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [tokens, kv_heads, head_dim] of the tokens at ``slots`` (``_C_ops.read_quantised``)."""
        return _C.read_quantised(self.k, self.v, self.k_scales, self.v_scales, slots)


class PagedAttentionBlock(nn.Module):
    """The attention part of a decoder block for serving.

    ``qkv``: in_features -> (q_heads + 2 kv_heads) head_dim; ``proj``: q_heads head_dim -> in_features.  Either may have
    ``LowRankAdapters`` beside it, one adapter (or none, -1) per token in ``forward``'s ``ids``."""

    def __init__(self, qkv: OrthoLinear, proj: OrthoLinear, q_heads: int, kv_heads: int, table: torch.Tensor,
                 sections: Optional[Sequence[int]] = None, interleaved: bool = False, window: int = 0,
                 qkv_adapters: Optional[LowRankAdapters] = None, proj_adapters: Optional[LowRankAdapters] = None):
        super().__init__()
        if qkv.out_features % (q_heads + 2 * kv_heads):
            raise ValueError("qkv.out_features must be (q_heads + 2 kv_heads) heads")
        self.head_dim = qkv.out_features // (q_heads + 2 * kv_heads)
        if proj.in_features != q_heads * self.head_dim:
            raise ValueError("proj.in_features must be q_heads * head_dim")
        self.qkv, self.proj, self.q_heads, self.kv_heads = qkv, proj, q_heads, kv_heads
        self.qkv_adapters, self.proj_adapters = qkv_adapters, proj_adapters
        self.sections, self.interleaved, self.window = sections, interleaved, window
        self.register_buffer("table", table, persistent=False)

    def _apply(self, fn, recurse=True):
        table = self.table
        out = super()._apply(fn, recurse)
        if self.table.dtype != table.dtype:        # .half() and the like are for weights: angles of late positions do not fit 16 bits
            self.table = table.to(self.table.device)
        return out

    def forward(self, x: torch.Tensor, cache: Union[PagedCache, QuantisedCache], pool: PagePool, step: PageStep, ids: Optional[torch.Tensor] = None,
                positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``x`` [tokens, in_features]: the step's new tokens, request after request, as ``step`` lists them.
        ``positions``: rotary positions where they are not those in the request, [tokens] or [axes, tokens].  Every token sees its
        request up to itself and reads its keys for itself: meant for decoding and short prompts.  A ``cache`` of another kind is asked for ``append`` and
        ``attention``; one that only has tensors ``k`` and ``v`` is taken as a ``PagedCache``'s.  Places behind the step's
        last token give what an empty attention gives."""
        T, D = x.shape[0], self.head_dim
        qkv = self.qkv(x)
        if self.qkv_adapters is not None and ids is not None:
            qkv = self.qkv_adapters(x, qkv, ids, out=qkv)
        heads = qkv.view(T, self.q_heads + 2 * self.kv_heads, D)
        q, k, v = heads.split((self.q_heads, self.kv_heads, self.kv_heads), dim=1)
        kind = cache if hasattr(cache, "append") and hasattr(cache, "attention") else _Plain(cache)
        q = kind.append(q, k, v, step.slots, step.positions if positions is None else positions, self.table,
                        sections=self.sections, interleaved=self.interleaved)
        o = kind.attention(q, pool.block_table, step.positions + 1, window=self.window, rows=step.requests)
        o = o.view(T, self.q_heads * D)
        y = self.proj(o)
        if self.proj_adapters is not None and ids is not None:
            y = self.proj_adapters(o, y, ids, out=y)
        return y
