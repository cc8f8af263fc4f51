"""Low-rank adapters of many requests beside one projection.

The reference leaves adapter matrices alone when it rewrites a model's weights
(``experiments/complete_real_model_experiments.py:269-327``); here they run beside the packed projection, a different
adapter for every token of a batch if need be.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import _C_ops as _C


class LowRankAdapters(nn.Module):
    """``count`` adapters of rank up to ``max_rank`` beside a projection ``in_features -> out_features``.

    ``load(i, down, up, scale)`` places one (``down`` [rank, in_features], ``up`` [out_features, rank]); an adapter that
    was never loaded, or was removed, adds nothing.  ``forward(x, y, ids)`` returns ``y + scale * up (down x)`` per token, in one pass over the batch whatever
    mix of adapters it holds; ``out=y`` adds in place."""

    def __init__(self, count: int, in_features: int, out_features: int, max_rank: int, device=None, dtype=torch.float16):
        super().__init__()
        if count < 1 or in_features < 8 or in_features % 8 or out_features < 1 or not 1 <= max_rank <= 256:
            raise ValueError("need at least one adapter, in_features a multiple of 8 and a rank of 1 to 256")
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError("adapters are float16 or bfloat16")
        self.count, self.in_features, self.out_features, self.max_rank = count, in_features, out_features, max_rank
        room = (max_rank + 7) // 8 * 8             # whole 16-byte rows of `up`; what a rank leaves over is zero
        self.register_buffer("down", torch.zeros(count, room, in_features, dtype=dtype, device=device))
        self.register_buffer("up", torch.zeros(count, out_features, room, dtype=dtype, device=device))
        self.register_buffer("scales", torch.zeros(count, dtype=torch.float32, device=device))
        self.register_buffer("ranks", torch.zeros(count, dtype=torch.int32, device=device))

    @torch.no_grad()
    def load(self, index: int, down: torch.Tensor, up: torch.Tensor, scale: float = 1.0) -> None:
        rank = down.shape[0]
        if not 0 <= index < self.count:
            raise IndexError(f"adapter {index} of {self.count}")
        if (tuple(down.shape) != (rank, self.in_features) or tuple(up.shape) != (self.out_features, rank)
                or not 1 <= rank <= self.max_rank):
            raise ValueError("down must be [rank, in_features] and up [out_features, rank], of a rank up to max_rank")
        self.down[index].zero_()
        self.up[index].zero_()
        self.down[index, :rank].copy_(down)
        self.up[index, :, :rank].copy_(up)
        self.scales[index].fill_(scale)
        self.ranks[index].fill_(rank)

    @torch.no_grad()
    def remove(self, index: int) -> None:
        if not 0 <= index < self.count:
            raise IndexError(f"adapter {index} of {self.count}")
        self.ranks[index].zero_()
        self.scales[index].zero_()

    def _apply(self, fn, recurse=True):
        scales = self.scales
        out = super()._apply(fn, recurse)
        if self.scales.dtype != torch.float32:     # .half() and the like are for the matrices
            self.scales = scales.to(self.scales.device)
        return out

    def forward(self, x: torch.Tensor, y: torch.Tensor, ids: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        return _C.low_rank_add(x, y, self.down, self.up, ids, scales=self.scales, ranks=self.ranks, out=out)

    def extra_repr(self) -> str:
        return f"count={self.count}, in_features={self.in_features}, out_features={self.out_features}, max_rank={self.max_rank}"
