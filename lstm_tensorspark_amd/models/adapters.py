"""Low-rank adapters of an LSTMModel: a set of fine-tunings that share one
frozen base, one of them (or none) for every sequence of a batch.

An adapter covers every layer's input projection W_x and the head; the
recurrent W_h stays the base's (it runs inside the sequence kernels).  Names
follow the model's flat weight dict: layer{i}/A, layer{i}/B, head/A, head/B.

    adapters = AdapterSet(model.cfg, rank=16, count=3).to(device, dtype)
    out, state = model(x, state, adapters=adapters.rows([0, 2, -1, 0]))
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Union

import torch
import torch.nn as nn

from ..config import ModelConfig
from ..ops.adapters import (MAX_RANK, AdapterRows, lowrank_add, lowrank_add_)


class AdapterSet(nn.Module):
    """`count` adapters of rank `rank`; a new one changes nothing (B = 0).
    alpha / rank scales what an adapter adds (alpha = rank by default)."""

    def __init__(self, cfg: ModelConfig, rank: int, count: int = 1,
                 alpha: Optional[float] = None):
        super().__init__()
        if not 1 <= rank <= MAX_RANK:
            raise ValueError(f"rank must be in [1, {MAX_RANK}], got {rank}")
        if count < 1:
            raise ValueError(f"count must be positive, got {count}")
        self.rank, self.count = rank, count
        self.scale = (rank if alpha is None else alpha) / rank
        self._params: dict[str, nn.Parameter] = {}
        H, D = cfg.hidden_size, cfg.num_directions
        for l in range(cfg.num_layers):
            for rev in ("", "_rev") if cfg.bidirectional else ("",):
                self._site(f"layer{l}{rev}",
                           cfg.input_size if l == 0 else H * D, 4 * H)
        if cfg.head != "none":
            self._site("head", H * D, cfg.vocab_size if cfg.head == "lm"
                       else cfg.num_classes)

    def _site(self, name: str, k: int, m: int):
        bound = 1.0 / math.sqrt(k)
        for part, t in (
                ("A", torch.empty(self.count, k, self.rank)
                 .uniform_(-bound, bound)),
                ("B", torch.zeros(self.count, self.rank, m))):
            p = nn.Parameter(t)
            self.register_parameter(f"{name}__{part}", p)
            self._params[f"{name}/{part}"] = p

    def weight_dict(self) -> dict[str, nn.Parameter]:
        """Flat named weights, as LSTMModel.weight_dict."""
        return {n: self.get_parameter(n.replace("/", "__"))
                for n in self._params}

    def rows(self, index: Union[Sequence[int], torch.Tensor]) -> "AdapterBatch":
        """The adapters of a batch's columns: one in [0, count) or -1 (the
        base alone) for each."""
        dev = next(self.parameters()).device
        return AdapterBatch(self, AdapterRows(index, self.count, device=dev))


class AdapterBatch:
    """An AdapterSet bound to the columns of one batch."""

    def __init__(self, adapters: AdapterSet, rows: AdapterRows):
        self.adapters, self.rows = adapters, rows

    def add(self, y: torch.Tensor, x: torch.Tensor, site: str) -> torch.Tensor:
        """y plus what the site's adapters make of x.  Without gradients y,
        which the caller has just computed, is updated in place."""
        a = self.adapters.get_parameter(site + "__A")
        b = self.adapters.get_parameter(site + "__B")
        f = lowrank_add if torch.is_grad_enabled() else lowrank_add_
        return f(y, x, a, b, self.rows, self.adapters.scale)
