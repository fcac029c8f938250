"""Penalties, biases and grammar masks on the logits of a decode step.

For a row (one request) with history h, of which the first `prompt_lengths`
tokens are the prompt and the rest was generated:

    seen  = v stands in h;  count = times v stands in the generated part
    z1 = seen ? (z > 0 ? z / repetition : z * repetition) : z
    z2 = z1 - frequency * count - presence * (count > 0)
    z3 = z2 + the sum of the row's biases for v
    out = allowed ? z3 : -inf

computed in fp32 and rounded once to the logits' type, in one launch
(csrc/logits.hip) that keeps nothing between steps: a request may join,
leave, or be rewound by handing in another history.  bf16, fp16 and fp32 run
the kernel on the GPU, the CPU and fp64 the reference below.
"""
from __future__ import annotations

import dataclasses
import math
from typing import Callable, Dict, List, Optional, Sequence, Union

import torch

from . import extension
from .functional import _acc_dtype

PerRow = Union[float, torch.Tensor, None]


def pack_allowed(allowed: torch.Tensor) -> torch.Tensor:
    """(B, V) truth values -> (B, ceil(V / 32)) int32: token v is bit v % 32
    of word v // 32."""
    if allowed.dim() != 2 or allowed.dtype != torch.bool:
        raise ValueError("allowed must be (B, V) bool")
    B, V = allowed.shape
    pad = torch.nn.functional.pad(allowed, (0, -V % 32)).view(B, -1, 32)
    bit = 1 << torch.arange(32, device=allowed.device)
    word = (pad.long() * bit).sum(dim=2)
    return torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)


def _ref_adjust(logits, history, lengths, prompt_lengths, repetition,
                presence, frequency, bias_index, bias, allowed):
    B, V = logits.shape
    dev = logits.device
    z = logits.to(_acc_dtype(logits.dtype))

    def column(x):
        return x.to(z.dtype)[:, None] if isinstance(x, torch.Tensor) else x

    if history is not None:
        h = history.long()
        at = torch.arange(h.shape[1], device=dev)
        n = h.new_full((B,), h.shape[1]) if lengths is None else lengths
        p = h.new_zeros(B) if prompt_lengths is None else prompt_lengths
        inside = (at < n[:, None]) & (h >= 0) & (h < V)
        h = torch.where(inside, h, 0)
        zero = torch.zeros(B, V, dtype=torch.long, device=dev)
        seen = zero.scatter_add(1, h, inside.long()) > 0
        count = zero.scatter_add(1, h, (inside & (at >= p[:, None])).long())
        rho = column(repetition)
        z = torch.where(seen, torch.where(z > 0, z / rho, z * rho), z)
        z = torch.where(count > 0, z - column(frequency) * count
                        - column(presence), z)
    if bias_index is not None:
        i = bias_index.long()
        inside = (i >= 0) & (i < V)
        z = z + torch.zeros_like(z).scatter_add(
            1, torch.where(inside, i, 0),
            torch.where(inside, bias.to(z.dtype), 0.0))
    if allowed is not None:
        v = torch.arange(V, device=dev)
        bit = (allowed[:, v // 32] >> (v % 32).to(torch.int32)) & 1
        z = z.masked_fill(bit == 0, -math.inf)
    return z.to(logits.dtype)


def _check(logits, history, lengths, prompt_lengths, per_row, bias_index,
           bias, allowed):
    """What the kernel's path refuses in csrc/lm_ops.cpp."""
    if logits.dim() != 2 or not logits.dtype.is_floating_point:
        raise ValueError(
            f"logits must be (B, V) floating, got {tuple(logits.shape)}")
    B, V = logits.shape
    index = (torch.int32, torch.int64)
    if history is not None and (
            history.dim() != 2 or history.shape[0] != B
            or history.dtype not in index):
        raise ValueError(f"history must be (B={B}, L) int32 or int64")
    for t, name in ((lengths, "lengths"), (prompt_lengths, "prompt_lengths")):
        if t is not None and (t.shape != (B,) or t.dtype not in index):
            raise ValueError(f"{name} must be (B={B},) int32 or int64")
    for t in per_row:
        if t is not None and (t.shape != (B,)
                              or not t.dtype.is_floating_point):
            raise ValueError(
                f"penalties must be numbers or (B={B},) floating")
    if bias is not None and (
            bias_index.dim() != 2 or bias_index.shape[0] != B
            or bias.shape != bias_index.shape
            or bias_index.dtype not in index
            or not bias.dtype.is_floating_point):
        raise ValueError(f"bias_index must be (B={B}, K) int32 or int64 and "
                         "bias floating of the same shape")
    if allowed is not None and (allowed.dtype != torch.int32 or allowed.shape
                                != (B, (V + 31) // 32)):
        raise ValueError(f"allowed must be (B={B}, {(V + 31) // 32}) int32")
    for t in (history, lengths, prompt_lengths, *per_row, bias_index, bias,
              allowed):
        if t is not None and t.device != logits.device:
            raise ValueError(f"all tensors must be on {logits.device}")


def _per_row(x: PerRow, none: float, name: str):
    """-> (tensor or None, number used without one)."""
    if x is None:
        return None, none
    if isinstance(x, torch.Tensor):
        return x, none
    x = float(x)
    if not math.isfinite(x):
        raise ValueError(f"{name} must be finite, got {x}")
    return None, x


def adjust_logits(logits: torch.Tensor,
                  history: Optional[torch.Tensor] = None,
                  lengths: Optional[torch.Tensor] = None,
                  prompt_lengths: Optional[torch.Tensor] = None, *,
                  repetition: PerRow = None, presence: PerRow = None,
                  frequency: PerRow = None,
                  bias_index: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None,
                  allowed: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Adjusted logits, a new (B, V) tensor of the logits' type.

    logits: (B, V), rows of any stride.
    history: (B, L) int32 / int64 tokens; row b counts its first lengths[b]
    (all L without `lengths`, never more than L) and takes the first
    prompt_lengths[b] of them as prompt (none without).  Tokens outside
    [0, V) are no tokens.
    repetition (> 0, 1 changes nothing), presence, frequency: a number for
    all rows or a floating (B,) tensor; they need a history.
    bias_index, bias: (B, K) tokens and what is added to them; an index
    outside [0, V) is none, the same index twice adds both.
    allowed: (B, ceil(V / 32)) int32 as `pack_allowed` makes it.  A row that
    allows nothing comes back as -inf throughout; a masked NaN is -inf.
    Not differentiable: this is the serving path.  The kernel refuses tensors
    that carry a forward-mode tangent.
    """
    if history is None:
        if not (lengths is prompt_lengths is repetition is presence
                is frequency is None):
            raise ValueError("penalties and lengths need a history")
    if (bias_index is None) != (bias is None):
        raise ValueError("bias_index and bias come together")
    rep, rep_all = _per_row(repetition, 1.0, "repetition")
    if rep_all <= 0.0:
        raise ValueError(f"repetition must be positive, got {rep_all}")
    pres, pres_all = _per_row(presence, 0.0, "presence")
    freq, freq_all = _per_row(frequency, 0.0, "frequency")
    if extension.use_hip_lm(logits):
        return extension.get_extension().adjust_logits(
            logits, history, lengths, prompt_lengths, rep, rep_all, pres,
            pres_all, freq, freq_all, bias_index, bias, allowed)
    _check(logits, history, lengths, prompt_lengths, (rep, pres, freq),
           bias_index, bias, allowed)
    with torch.no_grad():
        return _ref_adjust(logits, history, lengths, prompt_lengths,
                           rep_all if rep is None else rep,
                           pres_all if pres is None else pres,
                           freq_all if freq is None else freq, bias_index,
                           bias, allowed)


@dataclasses.dataclass
class LogitRules:
    """What one request wants done to its logits before a token is chosen.

    bias: token -> what is added to its logit.
    grammar: called with the request's tokens so far (prompt included) before
    every token; returns the tokens that may follow as a (V,) bool tensor, on
    any device.
    """
    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    bias: Optional[Dict[int, float]] = None
    grammar: Optional[Callable[[List[int]], torch.Tensor]] = None

    def check(self, vocab_size: int):
        """Refuses what could leave a row without a finite logit to sample
        from: the limits keep every adjusted logit finite in bf16 and fp32
        (fp16's range ends at seven repeats; RowRules adjusts in fp32)."""
        if not 0.01 <= self.repetition <= 100.0:
            raise ValueError("repetition must be in [0.01, 100], got "
                             f"{self.repetition}")
        for x in (self.presence, self.frequency):
            if not abs(x) <= 1e4:
                raise ValueError(f"penalties must be in [-1e4, 1e4], got {x}")
        bias = self.bias or {}
        if any(not hasattr(t, "__index__") or t < 0 or t >= vocab_size
               for t in bias):
            raise ValueError("bias tokens must be whole numbers in "
                             f"[0, {vocab_size})")
        if not all(f == -math.inf or abs(f) <= 1e4 for f in bias.values()):
            raise ValueError("a bias must be in [-1e4, 1e4] or -inf")
        if sum(f == -math.inf for f in bias.values()) == vocab_size:
            raise ValueError("the biases rule out every token")

    @property
    def penalizes(self) -> bool:
        return (self.repetition != 1.0 or self.presence != 0.0
                or self.frequency != 0.0)

    def allows(self, tokens: List[int], vocab_size: int) -> torch.Tensor:
        """The grammar's answer as a (V,) bool tensor, with a token in it
        that no bias rules out."""
        ok = self.grammar(tokens)
        if (not isinstance(ok, torch.Tensor) or ok.dtype != torch.bool
                or ok.shape != (vocab_size,)):
            raise ValueError(f"a grammar returns a ({vocab_size},) bool tensor")
        # a copy: the grammar may fill the same tensor for the next row
        ok = ok.clone()
        banned = [t for t, f in (self.bias or {}).items() if f == -math.inf]
        if banned:
            ok[banned] = False
        if not bool(ok.any()):
            raise ValueError(f"the grammar allows no token after {len(tokens)}")
        return ok


class RowRules:
    """The rules (or None) of a batch's rows, for as long as the batch stays
    the same: what does not change from token to token is uploaded once."""

    def __init__(self, rules: Sequence[Optional[LogitRules]],
                 prompt_lengths: Sequence[int], vocab_size: int, device):
        self.rules = [r or LogitRules() for r in rules]
        self.vocab_size, self.device = vocab_size, device
        self.penalizes = any(r.penalizes for r in self.rules)
        self.constant: dict = {}
        if self.penalizes:
            number = torch.tensor(
                [[getattr(r, n) for r in self.rules]
                 for n in ("repetition", "presence", "frequency")],
                dtype=torch.float32).to(device)
            self.constant.update(
                repetition=number[0], presence=number[1], frequency=number[2],
                prompt_lengths=torch.tensor(list(prompt_lengths)).to(device))
        K = max(len(r.bias or ()) for r in self.rules)
        if K:
            pairs = [list((r.bias or {}).items()) for r in self.rules]
            pairs = [p + [(-1, 0.0)] * (K - len(p)) for p in pairs]
            self.constant["bias_index"] = torch.tensor(
                [[t for t, _ in p] for p in pairs]).to(device)
            self.constant["bias"] = torch.tensor(
                [[f for _, f in p] for p in pairs],
                dtype=torch.float32).to(device)

    def apply(self, logits: torch.Tensor, history: Optional[torch.Tensor],
              lengths: Optional[torch.Tensor],
              allowed: Sequence[Optional[torch.Tensor]] = ()) -> torch.Tensor:
        """`adjust_logits` on the rows' (B, V) logits, fp16 ones as fp32.
        history (B, L) and lengths (B,) are needed where a row penalizes;
        allowed: what the grammars (LogitRules.allows) said for each row, None
        without one."""
        args = dict(self.constant)
        if self.penalizes:
            args.update(history=history, lengths=lengths)
        if any(ok is not None for ok in allowed):
            every = torch.ones(self.vocab_size, dtype=torch.bool)
            args["allowed"] = pack_allowed(torch.stack(
                [(every if ok is None else ok).to(self.device)
                 for ok in allowed]))
        if not args:
            return logits
        if logits.dtype == torch.float16:
            logits = logits.float()
        return adjust_logits(logits, **args)
