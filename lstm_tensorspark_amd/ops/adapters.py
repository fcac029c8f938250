"""Low-rank adapters of many requests at once beside a shared projection.

    out_i = y_i + s_l (x_i @ A_l) @ B_l          l = the adapter of row i

y is what the shared projection made of x (y = x @ W + b), A_l (K, R) and
B_l (R, M) are one tenant's or one task's fine-tuning of W, and rows of one
batch may belong to different adapters, or to none.

The engine is time-major, (T, B, .), and an adapter belongs to a sequence:
`AdapterRows` groups the B columns of a batch by adapter once, on the host,
and serves every projection of every step until the batch changes.

bf16 and fp16 run the kernels of csrc/adapters.hip on the GPU (fp32
throughout, x @ A included; the result is rounded once); the CPU, fp32 and
fp64 run the reference below, as the LSTM layers do.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Union

import torch

from . import extension
from .functional import _acc_dtype

MAX_RANK = 128


class AdapterRows:
    """The B columns of a batch, grouped by adapter.

    index: an adapter in [0, num_adapters) or -1 (none) for each column; a
    host list, or a tensor (a GPU tensor is copied to the host).  The
    grouping is fixed: a captured graph replays with the rows it was
    captured with, which have to live as long as the graph.
    """

    def __init__(self, index: Union[Sequence[int], torch.Tensor],
                 num_adapters: int, device=None):
        if isinstance(index, torch.Tensor):
            if index.dim() != 1 or index.dtype not in (torch.int32,
                                                       torch.int64):
                raise ValueError("index must be (B,) int32 or int64")
            device = index.device if device is None else device
            index = index.tolist()
        index = [int(i) for i in index]
        if not index:
            raise ValueError("index names no column")
        if num_adapters < 1 or any(i < -1 or i >= num_adapters
                                   for i in index):
            raise ValueError(f"adapters must be in [-1, {num_adapters})")
        self.index = tuple(index)
        self.num_adapters = num_adapters
        self.device = torch.device("cpu" if device is None else device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        # stable: a group of every column keeps their order
        order = sorted(range(len(index)), key=index.__getitem__)
        groups: dict[int, int] = {}
        for i in order:
            groups[index[i]] = groups.get(index[i], 0) + 1
        self.counts = list(groups.values())
        self.groups = len(groups) - (-1 in groups)  # adapters with rows
        segs, start = [], 0
        for adapter, count in groups.items():
            segs += [adapter, start, count, 0]
            start += count
        n = len(index)
        # one upload: segments first (16-byte entries), then the two lists
        flat = torch.tensor(segs + order + index, dtype=torch.int32)
        flat = flat.to(self.device)
        self.segs = flat[:len(segs)]
        self.order = flat[len(segs):len(segs) + n]
        self.adapter = flat[len(segs) + n:]

    def __len__(self) -> int:
        return len(self.index)


def _ref_lowrank(y, x, a, b, rows: AdapterRows, scale):
    """Plain-torch semantics (CPU path and test oracle); autograd gives its
    gradients."""
    acc = _acc_dtype(x.dtype)
    out = y.to(acc)
    at = {}
    for column, l in enumerate(rows.index):
        if l >= 0:
            at.setdefault(l, []).append(column)
    for l, columns in at.items():
        c = torch.tensor(columns, device=x.device)
        s = scale[l].to(acc) if isinstance(scale, torch.Tensor) else scale
        v = x.index_select(-2, c).to(acc) @ a[l].to(acc)
        out = out.index_add(out.dim() - 2, c, (s * v) @ b[l].to(acc))
    return out.to(y.dtype)


def _check(y, x, a, b, rows, scale):
    """What the kernels' path refuses in csrc/lm_ops.cpp."""
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] \
            or a.shape[2] != b.shape[1]:
        raise ValueError("a must be (L, K, R) and b (L, R, M), got "
                         f"{tuple(a.shape)}, {tuple(b.shape)}")
    L, K, R = a.shape
    if not 1 <= R <= MAX_RANK:
        raise ValueError(f"rank must be in [1, {MAX_RANK}], got {R}")
    if x.dim() < 2 or x.shape[:-1] != y.shape[:-1] or x.shape[-1] != K \
            or y.shape[-1] != b.shape[2]:
        raise ValueError(
            f"x must be (..., B, {K}) and y (..., B, {b.shape[2]}), got "
            f"{tuple(x.shape)}, {tuple(y.shape)}")
    if not isinstance(rows, AdapterRows) or len(rows) != x.shape[-2] \
            or rows.num_adapters != L:
        raise ValueError(f"rows must be AdapterRows of {x.shape[-2]} columns "
                         f"and {L} adapters")
    if not x.dtype.is_floating_point or any(
            t.dtype != x.dtype for t in (y, a, b)):
        raise ValueError("y, x, a and b must have one floating type")
    dev = x.device
    if isinstance(scale, torch.Tensor):
        if scale.shape != (L,) or not scale.dtype.is_floating_point:
            raise ValueError(f"scale must be a number or (L={L},) floating")
        if scale.requires_grad:
            raise ValueError("scale gets no gradient: detach it")
    elif not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    for t in (y, a, b, scale if isinstance(scale, torch.Tensor) else x):
        if t.device != dev:
            raise ValueError(f"all tensors must be on {dev}")
    if rows.device != dev:
        raise ValueError(f"rows are on {rows.device}, the tensors on {dev}")


def _kernels(y, x) -> bool:
    return extension.use_hip_lm(x) and x.dtype != torch.float32 \
        and x.numel() > 0 and y.numel() > 0


def _launch(y, x, a, b, rows, scale, inplace: bool):
    if not isinstance(rows, AdapterRows):
        raise ValueError("rows must be AdapterRows")
    each = None
    if isinstance(scale, torch.Tensor):
        each, scale = scale, 1.0
    elif not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    return extension.get_extension().lowrank_add(
        y, x, a, b, rows.order, rows.segs, rows.adapter, rows.counts,
        rows.groups, each, float(scale), inplace, rows.num_adapters)


def lowrank_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor,
                b: torch.Tensor, rows: AdapterRows,
                scale: Union[float, torch.Tensor] = 1.0) -> torch.Tensor:
    """y + scale * (x @ a[l]) @ b[l] with l the adapter of each row's column;
    rows without an adapter are y's.  Differentiable in y, x, a and b, once and
    backward: the kernels refuse a tensor that carries a forward-mode tangent.

    y (..., B, M), x (..., B, K); a (L, K, R), b (L, R, M), R <= 128; rows of
    the B columns; scale a number or one for each adapter (L,), a constant.
    """
    if _kernels(y, x):
        return _launch(y, x, a, b, rows, scale, False)
    _check(y, x, a, b, rows, scale)
    return _ref_lowrank(y, x, a, b, rows, scale)


def lowrank_add_(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor,
                 b: torch.Tensor, rows: AdapterRows,
                 scale: Union[float, torch.Tensor] = 1.0) -> torch.Tensor:
    """`lowrank_add` into a contiguous y itself, the serving form: rows
    without an adapter are not touched.  No gradient."""
    if _kernels(y, x):
        _launch(y, x, a, b, rows, scale, True)
        return y
    _check(y, x, a, b, rows, scale)
    if not y.is_contiguous():
        raise ValueError("y must be contiguous")
    with torch.no_grad():
        return y.copy_(_ref_lowrank(y, x, a, b, rows, scale))
