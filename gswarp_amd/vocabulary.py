"""Vocabulary operators: what Gaussians and pixels that hold tokens are trained with.

A scene whose Gaussians carry more than a colour keeps it in a learned table shared by all of them:
a codebook of attributes, or of language features.  Each Gaussian holds a token, its features are a
row of the table (:func:`embed_tokens`), they are rasterized, and a pixel's rendered feature is
scored against every row of a vocabulary (:func:`linear_cross_entropy`).  Both give the gradient of
the table; with one table at both ends (:class:`Vocabulary`) the two are added by autograd.

Tables and features are float32, bfloat16 or float16 on a ROCm device; sums are held in 32 bits or
more whatever the type is and rounded once.  Work is enqueued on the current stream, nothing is read
back, and results do not change from run to run.
"""

from __future__ import annotations

import functools
import math

import torch
import torch.nn as nn

from . import _lib, _workspace
from ._pipeline import _device_guard, _stream

_DTYPES = {torch.float32: _lib.GS_FP32, torch.bfloat16: _lib.GS_BF16, torch.float16: _lib.GS_FP16}
_INDEX_BITS = {torch.int32: 32, torch.int64: 64}
_REDUCTIONS = {"none": _lib.GS_REDUCE_NONE, "sum": _lib.GS_REDUCE_SUM, "mean": _lib.GS_REDUCE_MEAN}
_INT32_MAX = 2**31 - 1
_MAX_DIM = 2**21 - 8
_MAX_CLASSES = 2**29
_FP32_MAX = torch.finfo(torch.float32).max


def _check_table(table, name: str, most: int = _INT32_MAX) -> None:
    if isinstance(table, torch.Tensor) and table.is_cuda and table.dtype in _DTYPES and table.ndim == 2:
        vocab, dim = table.shape
        if 0 < vocab <= most and 0 < dim <= _MAX_DIM:
            return
    if not isinstance(table, torch.Tensor) or not table.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if table.dtype not in _DTYPES:
        raise ValueError(f"{name} must have dtype float32, bfloat16 or float16, got {table.dtype}")
    if table.ndim != 2 or table.shape[0] == 0 or table.shape[1] == 0:
        raise ValueError(f"{name} must have shape (vocabulary, dim), got {tuple(table.shape)}")
    raise ValueError(f"{name} must have at most {most} rows of at most {_MAX_DIM} values")


def _check_indices(indices, name: str, device: torch.device) -> None:
    if (isinstance(indices, torch.Tensor) and indices.dtype in _INDEX_BITS and indices.device == device
            and indices.numel() <= _INT32_MAX):
        return
    if not isinstance(indices, torch.Tensor):
        raise ValueError(f"{name} must be a torch.Tensor")
    if indices.device != device:
        raise ValueError(f"{name} must be on {device}, got {indices.device}")
    if indices.dtype not in _INDEX_BITS:
        raise ValueError(f"{name} must have dtype int32 or int64, got {indices.dtype}")
    raise ValueError(f"{name} must have at most 2**31 - 1 elements")


def _check_factor(value, name: str) -> float:
    value = float(value)
    if not -_FP32_MAX <= value <= _FP32_MAX:
        raise ValueError(f"{name} must be finite in float32")
    return value


def _rows(t: torch.Tensor, alignment: int = 1) -> torch.Tensor:
    """The matrix, or a copy of it, with contiguous rows that do not overlap, on `alignment` bytes."""
    if t.is_contiguous():
        if t.data_ptr() % alignment == 0:
            return t
    elif (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() % alignment else t


def _row_stride(t: torch.Tensor) -> int:
    if t.is_contiguous():
        return t.shape[1]
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


def _workspace_of(nbytes: int, device: torch.device) -> torch.Tensor:
    return torch.empty(nbytes + 255, dtype=torch.uint8, device=device)


def _aligned(space: torch.Tensor) -> int:
    return (space.data_ptr() + 255) & ~255


# Workspace sizes are functions of the sizes alone; a training loop asks for the same ones again.
@functools.lru_cache(maxsize=256)
def _embed_bwd_bytes(n, vocab, dim, code) -> int:
    return _lib.load().gs_embed_bwd_workspace_bytes(n, vocab, dim, code)


@functools.lru_cache(maxsize=256)
def _entropy_fwd_bytes(n, vocab, dim, code, ldf, ldt) -> tuple[int, int]:
    """(workspace, state)"""
    lib = _lib.load()
    return (lib.gs_xent_fwd_workspace_bytes(n, vocab, dim, code, ldf, ldt),
            lib.gs_xent_state_bytes(n, vocab, dim, code, ldf, ldt))


@functools.lru_cache(maxsize=256)
def _entropy_bwd_bytes(n, vocab, dim, code, ldf, ldt, want_features, want_table) -> int:
    return _lib.load().gs_xent_bwd_workspace_bytes(n, vocab, dim, code, ldf, ldt, want_features, want_table)


# ---------------------------------------------------------------- lookup

def _embed_forward(tokens, table, scale):
    device, (vocab, dim) = table.device, table.shape
    lib = _lib.load()
    tokens, rows = tokens.contiguous(), _rows(table)
    out = torch.empty((*tokens.shape, dim), dtype=table.dtype, device=device)
    with _device_guard(device), _workspace.device_lock(device):
        lib.call("gs_embed_fwd", tokens.numel(), vocab, dim, _DTYPES[table.dtype], tokens.data_ptr(),
                 _INDEX_BITS[tokens.dtype], rows.data_ptr(), _row_stride(rows), scale, out.data_ptr(), _stream(device))
    return out


class EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, scale, padding_idx):
        ctx.save_for_backward(tokens)
        ctx.table_shape, ctx.table_dtype = tuple(table.shape), table.dtype
        ctx.scale, ctx.padding_idx = scale, padding_idx
        return _embed_forward(tokens, table, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        (tokens,) = ctx.saved_tensors
        (vocab, dim), dtype, device = ctx.table_shape, ctx.table_dtype, grad_out.device
        lib = _lib.load()
        tokens, grad_out = tokens.contiguous(), grad_out.contiguous()
        grad = torch.empty((vocab, dim), dtype=dtype, device=device)
        n, code = tokens.numel(), _DTYPES[dtype]
        nbytes = _embed_bwd_bytes(n, vocab, dim, code)
        space = _workspace_of(nbytes, device)
        with _device_guard(device), _workspace.device_lock(device):
            lib.call("gs_embed_bwd", n, vocab, dim, code, tokens.data_ptr(), _INDEX_BITS[tokens.dtype],
                     grad_out.data_ptr(), ctx.scale, -1 if ctx.padding_idx is None else ctx.padding_idx,
                     grad.data_ptr(), _aligned(space), nbytes, _stream(device))
        return None, grad, None, None


def embed_tokens(tokens: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0,
                 padding_idx: int | None = None) -> torch.Tensor:
    """``scale * table[tokens]``: (..., dim) for tokens of shape (...), in the table's dtype.

    tokens: int32 or int64, any shape, on the table's device; a token outside the table reads
    nothing and gives a row of NaN.  table: (vocabulary, dim), any strides.  The gradient of row v is
    ``scale`` times the sum of the gradients at its positions, in a fixed order; the positions of
    ``padding_idx`` bring none.
    """
    _check_table(table, "table")
    _check_indices(tokens, "tokens", table.device)
    scale = _check_factor(scale, "scale")
    if padding_idx is not None and not (isinstance(padding_idx, int) and 0 <= padding_idx < table.shape[0]):
        raise ValueError(f"padding_idx must be a row of the table, got {padding_idx!r}")
    if table.requires_grad and torch.is_grad_enabled():
        return EmbedTokens.apply(tokens, table, scale, padding_idx)
    return _embed_forward(tokens, table, scale)


# ---------------------------------------------------------------- cross entropy

def _entropy_forward(features, table, targets, ignore_index, reduction, logit_scale, keep: bool):
    """(loss, what the backward needs or None) for 2-D features and 1-D targets."""
    device, n, (vocab, dim) = table.device, features.shape[0], table.shape
    lib = _lib.load()
    code, ldf, ldt = _DTYPES[table.dtype], _row_stride(features), _row_stride(table)
    loss = torch.empty((n,) if reduction == "none" else (), dtype=torch.float32, device=device)
    # the count of rows sits in front of the workspace, or of the state
    nbytes, state_bytes = _entropy_fwd_bytes(n, vocab, dim, code, ldf, ldt)
    space = _workspace_of(256 + nbytes, device)
    state = _workspace_of(256 + state_bytes, device) if keep else None
    count = _aligned(state if keep else space)
    with _device_guard(device), _workspace.device_lock(device):
        lib.call("gs_xent_fwd", n, vocab, dim, code, features.data_ptr(), ldf, table.data_ptr(), ldt,
                 targets.data_ptr(), _INDEX_BITS[targets.dtype], ignore_index, logit_scale, _REDUCTIONS[reduction],
                 loss.data_ptr(), count + 256 if keep else None, count, _aligned(space) + 256, nbytes, _stream(device))
    return loss, state


class LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, features, table, targets, ignore_index, reduction, logit_scale):
        loss, state = _entropy_forward(features, table, targets, ignore_index, reduction, logit_scale, True)
        ctx.save_for_backward(features, table, targets, state)
        ctx.options = (ignore_index, reduction, logit_scale)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        features, table, targets, state = ctx.saved_tensors
        ignore_index, reduction, logit_scale = ctx.options
        want_features, want_table = ctx.needs_input_grad[:2]
        device, n, (vocab, dim) = table.device, features.shape[0], table.shape
        lib = _lib.load()
        code, ldf, ldt = _DTYPES[table.dtype], _row_stride(features), _row_stride(table)
        grad_loss = grad_loss.contiguous()
        grad_features = torch.empty((n, dim), dtype=table.dtype, device=device) if want_features else None
        grad_table = torch.empty((vocab, dim), dtype=table.dtype, device=device) if want_table else None
        nbytes = _entropy_bwd_bytes(n, vocab, dim, code, ldf, ldt, want_features, want_table)
        space = _workspace_of(nbytes, device)
        count = _aligned(state)
        with _device_guard(device), _workspace.device_lock(device):
            lib.call("gs_xent_bwd", n, vocab, dim, code, features.data_ptr(), ldf, table.data_ptr(), ldt,
                     targets.data_ptr(), _INDEX_BITS[targets.dtype], ignore_index, logit_scale, _REDUCTIONS[reduction],
                     count + 256, count, grad_loss.data_ptr(), _lib.ptr(grad_features), _lib.ptr(grad_table),
                     _aligned(space), nbytes, _stream(device))
        return grad_features, grad_table, None, None, None, None


def linear_cross_entropy(features: torch.Tensor, table: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100, reduction: str = "mean",
                         logit_scale: float = 1.0) -> torch.Tensor:
    """Softmax cross entropy of ``logit_scale * features @ table.T`` against ``targets``.

    features: (..., dim); table: (vocabulary, dim) of the same dtype, any strides; targets: int32 or
    int64 of shape (...).  The logits are never kept: neither their matrix nor its gradient exists
    beyond a piece.  float32 loss: of shape (...) for ``reduction="none"``, else the ``"sum"`` or the
    ``"mean"`` over the rows that count (NaN over none).  Rows whose target is ``ignore_index`` do not
    count: their loss and gradient are zero and they bring nothing to the table's gradient, whatever
    their features hold.  Any other target outside the vocabulary makes its row's loss NaN.
    The logits' gradients enter the products in the inputs' type (in two parts of it where there are
    few; float32: with 22 bits or more, in steps of 2**-62 of the largest row's), and so rounded they
    decide the gradients' precision.
    """
    _check_table(table, "table", _MAX_CLASSES)
    device, dim = table.device, table.shape[1]
    if not isinstance(features, torch.Tensor) or features.device != device:
        raise ValueError(f"features must be a tensor on {device}")
    if features.dtype != table.dtype:
        raise ValueError(f"features must have the table's dtype {table.dtype}, got {features.dtype}")
    if features.ndim == 0 or features.shape[-1] != dim:
        raise ValueError(f"features must have shape (..., {dim}), got {tuple(features.shape)}")
    _check_indices(targets, "targets", device)
    if targets.shape != features.shape[:-1]:
        raise ValueError(f"targets must have shape {tuple(features.shape[:-1])}, got {tuple(targets.shape)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of 'none', 'sum', 'mean', got {reduction!r}")
    if not isinstance(ignore_index, int) or not -2**63 <= ignore_index < 2**63:
        raise ValueError("ignore_index must be an integer of 64 bits")
    logit_scale = _check_factor(logit_scale, "logit_scale")
    shape = targets.shape
    features = features if features.ndim == 2 else features.reshape(-1, dim)
    features, table = _rows(features, 16), _rows(table, 16)
    targets = (targets if len(shape) == 1 else targets.reshape(-1)).contiguous()
    if torch.is_grad_enabled() and (features.requires_grad or table.requires_grad):
        loss = LinearCrossEntropy.apply(features, table, targets, ignore_index, reduction, logit_scale)
    else:
        loss = _entropy_forward(features, table, targets, ignore_index, reduction, logit_scale, False)[0]
    return loss.reshape(shape) if reduction == "none" and len(shape) != 1 else loss


class Vocabulary(nn.Module):
    """A learned table used at both ends: looked up by token, and scored against.

    ``forward(tokens)`` is :func:`embed_tokens` with the module's scale and padding row,
    ``loss(features, targets)`` is :func:`linear_cross_entropy` with its logit scale.
    """

    def __init__(self, size: int, dim: int, *, scale: float = 1.0, padding_idx: int | None = None,
                 logit_scale: float = 1.0, dtype: torch.dtype = torch.float32, device=None):
        super().__init__()
        self.scale, self.padding_idx, self.logit_scale = scale, padding_idx, logit_scale
        self.weight = nn.Parameter(torch.randn(size, dim, device=device).div_(math.sqrt(dim)).to(dtype))

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return embed_tokens(tokens, self.weight, scale=self.scale, padding_idx=self.padding_idx)

    def loss(self, features: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
             reduction: str = "mean") -> torch.Tensor:
        return linear_cross_entropy(features, self.weight, targets, ignore_index=ignore_index, reduction=reduction,
                                    logit_scale=self.logit_scale)


__all__ = ["embed_tokens", "linear_cross_entropy", "Vocabulary"]
