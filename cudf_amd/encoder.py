"""Operators between the tokenizer's column of ids and a model that learns from it, over the C ABI of
include/nvtext_amd_encoder.h: embedding, dropout, layer norm and linear, each with its gradient.

Tensors are torch's, in HBM, of float32, float16 or bfloat16; the last dimension is contiguous, rows may lie apart.
Tensors of more than two dimensions are taken as the rows of their last one; what belongs
to another's rows has its shape, or has them in two dimensions.  As in cudf_amd.nvtext, torch owns memory and
provides the stream, and every computation happens in libnvtext_amd.so: ValueError for arguments that do not fit.
Nothing is recorded for torch's autograd: a result does not require a gradient, whatever its arguments do, and the gradients are
the calls named *_backward.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple

import numpy as np
import torch

from . import _capi
from .nvtext import DeviceListColumn, _mr, _raise, _stream_handle

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}

_TYPES = {torch.float32: _capi.TYPE_FLOAT32, torch.float16: _capi.TYPE_FLOAT16, torch.bfloat16: _capi.TYPE_BFLOAT16}
_INT32 = np.dtype(np.int32)
_Matrix = _capi.Matrix


class UnevenRowsError(ValueError, RuntimeError):
    """The rows of a tensor of more than two dimensions do not lie at equal distances (a RuntimeError as well, which is what
    torch's view() raises for them)."""


class LayerNormSaved(NamedTuple):
    """What layer_norm keeps for its gradient: what was normalized, and the mean and the reciprocal deviation of each row."""
    sum: torch.Tensor
    mean: torch.Tensor
    rstd: torch.Tensor


def _matrix(t: torch.Tensor, name: str) -> _capi.Matrix:
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16")
    if not t.is_cuda:
        raise ValueError(f"{name} must be in device memory")
    shape, strides = t.shape, t.stride()
    n = len(shape)
    if n == 0:
        raise ValueError(f"{name} must have a last dimension")
    cols = shape[-1]
    if strides[-1] != 1 and cols > 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    if n == 2:
        rows, stride = shape[0], strides[0]
    elif n == 1:
        rows, stride = 1, cols
    elif t.is_contiguous():
        rows, stride = t.numel() // cols if cols else shape[:-1].numel(), cols
    else:
        try:
            u = t.view(-1, cols)
        except RuntimeError as error:
            raise UnevenRowsError(f"the rows of {name} must be evenly spaced") from error
        rows, stride = u.shape[0], u.stride(0)
    if rows < 2 and stride < cols:
        stride = cols
    return _Matrix(t.data_ptr(), rows, cols, stride, kind)


def _new(t: torch.Tensor, rows: int, cols: int) -> _capi.Matrix:
    """The view of a contiguous tensor that was made here."""
    return _Matrix(t.data_ptr(), rows, cols, cols, _TYPES[t.dtype])


def _like(t: torch.Tensor) -> torch.Tensor:
    # (empty_like costs a third of empty, but would take over the strides of a view)
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _vector(t: torch.Tensor, name: str) -> _capi.Matrix:
    if t.dim() != 1:
        raise ValueError(f"{name} must be a vector")
    return _matrix(t, name)


def _like_shape(t: Optional[torch.Tensor], shape, name: str) -> Optional[_capi.Matrix]:
    """t's rows, which must be those of a tensor of `shape`: given as such or as the rows alone, in at most two dimensions."""
    if t is None:
        return None
    if t.dim() > 2 and len(shape) > 2 and t.shape != shape:
        raise ValueError(f"{name} must be of shape {tuple(shape)}, or its rows")
    return _matrix(t, name)


def _ids(tokens: DeviceListColumn) -> _capi.ListColumn:
    if tokens.child_dtype != _INT32:
        raise ValueError("tokens must be a LIST<INT32> column")
    return _capi.ListColumn(tokens.size, tokens.null_count, _capi.TYPE_INT32, tokens.size + 1 if tokens.offsets is not None else 0,
                            tokens.offsets.data_ptr() if tokens.offsets is not None else None,
                            tokens.child.data_ptr() if tokens.child is not None else None, tokens.child_size, None, 0, 0, 0)


def _seed(seed: int, offset: int) -> Tuple[int, int]:
    if not (0 <= seed < 2**64):
        raise ValueError("seed must fit uint64")
    if not (0 <= offset < 2**32):
        raise ValueError("offset must fit uint32")
    return seed, offset


def embedding(tokens: DeviceListColumn, token_table: torch.Tensor, position_table: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[tokens, width]: of every token of the column the row of `token_table` that its id names, plus the row of
    `position_table` for its place in its row.  An id that is no row of the table (-1) and a place beyond the last row of
    the other add nothing."""
    column, table = _ids(tokens), _matrix(token_table, "token_table")
    positions = None if position_table is None else _matrix(position_table, "position_table")
    out = token_table.new_empty((tokens.child_size, table.cols))
    st = _capi.load().nvtext_amd_embedding(column, table, positions, _stream_handle(), _new(out, tokens.child_size, table.cols))
    if st != _capi.SUCCESS:
        _raise(st)
    return out


def embedding_backward(tokens: DeviceListColumn, grad: torch.Tensor, vocabulary_size: int, positions: int = 0,
                       dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The gradients of embedding()'s tables, of `vocabulary_size` and `positions` rows (none for 0), in grad's type or in
    `dtype` (float32).  Sums are held in 32 bits and added in the same order at every call."""
    if vocabulary_size < 0 or positions < 0:
        raise ValueError("the tables' sizes must not be negative")
    column, g = _ids(tokens), _matrix(grad, "grad")
    width = g.cols
    token_grad = grad.new_empty((vocabulary_size, width), dtype=dtype)
    position_grad = grad.new_empty((positions, width), dtype=dtype) if positions else None
    st = _capi.load().nvtext_amd_embedding_backward(column, g, _stream_handle(), _mr().struct, _matrix(token_grad, "the gradient"),
                                                    None if position_grad is None else _new(position_grad, positions, width))
    if st != _capi.SUCCESS:
        _raise(st)
    return token_grad, position_grad


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """x with each value dropped (0) with probability `p`, which is rounded to 1/65536, and the others multiplied by
    1 / (1 - p).  What is dropped follows from `seed`, `offset` (a call's own number under that seed) and the place of the
    value alone, so no mask is kept: dropout(grad, p, seed, offset) is the gradient."""
    seed, offset = _seed(seed, offset)
    m = _matrix(x, "x")
    out = _like(x)
    st = _capi.load().nvtext_amd_dropout(m, p, seed, offset, _stream_handle(), _new(out, m.rows, m.cols))
    if st != _capi.SUCCESS:
        _raise(st)
    return out


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-5, residual: Optional[torch.Tensor] = None,
               p: float = 0.0, seed: int = 0, offset: int = 0, keep: bool = False):
    """The layer norm of residual + dropout(x, p, seed, offset) over the last dimension.  keep: returns (out,
    LayerNormSaved) for layer_norm_backward; saved.sum is also what goes on along the residual stream (x itself where
    there is neither a residual nor dropout).  weight and bias are of x's type or float32."""
    seed, offset = _seed(seed, offset)
    m = _matrix(x, "x")
    rows, cols = m.rows, m.cols
    out = _like(x)
    total = mean = rstd = m_total = None
    if keep:
        total = x
        if residual is not None or p != 0:
            total = _like(x)
            m_total = _new(total, rows, cols)
        mean, rstd = x.new_empty(x.shape[:-1], dtype=torch.float32), x.new_empty(x.shape[:-1], dtype=torch.float32)
    st = _capi.load().nvtext_amd_layer_norm(
        m, _like_shape(residual, x.shape, "residual"), _vector(weight, "weight"), _vector(bias, "bias"), eps, p, seed, offset, _stream_handle(),
        _new(out, rows, cols), m_total, mean.data_ptr() if keep else None, rstd.data_ptr() if keep else None)
    if st != _capi.SUCCESS:
        _raise(st)
    return (out, LayerNormSaved(total, mean, rstd)) if keep else out


def layer_norm_backward(grad: torch.Tensor, saved: LayerNormSaved, weight: torch.Tensor, p: float = 0.0, seed: int = 0, offset: int = 0,
                        sum_grad: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(grad of x, grad of the residual, grad of weight, grad of bias) from the gradient of layer_norm's output and, where
    saved.sum went on along the residual stream, that of saved.sum.  Without dropout the first two are one tensor."""
    seed, offset = _seed(seed, offset)
    g = _matrix(grad, "grad")
    for t in (saved.mean, saved.rstd):
        if t.dtype != torch.float32 or not t.is_contiguous() or t.numel() != g.rows or not t.is_cuda:
            raise ValueError("mean and rstd must be contiguous float32 tensors of one value a row")
    rows, cols = g.rows, g.cols
    m_weight = _vector(weight, "weight")
    residual_grad, weight_grad, bias_grad = _like(grad), _like(weight), _like(weight)
    x_grad = _like(grad) if p != 0 else residual_grad
    st = _capi.load().nvtext_amd_layer_norm_backward(
        g, _like_shape(saved.sum, grad.shape, "sum"), saved.mean.data_ptr(), saved.rstd.data_ptr(), m_weight, _like_shape(sum_grad, grad.shape, "sum_grad"),
        p, seed, offset, _stream_handle(), _mr().struct, _new(x_grad, rows, cols) if p != 0 else None, _new(residual_grad, rows, cols),
        _new(weight_grad, 1, m_weight.cols), _new(bias_grad, 1, m_weight.cols))
    if st != _capi.SUCCESS:
        _raise(st)
    return x_grad, residual_grad, weight_grad, bias_grad


def _activation(name: str) -> int:
    code = ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}")
    return code


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None, keep: bool = False):
    """activation(x @ weight.T + bias) + residual; weight is [outputs, inputs].  keep: returns (out, what the activation
    was applied to) for linear_backward."""
    act = _activation(activation)
    m, w = _matrix(x, "x"), _matrix(weight, "weight")
    rows, outputs = m.rows, w.rows
    shape = (rows, outputs) if x.dim() == 2 else x.shape[:-1] + (outputs,)
    out = x.new_empty(shape)
    z = torch.empty_like(out) if keep else None
    st = _capi.load().nvtext_amd_linear(m, w, None if bias is None else _vector(bias, "bias"), act, _like_shape(residual, shape, "residual"),
                                        _stream_handle(), _mr().struct, _new(out, rows, outputs), _new(z, rows, outputs) if keep else None)
    if st != _capi.SUCCESS:
        _raise(st)
    return (out, z) if keep else out


def linear_backward(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, activation: str = "none",
                    preactivation: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(grad of x, grad of weight, grad of bias) of linear(); the residual's gradient is grad itself.  grad times the activation's
    slope is rounded to the tensors' type before it is multiplied."""
    act = _activation(activation)
    m, w = _matrix(x, "x"), _matrix(weight, "weight")
    g = _like_shape(grad, x.shape[:-1] + (w.rows,), "grad")
    x_grad, weight_grad = _like(x), _like(weight)
    bias_grad = weight.new_empty(w.rows)
    st = _capi.load().nvtext_amd_linear_backward(g, m, w, act, _like_shape(preactivation, grad.shape, "preactivation"), _stream_handle(), _mr().struct,
                                                 _new(x_grad, m.rows, m.cols), _new(weight_grad, w.rows, w.cols), _new(bias_grad, 1, w.rows))
    if st != _capi.SUCCESS:
        _raise(st)
    return x_grad, weight_grad, bias_grad
