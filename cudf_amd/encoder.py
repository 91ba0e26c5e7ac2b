"""Operators between the tokenizer's column of ids and a model that learns from it, over the C ABI of
include/nvtext_amd_encoder.h: embedding, dropout, layer norm and linear, each with its gradient.

Tensors are torch's, in HBM, of float32, float16 or bfloat16; the last dimension is contiguous, rows may lie apart.
Tensors of more than two dimensions are taken as the rows of their last one.  As in cudf_amd.nvtext, torch owns memory and
provides the stream, and every computation happens in libnvtext_amd.so: ValueError for arguments that do not fit.
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
    else:
        t = t.view(-1, cols)  # raises where the rows are not evenly spaced
        rows, stride = t.shape[0], t.stride(0)
    if rows < 2 and stride < cols:
        stride = cols
    return _capi.Matrix(t.data_ptr(), rows, cols, stride, kind)


def _optional(t: Optional[torch.Tensor], name: str):
    return None if t is None else _matrix(t, name)


def _vector(t: torch.Tensor, name: str) -> _capi.Matrix:
    if t.dim() != 1:
        raise ValueError(f"{name} must be a vector")
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
    positions = _optional(position_table, "position_table")
    out = torch.empty((tokens.child_size, token_table.shape[-1]), dtype=token_table.dtype, device=token_table.device)
    st = _capi.load().nvtext_amd_embedding(column, table, positions, _stream_handle(), _matrix(out, "out"))
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
    dtype = dtype or grad.dtype
    width = grad.shape[-1]
    token_grad = torch.empty((vocabulary_size, width), dtype=dtype, device=grad.device)
    position_grad = torch.empty((positions, width), dtype=dtype, device=grad.device) if positions else None
    st = _capi.load().nvtext_amd_embedding_backward(column, g, _stream_handle(), _mr().struct, _matrix(token_grad, "token_grad"),
                                                    _optional(position_grad, "position_grad"))
    if st != _capi.SUCCESS:
        _raise(st)
    return token_grad, position_grad


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """x with each value dropped (0) with probability `p`, which is rounded to 1/65536, and the others multiplied by
    1 / (1 - p).  What is dropped follows from `seed`, `offset` (a call's own number under that seed) and the place of the
    value alone, so no mask is kept: dropout(grad, p, seed, offset) is the gradient."""
    seed, offset = _seed(seed, offset)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    st = _capi.load().nvtext_amd_dropout(_matrix(x, "x"), p, seed, offset, _stream_handle(), _matrix(out, "out"))
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
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    total = mean = rstd = None
    if keep:
        total = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None or p != 0 else x
        mean, rstd = torch.empty((2,) + x.shape[:-1], dtype=torch.float32, device=x.device)
    st = _capi.load().nvtext_amd_layer_norm(
        m, _optional(residual, "residual"), _vector(weight, "weight"), _vector(bias, "bias"), eps, p, seed, offset, _stream_handle(),
        _matrix(out, "out"), _matrix(total, "sum") if keep and total is not x else None, mean.data_ptr() if keep else None,
        rstd.data_ptr() if keep else None)
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
    residual_grad = torch.empty(grad.shape, dtype=grad.dtype, device=grad.device)
    x_grad = torch.empty(grad.shape, dtype=grad.dtype, device=grad.device) if p != 0 else residual_grad
    weight_grad, bias_grad = torch.empty((2,) + weight.shape, dtype=weight.dtype, device=weight.device)
    st = _capi.load().nvtext_amd_layer_norm_backward(
        g, _matrix(saved.sum, "sum"), saved.mean.data_ptr(), saved.rstd.data_ptr(), _vector(weight, "weight"), _optional(sum_grad, "sum_grad"),
        p, seed, offset, _stream_handle(), _mr().struct, _matrix(x_grad, "x_grad") if p != 0 else None, _matrix(residual_grad, "residual_grad"),
        _vector(weight_grad, "weight_grad"), _vector(bias_grad, "bias_grad"))
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
    out = torch.empty(x.shape[:-1] + weight.shape[:1], dtype=x.dtype, device=x.device)
    z = torch.empty_like(out) if keep else None
    st = _capi.load().nvtext_amd_linear(m, w, None if bias is None else _vector(bias, "bias"), act, _optional(residual, "residual"), _stream_handle(),
                                        _mr().struct, _matrix(out, "out"), _optional(z, "preactivation"))
    if st != _capi.SUCCESS:
        _raise(st)
    return (out, z) if keep else out


def linear_backward(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, activation: str = "none",
                    preactivation: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(grad of x, grad of weight, grad of bias) of linear(); the residual's gradient is grad itself."""
    act = _activation(activation)
    g, m, w = _matrix(grad, "grad"), _matrix(x, "x"), _matrix(weight, "weight")
    x_grad = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    weight_grad = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device)
    bias_grad = torch.empty(weight.shape[:1], dtype=weight.dtype, device=weight.device)
    st = _capi.load().nvtext_amd_linear_backward(g, m, w, act, _optional(preactivation, "preactivation"), _stream_handle(), _mr().struct,
                                                 _matrix(x_grad, "x_grad"), _matrix(weight_grad, "weight_grad"), _vector(bias_grad, "bias_grad"))
    if st != _capi.SUCCESS:
        _raise(st)
    return x_grad, weight_grad, bias_grad
