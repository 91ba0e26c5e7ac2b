"""Operators between the tokenizer's column of ids and a model that learns from it, over the C ABI of
include/nvtext_amd_encoder.h: embedding, dropout, layer norm, linear, rotary positions and attention, each with its gradient.

Tensors are torch's, in HBM, of float32, float16 or bfloat16; the last dimension is contiguous, rows may lie apart.
Tensors of more than two dimensions are taken as the rows of their last one; what belongs
to another's rows has its shape, or has them in two dimensions.  As in cudf_amd.nvtext, torch owns memory and
provides the stream, and every computation happens in libnvtext_amd.so: ValueError for arguments that do not fit.
Nothing is recorded for torch's autograd: a result does not require a gradient, whatever its arguments do, and the gradients are
the calls named *_backward.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Tuple, Union

import numpy as np
import torch

from . import _capi
from .nvtext import DeviceListColumn, _mr, _raise, _stream_handle

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}

ROTARY_LAYOUTS = {"half": 0, "interleaved": 1}

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


class AttentionSaved(NamedTuple):
    """What attention keeps for its gradient: its result, of every head of a token the logarithm of what its exponentials
    add up to, [heads, tokens], and, of 16-bit types, what rounding left off the result, an int8 for each of its values,
    [heads, tokens, width].
    (Without that, the gradients of q and k are off by a rounding more.)"""
    out: torch.Tensor
    logsum: torch.Tensor
    rest: Optional[torch.Tensor] = None


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


Rows = Union[DeviceListColumn, torch.Tensor]


def _heads(t: torch.Tensor, name: str) -> _capi.Heads:
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16")
    if t.dim() != 3:
        raise ValueError(f"{name} must be of shape [tokens, heads, width]")
    _here(t, name)
    (tokens, heads, width), (stride, head_stride, step) = t.shape, t.stride()
    if step != 1 and width > 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    return _capi.Heads(t.data_ptr(), tokens, heads, width, stride, head_stride, kind)


def _here(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be in device memory")
    # (the calls run on the current device's stream, and take their temporaries there)
    if t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"{name} must be on the current device")


def _int32s(t: Optional[torch.Tensor], count: Optional[int], name: str) -> Optional[int]:
    """The address of a tensor of `count` int32 values."""
    if t is None:
        return None
    _here(t, name)
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of int32")
    if count is not None and t.numel() != count:
        raise ValueError(f"{name} must have {count} values")
    return t.data_ptr()


def _rows(rows: Rows) -> Tuple[int, Optional[int]]:
    """(how many there are, the address of their offsets)."""
    if isinstance(rows, DeviceListColumn):
        if rows.size > 0:
            _here(rows.offsets, "the column")
        return rows.size, rows.offsets.data_ptr() if rows.offsets is not None else None
    address = _int32s(rows, None, "offsets")
    if rows.numel() == 0:
        raise ValueError("offsets must have a value more than there are rows")
    return rows.numel() - 1, address


def rotary_frequencies(width: int, base: float = 10000.0, factor: float = 1.0, length: int = 0, slow: float = 1.0, fast: float = 4.0,
                       device: Union[str, torch.device] = "cuda") -> torch.Tensor:
    """The frequencies that rotary() takes for `width` values of a head, width / 2 of them, in radians a position: base^(-2 n / width).
    For contexts `factor` times longer than a model has learned, all of them divided by that; or, where `length` names
    the positions it has learned, only those that turn up to `slow` times within it, with those that turn `fast` times and
    more left as they are and those in between passing from one to the other with their turns."""
    if width < 2 or width % 2:
        raise ValueError("width must be even, and at least 2")
    if not (base > 0 and factor > 0 and math.isfinite(base) and math.isfinite(factor)):
        raise ValueError("base and factor must be positive")
    if length < 0 or (length and not 0 <= slow < fast):
        raise ValueError("length must not be negative, and slow less than fast")
    f = base ** (-np.arange(0, width, 2, dtype=np.float64) / width)
    share = np.clip((f * length / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0) if length else 0.0  # of what is left as it is
    return torch.from_numpy(f * share + f / factor * (1 - share)).to(device)


def rotary(x: torch.Tensor, rows: Rows, frequencies: torch.Tensor, starts: Optional[torch.Tensor] = None, layout: str = "half", inverse: bool = False,
           magnitude: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x, [tokens, heads, width], with the first 2 * len(frequencies) values of every head rotated in pairs by its token's position in its
    row times the pair's frequency (float64, as rotary_frequencies() gives them), and multiplied by `magnitude`.  The pairs of
    layout "half" are n and n + len(frequencies), those of "interleaved" 2 n and 2 n + 1.  rows: the tokenizer's column, or int32 offsets;
    starts: int32, the position of every row's first token (of a text under way).  Query and key heads that lie next to each
    other take one call.  inverse=True on the gradient of the result gives that of x.  out: where the result goes, x itself
    if wanted, but nothing that holds values of x in other places."""
    code = ROTARY_LAYOUTS.get(layout)
    if code is None:
        raise ValueError(f"layout must be one of {', '.join(ROTARY_LAYOUTS)}")
    m = _heads(x, "x")
    count, offsets = _rows(rows)
    _here(frequencies, "frequencies")
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or not frequencies.is_contiguous():
        raise ValueError("frequencies must be a contiguous vector of float64")
    if out is None:
        out = _like(x)
    st = _capi.load().nvtext_amd_rotary(m, count, offsets, _int32s(starts, count, "starts"), frequencies.data_ptr(), frequencies.numel(), code, inverse, magnitude,
                                        _stream_handle(), _heads(out, "out"))
    if st != _capi.SUCCESS:
        _raise(st)
    return out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rows: Rows, key_rows: Optional[Rows] = None, key_lengths: Optional[torch.Tensor] = None,
              causal: bool = False, scale: Optional[float] = None, keep: bool = False):
    """softmax(scale * q @ k.T) @ v of every row's tokens by themselves, head by head.  q is [tokens, heads, width] with width up to 256, k and v
    [key tokens, a divisor of heads, width]: as many neighbouring heads of q see one of them.  Any of them may be a part of
    another tensor (of a projection's result, viewed as heads).  rows: the tokenizer's column, or int32 offsets.
    Keys and values of other rows than q's (those of texts under way, kept from call to call) have offsets of their own, key_rows, and
    where these leave room for more, key_lengths, int32.  causal: the last token of a row sees all its keys, each one before it one less.
    scale: 1 / sqrt(width) if not given.  A token that sees no key has zeros.  keep: returns (out, AttentionSaved) for attention_backward."""
    m = _heads(q, "q")
    count, offsets, *keys = _key_rows(rows, key_rows, key_lengths)
    out = q.new_empty(q.shape)
    logsum = q.new_empty((m.heads, m.tokens), dtype=torch.float32) if keep else None
    rest = q.new_empty((m.heads, m.tokens, m.width), dtype=torch.int8) if keep and q.dtype != torch.float32 else None
    st = _capi.load().nvtext_amd_attention(m, _heads(k, "k"), _heads(v, "v"), count, offsets, *keys, causal, _scale(scale, m.width), _stream_handle(),
                                           _mr().struct, _heads(out, "out"), logsum.data_ptr() if keep else None,
                                           None if rest is None else rest.data_ptr())
    if st != _capi.SUCCESS:
        _raise(st)
    return (out, AttentionSaved(out, logsum, rest)) if keep else out


def attention_backward(grad: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, saved: AttentionSaved, rows: Rows, key_rows: Optional[Rows] = None,
                       key_lengths: Optional[torch.Tensor] = None, causal: bool = False, scale: Optional[float] = None,
                       out: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(grad of q, grad of k, grad of v) of attention().  The gradient of a key head is the sum over the heads that see it.  out: where they go,
    views of one projection's gradient for instance, which hold no value of the other arguments."""
    g, m = _heads(grad, "grad"), _heads(q, "q")
    count, offsets, *keys = _key_rows(rows, key_rows, key_lengths)
    _here(saved.logsum, "logsum")
    if saved.logsum.dtype != torch.float32 or not saved.logsum.is_contiguous() or saved.logsum.shape != (m.heads, m.tokens):
        raise ValueError("logsum must be a contiguous float32 tensor of shape [heads, tokens]")
    if saved.rest is not None:
        _here(saved.rest, "rest")
        if saved.rest.dtype != torch.int8 or not saved.rest.is_contiguous() or saved.rest.shape != (m.heads, m.tokens, m.width):
            raise ValueError("rest must be a contiguous int8 tensor of shape [heads, tokens, width]")
    q_grad, k_grad, v_grad = out if out is not None else (_like(q), _like(k), _like(v))
    st = _capi.load().nvtext_amd_attention_backward(g, m, _heads(k, "k"), _heads(v, "v"), _heads(saved.out, "out"), saved.logsum.data_ptr(),
                                                    None if saved.rest is None else saved.rest.data_ptr(), count, offsets, *keys, causal, _scale(scale, m.width),
                                                    _stream_handle(), _mr().struct, _heads(q_grad, "the gradient of q"), _heads(k_grad, "the gradient of k"), _heads(v_grad, "the gradient of v"))
    if st != _capi.SUCCESS:
        _raise(st)
    return q_grad, k_grad, v_grad


def _scale(scale: Optional[float], width: int) -> float:
    return scale if scale is not None else max(width, 1) ** -0.5


def _key_rows(rows: Rows, key_rows: Optional[Rows], key_lengths: Optional[torch.Tensor]):
    """(rows, the addresses of their offsets, of their keys' offsets and of their keys' lengths)."""
    count, offsets = _rows(rows)
    key_offsets = None
    if key_rows is not None:
        key_count, key_offsets = _rows(key_rows)
        if key_count != count:
            raise ValueError("there must be as many rows of keys as of tokens")
    elif key_lengths is not None:
        raise ValueError("key_lengths need key_rows")
    return count, offsets, key_offsets, _int32s(key_lengths, count, "key_lengths")
