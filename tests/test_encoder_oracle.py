"""The 64-bit definitions of the encoder operators against published values, against each other and against differences
(CPU), and what the entry points refuse (no GPU work)."""
import ctypes as C

import numpy as np
import pytest

from cudf_amd import _capi
from oracle import encoder_py as orc

ACTIVATIONS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


@pytest.mark.parametrize("counter,key,words", [
    # the known answers that the authors of Philox publish with it
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_philox_known_answers(counter, key, words):
    assert tuple(int(w) for w in orc.philox4x32(counter, key)) == words


def test_multipliers_keep_the_mean():
    m = orc.multipliers(400, 1000, 0.25, 7, 3)
    kept = (m > 0).mean()
    assert abs(kept - 0.75) < 5 * (0.25 * 0.75 / m.size) ** 0.5
    assert set(np.unique(m)) == {0.0, 65536 / 49152}
    assert (orc.multipliers(3, 9, 1.0, 7, 3) == 0).all() and (orc.multipliers(3, 9, 0.0, 7, 3) == 1).all()


def _difference(f, at, direction, h):
    return (f(at + h * direction) - f(at - h * direction)) / (2 * h)


# Central differences in 64 bits with h = 1e-5: rounding gives 1e-16 / h, the third derivative h^2; sums of some hundred terms
CLOSE = dict(rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_linear_gradients_against_differences(activation):
    rng = np.random.default_rng(1)
    x, w, b, r, g = (rng.standard_normal(s) for s in ((5, 7), (4, 7), 4, (5, 4), (5, 4)))
    _, z, _ = orc.linear(x, w, b, activation, r)
    (dx, dw, db), _ = orc.linear_backward(g, x, w, activation, z)
    for value, grad, f in ((x, dx, lambda v: orc.linear(v, w, b, activation, r)), (w, dw, lambda v: orc.linear(x, v, b, activation, r)),
                           (b, db, lambda v: orc.linear(x, w, v, activation, r))):
        v = rng.standard_normal(value.shape)
        np.testing.assert_allclose((grad * v).sum(), _difference(lambda a: (f(a)[0] * g).sum(), value, v, 1e-5), **CLOSE)


@pytest.mark.parametrize("with_sum_grad", [False, True])
def test_layer_norm_gradients_against_differences(with_sum_grad):
    rng = np.random.default_rng(2)
    x, res, g, e = (rng.standard_normal((6, 11)) for _ in range(4))
    w, b = rng.standard_normal(11), rng.standard_normal(11)
    m = orc.multipliers(6, 11, 0.3, 99, 4)

    def loss(x=x, res=res, w=w, b=b):
        out, s, _, _ = orc.layer_norm(x, w, b, 1e-5, res, m)
        return (out * g).sum() + ((s * e).sum() if with_sum_grad else 0.0)
    _, s, mean, rstd = orc.layer_norm(x, w, b, 1e-5, res, m)
    dx, ds, dw, db = orc.layer_norm_backward(g, s, mean, rstd, w, e if with_sum_grad else None, m)[:4]
    for name, value, grad in (("x", x, dx), ("res", res, ds), ("w", w, dw), ("b", b, db)):
        v = rng.standard_normal(value.shape)
        np.testing.assert_allclose((grad * v).sum(), _difference(lambda a: loss(**{name: a}), value, v, 1e-5), **CLOSE)


def test_embedding_gradients_are_its_transpose():
    rng = np.random.default_rng(3)
    offsets, ids = np.array([2, 2, 7, 8, 8, 20]), rng.integers(-2, 9, 23)
    table, positions, g = rng.standard_normal((7, 5)), rng.standard_normal((4, 5)), rng.standard_normal((23, 5))
    out, _ = orc.embedding(offsets, ids, table, positions)
    (dt, dp), _ = orc.embedding_backward(offsets, ids, g, 7, 4)
    np.testing.assert_allclose((out * g).sum(), (table * dt).sum() + (positions * dp).sum(), rtol=1e-12)
    assert (out[:2] == 0).all() and (out[20:] == 0).all()


# ---- refusals: decided from the arguments alone

BF, F16, F32 = _capi.TYPE_BFLOAT16, _capi.TYPE_FLOAT16, _capi.TYPE_FLOAT32
AT = 4096  # an address that no call follows


def m(rows, cols, type=BF, stride=None, data=AT):
    return _capi.Matrix(data, rows, cols, cols if stride is None else stride, type)


def column(rows=3, count=10, child_type=_capi.TYPE_INT32, offsets=AT, child=AT):
    return _capi.ListColumn(rows, 0, child_type, rows + 1, offsets, child, count, None, 0, 0, 0)


def refused(st, text):
    assert st == _capi.INVALID_ARGUMENT
    assert text in _capi.load().nvtext_amd_last_error().decode()


@pytest.mark.parametrize("args,text", [
    ((None, m(5, 8), None, m(10, 8)), "null"),
    ((column(), None, None, m(10, 8)), "null"),
    ((column(), m(5, 8), None, None), "null"),
    ((column(child_type=_capi.TYPE_UINT32), m(5, 8), None, m(10, 8)), "INT32"),
    ((column(rows=-1), m(5, 8), None, m(10, 8)), "sizes"),
    ((column(count=-1), m(5, 8), None, m(10, 8)), "sizes"),
    ((column(offsets=None), m(5, 8), None, m(10, 8)), "no data"),
    ((column(child=None), m(5, 8), None, m(10, 8)), "no data"),
    ((column(), m(5, 8, F16), None, m(10, 8)), "one type"),
    ((column(), m(5, 16), None, m(10, 8)), "width"),
    ((column(), m(5, 8), m(5, 8, F32), m(10, 8)), "one type"),
    ((column(), m(5, 8), m(5, 9), m(10, 8)), "width"),
    ((column(), m(5, 8), None, m(11, 8)), "every token"),
    ((column(), m(5, 8, stride=7), None, m(10, 8)), "stride"),
    ((column(), m(5, 8, type=7), None, m(10, 8)), "FLOAT32"),
    ((column(), m(5, 8, data=None), None, m(10, 8)), "no data"),
    ((column(), m(5, 8, data=4097), None, m(10, 8)), "aligned"),
    ((column(), m(-5, 8), None, m(10, 8)), "sizes"),
])
def test_embedding_refusals(args, text):
    tokens, table, positions, out = args
    refused(_capi.load().nvtext_amd_embedding(tokens, table, positions, None, out), text)


def test_embedding_too_many_tokens():
    st = _capi.load().nvtext_amd_embedding(column(count=2**31), m(5, 8), None, None, m(2**31, 8))
    assert st == _capi.OVERFLOW


@pytest.mark.parametrize("args,text", [
    ((None, m(10, 8), m(5, 8), None), "null"),
    ((column(), None, m(5, 8), None), "null"),
    ((column(), m(10, 8), None, None), "null"),
    ((column(), m(9, 8), m(5, 8), None), "every token"),
    ((column(), m(10, 8), m(5, 9), None), "width"),
    ((column(), m(10, 8), m(5, 8, F16), None), "type"),
    ((column(), m(10, 8), m(5, 8), m(5, 8, F32)), "both"),
    ((column(), m(10, 8), m(5, 8), m(5, 7)), "width"),
])
def test_embedding_backward_refusals(args, text):
    tokens, grad, table, positions = args
    refused(_capi.load().nvtext_amd_embedding_backward(tokens, grad, None, None, table, positions), text)


@pytest.mark.parametrize("x,p,out,text", [
    (None, 0.1, m(4, 8), "null"), (m(4, 8), 0.1, None, "null"), (m(4, 8), -0.1, m(4, 8), "p must"), (m(4, 8), 1.5, m(4, 8), "p must"),
    (m(4, 8), float("nan"), m(4, 8), "p must"), (m(4, 8), 0.1, m(4, 9), "size"), (m(4, 8), 0.1, m(4, 8, F32), "type"),
    (m(4, 8, data=None), 0.1, m(4, 8), "no data"),
])
def test_dropout_refusals(x, p, out, text):
    refused(_capi.load().nvtext_amd_dropout(x, p, 1, 0, None, out), text)


@pytest.mark.parametrize("change,text", [
    (dict(x=None), "null"), (dict(weight=None), "null"), (dict(bias=None), "null"), (dict(out=None), "null"),
    (dict(x=m(4, 0), out=m(4, 0), weight=m(1, 0), bias=m(1, 0)), "width of 1"), (dict(residual=m(4, 9)), "residual"),
    (dict(residual=m(4, 8, F32)), "residual"), (dict(out=m(3, 8)), "out"), (dict(sum=m(4, 8, F16)), "sum"), (dict(weight=m(1, 7)), "weight"),
    (dict(weight=m(1, 8, F16), bias=m(1, 8, F16)), "weight"), (dict(bias=m(1, 8, F32)), "both"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(p=2.0), "p must"),
])
def test_layer_norm_refusals(change, text):
    a = dict(x=m(4, 8), residual=None, weight=m(1, 8), bias=m(1, 8), eps=1e-5, p=0.0, out=m(4, 8), sum=None)
    a.update(change)
    refused(_capi.load().nvtext_amd_layer_norm(a["x"], a["residual"], a["weight"], a["bias"], a["eps"], a["p"], 0, 0, None, a["out"], a["sum"], None, None), text)


@pytest.mark.parametrize("change,text", [
    (dict(grad=None), "null"), (dict(sum=None), "null"), (dict(weight=None), "null"), (dict(residual_grad=None), "null"), (dict(mean=None), "null"),
    (dict(rstd=None), "null"), (dict(sum=m(4, 9)), "sum"), (dict(sum_grad=m(4, 8, F32)), "sum_grad"), (dict(weight=m(1, 9)), "weight"),
    (dict(bias_grad=None), "come together"), (dict(weight_grad=m(1, 8, F32)), "weight_grad"), (dict(p=0.5, x_grad=None), "x_grad"),
    (dict(p=-1.0), "p must"), (dict(grad=m(4, 0), sum=m(4, 0), residual_grad=m(4, 0)), "width of 1"),
])
def test_layer_norm_backward_refusals(change, text):
    a = dict(grad=m(4, 8), sum=m(4, 8), mean=AT, rstd=AT, weight=m(1, 8), sum_grad=None, p=0.0, x_grad=m(4, 8), residual_grad=m(4, 8),
             weight_grad=m(1, 8), bias_grad=m(1, 8))
    a.update(change)
    refused(_capi.load().nvtext_amd_layer_norm_backward(a["grad"], a["sum"], a["mean"], a["rstd"], a["weight"], a["sum_grad"], a["p"], 0, 0, None, None,
                                                        a["x_grad"], a["residual_grad"], a["weight_grad"], a["bias_grad"]), text)


@pytest.mark.parametrize("change,text", [
    (dict(x=None), "null"), (dict(weight=None), "null"), (dict(out=None), "null"), (dict(weight=m(5, 9)), "inputs"), (dict(bias=m(1, 4)), "bias"),
    (dict(bias=m(1, 5, F32)), "one type"), (dict(residual=m(4, 4)), "residual"), (dict(out=m(3, 5)), "out"), (dict(preactivation=m(4, 6)), "preactivation"),
    (dict(activation=5), "activation"), (dict(activation=-1), "activation"), (dict(x=m(4, 8, stride=6)), "stride"),
])
def test_linear_refusals(change, text):
    a = dict(x=m(4, 8), weight=m(5, 8), bias=m(1, 5), activation=0, residual=None, out=m(4, 5), preactivation=None)
    a.update(change)
    refused(_capi.load().nvtext_amd_linear(a["x"], a["weight"], a["bias"], a["activation"], a["residual"], None, None, a["out"], a["preactivation"]), text)


@pytest.mark.parametrize("change,text", [
    (dict(grad=None), "null"), (dict(x=None), "null"), (dict(weight=None), "null"), (dict(grad=m(4, 6)), "grad"), (dict(preactivation=m(3, 5)), "preactivation"),
    (dict(activation=2), "applied to"), (dict(activation=9), "activation"), (dict(x_grad=m(4, 7)), "x_grad"), (dict(weight_grad=m(8, 5)), "weight_grad"),
    (dict(bias_grad=m(1, 8)), "bias_grad"), (dict(weight=m(5, 8, F16)), "one type"),
])
def test_linear_backward_refusals(change, text):
    a = dict(grad=m(4, 5), x=m(4, 8), weight=m(5, 8), activation=0, preactivation=None, x_grad=m(4, 8), weight_grad=m(5, 8), bias_grad=m(1, 5))
    a.update(change)
    refused(_capi.load().nvtext_amd_linear_backward(a["grad"], a["x"], a["weight"], a["activation"], a["preactivation"], None, None, a["x_grad"],
                                                    a["weight_grad"], a["bias_grad"]), text)


def test_calls_without_values_need_no_gpu():
    """Nothing to compute: no launch, whatever the other sizes are."""
    L = _capi.load()
    assert L.nvtext_amd_dropout(m(0, 8, data=None), 0.1, 1, 0, None, m(0, 8, data=None)) == _capi.SUCCESS
    assert L.nvtext_amd_embedding(column(0, 0, offsets=None, child=None), m(5, 8), None, None, m(0, 8, data=None)) == _capi.SUCCESS
    assert L.nvtext_amd_layer_norm(m(0, 8, data=None), None, m(1, 8), m(1, 8), 1e-5, 0.0, 0, 0, None, m(0, 8, data=None), None, None, None) == _capi.SUCCESS
    assert L.nvtext_amd_linear(m(0, 8, data=None), m(5, 8), None, 0, None, None, None, m(0, 5, data=None), None) == _capi.SUCCESS
