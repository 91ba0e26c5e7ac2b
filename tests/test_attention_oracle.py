"""Rotary positions' and attention's formulas in 64 bits (gradients against differences), and what the calls refuse from their
arguments alone."""
import math

import numpy as np
import pytest

from cudf_amd import _capi
from oracle import encoder_py as orc


def test_rotary_keeps_lengths_and_turns_back():
    rng = np.random.default_rng(0)
    x, f = rng.standard_normal((9, 2, 10)), 10000.0 ** (-np.arange(4) / 4)
    for layout in ("half", "interleaved"):
        y, _ = orc.rotary(x, [1, 4, 8], f, [5, 0], layout, magnitude=1.25)
        assert np.allclose((y[1:8] ** 2)[..., :8].sum(-1), (x[1:8] ** 2)[..., :8].sum(-1) * 1.25**2)
        assert np.array_equal(y[0], x[0]) and np.array_equal(y[8], x[8]) and np.array_equal(y[..., 8:], x[..., 8:])
        back, _ = orc.rotary(y, [1, 4, 8], f, [5, 0], layout, inverse=True, magnitude=1 / 1.25)
        assert np.allclose(back, x)
        # products of two tokens of a row depend on how far they are apart alone
        z, _ = orc.rotary(x, [1, 4, 8], f, [1005, 1000], layout)
        w, _ = orc.rotary(x, [1, 4, 8], f, None, layout)
        assert np.allclose((z[1] * z[3]).sum(), (w[1] * w[3]).sum()) and np.allclose((z[4] * z[7]).sum(), (w[4] * w[7]).sum())


def test_rotary_of_pairs():
    f = [math.pi / 2, math.pi / 6]
    y, _ = orc.rotary(np.array([[[0.0] * 4], [[1.0, 2.0, 3.0, 4.0]]]), [0, 2], f, None, "interleaved")
    c, s = math.sqrt(3) / 2, 0.5
    assert np.allclose(y[1, 0], [-2, 1, 3 * c - 4 * s, 3 * s + 4 * c])
    y, _ = orc.rotary(np.array([[[0.0] * 4], [[1.0, 2.0, 3.0, 4.0]]]), [0, 2], f, None, "half")
    assert np.allclose(y[1, 0], [-3, 2 * c - 4 * s, 1, 2 * s + 4 * c])


def test_attention_of_a_row():
    """Weights that are known: scores of log 1, log 2 and log 3."""
    q, k = np.array([[[1.0]]]), np.log([1.0, 2.0, 3.0]).reshape(3, 1, 1)
    v = np.array([6.0, 12.0, 18.0]).reshape(3, 1, 1)
    out, logsum, _, _ = orc.attention(q, k, v, [0, 1], [0, 3], scale=1.0)
    assert np.allclose(out, (6 + 24 + 54) / 6) and np.allclose(logsum, math.log(6))


@pytest.mark.parametrize("causal", [False, True])
def test_attention_gradients_against_differences(causal):
    rng = np.random.default_rng(1)
    offsets, key_offsets, key_lengths = [0, 3, 3, 8], [1, 3, 6, 14], [2, 3, 7]  # (of the first row's tokens, the first sees nothing if causal)
    q, k, v = rng.standard_normal((8, 4, 5)), rng.standard_normal((15, 2, 5)), rng.standard_normal((15, 2, 5))
    g = rng.standard_normal(q.shape)

    def value(q, k, v):
        return (orc.attention(q, k, v, offsets, key_offsets, key_lengths, causal)[0] * g).sum()

    out, logsum, _, _ = orc.attention(q, k, v, offsets, key_offsets, key_lengths, causal)
    assert (not causal) or (np.isinf(logsum[:, 0]).all() and (out[0] == 0).all())
    grads, _ = orc.attention_backward(g, q, k, v, out, logsum, offsets, key_offsets, key_lengths, causal)
    for i, x in enumerate((q, k, v)):
        direction, step = rng.standard_normal(x.shape), 1e-6
        args = [q, k, v]
        args[i] = x + step * direction
        up = value(*args)
        args[i] = x - step * direction
        assert math.isclose((up - value(*args)) / (2 * step), (grads[i] * direction).sum(), rel_tol=1e-6, abs_tol=1e-8)


# ---- refusals: decided from the arguments alone

BF, F16, F32 = _capi.TYPE_BFLOAT16, _capi.TYPE_FLOAT16, _capi.TYPE_FLOAT32
AT = 4096  # an address that no call follows


def h(tokens=10, heads=4, width=8, stride=None, head_stride=None, type=BF, data=AT):
    return _capi.Heads(data, tokens, heads, width, heads * width if stride is None else stride, width if head_stride is None else head_stride, type)


def refused(st, text):
    assert st == _capi.INVALID_ARGUMENT
    assert text in _capi.load().nvtext_amd_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(x=None), "null"), (dict(out=None), "null"), (dict(x=h(type=7)), "FLOAT32"), (dict(x=h(-1)), "sizes"), (dict(x=h(2**31)), "sizes"), (dict(x=h(stride=-8)), "negative"),
    (dict(x=h(head_stride=-8)), "negative"), (dict(x=h(data=None)), "no data"), (dict(x=h(data=4097)), "aligned"), (dict(out=h(9)), "size"), (dict(out=h(heads=3)), "size"),
    (dict(out=h(width=9)), "size"), (dict(out=h(type=F16)), "type"), (dict(out=h(stride=0)), "overlap"), (dict(out=h(stride=31)), "overlap"), (dict(out=h(head_stride=7)), "overlap"),
    (dict(out=h(stride=8, head_stride=79)), "overlap"), (dict(rows=-1), "number of rows"), (dict(offsets=None), "need offsets"), (dict(pairs=-1), "frequencies"), (dict(pairs=5), "frequencies"),
    (dict(frequencies=None), "frequencies"), (dict(layout=2), "layout"), (dict(layout=-1), "layout"), (dict(magnitude=float("nan")), "magnitude"), (dict(magnitude=float("inf")), "magnitude"),
    (dict(x=h(width=8192), out=h(width=8192), pairs=2049), "2048"), (dict(x=h(stride=64)), "another order"),
])
def test_rotary_refusals(change, text):
    a = dict(x=h(), rows=2, offsets=AT, starts=None, frequencies=AT, pairs=4, layout=0, inverse=0, magnitude=1.0, out=h())
    a.update(change)
    refused(_capi.load().nvtext_amd_rotary(a["x"], a["rows"], a["offsets"], a["starts"], a["frequencies"], a["pairs"], a["layout"], a["inverse"], a["magnitude"], None, a["out"]), text)


def test_rotary_of_too_many_values():
    big = dict(tokens=1, heads=2**20, width=2**10)
    assert _capi.load().nvtext_amd_rotary(h(**big), 1, AT, None, AT, 4, 0, 0, 1.0, None, h(**big)) == _capi.OVERFLOW


SHARED = [
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(q=h(type=7)), "FLOAT32"), (dict(k=h(heads=2, type=F32)), "one type"), (dict(v=h(heads=2, type=F16)), "one type"),
    (dict(v=h(11, 2)), "k's size"), (dict(v=h(heads=4)), "k's size"), (dict(k=h(heads=2, width=9), v=h(heads=2, width=9)), "width"), (dict(k=h(heads=3), v=h(heads=3)), "divisor"),
    (dict(k=h(heads=0), v=h(heads=0)), "divisor"), (dict(q=h(width=257), k=h(heads=2, width=257), v=h(heads=2, width=257)), "256"), (dict(rows=-3), "number of rows"),
    (dict(offsets=None), "need offsets"), (dict(key_lengths=AT), "key_offsets"), (dict(k=h(11, 2), v=h(11, 2)), "q's tokens"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=1e300), "scale"), (dict(k=h(heads=2, stride=-16)), "negative"), (dict(q=h(data=4097)), "aligned"),
]


@pytest.mark.parametrize("change,text", SHARED + [(dict(out=None), "null"), (dict(out=h(9)), "q's size"), (dict(out=h(type=F32)), "type"), (dict(out=h(stride=16)), "overlap")])
def test_attention_refusals(change, text):
    a = dict(q=h(), k=h(heads=2), v=h(heads=2), rows=2, offsets=AT, key_offsets=None, key_lengths=None, causal=0, scale=1.0, out=h(), logsum=None)
    a.update(change)
    refused(_capi.load().nvtext_amd_attention(a["q"], a["k"], a["v"], a["rows"], a["offsets"], a["key_offsets"], a["key_lengths"], a["causal"], a["scale"], None, None, a["out"], a["logsum"], None), text)


@pytest.mark.parametrize("change,text", SHARED + [
    (dict(grad=None), "null"), (dict(out=None), "null"), (dict(logsum=None), "null"), (dict(dq=None), "null"), (dict(dk=None), "null"), (dict(dv=None), "null"), (dict(grad=h(9)), "q's size"),
    (dict(out=h(heads=2)), "q's size"), (dict(grad=h(type=F16)), "type"), (dict(dq=h(heads=2)), "those of"), (dict(dk=h()), "those of"), (dict(dv=h(heads=2, type=F32)), "those of"),
    (dict(dk=h(heads=2, stride=0)), "overlap"),
])
def test_attention_backward_refusals(change, text):
    a = dict(grad=h(), q=h(), k=h(heads=2), v=h(heads=2), out=h(), logsum=AT, rows=2, offsets=AT, key_offsets=None, key_lengths=None, causal=0, scale=1.0, dq=h(), dk=h(heads=2), dv=h(heads=2))
    a.update(change)
    refused(_capi.load().nvtext_amd_attention_backward(a["grad"], a["q"], a["k"], a["v"], a["out"], a["logsum"], None, a["rows"], a["offsets"], a["key_offsets"], a["key_lengths"], a["causal"], a["scale"],
                                                       None, None, a["dq"], a["dk"], a["dv"]), text)


def test_calls_without_values_need_no_gpu():
    L = _capi.load()
    none = h(0, data=None)
    assert L.nvtext_amd_rotary(none, 0, None, None, AT, 4, 0, 0, 1.0, None, none) == _capi.SUCCESS
    assert L.nvtext_amd_rotary(h(heads=0), 2, AT, None, AT, 4, 0, 0, 1.0, None, h(heads=0)) == _capi.SUCCESS
    assert L.nvtext_amd_attention(none, none, none, 0, None, None, None, 0, 1.0, None, None, none, None, None) == _capi.SUCCESS
    assert L.nvtext_amd_attention(none, h(), h(), 2, AT, AT, None, 0, 1.0, None, None, none, None, None) == _capi.SUCCESS
    assert L.nvtext_amd_attention_backward(none, none, none, none, none, None, None, 0, None, None, None, 0, 1.0, None, None, none, none, none) == _capi.SUCCESS


def test_rotary_frequencies():
    encoder = pytest.importorskip("cudf_amd.encoder")
    f = encoder.rotary_frequencies(8, 100.0, device="cpu").numpy()
    assert f.dtype == np.float64 and np.allclose(f, [1, 100**-0.25, 0.1, 100**-0.75])
    assert np.allclose(encoder.rotary_frequencies(8, 100.0, factor=4.0, device="cpu").numpy(), f / 4)
    turns = f * 100 / (2 * math.pi)  # 15.9, 5.03, 1.59, 0.503
    g = encoder.rotary_frequencies(8, 100.0, factor=4.0, length=100, slow=1.0, fast=5.0, device="cpu").numpy()
    assert np.allclose(g[:2], f[:2]) and math.isclose(g[3], f[3] / 4)
    share = (turns[2] - 1) / 4
    assert math.isclose(g[2], f[2] * share + f[2] / 4 * (1 - share))
    for bad in (dict(width=7), dict(width=0), dict(width=8, base=0.0), dict(width=8, factor=-1.0), dict(width=8, factor=float("nan")), dict(width=8, length=-1), dict(width=8, length=5, slow=2.0, fast=2.0)):
        with pytest.raises(ValueError):
            encoder.rotary_frequencies(device="cpu", **bad)


@pytest.mark.parametrize("tokens,count,kv,text", [(2**31 - 1, 1, 1, "at most"), (1, 65537, 1, "at most"), (1, 65537, 65537, "at most"), (2**31 - 2000, 65536, 1, "too many tokens")])
def test_sizes_that_are_not_counted(tokens, count, kv, text):
    """More tokens than 32 bits count to a tile's end, and heads without end."""
    q, k = (_capi.Heads(4096, tokens, n, 8, 0, 0, _capi.TYPE_FLOAT32) for n in (count, kv))
    out, more = (_capi.Heads(4096, tokens, n, 8, n * 8, 8, _capi.TYPE_FLOAT32) for n in (count, kv))
    lib = _capi.load()
    refused(lib.nvtext_amd_attention(q, k, k, 1, 4096, None, None, 0, 1.0, None, None, out, None, None), text)
    refused(lib.nvtext_amd_attention_backward(q, q, k, k, q, 4096, None, 1, 4096, None, None, 0, 1.0, None, None, out, more, more), text)
