"""Results of the C interface: into rows that lie apart, at any address, each wanted or not, and over the inputs that the header allows.

What the Python calls give for the same inputs is asked for bit for bit; what lies between and around the rows of a result
stays as it was.
"""
import numpy as np
import pytest
import torch

from cudf_amd import _capi, encoder, nvtext

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
GUARD = -77.0  # what lies around a result


class Result:
    """Rows of a larger matrix that holds nothing but GUARD, `shift` values from its beginning and `gap` values apart."""

    def __init__(self, rows, cols, dtype, shift=3, gap=5, fill=None):
        self.whole = torch.full((rows * (cols + gap) + 2 * shift + 64,), GUARD, device="cuda", dtype=dtype)
        self.view = self.whole[32 + shift:].as_strided((rows, cols), (cols + gap, 1))
        if fill is not None:
            self.view.copy_(fill)
        self.matrix = _capi.Matrix(self.view.data_ptr(), rows, cols, cols + gap, encoder._TYPES[dtype])

    def check(self, want):
        assert torch.equal(self.view, want.view(self.view.shape)), (self.view, want)
        self.view.fill_(GUARD)
        assert (self.whole == GUARD).all()


def vector(t):
    return encoder._matrix(t, "a vector")


def call(name, *args):
    assert getattr(_capi.load(), "nvtext_amd_" + name)(*args) == _capi.SUCCESS, _capi.load().nvtext_amd_last_error()


def randn(seed, *shape, dtype):
    return torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dtype)


def M(t):
    return encoder._matrix(t, "a matrix")


ROWS = [(1, 1), (3, 7), (5, 8), (9, 9), (70, 64), (33, 129), (17, 250), (9, 1021), (5, 2056), (3, 5003), (2, 16391)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols", ROWS)
def test_dropout_and_layer_norm(rows, cols, dtype):
    x, r, w, b = randn(1, rows, cols, dtype=dtype), randn(2, rows, cols, dtype=dtype), randn(3, cols, dtype=dtype), randn(4, cols, dtype=dtype)
    g, e = randn(5, rows, cols, dtype=dtype), randn(6, rows, cols, dtype=dtype)
    stream, mr = nvtext._stream_handle(), nvtext._mr().struct
    want = encoder.dropout(x, 0.3, 7, 8)
    out = Result(rows, cols, dtype)
    call("dropout", M(x), 0.3, 7, 8, stream, out.matrix)
    out.check(want)
    over = Result(rows, cols, dtype, fill=x)
    call("dropout", over.matrix, 0.3, 7, 8, stream, over.matrix)
    over.check(want)

    want, saved = encoder.layer_norm(x, w, b, 1e-5, r, 0.3, 7, 8, keep=True)

    def norm(xs, rs, out, total, mean=None, rstd=None):
        call("layer_norm", xs, rs, vector(w), vector(b), 1e-5, 0.3, 7, 8, stream, out, total, mean, rstd)
    out, total = Result(rows, cols, dtype), Result(rows, cols, dtype, 1, 2)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    norm(M(x), M(r), out.matrix, total.matrix, mean.data_ptr(), rstd.data_ptr())
    out.check(want)
    total.check(saved.sum)
    assert torch.equal(mean, saved.mean) and torch.equal(rstd, saved.rstd)
    norm(M(x), M(r), out.matrix, None)
    out.check(want)
    norm(M(x), M(r), out.matrix, None, None, rstd.fill_(0).data_ptr())
    out.check(want)
    assert torch.equal(rstd, saved.rstd)
    for out_is, sum_is in (("x", "r"), ("r", "x"), ("x", None), (None, "r"), (None, "x"), ("r", None)):
        xs, rs = Result(rows, cols, dtype, fill=x), Result(rows, cols, dtype, 1, 3, fill=r)
        out, total = Result(rows, cols, dtype), Result(rows, cols, dtype)
        at = {"x": xs, "r": rs}
        out, total = at.get(out_is, out), at.get(sum_is, total)
        norm(xs.matrix, rs.matrix, out.matrix, total.matrix)
        out.check(want)
        total.check(saved.sum)

    wants = encoder.layer_norm_backward(g, saved, w, 0.3, 7, 8, e)

    def back(gs, ss, es, xg, rg, wg, bg, p=0.3):
        call("layer_norm_backward", gs, ss, saved.mean.data_ptr(), saved.rstd.data_ptr(), vector(w), es, p, 7, 8, stream, mr, xg, rg, wg, bg)
    xg, rg, wg, bg = Result(rows, cols, dtype), Result(rows, cols, dtype, 1, 2), Result(1, cols, dtype), Result(1, cols, dtype, 1)
    back(M(g), M(saved.sum), M(e), xg.matrix, rg.matrix, wg.matrix, bg.matrix)
    for result, value in zip((xg, rg, wg, bg), wants):
        result.check(value)
    back(M(g), M(saved.sum), M(e), xg.matrix, rg.matrix, None, None)
    xg.check(wants[0])
    rg.check(wants[1])
    for over in range(3):
        ins = [Result(rows, cols, dtype, 1, 1 + i, fill=t) for i, t in enumerate((g, saved.sum, e))]
        back(*(i.matrix for i in ins), xg.matrix, ins[over].matrix, wg.matrix, bg.matrix)
        for result, value in zip((xg, ins[over], wg, bg), wants):
            result.check(value)
    plain = encoder.layer_norm_backward(g, saved, w)
    back(M(g), M(saved.sum), None, None, rg.matrix, wg.matrix, bg.matrix, 0.0)
    for result, value in zip((rg, wg, bg), plain[1:]):
        result.check(value)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 77, 333), (3, 130, 17), (16, 512, 128), (33, 100, 301), (64, 64, 64), (100, 31, 260), (129, 264, 136), (300, 40, 301), (513, 1003, 72),
                                   (700, 75, 1103), (2000, 16, 24)])
def test_linear(m, k, n, dtype):
    x, w, b, r = randn(1, m, k, dtype=dtype), randn(2, n, k, dtype=dtype), randn(3, n, dtype=dtype), randn(4, m, n, dtype=dtype)
    stream, mr = nvtext._stream_handle(), nvtext._mr().struct
    want, want_z = encoder.linear(x, w, b, "gelu", r, keep=True)
    out, z = Result(m, n, dtype), Result(m, n, dtype, 1, 2)
    call("linear", M(x), M(w), vector(b), 2, M(r), stream, mr, out.matrix, z.matrix)
    out.check(want)
    z.check(want_z)
    call("linear", M(x), M(w), vector(b), 2, M(r), stream, mr, out.matrix, None)
    out.check(want)
    over = Result(m, n, dtype, fill=r)
    call("linear", M(x), M(w), vector(b), 2, over.matrix, stream, mr, over.matrix, z.matrix)
    over.check(want)
    z.check(want_z)
    g = randn(5, m, n, dtype=dtype)
    for activation in ("none", "gelu"):
        code = encoder.ACTIVATIONS[activation]
        wants = encoder.linear_backward(g, x, w, activation, want_z)
        results = [Result(m, k, dtype), Result(n, k, dtype, 1, 2), Result(1, n, dtype)]
        for wanted in range(8):
            some = [result.matrix if wanted >> i & 1 else None for i, result in enumerate(results)]
            call("linear_backward", M(g), M(x), M(w), code, M(want_z) if code else None, stream, mr, *some)
            for i, (result, value) in enumerate(zip(results, wants)):
                if wanted >> i & 1:
                    result.check(value)
                else:
                    assert (result.whole == GUARD).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,width", [(1, 1), (70, 7), (300, 8), (333, 129), (65, 1031), (9001, 24), (40000, 5)])
def test_embedding(tokens, width, dtype):
    vocabulary, places = 51, 9
    ids = torch.randint(-1, vocabulary + 1, (tokens,), generator=torch.Generator("cuda").manual_seed(1), device="cuda", dtype=torch.int32)
    offsets = torch.tensor([0, tokens // 3, tokens // 3, tokens], device="cuda", dtype=torch.int32)
    column = nvtext.DeviceListColumn(offsets, ids, None, 3, 0, np.dtype(np.int32), tokens)
    table, positions, g = randn(1, vocabulary, width, dtype=dtype), randn(2, places, width, dtype=dtype), randn(3, tokens, width, dtype=dtype)
    stream, mr = nvtext._stream_handle(), nvtext._mr().struct
    out = Result(tokens, width, dtype)
    call("embedding", encoder._ids(column), M(table), M(positions), stream, out.matrix)
    out.check(encoder.embedding(column, table, positions))
    for kind in {dtype, F32}:
        tg, pg = Result(vocabulary, width, kind), Result(places, width, kind, 1, 2)
        wants = encoder.embedding_backward(column, g, vocabulary, places, dtype=kind)
        call("embedding_backward", encoder._ids(column), M(g), stream, mr, tg.matrix, pg.matrix)
        tg.check(wants[0])
        pg.check(wants[1])
        call("embedding_backward", encoder._ids(column), M(g), stream, mr, tg.matrix, None)
        tg.check(wants[0])
