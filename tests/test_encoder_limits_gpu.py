"""The encoder's operators at the limits of what they count in 32 bits.

Values are whole numbers whose sums stay below 2^24, so that every sum is exact and a result may differ from the formula by
nothing but its one rounding: equality is asked for.
"""
import numpy as np
import pytest
import torch

from cudf_amd import encoder, nvtext

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def whole(shape, dtype, seed, most=1):
    gen = torch.Generator("cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=gen, device="cuda", dtype=torch.int8).to(dtype)


def product(a, b, step=1 << 18):
    """a b^T in 64 bits, a piece of k at a time."""
    total = torch.zeros(a.shape[0], b.shape[0], device="cuda", dtype=torch.float64)
    for k in range(0, a.shape[1], step):
        total += a[:, k:k + step].double() @ b[:, k:k + step].double().t().contiguous()
    return total


def by_rows(f, rows, step=1 << 18):
    return torch.cat([f(slice(i, i + step)) for i in range(0, rows, step)])


# ------------------------------------------------------------------ linear: lines whose bytes, in a tile, are about 2^31 and more

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,n,k", [(70, 24, 2**22 + 72), (200, 20, 2**23), (200, 20, 2**23 + 40), (130, 3, 2**23 + 3), (66, 5, 2**25 + 9)])
def test_linear_of_very_wide_rows(m, n, k, dtype):
    x, w, b = whole((m, k), dtype, 1), whole((n, k), dtype, 2), whole((n,), dtype, 3)
    out, z = encoder.linear(x, w, b, "relu", keep=True)
    want = (product(x, w) + b.double())
    assert torch.equal(z, want.to(dtype)) and torch.equal(out, want.clamp(min=0).to(dtype))


@pytest.mark.parametrize("activation", ["none", "relu"])
@pytest.mark.parametrize("m,n,k", [(130, 2**23 + 40, 16), (129, 2**24 + 72, 9), (130, 24, 2**24 + 8), (140, 33, 2**23 + 3)])
def test_linear_backward_of_very_wide_rows(m, n, k, activation):
    g, x, w = whole((m, n), BF16, 1), whole((m, k), BF16, 2), whole((n, k), BF16, 3)
    z = whole((m, n), BF16, 4) if activation == "relu" else None
    dx, dw, db = encoder.linear_backward(g, x, w, activation, z)
    d = g if z is None else torch.where(z > 0, g, torch.zeros((), device="cuda", dtype=BF16))
    if n > k:
        want_x = product(d, w.t().contiguous())
        want_w = by_rows(lambda s: (d[:, s].double().t().contiguous() @ x.double()).to(BF16), n)
        want_b = torch.cat([d[:, i:i + 2**18].double().sum(0) for i in range(0, n, 2**18)])
    else:
        want_x = torch.cat([(d.double() @ w[:, i:i + 2**18].double()).to(BF16) for i in range(0, k, 2**18)], 1)
        want_w = torch.cat([(d.double().t().contiguous() @ x[:, i:i + 2**18].double()).to(BF16) for i in range(0, k, 2**18)], 1)
        want_b = d.double().sum(0)
    assert torch.equal(dx, want_x.to(BF16)) and torch.equal(dw, want_w.to(BF16)) and torch.equal(db, want_b.to(BF16))


# ------------------------------------------------------------------ embedding

def test_embedding_of_as_many_tokens_as_a_column_holds():
    n, length, vocabulary, places = 2**31 - 5, 4096, 1000, 3
    gen = torch.Generator("cuda").manual_seed(5)
    ids = torch.empty(n, device="cuda", dtype=torch.int32)
    grad = torch.empty(n, 1, device="cuda", dtype=BF16)
    pieces = [slice(i, min(i + 2**26, n)) for i in range(0, n, 2**26)]
    for s in pieces:
        ids[s] = torch.randint(-1, vocabulary, (s.stop - s.start,), generator=gen, device="cuda", dtype=torch.int32)
        grad[s, 0] = torch.randint(-1, 2, (s.stop - s.start,), generator=gen, device="cuda", dtype=torch.int8).to(BF16)
    rows = n // length  # what is behind them belongs to no row
    offsets = torch.arange(rows + 1, device="cuda", dtype=torch.int32) * length
    tokens = nvtext.DeviceListColumn(offsets, ids, None, rows, 0, np.dtype(np.int32), n)
    inside = rows * length
    want_tokens = torch.zeros(vocabulary + 1, device="cuda", dtype=torch.float64)
    for s in pieces:
        s = slice(s.start, min(s.stop, inside))
        want_tokens += torch.bincount(ids[s] + 1, grad[s, 0].double(), vocabulary + 1)
    want_places = grad[:inside, 0].view(rows, length)[:, :places].double().sum(0)
    got_tokens, got_places = encoder.embedding_backward(tokens, grad, vocabulary, places, dtype=F32)
    assert torch.equal(got_tokens[:, 0].double(), want_tokens[1:]) and torch.equal(got_places[:, 0].double(), want_places)
    del grad
    table, positions = whole((vocabulary, 1), BF16, 6, 9), whole((length, 1), BF16, 7, 9)
    got = encoder.embedding(tokens, table, positions)
    at = torch.arange(2**26, device="cuda") % length
    for s in pieces:
        count = s.stop - s.start
        want = torch.where(ids[s] >= 0, table[ids[s].clamp(min=0).long(), 0], 0.0) + positions[at[:count], 0]
        if s.stop > inside:
            want[inside - s.start:] = 0
        assert torch.equal(got[s, 0], want)


# ------------------------------------------------------------------ launches of 2^32 threads and more

def poison(*bytes_each):
    """What is allocated next has held NaN: a result that is not written shows."""
    torch.cuda.empty_cache()
    held = [torch.full((n // 4,), float("nan"), device="cuda") for n in bytes_each]
    torch.cuda.synchronize()
    del held


def test_embedding_backward_of_many_places():
    rows, places, width = 32769, 131072, 1024
    tokens = nvtext.DeviceListColumn(torch.arange(rows + 1, device="cuda", dtype=torch.int32), torch.zeros(rows, device="cuda", dtype=torch.int32), None, rows, 0,
                                     np.dtype(np.int32), rows)
    grad = whole((rows, width), F32, 1)
    poison(places * width * 4, 3 * width * 4, 16 * places * width * 4 + 2**26)
    got_tokens, got_places = encoder.embedding_backward(tokens, grad, 3, places)
    want = grad.double().sum(0).float()
    assert torch.equal(got_places[0], want) and (got_places[1:] == 0).all()
    assert torch.equal(got_tokens[0], want) and (got_tokens[1:] == 0).all()


def test_linear_of_many_rows_that_are_copied():
    m, k = 2**31 + 5, 9
    w, b = whole((1, k), BF16, 1), whole((1,), BF16, 2)
    x = torch.empty(m, k, device="cuda", dtype=BF16)
    pieces = [slice(i, min(i + 2**25, m)) for i in range(0, m, 2**25)]
    for i, s in enumerate(pieces):
        x[s] = whole((s.stop - s.start, k), BF16, i)
    poison(m * 2, m * 32)
    got = encoder.linear(x, w, b)
    for s in pieces:
        assert torch.equal(got[s, 0], ((x[s] * w).float().sum(1) + b.float()).to(BF16))


def test_linear_of_many_rows():
    m = 2**31 + 400
    x = torch.arange(m, device="cuda", dtype=torch.int8).float().view(m, 1)
    w, b = torch.full((1, 1), 3.0, device="cuda"), torch.ones(1, device="cuda")
    poison(m * 4)
    got = encoder.linear(x, w, b)
    for i in range(0, m, 2**27):
        assert torch.equal(got[i:i + 2**27], x[i:i + 2**27] * 3 + 1)


def test_linear_of_many_outputs():
    n = 2**28 + 40
    b = whole((n,), BF16, 1, 9)
    poison(n * 2)
    assert torch.equal(encoder.linear(torch.empty(1, 0, device="cuda", dtype=BF16), torch.empty(n, 0, device="cuda", dtype=BF16), b)[0], b)


def test_linear_backward_of_a_row_of_many_inputs():
    k = 2**30 + 200
    x, w, g = whole((1, k), BF16, 1), whole((1, k), BF16, 2), torch.full((1, 1), 3.0, device="cuda", dtype=BF16)
    poison(k * 2, k * 2)
    dx, dw, db = encoder.linear_backward(g, x, w)
    assert torch.equal(dx, w * 3) and torch.equal(dw, x * 3) and db.item() == 3


def test_layer_norm_backward_of_rows_of_many_values():
    rows, cols = 2, 2**29 + 100
    s, g, w = whole((rows, cols), BF16, 1), whole((rows, cols), BF16, 2), torch.ones(cols, device="cuda", dtype=BF16)
    saved = encoder.LayerNormSaved(s, torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda"))
    poison(cols * 4, cols * 2, cols * 2, 4 * cols * 4)
    _, _, dw, db = encoder.layer_norm_backward(g, saved, w)
    for i in range(0, cols, 2**27):
        j = slice(i, i + 2**27)
        assert torch.equal(dw[j], (g[:, j] * s[:, j]).sum(0)) and torch.equal(db[j], g[:, j].sum(0))


# ------------------------------------------------------------------ the same values elsewhere

def elsewhere(t):
    """The same values, one value further on and with one value between the rows."""
    far = torch.empty(t.shape[0], t.shape[1] + 1, device="cuda", dtype=t.dtype)[:, 1:]
    return far.copy_(t)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k,n", [(1, 4096, 1024), (16, 4096, 1024), (17, 1024, 4096), (32, 2304, 1024), (48, 1536, 1003), (64, 1024, 512), (64, 2056, 300), (65, 1024, 64), (200, 768, 512),
                                   (300, 1003, 264)])
def test_results_do_not_depend_on_where_matrices_lie(m, k, n, dtype):
    gen = torch.Generator("cuda").manual_seed(m + k)
    x, w, g = (torch.randn(s, generator=gen, device="cuda").to(dtype) for s in ((m, k), (n, k), (m, n)))
    b = torch.randn(n, generator=gen, device="cuda").to(dtype)
    fx, fw, fg = elsewhere(x), elsewhere(w), elsewhere(g)
    for one, other in zip(encoder.linear(x, w, b, "gelu", g, keep=True), encoder.linear(fx, fw, b, "gelu", fg, keep=True)):
        assert torch.equal(one, other)
    for activation in ("none", "silu"):
        for one, other in zip(encoder.linear_backward(g, x, w, activation, g), encoder.linear_backward(fg, fx, fw, activation, fg)):
            assert torch.equal(one, other)
    scale = torch.randn(k, generator=gen, device="cuda").to(dtype)
    (one, saved), (other, far) = (encoder.layer_norm(a, scale, scale, residual=a, p=0.2, seed=1, keep=True) for a in (x, fx))
    assert torch.equal(one, other) and all(torch.equal(u, v) for u, v in zip(saved, far))
    for one, other in zip(*(encoder.layer_norm_backward(a, encoder.LayerNormSaved(s, saved.mean, saved.rstd), scale, 0.2, 1) for a, s in ((x, saved.sum), (fx, elsewhere(saved.sum))))):
        assert torch.equal(one, other)
    ids = (torch.arange(m, device="cuda") % 7).int()
    tokens = nvtext.DeviceListColumn(torch.tensor([0, m // 3, m], device="cuda", dtype=torch.int32), ids, None, 2, 0, np.dtype(np.int32), m)
    for one, other in zip(encoder.embedding_backward(tokens, x, 9, 5), encoder.embedding_backward(tokens, fx, 9, 5)):
        assert torch.equal(one, other)
    assert torch.equal(encoder.embedding(tokens, w[:7], w[:5]), encoder.embedding(tokens, fw[:7], fw[:5])) and torch.equal(encoder.dropout(x, 0.3, 2), encoder.dropout(fx, 0.3, 2))
