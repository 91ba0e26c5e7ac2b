"""The encoder operators' kernels against their definitions in 64 bits.

How far a value may be off follows from the arithmetic: u is half the distance from 1 to the next value of the result's
type (the one rounding at the end), and what is held in 32 bits is off by 2^-24 of the magnitudes that were added up, times
the longest chain of additions.  Matrix instructions may cut off where others round, so products count twice.
"""
import numpy as np
import pytest
import torch

from cudf_amd import encoder, nvtext
from oracle import encoder_py as orc

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
UNIT = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}
TINY = {F32: 2.0**-149, F16: 2.0**-24, BF16: 2.0**-133}  # results below the smallest normal number
EPS = 2.0**-24
TYPES = [F32, F16, BF16]
ACTIVATIONS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def make(rng, shape, dtype, scale=1.0, mean=0.0, pad=0):
    """A tensor on the device and its values in 64 bits; pad: rows lie that many values further apart."""
    a = rng.standard_normal(tuple(shape[:-1]) + (shape[-1] + pad,)) * scale + mean
    t = torch.from_numpy(a).to(dtype).cuda()
    t = t[..., pad // 2: pad // 2 + shape[-1]] if pad else t
    return t, t.double().cpu().numpy()


def near(got, want, size, chain, dtype=None, twice=1):
    """got within what its type and `chain` additions of magnitude `size` allow of want."""
    dtype = dtype or got.dtype
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    off = np.abs(got - want)
    most = UNIT[dtype] * np.abs(want) * (1 + UNIT[dtype]) + twice * (chain + 2) * EPS * size * 1.01 + TINY[dtype]
    assert np.isfinite(got).all()
    worst = np.unravel_index(np.argmax(off - most), off.shape) if off.size else ()
    assert (off <= most).all(), f"at {worst}: {got[worst]} for {want[worst]}, off {off[worst]:.3g}, at most {most[worst]:.3g}"


def column(offsets, ids):
    return nvtext.DeviceListColumn(torch.tensor(offsets, dtype=torch.int32).cuda().view(torch.uint8), torch.tensor(ids, dtype=torch.int32).cuda().view(torch.uint8),
                                   None, len(offsets) - 1, 0, np.dtype(np.int32), len(ids))


def ragged(rng, rows, tokens, vocabulary):
    """Offsets with empty rows among them, and ids of which some are no entries and one makes up a third."""
    cuts = np.sort(rng.integers(0, tokens + 1, rows - 1)) if rows > 1 else np.zeros(0, np.int64)
    offsets = np.concatenate([[0], cuts, [tokens]]).astype(np.int32)
    ids = rng.integers(0, vocabulary, tokens)
    ids = np.where(rng.random(tokens) < 0.3, vocabulary // 2, ids)
    ids = np.where(rng.random(tokens) < 0.05, rng.choice([-1, vocabulary, -(2**31), 2**31 - 1], tokens), ids).astype(np.int32)
    return offsets, ids


# ------------------------------------------------------------------ embedding

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,tokens,vocabulary,places,width,pad", [
    (1, 1, 1, 1, 1, 0), (3, 70, 11, 5, 768, 0), (40, 333, 1000, 512, 129, 0), (5, 65, 7, 64, 1031, 3), (300, 100, 50, 2, 64, 8), (2, 5000, 300, 2000, 24, 0),
    (1, 3, 40, 0, 2056, 0),
])
def test_embedding(dtype, rows, tokens, vocabulary, places, width, pad):
    rng = np.random.default_rng(tokens)
    offsets, ids = ragged(rng, rows, tokens, vocabulary)
    table, t64 = make(rng, (vocabulary, width), dtype, pad=pad)
    positions, p64 = make(rng, (places, width), dtype, pad=pad) if places else (None, None)
    want, size = orc.embedding(offsets, ids, t64, p64)
    near(encoder.embedding(column(offsets, ids), table, positions), want, size, 1)


def test_embedding_of_values_outside_all_rows():
    rng = np.random.default_rng(5)
    table, t64 = make(rng, (9, 40), F32)
    positions, p64 = make(rng, (3, 40), F32)
    offsets, ids = [4, 4, 9, 20], rng.integers(0, 9, 25)
    got = encoder.embedding(column(offsets, ids), table, positions)
    near(got, *orc.embedding(np.array(offsets), ids, t64, p64), 1)
    assert (got[:4] == 0).all() and (got[20:] == 0).all()
    grad, g64 = make(rng, (25, 40), F32)
    (dt, dp), (st, sp) = orc.embedding_backward(np.array(offsets), ids, g64, 9, 3)
    got_t, got_p = encoder.embedding_backward(column(offsets, ids), grad, 9, 3)
    near(got_t, dt, st, 25)
    near(got_p, dp, sp, 25)


def test_embedding_without_tokens():
    table, positions = torch.ones(5, 8, device="cuda"), torch.ones(3, 8, device="cuda")
    for offsets in ([0], [0, 0, 0]):
        c = column(offsets, [])
        assert encoder.embedding(c, table, positions).shape == (0, 8)
        t, p = encoder.embedding_backward(c, torch.empty(0, 8, device="cuda"), 5, 3)
        assert (t == 0).all() and (p == 0).all() and t.shape == (5, 8) and p.shape == (3, 8)


def test_embedding_of_the_tokenizers_result():
    from cudf_amd.arrow_host import HostStringsColumn
    vocabulary = ["[PAD]", "a", "bc", "##d", "e"]
    words = nvtext.WordPieceVocabulary(nvtext.DeviceStringsColumn.from_host(HostStringsColumn.from_pylist(vocabulary)))
    text = nvtext.DeviceStringsColumn.from_host(HostStringsColumn.from_pylist(["a bcd e", None, "", "zz a", "e"]))
    tokens = nvtext.wordpiece_tokenize(text, words)
    host = tokens.to_host()
    assert -1 in host.child  # no [UNK] in this vocabulary
    rng = np.random.default_rng(6)
    table, t64 = make(rng, (5, 96), BF16)
    positions, p64 = make(rng, (2, 96), BF16)
    near(encoder.embedding(tokens, table, positions), *orc.embedding(host.offsets, host.child, t64, p64), 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,tokens,vocabulary,places,width,pad", [
    (1, 1, 1, 1, 1, 0), (3, 70, 11, 5, 768, 0), (40, 333, 1000, 512, 129, 0), (5, 65, 7, 64, 1031, 3), (300, 100, 50, 2, 64, 8), (2, 5000, 300, 2000, 24, 0),
    (1, 3, 40, 0, 2056, 0), (7, 2048, 255, 3, 40, 0), (7, 2049, 256, 3, 40, 0), (900, 9000, 70000, 30, 8, 0), (5000, 20000, 3000, 9, 260, 0), (40000, 50000, 100, 6, 4, 0),
    (60, 8192, 3, 200, 3, 1), (60, 8193, 70000, 200, 5, 0), (3, 64, 2, 64, 4, 0), (3, 65, 1, 64, 300, 0), (3, 128, 5, 64, 2, 0),
])
def test_embedding_backward(dtype, rows, tokens, vocabulary, places, width, pad):
    rng = np.random.default_rng(tokens + 1)
    offsets, ids = ragged(rng, rows, tokens, vocabulary)
    grad, g64 = make(rng, (tokens, width), dtype, pad=pad)
    (dt, dp), (st, sp) = orc.embedding_backward(offsets, ids, g64, vocabulary, places)
    most = int(max(np.bincount(np.clip(ids, 0, vocabulary - 1)).max(), rows))
    for result in {dtype, F32}:
        got_t, got_p = encoder.embedding_backward(column(offsets, ids), grad, vocabulary, places, dtype=result)
        near(got_t, dt, st, most)
        if places:
            near(got_p, dp, sp, most)
        else:
            assert got_p is None
        again = encoder.embedding_backward(column(offsets, ids), grad, vocabulary, places, dtype=result)
        assert torch.equal(got_t, again[0]) and (not places or torch.equal(got_p, again[1]))


def test_embedding_backward_of_many_tokens():
    """More tiles than a workgroup adds up the counts of: in whole numbers, so that every sum is exact."""
    n, vocabulary, width = 256 * 2048 + 77, 300, 4
    rng = np.random.default_rng(4)
    ids = rng.integers(-1, vocabulary, n).astype(np.int32)
    offsets = np.arange(0, n + 1, 7, dtype=np.int32)
    g = rng.integers(-4, 5, (n, width)).astype(np.float32)
    dt, dp = encoder.embedding_backward(column(offsets, ids), torch.from_numpy(g).cuda(), vocabulary, 8)
    rows, inside = len(offsets) - 1, int(offsets[-1])
    want = np.stack([np.bincount(ids[:inside][ids[:inside] >= 0], g[:inside, k][ids[:inside] >= 0], vocabulary) for k in range(width)], 1)
    assert (dt.cpu().numpy() == want).all()
    assert (dp.cpu().numpy() == np.concatenate([g[:inside].reshape(rows, 7, width).sum(0), np.zeros((1, width))])).all()


def whole_numbers(tokens, vocabulary, width=4, length=7):
    """Gradients in whole numbers, so that every sum is exact."""
    rng = np.random.default_rng(tokens + vocabulary)
    ids = rng.integers(-1, vocabulary, tokens).astype(np.int32)
    ids[:2] = vocabulary - 1, 0
    offsets = np.arange(0, tokens + 1, length, dtype=np.int32)
    g = rng.integers(-4, 5, (tokens, width)).astype(np.float32)
    dt, _ = encoder.embedding_backward(column(offsets, ids), torch.from_numpy(g).cuda(), vocabulary, 0)
    inside = int(offsets[-1])
    known = ids[:inside] >= 0
    want = np.stack([np.bincount(ids[:inside][known], g[:inside, k][known], vocabulary) for k in range(width)], 1)
    assert (dt.cpu().numpy() == want).all()


@pytest.mark.parametrize("vocabulary", [254, 255, 256, 511, 512, 1022, 1023, 1024, 65535, 65536, 262143, 262144, 1048575, 1048576])
@pytest.mark.parametrize("tokens", [700, 9001])
def test_embedding_backward_sizes_of_ids(vocabulary, tokens):
    """Around the sizes at which the sort takes other digits."""
    whole_numbers(tokens, vocabulary)


@pytest.mark.parametrize("vocabulary", [1000, 40000, 250000])
def test_embedding_backward_of_many_tokens_of_other_ids(vocabulary):
    whole_numbers(256 * 2048 + 2050, vocabulary)


@pytest.mark.parametrize("tokens", [15, 16, 17, 31, 32, 33, 32767, 32768, 32769])
@pytest.mark.parametrize("vocabulary", [1, 3])
def test_embedding_backward_around_chunks(tokens, vocabulary):
    whole_numbers(tokens, vocabulary, width=8, length=1)


# ------------------------------------------------------------------ dropout

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (1, 7, 0), (3, 8, 0), (5, 9, 0), (257, 129, 0), (64, 1024, 0), (33, 1021, 3), (2000, 16, 8)])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_dropout(dtype, rows, cols, pad, p):
    rng = np.random.default_rng(rows)
    x, x64 = make(rng, (rows, cols), dtype, pad=pad)
    seed, offset = (1 << 63) + 12345, 2**32 - 1
    m = orc.multipliers(rows, cols, p, seed, offset)
    got = encoder.dropout(x, p, seed, offset)
    near(got, orc.dropped(x64, m), np.abs(x64) * m, 1)
    assert ((got == 0).cpu().numpy() | (m > 0)).all()


def test_dropout_of_nothing_and_of_everything():
    x = torch.randn(9, 33, device="cuda")
    x[3, 4], x[5, 6] = float("nan"), float("inf")
    assert torch.equal(encoder.dropout(x, 0.0, 1).nan_to_num(7.0), x.nan_to_num(7.0))
    assert (encoder.dropout(x, 1.0, 1) == 0).all()
    kept = torch.from_numpy(orc.multipliers(9, 33, 0.5, 1, 0) > 0).cuda()
    y = encoder.dropout(torch.full((9, 33), float("nan"), device="cuda"), 0.5, 1)
    assert torch.equal(y.isnan(), kept) and (y[~kept] == 0).all()
    assert encoder.dropout(torch.empty(0, 5, device="cuda"), 0.5, 1).shape == (0, 5)
    assert encoder.dropout(torch.empty(5, 0, device="cuda"), 0.5, 1).shape == (5, 0)


def test_dropout_of_more_dimensions_is_that_of_its_rows():
    x = torch.randn(3, 4, 5, 21, device="cuda")
    assert torch.equal(encoder.dropout(x, 0.3, 5, 6).view(-1, 21), encoder.dropout(x.view(-1, 21), 0.3, 5, 6))
    assert torch.equal(encoder.dropout(x[0, 0, 0], 0.3, 5, 6), encoder.dropout(x[0, 0, :1], 0.3, 5, 6)[0])


# ------------------------------------------------------------------ layer norm

NORMS = [(1, 1, 0), (1, 1024, 0), (3, 7, 0), (5, 64, 0), (130, 129, 0), (9, 512, 0), (70, 768, 8), (33, 1021, 3), (6, 2048, 0), (5, 2056, 0), (3, 5000, 0), (4, 8192, 0),
         (2, 8200, 0), (3, 16384, 0), (2, 20011, 1), (2, 40000, 0), (2, 70001, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pad", NORMS)
@pytest.mark.parametrize("p,with_residual,w32", [(0.0, False, False), (0.0, True, True), (0.3, True, False), (0.3, False, True)])
def test_layer_norm(dtype, rows, cols, pad, p, with_residual, w32):
    rng = np.random.default_rng(cols)
    x, x64 = make(rng, (rows, cols), dtype, mean=0.5, pad=pad)
    r, r64 = make(rng, (rows, cols), dtype, pad=2 * pad) if with_residual else (None, None)
    w, w64 = make(rng, (cols,), F32 if w32 else dtype, mean=1.0)
    b, b64 = make(rng, (cols,), F32 if w32 else dtype)
    m = orc.multipliers(rows, cols, p, 77, 3)
    want, s, mean, rstd = orc.layer_norm(x64, w64, b64, 1e-5, r64, m)
    out, saved = encoder.layer_norm(x, w, b, 1e-5, r, p, 77, 3, keep=True)
    terms = np.abs(x64) * m + (np.abs(r64) if with_residual else 0.0)
    # the longest chain of additions in a row's sums: what one of 64 lanes takes, then the lanes and wavefronts
    chain = cols / 64 + 32
    assert saved.mean.shape == (rows,) and saved.mean.dtype == F32
    near(saved.sum, s, terms, 2)
    near(saved.mean, mean, terms.mean(1), chain)
    # the mean of squares: every (s - mean)^2 is off by twice |s - mean| times what s and the mean are off by, on top of the sum
    spread = np.abs(s - mean[:, None])
    off_s = 3 * terms + chain * terms.mean(1, keepdims=True)
    of_var = chain / rstd**2 + 2 * (spread * off_s).mean(1) + EPS * np.square(off_s).mean(1)
    of_rstd = 0.5 * rstd**3 * of_var + 4 * rstd
    near(saved.rstd, rstd, of_rstd, 0)
    size = np.abs(w64) * (rstd[:, None] * off_s + spread * of_rstd[:, None]) + 3 * np.abs(w64) * spread * rstd[:, None] + np.abs(b64) + np.abs(want)
    near(out, want, size, 0)
    alone = encoder.layer_norm(x, w, b, 1e-5, r, p, 77, 3)
    assert torch.equal(alone, out)


def test_layer_norm_of_equal_values():
    """Nothing left of a row but its mean: the bias comes out, and no division by zero."""
    x = torch.full((4, 300), 3.0, device="cuda", dtype=BF16)
    w, b = torch.randn(300, device="cuda"), torch.randn(300, device="cuda")
    out, saved = encoder.layer_norm(x, w, b, 1e-5, keep=True)
    assert torch.equal(out, b.to(BF16).expand(4, 300)) and (saved.mean == 3).all()
    assert saved.sum is x
    assert encoder.layer_norm(x[:0], w, b).shape == (0, 300)


def test_layer_norm_keeps_rows_apart():
    """A row of infinities or NaN makes no other row wrong."""
    x = torch.randn(64, 200, device="cuda")
    w, b = torch.ones(200, device="cuda"), torch.zeros(200, device="cuda")
    clean, s = encoder.layer_norm(x, w, b, keep=True)
    y = x.clone()
    y[7], y[20, 3] = float("inf"), float("nan")
    got, t = encoder.layer_norm(y, w, b, keep=True)
    others = [i for i in range(64) if i not in (7, 20)]
    assert torch.equal(got[others], clean[others]) and got[7].isnan().all() and got[20].isnan().all()
    g = torch.randn(64, 200, device="cuda")
    a, c = encoder.layer_norm_backward(g, s, w), encoder.layer_norm_backward(g, t, w)
    assert torch.equal(a[0][others], c[0][others])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pad", NORMS + [(3000, 64, 0), (2500, 1536, 0), (700, 2504, 0)])
@pytest.mark.parametrize("p,with_sum_grad,w32", [(0.0, False, False), (0.0, True, True), (0.3, True, False), (0.3, False, True)])
def test_layer_norm_backward(dtype, rows, cols, pad, p, with_sum_grad, w32):
    rng = np.random.default_rng(cols + 1)
    g, g64 = make(rng, (rows, cols), dtype, pad=pad)
    s, s64 = make(rng, (rows, cols), dtype, mean=0.5, pad=2 * pad)
    e, e64 = make(rng, (rows, cols), dtype, pad=pad) if with_sum_grad else (None, None)
    w, w64 = make(rng, (cols,), F32 if w32 else dtype, mean=1.0)
    mean = torch.from_numpy(s64.mean(1)).float().cuda()
    rstd = torch.from_numpy(1 / np.sqrt(s64.var(1) + 1e-5)).float().cuda()
    m = orc.multipliers(rows, cols, p, 78, 4)
    mean64, rstd64 = mean.double().cpu().numpy(), rstd.double().cpu().numpy()
    dx, ds, dw, db, size, size_w, size_b = orc.layer_norm_backward(g64, s64, mean64, rstd64, w64, e64, m)
    saved = encoder.LayerNormSaved(s, mean, rstd)
    got = encoder.layer_norm_backward(g, saved, w, p, 78, 4, e)
    chain = cols / 64 + 32
    # h = (s - mean) * rstd cancels: it is off by what s and the mean are of
    cancel = (np.abs(s64) + np.abs(mean64[:, None])) * rstd64[:, None]
    h = np.abs(s64 - mean64[:, None]) * rstd64[:, None]
    a = np.abs(g64 * w64)
    size = size + rstd64[:, None] * (cancel * (a * h).mean(1, keepdims=True) + h * (a * cancel).mean(1, keepdims=True))
    near(got[1], ds, size, chain + 8)
    near(got[0], dx, size * m, chain + 9)
    if p == 0:
        assert got[0] is got[1]
    assert got[2].dtype == w.dtype
    near(got[2], dw, size_w + np.abs(g64 * cancel).sum(0), rows + 8)
    near(got[3], db, size_b, rows)
    again = encoder.layer_norm_backward(g, saved, w, p, 78, 4, e)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


def test_layer_norm_backward_without_rows():
    w = torch.ones(40, device="cuda")
    empty = torch.empty(0, 40, device="cuda")
    saved = encoder.LayerNormSaved(empty, torch.empty(0, device="cuda"), torch.empty(0, device="cuda"))
    x, r, dw, db = encoder.layer_norm_backward(empty, saved, w)
    assert x.shape == (0, 40) and (dw == 0).all() and (db == 0).all()


def test_layer_norm_gradient_against_differences():
    """In 32 bits: with a step of 2^-6 a difference is off by the rounding of two sums over all values, 2^-24 * 64 of their
    magnitude, and by the step squared times a third derivative of some units a row."""
    rng = np.random.default_rng(8)
    x, _ = make(rng, (20, 96), F32)
    r, _ = make(rng, (20, 96), F32)
    w, _ = make(rng, (96,), F32, mean=1.0)
    b, _ = make(rng, (96,), F32)
    g, _ = make(rng, (20, 96), F32)
    _, saved = encoder.layer_norm(x, w, b, 1e-5, r, 0.3, 5, 6, keep=True)
    grads = encoder.layer_norm_backward(g, saved, w, 0.3, 5, 6)
    h = 2.0**-6
    for i, (value, grad) in enumerate(zip((x, r, w, b), grads)):
        v = torch.from_numpy(rng.standard_normal(tuple(value.shape))).float().cuda()

        def loss(step):
            args = [x, w, b, r]
            at = [0, 3, 1, 2][i]
            args[at] = value + step * v
            return (encoder.layer_norm(args[0], args[1], args[2], 1e-5, args[3], 0.3, 5, 6).double() * g.double()).sum()
        want = (grad.double() * v.double()).sum().item()
        got = ((loss(h) - loss(-h)) / (2 * h)).item()
        size = (grad.double() * v.double()).abs().sum().item()
        assert abs(got - want) <= size * (2.0**-18 / h + 8 * h * h)


# ------------------------------------------------------------------ linear

# tokens, inputs, outputs, padding of the rows
PRODUCTS = [(1, 1, 1, 0), (1, 1024, 64, 0), (1, 77, 333, 0), (2, 256, 48, 8), (3, 130, 17, 3), (5, 4096, 96, 0), (8, 64, 200, 0), (15, 33, 31, 1), (16, 512, 128, 0), (17, 96, 40, 8),
            (31, 1000, 64, 0), (64, 64, 64, 0), (1, 2100, 40, 0), (20, 2051, 33, 3), (50, 2304, 24, 0), (40, 2048, 4200, 0), (65, 65, 65, 1), (100, 31, 260, 0), (128, 256, 128, 0), (129, 264, 136, 8), (255, 72, 257, 0), (256, 128, 512, 0), (300, 40, 300, 4),
            (513, 200, 520, 0), (700, 1032, 72, 0), (1, 8, 1000, 0), (2000, 16, 24, 0), (640, 320, 768, 0), (40, 2051, 24, 0)]
# how much larger a slope than 1 an activation has, and what its own evaluation is off by, in units of 2^-24 of |z| + |result|
STEEP = 1.15
OWN = 16


def check_linear(dtype, m, k, n, pad, activation, with_bias, with_residual, keep, seed=0):
    rng = np.random.default_rng(m * 7 + n + seed)
    x, x64 = make(rng, (m, k), dtype, pad=pad)
    w, w64 = make(rng, (n, k), dtype, scale=k**-0.5, pad=2 * pad)
    b, b64 = make(rng, (n,), dtype) if with_bias else (None, None)
    r, r64 = make(rng, (m, n), dtype, pad=pad) if with_residual else (None, None)
    want, z, size = orc.linear(x64, w64, b64, activation, r64)
    got = encoder.linear(x, w, b, activation, r, keep=keep)
    if keep:
        got, got_z = got
        near(got_z, z, size, k + 1, twice=2)
    most = size * STEEP * 2 * (k + 3) + OWN * (np.abs(z) + np.abs(want)) + (2 * np.abs(r64) if with_residual else 0.0)
    near(got, want, most, -1)  # (the chain is in `most`)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n,pad", PRODUCTS)
def test_linear(dtype, m, k, n, pad):
    check_linear(dtype, m, k, n, pad, "none", True, False, False)
    check_linear(dtype, m, k, n, pad, "gelu", True, True, True)
    check_linear(dtype, m, k, n, pad, "relu", False, True, False)


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("m", [1, 70, 300])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_activations(activation, m, dtype):
    check_linear(dtype, m, 72, 88, 0, activation, True, False, True)
    check_linear(dtype, m, 72, 88, 0, activation, False, True, True)


def test_activations_far_from_zero():
    """Where exp and tanh run out of range: the limits, no NaN."""
    x = torch.tensor([[-1e4, -300.0, -90.0, -20.0, 0.0, 20.0, 90.0, 300.0, 1e4]], device="cuda").t().contiguous()
    one = torch.ones(1, 1, device="cuda")
    for activation in ACTIVATIONS[1:]:
        y, z = encoder.linear(x, one, None, activation, keep=True)
        assert torch.equal(z, x) and y.isfinite().all()
        assert torch.equal(y[5:], x[5:]) and (y[:3].abs() < 1e-30).all() and y[4] == 0
        d = encoder.linear_backward(torch.ones_like(x), x, one, activation, z)[0]
        assert d.isfinite().all() and (d[5:] == 1).all() and (d[:3].abs() < 1e-30).all()


def test_linear_keeps_rows_apart():
    """A row of NaN stays in its row."""
    for m, k, n in ((5, 100, 40), (200, 136, 150)):
        x, w = torch.randn(m, k, device="cuda", dtype=BF16), torch.randn(n, k, device="cuda", dtype=BF16)
        y = x.clone()
        y[3] = float("nan")
        clean, got = encoder.linear(x, w), encoder.linear(y, w)
        others = [i for i in range(m) if i != 3]
        assert torch.equal(clean[others], got[others]) and got[3].isnan().all()


def test_linear_without_values():
    x, w, b = torch.empty(4, 0, device="cuda"), torch.empty(5, 0, device="cuda"), torch.randn(5, device="cuda")
    assert torch.equal(encoder.linear(x, w, b), b.expand(4, 5))
    assert encoder.linear(torch.empty(0, 3, device="cuda"), torch.ones(5, 3, device="cuda")).shape == (0, 5)
    dx, dw, db = encoder.linear_backward(torch.empty(0, 5, device="cuda"), torch.empty(0, 3, device="cuda"), torch.ones(5, 3, device="cuda"))
    assert dx.shape == (0, 3) and (dw == 0).all() and (db == 0).all()
    dx, dw, db = encoder.linear_backward(torch.ones(4, 0, device="cuda"), torch.ones(4, 3, device="cuda"), torch.empty(0, 3, device="cuda"))
    assert (dx == 0).all() and dx.shape == (4, 3) and dw.shape == (0, 3)


def test_linear_into_its_residual():
    """The C interface lets out be the residual."""
    import ctypes  # noqa: F401
    from cudf_amd import _capi
    for m, k, n in ((3, 64, 96), (300, 72, 200)):
        x, w, r = (torch.randn(s, device="cuda", dtype=BF16) for s in ((m, k), (n, k), (m, n)))
        want = encoder.linear(x, w, None, "silu", r)
        a, b, c = encoder._matrix(x, "x"), encoder._matrix(w, "w"), encoder._matrix(r, "r")
        assert _capi.load().nvtext_amd_linear(a, b, None, 4, c, nvtext._stream_handle(), nvtext._mr().struct, c, None) == _capi.SUCCESS
        assert torch.equal(r, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n,pad", PRODUCTS + [(3000, 64, 72, 0), (5001, 40, 33, 0), (1500, 264, 256, 8)])
@pytest.mark.parametrize("activation", ["none", "gelu"])
def test_linear_backward(dtype, m, k, n, pad, activation):
    rng = np.random.default_rng(m * 5 + n)
    g, g64 = make(rng, (m, n), dtype, pad=pad)
    x, x64 = make(rng, (m, k), dtype, pad=pad)
    w, w64 = make(rng, (n, k), dtype, scale=k**-0.5, pad=2 * pad)
    z, z64 = make(rng, (m, n), dtype, pad=pad) if activation != "none" else (None, None)
    got = encoder.linear_backward(g, x, w, activation, z)
    wants, sizes = orc.linear_backward(g64, x64, w64, activation, z64)
    # d is rounded to the matrices' type before it is multiplied; the slope's own evaluation is OWN units of |grad|
    rounding = UNIT[dtype] if activation != "none" else 0.0
    own = (OWN * EPS) if activation != "none" else 0.0
    slack = np.abs(g64) * own + TINY[dtype]
    offs = (slack @ np.abs(w64), slack.T @ np.abs(x64), slack.sum(0))
    for value, want, size, off, chain, rounded in zip(got, wants, sizes, offs, (n, m, m), (rounding, rounding, 0.0)):
        near(value, want, size * (2 * (chain + 3) + rounded * 1.01 / EPS) + off / EPS, -1)
    again = encoder.linear_backward(g, x, w, activation, z)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


# few rows and many outputs or inputs, which are cut into parts; the most rows that are few, and one more
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,k,n,pad", [(7, 64, 6400, 0), (33, 100, 3001, 1), (48, 3000, 70, 0), (63, 130, 2049, 3), (64, 72, 64, 8), (96, 200, 1500, 0), (127, 9, 700, 1), (128, 1000, 1048, 0),
                                       (128, 1024, 1032, 0), (100, 1101, 1003, 0)])
@pytest.mark.parametrize("activation", ["none", "relu", "gelu_tanh", "silu"])
def test_linear_backward_few_rows(dtype, m, k, n, pad, activation):
    test_linear_backward(dtype, m, k, n, pad, activation)


@pytest.mark.parametrize("activation", ACTIVATIONS[1:])
def test_linear_backward_activations(activation):
    rng = np.random.default_rng(12)
    g, g64 = make(rng, (70, 40), F32)
    x, x64 = make(rng, (70, 24), F32)
    w, w64 = make(rng, (40, 24), F32)
    z, z64 = make(rng, (70, 40), F32, scale=3.0)
    got = encoder.linear_backward(g, x, w, activation, z)
    wants, sizes = orc.linear_backward(g64, x64, w64, activation, z64)
    slack = np.abs(g64) * OWN * (1 + np.abs(z64))
    offs = (slack @ np.abs(w64), slack.T @ np.abs(x64), slack.sum(0))
    for value, want, size, off, chain in zip(got, wants, sizes, offs, (40, 70, 70)):
        near(value, want, size * 2 * (chain + 3) + off, -1)


def test_linear_gradient_against_differences():
    """linear is linear in x, weight and bias: a difference over a whole step is exact but for rounding."""
    rng = np.random.default_rng(9)
    x, _ = make(rng, (50, 72), F32)
    w, _ = make(rng, (40, 72), F32)
    b, _ = make(rng, (40,), F32)
    g, _ = make(rng, (50, 40), F32)
    grads = encoder.linear_backward(g, x, w)
    for i, (value, grad) in enumerate(zip((x, w, b), grads)):
        v = torch.from_numpy(rng.standard_normal(tuple(value.shape))).float().cuda()
        args = [x, w, b]
        losses = []
        for step in (1.0, -1.0):
            args[i] = value + step * v
            losses.append((encoder.linear(*args).double() * g.double()).sum().item())
        want = (grad.double() * v.double()).sum().item()
        size = (encoder.linear(x.abs(), w.abs(), b.abs()).double() * g.abs().double()).sum().item() + (grad.abs() * v.abs()).double().sum().item()
        assert abs((losses[0] - losses[1]) / 2 - want) <= size * 2 * 80 * EPS * 4


# ------------------------------------------------------------------ all

def test_on_another_stream():
    """Calls go to the current stream, and their temporaries with them."""
    rng = np.random.default_rng(10)
    x, _ = make(rng, (300, 256), BF16)
    w, _ = make(rng, (512, 256), BF16)
    g, _ = make(rng, (300, 512), BF16)
    offsets, ids = ragged(rng, 20, 300, 50)
    c = column(offsets, ids)

    def calls():
        lw = w[0].contiguous()
        y, saved = encoder.layer_norm(x, lw, lw, p=0.2, seed=3, keep=True)
        return [encoder.linear(x, w, None, "gelu"), *encoder.linear_backward(g, x, w), encoder.dropout(x, 0.4, 9), y, *encoder.layer_norm_backward(x, saved, lw, 0.2, 3),
                *encoder.embedding_backward(c, x, 50, 7), encoder.embedding(c, w[:50], w[:7])]
    want = calls()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = calls()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_more_dimensions_and_other_strides():
    """Tensors of more dimensions are taken as the rows of their last; results are contiguous whatever the strides."""
    big = torch.randn(3, 5, 4, 96, device="cuda", dtype=F16)
    w, b = torch.randn(64, 64, device="cuda", dtype=F16), torch.randn(64, device="cuda", dtype=F16)
    x = big[:, :, :, 16:80]
    flat = x.reshape(60, 64)
    y, z = encoder.linear(x, w, b, "silu", x, keep=True)
    y2, z2 = encoder.linear(flat, w, b, "silu", flat, keep=True)
    assert y.shape == x.shape and y.is_contiguous() and torch.equal(y.view(60, 64), y2) and torch.equal(z.view(60, 64), z2)
    for a, c in zip(encoder.linear_backward(x, x, w, "silu", z), encoder.linear_backward(flat, flat, w, "silu", z2)):
        assert torch.equal(a.reshape(c.shape), c)
    n, saved = encoder.layer_norm(x, b, b, p=0.2, seed=1, residual=x, keep=True)
    n2, saved2 = encoder.layer_norm(flat, b, b, p=0.2, seed=1, residual=flat, keep=True)
    assert torch.equal(n.view(60, 64), n2) and saved.mean.shape == (3, 5, 4) and torch.equal(saved.rstd.view(60), saved2.rstd)
    for a, c in zip(encoder.layer_norm_backward(x, saved, b, 0.2, 1), encoder.layer_norm_backward(flat, saved2, b, 0.2, 1)):
        assert torch.equal(a.reshape(c.shape), c)
    with pytest.raises(RuntimeError):
        encoder.dropout(big.transpose(0, 1), 0.1, 1)  # rows that are not evenly spaced
    wide = torch.randn(8, 128, device="cuda")[:, :64]
    assert encoder.dropout(wide, 0.1, 1).is_contiguous() and torch.equal(encoder.dropout(wide, 0.1, 1), encoder.dropout(wide.contiguous(), 0.1, 1))


def test_refusals():
    x, w = torch.randn(4, 8, device="cuda"), torch.randn(5, 8, device="cuda")
    b8 = torch.ones(8, device="cuda")
    with pytest.raises(ValueError, match="one of"):
        encoder.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="float32, float16"):
        encoder.linear(x.double(), w.double())
    with pytest.raises(ValueError, match="device memory"):
        encoder.linear(x.cpu(), w)
    with pytest.raises(ValueError, match="last dimension"):
        encoder.linear(x.t().contiguous().t(), w)
    with pytest.raises(ValueError, match="vector"):
        encoder.linear(x, w, w)
    with pytest.raises(ValueError, match="inputs"):
        encoder.linear(x, w[:, :7])
    with pytest.raises(ValueError, match="one type"):
        encoder.linear(x, w.half())
    with pytest.raises(ValueError, match="applied to"):
        encoder.linear_backward(torch.randn(4, 5, device="cuda"), x, w, "gelu")
    with pytest.raises(ValueError, match="seed"):
        encoder.dropout(x, 0.1, -1)
    with pytest.raises(ValueError, match="offset"):
        encoder.dropout(x, 0.1, 1, 2**32)
    with pytest.raises(ValueError, match="p must"):
        encoder.dropout(x, 1.1, 1)
    with pytest.raises(ValueError, match="weight"):
        encoder.layer_norm(x, b8[:7], b8)
    with pytest.raises(ValueError, match="mean and rstd"):
        encoder.layer_norm_backward(x, encoder.LayerNormSaved(x, b8, b8), b8)
    with pytest.raises(ValueError, match="sizes"):
        encoder.embedding_backward(column([0, 4], [1, 2, 3, 4]), x, -1)
    with pytest.raises(ValueError, match="INT32"):
        c = column([0, 4], [1, 2, 3, 4])
        c.child_dtype = np.dtype(np.uint32)
        encoder.embedding(c, w)


def test_no_memory_for_temporaries():
    mr = nvtext._mr()
    x, w, g = torch.randn(300, 64, device="cuda"), torch.randn(50, 64, device="cuda"), torch.randn(300, 50, device="cuda")
    live = len(mr.live)
    mr.fail_after = 0
    try:
        with pytest.raises(MemoryError):
            encoder.linear_backward(g, x, w, "relu", g)
        with pytest.raises(MemoryError):
            encoder.layer_norm_backward(x, encoder.LayerNormSaved(x, x[:, 0].contiguous(), x[:, 0].contiguous()), w[0])
        with pytest.raises(MemoryError):
            encoder.embedding_backward(column([0, 300], [1] * 300), x, 5)
    finally:
        mr.fail_after = None
    assert len(mr.live) == live


# rows that one workgroup goes through alone, one round more and less, at each number of lanes
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(191, 100), (192, 128), (193, 127), (95, 250), (96, 256), (97, 129), (47, 600), (48, 1024), (49, 2047), (12, 4000), (13, 8191), (6, 16000), (7, 16383)])
def test_layer_norm_backward_around_one_workgroup(dtype, rows, cols):
    test_layer_norm_backward(dtype, rows, cols, 0, 0.3, True, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [3, 70])
def test_rows_far_apart(dtype, m):
    """Values more than 2^31 values (and 2^32 bytes) from the first: what the same rows next to each other give."""
    stride, width = 2**31 // (m - 1) + 24, 72
    far = torch.empty(stride * (m - 1) + 2 * width, device="cuda", dtype=dtype)

    def spread(rows, at):
        view = far.as_strided((rows.shape[0], rows.shape[1]), (stride, 1), at)
        view.copy_(rows)
        return view
    x, g = torch.randn(m, width, device="cuda", dtype=dtype), torch.randn(m, width, device="cuda", dtype=dtype)
    w, b = torch.randn(width, width, device="cuda", dtype=dtype) * 0.1, torch.randn(width, device="cuda", dtype=dtype)
    fx, fg = spread(x, 0), spread(g, width)
    offsets, ids = np.array([0, m], np.int32), np.arange(m)[::-1].astype(np.int32)
    tokens = column(offsets, ids)

    def same(a, c):
        for u, v in zip(a, c):
            assert torch.equal(u, v)
    same([encoder.dropout(fx, 0.3, 5)], [encoder.dropout(x, 0.3, 5)])
    same([encoder.embedding(tokens, fx, fg)], [encoder.embedding(tokens, x, g)])
    same(encoder.embedding_backward(tokens, fx, 100, 3), encoder.embedding_backward(tokens, x, 100, 3))
    n, s = encoder.layer_norm(fx, b, b, residual=fg, p=0.2, seed=1, keep=True)
    n2, s2 = encoder.layer_norm(x, b, b, residual=g, p=0.2, seed=1, keep=True)
    same([n, *s], [n2, *s2])
    same(encoder.layer_norm_backward(fg, encoder.LayerNormSaved(fx, s.mean, s.rstd), b, 0.2, 1), encoder.layer_norm_backward(g, encoder.LayerNormSaved(x, s.mean, s.rstd), b, 0.2, 1))
    same(encoder.linear(fx, w, b, "gelu", fg, keep=True), encoder.linear(x, w, b, "gelu", g, keep=True))
    same([encoder.linear(w, fx)], [encoder.linear(w, x)])
    same(encoder.linear_backward(fg, fx, w, "silu", fx), encoder.linear_backward(g, x, w, "silu", x))
