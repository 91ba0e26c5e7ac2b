"""Every form of the encoder's kernels at sizes that take it: products by their plans, loops by more work than one turn does.

Products are of whole numbers whose sums stay below 2^24: every sum is exact in any order, and a result may differ from the
formula by nothing but its one rounding.  Which form a call took is read from the library's timing record, so that a plan fitted anew
cannot leave a form without a test unnoticed.
"""
import pytest
import torch

from cudf_amd import _capi, encoder, nvtext
from tests import test_encoder_gpu as checks
from tests.test_encoder_limits_gpu import whole

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def launches(call):
    """(the call's result, the names of its kernels in the order of their launches)"""
    _capi.profile_enable(True)
    _capi.profile_read()
    try:
        result = call()
        return result, [name for name, _ in _capi.profile_read()]
    finally:
        _capi.profile_enable(False)


def turns(edge, m, n):
    """Tiles of edge (256: square, 128: square, 64: 128 rows) per workgroup that runs at a time."""
    rows, cols = max(edge, 128), edge
    tiles = -(-m // rows) * -(-n // cols)
    return tiles / (torch.cuda.get_device_properties(0).multi_processor_count * (1 if edge == 256 else 2))


# tokens, inputs, outputs; rows of a tile's edge, whether a workgroup takes several tiles, whether k is cut into parts
FORWARD = [
    ((4490, 72, 5000), 256, True, False), ((4487, 75, 4999), 256, True, False), ((2051, 72, 6150), 256, False, False), ((2051, 4104, 2051), 256, False, True),
    ((260, 520, 6150), 128, False, False), ((4090, 1003, 4490), 128, True, False), ((129, 4104, 4490), 128, False, True),
    ((2051, 72, 2051), 64, True, False), ((100, 72, 100), 64, False, False), ((129, 2051, 4090), 64, False, True), ((100, 1003, 100), 64, False, True),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes,edge,several,cut", FORWARD)
def test_linear_in_every_tile(sizes, edge, several, cut, dtype):
    m, k, n = sizes
    x, w, b, r = whole((m, k), dtype, 1), whole((n, k), dtype, 2), whole((n,), dtype, 3, 9), whole((m, n), dtype, 4, 9)
    (out, z), names = launches(lambda: encoder.linear(x, w, b, "relu", r, keep=True))
    assert names == (["linear_prepare"] if k % 8 else []) + [f"linear_tiles_{edge}"] + (["linear_join"] if cut else [])
    assert cut or (turns(edge, m, n) > 1) == several
    want = x.double() @ w.double().t() + b.double()
    assert torch.equal(z, want.to(dtype)) and torch.equal(out, (want.clamp(min=0) + r.double()).to(dtype))


@pytest.mark.parametrize("sizes,edge,cut", [((129, 520, 4490), 128, True), ((260, 72, 6150), 128, False), ((129, 1003, 2051), 128, True), ((100, 72, 100), 64, False), ((129, 520, 4090), 64, True),
                                            ((3001, 75, 2953), 128, False)])
def test_linear_of_floats_in_every_tile(sizes, edge, cut):
    m, k, n = sizes
    x, w, b, r = whole((m, k), F32, 1), whole((n, k), F32, 2), whole((n,), F32, 3, 9), whole((m, n), F32, 4, 9)
    (out, z), names = launches(lambda: encoder.linear(x, w, b, "relu", r, keep=True))
    assert names == [f"linear_product_{edge}"] + (["linear_join"] if cut else [])
    want = x.double() @ w.double().t() + b.double()
    assert torch.equal(z, want.float()) and torch.equal(out, (want.clamp(min=0) + r.double()).float())


# tokens, inputs, outputs; the tiles of x's gradient and of the weight's, None: both in one launch
BACKWARD = [
    ((4090, 4104, 100), 256, 128), ((100, 4104, 4090), 128, 256), ((4090, 4104, 1003), 128, 256), ((1003, 4104, 4090), 256, 128), ((4100, 4104, 96), 256, 128), ((104, 4100, 4096), 128, 256),
    ((4200, 2056, 4300), 256, 256), ((4090, 4104, 1500), None, None), ((1500, 4104, 4090), None, None), ((129, 4104, 2051), 128, 256), ((129, 1500, 2056), None, None), ((513, 72, 104), None, None),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("activation", ["none", "relu"])
@pytest.mark.parametrize("sizes,of_x,of_weight", BACKWARD)
def test_linear_backward_in_every_tile(sizes, of_x, of_weight, activation, dtype):
    m, k, n = sizes
    g, x, w = whole((m, n), dtype, 1), whole((m, k), dtype, 2), whole((n, k), dtype, 3)
    z = whole((m, n), dtype, 4) if activation == "relu" else None
    got, names = launches(lambda: encoder.linear_backward(g, x, w, activation, z))
    tiles = [name for name in names if name not in ("linear_prepare_backward", "linear_join_backward")]
    assert tiles == (["linear_products_backward"] if of_x is None else [f"linear_tiles_{of_x}", f"linear_tiles_{of_weight}"])
    d = g.double() if z is None else torch.where(z > 0, g.double(), 0.0)
    for value, want in zip(got, (d @ w.double(), d.t() @ x.double(), d.sum(0))):
        assert torch.equal(value, want.to(dtype))


@pytest.mark.parametrize("activation", ["none", "relu"])
@pytest.mark.parametrize("sizes,of_x,of_weight", [((4090, 75, 4303), 64, 128), ((2500, 4200, 4300), 128, 64), ((5000, 2100, 2151), 128, 64), ((300, 610, 700), 64, 64)])
def test_linear_backward_of_floats_in_every_tile(sizes, of_x, of_weight, activation):
    m, k, n = sizes
    g, x, w = whole((m, n), F32, 1), whole((m, k), F32, 2), whole((n, k), F32, 3)
    z = whole((m, n), F32, 4) if activation == "relu" else None
    got, names = launches(lambda: encoder.linear_backward(g, x, w, activation, z))
    assert [name for name in names if "product" in name] == [f"linear_product_{of_x}", f"linear_product_{of_weight}"]
    d = g.double() if z is None else torch.where(z > 0, g.double(), 0.0)
    for value, want in zip(got, (d @ w.double(), d.t() @ x.double(), d.sum(0))):
        assert torch.equal(value, want.float())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k,n", [(1, 1024, 300), (16, 72, 40), (16, 2048, 4096), (32, 1024, 4096), (17, 2056, 1000), (64, 1024, 1024), (33, 1000, 4096), (48, 1003, 4090)])
def test_linear_of_few_rows(m, k, n, dtype):
    x, w, b, r = whole((m, k), dtype, 1), whole((n, k), dtype, 2), whole((n,), dtype, 3, 9), whole((m, n), dtype, 4, 9)
    (out, z), names = launches(lambda: encoder.linear(x, w, b, "relu", r, keep=True))
    assert names == ["linear_few_rows"]
    want = x.double() @ w.double().t() + b.double()
    assert torch.equal(z, want.to(dtype)) and torch.equal(out, (want.clamp(min=0) + r.double()).to(dtype))


# ------------------------------------------------------------------ several turns of a loop

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens,width", [(60011, 260), (300007, 40), (200003, 100), (100003, 250), (150001, 5), (70001, 1031)])
def test_embedding_of_several_tokens_a_wavefront(tokens, width, dtype):
    """More than a wavefront asks for at a time, at each number of rows side by side that can have so many."""
    gen = torch.Generator("cuda").manual_seed(tokens)
    vocabulary, places, length = 500, 40, 64
    ids = torch.randint(-1, vocabulary + 1, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    rows = tokens // length
    offsets = torch.arange(rows + 1, device="cuda", dtype=torch.int32) * length
    column = nvtext.DeviceListColumn(offsets, ids, None, rows, 0, checks.np.dtype(checks.np.int32), tokens)
    table, positions = whole((vocabulary, width), dtype, 1, 9), whole((places, width), dtype, 2, 9)
    want = torch.where(((ids >= 0) & (ids < vocabulary))[:, None], table[ids.clamp(0, vocabulary - 1).long()], 0.0)
    at = torch.arange(tokens, device="cuda") % length
    want = want + torch.where((at < places)[:, None], positions[at.clamp(max=places - 1)], 0.0)
    want[rows * length:] = 0
    assert torch.equal(encoder.embedding(column, table, positions), want)


@pytest.mark.parametrize("dtype,rows,cols", [(F32, 9001, 1021), (BF16, 140003, 64), (F16, 70003, 131)])
def test_dropout_of_several_turns(dtype, rows, cols):
    checks.test_dropout(dtype, rows, cols, 0, 0.3)


# more rows than the workgroups that run at a time have, at each number of lanes a row
TURNS = [(BF16, 33001, 100), (F32, 17001, 250), (BF16, 9001, 513), (F16, 8301, 1024), (BF16, 2101, 4000), (F32, 2101, 2100), (BF16, 601, 16000), (F16, 2101, 16392)]


@pytest.mark.parametrize("dtype,rows,cols", TURNS)
def test_layer_norm_of_several_turns(dtype, rows, cols):
    checks.test_layer_norm(dtype, rows, cols, 0, 0.3, True, True)


@pytest.mark.parametrize("dtype,rows,cols", TURNS)
def test_layer_norm_backward_of_several_turns(dtype, rows, cols):
    checks.test_layer_norm_backward(dtype, rows, cols, 0, 0.3, True, True)


# ------------------------------------------------------------------ NaN and infinities stay where the formula has them

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k,n", [(5, 72, 40), (64, 100, 301), (120, 72, 104), (300, 75, 260), (513, 72, 104), (1003, 4104, 4090), (4090, 4104, 100)])
def test_linear_backward_keeps_rows_and_columns_apart(m, k, n, dtype):
    g, x, w = whole((m, n), dtype, 1), whole((m, k), dtype, 2), whole((n, k), dtype, 3)
    clean = encoder.linear_backward(g, x, w)
    bad = g.clone()
    bad[3], bad[:, n - 1] = float("nan"), float("inf")
    dx, dw, db = encoder.linear_backward(bad, x, w)
    assert dx[3].isnan().all() and db[n - 1] == float("inf") and db[:-1].isnan().all()
    bad = g.clone()
    bad[m - 2] = float("nan")
    dx, dw, _ = encoder.linear_backward(bad, x, w)
    others = torch.arange(m, device="cuda") != m - 2
    assert torch.equal(dx[others], clean[0][others]) and dx[m - 2].isnan().all() and dw.isnan().all()
    bad = g.clone()
    bad[:, n - 1] = float("nan")
    dx, dw, db = encoder.linear_backward(bad, x, w)
    assert torch.equal(dw[:-1], clean[1][:-1]) and torch.equal(db[:-1], clean[2][:-1]) and dw[-1].isnan().all() and dx.isnan().all()
    bad = x.clone()
    bad[:, k - 1] = float("nan")
    dx, dw, _ = encoder.linear_backward(g, bad, w)
    assert torch.equal(dx, clean[0]) and torch.equal(dw[:, :-1], clean[1][:, :-1]) and dw[:, -1].isnan().all()
    bad = w.clone()
    bad[:, k - 1] = float("nan")
    dx, dw, _ = encoder.linear_backward(g, x, bad)
    assert torch.equal(dw, clean[1]) and torch.equal(dx[:, :-1], clean[0][:, :-1]) and dx[:, -1].isnan().all()


def test_embedding_keeps_entries_apart():
    """NaN in the gradient of a token reaches its entry and its place alone, and none where it belongs to neither."""
    ids = torch.tensor([0, 1, 2, -1, 1, 7], device="cuda", dtype=torch.int32)
    column = nvtext.DeviceListColumn(torch.tensor([0, 4, 5], device="cuda", dtype=torch.int32), ids, None, 2, 0, checks.np.dtype(checks.np.int32), 6)
    g = torch.ones(6, 40, device="cuda")
    g[2], g[3], g[5] = float("nan"), float("inf"), float("nan")
    t, p = encoder.embedding_backward(column, g, 8, 2)
    assert t[2].isnan().all() and t[[0, 1, 3, 4, 5, 6, 7]].sum(1).tolist() == [40, 80, 0, 0, 0, 0, 0] and p.sum(1).tolist() == [80, 40]
    table = torch.ones(8, 40, device="cuda")
    table[3:] = float("nan")
    assert encoder.embedding(column, table).sum(1).tolist() == [40, 40, 40, 0, 40, 0]
