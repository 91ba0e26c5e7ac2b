"""The encoder's operators at the limits of what they count in 32 bits.

Values are whole numbers whose sums stay below 2^24, so that every sum is exact and a result may differ from the formula by
nothing but its one rounding: equality is asked for.
"""
import pytest
import torch

from cudf_amd import encoder

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
