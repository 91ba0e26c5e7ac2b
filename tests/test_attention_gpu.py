"""Rotary positions and attention against their definitions in 64 bits.

A value may be off by the one rounding of its type at the end, and by what the oracle adds up for it: of everything held in 32 bits
2^-24 of the magnitudes that were added, times the longest chain of additions, and of the exponentials that 16-bit types have
rounded before they are multiplied, half a step of the type (the oracle's `unit`)."""
import numpy as np
import pytest
import torch

from cudf_amd import encoder, nvtext
from oracle import encoder_py as orc

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
UNIT = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}
TINY = {F32: 2.0**-149, F16: 2.0**-24, BF16: 2.0**-133}
TYPES = [F32, F16, BF16]


def rounding(dtype):
    """How far what is rounded before it is multiplied may be off: half a step of its value, or of the smallest one."""
    return {F32: dict(unit=0.0), F16: dict(unit=2.0**-11, tiny=2.0**-25), BF16: dict(unit=2.0**-8)}[dtype]


def near(got, want, off, dtype=None):
    dtype = dtype or got.dtype
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    wrong = np.abs(np.where(np.isinf(want), 0, got) - np.where(np.isinf(want), 0, want))
    most = UNIT[dtype] * np.abs(np.where(np.isinf(want), 0, want)) * (1 + UNIT[dtype]) + 1.01 * off + 2 * TINY[dtype]
    assert np.array_equal(np.isinf(got), np.isinf(want)) and not np.isnan(got).any()
    assert (got[np.isinf(want)] == want[np.isinf(want)]).all()
    worst = np.unravel_index(np.argmax(wrong - most), wrong.shape) if wrong.size else ()
    assert (wrong <= most).all(), f"at {worst}: {got[worst]} for {want[worst]}, off {wrong[worst]:.3g}, at most {most[worst]:.3g}"


def heads(rng, tokens, count, width, dtype, scale=1.0, pad=0):
    """Heads and their values in 64 bits; pad: the tokens lie so many values further apart."""
    a = rng.standard_normal((tokens, count * width + pad)) * scale
    t = torch.from_numpy(a).to(dtype).cuda()[:, pad // 2: pad // 2 + count * width].unflatten(1, (count, width))
    return t, t.double().cpu().numpy()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def unrounded(saved):
    """out's values with what rounding left off them: its bits as float32 with the rest's behind them."""
    if saved.rest is None:
        return saved.out.double().cpu().numpy()
    shift = {F16: 5, BF16: 8}[saved.out.dtype]
    return (saved.out.float().view(torch.int32) + saved.rest.transpose(0, 1).int() * 2**shift).view(torch.float32).double().cpu().numpy()


def offsets_of(lengths, first=0):
    return np.concatenate([[first], first + np.cumsum(lengths)]).astype(np.int32)


# ------------------------------------------------------------------ rotary positions

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("lengths,count,width,pairs,pad", [
    ([1], 1, 2, 1, 0), ([1], 40, 128, 64, 0), ([3, 0, 5], 4, 64, 32, 0), ([70, 1], 3, 80, 20, 16), ([9], 5, 33, 16, 1), ([2, 2], 2, 7, 3, 3), ([300], 2, 12, 5, 0), ([4], 1, 10, 0, 0),
    ([5000], 1, 8, 4, 0), ([3], 2, 4096, 2048, 0),
])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary(dtype, layout, lengths, count, width, pairs, pad, inverse):
    """A product and the sum of two: three roundings of 32 bits of the magnitudes, and sine and cosine off by 2^-22."""
    rng = np.random.default_rng(width)
    offsets = offsets_of(lengths, 2)
    tokens = int(offsets[-1]) + 3
    x, x64 = heads(rng, tokens, count, width, dtype, pad=pad)
    f = encoder.rotary_frequencies(2 * pairs, 1000.0) if pairs else torch.zeros(0, dtype=torch.float64, device="cuda")
    starts = rng.integers(0, 100000, len(lengths))
    want, size = orc.rotary(x64, offsets, f.cpu().numpy(), starts, layout, inverse, 1.37)
    got = encoder.rotary(x, ints(offsets), f, ints(starts), layout, inverse, 1.37)
    near(got, want, size * (2.0**-22 + 4 * 2.0**-24))
    kept = np.broadcast_to(np.arange(width) >= 2 * pairs, x64.shape).copy()
    kept[:2] = kept[int(offsets[-1]):] = True
    kept = torch.from_numpy(kept).cuda()
    assert torch.equal(got[kept], x[kept])
    again = encoder.rotary(x, ints(offsets), f, ints(starts), layout, inverse, 1.37, out=x)
    assert again is x and torch.equal(x, got)


def test_rotary_of_far_positions():
    """Angles of 2^31 and of frequencies that are no round part of a turn: in 32 bits nothing would be left of them."""
    rng = np.random.default_rng(3)
    x, x64 = heads(rng, 6, 2, 64, F32)
    f = encoder.rotary_frequencies(64)
    starts = [2**31 - 4, 10**9]
    want, size = orc.rotary(x64, [0, 3, 6], f.cpu().numpy(), starts)
    near(encoder.rotary(x, ints([0, 3, 6]), f, ints(starts)), want, size * (2.0**-22 + 2.0**31 * 2.0**-52 + 4 * 2.0**-24))


def test_rotary_copies_bits_outside_rows():
    x = torch.full((5, 2, 8), float("inf"), device="cuda")
    x[0, 0, 0] = float("nan")
    f = encoder.rotary_frequencies(8)
    got = encoder.rotary(x, ints([2, 3]), f)
    for t in (0, 1, 3, 4):
        assert torch.equal(got[t].view(torch.int32), x[t].view(torch.int32))
    assert torch.equal(encoder.rotary(x, ints([0]), f).view(torch.int32), x.view(torch.int32))


def test_rotary_into_another_layout():
    """Query and key heads of a projection in place, and tokens within heads."""
    rng = np.random.default_rng(4)
    projection = torch.from_numpy(rng.standard_normal((50, 12 * 16))).to(BF16).cuda()
    f = encoder.rotary_frequencies(16)
    rows = ints([0, 20, 50])
    view = projection.view(50, 12, 16)[:, :8]
    want = encoder.rotary(view, rows, f)
    before = projection.clone()
    encoder.rotary(view, rows, f, out=view)
    assert torch.equal(view, want) and torch.equal(projection[:, 128:], before[:, 128:])
    turned = torch.empty(8, 50, 16, dtype=BF16, device="cuda").transpose(0, 1)
    assert torch.equal(encoder.rotary(before.view(50, 12, 16)[:, :8], rows, f, out=turned), want)


def test_rotary_gradient_is_the_inverse_call():
    """(R x, g) = (x, R^T g) for any x and g; both sums are of 2400 products in 64 bits of values rounded to 32."""
    rng = np.random.default_rng(5)
    x, x64 = heads(rng, 30, 5, 16, F32)
    g, g64 = heads(rng, 30, 5, 16, F32)
    f = encoder.rotary_frequencies(12)
    for layout in ("half", "interleaved"):
        y = encoder.rotary(x, ints([0, 30]), f, None, layout, magnitude=1.5).double().cpu().numpy()
        b = encoder.rotary(g, ints([0, 30]), f, None, layout, inverse=True, magnitude=1.5).double().cpu().numpy()
        size = (np.abs(x64) * 3).sum() * np.abs(g64).max()
        assert abs((y * g64).sum() - (x64 * b).sum()) <= 2 * size * (2.0**-22 + 5 * 2.0**-24)


# ------------------------------------------------------------------ attention

# (tokens of the rows, keys of the rows or None for the same, heads, key heads, width, values that tokens lie further apart)
CASES = [
    ([1], None, 1, 1, 1, 0), ([1], None, 4, 4, 64, 0), ([3, 0, 2], None, 2, 1, 8, 0), ([64], None, 2, 2, 64, 0), ([65, 63], None, 3, 3, 64, 64), ([31, 33, 1, 0, 7], None, 4, 2, 32, 0),
    ([129], None, 2, 1, 128, 8), ([40, 5, 100], None, 2, 2, 72, 0), ([17, 50], None, 2, 2, 80, 16), ([257], None, 1, 1, 96, 0), ([70, 10], None, 2, 1, 256, 0), ([50], None, 1, 1, 200, 0),
    ([37, 9], None, 6, 3, 5, 1), ([66], None, 2, 2, 33, 0), ([20], None, 1, 1, 255, 1), ([300, 200], None, 8, 2, 16, 0), ([12, 200], None, 5, 1, 160, 0),
    ([1, 1, 1], [5, 130, 1], 8, 2, 64, 0), ([1], [1000], 4, 1, 128, 0), ([1, 1], [300, 0], 16, 16, 64, 0), ([2, 1, 3], [90, 64, 257], 6, 2, 128, 0), ([5], [3], 2, 2, 64, 0), ([70, 6], [20, 200], 2, 1, 64, 0),
    ([130], [300], 2, 2, 128, 0), ([4, 4], [500, 33], 3, 3, 40, 4), ([1, 0, 1], [7, 9, 65], 40, 8, 256, 0), ([1], [700], 3, 1, 50, 1),
]


# what one or another way through the kernels needs: rows of many columns among rows of few, chunks and shares of many tiles, and of causal ones that end
# before others
CASES += [
    ([40, 1, 1, 1, 0, 2], [900, 300, 129, 128, 700, 127], 2, 2, 64, 0), ([1, 9], [2000, 1500], 4, 1, 128, 0), ([200], [1500], 2, 1, 64, 0), ([150, 3], [900, 1200], 2, 2, 128, 0),
    ([1300], None, 2, 1, 64, 0), ([900, 40], None, 1, 1, 128, 0), ([700, 1], None, 2, 2, 256, 0), ([260], [1000], 8, 1, 40, 0), ([800], [200], 2, 1, 64, 0),
]


class Made:
    """A case's tensors, with tokens in front of the first row and behind the last, and keys in places with room."""

    def __init__(self, case, dtype, roomy=False, seed=0, scale=1.5):
        lengths, keys, self.count, self.kv, self.width, pad = case
        rng = self.rng = np.random.default_rng(seed + sum(lengths) + self.width)
        self.dtype = dtype
        self.offsets = offsets_of(lengths, 1)
        tokens = int(self.offsets[-1]) + 2
        self.q, self.q64 = heads(rng, tokens, self.count, self.width, dtype, scale, pad)
        self.key_offsets = self.key_lengths = None
        key_tokens = tokens
        if keys is not None or roomy:
            keys = lengths if keys is None else keys
            self.key_offsets = offsets_of([n + (i * 5 + 3 if roomy else 0) for i, n in enumerate(keys)], 2)
            self.key_lengths = np.array(keys, np.int32) if roomy else None
            key_tokens = int(self.key_offsets[-1]) + 3
        self.k, self.k64 = heads(rng, key_tokens, self.kv, self.width, dtype, 1.0, pad)
        self.v, self.v64 = heads(rng, key_tokens, self.kv, self.width, dtype, 1.0, pad)
        self.g, self.g64 = heads(rng, tokens, self.count, self.width, dtype, 1.0, pad)

    def rows(self):
        return [ints(self.offsets), None if self.key_offsets is None else ints(self.key_offsets), None if self.key_lengths is None else ints(self.key_lengths)]

    def oracle_rows(self):
        return dict(offsets=self.offsets, key_offsets=self.key_offsets, key_lengths=self.key_lengths)

    def check_forward(self, causal, scale=None):
        want, log, off, log_off = orc.attention(self.q64, self.k64, self.v64, **self.oracle_rows(), causal=causal, scale=scale, **rounding(self.dtype))
        out, saved = encoder.attention(self.q, self.k, self.v, *self.rows(), causal=causal, scale=scale, keep=True)
        assert saved.out is out
        near(out, want, off)
        near(saved.logsum, log, log_off)
        assert torch.equal(encoder.attention(self.q, self.k, self.v, *self.rows(), causal=causal, scale=scale), out)
        return want, log

    def check_backward(self, causal, scale=None):
        want, log, _, _ = orc.attention(self.q64, self.k64, self.v64, **self.oracle_rows(), causal=causal, scale=scale)
        out = torch.from_numpy(want).to(self.dtype).cuda()
        logsum = torch.from_numpy(log).float().cuda()
        wants, offs = orc.attention_backward(self.g64, self.q64, self.k64, self.v64, out.double().cpu().numpy(), logsum.double().cpu().numpy(), **self.oracle_rows(), causal=causal, scale=scale, **rounding(self.dtype))
        saved = encoder.AttentionSaved(out, logsum)
        got = encoder.attention_backward(self.g, self.q, self.k, self.v, saved, *self.rows(), causal=causal, scale=scale)
        for name, x, w, o in zip("qkv", got, wants, offs):
            try:
                near(x, w, o)
            except AssertionError as e:
                raise AssertionError(f"gradient of {name}: {e}") from None
        again = encoder.attention_backward(self.g, self.q, self.k, self.v, saved, *self.rows(), causal=causal, scale=scale)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention(case, causal, dtype):
    Made(case, dtype).check_forward(causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention_backward(case, causal, dtype):
    Made(case, dtype).check_backward(causal)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", [CASES[2], CASES[5], CASES[12], CASES[15], CASES[17], CASES[21], CASES[25]], ids=str)
def test_what_rounding_leaves_off(case, dtype):
    """Both directions together: the gradients from the out that was rounded and its rest are those from out as it is, up to a 2^-8 of a step
    of it, and what the forward pass may be off by."""
    m = Made(case, dtype, seed=3)
    want, log, off, log_off = orc.attention(m.q64, m.k64, m.v64, **m.oracle_rows(), causal=True, **rounding(dtype))
    out, saved = encoder.attention(m.q, m.k, m.v, *m.rows(), causal=True, keep=True)
    assert saved.rest.dtype == torch.int8 and saved.rest.shape == out.transpose(0, 1).shape
    more = unrounded(saved)
    assert (np.abs(more - want) <= off * 1.01 + UNIT[dtype] * 2.0**-7 * np.abs(want) + 2 * TINY[dtype]).all()
    wants, offs = orc.attention_backward(m.g64, m.q64, m.k64, m.v64, more, saved.logsum.double().cpu().numpy(), **m.oracle_rows(), causal=True, **rounding(dtype))
    got = encoder.attention_backward(m.g, m.q, m.k, m.v, saved, *m.rows(), causal=True)
    for x, w, o in zip(got, wants, offs):
        near(x, w, o)


@pytest.mark.parametrize("case", [CASES[1], CASES[5], CASES[11], CASES[17], CASES[20], CASES[22], CASES[25]], ids=str)
def test_keys_in_places_with_room(case):
    """What lies behind a row's keys is not read: NaN there."""
    for dtype in TYPES:
        m = Made(case, dtype, roomy=True)
        for first, last, n in zip(m.key_offsets[:-1], m.key_offsets[1:], m.key_lengths):
            m.k[first + n:last] = m.v[first + n:last] = float("nan")
        m.check_forward(True)
        m.check_forward(False)
        m.check_backward(True)


@pytest.mark.parametrize("scale", [0.0, 0.02, 3.0])
def test_scales(scale):
    """A scale of 0 is a mean over the keys; with a large one, a single key has nearly all of the weight."""
    for dtype in TYPES:
        m = Made(([40, 3], None, 2, 1, 64, 0), dtype)
        m.check_forward(True, scale)
        m.check_backward(True, scale)


def test_scores_far_apart():
    """Keys whose scores rise by hundreds from one to the next, and fall: what was added up before fades to nothing, without overflow."""
    for dtype in (F32, BF16):
        for order in (1, -1):
            rng = np.random.default_rng(8)
            n, width = 200, 64
            q = torch.ones(1, 1, width, dtype=dtype, device="cuda")
            k = torch.from_numpy(np.arange(n)[::order].astype(np.float64)[:, None, None] * np.ones(width)).to(dtype).cuda()
            v, v64 = heads(rng, n, 1, width, dtype)
            want, log, off, log_off = orc.attention(q.double().cpu().numpy(), k.double().cpu().numpy(), v64, [0, 1], [0, n], **rounding(dtype))
            out, saved = encoder.attention(q, k, v, ints([0, 1]), ints([0, n]), keep=True)
            near(out, want, off)
            near(saved.logsum, log, log_off)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_what_is_not_seen_has_no_effect(dtype, value):
    """A token's k and v, and what lies in no row, are anything at all: the tokens that do not see them have what they have without."""
    m = Made(([70, 40, 130], None, 4, 2, 64, 0), dtype)
    bad = int(m.offsets[1]) + 21  # a token of the second row
    want, log, off, log_off = orc.attention(m.q64, m.k64, m.v64, m.offsets, causal=True, **rounding(dtype))
    grads = None
    for where in ("k", "v", "both"):
        q, k, v, g = m.q.clone(), m.k.clone(), m.v.clone(), m.g.clone()
        for t in (0, bad, len(k) - 1):
            if where != "v":
                k[t] = value
            if where != "k":
                v[t] = value
        out, saved = encoder.attention(q, k, v, ints(m.offsets), causal=True, keep=True)
        untouched = np.ones(len(q), bool)
        untouched[bad:int(m.offsets[2])] = False
        pick = torch.from_numpy(untouched).cuda()
        near(out[pick], want[untouched], off[untouched])
        near(saved.logsum[:, pick], log[:, untouched], log_off[:, untouched])
        if where != "k":
            assert not torch.isfinite(out[bad]).any()
        # and the way back: of q, what does not see it; of k and v, what only tokens see that do not (none in its row behind it)
        clean = encoder.attention(m.q, m.k, m.v, ints(m.offsets), causal=True, keep=True)[1]
        saved = encoder.AttentionSaved(torch.where(pick[:, None, None], clean.out, out), torch.where(pick[None], clean.logsum, saved.logsum),
                                       None if saved.rest is None else torch.where(pick[None, :, None], clean.rest, saved.rest))
        grads = encoder.attention_backward(g, q, k, v, saved, ints(m.offsets), causal=True)
        wants, offs = orc.attention_backward(m.g64, m.q64, m.k64, m.v64, unrounded(clean), clean.logsum.double().cpu().numpy(), m.offsets, causal=True, **rounding(dtype))
        near(grads[0][pick], wants[0][untouched], offs[0][untouched])
        others = np.ones(len(q), bool)
        others[int(m.offsets[1]):int(m.offsets[2])] = False
        pick_others = torch.from_numpy(others).cuda()
        for x, w, o in zip(grads[1:], wants[1:], offs[1:]):
            near(x[pick_others], w[others], o[others])
    # a query's and its gradient's: k and v behind it do not see it
    q, g = m.q.clone(), m.g.clone()
    q[bad], g[bad] = value, value
    out, saved = encoder.attention(q, m.k, m.v, ints(m.offsets), causal=True, keep=True)
    others = np.ones(len(q), bool)
    others[bad] = False
    pick = torch.from_numpy(others).cuda()
    near(out[pick], want[others], off[others])
    grads = encoder.attention_backward(g, q, m.k, m.v, saved, ints(m.offsets), causal=True)
    wants, offs = orc.attention_backward(m.g64, m.q64, m.k64, m.v64, unrounded(clean), clean.logsum.double().cpu().numpy(), m.offsets, causal=True, **rounding(dtype))
    near(grads[0][pick], wants[0][others], offs[0][others])
    behind = np.ones(len(q), bool)
    behind[int(m.offsets[1]):bad + 1] = False
    pick = torch.from_numpy(behind).cuda()
    for x, w, o in zip(grads[1:], wants[1:], offs[1:]):
        near(x[pick], w[behind], o[behind])


def test_scores_of_minus_infinity():
    """A key whose score is -infinity has no weight; where all seen have it, there is no result."""
    for dtype in TYPES:
        q = torch.ones(2, 1, 16, dtype=dtype, device="cuda")
        k = torch.ones(80, 1, 16, dtype=dtype, device="cuda")
        k[3:60] = float("-inf")
        v = torch.zeros(80, 1, 16, dtype=dtype, device="cuda")
        v[:3], v[60:] = 1.0, 2.0
        out = encoder.attention(q, k, v, ints([0, 2]), ints([0, 80]))
        want = (3 + 20 * 2) / 23
        assert (out.double() - want).abs().max() <= want * (2 * UNIT[dtype] + 100 * 2.0**-24)
        k[:] = float("-inf")
        assert torch.isnan(encoder.attention(q, k, v, ints([0, 2]), ints([0, 80]))).all()


def test_gradient_against_differences():
    """The loss (out, g) along a direction, by differences of the float32 kernel itself: with a step of 2^-6 the cubic term is
    2^-12 of a third derivative of the size of the loss, and rounding 2^-24 * 2^6 of the sums' magnitudes."""
    m = Made(([9, 14], [12, 14], 4, 2, 24, 0), F32)
    out, saved = encoder.attention(m.q, m.k, m.v, *m.rows(), causal=True, keep=True)
    grads = encoder.attention_backward(m.g, m.q, m.k, m.v, saved, *m.rows(), causal=True)
    for i in range(3):
        args = [m.q, m.k, m.v]
        direction = torch.from_numpy(m.rng.standard_normal(args[i].shape)).float().cuda()
        values = []
        for sign in (1, -1):
            moved = list(args)
            moved[i] = args[i] + sign * 2.0**-6 * direction
            values.append((encoder.attention(*moved, *m.rows(), causal=True).double() * m.g.double()).sum().item())
        got, want = (grads[i].double() * direction.double()).sum().item(), (values[0] - values[1]) * 2.0**5
        size = (grads[i].double().abs() * direction.double().abs()).sum().item()
        assert abs(got - want) <= size * (8 * 2.0**-12 + 2.0**-14), (i, got, want, size)


def test_layouts():
    """Parts of a projection, tokens within heads, broadcast keys; gradients into the parts of a projection's gradient."""
    rng = np.random.default_rng(12)
    rows = ints([0, 30, 77])
    projection = torch.from_numpy(rng.standard_normal((77, 8, 64))).to(BF16).cuda()
    q, k, v = projection[:, :4], projection[:, 4:6], projection[:, 6:]
    out, saved = encoder.attention(q, k, v, rows, causal=True, keep=True)
    plain = [x.contiguous() for x in (q, k, v)]
    assert torch.equal(encoder.attention(*plain, rows, causal=True), out)
    within = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(encoder.attention(*within, rows, causal=True), out)
    g = torch.randn(77, 4, 64, device="cuda").to(BF16)
    want = encoder.attention_backward(g, *plain, saved, rows, causal=True)
    whole = torch.full((77, 10, 64), 5.0, dtype=BF16, device="cuda")
    got = encoder.attention_backward(g, q, k, v, saved, rows, causal=True, out=(whole[:, 1:5], whole[:, 5:7], whole[:, 7:9]))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and (whole[:, 0] == 5).all() and (whole[:, 9] == 5).all()
    assert torch.equal(encoder.attention_backward(g.transpose(0, 1).contiguous().transpose(0, 1), *within, saved, rows, causal=True)[1], want[1])
    one = k[:1].expand(77, 2, 64)
    assert torch.equal(encoder.attention(q, one, v, rows), encoder.attention(q, one.contiguous(), v, rows))
    assert torch.equal(encoder.attention_backward(g, q, one, v, saved, rows)[1], encoder.attention_backward(g, q, one.contiguous(), v, saved, rows)[1])


def test_a_column_of_tokens_as_rows():
    child = torch.arange(12, dtype=torch.int32, device="cuda").view(torch.uint8)
    column = nvtext.DeviceListColumn(ints([0, 5, 5, 12]).view(torch.uint8), child, None, 3, 0, np.dtype(np.int32), 12)
    q = torch.randn(12, 2, 32, device="cuda")
    assert torch.equal(encoder.attention(q, q, q, column), encoder.attention(q, q, q, ints([0, 5, 5, 12])))
    f = encoder.rotary_frequencies(32)
    assert torch.equal(encoder.rotary(q, column, f), encoder.rotary(q, ints([0, 5, 5, 12]), f))


def test_rows_at_odd_places():
    """The same values at addresses and distances that no wide load has: the same results."""
    for dtype in TYPES:
        for width in (64, 72, 128):
            m = Made(([50, 70, 1], None, 2, 1, width, 0), dtype)
            out, saved = encoder.attention(m.q, m.k, m.v, *m.rows(), causal=True, keep=True)
            grads = encoder.attention_backward(m.g, m.q, m.k, m.v, saved, *m.rows(), causal=True)

            def odd(x):
                tokens, count, width = x.shape
                y = torch.empty(tokens * (count * (width + 1) + 1) + 1, dtype=dtype, device="cuda")[1:].as_strided(x.shape, (count * (width + 1) + 1, width + 1, 1), 1)
                y.copy_(x)
                return y
            q, k, v, g = odd(m.q), odd(m.k), odd(m.v), odd(m.g)
            want, log, off, log_off = orc.attention(m.q64, m.k64, m.v64, m.offsets, causal=True, **rounding(dtype))
            got, kept = encoder.attention(q, k, v, *m.rows(), causal=True, keep=True)
            near(got, want, off)
            near(kept.logsum, log, log_off)
            into = tuple(odd(torch.zeros_like(x)) for x in (q, k, v))
            for a, b in zip(encoder.attention_backward(g, q, k, v, saved._replace(out=odd(out)), *m.rows(), causal=True, out=into), grads):
                assert torch.equal(a, b)


def test_no_tokens_no_rows_no_keys():
    for dtype in TYPES:
        x, none = torch.randn(5, 2, 16, device="cuda").to(dtype), torch.empty(0, 2, 16, dtype=dtype, device="cuda")
        out, saved = encoder.attention(x, x, x, ints([0]), keep=True)  # no rows: nobody sees anything
        assert (out == 0).all() and (saved.logsum == float("-inf")).all()
        assert all((g == 0).all() for g in encoder.attention_backward(x, x, x, x, saved, ints([0])))
        out, saved = encoder.attention(x, none, none, ints([0, 5]), ints([0, 0]), keep=True)  # no keys
        assert (out == 0).all() and (saved.logsum == float("-inf")).all()
        dq, dk, dv = encoder.attention_backward(x, x, none, none, saved, ints([0, 5]), ints([0, 0]))
        assert (dq == 0).all() and dk.shape == dv.shape == none.shape
        assert encoder.attention(none, x, x, ints([0, 0]), ints([0, 5])).shape == (0, 2, 16)  # no tokens
        dq, dk, dv = encoder.attention_backward(none, none, x, x, encoder.AttentionSaved(none, torch.empty(2, 0, device="cuda")), ints([0, 0]), ints([0, 5]))
        assert dq.shape == none.shape and (dk == 0).all() and (dv == 0).all()
        assert encoder.rotary(none, ints([0, 0]), encoder.rotary_frequencies(16)).shape == none.shape


def test_offsets_out_of_range_read_and_write_nothing_outside():
    """Offsets that point in front of the tokens and behind them, and lengths below zero and above what is there, are cut to what is."""
    m = Made(([60, 50], None, 2, 2, 64, 0), BF16)
    tokens = len(m.q)
    got = encoder.attention(m.q, m.k, m.v, ints([-7, 60, tokens + 1000]), causal=True)
    assert torch.equal(got, encoder.attention(m.q, m.k, m.v, ints([0, 60, tokens]), causal=True))
    got = encoder.attention(m.q, m.k, m.v, ints([0, 60, tokens]), ints([0, 60, tokens]), ints([-3, 2**31 - 1]))
    assert torch.equal(got, encoder.attention(m.q, m.k, m.v, ints([0, 60, tokens]), ints([0, 60, tokens]), ints([0, tokens - 60])))


def test_many_short_rows():
    rng = np.random.default_rng(14)
    lengths = rng.integers(0, 5, 5000)
    offsets = offsets_of(lengths)
    tokens = int(offsets[-1])
    for dtype in (F32, BF16):
        q, q64 = heads(rng, tokens, 2, 16, dtype)
        out, saved = encoder.attention(q, q, q, ints(offsets), keep=True)
        g, g64 = heads(rng, tokens, 2, 16, dtype)
        grads = encoder.attention_backward(g, q, q, q, saved, ints(offsets))
        want, log, off, log_off = orc.attention(q64, q64, q64, offsets, **rounding(dtype))
        near(out, want, off)
        near(saved.logsum, log, log_off)
        wants, offs = orc.attention_backward(g64, q64, q64, q64, unrounded(saved), saved.logsum.double().cpu().numpy(), offsets, **rounding(dtype))
        for x, w, o in zip(grads, wants, offs):
            near(x, w, o)


def test_on_another_stream_and_captured():
    """A graph of a rotation, an attention and both ways back, replayed on other values, against the calls themselves."""
    rng = np.random.default_rng(15)
    rows, f = ints([0, 33, 100, 260]), encoder.rotary_frequencies(64)
    projection = torch.from_numpy(rng.standard_normal((260, 8, 64))).to(BF16).cuda()
    cache = torch.from_numpy(rng.standard_normal((900, 2, 64))).to(BF16).cuda()
    key_rows, key_lengths = ints([0, 200, 500, 900]), ints([150, 300, 390])
    single = ints([0, 1, 2, 3])

    def step():
        turned = encoder.rotary(projection[:, :6], rows, f)
        q, k, v = turned[:, :4], turned[:, 4:], projection[:, 6:]
        out, saved = encoder.attention(q, k, v, rows, causal=True, keep=True)
        grads = encoder.attention_backward(out, q, k, v, saved, rows, causal=True)
        return (turned, out, saved.logsum, *grads, encoder.rotary(grads[0], rows, f, inverse=True), encoder.attention(q[:3], cache, cache, single, key_rows, key_lengths, causal=True))

    want = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for replay in range(4):
        projection.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        kept = [x.clone() for x in got]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want)), replay


def test_refusals():
    x, f = torch.randn(6, 4, 16, device="cuda"), encoder.rotary_frequencies(16)
    rows = ints([0, 6])
    for text, call in [
        ("layout", lambda: encoder.rotary(x, rows, f, layout="thirds")),
        ("float64", lambda: encoder.rotary(x, rows, f.float())),
        ("float64", lambda: encoder.rotary(x, rows, f[::2])),
        ("frequencies", lambda: encoder.rotary(x, rows, encoder.rotary_frequencies(18))),
        ("starts must have", lambda: encoder.rotary(x, rows, f, ints([0, 0]))),
        ("int32", lambda: encoder.rotary(x, rows.long(), f)),
        ("a value more", lambda: encoder.rotary(x, rows[:0], f)),
        ("tokens, heads, width", lambda: encoder.rotary(x[0], rows, f)),
        ("float32, float16", lambda: encoder.rotary(x.double(), rows, f)),
        ("device memory", lambda: encoder.rotary(x.cpu(), rows, f)),
        ("device memory", lambda: encoder.rotary(x, rows.cpu(), f)),
        ("size and type", lambda: encoder.rotary(x, rows, f, out=x[:5])),
        ("overlap", lambda: encoder.rotary(x, rows, f, out=x[:1].expand(6, 4, 16))),
        ("last dimension", lambda: encoder.attention(x.transpose(1, 2), x, x, rows)),
        ("divisor", lambda: encoder.attention(x, x[:, :3], x[:, :3], rows)),
        ("one type", lambda: encoder.attention(x, x.half(), x, rows)),
        ("q's tokens", lambda: encoder.attention(x, x[:5], x[:5], rows)),
        ("as many rows", lambda: encoder.attention(x, x, x, rows, ints([0, 3, 6]))),
        ("key_rows", lambda: encoder.attention(x, x, x, rows, None, ints([6]))),
        ("key_lengths must have", lambda: encoder.attention(x, x, x, rows, rows, ints([6, 6]))),
        ("scale", lambda: encoder.attention(x, x, x, rows, scale=-0.5)),
        ("256", lambda: encoder.attention(*[torch.zeros(6, 1, 257, device="cuda")] * 3, rows)),
        ("logsum", lambda: encoder.attention_backward(x, x, x, x, encoder.AttentionSaved(x, torch.zeros(6, 4, device="cuda")), rows)),
        ("rest", lambda: encoder.attention_backward(x, x, x, x, encoder.AttentionSaved(x, torch.zeros(4, 6, device="cuda"), x.to(torch.int8)[:5]), rows)),
        ("grad and out", lambda: encoder.attention_backward(x[:5], x, x, x, encoder.AttentionSaved(x, torch.zeros(4, 6, device="cuda")), rows)),
        ("those of", lambda: encoder.attention_backward(x, x, x, x, encoder.AttentionSaved(x, torch.zeros(4, 6, device="cuda")), rows, out=(x, x, x[:, :2]))),
    ]:
        with pytest.raises(ValueError, match=text):
            call()


def test_no_memory_for_temporaries():
    mr = nvtext._mr()
    x, rows = torch.randn(100, 2, 16, device="cuda"), ints([0, 100])
    _, saved = encoder.attention(x, x, x, rows, keep=True)
    live = len(mr.live)
    mr.fail_after = 0
    try:
        with pytest.raises(MemoryError):
            encoder.attention_backward(x, x, x, x, saved, rows)
    finally:
        mr.fail_after = None
    assert len(mr.live) == live


# rows of few tokens among rows of many: some go in chunks of their keys and some in tiles, or a row of many columns through the chunks that it has
MIXED = [
    ([1] * 40 + [60], [3 * i for i in range(40)] + [300], 8, 2, 64, 0),
    ([0] * 30 + [20, 1, 1, 1], [5] * 30 + [700, 200, 0, 129], 8, 2, 64, 0),
    ([1, 2, 5, 9, 17, 40, 0, 3] * 4, None, 8, 2, 72, 0),
    ([1, 1, 30], [900, 129, 1100], 2, 1, 128, 0),
    ([2] * 9 + [33, 16, 17], [128, 127, 129, 1, 0, 2, 256, 257, 700, 128, 128, 129], 4, 2, 40, 8),
    ([1] * 300, [1 + i % 140 for i in range(300)], 40, 8, 32, 0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("roomy", [False, True])
@pytest.mark.parametrize("case", MIXED, ids=lambda c: f"{len(c[0])}x{sum(c[0])}")
def test_rows_of_few_tokens_among_others(case, roomy, causal, dtype):
    m = Made(case, dtype, roomy)
    if roomy:
        for first, last, n in zip(m.key_offsets[:-1], m.key_offsets[1:], m.key_lengths):
            m.k[first + n:last] = m.v[first + n:last] = float("nan")
    m.check_forward(causal)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_offsets_over_more_keys_than_tokens(dtype):
    """One array of offsets for both, that ends behind the tokens: they are its first ones, and the keys are all there."""
    rng = np.random.default_rng(16)
    q, q64 = heads(rng, 12, 4, 64, dtype)
    k, k64 = heads(rng, 1200, 2, 64, dtype)
    rows = ints([0, 10, 1200])
    for causal in (False, True):
        want, log, off, log_off = orc.attention(q64, k64, k64, [0, 10, 12], [0, 10, 1200], causal=causal, **rounding(dtype))
        out, saved = encoder.attention(q, k, k, rows, rows, causal=causal, keep=True)
        near(out, want, off)
        near(saved.logsum, log, log_off)


@pytest.mark.parametrize("lengths,keys", [([4, 3, 1], [300, 200, 500]), ([150, 60], [1500, 100])])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_key_that_only_the_last_tokens_see(lengths, keys, value):
    """In chunks and in shares of tiles: the tokens in front of it have what they have without."""
    for dtype in TYPES:
        m = Made((lengths, keys, 4, 2, 64, 0), dtype)
        want, log, off, log_off = orc.attention(m.q64, m.k64, m.v64, **m.oracle_rows(), causal=True, **rounding(dtype))
        last = [int(m.key_offsets[1]) - 1, int(m.key_offsets[2]) - 1]
        m.k[last[0]] = value
        m.v[last] = value
        out, saved = encoder.attention(m.q, m.k, m.v, *m.rows(), causal=True, keep=True)
        seen = [int(m.offsets[1]) - 1, int(m.offsets[2]) - 1]
        pick = np.ones(len(m.q), bool)
        pick[seen] = False
        where = torch.from_numpy(pick).cuda()
        near(out[where], want[pick], off[pick])
        near(saved.logsum[:, where], log[:, pick], log_off[:, pick])
        assert not torch.isfinite(out[seen[1]]).any()


def test_two_streams_at_once():
    rng = np.random.default_rng(17)
    made = [Made((lengths, keys, 8, 2, 64, 0), BF16, seed=i) for i, (lengths, keys) in enumerate([([1] * 20, [400] * 20), ([500, 20], None), ([3000], None), ([1, 50], [900, 2000])])]
    calls = [lambda m=m: encoder.attention(m.q, m.k, m.v, *m.rows(), causal=True) for m in made]
    calls += [lambda m=m: encoder.attention_backward(m.g, m.q, m.k, m.v, m.saved, *m.rows(), causal=True) for m in made]
    for m in made:
        m.saved = encoder.attention(m.q, m.k, m.v, *m.rows(), causal=True, keep=True)[1]
    wants = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for order in range(len(calls)):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[s].append(calls[order if s == 0 else len(calls) - 1 - order]())
    torch.cuda.synchronize()
    got[1].reverse()
    for results in got:
        for a, b in zip(results, wants):
            assert all(torch.equal(x, y) for x, y in zip(a, b)) if isinstance(b, tuple) else torch.equal(a, b)


@pytest.mark.parametrize("single", [True, False])
def test_a_cache_of_more_than_2_to_31_values(single):
    """Rows at its begin, across the value that no 32 bits count, and at its end, against the same rows in caches of their own."""
    torch.manual_seed(18)
    tokens, lengths = 17 * 2**20 + 5, [700, 600, 900]
    cache = torch.empty(tokens, 1, 128, dtype=BF16, device="cuda")
    starts = [3, 2**24 - 300, tokens - 900]
    assert starts[1] * 128 < 2**31 < (starts[1] + 600) * 128
    key_offsets = ints([starts[0], starts[1], starts[2], tokens])
    for first, n in zip(starts, lengths):
        cache[first:first + n] = torch.randn(n, 1, 128, device="cuda")
    count = 1 if single else 140
    offsets = ints([0, count, 2 * count, 3 * count])
    q = torch.randn(3 * count, 4, 128, device="cuda").to(BF16)
    out, saved = encoder.attention(q, cache, cache, offsets, key_offsets, ints(lengths), causal=True, keep=True)
    small = torch.cat([cache[first:first + n] for first, n in zip(starts, lengths)])
    want, want_saved = encoder.attention(q, small, small, offsets, ints(offsets_of(lengths)), causal=True, keep=True)
    # (other numbers of chunks and shares: sums in another order, of exponentials that another maximum rounds)
    assert ((out.float() - want.float()).abs() <= 2 * 2.0**-8 * (want.float().abs() + small.float().abs().max())).all()
    assert ((saved.logsum - want_saved.logsum).abs() <= 1e-5 * (1 + want_saved.logsum.abs())).all()
    del out
    grads = encoder.attention_backward(q, q, cache, cache, saved, offsets, key_offsets, ints(lengths), causal=True)
    wants = encoder.attention_backward(q, q, small, small, saved, offsets, ints(offsets_of(lengths)), causal=True)
    bounds = [2.0**-7 * (w.float().abs() + w.float().abs().max()) for w in wants]
    assert ((grads[0].float() - wants[0].float()).abs() <= bounds[0]).all()
    for g, w, b in zip(grads[1:], wants[1:], bounds[1:]):
        got = torch.cat([g[first:first + n] for first, n in zip(starts, lengths)])
        assert ((got.float() - w.float()).abs() <= b).all()
        assert not g[starts[0] + 700:starts[0] + 5000].any() and not g[starts[1] + 600:starts[1] + 5000].any()


def test_tokens_far_apart():
    """Tokens 2^23 values and more from one to the next."""
    rng = np.random.default_rng(19)
    for dtype in (F32, BF16):
        m = Made(([3, 17], None, 2, 1, 64, 0), dtype)
        far = torch.zeros(len(m.k), 2**23 + 8, dtype=dtype, device="cuda")
        for i, x in enumerate((m.k, m.v)):
            far[:, 64 * i:64 * i + 64] = x[:, 0]
        m.k, m.v = far[:, None, :64], far[:, None, 64:128]
        m.check_forward(True)
        m.check_backward(True)


@pytest.mark.parametrize("dtype", TYPES)
def test_broadcast_inputs(dtype):
    """One head's, or one token's, values in place of all: the gradients are those of every one of them."""
    m = Made(([30, 45, 1], None, 4, 4, 64, 0), dtype)
    for name in ("k", "v", "g"):
        x = getattr(m, name)[:, :1].expand(-1, 4, -1)
        setattr(m, name, x)
        setattr(m, name + "64", x.double().cpu().numpy())
    m.check_forward(True)
    m.check_backward(True)
    x = m.k[:1, :1].expand(len(m.q), 4, -1)
    m.k, m.k64 = x, x.double().cpu().numpy()
    m.check_forward(False)
    m.check_backward(False)


def test_heads_without_values():
    """Nothing to add up: every score is 0, and a token's logsum the logarithm of the number of its keys."""
    for dtype in TYPES:
        q, k = torch.empty(9, 4, 0, dtype=dtype, device="cuda"), torch.empty(300, 2, 0, dtype=dtype, device="cuda")
        rows, keys = ints([0, 1, 8]), ints([0, 200, 300])
        out, saved = encoder.attention(q, k, k, rows, keys, causal=True, keep=True)
        counts = np.concatenate([[200.0], np.arange(94.0, 101.0)])
        assert out.shape == q.shape and (saved.logsum[:, 8] == float("-inf")).all()
        near(saved.logsum[:, :8], np.broadcast_to(np.log(counts), (4, 8)), np.full((4, 8), 2.0**-20))
        assert encoder.attention(q, k, k, rows, keys).shape == q.shape
        assert [g.shape for g in encoder.attention_backward(q, q, k, k, saved, rows, keys, causal=True)] == [q.shape, k.shape, k.shape]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [64, 72, 128, 160, 256])
@pytest.mark.parametrize("count,kv", [(3, 3), (4, 2), (4, 1)])
def test_short_rows_among_longer_ones(count, kv, width, dtype):
    """Rows that a wavefront has alone, of no token up to several of its blocks."""
    m = Made(([3, 32, 0, 33, 1, 64, 20, 150, 2, 31] * 3, None, count, kv, width, 0), dtype)
    for causal in (False, True):
        m.check_forward(causal)
        m.check_backward(causal)
