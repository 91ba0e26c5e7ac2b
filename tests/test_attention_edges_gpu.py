"""Attention where its kernels could go wrong unnoticed: tokens that see nothing next to tokens that do, keys of no weight in front of others, and
float16 where what is multiplied is far below 1."""
import numpy as np
import pytest
import torch

from cudf_amd import encoder
from oracle import encoder_py as orc
from tests.test_attention_gpu import BF16, F16, F32, TYPES, UNIT, Made, ints, near, offsets_of, rounding

pytestmark = pytest.mark.gpu

# Rows with fewer keys than tokens, whose first tokens see nothing if causal: in chunks, in tiles of one and of four wavefronts, in shares.
UNSEEING = [
    ([5], [3], 2, 2, 64, 0), ([70, 6], [20, 200], 2, 1, 64, 0), ([3, 1, 0, 9], [1, 300, 7, 2], 8, 2, 128, 0), ([40, 33], [30, 2], 4, 4, 72, 0), ([800], [400], 2, 1, 64, 0),
    ([300, 200], [129, 64], 3, 3, 256, 0), ([20, 1, 1, 1], [11, 900, 0, 5], 4, 1, 160, 0),
]


def unseeing(m):
    """Of every token whether it sees nothing."""
    none = np.ones(len(m.q), bool)
    for r, keys in enumerate(np.diff(m.key_offsets)):
        first, last = int(m.offsets[r]), int(m.offsets[r + 1])
        none[max(first, last - int(keys)):last] = False
    return none


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", UNSEEING, ids=str)
def test_a_scale_of_zero_and_tokens_that_see_nothing(case, dtype):
    m = Made(case, dtype)
    m.check_forward(True, 0.0)
    none = torch.from_numpy(unseeing(m)).cuda()
    out, saved = encoder.attention(m.q, m.k, m.v, *m.rows(), causal=True, scale=0.0, keep=True)
    assert not out[none].any() and (saved.logsum[:, none] == float("-inf")).all() and not (saved.rest is not None and saved.rest[:, none].any())
    m.check_backward(True, 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("case", UNSEEING, ids=str)
def test_tokens_that_see_nothing(case, value, dtype):
    """The last key of every row, which its last token alone sees, holds anything: those that see nothing have zeros, the others what they have without."""
    m = Made(case, dtype)
    want, log, off, log_off = orc.attention(m.q64, m.k64, m.v64, **m.oracle_rows(), causal=True, **rounding(dtype))
    last = [int(b) - 1 for a, b in zip(m.key_offsets[:-1], m.key_offsets[1:]) if b > a]
    m.v[last] = value
    if value != value:
        m.k[last] = value
    out, saved = encoder.attention(m.q, m.k, m.v, *m.rows(), causal=True, keep=True)
    pick = np.ones(len(m.q), bool)
    pick[[int(b) - 1 for a, b in zip(m.offsets[:-1], m.offsets[1:]) if b > a]] = False
    where, none = torch.from_numpy(pick).cuda(), torch.from_numpy(unseeing(m)).cuda()
    near(out[where], want[pick], off[pick])
    near(saved.logsum[:, where], log[:, pick], log_off[:, pick])
    assert not out[none].any() and (saved.logsum[:, none] == float("-inf")).all() and not (saved.rest is not None and saved.rest[:, none].any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("case", UNSEEING, ids=str)
def test_gradients_of_tokens_that_see_nothing(case, value, dtype):
    """The same on the way back, with infinities in keys too."""
    m = Made(case, dtype)
    want, log, _, _ = orc.attention(m.q64, m.k64, m.v64, **m.oracle_rows(), causal=True)
    out, logsum = torch.from_numpy(want).to(dtype).cuda(), torch.from_numpy(log).float().cuda()
    wants, offs = orc.attention_backward(m.g64, m.q64, m.k64, m.v64, out.double().cpu().numpy(), logsum.double().cpu().numpy(), **m.oracle_rows(), causal=True, **rounding(dtype))
    last = [int(b) - 1 for a, b in zip(m.key_offsets[:-1], m.key_offsets[1:]) if b > a]
    m.k[last] = m.v[last] = value
    q_grad, _, _ = encoder.attention_backward(m.g, m.q, m.k, m.v, encoder.AttentionSaved(out, logsum), *m.rows(), causal=True)
    pick = np.ones(len(m.q), bool)
    pick[[int(b) - 1 for a, b in zip(m.offsets[:-1], m.offsets[1:]) if b > a]] = False
    near(q_grad[torch.from_numpy(pick).cuda()], wants[0][pick], offs[0][pick])
    assert not q_grad[torch.from_numpy(unseeing(m)).cuda()].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,kv", [(2, 2), (4, 1)])
def test_keys_of_no_weight_in_front_of_others(count, kv, dtype):
    """The first 64 keys have scores of -infinity, so the first 64 tokens have no result, and a key that the last token alone sees holds NaN: the tokens
    between have what the keys from 64 on come to."""
    m = Made(([150], None, count, kv, 64, 0), dtype)
    first, last = int(m.offsets[0]), int(m.offsets[1])
    m.q[:, :, 0] = 1.0
    m.k[first:first + 64, :, 0] = float("-inf")
    q64, k64 = m.q.double().cpu().numpy(), m.k.double().cpu().numpy()
    want, log, off, log_off = orc.attention(q64[first + 64:last], k64[first + 64:last], m.v64[first + 64:last], [0, 86], causal=True, **rounding(dtype))
    m.v[last - 1] = float("nan")
    out, saved = encoder.attention(m.q, m.k, m.v, *m.rows(), causal=True, keep=True)
    near(out[first + 64:last - 1], want[:-1], off[:-1])
    near(saved.logsum[:, first + 64:last - 1], log[:, :-1], log_off[:, :-1])
    assert torch.isnan(out[first:first + 64]).all() and torch.isnan(out[last - 1]).all()


class Long:
    """Rows of many tokens in float16, and the gradients in 64 bits from out and logsum as they are given, with how far off a kernel's are to be expected: next to the rounding
    of a result, of each product that is added up half a step of the value (`unit`) that is rounded before it is multiplied, wherever that value lies, and what 32 bits leave of it.
    Roundings are independent of one another, so it is their squares that add up."""

    def __init__(self, lengths, count, kv, width, causal, grad, raise_first=0.0, q_scale=1.0):
        torch.manual_seed(len(lengths) + width)
        self.lengths, self.causal, self.each, tokens = lengths, causal, count // kv, sum(lengths)
        self.q, self.k, self.v, self.g = (torch.randn(tokens, n, width, device="cuda") * s for n, s in ((count, q_scale), (kv, 1.0), (kv, 1.0), (count, grad)))
        self.offsets = offsets_of(lengths)
        if raise_first:  # the first key of every row is what all its tokens look at
            self.q[:, :, 0] = raise_first**0.5 * width**0.25
            self.k[:, :, 0] = 0.0
            self.k[self.offsets[:-1].tolist(), :, 0] = raise_first**0.5 * width**0.25
        self.q, self.k, self.v, self.g = (x.to(F16) for x in (self.q, self.k, self.v, self.g))
        self.scale = width**-0.5

    def check(self):
        unit, eps, width = 2.0**-11, 2.0**-24, self.q.shape[2]
        out, logsum = torch.zeros_like(self.q), torch.full((self.q.shape[1], len(self.q)), float("-inf"), device="cuda")
        wants = [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (self.q, self.k, self.v)]
        squares = [torch.zeros_like(w) for w in wants]
        for first, last in zip(self.offsets[:-1], self.offsets[1:]):
            for h in range(self.q.shape[1]):
                t, u = slice(first, last), h // self.each
                q, k, v, g = self.q[t, h].double(), self.k[t, u].double(), self.v[t, u].double(), self.g[t, h].double()
                s = q @ k.T.contiguous() * self.scale
                if self.causal:
                    s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), float("-inf"))
                log = torch.logsumexp(s, 1)
                out[t, h], logsum[h, t] = (torch.exp(s - log[:, None]) @ v).to(F16), log.float()
                o, log = out[t, h].double(), logsum[h, t].double()
                p = torch.exp(s - log[:, None])
                product = g @ v.T.contiguous()
                ds = p * (product - (g * o).sum(1)[:, None])
                size = self.scale * (q.abs() @ k.abs().T.contiguous())
                e = unit + orc.score_error(size, log.abs()[:, None], width, eps) + 8 * eps
                more = 2 * (width + 4) * eps * (g.abs() @ v.abs().T.contiguous() + (g * o).abs().sum(1)[:, None])
                ds_off, p_off = (e * ds.abs() + p * more) ** 2, (e * p) ** 2
                wants[0][t, h] = self.scale * (ds @ k)
                squares[0][t, h] = self.scale**2 * (ds_off @ k**2)
                wants[1][t, u] += self.scale * (ds.T.contiguous() @ q)
                squares[1][t, u] += self.scale**2 * (ds_off.T.contiguous() @ q**2)
                wants[2][t, u] += p.T.contiguous() @ g
                squares[2][t, u] += p_off.T.contiguous() @ g**2
        self.wants, self.squares = wants, squares
        got = encoder.attention_backward(self.g, self.q, self.k, self.v, encoder.AttentionSaved(out, logsum), ints(self.offsets), causal=self.causal)
        return [self.error(x, w, s) for x, w, s in zip(got, wants, squares)]

    def error(self, got, want, square, pick=slice(None)):
        """(how far off, how far to be expected): (of a result, half a step, which is 2^-25 where it is smallest).  A result of more than float16 holds,
        65520 and more as it is rounded, is an infinity; those that are off by less from that than by 2^-8 may be either."""
        got, want, square = got[pick].double(), want[pick], square[pick]
        beyond, below = want.abs() >= 65520 * (1 + 2.0**-8), want.abs() <= 65520 * (1 - 2.0**-8)
        assert torch.equal(got[beyond], torch.copysign(torch.full_like(want[beyond], float("inf")), want[beyond]))
        got, want, square = got[below], want[below], square[below]
        half = torch.maximum(2.0**-11 * want.abs(), torch.full_like(want, 2.0**-25))
        return (got - want).norm().item(), (square + half**2).sum().sqrt().item()


@pytest.mark.parametrize("lengths,count,kv,width,causal,grad", [
    ([4096], 2, 2, 64, False, 1e-3), ([2000], 4, 1, 64, True, 1e-3), ([2000], 4, 1, 128, True, 1e-4), ([8192], 1, 1, 64, False, 1e-4), ([1500, 700], 2, 1, 72, True, 1e-3),
    ([300] * 12, 12, 6, 64, True, 1e-3), ([300] * 12, 12, 6, 128, False, 1e-3), ([40] * 50, 4, 2, 64, True, 1e-4), ([40] * 50, 4, 2, 256, False, 1e-4), ([1000], 2, 2, 256, True, 1e-3),
    ([500], 2, 2, 64, False, 8e3), ([40] * 50, 4, 2, 128, True, 8e3),
])
def test_float16_gradients_keep_their_bits(lengths, count, kv, width, causal, grad):
    """Probabilities of some thousandths and gradients of a loss that is a mean, or that has been scaled up: what is rounded before it is multiplied lies below float16's normal
    numbers, or beyond its largest, but its sums do not."""
    for name, (error, expected) in zip("qkv", Long(lengths, count, kv, width, causal, grad).check()):
        assert error <= expected, (name, error, expected)


def self_log(m, first, last, h):
    s = m.q[first:last, h].double() @ m.k[first:last, h // m.each].double().T.contiguous() * m.scale
    if m.causal:
        s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), float("-inf"))
    return torch.logsumexp(s, 1).float()


@pytest.mark.parametrize("lengths,count,kv,width,causal", [([2000], 2, 1, 64, True), ([900] * 3, 4, 4, 128, False), ([60] * 40, 4, 2, 64, True), ([500] * 4, 4, 4, 256, False)])
def test_float16_probabilities_keep_their_bits(lengths, count, kv, width, causal):
    """One key has nearly all the weight of all tokens: the gradients of the others' values are sums of probabilities of 2^-20."""
    m = Long(lengths, count, kv, width, causal, 50.0, raise_first=14.0, q_scale=0.3)
    m.check()
    out = torch.zeros_like(m.q)
    others = torch.ones(len(m.q), dtype=torch.bool, device="cuda")
    others[m.offsets[:-1].tolist()] = False
    logsum = torch.stack([torch.cat([self_log(m, a, b, h) for a, b in zip(m.offsets[:-1], m.offsets[1:])]) for h in range(count)])
    v_grad = encoder.attention_backward(m.g, m.q, m.k, m.v, encoder.AttentionSaved(out, logsum), ints(m.offsets), causal=causal)[2]
    error, expected = m.error(v_grad, m.wants[2], m.squares[2], others)
    assert error <= expected, (error, expected)


@pytest.mark.parametrize("gap", [16.0, 22.0, 22.59375, 24.40625])
@pytest.mark.parametrize("tokens,count", [(128, 1024), (33, 512)])
def test_float16_weights_far_below_the_largest(gap, tokens, count):
    """One key's weight is 2^gap times that of each of 131071 others, which have values of 1 where it has 0: a weight is off by half a step of it (unit) or by 2^-32, half of
    float16's smallest number next to a largest weight of 2^7 and more; of their two sums, the scores and the exponentials 32 bits are left, n additions of 2^-24."""
    n, unit = 131072, 2.0**-11
    q, k, v = (torch.zeros(t, c, 64, dtype=F16, device="cuda") for t, c in ((tokens, count), (n, 1), (n, 1)))
    q[:, :, 0], k[0, :, 0], v[1:] = 1.0, gap, 1.0
    out, saved = encoder.attention(q, k, v, ints([0, tokens]), ints([0, n]), scale=float(np.log(2.0)), keep=True)
    mass = (n - 1) * 2.0**-gap
    want = mass / (1 + mass)
    most = want * (3 * unit + 2 * n * 2.0**-24 + 2.0**-18) + n * 2.0**-32
    assert (out.double() - want).abs().max().item() <= most
    assert (saved.logsum.double() - (gap * np.log(2.0) + np.log1p(mass))).abs().max().item() <= 2.0**-18 * gap + n * 2.0**-24


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_over_their_own_keys_take_no_memory_for_parts(dtype):
    """No row of few tokens over its own keys is in several chunks: the call needs no memory but its result."""
    q, k = torch.randn(8192, 8, 128, device="cuda").to(dtype), torch.randn(8192, 1, 128, device="cuda").to(dtype)
    rows = torch.arange(0, 8193, 4, dtype=torch.int32, device="cuda")
    encoder.attention(q, k, k, rows)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = encoder.attention(q, k, k, rows)
    assert torch.cuda.max_memory_allocated() - before <= out.numel() * out.element_size() + 4096


def by_what_is_seen(m):
    """Forward results and gradients in 64 bits where inputs are infinite or NaN: each token's sums over what it sees alone, with 0 times such a value NaN; out and logsum
    of the forward pass go on as they are."""
    q, k, v, g = (x.double().cpu().numpy() for x in (m.q, m.k, m.v, m.g))
    scale, each = q.shape[2] ** -0.5, q.shape[1] // k.shape[1]
    out, log = np.zeros(q.shape), np.full(q.shape[:2][::-1], -np.inf)
    grads = [np.zeros(x.shape) for x in (q, k, v)]
    with np.errstate(all="ignore"):
        for first, last in zip(m.offsets[:-1], m.offsets[1:]):
            for h in range(q.shape[1]):
                for t in range(first, last):
                    keys = slice(first, t + 1)
                    kk, vv = k[keys, h // each], v[keys, h // each]
                    s = scale * (kk * q[t, h]).sum(1)
                    top = s.max()
                    e = np.exp(s - (0.0 if top == -np.inf else top))
                    log[h, t] = top + np.log(e.sum())
                    p = e / e.sum()
                    out[t, h] = (p[:, None] * vv).sum(0)
                    ds = p * ((vv * g[t, h]).sum(1) - (g[t, h] * out[t, h]).sum())
                    grads[0][t, h] = scale * (ds[:, None] * kk).sum(0)
                    grads[1][keys, h // each] += scale * ds[:, None] * q[t, h]
                    grads[2][keys, h // each] += p[:, None] * g[t, h]
    return out, log, grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,count,kv,width", [([150, 40, 3], 2, 1, 64), ([33] * 6, 4, 2, 72), ([700], 2, 2, 64), ([140, 20], 2, 1, 256)])
@pytest.mark.parametrize("where", ["v", "g", "k", "tokens", "all of g"])
def test_what_is_not_finite_stays_with_those_that_see_it(where, lengths, count, kv, width, dtype):
    """Infinities and NaN here and there in values or gradients, in keys, of whole tokens, and everywhere: results are finite where they are for what is seen, and as they are without the
    others (to twice what a kernel's may be off by: 16-bit types and sums of 700 in 32 bits, of magnitudes of about 1)."""
    m = Made((lengths, None, count, kv, width, 0), dtype, seed=5)
    odd = torch.tensor([float("inf"), float("-inf"), float("nan")], device="cuda").to(dtype)
    pick = lambda shape, n: tuple(torch.from_numpy(m.rng.integers(0, s, n)).cuda() for s in shape)
    tokens = sum(lengths)
    if where in ("v", "g", "k"):
        x = getattr(m, where)
        at = pick(x.shape, tokens // 8)
        x[at] = odd[torch.from_numpy(m.rng.integers(0, 3, tokens // 8)).cuda()] if where != "k" else float("nan")
    elif where == "tokens":
        for t in m.rng.integers(m.offsets[0], m.offsets[-1], 3):
            m.q[t] = m.k[t] = m.v[t] = m.g[t] = float("nan")
    else:
        m.g[:] = float("inf")
    want, log, wants = by_what_is_seen(m)
    out, saved = encoder.attention(m.q, m.k, m.v, *m.rows(), causal=True, keep=True)
    grads = encoder.attention_backward(m.g, m.q, m.k, m.v, saved, *m.rows(), causal=True)
    near_where_finite(out, want, dtype, 1.0)
    near_where_finite(saved.logsum, log, F32, 16.0)
    for x, w in zip(grads, wants):
        near_where_finite(x, w, dtype, 32.0)


def near_where_finite(got, want, dtype, size):
    got = got.double().cpu().numpy()
    finite = np.isfinite(want) | (want == -np.inf if got.ndim == 2 else False)
    assert np.array_equal(np.isfinite(got) | (got == -np.inf if got.ndim == 2 else False), finite)
    inside = np.isfinite(want)
    assert (np.abs(got[inside] - want[inside]) <= 4 * (UNIT[dtype] + 2.0**-13) * (np.abs(want[inside]) + size)).all()


@pytest.mark.parametrize("back", [3, 11])
def test_tokens_that_overlap(back):
    """Keys and values that lie a few values apart, each within the last: NaN behind the last one's 64 values (which end 8 in front of the memory's end) is nobody's, and among them it
    is that key's, and nobody else's."""
    for dtype in TYPES:
        memory = torch.randn(33 * 8 + 64, device="cuda").to(dtype)
        x = memory.as_strided((33, 1, 64), (8, 64, 1))
        q = torch.randn(33, 2, 64, device="cuda").to(dtype)
        memory[-back] = float("nan")
        apart = x.contiguous()
        assert torch.isnan(apart).sum() == (1 if back > 8 else 0)
        out, want = encoder.attention(q, x, x, ints([0, 33])), encoder.attention(q, apart, apart, ints([0, 33]))
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        k = torch.randn(33, 1, 64, device="cuda").to(dtype)
        out, want = encoder.attention(q, k, x, ints([0, 33])), encoder.attention(q, k, apart, ints([0, 33]))
        odd = torch.isnan(apart).any(0)[0]
        assert torch.equal(torch.isnan(out), odd.expand(33, 2, 64)) and torch.equal(out[:, :, ~odd], want[:, :, ~odd])


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("which", ["token", "tokens", "gradient", "gradients"])
def test_what_is_not_finite_does_not_take_long(which, causal):
    """NaN in one token or in all, or a gradient that has overflowed: a step over 4096 tokens takes less than 30 times as long as one without (it took 300 to 1000 times as long
    where every row that is not finite was made once more)."""
    torch.manual_seed(3)
    n = 4096
    q, k, v, g = (torch.randn(n, h, 64, device="cuda").to(BF16) for h in (8, 4, 4, 8))

    def step(q, k, v, g):
        out, saved = encoder.attention(q, k, v, ints([0, n]), causal=causal, keep=True)
        return encoder.attention_backward(g, q, k, v, saved, ints([0, n]), causal=causal)

    def time(*args):
        step(*args)
        torch.cuda.synchronize()
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(3):
            step(*args)
        end.record()
        torch.cuda.synchronize()
        return begin.elapsed_time(end)

    clean = time(q, k, v, g)
    if which in ("token", "tokens"):
        for x in (q, k, v, g):
            x[7 if which == "token" else slice(None)] = float("nan")
    else:
        g[n - 7 if which == "gradient" else slice(None)] = float("inf")
    assert time(q, k, v, g) < 30 * clean


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,keys", [([40, 33, 0, 50] * 8, [150, 90, 3, 260] * 8), ([20, 90] * 12, [30, 95] * 12), ([60] * 20, [61] * 20)])
def test_short_rows_over_more_keys_than_tokens(lengths, keys, dtype):
    """Short rows of tokens over caches of more keys, which four wavefronts share, and over few, which one has alone."""
    m = Made((lengths, keys, 8, 8, 64, 0), dtype, roomy=True)
    m.check_forward(True)
    m.check_backward(True)
