"""Attention where its kernels could go wrong unnoticed: tokens that see nothing next to tokens that do, keys of no weight in front of others."""
import numpy as np
import pytest
import torch

from cudf_amd import encoder
from oracle import encoder_py as orc
from tests.test_attention_gpu import TYPES, Made, near, rounding

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
