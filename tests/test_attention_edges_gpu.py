"""Attention where its kernels could go wrong unnoticed: tokens that see nothing next to tokens that do."""
import numpy as np
import pytest
import torch

from cudf_amd import encoder
from tests.test_attention_gpu import TYPES, Made

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
