"""Token log probabilities of rows at the ends of the number range."""
import math

import numpy as np
import pytest
import torch

from test_gpu_logprobs import logits, plain
from vates_b200.logprobs import token_logprobs

pytestmark = pytest.mark.gpu

# one logit per thread, one CTA, several slices of a row
SIZES = [300, 8001, 151936]


def ints(a):
    return torch.tensor([int(x) for x in a], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, (0x7FC0, 0x7FFF, 0xFF81, 0xFFFF)),
                                        (torch.float32, (0x7FC00000, 0x7FFFFFFF, 0xFF800001,
                                                         0xFFFFFFFF))])
def test_nothing_is_ahead_of_a_nan(cuda, V, dtype, bits):
    """Every NaN pattern, as the token's own logit: rank 0, NaN results."""
    rng = np.random.default_rng(V)
    x = logits(rng, len(bits), V, dtype)
    raw = x.view(torch.int16 if dtype == torch.bfloat16 else torch.int32)
    tok = [0, V - 1, V // 2, V // 3]
    for r, (t, b) in enumerate(zip(tok, bits)):
        raw[r, t] = b - (1 << (16 if dtype == torch.bfloat16 else 32)) if b >> (
            15 if dtype == torch.bfloat16 else 31) else b
    assert x[range(4), tok].isnan().all()
    got = token_logprobs(x.cuda(), ints(tok), top=3)
    assert got.rank.tolist() == [0] * 4
    assert got.logprob.isnan().all() and got.entropy.isnan().all()
