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


def compare(x, tok, top, T):
    """Against float64: in float32's range of results to 2^-20 of them (three float32
    roundings, and the sums' share as in `plain`), beyond it infinite."""
    got = token_logprobs(x.cuda(), ints(tok), top=top, temperature=T)
    with np.errstate(over="ignore"):
        want = plain(x.float().numpy(), np.asarray(tok), top, T)
    assert np.array_equal(got.rank.cpu().numpy(), want["rank"])
    assert np.array_equal(got.top_ids.cpu().numpy(), want["ids"])
    for name, key in (("logprob", "logprob"), ("entropy", "entropy"), ("top_logprobs", "top")):
        g = getattr(got, name).cpu().numpy().astype(np.float64)
        ref, tol = want[key]
        out = ref < -float(np.finfo(np.float32).max)
        assert np.isneginf(g[out]).all()
        assert (np.abs(g[~out] - ref[~out]) <= tol[~out]).all(), (name, g, ref)


@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1.0, 0.7, 20.0])
def test_rows_of_the_lowest_values(cuda, V, dtype, T):
    """Allowed logits that all hold the type's lowest value beside -inf for the others,
    a few of them larger but still enormous, and all of them alike."""
    rng = np.random.default_rng(V)
    low = torch.finfo(dtype).min
    x = torch.full((4, V), -math.inf, dtype=dtype)
    allowed = rng.choice(V, (4, 37), replace=True)
    for r in range(4):
        x[r, allowed[r]] = low
    x[1, allowed[1][5]] = x[1, allowed[1][9]] = -2e32
    x[2, allowed[2][3]] = -1.5
    x[3] = low
    compare(x, [allowed[0][0], allowed[1][5], allowed[2][4], V - 1], 20, T)
    compare(x, [allowed[0][3], allowed[1][6], allowed[2][3], 0], 0, T)


@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1.0, 1.7])
def test_tokens_masked_with_the_lowest_value(cuda, V, dtype, T):
    """Their log probability is the lowest value over T, not just something low."""
    rng = np.random.default_rng(V + 1)
    x = logits(rng, 3, V, dtype)
    x[torch.from_numpy(rng.random((3, V)) < 0.6)] = torch.finfo(dtype).min
    x[1] = torch.finfo(dtype).min
    x[1, 7] = 3.0
    tok = [int((x[r] == torch.finfo(dtype).min).nonzero()[-1]) for r in range(3)]
    compare(x, tok, 20, T)
