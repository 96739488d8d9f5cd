"""Shared prefixes with queries that are not finite: what attention of every sequence
by itself gives, in every form that the call takes."""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv8 import bf16, ints, make_cache
from test_gpu_kv8_shared import share

pytestmark = pytest.mark.gpu

# batch, rows, heads per kv head, dim, page, prefix, own keys: both parts in one launch;
# by the decode kernel, beside each other; the prefix, or both, by the prompt kernel (one
# row tile, several, dealt); rows joined by 1024 / dim threads, by two and by one
FORMS = [(2, 1, 4, 128, 32, 384, 40), (3, 2, 5, 64, 16, 256, 200), (2, 2, 8, 256, 64, 16384, 900),
         (4, 1, 8, 64, 16, 8192, 3000), (12, 1, 8, 128, 64, 640, 90), (64, 4, 6, 256, 64, 2048, 70),
         (3, 40, 2, 128, 128, 512, 300), (9, 130, 2, 64, 32, 320, 150), (40, 2, 10, 64, 16, 800, 33)]


def spoiled(rng, B, L, rep, dim):
    """Queries, clean and with values that are not finite, and the mask of the rows."""
    q = bf16(rng, (B, 2 * rep, L, dim), 1.5).cuda()
    bad = torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")
    p = q.clone()
    for k, x in enumerate((math.nan, math.inf, -math.inf, math.nan)):
        b, h, i = k * (B - 1) // 3, k * (2 * rep - 1) // 3, (L - 1) * (k % 2)
        p[b, h, i, (11 * k + 5) % dim] = x
        bad[b, h, i] = True
    p[B // 2, rep, L // 2] = math.nan  # a whole row
    bad[B // 2, rep, L // 2] = True
    return q, p, bad


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,L,rep,dim,page,prefix,own", FORMS)
def test_nonfinite_queries_stay_in_their_row(cuda, B, L, rep, dim, page, prefix, own, causal):
    rng = np.random.default_rng(B + L + dim)
    c = make_cache(rng, B, 2, dim, page, -(-(prefix + own) // page))
    q, p, bad = spoiled(rng, B, L, rep, dim)
    plan = share(c, [(0, B, prefix)])
    lens = ints([prefix + max(L, int(x)) for x in rng.integers(1, own, B)])
    clean, cl = c.attend_shared(q, lens, plan, causal=causal, return_lse=True)
    out, lse = c.attend_shared(p, lens, plan, causal=causal, return_lse=True)
    assert out[bad].isnan().all() and lse[bad].isnan().all()
    assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse[~bad], cl[~bad])
    # and so in the attention of every sequence by itself
    each, el = c.attend(p, lens, causal=causal, return_lse=True)
    assert torch.equal(each.isnan(), out.isnan()) and torch.equal(el.isnan(), lse.isnan())


def test_a_sequence_without_own_keys_or_prefix(cuda):
    """Rows that have keys in one of the parts only, and rows without keys beside them."""
    rng = np.random.default_rng(5)
    c = make_cache(rng, 5, 2, 64, 16, 40)
    q, p, bad = spoiled(rng, 5, 2, 8, 64)
    p[0, 1, 1] = p[1, 2, 0] = p[2, 3, 0] = p[4, 4, 1] = math.nan
    plan = share(c, [(0, 4, 320)])
    lens, ql = ints([320, 200, 0, 322, 50]), ints([2, 1, 0, 2, 2])
    out, lse = c.attend_shared(p, lens, plan, ql, return_lse=True)
    each, el = c.attend(p, lens, ql, return_lse=True)
    assert lse[0, 1, 1].isnan() and lse[1, 2, 0].isnan() and lse[4, 4, 1].isnan()
    assert torch.isneginf(lse[2]).all() and not out[2].any()
    assert torch.equal(each.isnan(), out.isnan()) and torch.equal(el.isnan(), lse.isnan())
    assert torch.equal(torch.isneginf(el), torch.isneginf(lse))


def test_scores_that_overflow(cuda):
    """Scores past float32, of one sign or both, in both parts or one of them."""
    rng = np.random.default_rng(6)
    c = make_cache(rng, 4, 1, 128, 32, 30)
    c.k_scales.mul_(2.0 ** 20)
    plan = share(c, [(0, 4, 640)])
    q = bf16(rng, (4, 4, 2, 128))
    q[0, 0, 0] *= 2.0 ** 126
    q[1, 1, 1] *= 2.0 ** 126
    q[3, 3, 0] *= 2.0 ** 126
    lens = ints([700, 643, 900, 642])
    out, lse = c.attend_shared(q.cuda(), lens, plan, return_lse=True)
    each, el = c.attend(q.cuda(), lens, return_lse=True)
    assert int((~torch.isfinite(el)).sum()) == 3
    assert torch.equal(torch.isfinite(el), torch.isfinite(lse))
    assert torch.equal(torch.isfinite(each), torch.isfinite(out))
