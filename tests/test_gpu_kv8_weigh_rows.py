"""Accumulated attention weight of more than 32 query rows per kv head: rows that do
not count, and sequences without rows."""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv8 import bf16, ints, make_cache
from test_gpu_kv8_evict import check_weigh
from vates_b200 import _lib
from vates_b200.kv8 import PagedKV8Cache

pytestmark = pytest.mark.gpu


def spoil(q, rows, xs=(math.nan, math.inf, -math.inf)):
    """One value of each (head, row) of sequence 0 that is not finite; the mask of the rows."""
    bad = torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")
    for k, (h, i) in enumerate(rows):
        q[0, h, i, (7 * k + 3) % q.shape[3]] = xs[k % len(xs)]
        bad[0, h, i] = True
    return bad


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,page,L,rep,keys", [(64, 16, 40, 8, 700), (128, 32, 33, 1, 515),
                                                 (256, 64, 64, 8, 1500), (128, 128, 100, 7, 300),
                                                 (64, 64, 5, 7, 1), (256, 16, 300, 2, 4000)])
def test_rows_that_are_not_finite_add_nothing(cuda, dim, page, L, rep, keys, causal):
    """A NaN or an infinity in a query makes its lse NaN: the row adds nothing, and every
    other row what it adds without it, in each of several passes over the rows."""
    rng = np.random.default_rng(dim + L + keys)
    c = make_cache(rng, 2, 2, dim, page, -(-keys // page))
    q = bf16(rng, (2, 2 * rep, L, dim), 1.5).cuda()
    lens, ql = [keys, max(1, keys // 2)], [min(L, keys), min(L, max(1, keys // 2))]
    last = ql[0] - 1
    bad = spoil(q, {(0, 0), (rep - 1, last), (rep, last // 2), (2 * rep - 1, last // 3), (0, last)})
    _, lse = c.attend(q, ints(lens), ints(ql), causal=causal, return_lse=True)
    assert lse[bad].isnan().all()
    check_weigh(c, q, lens, ql, causal=causal, lse=lse)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    w = torch.zeros((2, 2, keys + 3), device="cuda")
    c.weigh(q, lse, ints(lens), w, ints(ql), causal=causal, status=status)
    assert int(status) == _lib.VB_STATUS_NONFINITE and torch.isfinite(w).all()
    # the same rows left out by their lse alone
    status.zero_()
    want = torch.zeros_like(w)
    c.weigh(torch.where(bad[..., None], 1.0, q), torch.where(bad, -math.inf, lse), ints(lens), want,
            ints(ql), causal=causal, status=status)
    assert int(status) == 0 and torch.equal(w, want)


def test_scores_that_overflow_add_nothing(cuda):
    """Scores past float32: lse is not finite although every query value is."""
    rng = np.random.default_rng(3)
    c = make_cache(rng, 1, 1, 128, 32, 20)
    c.k_scales.mul_(2.0 ** 20)
    q = bf16(rng, (1, 4, 20, 128))
    q[0, 1, 3] *= 2.0 ** 126
    q[0, 3, 19] *= 2.0 ** 126
    q = q.cuda()
    lens = ints([600])
    _, lse = c.attend(q, lens, return_lse=True)
    bad = ~torch.isfinite(lse)
    assert bad[0, 1, 3] and bad[0, 3, 19] and int(bad.sum()) == 2
    check_weigh(c, q, [600], lse=lse)


def test_no_row_counts(cuda):
    rng = np.random.default_rng(4)
    c = make_cache(rng, 2, 1, 64, 16, 30)
    q = torch.full((2, 4, 40, 64), math.nan, dtype=torch.bfloat16, device="cuda")
    lens = [480, 100]
    _, lse = c.attend(q, ints(lens), return_lse=True)
    assert lse.isnan().all()
    w = check_weigh(c, q, lens, new=[0, 7], lse=lse)
    assert not w[1, :, 93:100].any()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("L", [2, 33, 200])
def test_scales_of_zero_and_tiny_ones(cuda, L, causal):
    """A page with scale 0 has scores of 0 whatever its codes and the queries are, and the
    smallest scales count as any other."""
    rng = np.random.default_rng(L)
    c = make_cache(rng, 2, 2, 128, 16, 40)
    q = bf16(rng, (2, 4, L, 128)) * 2.0 ** 100
    c.k_scales.fill_(0)
    check_weigh(c, q.cuda(), [640, 201], causal=causal)
    c.k_scales[::2] = 2.0 ** -110
    check_weigh(c, q.cuda(), [640, 201], causal=causal, scale=2.0 ** -3)


@pytest.mark.parametrize("L", [4, 40])
def test_longest_sequence(cuda, L):
    """As many keys as a table may have, less than 2^31 - 65536, which all lie in one page:
    new rows alone, without query rows, and then a row that sees them all."""
    keys, pad = (1 << 31) - 65536 - 128, 1 << 31
    c = PagedKV8Cache.empty(1, 1, 64, 1, keys // 128, 128)
    c.page_table.zero_()
    # what lies in front of the weights is not written
    room = torch.ones(pad + keys, device="cuda")
    w = room[pad:].view(1, 1, keys)
    q, lse = torch.zeros((1, 1, L, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((1, 1, L), device="cuda")
    c.weigh(q, lse, ints([keys]), w, ints([0]), new=ints([100_000]))
    assert float(room[:-100_000].min()) == float(room[:-100_000].max()) == 1
    assert not room[-100_000:].any()
    c.weigh(q, lse, ints([keys]), w, ints([1]), new=ints([9]), causal=False)
    assert float(room[:pad].min()) == float(room[:pad].max()) == 1
    assert float(w[..., :-100_000].min()) == float(w[..., :-100_000].max()) == 2
    assert float(w[..., -100_000:].min()) == float(w[..., -100_000:].max()) == 1
