"""Attention over the 8-bit cache at its edges, by both kernels: up to 32 query rows
per key/value head (``few``) and more (``many``), with the keys in one tile, in
several tiles and in several ranges."""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv8 import Plain, attend_plain, bf16, check_attend, ints, make_cache
from vates_b200 import _lib

pytestmark = pytest.mark.gpu

ROWS = [pytest.param(1, 2, id="few"), pytest.param(20, 4, id="many")]
KEYS = [pytest.param(100, id="tile"), pytest.param(380, id="tiles"),
        pytest.param(3000, id="ranges")]


def both(fn):
    for mark in (pytest.mark.parametrize("L,rep", ROWS), pytest.mark.parametrize("keys", KEYS),
                 pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (256, 64)])):
        fn = mark(fn)
    return fn


def setup(L, rep, keys, dim, page, seed=0, heads=1, amp=1.0):
    rng = np.random.default_rng(seed + 7 * L + keys + dim)
    c = make_cache(rng, 1, heads, dim, page, -(-keys // page) + 2)
    return c, bf16(rng, (1, heads * rep, L, dim), amp)


def pages(c, *which):
    """Pool pages of the table's entries at these fractions of it."""
    n = c.page_table.shape[1] - 2
    return [int(c.page_table[0, min(n - 1, int(f * n))]) for f in which]


@both
def test_pages_blanked_by_their_scale(cuda, L, rep, keys, dim, page):
    """Scale 0 makes a page's keys or values 0 whatever its codes are."""
    c, q = setup(L, rep, keys, dim, page)
    a, b, d = pages(c, 0.0, 0.4, 0.9)
    c.k_scales[a] = 0
    c.v_scales[b] = 0
    c.k_scales[d] = c.v_scales[d] = 0
    check_attend(c, q.cuda(), [keys], None)
    check_attend(c, q.cuda(), [keys], None, causal=False)
    c.v_scales.zero_()
    out, lse = c.attend(q.cuda(), ints([keys]), return_lse=True)
    assert not out.any()
    c.k_scales.zero_()
    out, lse = c.attend(q.cuda(), ints([keys]), return_lse=True)
    seen = torch.arange(keys - L + 1, keys + 1, dtype=torch.float64).log()
    # equal weights of 2^6 to 2^15.5 whose sum is exact: log2 of it (below 2^5 each,
    # within an ulp) and two float32 steps
    assert (lse.cpu() - seen).abs().max() <= 2.0 ** -17


@both
def test_keys_of_vanishing_values_keep_their_weight(cuda, L, rep, keys, dim, page):
    """Equal scores over pages whose V scales lie 2^140 apart: the small values add
    nothing, but their keys are as likely as the others."""
    c, q = setup(L, rep, keys, dim, page)
    c.k_scales.zero_()
    c.v_scales.fill_(2.0 ** -40)
    c.v_scales[pages(c, 0.0, 0.5)] = 2.0 ** 100
    check_attend(c, q.cuda(), [keys], None, causal=False)
