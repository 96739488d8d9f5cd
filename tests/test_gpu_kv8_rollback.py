"""Rows of the 8-bit cache that are taken back (rejected drafts of a verify step) and
written again: what they leave behind, and where it ends."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import Plain, bf16, ints, make_cache, same_cache

pytestmark = pytest.mark.gpu


def write(c, ref, x, pos):
    c.append(x.cuda(), x.cuda(), ints([pos]))
    for kv in (0, 1):
        ref.append(kv, x.float().numpy(), [pos], [x.shape[2]])


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("amp", [3.0, 200.0])
def test_a_large_row_in_the_middle_of_a_page(cuda, page, amp):
    """The page keeps the scale s1 that the large row gave it, and its older codes were
    rounded again: up to (s0 + s1) / 2 off for rows before, s1 / 2 for rows after. The
    next page knows nothing of it."""
    rng = np.random.default_rng(page)
    H, D, n0 = 2, 64, page // 2
    c, clean = (make_cache(np.random.default_rng(3), 1, H, D, page, 4) for _ in range(2))
    ref, ref_clean = Plain(c), Plain(clean)
    rows = bf16(rng, (1, H, 2 * page, D))
    drafts = bf16(rng, (1, H, 3, D), amp)
    for cache, r, drafted in ((c, ref, True), (clean, ref_clean, False)):
        write(cache, r, rows[:, :, :n0], 0)
        if drafted:
            s0 = [t[c.page_table[0, 0]].cpu().numpy().copy() for t in (c.k_scales, c.v_scales)]
            write(cache, r, drafts, n0)
        for i in range(n0, 2 * page):
            write(cache, r, rows[:, :, i:i + 1], i)
        same_cache(cache, r)
    x = rows[0].double().numpy()
    ids = c.page_table[0].cpu().numpy()
    for kv in (0, 1):
        got, plain = ref.rows(kv, 0, 2 * page), ref_clean.rows(kv, 0, 2 * page)
        s1 = ref.scales[kv][ids[0]].astype(np.float64)[:, None, None]
        assert (s1[:, 0, 0] >= float(drafts.float().abs().max()) / 127 * 0.3).all()
        old = (s0[kv].astype(np.float64)[:, None, None] + s1) / 2
        slop = 1 + 2.0 ** -18
        assert (np.abs(got[:, :n0] - x[:, :n0]) <= old * slop).all()
        assert (np.abs(got[:, n0:page] - x[:, n0:page]) <= s1 / 2 * slop).all()
        assert np.array_equal(got[:, page:], plain[:, page:])


def test_a_large_row_that_began_its_page(cuda):
    """The page starts afresh with its first row: nothing is left."""
    rng = np.random.default_rng(5)
    H, D, page = 2, 128, 32
    c, clean = (make_cache(np.random.default_rng(3), 1, H, D, page, 3) for _ in range(2))
    rows, drafts = bf16(rng, (1, H, 2 * page, D)), bf16(rng, (1, H, 4, D), 100.0)
    for cache in (c, clean):
        cache.append(rows[:, :, :page].cuda(), rows[:, :, :page].cuda(), ints([0]))
        if cache is c:
            c.append(drafts.cuda(), drafts.cuda(), ints([page]))
        cache.append(rows[:, :, page:].cuda(), rows[:, :, page:].cuda(), ints([page]))
    for a, b in zip(c.read(ints([2 * page]), 2 * page), clean.read(ints([2 * page]), 2 * page)):
        assert torch.equal(a, b)
    used = c.page_table[0, :2].long()
    assert torch.equal(c.k_scales[used], clean.k_scales[used])
