"""Eviction where pages are not there: rows to or from them do not move, in the cache,
the weights and the positions alike, and what stays keeps its value."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import Plain, ints, make_cache
from vates_b200 import _lib

pytestmark = pytest.mark.gpu
F32 = np.float32


def evict_plain(ref, pages, w, p, lens, keep, first, recent):
    """The rule row by row, in place. The rows of a page that is not there have no new row
    and give none, so the row that one of them would have replaced is there still."""
    page = ref.page
    there = lambda i: 0 <= i < pages
    for b, n in enumerate(lens):
        if n <= keep:
            continue
        for h in range(w.shape[1]):
            at = p[b, h, :n].astype(np.int64)
            safe = (np.arange(n) < first) | (at > at.max() - recent)
            order = np.lexsort((np.arange(n), -w[b, h, :n], ~safe))
            kept = np.zeros(n, bool)
            kept[order[:keep]] = True
            holes, tail = np.flatnonzero(~kept[:keep]), keep + np.flatnonzero(kept[keep:])
            moves = [(d, s) for d, s in zip(holes, tail)
                     if there(ref.table[b, d // page]) and there(ref.table[b, s // page])]
            old = [s.copy() for s in ref.scales]
            for pg in sorted({d // page for d, _ in moves}):
                pid = ref.table[b, pg]
                mine = [(d, s, ref.table[b, s // page]) for d, s in moves if d // page == pg]
                rows = np.arange(pg * page, min((pg + 1) * page, keep))
                stay = np.setdiff1d(rows, [d for d, _, _ in mine])
                for kv in range(2):
                    codes, scales = ref.codes[kv], ref.scales[kv]
                    top = F32(max([old[kv][i, h] for _, _, i in mine]
                                  + ([old[kv][pid, h]] if len(stay) else [])))
                    if top > 0 and len(stay) and old[kv][pid, h] != top:
                        r = F32(old[kv][pid, h] / top)
                        codes[pid, h, stay % page] = np.rint(codes[pid, h, stay % page].astype(F32) * r)
                    for d, s, i in mine:
                        r = F32(old[kv][i, h] / top) if top > 0 else F32(1)
                        codes[pid, h, d % page] = np.rint(codes[i, h, s % page].astype(F32) * r)
                    scales[pid, h] = top
            for x in (w, p):
                d, s = [d for d, _ in moves], [s for _, s in moves]
                x[b, h, d] = x[b, h, s]
    return [min(n, keep) for n in lens]


# of a table of ten pages: no source; some; some that rows go to; all but the first; the one
# in which `keep` falls, whose rows move and are moved to
MISSING = {"sources": range(4, 10), "some sources": (5, 8), "targets": (0, 2),
           "both": range(1, 10, 2), "edge": (3,), "all but one": range(1, 10), "all": range(10)}


@pytest.mark.parametrize("what", MISSING)
@pytest.mark.parametrize("dim,page", [(64, 16), (64, 64), (128, 32), (256, 64), (256, 128)])
def test_rows_of_missing_pages_do_not_move(cuda, dim, page, what):
    rng = np.random.default_rng(dim + page)
    B, H, n = 3, 2, 10 * page
    c = make_cache(rng, B, H, dim, page, 10)
    # scales far apart: a row that should not have moved, or been rounded again, shows
    for t in (c.k_scales, c.v_scales):
        t.copy_(torch.from_numpy((2.0 ** rng.uniform(-8, 0, t.shape)).astype(F32)))
    bad = np.array([-1, c.pages, 10 ** 6, -7])
    table = c.page_table.cpu().numpy()
    for b in range(2):  # the last sequence has all of its pages
        for k, pg in enumerate(MISSING[what]):
            table[b, pg] = bad[(k + b) % 4]
    c.page_table.copy_(torch.from_numpy(table))
    keep = 3 * page + page // 2 + 1
    w = rng.exponential(1.0, (B, H, n)).astype(F32)
    w[0, :, page:2 * page] = 0  # a page that is refilled whole
    w[:, :, keep:] *= 3
    p = rng.permuted(np.tile(np.arange(n, dtype=np.int32), (B, H, 1)), axis=-1)
    ref, status = Plain(c), torch.zeros(1, dtype=torch.int32, device="cuda")
    tw, tp = torch.from_numpy(w).cuda(), torch.from_numpy(p).cuda()
    lens = [n, n - 5, n - 1]
    after = c.evict(tw, ints(lens), keep, first=3, recent=page // 2, positions=tp, status=status)
    want = evict_plain(ref, c.pages, w, p, lens, keep, 3, page // 2)
    assert after.tolist() == want and int(status) == _lib.VB_STATUS_BOUNDS
    assert np.array_equal(tw.cpu().numpy(), w)
    assert np.array_equal(tp.cpu().numpy(), p)
    for t, r in zip((c.k_scales, c.v_scales, c.k_codes, c.v_codes), ref.scales + ref.codes):
        assert np.array_equal(t.cpu().numpy(), r)
