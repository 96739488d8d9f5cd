"""Accumulated attention weight and eviction over the paged 8-bit cache against
plain forms: 64-bit for the weights, exact for what is evicted and moved."""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv8 import Plain, bf16, ints, make_cache
from vates_b200 import _lib
from vates_b200.kv8 import PagedKV8Cache, SharedPrefix

pytestmark = pytest.mark.gpu
F32 = np.float32


# -------------------------------------------------------------------- weigh
def weigh_plain(ref, q, lse, lens, q_lens, scale, causal):
    """float64 sums [B, H, keys] per sequence, and a bound on the kernel's error.

    A term e = exp(z - lse) is off by the score's error (a float32 sum of D
    products: D 2^-24 of sum |q k|, and 2^-22 for the steps after it), by lse in
    units of log 2 (2^-22 of it) and by the exponential (2^-20), each relative to e;
    a sum of R terms by R 2^-23 of it."""
    B, Hq, L, D = q.shape
    H = ref.codes[0].shape[1]
    rep = Hq // H
    sums, tols = [], []
    for b in range(B):
        n, ql = lens[b], q_lens[b]
        K = ref.rows(0, b, n)
        s, t = np.zeros((H, n)), np.zeros((H, n))
        for h in range(Hq):
            k = K[h // rep]
            for i in range(ql):
                m = max(0, n - ql + i + 1) if causal else n
                if m == 0 or not np.isfinite(lse[b, h, i]):
                    continue
                z = k[:m] @ q[b, h, i] * scale
                mag = np.abs(k[:m]) @ np.abs(q[b, h, i]) * scale
                e = np.exp(z - lse[b, h, i])
                rel = mag * (D * 2.0 ** -24 + 2.0 ** -22) + abs(lse[b, h, i]) * 2.0 ** -22 + 2.0 ** -20
                s[h // rep, :m] += e
                t[h // rep, :m] += e * (rel + rep * ql * 2.0 ** -23)
        sums.append(s)
        tols.append(t)
    return sums, tols


def check_weigh(c, q, lens, q_lens=None, new=None, causal=True, len_add=0, extra=5, lse=None,
                positions=True, scale=None, seed=0):
    B, Hq, L, D = q.shape
    H = c.kv_heads
    rng = np.random.default_rng(seed)
    room = max(max(lens), 1) + extra
    w0 = rng.exponential(1.0, (B, H, room)).astype(F32)
    p0 = rng.integers(0, 1000, (B, H, room)).astype(np.int32)
    seen = [n + 17 * b for b, n in enumerate(lens)]
    w, p = torch.from_numpy(w0).cuda(), torch.from_numpy(p0).cuda()
    given = [n - len_add for n in lens]
    ql = q_lens or [L] * B
    if lse is None:
        _, lse = c.attend(q, ints(given), None if q_lens is None else ints(q_lens),
                          len_add=len_add, causal=causal, scale=scale, return_lse=True)
    c.weigh(q, lse, ints(given), w, None if q_lens is None else ints(q_lens),
            new=None if new is None else ints(new), len_add=len_add, causal=causal, scale=scale,
            positions=p if positions else None, seen=ints(seen) if positions else None)
    sums, tols = weigh_plain(Plain(c), q.float().cpu().numpy().astype(np.float64),
                             lse.cpu().numpy().astype(np.float64), lens, ql,
                             D ** -0.5 if scale is None else scale, causal)
    want, tol, pos = w0.astype(np.float64), np.zeros(w0.shape), p0.copy()
    for b in range(B):
        n, m = lens[b], min(lens[b], ql[b] if new is None else new[b])
        want[b, :, n - m:n] = 0
        want[b, :, :n] += sums[b]
        # What a weight grows by comes in passes over 256 query rows (one for few rows). Each
        # is added to the float32 weight, which only grows: off by half a step, 2^-24, of
        # `want` at most. With 5 passes and terms that are small beside the weight, that is
        # 5 2^-24 of it, not the 2^-23 that one or two take.
        passes = max(2, -(-ql[b] * (Hq // H) // 256))
        tol[b, :, :n] = tols[b] + want[b, :, :n] * passes * 2.0 ** -24
        if positions:
            pos[b, :, n - m:n] = seen[b] - m + np.arange(m)
    got = w.cpu().numpy()
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), (np.abs(got - want) - tol).max())
    for b in range(B):  # rows behind the last one
        assert np.array_equal(got[b, :, lens[b]:], w0[b, :, lens[b]:])
    assert np.array_equal(p.cpu().numpy(), pos)
    return w


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("L,rep", [(1, 1), (1, 8), (4, 4), (3, 7), (2, 16), (1, 48)])
def test_weigh_small(cuda, dim, page, L, rep):
    rng = np.random.default_rng(dim + page + 10 * L + rep)
    c = make_cache(rng, 3, 2, dim, page, -(-640 // page))
    q = bf16(rng, (3, 2 * rep, L, dim), 2.0).cuda()
    check_weigh(c, q, [601, L, 255])
    check_weigh(c, q, [64, 0, 300], [L, 0, max(1, L - 1)], causal=False)


@pytest.mark.parametrize("keys", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1023])
def test_weigh_edges(cuda, keys):
    rng = np.random.default_rng(keys)
    c = make_cache(rng, 2, 1, 128, 16, 66)
    q = bf16(rng, (2, 4, 2, 128)).cuda()
    check_weigh(c, q, [keys, max(1, keys - 1)], [min(2, keys), 1])
    check_weigh(c, q, [keys, keys], [0, 1], new=[keys, 0], positions=False, extra=0)


@pytest.mark.parametrize("dim,page,L,rep,keys", [(64, 16, 33, 3, 700), (128, 64, 70, 5, 515),
                                                 (256, 64, 64, 8, 1500), (256, 128, 5, 16, 2100),
                                                 (64, 32, 300, 4, 300), (128, 32, 257, 1, 4000),
                                                 (64, 64, 600, 2, 20000), (256, 32, 96, 8, 900)])
def test_weigh_windows(cuda, dim, page, L, rep, keys):
    """More query rows than one pass over them takes; windows at a prompt's end."""
    rng = np.random.default_rng(dim + L)
    c = make_cache(rng, 2, 2, dim, page, -(-keys // page))
    q = bf16(rng, (2, 2 * rep, L, dim), 1.5).cuda()
    check_weigh(c, q, [keys, keys // 2 + L // 2], [L, L // 2])
    check_weigh(c, q, [keys, keys - 3], [L - 1, L], new=[keys, 5], causal=False)


def test_weigh_sums_to_the_rows(cuda):
    """The weights of a row add up to 1: a step adds the query heads of a kv head."""
    rng = np.random.default_rng(9)
    c = make_cache(rng, 2, 2, 128, 32, 40)
    q = bf16(rng, (2, 12, 3, 128)).cuda()
    lens = ints([1200, 77])
    _, lse = c.attend(q, lens, return_lse=True)
    w = torch.zeros((2, 2, 1280), device="cuda")
    for _ in range(4):
        c.weigh(q, lse, lens, w, new=ints([0, 0]))
    # 18 rows 4 times over; each term is right to about 2^-16 (scores of up to 30)
    assert (w.double().sum(-1) - 72).abs().max() < 72 * 2.0 ** -14


def test_weigh_lse_that_is_not_finite(cuda):
    rng = np.random.default_rng(10)
    c = make_cache(rng, 1, 1, 64, 16, 8)
    q = bf16(rng, (1, 5, 2, 64)).cuda()
    lens = ints([100])
    _, lse = c.attend(q, lens, return_lse=True)
    lse[0, 0, 0], lse[0, 1, 1], lse[0, 2, 0] = math.nan, math.inf, -math.inf
    check_weigh(c, q, [100], lse=lse)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    w = torch.zeros((1, 1, 128), device="cuda")
    c.weigh(q, lse, lens, w, status=status)
    assert int(status) == _lib.VB_STATUS_NONFINITE and torch.isfinite(w).all()
    status.zero_()
    c.weigh(q, torch.full_like(lse, -math.inf), lens, w.zero_(), status=status)
    assert int(status) == 0 and not w.any()


def test_weigh_bounds(cuda):
    """Pages that are not there, and sequences longer than the weights have room."""
    rng = np.random.default_rng(11)
    c = make_cache(rng, 2, 1, 64, 16, 8)
    q = bf16(rng, (2, 2, 1, 64)).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    w = torch.ones((2, 1, 99), device="cuda")
    lse = torch.zeros((2, 2, 1), device="cuda")
    c.weigh(q, lse, ints([100, 50]), w, status=status)
    assert int(status) == _lib.VB_STATUS_BOUNDS
    assert (w[0] == 1).all() and not (w[1, :, :50] == 1).any()
    status.zero_()
    c.page_table[1, 1], c.page_table[1, 2] = -1, 10 ** 6
    w.fill_(1)
    c.weigh(q, lse, ints([20, 50]), w, status=status)
    assert int(status) == _lib.VB_STATUS_BOUNDS
    assert (w[1, :, 16:48] == 1).all() and not (w[1, :, :16] == 1).any()


def test_weigh_strides_streams_and_graphs(cuda):
    rng = np.random.default_rng(12)
    c = make_cache(rng, 2, 2, 128, 64, 10)
    base = bf16(rng, (2, 3, 8 * 128 + 5)).cuda()
    for shift in (0, 3):
        q = base[..., shift:shift + 8 * 128].unflatten(-1, (8, 128)).transpose(1, 2)
        check_weigh(c, q, [640, 333])
    q = bf16(rng, (2, 8, 1, 128)).cuda()
    lens, lse = ints([600, 35]), torch.empty((2, 8, 1), device="cuda")
    lse.copy_(c.attend(q, lens, return_lse=True)[1])
    want = torch.zeros((2, 2, 640), device="cuda")
    c.weigh(q, lse, lens, want)
    side = torch.cuda.Stream()
    got = torch.zeros_like(want)
    side.wait_stream(torch.cuda.current_stream())
    c.weigh(q, lse, lens, got, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.weigh(q, lse, lens, got)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for _ in range(3):
        c.weigh(q, lse, lens, want)
    assert torch.equal(got, want)
    del g


# -------------------------------------------------------------------- evict
def evict_plain(ref, w, p, lens, keep, first, recent):
    """The rule row by row, in place; returns the new lengths and the rows kept."""
    B, H = w.shape[:2]
    page = ref.page
    for b in range(B):
        n = lens[b]
        if n <= keep:
            continue
        for h in range(H):
            at = p[b, h, :n].astype(np.int64) if p is not None else np.arange(n)
            safe = (np.arange(n) < first) | (at > at.max() - recent)
            v = np.where(np.isnan(w[b, h, :n]), -np.inf, w[b, h, :n].astype(np.float64))
            nan = np.isnan(w[b, h, :n])
            order = np.lexsort((np.arange(n), -v, nan, ~safe))
            # protected rows are alike: the lower ones first
            s = np.flatnonzero(safe)
            order = np.concatenate((s, order[len(s):]))
            kept = np.zeros(n, bool)
            kept[order[:keep]] = True
            holes, tail = np.flatnonzero(~kept[:keep]), keep + np.flatnonzero(kept[keep:])
            assert len(holes) == len(tail)
            old = [s.copy() for s in ref.scales]
            for pg in np.unique(holes // page):
                mine = holes // page == pg
                to, src = holes[mine], tail[mine]
                pid = ref.table[b, pg]
                rows = np.arange(pg * page, min((pg + 1) * page, keep))
                stay = np.setdiff1d(rows, to)
                for kv in range(2):
                    codes, scales = ref.codes[kv], ref.scales[kv]
                    sid = ref.table[b, src // page]
                    top = F32(max([old[kv][i, h] for i in sid] + ([old[kv][pid, h]] if len(stay) else [])))
                    if top > 0:
                        r = F32(old[kv][pid, h] / top)
                        if len(stay) and old[kv][pid, h] != top:
                            codes[pid, h, stay % page] = np.rint(codes[pid, h, stay % page].astype(F32) * r)
                    for d, s, i in zip(to, src, sid):
                        r = F32(old[kv][i, h] / top) if top > 0 else F32(1)
                        codes[pid, h, d % page] = np.rint(codes[i, h, s % page].astype(F32) * r)
                    scales[pid, h] = top
            for x in (w, p) if p is not None else (w,):
                x[b, h, holes] = x[b, h, tail]
    return [min(n, keep) for n in lens]


def check_evict(c, rng, lens, keep, first=0, recent=0, weights=None, positions="shuffled", room=None,
                status=None):
    B, H = c.batch, c.kv_heads
    room = c.page_table.shape[1] * c.page if room is None else room
    w = rng.exponential(1.0, (B, H, room)).astype(F32) if weights is None else weights
    p = None
    if positions == "shuffled":
        p = rng.permuted(np.tile(np.arange(room, dtype=np.int32), (B, H, 1)), axis=-1)
    ref = Plain(c)
    tw, tp = torch.from_numpy(w).cuda(), None if p is None else torch.from_numpy(p).cuda()
    after = c.evict(tw, ints(lens), keep, first=first, recent=recent, positions=tp, status=status)
    want = evict_plain(ref, w, p, lens, keep, first, recent)
    assert after.tolist() == want
    assert np.array_equal(tw.cpu().numpy(), w, equal_nan=True)
    assert p is None or np.array_equal(tp.cpu().numpy(), p)
    for t, r in zip((c.k_scales, c.v_scales, c.k_codes, c.v_codes), ref.scales + ref.codes):
        assert np.array_equal(t.cpu().numpy(), r)
    return tw, tp, after


@pytest.mark.parametrize("dim,page", [(64, 16), (64, 128), (128, 32), (256, 64), (256, 16), (128, 128)])
@pytest.mark.parametrize("keep,rows", [(1, 2), (16, 17), (64, 128), (100, 101), (127, 300), (128, 511),
                                       (500, 512), (300, 2000)])
@pytest.mark.parametrize("first,recent", [(0, 0), (0.1, 0.4), (0.5, 0.5)])
def test_evict(cuda, dim, page, keep, rows, first, recent):
    rng = np.random.default_rng(dim + page + keep + rows)
    c = make_cache(rng, 4, 2, dim, page, -(-rows // page))
    check_evict(c, rng, [rows, keep, keep + (rows - keep) // 2, keep + 1], keep, int(first * keep),
                int(recent * keep))


def test_evict_positions_are_rows_without_them(cuda):
    rng = np.random.default_rng(1)
    c = make_cache(rng, 2, 3, 64, 16, 20)
    check_evict(c, rng, [320, 211], 123, first=4, recent=40, positions=None)


@pytest.mark.parametrize("kind", ["equal", "few", "nan", "infinite", "negative", "zeros", "tiny"])
def test_evict_order(cuda, kind):
    """Ties go to the lower row, whatever their number; any bits are ordered."""
    rng = np.random.default_rng(2)
    B, H, N = 3, 2, 1024
    w = {"equal": np.full((B, H, N), 0.25),
         "few": rng.integers(0, 3, (B, H, N)),
         "nan": np.where(rng.random((B, H, N)) < 0.6, np.nan, rng.random((B, H, N))),
         "infinite": rng.choice([np.inf, -np.inf, 1.0, np.nan], (B, H, N)),
         "negative": rng.standard_normal((B, H, N)),
         "zeros": rng.choice([0.0, -0.0], (B, H, N)),
         "tiny": rng.random((B, H, N)) * 1e-44}[kind].astype(F32)
    c = make_cache(rng, B, H, 64, 32, N // 32)
    check_evict(c, rng, [N, N - 1, N // 2 + 3], 500, first=3, recent=17, weights=w)


def test_evict_more_protected_than_kept(cuda):
    """Positions that repeat can protect more rows than stay: the lower ones do."""
    rng = np.random.default_rng(3)
    c = make_cache(rng, 1, 1, 64, 16, 20)
    w = torch.rand((1, 1, 320), device="cuda")
    p = torch.full((1, 1, 320), 7, dtype=torch.int32, device="cuda")
    before = c.k_codes.clone()
    assert c.evict(w, ints([320]), 100, recent=50, positions=p).tolist() == [100]
    assert torch.equal(c.k_codes, before)


def test_evict_many_heads(cuda):
    """More (sequence, head) pairs than a grid has rows in its second dimension."""
    rng = np.random.default_rng(14)
    heads = 16384
    c = PagedKV8Cache.empty(9, heads, 64, 5, 2, 16)
    c.page_table.copy_(torch.arange(10, dtype=torch.int32).view(5, 2).clamp(max=8))
    c.k_codes.random_(-127, 128)
    c.v_codes.random_(-127, 128)
    c.k_scales.fill_(0.5)
    c.v_scales.fill_(0.25)
    w = torch.rand((5, heads, 32), device="cuda")
    lens = [20, 3, 31, 28, 16]
    before, w0 = [t.clone() for t in (c.k_codes, c.v_codes)], w.clone()
    assert c.evict(w, ints(lens), 12).tolist() == [min(n, 12) for n in lens]
    for b, n in enumerate(lens[:4]):
        kept = torch.argsort(-w0[b, :, :n], dim=-1, stable=True)[:, :min(n, 12)].sort(-1).values
        assert torch.equal(w[b, :, :min(n, 12)].sort(-1).values,
                           w0[b, :, :n].gather(-1, kept).sort(-1).values)
        # equal scales: the kept rows themselves, in some order
        for t, old in zip((c.k_codes, c.v_codes), before):
            rows = [x[c.page_table[b].long()].permute(1, 0, 2, 3).reshape(heads, 32, 64).double().sum(-1)
                    for x in (t, old)]
            m = min(n, 12)
            assert torch.equal(rows[0][:, :m].sort(-1).values, rows[1].gather(-1, kept).sort(-1).values)


@pytest.mark.parametrize("rows,keep,units", [(5000, 4000, 1), (20000, 3000, 1), (70000, 5001, 2),
                                             (70000, 60000, 1), (300000, 70000, 1)])
def test_evict_long(cuda, rows, keep, units):
    """Several CTAs for a head; more keys than their shared memory holds."""
    rng = np.random.default_rng(rows)
    c = make_cache(rng, 1, units, 64, 128, -(-rows // 128))
    w = rng.integers(0, 5000, (1, units, c.page_table.shape[1] * 128)).astype(F32)
    check_evict(c, rng, [rows], keep, first=64, recent=keep // 3, weights=w)


def test_evict_long_and_many(cuda):
    """One CTA for each of more heads than there are SMs, over more keys than it holds."""
    rng = np.random.default_rng(19)
    c = make_cache(rng, 10, 16, 64, 128, 72)
    w = rng.exponential(1.0, (10, 16, 72 * 128)).astype(F32)
    lens = [9216, 9001, 8193, 8192, 700, 129, 128, 1, 0, 9215]
    check_evict(c, rng, lens, 128, first=4, recent=30, weights=w)


def test_evict_scales(cuda):
    """Scales of zero, pages whose rows all leave, and equal scales, which leave the
    codes as they are."""
    rng = np.random.default_rng(4)
    c = make_cache(rng, 2, 2, 64, 16, 32)
    for t in (c.k_scales, c.v_scales):
        t[torch.rand_like(t) < 0.3] = 0
    w = rng.random((2, 2, 512)).astype(F32)
    w[:, :, :64] = 0       # four pages are refilled whole
    w[:, :, 400:] += 1
    check_evict(c, rng, [512, 470], 200, weights=w)
    c.k_scales.fill_(0.5)
    c.v_scales.fill_(0.5)
    check_evict(c, rng, [512, 300], 100)


def test_evict_rounding_is_half_a_step(cuda):
    rng = np.random.default_rng(5)
    c = make_cache(rng, 1, 1, 128, 16, 40)
    c.v_scales.mul_(torch.rand_like(c.v_scales) * 10 + 0.1)
    ref = Plain(c)
    tw, tp, after = check_evict(c, rng, [640], 300, positions="shuffled", recent=100)
    now = Plain(c)
    # the kept rows' values before, found by their position
    before, got = ref.rows(1, 0, 640)[0], now.rows(1, 0, 300)[0]
    scale = np.repeat(now.scales[1][now.table[0, :19], 0], 16)[:300]
    rng = np.random.default_rng(5)
    make_cache(rng, 1, 1, 128, 16, 40)
    rng.exponential(1.0, (1, 1, 640))
    p0 = rng.permuted(np.tile(np.arange(640, dtype=np.int32), (1, 1, 1)), axis=-1)[0, 0]
    was = np.argsort(p0)[tp.cpu().numpy()[0, 0, :300]]
    assert (np.abs(got - before[was]) <= scale[:, None] * 0.50001).all()


def test_evict_bounds(cuda):
    """Lengths beyond the table and the weights, and pages that are not there."""
    rng = np.random.default_rng(6)
    c = make_cache(rng, 2, 1, 64, 16, 8)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    w = torch.rand((2, 1, 100), device="cuda")
    assert c.evict(w, ints([128, -3]), 100, status=status).tolist() == [100, 0]
    assert int(status) == _lib.VB_STATUS_BOUNDS
    status.zero_()
    c.page_table[0, 0], c.page_table[1, 5] = -1, 10 ** 6
    w = torch.rand((2, 1, 128), device="cuda")
    assert c.evict(w, ints([128, 128]), 40, status=status).tolist() == [40, 40]
    assert int(status) == _lib.VB_STATUS_BOUNDS


def test_evict_streams_and_graphs(cuda):
    """Replays use their own scratch and the lengths of the time."""
    rng = np.random.default_rng(7)
    c = make_cache(rng, 2, 2, 128, 32, 30)
    w0 = rng.random((2, 2, 960)).astype(F32)
    w, lens = torch.from_numpy(w0).cuda(), ints([0, 0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        after = c.evict(w, lens, 400, recent=9)
    for given in ([960, 300], [401, 777]):
        ref, want = Plain(c), w.cpu().numpy().copy()
        lens.copy_(ints(given))
        torch.empty(1 << 20, device="cuda").fill_(7)
        g.replay()
        torch.cuda.synchronize()
        assert after.tolist() == evict_plain(ref, want, None, given, 400, 0, 9)
        assert np.array_equal(w.cpu().numpy(), want)
        assert np.array_equal(c.k_codes.cpu().numpy(), ref.codes[0])
    del g
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ref, want = Plain(c), w.cpu().numpy().copy()
    got = c.evict(w, lens, 100, stream=side)
    side.synchronize()
    assert got.tolist() == evict_plain(ref, want, None, [401, 777], 100, 0, 0)
    assert np.array_equal(c.v_codes.cpu().numpy(), ref.codes[1])


def test_graphs_on_two_streams_at_once(cuda):
    """Captured windows and evictions have scratch of their own: replayed beside one
    another and beside eager calls."""
    rng = np.random.default_rng(17)
    caches = [make_cache(rng, 2, 2, 64, 16, 60) for _ in range(3)]
    qs = [bf16(rng, (2, 8, 40, 64)).cuda() for _ in range(3)]
    lens = ints([960, 700])
    lses = [c.attend(q, lens, return_lse=True)[1] for c, q in zip(caches, qs)]
    ws = [torch.zeros((2, 2, 960), device="cuda") for _ in range(3)]
    want = []
    for c, q, lse in zip(caches, qs, lses):
        w = torch.zeros((2, 2, 960), device="cuda")
        c.weigh(q, lse, lens, w)
        want.append(w.clone())
    graphs = []
    for c, q, lse, w in zip(caches[:2], qs, lses, ws):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            w.zero_()
            c.weigh(q, lse, lens, w)
            keep = w.clone()
            after = c.evict(w, lens, 300, recent=20)
        graphs.append((g, keep, after))
    refs = [(Plain(c), w.cpu().numpy().copy()) for c, w in zip(caches, want)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for (g, _, _), st in zip(graphs, streams):
        with torch.cuda.stream(st):
            g.replay()
    caches[2].weigh(qs[2], lses[2], lens, ws[2])
    done = caches[2].evict(ws[2], lens, 300, recent=20)
    torch.cuda.synchronize()
    for i, (c, (ref, w)) in enumerate(zip(caches, refs)):
        if i < 2:
            assert torch.equal(graphs[i][1], want[i])
        got = graphs[i][2] if i < 2 else done
        assert got.tolist() == evict_plain(ref, w, None, [960, 700], 300, 0, 20)
        assert np.array_equal(ws[i].cpu().numpy(), w)
        assert np.array_equal(c.k_codes.cpu().numpy(), ref.codes[0])
        assert np.array_equal(c.v_codes.cpu().numpy(), ref.codes[1])
    del g, graphs


def test_shared_pages_below_first_are_left(cuda):
    rng = np.random.default_rng(8)
    c = make_cache(rng, 3, 2, 64, 16, 20)
    c.page_table[1:, :4] = c.page_table[0, :4]
    ids = c.page_table[0, :4].long()
    old = [t[ids].clone() for t in (c.k_codes, c.v_codes, c.k_scales, c.v_scales)]
    c.evict(torch.rand((3, 2, 320), device="cuda"), ints([320, 200, 260]), 128, first=64, recent=20)
    for t, o in zip((c.k_codes, c.v_codes, c.k_scales, c.v_scales), old):
        assert torch.equal(t[ids], o)


def test_offsets_past_32_bits(cuda):
    """Pages at the end of a pool of more than 4 GB, by every kernel."""
    rng = np.random.default_rng(20)
    heads, dim, page, pages = 8, 256, 128, 17000  # 4.5 GB of K
    c = PagedKV8Cache.empty(pages, heads, dim, 2, 6, page)
    c.page_table.copy_(torch.tensor([[16999, 3, 16998, 8300, 16990, 16991],
                                     [16999, 3, 16000, 1, 16997, 16996]], dtype=torch.int32))
    small = make_cache(rng, 2, heads, dim, page, 6)
    small.page_table[1, :2] = small.page_table[0, :2]
    for a, b in ((c.k_codes, small.k_codes), (c.v_codes, small.v_codes),
                 (c.k_scales, small.k_scales), (c.v_scales, small.v_scales)):
        a[c.page_table.long()] = b[small.page_table.long()]
    lens = ints([768, 700])
    for L, rep in ((1, 4), (40, 2)):
        q = bf16(rng, (2, heads * rep, L, dim)).cuda()
        plan = [SharedPrefix(x, [(0, 2, 256)], 0) for x in (c, small)]
        (a, la), (b, lb) = (x.attend_shared(q, lens, p, return_lse=True)
                            for x, p in zip((c, small), plan))
        assert torch.equal(a, b) and torch.equal(la, lb)
        w = [torch.zeros((2, heads, 768), device="cuda") for _ in range(2)]
        c.weigh(q, la, lens, w[0])
        small.weigh(q, lb, lens, w[1])
        assert torch.equal(*w) and w[0].any()
    after = [x.evict(y, lens, 400, first=256) for x, y in zip((c, small), w)]
    assert torch.equal(*after) and torch.equal(*w)
    for a, b in zip(c.read(after[0], 400), small.read(after[0], 400)):
        assert torch.equal(a, b)
    del c


def test_python_refusals(cuda):
    rng = np.random.default_rng(13)
    c = make_cache(rng, 2, 2, 64, 16, 4)
    q, lens = bf16(rng, (2, 4, 1, 64)).cuda(), ints([9, 9])
    lse, w = torch.zeros((2, 4, 1), device="cuda"), torch.zeros((2, 2, 64), device="cuda")
    p = torch.zeros((2, 2, 64), dtype=torch.int32, device="cuda")
    ok = dict(q=q, lse=lse, lens=lens, weights=w)
    for bad in (dict(q=q.float()), dict(q=q[:1]), dict(q=q[:, :3]), dict(lse=lse[:, :3]),
                dict(lse=lse.double()), dict(lens=lens.long()), dict(weights=w[:1]),
                dict(weights=w.transpose(0, 1)), dict(weights=w.cpu()), dict(weights=w.half()),
                dict(positions=p), dict(positions=p[..., :9].contiguous(), seen=lens),
                dict(positions=w, seen=lens), dict(scale=-1.0), dict(new=lens[:1])):
        with pytest.raises((ValueError, RuntimeError)):
            c.weigh(**{**ok, **bad})
    ok = dict(weights=w, lens=lens, keep=8)
    for bad in (dict(keep=0), dict(keep=-1), dict(first=9), dict(first=-1), dict(recent=-1),
                dict(first=4, recent=5), dict(keep=(1 << 32) + 8), dict(first=1 << 32),
                dict(recent=-1 << 32), dict(weights=w[:, :1]), dict(lens=lens[:1]),
                dict(lens=lens.cpu()), dict(positions=p[:1]), dict(positions=p.float())):
        with pytest.raises((ValueError, RuntimeError)):
            c.evict(**{**ok, **bad})
