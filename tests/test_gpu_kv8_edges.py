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


@both
def test_unequal_pages(cuda, L, rep, keys, dim, page):
    """K and V scales of neighbouring pages up to 2^10 apart, a page of vanishing
    values, V scales that grow along the sequence (the sums so far are rescaled)."""
    c, q = setup(L, rep, keys, dim, page)
    rng = np.random.default_rng(keys)
    n = c.page_table.shape[1]
    ids = c.page_table[0].long()
    c.v_scales[ids] = torch.from_numpy((0.02 * 2.0 ** rng.uniform(-10, 0, (n, 1)))
                                       .astype(np.float32)).cuda()
    c.k_scales[ids] = torch.from_numpy((0.02 * 2.0 ** rng.uniform(-10, 0, (n, 1)))
                                       .astype(np.float32)).cuda()
    c.v_scales[pages(c, 0.6)] = 2.0 ** -30
    check_attend(c, q.cuda(), [keys], None)
    c.v_scales[ids] = torch.from_numpy((2.0 ** np.linspace(-14, -3, n))
                                       .astype(np.float32)[:, None]).cuda()
    check_attend(c, q.cuda(), [keys], None)


@both
def test_garbage_past_the_end_is_not_read(cuda, L, rep, keys, dim, page):
    c, q = setup(L, rep, keys, dim, page, heads=2)
    q = q.cuda()
    before = c.attend(q, ints([keys]), return_lse=True)
    ids = c.page_table[0].long()
    last = (keys - 1) // page
    c.k_codes[ids[last], :, (keys - 1) % page + 1:] = 127
    c.v_codes[ids[last], :, (keys - 1) % page + 1:] = -127
    c.k_scales[ids[last + 1:]] = math.nan
    c.v_scales[ids[last + 1:]] = math.inf
    c.page_table[0, last + 1:] = -1
    for a, b in zip(before, c.attend(q, ints([keys]), return_lse=True)):
        assert torch.equal(a, b)


@both
def test_missing_pages_are_masked(cuda, L, rep, keys, dim, page):
    """Entries without a page, and pages outside the pool, in the middle of the
    table: their keys have no weight, and the call says so."""
    c, q = setup(L, rep, keys, dim, page)
    n = -(-keys // page)
    gone = sorted({1 % n, n // 2})
    ref = Plain(c)
    for i, e in zip(gone, (-1, 10 ** 6)):
        c.page_table[0, i] = e
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = c.attend(q.cuda(), ints([keys]), causal=False, return_lse=True, status=status)
    assert int(status) == _lib.VB_STATUS_BOUNDS
    left = [p for p in range(keys) if p // page not in gone]
    rows = ref.rows
    ref.rows = lambda kv, b, m: rows(kv, b, keys)[:, left]
    want, wl, tol, ltol = attend_plain(ref, q.float().numpy().astype(np.float64), [len(left)],
                                       [L], dim ** -0.5, False)
    assert (np.abs(out.float().cpu().numpy() - want) <= tol).all()
    assert (np.abs(lse.cpu().numpy() - wl) <= ltol).all()


@both
def test_nonfinite_queries_stay_in_their_row(cuda, L, rep, keys, dim, page):
    c, q = setup(L, rep, keys, dim, page)
    q = q.cuda()
    clean, cl = c.attend(q, ints([keys]), return_lse=True)
    bad = torch.zeros((rep, L), dtype=torch.bool)
    for h, i, x in ((0, 0, math.nan), (1, L - 1, math.inf), (rep - 1, L // 2, -math.inf)):
        q[0, h, i, dim // 3] = x
        bad[h, i] = True
    out, lse = c.attend(q, ints([keys]), return_lse=True)
    bad = bad.cuda()
    assert out[0][bad].isnan().all() and lse[0][bad].isnan().all()
    assert torch.equal(out[0][~bad], clean[0][~bad]) and torch.equal(lse[0][~bad], cl[0][~bad])


@both
def test_large_and_small_queries(cuda, L, rep, keys, dim, page):
    """A power of two per row keeps queries of any size exact."""
    c, q = setup(L, rep, keys, dim, page)
    flat = q.view(-1, dim)
    flat[0] *= 2.0 ** 60
    flat[1] *= 2.0 ** -60
    flat[-1] = 0
    c.k_scales.mul_(2.0 ** -30)
    check_attend(c, q.cuda(), [keys], None)


@both
@pytest.mark.parametrize("odd", [0, 3])
def test_strided_queries(cuda, L, rep, keys, dim, page, odd):
    """Queries in a projection's layout, at an even and at an odd offset; rows that
    see no key among them."""
    rng = np.random.default_rng(keys + odd)
    c = make_cache(rng, 2, 2, dim, page, -(-keys // page))
    Hq = 2 * rep
    base = bf16(rng, (2, L, Hq * dim + 2 * odd), 2.0).cuda()
    q = base[..., odd:Hq * dim + odd].unflatten(-1, (Hq, dim)).transpose(1, 2)
    lens = [keys, max(1, L // 2)]
    a = check_attend(c, q, lens, None)
    assert torch.equal(a, c.attend(q.contiguous(), ints(lens)))
    check_attend(c, q, lens, [max(1, L - 1), max(1, L // 3)], causal=False)
    # a broadcast head
    wide = q[:, :1].expand(2, Hq, L, dim)
    assert torch.equal(c.attend(wide, ints(lens)), c.attend(wide.contiguous(), ints(lens)))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_many_rows_over_every_page_size(cuda, dim, page):
    rng = np.random.default_rng(dim + page)
    c = make_cache(rng, 2, 2, dim, page, -(-700 // page))
    q = bf16(rng, (2, 6, 50, dim), 2.0).cuda()
    for keys in (127, 128, 129, 257, 700):
        check_attend(c, q, [keys, 700 - keys], [50, min(50, 700 - keys)])


@pytest.mark.parametrize("L,rep", ROWS)
@pytest.mark.parametrize("ratio", [-10, -20, -26, -30])
@pytest.mark.parametrize("keys", [100, 1000])
def test_weight_on_a_page_of_small_values(cuda, L, rep, ratio, keys):
    """Nearly all of a row's weight on a page whose values lie far below another
    page's. A weight times its V scale over the largest one seen is an f16 number of
    at least 2^6 times (the weight over the row's largest); what it loses below f16's
    normal numbers is 2^-25 at most, of l >= 2^6: n 2^-31 of the largest value."""
    dim, page = 128, 16
    c, q = setup(L, rep, keys, dim, page, heads=1)
    ids = c.page_table[0].long()
    c.k_codes[ids[2:]] = 0
    c.k_codes[ids[0]] = 0
    c.k_codes[ids[1]] = 100
    c.k_scales[ids] = 0.05
    q = q.abs() + 0.5
    c.v_scales[ids] = 1.0
    c.v_scales[ids[1]] = 2.0 ** ratio
    out = c.attend(q.cuda(), ints([keys]), causal=False).float().cpu().numpy()
    want, _, tol, _ = attend_plain(Plain(c), q.float().numpy().astype(np.float64), [keys], [L],
                                   dim ** -0.5, False)
    # (every other key's weight is e^-28 or less, and its share of the row is in `tol`)
    assert (np.abs(out - want) <= tol + 2.0 ** -31 * keys * 127).all()


@both
@pytest.mark.parametrize("power", [18, 22, 24, 26, 27, 28, 30, 33, 40, 60])
def test_scores_of_any_size(cuda, L, rep, keys, dim, page, power):
    """Scores of 2^power, where float32 is coarser than the exponentials' range: one
    key stands out for each row (its codes are the signs of the row's query, the
    others' products are half as large at most), so its value is the result."""
    c, q = setup(L, rep, keys, dim, page, seed=power)
    rng = np.random.default_rng(power)
    sign = torch.from_numpy(rng.choice([-1, 1], (rep * L, dim)).astype(np.float32))
    # the row's own key, spread over the sequence
    at = torch.arange(rep * L) * (keys // (rep * L)) + (keys - 1) % max(1, keys // (rep * L))
    c.k_scales.fill_(2.0 ** -10)
    c.k_codes.clamp_(-30, 30)
    ids = c.page_table[0].long()[torch.div(at, page, rounding_mode="floor").cuda()]
    c.k_codes[ids, 0, (at % page).cuda()] = (sign * 120).to(torch.int8).cuda()
    # sum over dims of 120 |q| 2^-10 scale = 2^power ln 2
    amp = 2.0 ** power * math.log(2) / (dim * 120 * 2.0 ** -10 * dim ** -0.5)
    mag = torch.from_numpy(rng.uniform(0.9, 1.1, (rep * L, dim)).astype(np.float32)) * amp
    q = (sign * mag).to(torch.bfloat16).view(1, rep, L, dim)
    out, lse = c.attend(q.cuda(), ints([keys]), causal=False, return_lse=True)
    ref = Plain(c)
    V, K = ref.rows(1, 0, keys)[0], ref.rows(0, 0, keys)[0]
    z = (q.double().view(-1, dim).numpy() @ K.T) * dim ** -0.5
    best = z.argmax(1)
    assert np.array_equal(best, at.numpy())
    two = np.sort(z, 1)
    assert keys == 1 or (two[:, -1] - two[:, -2] >= 2.0 ** (power - 3)).all()
    # the value, rounded to f16 weights' 2^-11 of it, and to bf16
    want = V[best].reshape(rep, L, dim)
    got = out[0].double().cpu().numpy()
    assert (np.abs(got - want) <= np.abs(want) * (2.0 ** -8 + 2.0 ** -11)).all()
    zt = z.max(1).reshape(rep, L)
    # float32 sums of dim products and three float32 steps
    assert (np.abs(lse[0].cpu().numpy() - zt) <= zt * (dim * 2.0 ** -24 + 2.0 ** -21)).all()


@both
def test_scales_below_float32s_normal_numbers(cuda, L, rep, keys, dim, page):
    """They read as 0 or as what they are: nothing but numbers as small comes out."""
    c, q = setup(L, rep, keys, dim, page)
    for tiny in (2.0 ** -149, 2.0 ** -130, 2.0 ** -126):
        c.v_scales.fill_(tiny)
        c.k_scales.fill_(tiny)
        out, lse = c.attend(q.cuda(), ints([keys]), causal=False, return_lse=True)
        assert (out.abs().float() <= 128 * tiny).all()
        assert (lse - math.log(keys)).abs().max() <= 2.0 ** -17
