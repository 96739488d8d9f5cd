"""Paged 8-bit KV cache on the GPU against plain 64-bit (and, for the codes,
exact 32-bit) forms on the CPU."""
import math

import numpy as np
import pytest
import torch

from vates_b200 import _lib
from vates_b200.kv8 import PagedKV8Cache

pytestmark = pytest.mark.gpu
F32 = np.float32


def make_cache(rng, batch, heads, dim, page, max_pages, extra=3, filled=True):
    """Random codes and scales, the table's pages in shuffled order."""
    pages = batch * max_pages + extra
    c = PagedKV8Cache.empty(pages, heads, dim, batch, max_pages, page)
    c.page_table.copy_(torch.from_numpy(
        rng.permutation(pages)[:batch * max_pages].reshape(batch, max_pages).astype(np.int32)))
    if filled:
        for t in (c.k_codes, c.v_codes):
            t.copy_(torch.from_numpy(rng.integers(-127, 128, t.shape).astype(np.int8)))
        for t in (c.k_scales, c.v_scales):
            t.copy_(torch.from_numpy(rng.uniform(0.01, 0.04, t.shape).astype(F32)))
    return c


def ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def bf16(rng, shape, scale=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * scale).astype(F32)).to(torch.bfloat16)


class Plain:
    """The cache's rule in numpy float32, page by page."""

    def __init__(self, c):
        self.page = c.page
        self.table = c.page_table.cpu().numpy()
        self.codes = [t.cpu().numpy().copy() for t in (c.k_codes, c.v_codes)]
        self.scales = [t.cpu().numpy().copy() for t in (c.k_scales, c.v_scales)]

    def append(self, kv, x, pos, counts):
        codes, scales = self.codes[kv], self.scales[kv]
        for b in range(x.shape[0]):
            n, p0 = counts[b], pos[b]
            i = 0
            while i < n:
                pg, at = divmod(p0 + i, self.page)
                m = min(self.page - at, n - i)
                pid = self.table[b, pg]
                for h in range(x.shape[1]):
                    v = x[b, h, i:i + m]
                    fin = np.isfinite(v)
                    amax = F32(np.abs(np.where(fin, v, 0)).max())
                    s0 = scales[pid, h] if at else F32(0)
                    s = max(s0, max(F32(amax / F32(127)), F32(2.0 ** -40)) if amax > 0 else F32(0))
                    inv = F32(1) / s if s > 0 else F32(0)
                    if at and s > s0:
                        codes[pid, h, :at] = np.rint(codes[pid, h, :at].astype(F32) * F32(s0 / s))
                    with np.errstate(invalid="ignore"):
                        q = np.where(np.isnan(v), 0, np.rint(np.clip(v * inv, -127, 127)))
                    codes[pid, h, at:at + m] = (q if s > 0 else np.zeros_like(v)).astype(np.int8)
                    scales[pid, h] = s
                i += m

    def rows(self, kv, b, n):
        """float64 [heads, n, dim] of positions [0, n) of sequence b."""
        if n == 0:
            return np.zeros((self.codes[kv].shape[1], 0, self.codes[kv].shape[3]))
        ids = self.table[b, :-(-n // self.page)]
        x = self.codes[kv][ids].astype(np.float64) * self.scales[kv][ids][..., None, None]
        return x.transpose(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :n]


def same_cache(c, ref):
    for t, r in zip((c.k_codes, c.v_codes, c.k_scales, c.v_scales), ref.codes + ref.scales):
        assert np.array_equal(t.cpu().numpy(), r)


# ------------------------------------------------------------------- writing
@pytest.mark.parametrize("dim,page", [(64, 16), (64, 128), (128, 32), (256, 64), (256, 128),
                                      (128, 16)])
@pytest.mark.parametrize("n", [1, 3, 16, 77, 300])
def test_append_codes_and_scales(cuda, dim, page, n):
    rng = np.random.default_rng(n * 1000 + dim + page)
    B, H = 4, 3
    c = make_cache(rng, B, H, dim, page, (400 + page) // page + 2)
    ref = Plain(c)
    pos = [0, 1, page, 2 * page - 1]
    counts = [n, 0, max(1, n // 2), n]
    # amplitudes on both sides of the old scales' reach, so some pages grow
    for step, amp in enumerate((0.5, 3.0, 1.0)):
        k, v = bf16(rng, (B, H, n, dim), amp), bf16(rng, (B, H, n, dim), 2 * amp)
        c.append(k.cuda(), v.cuda(), ints(pos), counts=ints(counts))
        ref.append(0, k.float().numpy(), pos, counts)
        ref.append(1, v.float().numpy(), pos, counts)
        same_cache(c, ref)
        pos = [p + m for p, m in zip(pos, counts)]
        if max(pos) + n > c.page_table.shape[1] * page:
            break


def test_append_strides_alignment_and_offset(cuda):
    """Rows in a projection's layout (heads side by side), an odd element
    offset, unequal strides of K and V, and pos_add."""
    rng = np.random.default_rng(5)
    B, H, n, D, page = 2, 2, 19, 128, 16
    base = bf16(rng, (B, n, 3 * H * D + 5)).cuda()
    k = base[..., :H * D].unflatten(-1, (H, D)).transpose(1, 2)
    v = base[..., H * D + 3:2 * H * D + 3].unflatten(-1, (H, D)).transpose(1, 2)
    c = make_cache(rng, B, H, D, page, 8)
    ref = Plain(c)
    c.append(k, v, ints([4, 30]), pos_add=3)
    ref.append(0, k.float().cpu().numpy(), [7, 33], [n, n])
    ref.append(1, v.float().cpu().numpy(), [7, 33], [n, n])
    same_cache(c, ref)
    # dims that are not contiguous are copied
    rng = np.random.default_rng(5)
    bf16(rng, (B, n, 3 * H * D + 5))
    c2 = make_cache(rng, B, H, D, page, 8)
    c2.append(k.transpose(2, 3).contiguous().transpose(2, 3), v, ints([4, 30]), pos_add=3)
    same_cache(c2, ref)


def test_append_special_values(cuda):
    """Zero rows (scale 0), the smallest scale, the largest bf16, infinities
    and NaN (flagged; the page's other values keep their precision)."""
    rng = np.random.default_rng(6)
    D, page = 64, 16
    c = make_cache(rng, 5, 1, D, page, 2)
    x = bf16(rng, (5, 1, 4, D))
    x[0] = 0
    x[1] *= 2.0 ** -60
    x[2] *= 2.0 ** 120
    x[3, 0, 1, 3], x[3, 0, 2, 7] = math.inf, -math.inf
    x[4, 0, 0, 0], x[4, 0, 3, 9] = math.nan, math.inf
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ref = Plain(c)
    c.append(x[:3].cuda().repeat(2, 1, 1, 1)[:5], x.cuda(), ints([0] * 5), status=status)
    y = x[:3].repeat(2, 1, 1, 1)[:5]
    ref.append(0, y.float().numpy(), [0] * 5, [4] * 5)
    ref.append(1, x.float().numpy(), [0] * 5, [4] * 5)
    same_cache(c, ref)
    assert int(status) == _lib.VB_STATUS_NONFINITE
    k, v = c.read(ints([4] * 5), 4)
    assert torch.equal(k[0], torch.zeros_like(k[0])) and torch.isfinite(v).all()
    fin = torch.isfinite(x[3].float())
    step = float(x[3].float()[fin].abs().max()) / 127
    # half a step, and half a bf16 ulp of the value read back
    err = (v[3].cpu().float() - x[3].float())[fin].abs()
    assert (err <= step * 0.5001 + x[3].float()[fin].abs() * 2.0 ** -8).all()


def test_append_out_of_table_is_dropped(cuda):
    rng = np.random.default_rng(7)
    c = make_cache(rng, 3, 2, 64, 16, 2)
    c.page_table[1, 1] = 10 ** 6
    before = [t.clone() for t in (c.k_codes, c.v_codes, c.k_scales, c.v_scales)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = bf16(rng, (3, 2, 4, 64)).cuda()
    # past the table's end, a page that is not in the pool, a negative position
    c.append(x, x, ints([32, 16, -8]), status=status)
    assert int(status) == _lib.VB_STATUS_BOUNDS
    for t, old in zip((c.k_codes, c.v_codes, c.k_scales, c.v_scales), before):
        assert torch.equal(t, old)


# ------------------------------------------------------------------- reading
@pytest.mark.parametrize("dim,page,n", [(64, 16, 1), (128, 32, 45), (256, 64, 130),
                                        (256, 128, 700), (64, 128, 1000)])
def test_read_back(cuda, dim, page, n):
    rng = np.random.default_rng(dim + n)
    B, H = 3, 2
    c = make_cache(rng, B, H, dim, page, -(-(n + 40) // page))
    ref = Plain(c)
    lens, start = [n + 20, 0, n // 2 + 1], [17, 3, 0]
    for st in (None, start):
        k, v = c.read(ints(lens), n, start=None if st is None else ints(st))
        for kv, got in enumerate((k, v)):
            want = np.zeros((B, H, n, dim), F32)
            for b in range(B):
                lo = st[b] if st else 0
                # float32 product of the code and the scale, then bf16
                ids = ref.table[b]
                x = (ref.codes[kv][ids].astype(F32) * ref.scales[kv][ids][..., None, None])
                x = x.transpose(1, 0, 2, 3).reshape(H, -1, dim)[:, lo:min(lens[b], lo + n)]
                want[b, :, :x.shape[1]] = x
            assert torch.equal(got.cpu(), torch.from_numpy(want).to(torch.bfloat16))


# ----------------------------------------------------------------- attention
def attend_plain(ref, q, lens, q_lens, scale, causal):
    """float64 softmax attention, with the bounds on the kernel's error.

    Bounds: out is rounded to bf16 (2^-9 of it) after weights of 11 bits (2^-12
    each, of sum p |v|) whose scores carry at most dz; the scores are float32
    sums of D products of a q rounded nowhere and exact codes: dz = D 2^-24
    scale max_j sum |q k| (plus 2^-22 of the float32 steps after the sum)."""
    B, Hq, L, D = q.shape
    H = ref.codes[0].shape[1]
    out, lse = np.zeros((B, Hq, L, D)), np.full((B, Hq, L), -np.inf)
    tol, ltol = np.zeros_like(out), np.zeros_like(lse)
    for b in range(B):
        n, ql = lens[b], q_lens[b]
        K, V = ref.rows(0, b, n), ref.rows(1, b, n)
        for h in range(Hq):
            k, v = K[h // (Hq // H)], V[h // (Hq // H)]
            for i in range(ql):
                m = max(0, n - ql + i + 1) if causal else n
                if m == 0:
                    continue
                z = k[:m] @ q[b, h, i] * scale
                mag = (np.abs(k[:m]) @ np.abs(q[b, h, i])).max() * scale
                e = np.exp(z - z.max())
                p = e / e.sum()
                out[b, h, i] = p @ v[:m]
                lse[b, h, i] = np.log(e.sum()) + z.max()
                dz = mag * (D * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -20
                av = p @ np.abs(v[:m])
                tol[b, h, i] = np.abs(out[b, h, i]) * 2.0 ** -8 + av * (2.0 ** -11 + 2 * dz)
                ltol[b, h, i] = dz + 2.0 ** -20 * max(1, abs(lse[b, h, i]))
    return out, lse, tol, ltol


def check_attend(c, q, lens, q_lens, causal=True, scale=None, len_add=0, ref=None, **kw):
    B, Hq, L, D = q.shape
    out, lse = c.attend(q, ints([n - len_add for n in lens]),
                        None if q_lens is None else ints(q_lens), len_add=len_add, scale=scale,
                        causal=causal, return_lse=True, **kw)
    want, wl, tol, ltol = attend_plain(ref or Plain(c), q.float().cpu().numpy().astype(np.float64),
                                       lens, q_lens or [L] * B,
                                       D ** -0.5 if scale is None else scale, causal)
    got, gl = out.float().cpu().numpy(), lse.cpu().numpy()
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) - tol).max()
    empty = np.isinf(wl)
    assert np.array_equal(np.isneginf(gl), empty)
    assert (np.abs(gl - np.where(empty, 0, wl))[~empty] <= ltol[~empty]).all()
    return out


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("L,rep", [(1, 1), (1, 8), (4, 4), (3, 7), (2, 16), (1, 48)])
def test_attend_small(cuda, dim, page, L, rep):
    rng = np.random.default_rng(dim + page + 10 * L + rep)
    B, H = 3, 2
    c = make_cache(rng, B, H, dim, page, -(-640 // page))
    q = bf16(rng, (B, H * rep, L, dim), 2.0).cuda()
    check_attend(c, q, [601, L, 255], None)
    check_attend(c, q, [64, 0, 300], [L, 0, max(1, L - 1)], causal=False)


@pytest.mark.parametrize("keys", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_attend_tile_edges(cuda, keys):
    rng = np.random.default_rng(keys)
    for dim in (64, 256):
        c = make_cache(rng, 1, 1, dim, 32, -(-keys // 32))
        check_attend(c, bf16(rng, (1, 3, 1, dim), 2.0).cuda(), [keys], None)


@pytest.mark.parametrize("dim,rep,L,lens,q_lens,causal", [
    (64, 5, 40, [97, 40, 33], [40, 17, 0], True),       # an idle slot
    (128, 4, 70, [30, 200, 70], [70, 65, 3], True),     # rows before the first key see nothing
    (256, 8, 33, [500, 33, 1], [33, 33, 1], True),
    (128, 1, 129, [129, 300, 128], [129, 1, 128], True),
    (256, 2, 150, [0, 150, 700], [150, 150, 150], False),
    (64, 3, 260, [260, 513, 511], [260, 259, 100], True),
    (256, 12, 24, [24, 100, 129], [24, 24, 24], False),
])
def test_attend_many_rows(cuda, dim, rep, L, lens, q_lens, causal):
    rng = np.random.default_rng(dim + rep + L)
    H, page = 2, 16 if dim == 64 else 64
    c = make_cache(rng, 3, H, dim, page, -(-max(lens) // page) + 1)
    q = bf16(rng, (3, H * rep, L, dim), 2.0).cuda()
    check_attend(c, q, lens, q_lens, causal)


@pytest.mark.parametrize("dim,rep,L,batch,heads", [(256, 2, 64, 2, 8), (256, 8, 8, 16, 8),
                                                   (128, 8, 64, 2, 8), (64, 4, 70, 4, 8)])
def test_attend_every_key_tile_counts(cuda, dim, rep, L, batch, heads):
    """Equal keys and equal values: every weight is the same, so the result is
    the value itself, and a key tile that is missed (also for a moment, at the
    end of a short range of tiles) shows at once."""
    rng = np.random.default_rng(dim + L)
    page = 16
    for keys in (200, 300, 1100, 2182):
        c = make_cache(rng, batch, heads, dim, page, -(-keys // page))
        c.k_codes.zero_()
        c.v_codes.fill_(100)
        c.v_scales.fill_(0.02)
        q = bf16(rng, (batch, heads * rep, L, dim)).cuda()
        for _ in range(3):
            out, lse = c.attend(q, ints([keys] * batch), causal=False, return_lse=True)
            # one f16 rounding of equal weights (2^-11) and one to bf16 (2^-8)
            assert (out.float() - 2.0).abs().max() <= 2.0 * (2.0 ** -8 + 2.0 ** -11)
            assert (lse - math.log(keys)).abs().max() <= 2.0 ** -18 * math.log(keys)


def test_attend_long_sequence(cuda):
    """Splits over a long axis, one sequence beside short ones."""
    rng = np.random.default_rng(11)
    c = make_cache(rng, 2, 1, 128, 64, 320)
    ref = Plain(c)
    for L in (1, 4):
        check_attend(c, bf16(rng, (2, 2, L, 128), 3.0).cuda(), [20001, 5], None, ref=ref)


@pytest.mark.parametrize("batch,heads,rep,L,dim,keys", [
    (1, 1, 8, 1, 256, 400), (1, 2, 8, 1, 256, 4000),     # few results to join, and many
    (1, 1, 8, 4, 64, 600), (2, 8, 4, 4, 64, 1500),       # 32 rows; 16 units of 16
    (5, 4, 2, 4, 64, 1500), (17, 1, 3, 1, 128, 700),     # more units than 16
    (1, 1, 2, 40, 256, 3000), (1, 1, 4, 150, 128, 4000),  # prompts: ranges of few rows, of many
    (1, 2, 1, 300, 64, 2500)])
def test_attend_joined_ranges(cuda, batch, heads, rep, L, dim, keys):
    """Ranges of keys joined in every way, whose maxima differ by far more than the
    running maximum is let lag (queries along the key of one position), then again
    on the same workspace for shorter sequences. All values are 2, so that the result
    is 2 whatever the weights are (each rounded to f16 once, 2^-11, the result to
    bf16, 2^-8) and the log-sum-exp tells of them."""
    rng = np.random.default_rng(keys + dim + batch)
    c = make_cache(rng, batch, heads, dim, 64, -(-keys // 64))
    c.v_codes.fill_(100)
    c.v_scales.fill_(0.02)
    ref = Plain(c)
    q = bf16(rng, (batch, heads * rep, L, dim), 2.0)
    far = ref.rows(0, 0, keys)[:, keys * 2 // 3]
    q[0, ::rep] += torch.from_numpy(far).to(torch.bfloat16)[:, None]
    q = q.cuda()
    for lens in ([keys - 37 * b for b in range(batch)],
                 [max(L, keys // 5 - b) for b in range(batch)]):
        out, lse = c.attend(q, ints(lens), return_lse=True)
        _, want, _, ltol = attend_plain(ref, q.float().cpu().numpy().astype(np.float64), lens,
                                        [L] * batch, dim ** -0.5, True)
        assert (out.float() - 2.0).abs().max() <= 2.0 * (2.0 ** -8 + 2.0 ** -11)
        assert (np.abs(lse.cpu().numpy() - want) <= ltol).all()


def test_attend_strides_len_add_and_out(cuda):
    """Queries in a projection's layout at an odd offset, lengths given without
    this step's rows, a caller's output."""
    rng = np.random.default_rng(12)
    B, Hq, L, D = 2, 6, 3, 128
    c = make_cache(rng, B, 2, D, 32, 10)
    base = bf16(rng, (B, L, Hq * D + 7), 2.0).cuda()
    q = base[..., 3:Hq * D + 3].unflatten(-1, (Hq, D)).transpose(1, 2)
    out = torch.empty((B, Hq, L, D), dtype=torch.bfloat16, device="cuda")
    got = check_attend(c, q, [203, 40], None, len_add=L, scale=0.3, out=out)
    assert got is out
    assert torch.equal(out, check_attend(c, q.contiguous(), [203, 40], None, scale=0.3))


def test_attend_unequal_pages(cuda):
    """Pages whose scales differ by up to 2^30 and all-zero pages (scale 0)."""
    rng = np.random.default_rng(13)
    c = make_cache(rng, 1, 1, 128, 16, 24)
    ids = c.page_table[0].long()
    c.v_scales[ids[3]] = 0
    c.v_codes[ids[3]] = 0
    c.k_scales[ids[5]] = 0
    c.k_codes[ids[5]] = 0
    c.v_scales[ids[7]] = 2.0 ** -30
    q = bf16(rng, (1, 4, 2, 128), 1.0).cuda()
    check_attend(c, q, [24 * 16], None)
    c.v_scales.zero_()
    c.v_codes.zero_()
    assert not c.attend(q, ints([24 * 16])).any()


def test_attend_garbage_past_the_end_is_not_read(cuda):
    """Codes and scales past a sequence's last key, and pages the table names
    beyond it, change nothing (NaN and infinite scales in unused pages)."""
    rng = np.random.default_rng(14)
    c = make_cache(rng, 2, 2, 64, 32, 12)
    q = bf16(rng, (2, 4, 2, 64)).cuda()
    a, la = c.attend(q, ints([70, 200]), return_lse=True)
    for b, n in enumerate((70, 200)):
        ids = c.page_table[b].long()
        last = n // 32
        c.k_codes[ids[last], :, n % 32:] = 127
        c.v_codes[ids[last], :, n % 32:] = -127
        c.k_scales[ids[last + 1:]] = math.nan
        c.v_scales[ids[last + 1:]] = math.inf
        c.page_table[b, last + 2:] = -1
    b2, lb = c.attend(q, ints([70, 200]), return_lse=True)
    assert torch.equal(a, b2) and torch.equal(la, lb)


def test_attend_missing_page_is_masked(cuda):
    rng = np.random.default_rng(15)
    c = make_cache(rng, 1, 1, 128, 16, 8)
    q = bf16(rng, (1, 2, 1, 128)).cuda()
    c.page_table[0, 7] = -1
    want = c.attend(q, ints([112]), causal=False)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = c.attend(q, ints([128]), causal=False, status=status)
    assert int(status) == _lib.VB_STATUS_BOUNDS
    assert (got.float() - want.float()).abs().max() <= 2.0 ** -8 * want.float().abs().max()


def test_attend_nan_query_stays_in_its_row(cuda):
    rng = np.random.default_rng(16)
    c = make_cache(rng, 1, 1, 64, 16, 70)
    for keys in (30, 1100):
        q = bf16(rng, (1, 3, 2, 64)).cuda()
        clean, cl = c.attend(q, ints([keys]), return_lse=True)
        q[0, 1, 0, 5] = math.nan
        q[0, 2, 1, 5] = math.inf
        out, lse = c.attend(q, ints([keys]), return_lse=True)
        for h, i in ((1, 0), (2, 1)):
            assert out[0, h, i].isnan().all() and lse[0, h, i].isnan()
        for h, i in ((0, 0), (0, 1), (1, 1), (2, 0)):
            assert torch.equal(out[0, h, i], clean[0, h, i]) and lse[0, h, i] == cl[0, h, i]


def test_large_and_small_queries(cuda):
    """A power of two per row keeps queries of any size exact."""
    rng = np.random.default_rng(17)
    c = make_cache(rng, 1, 1, 128, 32, 6)
    q = bf16(rng, (1, 4, 1, 128))
    q[0, 1] *= 2.0 ** 60
    q[0, 2] *= 2.0 ** -60
    q[0, 3] = 0
    c.k_scales.mul_(2.0 ** -30)
    check_attend(c, q.cuda(), [180], None)


def test_write_then_attend_is_deterministic_on_another_stream(cuda):
    """Append and attend on a side stream, twice: the same bits, and the same
    as on the default stream."""
    rng = np.random.default_rng(18)
    B, H, D = 2, 2, 256
    k, v = bf16(rng, (B, H, 90, D)).cuda(), bf16(rng, (B, H, 90, D)).cuda()
    q = bf16(rng, (B, 16, 2, D)).cuda()
    pos, lens = ints([0, 0]), ints([90, 90])
    outs = []
    side = torch.cuda.Stream()
    for stream in (None, side, side):
        c = PagedKV8Cache.empty(4, H, D, B, 2, 64)
        c.page_table.copy_(torch.tensor([[2, 0], [1, 3]], dtype=torch.int32))
        if stream:
            stream.wait_stream(torch.cuda.current_stream())
        c.append(k, v, pos, stream=stream)
        outs.append(c.attend(q, lens, stream=stream))
        torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[1], outs[2])


def test_page_offsets_past_32_bits(cuda):
    """Pages whose byte offset passes 2^32 hold what was written to them."""
    rng = np.random.default_rng(19)
    H, D, page = 2, 256, 128
    pages = (1 << 32) // (H * D * page) + 8
    c = PagedKV8Cache.empty(pages, H, D, 1, 4, page)
    c.page_table.copy_(torch.tensor([[pages - 1, 1, pages - 3, 0]], dtype=torch.int32))
    k, v = bf16(rng, (1, H, 400, D)), bf16(rng, (1, H, 400, D))
    c.append(k.cuda(), v.cuda(), ints([0]))
    small = PagedKV8Cache.empty(4, H, D, 1, 4, page)
    small.page_table.copy_(torch.tensor([[3, 1, 2, 0]], dtype=torch.int32))
    small.append(k.cuda(), v.cuda(), ints([0]))
    for a, b in zip(c.read(ints([400]), 400), small.read(ints([400]), 400)):
        assert torch.equal(a, b)
    q = bf16(rng, (1, 8, 40, D)).cuda()
    for rows in (q[:, :, :1], q):
        assert torch.equal(c.attend(rows, ints([400])), small.attend(rows, ints([400])))


def test_graph_capture(cuda):
    """Append and attend in a CUDA graph; positions advance on the device."""
    rng = np.random.default_rng(20)
    H, D = 1, 128
    c = PagedKV8Cache.empty(8, H, D, 1, 8, 16)
    c.page_table.copy_(torch.arange(8, dtype=torch.int32)[None])
    k, v, q = (bf16(rng, (1, h, 1, D)).cuda() for h in (H, H, 4))
    pos = ints([0])
    c.append(k, v, pos)
    c.attend(q, pos, len_add=1)  # workspaces exist before the capture
    graph = torch.cuda.CUDAGraph()
    out = torch.empty((1, 4, 1, D), dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.append(k, v, pos)
        c.attend(q, pos, len_add=1, out=out)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph, stream=side):
        c.append(k, v, pos)
        c.attend(q, pos, len_add=1, out=out)
        pos += 1
    for i in range(40):
        k.copy_(bf16(rng, (1, H, 1, D)))
        graph.replay()
    assert int(pos) == 40
    check = c.attend(q, ints([40]))
    assert torch.equal(check, out)


def test_python_refusals(cuda):
    rng = np.random.default_rng(21)
    c = make_cache(rng, 2, 2, 64, 16, 4)
    x = bf16(rng, (2, 2, 3, 64)).cuda()
    with pytest.raises(ValueError):
        c.append(x.float(), x, ints([0, 0]))
    with pytest.raises(ValueError):
        c.append(x[:, :1], x[:, :1], ints([0, 0]))
    with pytest.raises(ValueError):
        c.append(x, x, ints([0]))
    with pytest.raises(ValueError):
        c.append(x, x, torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        c.attend(x[:, :, :, :32], ints([3, 3]))
    with pytest.raises(_lib.VbError):
        c.attend(bf16(rng, (2, 3, 1, 64)).cuda(), ints([3, 3]))  # 3 heads over 2
    with pytest.raises(ValueError):
        c.attend(x, ints([3, 3]), out=torch.empty_like(x).float())
