"""Token log probabilities on the GPU against float64 on the CPU."""
import math

import numpy as np
import pytest
import torch

from vates_b200 import _lib
from vates_b200.logprobs import token_logprobs

pytestmark = pytest.mark.gpu


def plain(x, tok, top, T):
    """float64 results and error bounds. A CTA's thread adds up to V / 512 + 8
    terms (slices and warps add 40 more joins) in float32, the exponentials and
    y = x c - m carry 2^-22 (1 + |y|): n 2^-24 + 2^-21 relative on the sums,
    and 2^-22 of |log p| for the rounding of c."""
    R, V = x.shape
    z = x.astype(np.float64) / T
    m = z.max(1, keepdims=True)
    e = np.exp(z - m)
    s = e.sum(1, keepdims=True)
    logp = z - m - np.log(s)
    p = e / s
    with np.errstate(invalid="ignore"):
        plogp = np.where(p > 0, p * logp, 0.0)
    order = np.lexsort((np.arange(V)[None].repeat(R, 0), -x), axis=-1)[:, :top]
    xt = x[np.arange(R), tok][:, None]
    ids = np.arange(V)[None]
    rank = ((x > xt) | ((x == xt) & (ids < tok[:, None]))).sum(1)
    eps = (V / 512 + 48) * 2.0 ** -24 + 2.0 ** -21
    lp = logp[np.arange(R), tok]
    tlp = np.take_along_axis(logp, order, 1)
    tol = lambda a: eps + 2.0 ** -21 * np.where(np.isfinite(a), np.abs(a), 0)  # noqa: E731
    return dict(logprob=(lp, tol(lp)), rank=rank, ids=order, top=(tlp, tol(tlp)),
                entropy=(-plogp.sum(1), eps * (2 + 2 * np.abs(plogp).sum(1))))


def close(got, want, tol):
    got = got.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    fin = np.isfinite(want)
    assert (np.abs(got[fin] - want[fin]) <= tol[fin]).all(), np.abs(got[fin] - want[fin]).max()


def check(x, tok, top=5, T=1.0):
    """x: torch CPU tensor in its type; tok numpy int."""
    got = token_logprobs(x.cuda(), torch.from_numpy(tok.astype(np.int32)).cuda(), top=top,
                         temperature=T)
    want = plain(x.float().numpy(), tok, top, T)
    assert np.array_equal(got.rank.cpu().numpy(), want["rank"])
    assert np.array_equal(got.top_ids.cpu().numpy(), want["ids"])
    close(got.logprob, *want["logprob"])
    close(got.entropy, *want["entropy"])
    close(got.top_logprobs, *want["top"])
    return got


def logits(rng, R, V, dtype, scale=2.5):
    x = rng.standard_normal((R, V)).astype(np.float32) * np.float32(scale)
    x[np.arange(R), rng.integers(0, V, R)] += 8
    return torch.from_numpy(x).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (1, 7, 7), (3, 8, 0), (2, 33, 32), (5, 1000, 20),
                                     (4, 4097, 5), (1, 151936, 20), (4, 151936, 5),
                                     (2, 50257, 32), (300, 2049, 1), (150, 9001, 8)])
@pytest.mark.parametrize("T", [1.0, 0.6])
def test_sizes(cuda, dtype, R, V, top, T):
    rng = np.random.default_rng(R * V + top)
    x = logits(rng, R, V, dtype)
    tok = rng.integers(0, V, R)
    tok[0] = 0
    if R > 1:
        tok[1] = V - 1
    check(x, tok, top, T)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_go_to_the_lowest_id(cuda, dtype):
    rng = np.random.default_rng(1)
    for V in (40, 5000, 151936):
        x = torch.from_numpy(rng.integers(-2, 3, (3, V)).astype(np.float32)).to(dtype)
        x[2] = 1.0  # a uniform row
        x[1] *= -0.0  # zeros of both signs are equal
        check(x, rng.integers(0, V, 3), 32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sorted_rows(cuda, dtype):
    """The best logits side by side, at either end of a row."""
    for V in (30000, 151936):
        up = torch.linspace(-40, 40, V)
        x = torch.stack([up, up.flip(0)]).to(dtype)
        check(x, np.array([V - 3, 2]), 32)


@pytest.mark.parametrize("mask", [-math.inf, torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_tokens(cuda, dtype, mask):
    """Tokens that cannot follow, as -inf or the type's lowest value; a few
    allowed tokens among many masked ones, masked tokens asked for."""
    rng = np.random.default_rng(2)
    for V in (300, 60000):
        x = logits(rng, 4, V, dtype)
        hide = torch.from_numpy(rng.random((4, V)) < 0.5)
        hide[1] = True
        hide[1, 17] = hide[1, V - 1] = False
        hide[2] = True
        hide[2, 200] = False
        x = torch.where(hide, torch.tensor(mask, dtype=dtype), x)
        tok = np.array([int(torch.nonzero(hide[0])[3]), 17, 200, int(torch.nonzero(~hide[3])[5])])
        got = token_logprobs(x.cuda(), torch.from_numpy(tok.astype(np.int32)).cuda(), top=20)
        want = plain(x.float().numpy(), tok, 20, 1.0)
        assert np.array_equal(got.rank.cpu().numpy(), want["rank"])
        assert np.array_equal(got.top_ids.cpu().numpy(), want["ids"])
        for name, w in (("logprob", "logprob"), ("entropy", "entropy"), ("top_logprobs", "top")):
            g, (ref, tol) = getattr(got, name).cpu().numpy().astype(np.float64), want[w]
            low = ref < -1e30  # the lowest value or -inf: as low in the result
            assert (g[low] < -1e30).all()
            assert (np.abs(g[~low] - ref[~low]) <= tol[~low]).all()


def test_rows_of_masks_alone_and_nonfinite_rows(cuda):
    rng = np.random.default_rng(3)
    for V in (100, 151936):
        x = logits(rng, 5, V, torch.bfloat16)
        x[1] = -math.inf
        x[2, 50] = math.nan
        x[3, 70] = math.inf
        tok = ints = torch.tensor([1, 2, 3, 4, 5], dtype=torch.int32).cuda()
        got = token_logprobs(x.cuda(), tok, top=4)
        for name in ("logprob", "entropy"):
            bad = getattr(got, name).isnan().cpu()
            assert bad.tolist() == [False, True, True, True, False]
        assert got.top_ids[1].tolist() == [0, 1, 2, 3]
        assert got.top_logprobs[1:4].isnan().all() and got.top_logprobs[4].isfinite().all()
        clean = token_logprobs(x[[0, 4]].cuda(), ints[[0, 4]].contiguous(), top=4)
        if V == 100:  # one CTA per row either way
            assert torch.equal(clean.logprob, got.logprob[[0, 4]])


def test_row_of_the_lowest_value_is_uniform(cuda):
    x = torch.full((1, 5000), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16)
    got = token_logprobs(x.cuda(), torch.zeros(1, dtype=torch.int32).cuda(), top=2)
    assert abs(float(got.logprob) + math.log(5000)) < 1e-3
    assert abs(float(got.entropy) - math.log(5000)) < 1e-3
    assert got.top_ids.tolist() == [[0, 1]]


def test_token_outside_the_vocabulary(cuda):
    rng = np.random.default_rng(4)
    x = logits(rng, 3, 999, torch.float32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = token_logprobs(x.cuda(), torch.tensor([-1, 5, 999], dtype=torch.int32).cuda(), top=3,
                         status=status)
    assert int(status) == _lib.VB_STATUS_BOUNDS
    assert got.rank.tolist()[0] == got.rank.tolist()[2] == -1
    assert got.logprob.isnan().tolist() == [True, False, True]
    want = plain(x.numpy(), np.array([0, 5, 0]), 3, 1.0)
    close(got.entropy, *want["entropy"])
    assert np.array_equal(got.top_ids.cpu().numpy(), want["ids"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(cuda, dtype):
    """Rows of an odd stride at every offset from a 16-byte boundary, a
    broadcast row, and columns that are not contiguous."""
    rng = np.random.default_rng(5)
    V = 9003
    wide = logits(rng, 6, V + 30, dtype).cuda()
    tok = rng.integers(0, V, 6)
    t32 = torch.from_numpy(tok.astype(np.int32)).cuda()
    for off in range(9):
        x = wide[:, off:off + V]
        a = token_logprobs(x, t32, top=6)
        want = plain(x.float().cpu().numpy(), tok, 6, 1.0)
        assert np.array_equal(a.top_ids.cpu().numpy(), want["ids"])
        assert np.array_equal(a.rank.cpu().numpy(), want["rank"])
        close(a.logprob, *want["logprob"])
        close(a.entropy, *want["entropy"])
    row = wide[:1, :V].expand(6, V)
    got = token_logprobs(row, t32, top=2)
    want = plain(row.float().cpu().numpy(), tok, 2, 1.0)
    close(got.logprob, *want["logprob"])
    cols = wide[:, :2 * (V // 2):2]
    got = token_logprobs(cols, t32 // 3, top=2)
    want = plain(cols.float().cpu().numpy(), tok // 3, 2, 1.0)
    close(got.logprob, *want["logprob"])


def test_repeatable_and_workspace_shared_by_sizes(cuda):
    """Split and unsplit calls in turn on one workspace, on two streams: the
    same bits every time."""
    rng = np.random.default_rng(6)
    sets = [(logits(rng, R, V, torch.bfloat16).cuda(),
             torch.from_numpy(rng.integers(0, V, R).astype(np.int32)).cuda(), k)
            for R, V, k in ((2, 151936, 20), (140, 9000, 3), (400, 3000, 5), (1, 70001, 32))]
    torch.cuda.synchronize()
    first = [token_logprobs(x, t, top=k) for x, t, k in sets]
    side = torch.cuda.Stream()
    for stream in (None, side, side):
        for (x, t, k), f in zip(sets, first):
            again = token_logprobs(x, t, top=k, stream=stream)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(f, again))


def test_python_refusals(cuda):
    x = torch.zeros((2, 10), device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        token_logprobs(x, t, top=11)
    with pytest.raises(ValueError):
        token_logprobs(x, t, top=-1)
    with pytest.raises(ValueError):
        token_logprobs(x, t.long())
    with pytest.raises(ValueError):
        token_logprobs(x.half(), t)
    with pytest.raises(_lib.VbError):
        token_logprobs(x, t, temperature=0.0)


@pytest.mark.parametrize("kind", ["equal", "few", "one_slice", "steps"])
@pytest.mark.parametrize("rows,top", [(1, 32), (3, 20), (40, 7)])
def test_best_across_slices(cuda, kind, rows, top):
    """Best logits that lie in one slice, in all, in fewer places than are asked for
    (the others -inf), and equal ones that go by id."""
    rng = np.random.default_rng(rows + top)
    V = 151936
    x = np.zeros((rows, V), np.float32)
    if kind == "few":
        x[:] = -np.inf
        x[:, rng.choice(V, 40, replace=False)] = rng.standard_normal(40).astype(np.float32)
    elif kind == "one_slice":
        x[:, 70000:70100] = 1 + np.arange(100, dtype=np.float32) / 32
    elif kind == "steps":
        x[:] = np.floor(np.arange(V) / 5000) / 4
    check(torch.from_numpy(x).to(torch.bfloat16), rng.integers(0, 40, rows) * 3001, top)
