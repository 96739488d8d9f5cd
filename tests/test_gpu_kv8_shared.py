"""Attention of batches that share prefixes in groups, against the plain 64-bit
form of attention with the bounds that hold for it (an exact sum is split in two,
whose float32 results are joined: within the bounds' float32 steps)."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import Plain, attend_plain, bf16, ints, make_cache
from vates_b200 import _lib
from vates_b200.kv8 import SharedPrefix

pytestmark = pytest.mark.gpu


def share(c, groups):
    """The pages of a group's first sequence in the tables of all of its sequences."""
    for first, count, rows in groups:
        n = rows // c.page
        c.page_table[first:first + count, :n] = c.page_table[first, :n].clone()
    return SharedPrefix(c, groups, least=0)  # however little it saves


def check(c, q, groups, lens, q_lens=None, causal=True, len_add=0, scale=None, plan=None, ref=None, **kw):
    B, Hq, L, D = q.shape
    plan = plan or share(c, groups)
    out, lse = c.attend_shared(q, ints([n - len_add for n in lens]), plan,
                               None if q_lens is None else ints(q_lens), len_add=len_add,
                               causal=causal, scale=scale, return_lse=True, **kw)
    want, wl, tol, ltol = attend_plain(ref or Plain(c), q.float().cpu().numpy().astype(np.float64),
                                       lens, q_lens or [L] * B, D ** -0.5 if scale is None else scale,
                                       causal)
    # Weights are f16 with the row's largest at 2^13 or more (2^6 where a part has more
    # than 32 rows of a kv head): what is lost below f16's last step is half of 2^-24 over
    # that, a key, of a value of at most 127 v (v the largest V scale), beside the 11 bits
    # that the bound above has. A part's largest weight is at most the row's.
    rows = L * Hq // c.kv_heads * max([1] + [n for _, n, _ in plan.groups])
    least = 2.0 ** -25 / (2.0 ** 13 if rows <= 32 else 2.0 ** 6)
    tol = tol + max(lens) * least * 127 * float(c.v_scales.max())
    got, gl = out.float().cpu().numpy(), lse.cpu().numpy()
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), (np.abs(got - want) - tol).max())
    empty = np.isinf(wl)
    assert np.array_equal(np.isneginf(gl), empty)
    assert (np.abs(gl - np.where(empty, 0, wl))[~empty] <= ltol[~empty]).all()
    return out, lse


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("L,rep,count", [(1, 1, 2), (1, 8, 2), (1, 8, 4), (2, 4, 5), (1, 7, 9),
                                         (4, 8, 3), (5, 8, 2), (1, 48, 2)])
def test_one_group(cuda, dim, page, L, rep, count):
    """Prefix by either kernel (up to 32 rows of a kv head together, or more), and so
    the sequences' own rows."""
    rng = np.random.default_rng(dim + page + 10 * L + rep)
    c = make_cache(rng, count, 2, dim, page, -(-700 // page))
    q = bf16(rng, (count, 2 * rep, L, dim), 2.0).cuda()
    lens = [384 + int(x) for x in rng.integers(L, 300, count)]
    check(c, q, [(0, count, 384)], lens)
    # idle sequences, the first among them, rows that end early, no mask
    idle = [0] + lens[1:]
    ql = [0] + [max(1, L - b % 2) for b in range(1, count)]
    check(c, q, [(0, count, 256)], idle, ql)
    check(c, q, [(0, count, 256)], idle, ql, causal=False)


@pytest.mark.parametrize("L", [1, 3])
def test_groups_and_sequences_without_one(cuda, L):
    rng = np.random.default_rng(L)
    B = 11
    c = make_cache(rng, B, 3, 128, 32, 20)
    q = bf16(rng, (B, 6, L, 128), 2.0).cuda()
    groups = [(1, 3, 96), (4, 1, 32), (5, 5, 512)]
    lens = [200, 97, 300, 99 + L, 77, 512 + L, 513 + L, 640, 600, 530, L]
    check(c, q, groups, lens)
    check(c, q, groups, [n - 1 for n in lens], len_add=0, causal=False, scale=0.3)
    check(c, q, groups, lens, len_add=L)
    check(c, q, [(4, 1, 32)], lens)   # nothing is shared
    check(c, q, [], lens)


def test_sequences_shorter_than_their_prefix(cuda):
    """A sequence that has not got all of the prefix, or has rows within it, sees what
    it has; pages behind that need not be in its table."""
    rng = np.random.default_rng(3)
    c = make_cache(rng, 5, 2, 64, 16, 40)
    q = bf16(rng, (5, 8, 4, 64)).cuda()
    plan = share(c, [(0, 5, 320)])
    ref = Plain(c)
    c.page_table[1, 7:] = -1
    c.page_table[2] = -1
    lens, ql = [400, 100, 0, 320, 322], [4, 4, 0, 4, 3]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(c, q, None, lens, ql, plan=plan, ref=ref, status=status)
    check(c, q, None, [50, 100, 0, 16, 3], [4, 2, 0, 4, 3], plan=plan, ref=ref, status=status)
    check(c, q, None, [0] * 5, [0] * 5, plan=plan, ref=ref, status=status)
    check(c, q, None, [2, 0, 0, 0, 1], [4, 2, 0, 4, 1], plan=plan, ref=ref, status=status)
    assert int(status) == 0


@pytest.mark.parametrize("B,L,rep,dim,page,rows,tail", [(64, 1, 8, 256, 64, 4096, 300),
                                                        (40, 4, 5, 64, 16, 2064, 90),
                                                        (3, 200, 4, 128, 128, 1280, 400),
                                                        (17, 2, 16, 128, 32, 8192, 33),
                                                        (33, 1, 1, 64, 16, 16384, 100)])
def test_long_prefixes(cuda, B, L, rep, dim, page, rows, tail):
    """Several row tiles and key ranges of the prefix; prompts behind a prefix."""
    rng = np.random.default_rng(B + L)
    c = make_cache(rng, B, 1, dim, page, (rows + tail) // page + 1)
    q = bf16(rng, (B, rep, L, dim), 1.5).cuda()
    lens = [rows + max(L, int(x)) for x in rng.integers(1, tail, B)]
    ql = [0 if b % 8 == 5 else max(1, L - b % 3) for b in range(B)]
    check(c, q, [(0, B, rows)], lens, ql)


@pytest.mark.parametrize("groups,count,L,rep", [(40, 20, 1, 4), (300, 2, 3, 12), (9, 40, 2, 20),
                                                (1, 520, 1, 2), (2, 3, 130, 2), (20, 20, 1, 16),
                                                (260, 2, 130, 2)])
def test_rows_that_are_not_there(cuda, groups, count, L, rep):
    """Row tiles are filled by the rows of this pass: many groups, sequences without
    rows, groups without any, groups whose rows begin anywhere in a tile."""
    rng = np.random.default_rng(groups + count)
    B = groups * count + 1
    c = make_cache(rng, B, 1, 64, 16, 32)
    q = bf16(rng, (B, rep, L, 64), 1.5).cuda()
    ql = [int(n) for n in rng.integers(0, L + 1, B)]
    for g in range(1, groups, 3):
        ql[g * count:(g + 1) * count] = [0] * count
    prefix = [16 * int(n) for n in rng.integers(1, 20, groups)]
    lens = [prefix[min(b // count, groups - 1)] + n + int(rng.integers(0, 40)) for b, n in enumerate(ql)]
    check(c, q, [(g * count, count, prefix[g]) for g in range(groups)], lens, ql)


def test_a_graph_deals_anew_in_each_replay(cuda):
    """Rows per sequence change under a captured call: from all to few, to none."""
    rng = np.random.default_rng(22)
    c = make_cache(rng, 33, 2, 128, 32, 70)
    q = bf16(rng, (33, 16, 4, 128)).cuda()
    plan = share(c, [(0, 16, 2048), (16, 17, 1024)])
    lens, ql = ints([2060 + b for b in range(16)] + [1030 + b for b in range(17)]), ints([4] * 33)
    ref = Plain(c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = c.attend_shared(q, lens, plan, ql, return_lse=True)
    for rows in ([4] * 33, [int(n) for n in rng.integers(0, 5, 33)], [0] * 16 + [1] * 17, [0] * 33,
                 [0] * 32 + [4]):
        ql.copy_(ints(rows))
        g.replay()
        a, la = check(c, q, None, lens.tolist(), rows, plan=plan, ref=ref)
        assert torch.equal(a, out) and torch.equal(la, lse)


def test_bad_row_counts_are_flagged(cuda):
    """Counts and lengths out of range are cut off, as in attention, and flagged."""
    rng = np.random.default_rng(21)
    c = make_cache(rng, 12, 1, 64, 16, 24)
    q = bf16(rng, (12, 40, 1, 64)).cuda()
    plan = share(c, [(0, 12, 160)])
    lens, ql = [170 + b for b in range(12)], [1] * 12
    for bad_lens, bad_ql in (({}, {3: 2}), ({}, {4: -1}), ({5: 385}, {}), ({6: -1}, {6: 0})):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        n = [bad_lens.get(b, x) for b, x in enumerate(lens)]
        m = [bad_ql.get(b, x) for b, x in enumerate(ql)]
        got = c.attend_shared(q, ints(n), plan, ints(m), status=status)
        assert int(status) == _lib.VB_STATUS_BOUNDS
        want = c.attend_shared(q, ints([min(max(x, 0), 384) for x in n]), plan,
                               ints([min(max(x, 0), 1) for x in m]))
        assert torch.equal(got, want)


def test_like_attention_of_each(cuda):
    """Scores of hundreds, where one key has all the weight, are split between the two
    parts too: compared with the attention of every sequence by itself."""
    rng = np.random.default_rng(7)
    c = make_cache(rng, 6, 2, 128, 32, 30)
    q = bf16(rng, (6, 16, 2, 128), 40.0).cuda()
    plan = share(c, [(0, 6, 640)])
    lens = [n - 2 for n in (960, 700, 643, 800, 642, 900)]
    check(c, q, None, lens, plan=plan)
    a, la = c.attend(q, ints(lens), return_lse=True)
    b, lb = c.attend_shared(q, ints(lens), plan, return_lse=True)
    # both within 2^-8 of the exact value (see the bounds above) and of one another
    assert (a.float() - b.float()).abs().max() <= 2 ** -6 * a.float().abs().max()
    assert (la - lb).abs().max() <= 1e-3 * la.abs().max()


def test_little_is_not_shared(cuda):
    """Groups that save little: the attention of every sequence by itself, bit for bit."""
    rng = np.random.default_rng(13)
    c = make_cache(rng, 6, 2, 128, 32, 30)
    lens = ints([960, 700, 643, 800, 642, 900])
    share(c, [(0, 6, 640)])
    saved = 5 * 640 * 2 * 128 * 2
    for L, least in ((2, None), (9, None), (2, saved + 1)):
        q = bf16(rng, (6, 16, L, 128)).cuda()
        plan = SharedPrefix(c, [(0, 6, 640)], least)
        a, la = c.attend(q, lens, return_lse=True)
        b, lb = c.attend_shared(q, lens, plan, return_lse=True)
        assert torch.equal(a, b) and torch.equal(la, lb)
        assert c.shared_workspace_size(plan, 16, L) == c.attend_workspace_size(16, L)
    q = bf16(rng, (6, 16, 2, 128)).cuda()
    check(c, q, None, lens.tolist(), plan=SharedPrefix(c, [(0, 6, 640)], saved))


def test_pages_that_are_not_there(cuda):
    rng = np.random.default_rng(8)
    for count in (3, 12):
        c = make_cache(rng, count, 1, 64, 16, 20)
        q = bf16(rng, (count, 8, 1, 64)).cuda()
        plan = share(c, [(0, count, 160)])
        c.page_table[:, 3], c.page_table[1, 12] = 10 ** 6, -1
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        lens = [200 + b for b in range(count)]
        out = c.attend_shared(q, ints(lens), plan, status=status)
        assert int(status) == _lib.VB_STATUS_BOUNDS
        assert torch.isfinite(out).all()
        # keys without a page have no weight
        want = c.attend(q, ints(lens))
        assert (out.float() - want.float()).abs().max() <= 2 ** -6 * want.float().abs().max()


def test_strides_out_streams_and_graphs(cuda):
    rng = np.random.default_rng(9)
    c = make_cache(rng, 8, 2, 128, 64, 12)
    base = bf16(rng, (8, 2, 8 * 128 + 5)).cuda()
    q = base[..., 3:3 + 8 * 128].unflatten(-1, (8, 128)).transpose(1, 2)
    plan = share(c, [(0, 8, 512)])
    lens = [514 + 30 * b for b in range(8)]
    check(c, q, None, lens, plan=plan)
    n = ints(lens)
    out = torch.empty((8, 8, 2, 128), dtype=torch.bfloat16, device="cuda")
    want = c.attend_shared(q, n, plan)
    assert c.attend_shared(q, n, plan, out=out) is out and torch.equal(out, want)
    ws = torch.zeros(c.shared_workspace_size(plan, 8, 2), dtype=torch.uint8, device="cuda")
    for _ in range(3):
        assert torch.equal(c.attend_shared(q, n, plan, workspace=ws), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = c.attend_shared(q, n, plan, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    # two graphs, replayed on two streams at once, and an eager call between
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = c.attend_shared(q, n, plan)
        graphs.append((g, o))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        eager = c.attend_shared(q, n, plan)
    torch.cuda.synchronize()
    assert torch.equal(eager, want) and all(torch.equal(o, want) for _, o in graphs)
    # lengths are read when it runs
    lens = [512 + b for b in range(2, 10)]
    n.copy_(ints(lens))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], c.attend_shared(q, n, plan))
    del g, graphs


def test_one_plan_for_several_layers(cuda):
    rng = np.random.default_rng(10)
    a, b = make_cache(rng, 4, 2, 64, 16, 30), make_cache(rng, 4, 1, 256, 16, 50)
    plan = share(a, [(0, 4, 320)])
    share(b, [(0, 4, 320)])
    check(a, bf16(rng, (4, 4, 1, 64)).cuda(), None, [330, 400, 321, 460], plan=plan)
    check(b, bf16(rng, (4, 3, 2, 256)).cuda(), None, [330, 400, 322, 700], plan=plan)


def test_python_refusals(cuda):
    rng = np.random.default_rng(11)
    c = make_cache(rng, 4, 2, 64, 16, 8)
    for bad in ([(0, 5, 16)], [(0, 0, 16)], [(-1, 2, 16)], [(0, 2, 8)], [(0, 2, 24)], [(0, 2, 0)],
                [(0, 2, 144)], [(0, 2, 16), (1, 2, 16)], [(2, 2, 16), (0, 2, 16)]):
        with pytest.raises(ValueError):
            SharedPrefix(c, bad)
    with pytest.raises(ValueError):
        SharedPrefix(c, [(0, 2, 16)], least=-1)
    plan = SharedPrefix(c, [(0, 4, 64)], 0)
    q, lens = bf16(rng, (4, 4, 1, 64)).cuda(), ints([70] * 4)
    for bad in (dict(q=q.float()), dict(q=q[:2]), dict(lens=lens[:2]), dict(scale=0.0),
                dict(shared=SharedPrefix(make_cache(rng, 3, 2, 64, 16, 8), [(0, 2, 16)])),
                dict(shared=SharedPrefix(make_cache(rng, 4, 2, 64, 32, 8), [(0, 2, 32)])),
                dict(shared=SharedPrefix(make_cache(rng, 4, 2, 64, 16, 9), [(0, 2, 144)], 0)),
                dict(workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            c.attend_shared(**{**dict(q=q, lens=lens, shared=plan), **bad})
