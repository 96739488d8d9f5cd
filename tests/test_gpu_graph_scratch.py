"""Attention over the 8-bit cache, log probabilities and the MoE block in CUDA
graphs: graphs that were captured without a warm-up, that outlive larger calls, and that run
side by side give what an eager call gives."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import bf16, ints, make_cache
from vates_b200 import _lib
from vates_b200.logprobs import token_logprobs

pytestmark = pytest.mark.gpu


class Attend:
    """Rows of a batch over one cache, split over key ranges."""

    def __init__(self, L, seed=0, batch=3, rep=2):
        rng = np.random.default_rng(seed)
        # (joined by the last of several CTAs: 24 units of up to 3,000 keys)
        self.c = make_cache(rng, batch, 8, 128, 32, 96)
        self.q = bf16(rng, (batch, 8 * rep, L, 128)).cuda()
        self.lens = ints([3000 - 700 * b for b in range(batch)])

    def __call__(self):
        return list(self.c.attend(self.q, self.lens, return_lse=True))


class Score:
    def __init__(self, rows, top, seed=0, vocab=151936):
        rng = np.random.default_rng(seed)
        self.x = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32)).cuda()
        self.t = ints(rng.integers(0, vocab, rows).tolist())
        self.top = top

    def __call__(self):
        return list(token_logprobs(self.x, self.t, top=self.top))


SETS = {"attend": (lambda: Attend(1), lambda: Attend(4, 1)),
        "prompt": (lambda: Attend(40, 2, 1), lambda: Attend(70, 3, 2)),
        "score": (lambda: Score(2, 5), lambda: Score(7, 32, 1))}


def capture(fn, stream=None):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        out = fn()
    return g, out


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


def clear(out):
    for t in out:
        t.fill_(7)


def warm(*fns):
    """Kernels loaded and attributes set, on a stream that nothing else uses."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [f() for f in fns]
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("kind", SETS)
def test_first_calls_inside_captures(cuda, kind):
    """Two graphs captured one after the other on a stream that has seen no call;
    the second runs first, then an eager call on that stream, then the first."""
    small, large = (f() for f in SETS[kind])
    want_s, want_l = warm(small, large)
    stream = torch.cuda.Stream()
    g1, o1 = capture(small, stream)
    g2, o2 = capture(small, stream)
    for t in o1 + o2:
        t.fill_(7)
    g2.replay()
    torch.cuda.synchronize()
    assert same(o2, want_s)
    with torch.cuda.stream(stream):
        eager = large()
    torch.cuda.synchronize()
    assert same(eager, want_l)
    for _ in range(2):
        clear(o1)
        g1.replay()
        torch.cuda.synchronize()
        assert same(o1, want_s)


@pytest.mark.parametrize("kind", SETS)
def test_a_larger_call_after_a_capture(cuda, kind):
    """A graph whose stream later needs more scratch, eagerly and in another
    graph, keeps its own: it writes into nobody else's memory."""
    small, large = (f() for f in SETS[kind])
    want_s, want_l = warm(small, large)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        small()
    torch.cuda.synchronize()
    g1, o1 = capture(small, stream)
    with torch.cuda.stream(stream):
        large()
    torch.cuda.synchronize()
    g2, o2 = capture(large, stream)
    with torch.cuda.stream(stream):  # whatever the stream has given back is taken again
        taken = [torch.full((n,), 0x5A, dtype=torch.uint8, device="cuda")
                 for n in [1 << 16] * 8 + [1 << 20] * 8 + [1 << 23] * 8]
    torch.cuda.synchronize()
    for _ in range(3):
        clear(o1 + o2)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert same(o1, want_s) and same(o2, want_l)
    assert all(bool((t == 0x5A).all()) for t in taken)


@pytest.mark.parametrize("kind", SETS)
def test_graphs_side_by_side(cuda, kind):
    """Two graphs captured on one stream, replayed on two at a time."""
    a, b = (f() for f in SETS[kind])
    want_a, want_b = warm(a, b)
    stream = torch.cuda.Stream()
    repeat = lambda f: lambda: [f() for _ in range(8)][-1]
    ga, oa = capture(repeat(a), stream)
    gb, ob = capture(repeat(b), stream)
    sides = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        clear(oa + ob)
        torch.cuda.synchronize()
        for s, g in zip(sides, (ga, gb)):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert same(oa, want_a) and same(ob, want_b)


def test_moe_block_graph_outlives_a_larger_call(cuda):
    """A block of one token captured, then one of eight called: the graph's scratch
    (its barrier's counter among it) is nobody else's. And a graph whose capture
    is the first call on its workspace."""
    from vates_b200.moe_block import Workspace
    from vates_b200.synth import config0, input_tokens
    blk, _ = config0(seed=0)
    x1, x8 = input_tokens(31, 1), input_tokens(32, 8)
    blk.workspace = Workspace()
    want1, want8 = (t.clone() for t in warm(lambda: blk.decode(x1), lambda: blk.decode(x8)))
    for first_in_capture in (False, True):
        blk.workspace = Workspace()
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.empty_like(want1)
        if not first_in_capture:
            blk.decode(x1)
        torch.cuda.synchronize()
        g, _ = capture(lambda: blk.decode(x1, out=out, status=status))
        assert torch.equal(blk.decode(x8), want8)
        taken = [torch.full((n,), 0x5A, dtype=torch.uint8, device="cuda")
                 for n in [1 << 14] * 8 + [1 << 17] * 8 + [1 << 20] * 8]
        for _ in range(3):
            out.fill_(7)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want1) and int(status) == 0
        assert all(bool((t == 0x5A).all()) for t in taken)


def test_callers_workspace(cuda):
    rng = np.random.default_rng(3)
    c = make_cache(rng, 3, 8, 128, 32, 96)
    for L in (1, 40):
        q = bf16(rng, (3, 16, L, 128)).cuda()
        lens = ints([3000, 2000, 1000])
        want = c.attend(q, lens)
        need = c.attend_workspace_size(16, L)
        ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for stream in (None, side):
            got = c.attend(q, lens, workspace=ws, stream=stream)
            torch.cuda.synchronize()  # (results on another stream than the comparison's)
            assert torch.equal(got, want)
        with pytest.raises(_lib.VbError, match="workspace"):
            c.attend(q, lens, workspace=ws[:need - 1])
        for bad in (ws.cpu(), ws.view(torch.int8)):
            with pytest.raises(ValueError, match="workspace"):
                c.attend(q, lens, workspace=bad)
