"""Rotary positions, shared prefixes, accumulated weight and eviction together, as
a server's decode loop uses them: the answers of several sequences behind one
prompt, in a cache that keeps a limited number of rows of each."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import Plain, attend_plain, ints
from test_gpu_kv8_evict import evict_plain, weigh_plain
from test_gpu_rotary import plain as rotate_plain
from vates_b200.kv8 import PagedKV8Cache, SharedPrefix
from vates_b200.rotary import pair_axes, rotate_axes

pytestmark = pytest.mark.gpu
B, HQ, H, D, PAGE = 4, 8, 2, 64, 16
PROMPT, KEEP, RECENT, SLACK = 64, 100, 12, 16
AXES = pair_axes((8, 4, 4), True)


class Loop:
    """One attention layer's buffers; lengths and token counts on the device."""

    def __init__(self):
        width = (KEEP + SLACK + PAGE - 1) // PAGE + 1
        shared, own = PROMPT // PAGE, width - PROMPT // PAGE
        self.cache = PagedKV8Cache.empty(shared + B * own + 1, H, D, B, width, PAGE)
        order = torch.randperm(shared + B * own, generator=torch.Generator().manual_seed(1)).int()
        table = torch.empty((B, width), dtype=torch.int32)
        table[:, :shared] = order[:shared]
        table[:, shared:] = order[shared:].view(B, own)
        self.cache.page_table.copy_(table)
        # (however little it saves)
        self.shared = SharedPrefix(self.cache, [(0, B, PROMPT)], least=0)
        room = width * PAGE
        self.weights = torch.zeros((B, H, room), device="cuda")
        self.positions = torch.zeros((B, H, room), dtype=torch.int32, device="cuda")
        self.lens, self.seen = ints([0] * B), ints([0] * B)
        bf = dict(dtype=torch.bfloat16, device="cuda")
        self.q, self.k = torch.zeros((B, 1, HQ, D), **bf), torch.zeros((B, 1, H, D), **bf)
        self.v = torch.zeros((B, 1, H, D), **bf)
        self.norm = (1 + 0.1 * torch.randn(D, device="cuda")).to(torch.bfloat16)

    def step(self, stream=None):
        """One token of every sequence, at its position in all axes."""
        q, k = rotate_axes(self.q.transpose(1, 2), self.k.transpose(1, 2),
                           self.seen.view(1, B, 1).expand(3, B, 1).contiguous(), AXES,
                           q_norm=self.norm, k_norm=self.norm, stream=stream)
        self.cache.append(k, self.v.transpose(1, 2), self.lens, stream=stream)
        self.lens += 1
        self.seen += 1
        out, lse = self.cache.attend_shared(q, self.lens, self.shared, return_lse=True, stream=stream)
        self.cache.weigh(q, lse, self.lens, self.weights, positions=self.positions, seen=self.seen,
                         stream=stream)
        return q, k, out, lse

    def evict(self):
        self.lens.copy_(self.cache.evict(self.weights, self.lens, KEEP, first=PROMPT, recent=RECENT,
                                         positions=self.positions))

    def tokens(self, rng):
        for t, s in ((self.q, 3.0), (self.k, 1.0), (self.v, 1.0)):
            t.copy_(torch.from_numpy((rng.standard_normal(t.shape) * s).astype(np.float32)))


def prompt(loop, rng):
    """The prompt, once: it is in the first sequence's pages and so in all of them."""
    n = PROMPT
    q, k, v = (torch.from_numpy(rng.standard_normal((1, h, n, D)).astype(np.float32))
               .to(torch.bfloat16).cuda() for h in (HQ, H, H))
    at = torch.arange(n, dtype=torch.int32, device="cuda").expand(3, 1, n).contiguous()
    q, k = rotate_axes(q, k, at, AXES, q_norm=loop.norm, k_norm=loop.norm)
    c = loop.cache
    first = PagedKV8Cache(c.k_codes, c.v_codes, c.k_scales, c.v_scales, c.page_table[:1].contiguous())
    first.append(k, v, ints([0]))
    _, lse = first.attend(q, ints([n]), return_lse=True)
    first.weigh(q, lse, ints([n]), loop.weights[:1], positions=loop.positions[:1], seen=ints([n]))
    loop.weights[1:], loop.positions[1:] = loop.weights[:1], loop.positions[:1]
    loop.lens.fill_(n)
    loop.seen.fill_(n)


def check_step(loop, before, q, k, out, lse, seen):
    """The step's results from what lies in the cache, in 64 bits."""
    c, lens = loop.cache, loop.lens.tolist()
    ref = Plain(c)
    raw = loop.k.transpose(1, 2)
    want, tol = rotate_plain(raw, torch.tensor(seen).view(1, B, 1).expand(3, B, 1), AXES,
                             10_000_000.0, loop.norm)
    assert ((k.double().cpu() - want).abs() <= tol).all()
    qn = q.float().cpu().numpy().astype(np.float64)
    want, wl, tol, ltol = attend_plain(ref, qn, lens, [1] * B, D ** -0.5, True)
    # (weights below the last step of f16: half of it, a key, of 127 scales; 2^13 at least
    # is the largest)
    tol = tol + max(lens) * 2.0 ** -38 * 127 * float(c.v_scales.max())
    assert (np.abs(out.float().cpu().numpy() - want) <= tol).all()
    assert (np.abs(lse.cpu().numpy() - wl) <= ltol).all()
    sums, tols = weigh_plain(ref, qn, lse.cpu().numpy().astype(np.float64), lens, [1] * B,
                             D ** -0.5, True)
    got, pos = loop.weights.cpu().numpy(), loop.positions.cpu().numpy()
    for b in range(B):
        n = lens[b]
        w = before[b].astype(np.float64)
        w[:, n - 1] = 0
        w[:, :n] += sums[b]
        assert (np.abs(got[b] - w)[:, :n] <= tols[b] + w[:, :n] * 2.0 ** -23).all()
        assert np.array_equal(got[b][:, n:], before[b][:, n:])
        assert (pos[b, :, n - 1] == seen[b]).all()


def test_decode_loop(cuda):
    rng = np.random.default_rng(1)
    torch.manual_seed(1)
    loop = Loop()
    prompt(loop, rng)
    shared = loop.cache.page_table[0, :PROMPT // PAGE].long()
    was = [t[shared].clone() for t in (loop.cache.k_codes, loop.cache.v_codes, loop.cache.k_scales,
                                       loop.cache.v_scales)]
    for step in range(3 * (KEEP - PROMPT + SLACK)):
        loop.tokens(rng)
        before, seen = loop.weights.cpu().numpy(), loop.seen.tolist()
        got = loop.step()
        if step % 7 == 0 or step > 100:
            check_step(loop, before, *got, seen)
        if int(loop.lens.max()) >= KEEP + SLACK:
            ref, w, p = Plain(loop.cache), loop.weights.cpu().numpy(), loop.positions.cpu().numpy()
            lens = loop.lens.tolist()
            loop.evict()
            assert loop.lens.tolist() == evict_plain(ref, w, p, lens, KEEP, PROMPT, RECENT)
            assert np.array_equal(loop.weights.cpu().numpy(), w)
            assert np.array_equal(loop.positions.cpu().numpy(), p)
            assert np.array_equal(loop.cache.k_codes.cpu().numpy(), ref.codes[0])
            assert np.array_equal(loop.cache.v_scales.cpu().numpy(), ref.scales[1])
            kept = loop.positions[:, :, :KEEP].sort(-1).values
            last = int(loop.seen[0])
            # the prompt and the newest tokens are all there, and nothing twice
            assert (kept[..., :PROMPT] == torch.arange(PROMPT, device="cuda")).all()
            assert (kept[..., -RECENT:] == torch.arange(last - RECENT, last, device="cuda")).all()
            assert (kept.diff(dim=-1) > 0).all()
    assert int(loop.seen[0]) == PROMPT + 3 * (KEEP - PROMPT + SLACK) and int(loop.lens.max()) < KEEP + SLACK
    for t, o in zip((loop.cache.k_codes, loop.cache.v_codes, loop.cache.k_scales,
                     loop.cache.v_scales), was):
        assert torch.equal(t[shared], o)


def test_decode_loop_as_a_graph(cuda):
    """A captured step, replayed between evictions: what the eager loop computes."""
    loops, outs = [Loop(), Loop()], [[], []]
    torch.manual_seed(2)
    norm = (1 + 0.1 * torch.randn(D, device="cuda")).to(torch.bfloat16)
    for loop in loops:
        loop.norm.copy_(norm)
        prompt(loop, np.random.default_rng(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = loops[1].step()
    torch.cuda.synchronize()
    for i, loop in enumerate(loops):
        rng = np.random.default_rng(3)
        for step in range(2 * (KEEP - PROMPT + SLACK)):
            loop.tokens(rng)
            if i:
                graph.replay()
                got = held
            else:
                got = loop.step()
            outs[i].append(got[2].clone())
            if int(loop.lens.max()) >= KEEP + SLACK:
                loop.evict()
    torch.cuda.synchronize()
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    for name in ("weights", "positions", "lens", "seen"):
        assert torch.equal(getattr(loops[0], name), getattr(loops[1], name))
    assert torch.equal(loops[0].cache.k_codes, loops[1].cache.k_codes)
    del graph, held
