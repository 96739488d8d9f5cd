"""The device memory of a SharedPrefix lives as long as kernels read it."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import bf16, ints, make_cache
from test_gpu_kv8_shared import share
from vates_b200.kv8 import SharedPrefix

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count,L", [(3, 2), (12, 4)])
@pytest.mark.parametrize("made_on_side", [False, True])
def test_a_plan_of_one_step_on_another_stream(cuda, count, L, made_on_side):
    """A plan that is made on one stream, used on another one that is busy, and let go: no
    tensor that is made on its own stream meanwhile gets its memory."""
    rng = np.random.default_rng(count)
    c = make_cache(rng, count, 2, 64, 16, 40)
    q, lens = bf16(rng, (count, 8, L, 64)).cuda(), ints([500 + 9 * b for b in range(count)])
    want = c.attend_shared(q, lens, share(c, [(0, count, 480)]))
    here, there = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(here):
        plan = SharedPrefix(c, [(0, count, 480)], 0)
        # (both streams have memory of their own before one is busy: asking for more may wait)
        others = [torch.empty(plan._words.numel(), dtype=torch.int32, device="cuda") for _ in range(64)]
    at, n = plan._segments, plan._words.numel()
    busy = here if made_on_side else there
    got = c.attend_shared(q, lens, plan, stream=busy)
    torch.cuda.synchronize()
    del got, others
    with torch.cuda.stream(busy):
        torch.cuda._sleep(1_000_000_000)
    got = c.attend_shared(q, lens, plan, stream=busy)
    del plan
    with torch.cuda.stream(here):
        others = [torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(64)]
    assert not busy.query()
    # (on the stream that used it the next tensor may have it: what writes it comes later)
    assert made_on_side or all(t.data_ptr() != at for t in others)
    busy.synchronize()
    assert torch.equal(got, want)


def test_a_captured_plan(cuda):
    """A plan of another stream in a capture, with other plans made and let go beside it."""
    rng = np.random.default_rng(5)
    c = make_cache(rng, 6, 2, 128, 32, 30)
    q, lens = bf16(rng, (6, 8, 2, 128)).cuda(), ints([700, 702, 800, 645, 900, 960])
    plan = share(c, [(0, 6, 640)])
    want = c.attend_shared(q, lens, plan)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = c.attend_shared(q, lens, plan)
    for _ in range(3):
        other = SharedPrefix(c, [(0, 6, 320)], 0)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del other
    del g
    del plan
    torch.cuda.synchronize()
    assert torch.equal(c.attend_shared(q, lens, SharedPrefix(c, [(0, 6, 640)], 0)), want)
