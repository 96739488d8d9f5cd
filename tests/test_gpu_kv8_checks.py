"""What the Python entry points of the 8-bit cache and the log probabilities refuse:
tensors of another device or type, before their addresses reach a kernel."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import bf16, ints, make_cache
from vates_b200 import kv8, logprobs
from vates_b200.kv8 import PagedKV8Cache
from vates_b200.logprobs import token_logprobs

pytestmark = pytest.mark.gpu


class Elsewhere:
    """A stream of a GPU that is not the tensors'."""
    device = torch.device("cuda", 77)


BAD_STATUS = [torch.zeros(1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32),
              torch.zeros(1, dtype=torch.int64)]


@pytest.fixture
def cache(cuda):
    rng = np.random.default_rng(1)
    return make_cache(rng, 2, 2, 64, 16, 4), bf16(rng, (2, 2, 3, 64)).cuda()


def test_host_output_is_refused(cache):
    c, x = cache
    with pytest.raises(ValueError, match="out"):
        c.attend(x, ints([3, 3]), out=torch.empty((2, 2, 3, 64), dtype=torch.bfloat16))


@pytest.mark.parametrize("bad", range(len(BAD_STATUS)))
@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_status_words(cache, bad, where):
    c, x = cache
    status = BAD_STATUS[bad].to(where)
    if where == "cuda" and bad == 0:
        c.append(x, x, ints([0, 0]), status=status)
        c.attend(x, ints([3, 3]), status=status)
        c.read(ints([3, 3]), 3, status=status)
        assert int(status) == 0
        return
    with pytest.raises(ValueError, match="status"):
        c.append(x, x, ints([0, 0]), status=status)
    with pytest.raises(ValueError, match="status"):
        c.attend(x, ints([3, 3]), status=status)
    with pytest.raises(ValueError, match="status"):
        c.read(ints([3, 3]), 3, status=status)
    with pytest.raises(ValueError, match="status"):
        token_logprobs(torch.zeros((2, 10), device="cuda"), ints([0, 0]), status=status)


def test_host_tensors_beside_device_ones(cache):
    c, x = cache
    two = ints([3, 3])
    with pytest.raises(ValueError, match="pos"):
        c.append(x, x, two.cpu())
    with pytest.raises(ValueError, match="counts"):
        c.append(x, x, two, counts=two.cpu())
    with pytest.raises(ValueError, match="values"):
        c.append(x, x.cpu(), two)
    with pytest.raises(ValueError, match="lens"):
        c.read(two.cpu(), 3)
    with pytest.raises(ValueError, match="start"):
        c.read(two, 3, start=two.cpu())
    with pytest.raises(ValueError, match="q_lens"):
        c.attend(x, two, q_lens=two.cpu())
    with pytest.raises(ValueError, match="page_table"):
        c.page_table = c.page_table.cpu()
    with pytest.raises(ValueError):
        PagedKV8Cache(c.k_codes, c.v_codes.cpu(), c.k_scales, c.v_scales, c.page_table)
    with pytest.raises(ValueError, match="tokens"):
        token_logprobs(torch.zeros((2, 10), device="cuda"), two.cpu())


def test_stream_of_another_device(cache):
    c, x = cache
    for call in (lambda s: c.append(x, x, ints([0, 0]), stream=s),
                 lambda s: c.read(ints([3, 3]), 3, stream=s),
                 lambda s: c.attend(x, ints([3, 3]), stream=s),
                 lambda s: token_logprobs(torch.zeros((2, 10), device="cuda"), ints([0, 0]),
                                          stream=s)):
        with pytest.raises(ValueError, match="stream"):
            call(Elsewhere())


def test_calls_move_to_the_tensors_device(cache, monkeypatch):
    """With another GPU current, a call runs on the tensors' own (faked: the current
    device is another one until the call has changed it)."""
    c, x = cache
    want = c.attend(x, ints([3, 3])), *c.read(ints([3, 3]), 3)
    score = token_logprobs(x[0, 0].float(), ints([0, 1, 2]))
    real, moved = kv8.on_device, []

    def on_device(device, stream):
        moved.append(device)
        return real(device, stream)

    for module in (kv8, logprobs):
        monkeypatch.setattr(module, "on_device", on_device)
        monkeypatch.setattr(module, "current_device",
                            lambda: x.device.index if len(moved) % 2 else 77)
    got = [c.attend(x, ints([3, 3]))]
    moved.append(None)
    got += c.read(ints([3, 3]), 3)
    moved.append(None)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    again = token_logprobs(x[0, 0].float(), ints([0, 1, 2]))
    moved.append(None)
    assert torch.equal(score.logprob, again.logprob)
    c.append(x, x, ints([0, 0]))
    assert moved == [x.device, None] * 3 + [x.device]
