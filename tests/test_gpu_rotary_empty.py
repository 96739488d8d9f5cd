"""Rotary positions of calls without heads or without tokens, whatever the strides of the
empty tensors are (those that come from an empty array have strides of 0)."""
import numpy as np
import pytest
import torch

from test_gpu_rotary import check, places, rows
from vates_b200.rotary import pair_axes, rotate_axes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(0, 3), (5, 0), (0, 0)])
def test_no_heads(cuda, heads, kv_heads, norm):
    rng = np.random.default_rng(heads + kv_heads)
    axes, pos = pair_axes((8, 8)), places(rng, (2, 2, 9), 500)
    w = rows(rng, (48,)) if norm else None
    x = [rows(rng, (2, h, 9, 48)) if h else
         torch.empty(1, dtype=torch.bfloat16, device="cuda").as_strided((2, 0, 9, 48), (0, 0, 0, 0))
         for h in (heads, kv_heads)]
    got = rotate_axes(*x, pos, axes, q_norm=w, k_norm=w)
    for y, z in zip(got, x):
        assert y.shape == z.shape
        if z.numel():
            check(y, z, pos, axes, norm=w)
    back = rotate_axes(*[z.clone() if z.numel() else z for z in x], pos, axes, q_norm=w, k_norm=w,
                       q_out=x[0], k_out=x[1])
    assert all(torch.equal(y, z) for y, z in zip(got, back))


def test_no_tokens(cuda):
    q = torch.empty(1, dtype=torch.bfloat16, device="cuda").as_strided((2, 3, 0, 64), (0, 0, 0, 0))
    pos = torch.empty((1, 2, 0), dtype=torch.int32, device="cuda")
    a, b = rotate_axes(q, q[:, :1], pos, pair_axes((16,)))
    assert a.shape == q.shape and b.shape == (2, 1, 0, 64)
