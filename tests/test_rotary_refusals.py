"""Refusals of the rotary positions' C entry, and the axes of pairs (no GPU)."""
import ctypes as C

import pytest
import torch

from vates_b200 import _lib
from vates_b200._lib import lib
from vates_b200.rotary import pair_axes, rotate_axes

FAKE = 0x10000


def _args(**bad):
    axis, turns = (C.c_uint8 * 128)(*[i % 3 for i in range(128)]), (C.c_double * 128)(*[0.1] * 128)
    d = dict(q=FAKE, k=FAKE, q_out=FAKE, k_out=FAKE, positions=FAKE, eps=1e-6, batch=1, L=2,
             q_heads=4, kv_heads=2, dim=128, rope_dims=64, axes=3,
             turns=C.cast(turns, C.c_void_p), axis=C.cast(axis, C.c_void_p))
    d.update(bad)
    a = _lib.VbRotateArgs(**d)
    a._keep = (axis, turns)
    return a


@pytest.mark.parametrize("bad", [dict(dim=0), dict(dim=24), dict(dim=272), dict(rope_dims=8),
                                 dict(rope_dims=144), dict(rope_dims=40), dict(batch=-1),
                                 dict(L=-1), dict(q_heads=-1), dict(axes=0), dict(axes=2),
                                 dict(eps=-1.0), dict(eps=float("nan")), dict(turns=None),
                                 dict(axis=None), dict(q=None), dict(k_out=None),
                                 dict(positions=None), dict(q=FAKE + 1), dict(k_norm=FAKE + 1)],
                         ids=lambda d: "-".join(d))
def test_refusals(bad):
    assert lib.vb_rotate_axes(C.byref(_args(**bad)), None) == 1
    assert b"vb_rotate_axes" in lib.vb_last_error()


@pytest.mark.parametrize("out", ["q_out_strides", "k_out_strides"])
@pytest.mark.parametrize("strides", [(0, 256, 128), (1024, 0, 128), (1024, 256, 0)])
def test_outputs_whose_rows_share_a_place(out, strides):
    """An expanded tensor, be it the input itself (whose rows may)."""
    three = C.c_int64 * 3
    dense = dict(q_out_strides=three(1024, 256, 128), k_out_strides=three(512, 256, 128))
    a = _args(batch=2, **{**dense, out: three(*strides)})
    assert lib.vb_rotate_axes(C.byref(a), None) == 1
    assert b"one place" in lib.vb_last_error()


def test_no_tokens_are_accepted():
    assert lib.vb_rotate_axes(C.byref(_args(L=0)), None) == 0
    assert lib.vb_rotate_axes(C.byref(_args(q_heads=0, kv_heads=0)), None) == 0


def test_pair_axes():
    assert pair_axes((2, 1, 1)) == (0, 0, 1, 2)
    assert pair_axes((3, 1, 2), True) == (0, 1, 2, 0, 2, 0)
    assert pair_axes(()) == pair_axes((), True) == ()
    assert pair_axes((0, 2)) == (1, 1)
    with pytest.raises(ValueError):
        pair_axes((4, -1))


def test_host_tensors_are_refused():
    x = torch.zeros((1, 1, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        rotate_axes(x, x, torch.zeros((1, 1, 2), dtype=torch.int32), pair_axes((8,)))
