"""Rotary positions with several axes against a plain 64-bit form."""
import math

import numpy as np
import pytest
import torch

from vates_b200.rotary import pair_axes, rotate_axes

pytestmark = pytest.mark.gpu
BASE = 10_000_000.0


def plain(x, positions, axes, base, norm, eps=1e-6):
    """float64 rows, and a bound on the kernel's error: the rounding to bf16
    (2^-8 of the value) after float32 steps. Sine and cosine are off by at most
    2^-21 (the turn as a float, 2^-23, and two units of the function's last place),
    the norm by 2^-20 (a sum of 16 products a lane and 4 steps over lanes, under a
    root, rsqrt and two products), each of |a| + |b| of the pair."""
    half = len(axes)
    x = x.double().cpu()
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double().cpu()
    pos = positions.double().cpu()
    freq = torch.tensor([base ** (-i / half) for i in range(half)], dtype=torch.float64)
    angle = torch.stack([pos[a] for a in axes], -1) * freq            # [B, L, half]
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    y = torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), -1)
    mag = a.abs() + b.abs()
    mag = torch.cat((mag, mag, x[..., 2 * half:].abs()), -1)
    return y, y.abs() * 2.0 ** -8 + mag * 2.0 ** -19


def rows(rng, shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(torch.bfloat16).cuda()


def places(rng, shape, far):
    return torch.from_numpy(rng.integers(-far, far, shape).astype(np.int32)).cuda()


def check(got, x, positions, axes, base=BASE, norm=None):
    want, tol = plain(x, positions, axes, base, norm)
    assert got.shape == x.shape and got.dtype == torch.bfloat16
    assert ((got.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("dim,rope", [(64, 64), (64, 32), (16, 16), (80, 80), (96, 48), (128, 128),
                                      (192, 64), (256, 64), (256, 256), (240, 176)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("B,L,Hq,Hk", [(1, 1, 16, 2), (3, 5, 4, 1), (2, 301, 7, 3)])
def test_rotate(cuda, dim, rope, norm, B, L, Hq, Hk):
    rng = np.random.default_rng(dim + rope + L)
    half = rope // 2
    axes = pair_axes((half // 4 + 1, half - half // 2 - half // 4 - 1, half // 2),
                     interleaved=L % 2 == 0 or dim == 80)
    q, k = rows(rng, (B, Hq, L, dim)), rows(rng, (B, Hk, L, dim))
    pos = places(rng, (3, B, L), 100000)
    w = [rows(rng, (dim,)) + 1 if norm else None for _ in range(2)]
    q2, k2 = rotate_axes(q, k, pos, axes, q_norm=w[0], k_norm=w[1])
    check(q2, q, pos, axes, norm=w[0])
    check(k2, k, pos, axes, norm=w[1])


def test_positions_far_and_extreme(cuda):
    """Where a float32 product of position and frequency is off by whole radians."""
    rng = np.random.default_rng(1)
    q, k = rows(rng, (1, 2, 6, 128)), rows(rng, (1, 1, 6, 128))
    pos = torch.tensor([[[0, -1, 2 ** 31 - 1, -2 ** 31, 99_999_999, 1 << 24]]], dtype=torch.int32,
                       device="cuda").repeat(2, 1, 1)
    axes = pair_axes((40, 24))
    for got, x in zip(rotate_axes(q, k, pos, axes, base=10000.0), (q, k)):
        # (the double product of 2^31 radians is itself off by up to 2^-22 turns)
        want, tol = plain(x, pos, axes, 10000.0, None)
        assert ((got.double().cpu() - want).abs() <= tol * 2).all()


def test_strides_alignment_and_in_place(cuda):
    """Views of a projection, odd element offsets, outputs with strides, and rows
    rotated where they are."""
    rng = np.random.default_rng(2)
    B, L, Hq, Hk, D = 2, 37, 6, 2, 64
    axes = pair_axes((5, 7, 4), True)
    pos = places(rng, (3, B, L), 5000)
    for shift in (0, 3, 8):
        base = rows(rng, (B, L, (Hq + Hk) * D + 16))
        q = base[..., shift:shift + Hq * D].unflatten(-1, (Hq, D)).transpose(1, 2)
        k = base[..., shift + Hq * D:shift + (Hq + Hk) * D].unflatten(-1, (Hk, D)).transpose(1, 2)
        q0, k0, outside = q.clone(), k.clone(), base.clone()
        q2, k2 = rotate_axes(q, k, pos, axes)
        check(q2, q0, pos, axes)
        check(k2, k0, pos, axes)
        room = torch.zeros((B, Hq, L + 3, D + 8), dtype=torch.bfloat16, device="cuda")
        part = room[:, :, 2:2 + L, :D]
        rotate_axes(q, k, pos, axes, q_out=part)
        assert torch.equal(part, q2)
        assert not room[:, :, :2].any() and not room[:, :, 2 + L:].any() and not room[..., D:].any()
        got = rotate_axes(q, k, pos, axes, q_out=q, k_out=k)
        assert got[0] is q and torch.equal(q, q2) and torch.equal(k, k2)
        keep = torch.ones_like(base, dtype=torch.bool)
        keep[..., shift:shift + (Hq + Hk) * D] = False
        assert torch.equal(base[keep], outside[keep])
    # dims that are not contiguous are copied
    t = rows(rng, (B, Hq, D, L)).transpose(2, 3)
    q2, _ = rotate_axes(t, k, pos, axes)
    check(q2, t, pos, axes)


def test_one_norm_only_and_in_place_norm(cuda):
    rng = np.random.default_rng(3)
    q, k = rows(rng, (1, 4, 9, 128)), rows(rng, (1, 2, 9, 128))
    w = rows(rng, (128,))
    pos, axes = places(rng, (1, 1, 9), 1000), pair_axes((32,))
    q0, k0 = q.clone(), k.clone()
    rotate_axes(q, k, pos, axes, k_norm=w, q_out=q, k_out=k)
    check(q, q0, pos, axes)
    check(k, k0, pos, axes, norm=w)
    # a zero row stays zero, a weight at an odd address is read
    k.zero_()
    odd = rows(rng, (129,))[1:]
    _, z = rotate_axes(q, k, pos, axes, k_norm=odd)
    assert not z.any()
    _, z = rotate_axes(q, k0, pos, axes, k_norm=odd)
    check(z, k0, pos, axes, norm=odd)


def test_special_values_stay_in_their_rows(cuda):
    rng = np.random.default_rng(4)
    q, k = rows(rng, (1, 3, 8, 64)), rows(rng, (1, 1, 8, 64))
    q[0, 1, 3, 5], q[0, 2, 6, 40] = math.nan, math.inf
    pos, axes = places(rng, (2, 1, 8), 1000), pair_axes((8, 8))
    got, _ = rotate_axes(q, k, pos, axes)
    bad = ~torch.isfinite(got)
    assert bad[0, 1, 3, 5] and bad[0, 1, 3, 21] and bad[0, 2, 6, 40]
    assert int(bad.sum()) == 3  # (the pair of dims 5 and 21; dim 40 is not rotated)
    got, _ = rotate_axes(q, k, pos, axes, q_norm=torch.ones_like(q[0, 0, 0]))
    rest = torch.isfinite(got).all(-1)
    assert not rest[0, 1, 3] and not rest[0, 2, 6] and int((~rest).sum()) == 2


def test_no_tokens_streams_and_graphs(cuda):
    rng = np.random.default_rng(5)
    axes = pair_axes((16, 16))
    e = torch.empty((2, 4, 0, 64), dtype=torch.bfloat16, device="cuda")
    p = torch.empty((2, 2, 0), dtype=torch.int32, device="cuda")
    q2, k2 = rotate_axes(e, e[:, :1], p, axes)
    assert q2.shape == e.shape and k2.shape == (2, 1, 0, 64)
    q, k = rows(rng, (2, 4, 65, 64)), rows(rng, (2, 1, 65, 64))
    pos = places(rng, (2, 2, 65), 3000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q2, _ = rotate_axes(q, k, pos, axes, stream=side)
    side.synchronize()
    check(q2, q, pos, axes)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q2, k2 = rotate_axes(q, k, pos, axes)
    pos.copy_(places(rng, (2, 2, 65), 3000))
    q.copy_(rows(rng, q.shape))
    g.replay()
    torch.cuda.synchronize()
    check(q2, q, pos, axes)
    check(k2, k, pos, axes)
    del g


def test_python_refusals(cuda):
    rng = np.random.default_rng(6)
    q, k = rows(rng, (1, 2, 3, 64)), rows(rng, (1, 1, 3, 64))
    pos, axes = places(rng, (2, 1, 3), 10), pair_axes((8, 8))
    ok = dict(q=q, k=k, positions=pos, axes=axes)
    for bad in (dict(q=q.float()), dict(k=k.half()), dict(k=k[:, :, :2]), dict(q=q[0]),
                dict(k=k.cpu()), dict(positions=pos.long()), dict(positions=pos[:1]),
                dict(positions=pos[:, :, :2]), dict(positions=pos.cpu()),
                dict(axes=pair_axes((8, 8, 1))), dict(axes=()), dict(axes=(0,) * 40),
                dict(axes=(-1,) * 8), dict(base=1.0), dict(base=math.nan),
                dict(q_norm=q[0, 0, 0, :32]), dict(k_norm=q[0, 0, 0].float()),
                dict(q_out=k), dict(k_out=k.transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises((ValueError, RuntimeError)):
            rotate_axes(**{**ok, **bad})
