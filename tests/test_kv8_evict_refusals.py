"""Refusals of the C entries of accumulated attention weight and eviction (no GPU)."""
import ctypes as C

import pytest

from test_kv8_refusals import FAKE, _cache
from vates_b200 import _lib
from vates_b200._lib import lib


@pytest.mark.parametrize("bad", [dict(dim=96), dict(page=48), dict(kv_heads=0), dict(pages=0),
                                 dict(max_pages=0), dict(k_codes=None)], ids=lambda d: "-".join(d))
def test_cache_refusals(bad):
    c = _cache(**bad)
    a = _lib.VbKv8WeighArgs(cache=c, q=FAKE, lse=FAKE, lens=FAKE, weights=FAKE, scale=1.0,
                            q_heads=4, L=1, room=64)
    assert lib.vb_kv8_weigh(C.byref(a), None) == 1
    e = _lib.VbKv8EvictArgs(cache=c, weights=FAKE, lens=FAKE, lens_out=FAKE + 64, room=64, keep=8)
    assert lib.vb_kv8_evict(C.byref(e), None) == 1
    assert lib.vb_kv8_evict_workspace_size(C.byref(e)) == 0


@pytest.mark.parametrize("bad", [dict(q_heads=3), dict(q_heads=0), dict(q_heads=512), dict(L=-1),
                                 dict(scale=0.0), dict(scale=float("nan")), dict(q=None),
                                 dict(lens=None), dict(lse=None), dict(weights=None),
                                 dict(room=-1), dict(positions=FAKE)], ids=lambda d: "-".join(d))
def test_weigh_refusals(bad):
    d = dict(q=FAKE, lse=FAKE, lens=FAKE, weights=FAKE, scale=1.0, q_heads=4, L=1, room=64)
    d.update(bad)
    a = _lib.VbKv8WeighArgs(cache=_cache(), **d)
    assert lib.vb_kv8_weigh(C.byref(a), None) == 1
    assert b"vb_kv8_weigh" in lib.vb_last_error()


@pytest.mark.parametrize("bad", [dict(keep=0), dict(keep=-4), dict(first=-1), dict(recent=-1),
                                 dict(first=5, recent=4), dict(room=-1), dict(lens=None),
                                 dict(lens_out=None), dict(lens_out=FAKE), dict(weights=None)],
                         ids=lambda d: "-".join(d))
def test_evict_refusals(bad):
    d = dict(weights=FAKE, lens=FAKE, lens_out=FAKE + 64, room=64, keep=8, workspace=FAKE,
             workspace_bytes=1 << 30)
    d.update(bad)
    a = _lib.VbKv8EvictArgs(cache=_cache(), **d)
    assert lib.vb_kv8_evict(C.byref(a), None) == 1
    assert b"vb_kv8_evict" in lib.vb_last_error()


def test_evict_workspace():
    a = _lib.VbKv8EvictArgs(cache=_cache(max_pages=64, pages=64), weights=FAKE, lens=FAKE,
                            lens_out=FAKE + 64, room=1024, keep=100)
    need = lib.vb_kv8_evict_workspace_size(C.byref(a))
    assert need > 0
    a.workspace, a.workspace_bytes = FAKE, need - 1
    assert lib.vb_kv8_evict(C.byref(a), None) == 3
    a.workspace, a.workspace_bytes = FAKE + 4, need + 16
    assert lib.vb_kv8_evict(C.byref(a), None) == 1
    a.keep = 1 << 20  # nothing can be over it
    assert lib.vb_kv8_evict_workspace_size(C.byref(a)) == 0


def test_no_rows_are_accepted():
    a = _lib.VbKv8WeighArgs(cache=_cache(), lens=FAKE, scale=1.0, q_heads=4, L=0, room=0)
    assert lib.vb_kv8_weigh(C.byref(a), None) == 0


def test_weigh_tiles_are_counted_in_31_bits():
    d = dict(q=FAKE, lse=FAKE, lens=FAKE, weights=FAKE, scale=1.0, room=1 << 29, workspace=FAKE,
             workspace_bytes=1)
    for L, rc in ((256 * 1022, 3), (256 * 1023, 1), (256 * 65536, 1)):
        a = _lib.VbKv8WeighArgs(cache=_cache(max_pages=1 << 25, kv_heads=1), q_heads=1, L=L, **d)
        a.cache.page = 16
        assert lib.vb_kv8_weigh(C.byref(a), None) == rc
        assert (lib.vb_kv8_weigh_workspace_size(C.byref(a)) > 0) == (rc == 3)
