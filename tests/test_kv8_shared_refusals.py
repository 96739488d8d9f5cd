"""Refusals of the C entry of attention over shared prefixes (no GPU)."""
import ctypes as C

import pytest

from test_kv8_refusals import FAKE, _cache
from vates_b200 import _lib
from vates_b200._lib import lib


def _args(groups=((0, 2, 64),), cache=None, attn=None, **kw):
    host = (C.c_int32 * (3 * len(groups)))(*[x for g in groups for x in g])
    t = dict(q=FAKE, lens=FAKE, out=FAKE, scale=1.0, q_heads=4, L=1, workspace=FAKE,
             workspace_bytes=1 << 40)
    t.update(attn or {})
    d = dict(segments=FAKE, group_of=FAKE, host_groups=C.addressof(host), groups=len(groups))
    d.update(kw)
    a = _lib.VbKv8SharedArgs(attn=_lib.VbKv8AttnArgs(cache=_cache(**{"batch": 3, **(cache or {})}), **t),
                             **d)
    a._keep = host
    return a


@pytest.mark.parametrize("groups", [((0, 4, 64),), ((0, 0, 64),), ((-1, 2, 64),), ((0, 2, 0),),
                                    ((0, 2, 65),), ((0, 2, 320),), ((1, 2, 64), (0, 1, 64)),
                                    ((0, 2, 64), (1, 2, 64)), ()])
def test_groups(groups):
    assert lib.vb_kv8_attn_shared(C.byref(_args(groups)), None) == 1
    assert b"vb_kv8_attn_shared" in lib.vb_last_error()
    assert lib.vb_kv8_attn_shared_workspace_size(C.byref(_args(groups))) == 0


@pytest.mark.parametrize("bad", [dict(attn=dict(q=None)), dict(attn=dict(lens=None)),
                                 dict(attn=dict(out=FAKE + 8)), dict(attn=dict(scale=0.0)),
                                 dict(attn=dict(q_heads=3)), dict(attn=dict(L=-1)),
                                 dict(attn=dict(workspace=FAKE + 8)), dict(segments=None),
                                 dict(segments=FAKE + 4), dict(group_of=None),
                                 dict(host_groups=None), dict(cache=dict(dim=96)),
                                 dict(cache=dict(batch=65535, kv_heads=256), attn=dict(q_heads=256))], ids=str)
def test_refusals(bad):
    assert lib.vb_kv8_attn_shared(C.byref(_args(**bad)), None) == 1
    assert lib.vb_last_error()


def test_workspace_and_no_rows():
    a = _args(least=0)
    need = lib.vb_kv8_attn_shared_workspace_size(C.byref(a))
    assert need > _lib.VB_KV8_ATTN_WORKSPACE_HEAD
    a.attn.workspace_bytes = need - 1
    assert lib.vb_kv8_attn_shared(C.byref(a), None) == 3
    a.attn.workspace = None
    assert lib.vb_kv8_attn_shared(C.byref(a), None) == 3
    a.attn.L = 0
    assert lib.vb_kv8_attn_shared(C.byref(a), None) == 0


def test_workspace_of_the_prefill_kernel():
    """It stores 32 bytes at a time."""
    for off in (16, 48):
        a = _args(attn=dict(q_heads=80, workspace=FAKE + off), least=0)
        assert lib.vb_kv8_attn_shared(C.byref(a), None) == 1
        assert b"alignment" in lib.vb_last_error()
        a = _args(attn=dict(q_heads=80, workspace=FAKE + off), cache=dict(max_pages=4096)).attn
        assert lib.vb_kv8_attn_workspace_size(C.byref(a)) > 0
        assert lib.vb_kv8_attn(C.byref(a), None) == 1
        assert b"alignment" in lib.vb_last_error()
