"""Argument checks of the paged 8-bit cache and the token log probabilities:
bad arguments are refused before anything is launched (no GPU needed)."""
import ctypes as C

import pytest
import torch

from vates_b200 import _lib
from vates_b200._lib import lib

FAKE = 1 << 20  # an aligned address that no accepted call reaches


def _cache(**kw):
    d = dict(k_codes=FAKE, v_codes=FAKE, k_scales=FAKE, v_scales=FAKE, page_table=FAKE, pages=4,
             kv_heads=2, page=64, dim=128, batch=1, max_pages=4)
    d.update(kw)
    return _lib.VbKv8Cache(**d)


BAD_CACHES = [dict(dim=96), dict(page=48), dict(pages=0), dict(kv_heads=0), dict(batch=0),
              dict(batch=70000), dict(max_pages=0), dict(k_codes=None), dict(v_scales=None),
              dict(page_table=None), dict(k_codes=FAKE + 8), dict(max_pages=1 << 26)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda d: "-".join(d))
def test_cache_refusals(bad):
    c = _cache(**bad)
    a = _lib.VbKv8AppendArgs(cache=c, keys=FAKE, values=FAKE, pos=FAKE, n=1)
    assert lib.vb_kv8_append(C.byref(a), None) == 1
    r = _lib.VbKv8ReadArgs(cache=c, lens=FAKE, keys=FAKE, values=FAKE, n=1)
    assert lib.vb_kv8_read(C.byref(r), None) == 1
    t = _lib.VbKv8AttnArgs(cache=c, q=FAKE, lens=FAKE, out=FAKE, scale=1.0, q_heads=4, L=1)
    assert lib.vb_kv8_attn(C.byref(t), None) == 1
    assert lib.vb_kv8_attn_workspace_size(C.byref(t)) == 0
    assert lib.vb_last_error()


@pytest.mark.parametrize("bad", [dict(q_heads=3), dict(q_heads=0), dict(q_heads=512), dict(L=-1),
                                 dict(scale=0.0), dict(scale=float("nan")), dict(q=None),
                                 dict(lens=None), dict(out=None), dict(out=FAKE + 8)],
                         ids=lambda d: "-".join(d))
def test_attention_refusals(bad):
    d = dict(q=FAKE, lens=FAKE, out=FAKE, scale=1.0, q_heads=4, L=1, workspace=FAKE,
             workspace_bytes=1 << 40)
    d.update(bad)
    a = _lib.VbKv8AttnArgs(cache=_cache(), **d)
    assert lib.vb_kv8_attn(C.byref(a), None) == 1
    assert b"vb_kv8_attn" in lib.vb_last_error()


def test_attention_workspace_too_small():
    a = _lib.VbKv8AttnArgs(cache=_cache(max_pages=64, pages=64), q=FAKE, lens=FAKE, out=FAKE,
                           scale=1.0, q_heads=4, L=1)
    need = lib.vb_kv8_attn_workspace_size(C.byref(a))
    assert need > 0
    a.workspace, a.workspace_bytes = FAKE, need - 1
    assert lib.vb_kv8_attn(C.byref(a), None) == 3
    assert b"workspace" in lib.vb_last_error()


def test_empty_calls_are_accepted():
    """Zero rows: nothing to do, nothing launched."""
    a = _lib.VbKv8AppendArgs(cache=_cache(), n=0)
    assert lib.vb_kv8_append(C.byref(a), None) == 0
    r = _lib.VbKv8ReadArgs(cache=_cache(), n=0)
    assert lib.vb_kv8_read(C.byref(r), None) == 0
    t = _lib.VbKv8AttnArgs(cache=_cache(), q_heads=4, L=0, scale=1.0)
    assert lib.vb_kv8_attn(C.byref(t), None) == 0
    p = _lib.VbTokenLogprobsArgs(rows=0, vocab=10, temperature=1.0)
    assert lib.vb_token_logprobs(C.byref(p), None) == 0


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(vocab=0), dict(top=33), dict(top=-1),
                                 dict(top=12, vocab=10, row_stride=10), dict(dtype=2),
                                 dict(temperature=0.0), dict(temperature=float("nan")),
                                 dict(temperature=-1.0), dict(logits=None), dict(tokens=None),
                                 dict(top_ids=None), dict(rank=None), dict(row_stride=99),
                                 dict(logits=FAKE + 1), dict(workspace=FAKE + 4)],
                         ids=lambda d: "-".join(d))
def test_logprob_refusals(bad):
    d = dict(logits=FAKE, tokens=FAKE, logprob=FAKE, entropy=FAKE, rank=FAKE, top_ids=FAKE,
             top_logprobs=FAKE, workspace=FAKE, workspace_bytes=1 << 30, row_stride=100,
             temperature=1.0, rows=2, vocab=100, top=5, dtype=0)
    d.update(bad)
    a = _lib.VbTokenLogprobsArgs(**d)
    assert lib.vb_token_logprobs(C.byref(a), None) == 1
    assert b"vb_token_logprobs" in lib.vb_last_error()


def test_logprob_workspace_too_small():
    need = lib.vb_token_logprobs_workspace_size(3, 100000, 5)
    a = _lib.VbTokenLogprobsArgs(logits=FAKE, tokens=FAKE, logprob=FAKE, entropy=FAKE, rank=FAKE,
                                 top_ids=FAKE, top_logprobs=FAKE, workspace=FAKE,
                                 workspace_bytes=need - 1, row_stride=100000, temperature=1.0,
                                 rows=3, vocab=100000, top=5, dtype=0)
    assert lib.vb_token_logprobs(C.byref(a), None) == 3


def test_python_refuses_host_tensors_and_shapes():
    from vates_b200.kv8 import PagedKV8Cache
    from vates_b200.logprobs import token_logprobs
    i8, f32 = torch.zeros((4, 2, 64, 128), dtype=torch.int8), torch.zeros((4, 2))
    table = torch.zeros((1, 4), dtype=torch.int32)
    with pytest.raises(ValueError):  # host tensors
        PagedKV8Cache(i8, i8, f32, f32, table)
    with pytest.raises(ValueError):  # page size
        PagedKV8Cache(i8[:, :, :40], i8[:, :, :40], f32, f32, table)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros((2, 10)), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(10), torch.zeros(1, dtype=torch.int32))
