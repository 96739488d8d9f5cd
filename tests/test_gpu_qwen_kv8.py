"""The decode stack with the 8-bit paged cache on its full-attention layers:
the layer's attention against float64 over the cache's rule, prompt scoring
against float64 over the forward's logits, and generation."""
import numpy as np
import pytest

from test_gpu_kv8 import Plain, attend_plain, same_cache

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(cuda):
    from vates_b200.qwen_next import QwenNextModel, tiny_config
    return QwenNextModel(tiny_config(), seed=4, cache_len=512, verify_len=4, drafts=3, kv="kv8")


def test_unknown_cache_is_refused():
    from vates_b200.qwen_next import QwenNextModel, tiny_config
    with pytest.raises(ValueError, match="isoquant"):
        QwenNextModel(tiny_config(), kv="kv9")


@gpu
def test_layer_attention_over_pages(model):
    """Chunks of 1 to 8 rows across the end of a page: cache contents exactly the
    rule's, attention within the operator's bound, its gate the separate one's."""
    import torch
    from vates_b200._lib import check, lib
    from vates_b200.pool import stream_handle
    from vates_b200.qwen_next import AttnLayer, SP_POS
    model.reset()
    b, cfg = model.buf, model.cfg
    lay = next(l for l in model.layers if isinstance(l.mixer, AttnLayer))
    D, H, Hq = cfg.head_dim, cfg.kv_heads, cfg.q_heads
    ref = Plain(lay.mixer.cache)
    gen = torch.Generator(device="cuda").manual_seed(3)
    pos = 50
    for T in (4, 1, 8, 3, 8, 2):
        b["state"][SP_POS] = pos
        b["x0"][:T] = torch.randn((T, cfg.hidden), device="cuda", generator=gen).bfloat16()
        model._attn(lay.mixer, lay, b["x0"], b["h"], T, None,
                    b["state"].data_ptr() + 4 * SP_POS)
        f = lambda k, n: b[k].view(-1)[:n * T * D].view(1, n, T, D).float().cpu().numpy()
        ref.append(0, f("krow", H), [pos], [T])
        ref.append(1, f("vrow", H), [pos], [T])
        same_cache(lay.mixer.cache, ref)
        pos += T
        want, _, tol, _ = attend_plain(ref, f("q", Hq).astype(np.float64), [pos], [T], D ** -0.5,
                                       True)
        got = f("attn", Hq)
        assert (np.abs(got - want) <= tol).all()
        # the gate is vb_attn_gate's own, bit for bit
        sep = torch.empty_like(b["gout"])
        check(lib.vb_attn_gate(b["attn"].data_ptr(), b["proj"].data_ptr(), cfg.attn_proj, T, Hq,
                               sep.data_ptr(), stream_handle()), "vb_attn_gate")
        n = T * Hq * D
        assert torch.equal(sep.view(-1)[:n], b["gout"].view(-1)[:n])
    assert int(b["status"].item()) == 0


@gpu
@pytest.mark.parametrize("n,top", [(2, 0), (70, 3), (129, 5)])
def test_score_vs_float64(model, n, top):
    """Log-sum-exp of 2048 float32 terms, each within 2^-22, and a float32 result:
    5e-5 covers both up to |z| of 100."""
    import torch
    ids = np.random.default_rng(n).integers(0, model.cfg.vocab, n).astype(np.int32)
    got = model.score(ids, top=top)
    rows = []
    model._prompt(ids[:-1], False, lambda done, T: rows.append(model.buf["logits"][:T].clone()))
    eager = model.score(ids, top=top, use_graphs=False)
    for a, e in zip(got, eager):
        assert torch.equal(a, e)
    z = torch.cat(rows).double().cpu().numpy()
    assert z.shape == (n - 1, model.cfg.vocab) and np.abs(z).max() < 100
    lp = z - z.max(1, keepdims=True)
    lp -= np.log(np.exp(lp).sum(1, keepdims=True))
    t, r = ids[1:], np.arange(n - 1)
    assert np.abs(got.logprob.cpu().numpy() - lp[r, t]).max() <= 5e-5
    order = np.argsort(-z, axis=1, kind="stable")
    place = np.empty_like(order)
    place[r[:, None], order] = np.arange(z.shape[1])
    assert np.array_equal(got.rank.cpu().numpy(), place[r, t])
    assert np.array_equal(got.top_ids.cpu().numpy(), order[:, :top])
    assert int(model.buf["status"].item()) == 0


@gpu
def test_generate_graph_eager_and_again(model):
    """Pages keep nothing of an earlier prompt, and speculation that is taken
    back leaves the tokens as they are."""
    rng = np.random.default_rng(8)
    a, b = (rng.integers(0, model.cfg.vocab, n).astype(np.int32) for n in (37, 90))
    first, st = model.generate(a, 40)
    model.generate(b, 30)
    again, _ = model.generate(a, 40)
    eager, _ = model.generate(a, 40, use_graphs=False)
    assert len(first) == 40 and st["status"] == 0
    assert np.array_equal(first, again) and np.array_equal(first, eager)
