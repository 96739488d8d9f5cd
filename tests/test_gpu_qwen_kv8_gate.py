"""The decode stack's attention over the 8-bit cache: its output gate against the exact
sigmoid, and the scratch that it uses."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_layer_gate_vs_float64(cuda):
    """Row t of the gated output is [q_heads, head_dim] of attention times the sigmoid of
    the gate half of the head's query projection. The sigmoid is rounded to bf16, so it is
    one of the two bf16 values beside the exact one (float32's own error, 2^-23, is far
    below their distance), and the product with either is rounded once: no other value
    can come out."""
    import torch
    from vates_b200.qwen_next import AttnLayer, QwenNextModel, SP_POS, tiny_config
    model = QwenNextModel(tiny_config(), seed=4, cache_len=256, verify_len=4, drafts=3, kv="kv8")
    b, cfg = model.buf, model.cfg
    lay = next(l for l in model.layers if isinstance(l.mixer, AttnLayer))
    D, Hq = cfg.head_dim, cfg.q_heads
    gen = torch.Generator(device="cuda").manual_seed(9)
    pos = 0
    for T in (3, 8, 1):
        b["state"][SP_POS] = pos
        b["x0"][:T] = 4 * torch.randn((T, cfg.hidden), device="cuda", generator=gen).bfloat16()
        model._attn(lay.mixer, lay, b["x0"], b["h"], T, None,
                    b["state"].data_ptr() + 4 * SP_POS)
        pos += T
        n = T * Hq * D
        o = b["attn"].view(-1)[:n].view(Hq, T, D).float().cpu().transpose(0, 1)
        proj = b["proj"].view(-1)[:T * cfg.attn_proj].view(T, cfg.attn_proj)
        gate = proj[:, :Hq * 2 * D].view(T, Hq, 2, D)[:, :, 1].double().cpu().numpy()
        s = 1 / (1 + np.exp(-gate))
        assert s.min() > 2.0 ** -12
        # bf16 values beside s: the float32 bits cut off, and the next one up
        down = s.astype(np.float32).view(np.uint32) & np.uint32(0xFFFF0000)
        got = b["gout"].view(-1)[:n].view(T, Hq, D).cpu()
        hit = torch.zeros(got.shape, dtype=torch.bool)
        for near in (down, down + np.uint32(0x10000)):
            f = torch.from_numpy(near.view(np.float32).copy())
            hit |= got == (o * f).bfloat16()
        assert hit.all()
        assert np.abs(gate).max() > 1 and s.std() > 0.1


def test_one_workspace_for_all_layers_and_graphs(cuda, monkeypatch):
    """The model's attention takes its scratch from the model, in every graph, and
    leaves the ticket words zero."""
    import torch
    from vates_b200 import _lib, kv8
    from vates_b200.qwen_next import QwenNextModel, tiny_config
    model = QwenNextModel(tiny_config(), seed=4, cache_len=4096, verify_len=4, drafts=3, kv="kv8")
    ids = np.random.default_rng(1).integers(0, model.cfg.vocab, 203).astype(np.int32)
    want, _ = model.generate(ids, 12, use_graphs=False)

    class Closed:
        def get(self, *a):
            raise AssertionError("scratch of the module")

    monkeypatch.setattr(kv8, "_scratch", Closed())
    got, stats = model.generate(ids, 12)
    assert np.array_equal(got, want) and stats["status"] == 0
    torch.cuda.synchronize()
    assert not model.kv8_ws[:_lib.VB_KV8_ATTN_WORKSPACE_HEAD].any()
