"""Error of attention over int8 pages beside the 4-bit keys and 3-bit values of the
other quantised cache, on the same rows."""
import math

import pytest
import torch

from vates_b200.kv8 import PagedKV8Cache
from vates_b200.quant_kv import (AsymmetricQuantizedKVCache, asym_quantized_sdpa, build_block_so4,
                                 rotate_last, so4_blocks)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,ratio", [("normal", 8), ("large tokens", 3)])
def test_output_error_beside_k4_v3(cuda, kind, ratio):
    """Normal rows: 64 rows of 256 reach some 4.1 sigma, so int8 errs by 4.1 / 127 /
    sqrt(12) = 0.0093 sigma; groups of 64 span some 4.8 sigma, 0.092 sigma at 4 bits and
    0.2 at 3: ten times as much and more. Values ten times as large in one token of two
    hundred raise the scale of about a quarter of the pages tenfold, 0.05 sigma on
    average, a quarter of what 3 bits err."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    D, H, Hq, n, L = 256, 2, 16, 4000, 4
    rand = lambda *s: torch.randn(s, device="cuda", generator=gen)
    k, v, q = rand(1, H, n, D), rand(1, H, n, D), 1.5 * rand(1, Hq, L, D)
    if kind == "large tokens":
        v[:, :, torch.randperm(n, device="cuda", generator=gen)[:n // 200]] *= 10
    k, v, q = k.bfloat16(), v.bfloat16(), q.bfloat16()
    z = q.double().view(1, H, Hq // H, L, D) @ k.double()[:, :, None].transpose(-1, -2)
    later = torch.arange(n, device="cuda") > torch.arange(n - L, n, device="cuda")[:, None]
    p = torch.softmax((z * D ** -0.5).masked_fill(later, -math.inf), -1)
    want = (p @ v.double()[:, :, None]).view(1, Hq, L, D)

    def error(o):
        return float((o.double() - want).square().mean().sqrt() / want.square().mean().sqrt())

    c = PagedKV8Cache.empty(-(-n // 64), H, D, 1, -(-n // 64), 64)
    c.page_table.copy_(torch.arange(c.pages, dtype=torch.int32)[None])
    c.append(k, v, torch.zeros(1, dtype=torch.int32, device="cuda"))
    eight = error(c.attend(q, torch.tensor([n], dtype=torch.int32, device="cuda")))
    rk, rv = (so4_blocks(build_block_so4(D, seed=s)) for s in (0, 1))
    keys, values = AsymmetricQuantizedKVCache().update_and_fetch(k, v, rk, rv)
    four = error(asym_quantized_sdpa(rotate_last(q, rk), keys, values, D ** -0.5, "causal", 64, 4,
                                     3, rv=rv))
    assert eight * ratio <= four, (eight, four)
