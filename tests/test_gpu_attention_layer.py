"""AttentionLayer against the layer in 64 bits, made from the checkpoint's tensors one by one (tests/attention_layer_ref.py)."""
from __future__ import annotations

import pytest
import torch

from tests import attention_layer_ref as lref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("heads,kv,d", [(6, 2, 64), (4, 4, 128), (5, 1, 64)])
@pytest.mark.parametrize("bias,sinks,window,scale", [(True, True, 5, None), (False, False, 0, None), (True, False, 0, 0.2), (False, True, 3, 0.05)])
def test_prompt_and_decode(heads, kv, d, bias, sinks, window, scale):
    from kcapw_klcquant_b200 import AttentionLayer, PagedKvCache

    hidden = 48
    t = lref.checkpoint(heads, kv, d, hidden, bias=bias, sinks=sinks, seed=heads)
    at = AttentionLayer.from_tensors(3, t, DEV, heads, kv, d, window=window)
    if scale is not None:
        at = AttentionLayer(at.qkv_weight, at.o_weight, heads, kv, d, at.qkv_bias, at.o_bias, at.sinks, window, scale)
    cos, sin = lref.tables(64, d)
    rope = (cos.to(DEV), sin.to(DEV))
    cache = PagedKvCache(layers=2, pages=8, page_size=16, kv_heads=kv, head_dim=d, rows=3, row_pages=2, device=DEV)
    seqs = {2: lref.tokens(8, hidden, 1), 0: lref.tokens(15, hidden, 2)}  # the second grows over a page's end
    steps = {r: lref.tokens(3, hidden, 3 + r) for r in seqs}
    want = {r: lref.layer(torch.cat([seqs[r], steps[r]]), t, cos, sin, heads, kv, d, window, scale) for r in seqs}

    def close(got, r, rows):
        y, bound = (a[rows] for a in want[r])
        off = (got.double().cpu() - y).abs()
        assert (off <= bound).all(), f"row {r}: {float((off / bound).max()):.3g} x the bound"

    cache.reserve(i32([15, 0, 8]))
    x = torch.cat([seqs[2], seqs[0]]).to(DEV)
    pos = torch.cat([torch.arange(8), torch.arange(15)]).to(torch.int32).to(DEV)
    y = at.prompt(x, cache, 1, rope, i32([0, 8, 23]), pos, i32([2] * 8 + [0] * 15))
    close(y[:8], 2, slice(0, 8))
    close(y[8:], 0, slice(0, 15))
    for n in range(3):
        before = cache.lens.clone()
        cache.reserve(i32([1, 0, 1]))
        x = torch.zeros(3, hidden, dtype=torch.bfloat16)
        for r in seqs:
            x[r] = steps[r][n]
        y = at.decode(x.to(DEV), cache, 1, rope, before, i32([0, -1, 2]))
        for r, s in seqs.items():
            close(y[r:r + 1], r, slice(s.shape[0] + n, s.shape[0] + n + 1))
    cache.check()
    assert (cache.pool[0] == 0).all()  # the other layer's pages
