"""AttentionLayer's weights from checkpoint names, and the reference that its GPU tests use: no GPU."""
from __future__ import annotations

import pytest
import torch

from tests import attention_layer_ref as lref
from kcapw_klcquant_b200 import AttentionLayer

H, KV, D, W = 6, 2, 64, 48


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("sinks", [False, True])
def test_from_tensors_projects_by_name(bias, sinks):
    t = lref.checkpoint(H, KV, D, W, bias=bias, sinks=sinks)
    at = AttentionLayer.from_tensors(3, t, "cpu", H, KV, D, window=7)
    assert (at.heads, at.kv_heads, at.head_dim, at.window, at.scale) == (H, KV, D, 7, None)
    x = lref.tokens(9, W, 1)
    for name, got in zip("qkv", at.project(x)):
        want, bound = lref.linear(x.double(), torch.zeros(9, W, dtype=torch.float64), t, name)
        assert got.shape == (9, H if name == "q" else KV, D)
        assert ((got.double().reshape(9, -1) - want).abs() <= bound).all(), name
    o = torch.randn(9, H, D, generator=torch.Generator().manual_seed(2)).bfloat16()
    want, bound = lref.linear(o.double().reshape(9, -1), torch.zeros(9, H * D, dtype=torch.float64), t, "o")
    assert ((at.output(o).double() - want).abs() <= bound).all()
    assert at.sinks is None if not sinks else torch.equal(at.sinks, t[f"{lref.PREFIX}.sinks"].float())


@pytest.mark.parametrize("gone", ["q", "k", "v"])
def test_from_tensors_refuses_some_biases_and_missing_weights(gone):
    t = lref.checkpoint(H, KV, D, W, bias=True, sinks=False)
    some = {k: v for k, v in t.items() if k != f"{lref.PREFIX}.{gone}_proj.bias"}
    with pytest.raises(ValueError):
        AttentionLayer.from_tensors(3, some, "cpu", H, KV, D)
    with pytest.raises(KeyError):
        AttentionLayer.from_tensors(3, {k: v for k, v in t.items() if k != f"{lref.PREFIX}.{gone}_proj.weight"}, "cpu", H, KV, D)
    with pytest.raises(KeyError):
        AttentionLayer.from_tensors(2, t, "cpu", H, KV, D)
    with pytest.raises(ValueError):
        AttentionLayer.from_tensors(3, t, "cpu", H + 2, KV, D)
    no_o = {k: v for k, v in t.items() if k != f"{lref.PREFIX}.o_proj.bias"}
    assert AttentionLayer.from_tensors(3, no_o, "cpu", H, KV, D).o_bias is None


def test_the_layer_reference_tells_mistakes_apart():
    """Each of these would have to fail the GPU tests: they differ from the reference by more than its bound."""
    t = lref.checkpoint(H, KV, D, W, bias=True, sinks=True)
    cos, sin = lref.tables(64, D)
    x = lref.tokens(8, W, 3)
    want, bound = lref.layer(x, t, cos, sin, H, KV, D, window=5)

    def off(t=t, cos=cos, sin=sin, **kw):
        got, _ = lref.layer(x, t, cos, sin, H, KV, D, **dict(dict(window=5), **kw))
        return ((got - want).abs() > bound).any()

    name = lambda n, what: f"{lref.PREFIX}.{n}_proj.{what}"  # noqa: E731
    assert not off()
    for n in "qkvo":
        assert off({**t, name(n, "bias"): torch.zeros_like(t[name(n, "bias")])}), n
        assert off({**t, name(n, "bias"): 2 * t[name(n, "bias")]}), n
    for what in ("weight", "bias"):
        assert off({**t, name("k", what): t[name("v", what)], name("v", what): t[name("k", what)]}), what
    heads = t[name("q", "weight")].view(H, D, W).flip(0).reshape(H * D, W)
    assert off({**t, name("q", "weight"): heads})
    assert off({k: v for k, v in t.items() if not k.endswith("sinks")}) and off({**t, f"{lref.PREFIX}.sinks": t[f"{lref.PREFIX}.sinks"].flip(0)})
    assert off(window=0) and off(window=4) and off(window=6) and off(scale=0.15) and off(sin=-sin) and off(cos=cos[::2], sin=sin[::2])
    inter = torch.arange(D).view(2, D // 2).T.reshape(-1)  # pairs next to each other instead of halves
    mixed = {n: t[name(n, "weight")].view(-1, D, W)[:, inter].reshape(-1, W) for n in "qk"}
    assert off({**t, name("q", "weight"): mixed["q"], name("k", "weight"): mixed["k"]})
