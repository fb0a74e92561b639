"""Host checks of the attention and cache entry points, and the plain forms of the benchmark cases: no GPU."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from kcapw_klcquant_b200 import _lib
from tests import attention_ref as ref

A = 1024  # an aligned address nothing reads


def dims(**kw):
    d = dict(dtype=_lib.KLC_BF16, heads=8, kv_heads=2, head_dim=64, window=0, scale=0.125)
    d.update(kw)
    return _lib.KlcAttnDims(*d.values())


def prompt(d=None, **kw):
    a = dict(q=A, n=4, qt=512, qh=64, k=A, kt=128, kh=64, v=A, vt=128, vh=64, m=4, cu_q=A, cu_k=A, batch=1, sinks=None, out=A, ot=512, oh=64,
             lse=None, status=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().klc_attn_prompt(ctypes.byref(d or dims()), *a.values())


def decode(d=None, **kw):
    a = dict(q=A, qt=512, qh=64, k=A, v=A, pages=4, ps=16, stride=2 * 16 * 64, table=A, width=4, tstride=4, lens=A, batch=2, gs=None, pl=None,
             groups=0, sinks=None, out=A, ot=512, oh=64, lse=None, ws=A, bytes=1 << 30, status=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().klc_attn_decode(ctypes.byref(d or dims()), *a.values())


def rope(d=None, **kw):
    a = dict(q=A, qt=512, qh=64, k=A, kt=128, kh=64, v=A, vt=128, vh=64, cos=A, sin=A, max_pos=8, pos=A, rows=A, n=3, qo=A, qot=512, qoh=64,
             ko=None, kot=0, koh=0, kp=A, vp=A, pages=4, ps=16, stride=2 * 16 * 64, table=A, trows=2, width=4, tstride=4, status=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().klc_rope_append(ctypes.byref(d or dims()), *a.values())


BAD_DIMS = [(dict(dtype=_lib.KLC_F32), _lib.KLC_ERR_INVALID), (dict(heads=7), _lib.KLC_ERR_INVALID), (dict(kv_heads=0), _lib.KLC_ERR_INVALID),
            (dict(heads=0), _lib.KLC_ERR_INVALID), (dict(head_dim=96), _lib.KLC_ERR_UNSUPPORTED), (dict(heads=130), _lib.KLC_ERR_UNSUPPORTED)]


@pytest.mark.parametrize("call", [prompt, decode, rope])
@pytest.mark.parametrize("bad,status", BAD_DIMS)
def test_bad_dims(call, bad, status):
    assert call(dims(**bad)) == status


@pytest.mark.parametrize("call", [prompt, decode])
@pytest.mark.parametrize("bad", [dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(window=-1)])
def test_bad_scale_or_window(call, bad):
    assert call(dims(**bad)) == _lib.KLC_ERR_INVALID


@pytest.mark.parametrize("bad", [dict(n=-1), dict(batch=-1), dict(n=1 << 30), dict(cu_q=None), dict(cu_k=None), dict(q=None), dict(q=A + 8),
                                 dict(out=None), dict(out=A + 2), dict(k=None), dict(qt=509), dict(qh=60), dict(qh=32), dict(kt=64 - 8),
                                 dict(vh=12), dict(ot=8)])
def test_prompt_refusals(bad):
    assert prompt(**bad) == _lib.KLC_ERR_INVALID


def test_empty_calls_do_nothing():
    assert prompt(n=0, q=None, out=None) == _lib.KLC_OK and prompt(batch=0, q=None) == _lib.KLC_OK
    assert decode(batch=0, q=None) == _lib.KLC_OK and rope(n=0, q=None) == _lib.KLC_OK


@pytest.mark.parametrize("bad,status", [(dict(ps=24), 1), (dict(ps=256), 1), (dict(pages=0), 1), (dict(width=-1), 1), (dict(tstride=3), 1),
                                        (dict(width=1 << 28, tstride=1 << 28), 1), (dict(batch=-1), 1), (dict(batch=4097), 2), (dict(groups=3), 1),
                                        (dict(groups=1), 1), (dict(k=None), 1), (dict(v=A + 8), 1), (dict(table=None), 1), (dict(lens=None), 1),
                                        (dict(stride=2 * 16 * 64 - 8), 1), (dict(stride=2 * 16 * 64 + 4), 1), (dict(q=A + 4), 1),
                                        (dict(ot=4), 1), (dict(ws=None), 1), (dict(bytes=64), _lib.KLC_ERR_WORKSPACE)])
def test_decode_refusals(bad, status):
    assert decode(**bad) == status


@pytest.mark.parametrize("bad", [dict(n=-1), dict(max_pos=-1), dict(ps=8), dict(pages=0), dict(trows=-1), dict(tstride=2), dict(cos=None), dict(sin=A + 4),
                                 dict(pos=None), dict(rows=None), dict(kp=None), dict(vp=A + 8), dict(stride=64), dict(q=None), dict(qo=None),
                                 dict(ko=A, kot=4, koh=64), dict(kt=66)])
def test_rope_refusals(bad):
    assert rope(**bad) == _lib.KLC_ERR_INVALID


def kv(**kw):
    c = dict(pool=A, planes=2, plane_stride=4 * 4096, page_bytes=4096, pages=4, refs=A, block_table=A, table_width=4, table_stride=4, lens=A, rows=2,
             page_size=16, status=None)
    assert set(kw) <= set(c)
    c.update(kw)
    return _lib.KlcKvCache(*c.values())


@pytest.mark.parametrize("bad", [dict(pages=0), dict(rows=-1), dict(page_size=48), dict(table_stride=3), dict(page_bytes=0), dict(page_bytes=4104),
                                 dict(plane_stride=4096), dict(refs=None), dict(refs=A + 4), dict(lens=None), dict(block_table=None), dict(pool=None),
                                 dict(pool=A + 8), dict(table_width=1 << 31, table_stride=1 << 31),
                                 dict(rows=1 << 20, table_width=1 << 12, table_stride=1 << 12)])
def test_cache_refusals(bad):
    L, c = _lib.lib(), kv(**bad)
    big = 1 << 20
    assert L.klc_kv_reserve(ctypes.byref(c), A, A, big, None) == _lib.KLC_ERR_INVALID
    assert L.klc_kv_fork(ctypes.byref(c), A, A, 1, 0, A, big, None) == _lib.KLC_ERR_INVALID
    assert L.klc_kv_free(ctypes.byref(c), A, 1, None) == _lib.KLC_ERR_INVALID
    assert L.klc_kv_compact(ctypes.byref(c), None, A, big, None) == _lib.KLC_ERR_INVALID


def test_cache_lists_and_workspace():
    L, c = _lib.lib(), kv()
    n = ctypes.c_size_t(0)
    assert L.klc_kv_workspace_size(ctypes.byref(c), ctypes.byref(n)) == _lib.KLC_OK and n.value > 0
    assert L.klc_kv_reserve(ctypes.byref(c), None, A, n.value, None) == _lib.KLC_ERR_INVALID
    assert L.klc_kv_reserve(ctypes.byref(c), A, A, n.value - 1, None) == _lib.KLC_ERR_WORKSPACE
    assert L.klc_kv_fork(ctypes.byref(c), A, A, 3, 0, A, n.value, None) == _lib.KLC_ERR_INVALID  # more than rows
    assert L.klc_kv_fork(ctypes.byref(c), None, A, 1, 0, A, n.value, None) == _lib.KLC_ERR_INVALID
    assert L.klc_kv_fork(ctypes.byref(c), None, None, 0, 0, None, 0, None) == _lib.KLC_OK
    assert L.klc_kv_free(ctypes.byref(c), None, 0, None) == _lib.KLC_OK
    assert L.klc_kv_compact(ctypes.byref(c), None, None, 0, None) == _lib.KLC_ERR_INVALID
    assert L.klc_kv_workspace_size(ctypes.byref(c), None) == _lib.KLC_ERR_INVALID


def test_cpu_tensors_are_refused():
    from kcapw_klcquant_b200 import PagedKvCache, attn_decode, attn_prompt, rope_append

    q = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16)
    for call in (lambda: attn_prompt(q, q, q, i), lambda: attn_decode(q, pool, pool, i[:, None], i),
                 lambda: rope_append(q, q, q, torch.zeros(4, 32), torch.zeros(4, 32), i, i, pool, pool, i[:, None]),
                 lambda: PagedKvCache(layers=1, pages=1, page_size=16, kv_heads=1, head_dim=64, rows=1, row_pages=1, device="cpu")):
        with pytest.raises(ValueError):
            call()


def test_reference_attention_against_scaled_rows():
    """The tests' reference itself: one key gives its value, equal scores the mean, a sink of the same score a share."""
    v = torch.randn(4, 1, 64)
    z = torch.zeros(4, 1, 64)
    out, lse, _ = ref.attention(z.half(), z.half(), v.half(), torch.arange(4), 1.0)
    for i in range(4):
        assert torch.allclose(out[i, 0], v.half().double()[:i + 1, 0].mean(0)) and math.isclose(float(lse[i, 0]), math.log(i + 1), abs_tol=1e-12)
    out, _, _ = ref.attention(z.half(), z.half(), v.half(), torch.arange(4), 1.0, window=1, sinks=torch.zeros(1))
    assert torch.allclose(out[:, 0], v.half().double()[:, 0] / 2)


@pytest.mark.parametrize("heads,kv,d", [(4, 2, 64), (3, 1, 128)])
@pytest.mark.parametrize("n,m,window,sink", [(1, 1, 0, False), (70, 70, 0, True), (9, 200, 30, True), (40, 41, 1, False)])
def test_plain_forms_of_the_cases(heads, kv, d, n, m, window, sink):
    """Plain and 64-bit form of the benchmark's attention against the tests' own reference (no case has fewer keys than queries, and
    the plain form divides by nothing there); its rotation against complex products."""
    from perf import operators as ops

    g = torch.Generator().manual_seed(n + m)
    q, k, v = torch.randn(n, heads, d, generator=g), torch.randn(m, kv, d, generator=g), torch.randn(m, kv, d, generator=g)
    sinks = torch.randn(heads, generator=g) if sink else None
    pos = torch.arange(n) + m - n
    want, _, _ = ref.attention(q.half(), k.half(), v.half(), pos, 0.3, window, sinks)
    q, k, v = q.half().float(), k.half().float(), v.half().float()
    # fp32: sums of d products and of m weights; the definition in 64 bits: to its own rounding
    assert (ops._plain_attention(q, k, v, m - n, 0.3, window, sinks) - want).abs().max() <= 2e-4
    assert (ops._exact_attention(q, k, v, m - n, 0.3, window, sinks) - want).abs().max() <= 1e-10
    assert ops._visible(m - n, m - 1, window) == sum(min(p + 1, window) if window else p + 1 for p in range(m - n, m))
    ang = torch.rand(n, d // 2, generator=g)
    turned = torch.view_as_real(torch.complex(*q.chunk(2, -1)) * torch.polar(torch.ones_like(ang), ang)[:, None])
    assert torch.allclose(ops._rotate(q, ang.cos()[:, None], ang.sin()[:, None]), torch.cat([turned[..., 0], turned[..., 1]], -1), atol=1e-5)
