"""Attention where the inputs are not finite, the numerators small, the pages gone or the calls unusual: against the definition."""
from __future__ import annotations

import pytest
import torch

from tests import attention_ref as ref
from tests.test_gpu_attention import BF, DEV, HF, check_decode, decode_case, rnd

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---- scores that are not finite --------------------------------------------------------


@pytest.mark.parametrize("dtype,heads,kv,d", [(BF, 64, 8, 64), (HF, 6, 2, 128), (BF, 20, 1, 64)])
@pytest.mark.parametrize("lens", [[777], [1], [40, 3000, 0, 130, 64], [90] * 200])
@pytest.mark.parametrize("sink", [False, True])
def test_decode_nan_query_is_a_nan_row(dtype, heads, kv, d, lens, sink):
    """Whether the row's keys are cut over many thread blocks or not; its neighbours keep their bits."""
    from kcapw_klcquant_b200 import attn_decode

    q, ks, vs, sinks = decode_case(dtype, heads, kv, d, lens, 32, 0, sink)
    kp, vp, table = ref.paged(ks, vs, 32)
    ln = i32(lens)
    clean, clean_lse = attn_decode(q, kp, vp, table, ln, sinks=sinks, return_lse=True)
    hit = torch.zeros(len(lens), heads, dtype=torch.bool, device=DEV)
    hit[0, 0] = hit[-1, heads - 1] = hit[len(lens) // 2, heads // 2] = True
    q[..., d - 1][hit] = float("nan")
    out, lse = attn_decode(q, kp, vp, table, ln, sinks=sinks, return_lse=True)
    hit &= (ln > 0)[:, None]  # a row without keys has no score to be a NaN
    assert out[hit].isnan().all() and lse[hit].isnan().all()
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])


@pytest.mark.parametrize("dtype,d", [(BF, 64), (HF, 128)])
@pytest.mark.parametrize("keys", [(0, 1), (0, 64), (100, 116), (512, 1024), (0, 3000), (2999, 3000)])
@pytest.mark.parametrize("window", [0, 200])
@pytest.mark.parametrize("prefix", [0, 1024])
def test_decode_nan_keys_make_the_rows_that_see_them_nan(dtype, d, keys, window, prefix):
    """One key, a warp's, a tile's, a whole share of them: output and log-sum-exp."""
    from kcapw_klcquant_b200 import attn_decode

    n = 3000
    q, ks, vs, _ = decode_case(dtype, 8, 2, d, [n, n], 64, 0, False)
    ks[1][:prefix], vs[1][:prefix] = ks[0][:prefix], vs[0][:prefix]
    kw = dict(window=window, return_lse=True)
    if prefix:
        kw.update(group_starts=i32([0, 2]), prefix_lens=i32([prefix]))
    ln = i32([n, n])
    clean, clean_lse = attn_decode(q, *ref.paged(ks, vs, 64), ln, **kw)
    for k in ks:
        k[keys[0]:keys[1], 1] = float("nan")
    out, lse = attn_decode(q, *ref.paged(ks, vs, 64), ln, **kw)
    assert torch.equal(out[:, :4], clean[:, :4]) and torch.equal(lse[:, :4], clean_lse[:, :4])
    if window == 0 or keys[1] > n - window:
        assert out[:, 4:].isnan().all() and lse[:, 4:].isnan().all()
    else:
        assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


# ---- small numerators ------------------------------------------------------------------


@pytest.mark.parametrize("dtype,d", [(HF, 64), (HF, 128), (BF, 64)])
@pytest.mark.parametrize("path,n", [("prompt", 5000), ("decode", 131000), ("prefix", 16384 + 70)])
@pytest.mark.parametrize("gap", [16.0, 18.0, 21.0])
def test_many_small_weights_behind_one_large(dtype, d, path, n, gap):
    """A first key whose value is 0 takes almost all of the softmax: what is left comes from the small weights alone.

    f16 numerators go up to 2^15 and the reference is at most 2^4 under the row's maximum, so that what a numerator loses
    below the type's normal range is 2^-25 / 2^11 = 2^-36 of the largest weight (attention_ref allows 2^-25)."""
    from kcapw_klcquant_b200 import attn_decode, attn_prompt

    q = torch.ones((1, 2, d), dtype=dtype, device=DEV)
    k, v = rnd((n, 1, d), dtype, 1, 0.02), 1 + rnd((n, 1, d), dtype, 2, 0.25)
    k[0], v[0] = gap / d, 0  # the scores of the others: 0, and 0.02 d^0.5 around it
    if path == "prompt":
        out = attn_prompt(q, k, v, i32([0, 1]), cu_seqlens_k=i32([0, n]), scale=1.0)
    elif path == "decode":
        out = attn_decode(q, *ref.paged([k], [v], 64), i32([n]), scale=1.0)
    else:
        out = attn_decode(q, *ref.paged([k], [v], 64), i32([n]), scale=1.0, group_starts=i32([0, 1]), prefix_lens=i32([16384]))
    want, _, bound = ref.attention(q, k, v, torch.tensor([n - 1], device=DEV), 1.0)
    if dtype == HF:
        bound = bound + (2.0 ** -36 - 2.0 ** -25) * n * v.double().abs().amax()
    assert (want > 4 * bound).all()  # the bound would not pass zeros
    ref.assert_close(out, want, bound, path)


# ---- infinite scores -------------------------------------------------------------------


def attend(path, q1, k, v, sinks, window=0):
    """The last token's attention: as the last of a prompt's rows, over the cache, or over the cache with a shared prefix."""
    from kcapw_klcquant_b200 import attn_decode, attn_prompt

    n, kw = k.shape[0], dict(sinks=sinks, window=window, return_lse=True)
    if path == "prompt":
        q = torch.cat([rnd((39, *q1.shape[1:]), q1.dtype, 3), q1])
        out, lse = attn_prompt(q, k, v, i32([0, 40]), cu_seqlens_k=i32([0, n]), **kw)
        return out[39:], lse[39:]
    if path == "prefix":
        kw.update(group_starts=i32([0, 1]), prefix_lens=i32([n // 2 // 64 * 64]))
    return attn_decode(q1, *ref.paged([k], [v], 64), i32([n]), **kw)


@pytest.mark.parametrize("dtype,d", [(BF, 64), (BF, 128), (HF, 64), (HF, 128)])
@pytest.mark.parametrize("path", ["prompt", "decode", "prefix"])
@pytest.mark.parametrize("sink", [False, True])
def test_infinite_scores(dtype, d, path, sink):
    n = 1200
    q, k, v = rnd((1, 4, d), dtype, 1).abs() + 0.5, rnd((n, 2, d), dtype, 4), rnd((n, 2, d), dtype, 5)
    sinks = torch.randn(4, device=DEV) if sink else None
    clean, clean_lse = attend(path, q, k, v, sinks)
    for j in (0, 130, 131, 390, 648, n - 1):  # +inf: not a number, in the heads that read it
        bad = k.clone()
        bad[j, 1, 5] = float("inf")
        out, lse = attend(path, q, bad, v, sinks)
        assert out[:, 2:].isnan().all() and lse[:, 2:].isnan().all(), j
        assert torch.equal(out[:, :2], clean[:, :2]) and torch.equal(lse[:, :2], clean_lse[:, :2])
    gone = [0, 130, 131, 390, 648, 649, n - 1]  # -inf: as if the key were not there
    bad = k.clone()
    bad[gone, 1, 5] = -float("inf")
    out, lse = attend(path, q, bad, v, sinks)
    left = torch.ones(n, dtype=torch.bool, device=DEV)
    left[gone] = False
    want, wl, bound = ref.attention(q[:, 2:], k[left, 1:], v[left, 1:], torch.tensor([n], device=DEV), d ** -0.5, 0, sinks[2:] if sink else None)
    ref.assert_close(out[:, 2:], want, bound, "-inf")
    ref.assert_lse(lse[:, 2:], wl, "-inf")
    bad[:, 1, 5] = -float("inf")  # nothing else: as a row that sees no key
    for window in (0, 100):
        out, lse = attend(path, q, bad, v, sinks, window)
        assert (out[:, 2:] == 0).all()
        assert torch.allclose(lse[:, 2:], sinks[2:] if sink else torch.full_like(lse[:, 2:], -float("inf")), rtol=1e-6, atol=1e-6)


# ---- whole layers ----------------------------------------------------------------------


def test_prompt_into_a_row_with_keys_is_reported_and_writes_nothing():
    """After a fork such a row shares its pages: parent and siblings keep their keys, the other prompts of the call are served."""
    from kcapw_klcquant_b200 import KlcError
    from tests.test_gpu_kv_cache import make_stack

    stack, alone = make_stack(5, 40, layers=2), make_stack(5, 40, layers=2)
    cache = stack.cache
    x = rnd((50, 256), BF, 1)
    stack.prompt(x[:40], i32([0, 40]), i32([1]))
    cache.fork(i32([1]), i32([2]))
    cache.check()

    def state():
        live = cache.refs > 0
        return cache.lens.tolist(), cache.block_table[:3].tolist(), cache.pool[:, :, live].clone()

    for rows in ([1], [2]):
        before = state()
        stack.prompt(x[:20], i32([0, 20]), i32(rows))
        with pytest.raises(KlcError):
            cache.check()
        after = state()
        assert after[:2] == before[:2] and torch.equal(after[2], before[2])
    before = state()
    out = stack.prompt(x, i32([0, 10, 30, 50]), i32([2, 3, 1]))  # the one in the middle goes to an empty row
    with pytest.raises(KlcError):
        cache.check()
    want = alone.prompt(x[10:30], i32([0, 20]), i32([3]))
    assert torch.equal(out[10:30], want)
    assert cache.lens.tolist() == [0, 40, 40, 20, 0] and cache.block_table[:3].tolist() == before[1]
    for r in (1, 2):
        held = cache.block_table[r, :3].long()
        assert torch.equal(cache.pool[:, :, held], alone_pages(x[:40])), r
    # the same row twice
    stack.prompt(x[:30], i32([0, 20, 30]), i32([4, 4]))
    with pytest.raises(KlcError):
        cache.check()
    assert cache.lens.tolist() == [0, 40, 40, 20, 0]


def alone_pages(x):
    """The pages a prompt of these tokens fills in a stack of its own."""
    from tests.test_gpu_kv_cache import make_stack

    stack = make_stack(5, 40, layers=2)
    stack.prompt(x, i32([0, x.shape[0]]), i32([1]))
    return stack.cache.pool[:, :, stack.cache.block_table[1, :3].long()]


def test_prompt_reports_rows_that_do_not_exist():
    from kcapw_klcquant_b200 import KlcError
    from tests.test_gpu_kv_cache import make_stack

    stack = make_stack(2, 20, layers=1)
    x = rnd((7, 256), BF, 1)
    for rows in ([0, -1], [0, 2], [0, -2 ** 31]):
        stack.prompt(x, i32([0, 4, 7]), i32(rows))
        with pytest.raises(KlcError):
            stack.cache.check()
        assert stack.cache.lens.tolist() == [4, 0]
        stack.cache.free(i32([0]))


# ---- scratch ---------------------------------------------------------------------------


def test_decode_leaves_a_moe_fault_to_be_read():
    """A layer's fault word lies in its stream's MoE workspace: a decode call on the stream does not touch it."""
    from kcapw_klcquant_b200 import KlcError, MoeLayer, attn_decode
    from kcapw_klcquant_b200 import synthetic as syn

    dims = syn.LayerDims(experts=16, hidden=256, intermediate=256, top_k=4)
    layer = MoeLayer.from_tensors(0, syn.make_layer(dims, seed=3, device=DEV), DEV, top_k=4)
    q, ks, vs, _ = decode_case(BF, 8, 2, 64, [100, 300], 16, 0, False)
    kp, vp, table = ref.paged(ks, vs, 16)
    attn_decode(q, kp, vp, table, i32([100, 300]))  # scratch of the size it needs is there
    idx = i32([[0, 1, 2, 3], [4, 5, 6, 99]])  # no such expert: recorded by the permute, the pair is left out
    layer.experts_forward(rnd((2, 256), BF, 1), idx, torch.full((2, 4), 0.25, dtype=BF, device=DEV), path="simt")
    attn_decode(q, kp, vp, table, i32([100, 300]))
    with pytest.raises(KlcError):
        layer.check_device_status()


def test_decode_calls_of_several_threads_on_one_stream():
    """Each call's kernels follow each other in the stream: no thread's shares reach another's rows."""
    import threading

    from kcapw_klcquant_b200 import attn_decode

    lens = [3000, 17, 900, 4000, 1]  # the same for all threads: only the queries differ
    _, ks, vs, sinks = decode_case(BF, 16, 2, 64, lens, 64, 0, True)
    kp, vp, table = ref.paged(ks, vs, 64)
    ln = i32(lens)
    qs = [rnd((len(lens), 16, 64), BF, 40 + i) for i in range(4)]
    want = [attn_decode(q, kp, vp, table, ln, sinks=sinks) for q in qs]
    outs = [[] for _ in qs]
    start = threading.Barrier(len(qs))

    def work(i):
        start.wait()
        for _ in range(200):
            outs[i].append(attn_decode(qs[i], kp, vp, table, ln, sinks=sinks))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(qs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert [sum(not torch.equal(o, w) for o in got) for got, w in zip(outs, want)] == [0] * len(qs)


def test_cache_calls_of_several_threads_on_one_stream():
    """A fork is a plan and the moves it asks for: another thread's plan does not come between them."""
    import threading

    from kcapw_klcquant_b200 import PagedKvCache

    n = 4
    cache = PagedKvCache(layers=1, pages=64, page_size=16, kv_heads=1, head_dim=64, rows=2 * n, row_pages=4, device=DEV)
    cache.reserve(i32([20] * n + [0] * n))
    cache.check()
    for r in range(n):
        cache.pool[:, :, cache.block_table[r, :2].long()] = r + 1
    parents, children = [i32([r]) for r in range(n)], [i32([n + r]) for r in range(n)]
    wrong = torch.zeros(n, dtype=torch.int32, device=DEV)
    start = threading.Barrier(n)

    def work(r):
        start.wait()
        for _ in range(100):
            cache.fork(parents[r], children[r], copy=True)
            page = cache.block_table.index_select(0, children[r].long())[0, :2].long().clamp(min=0)
            wrong[r] += (cache.pool.index_select(2, page) != r + 1).any()
            cache.free(children[r])

    threads = [threading.Thread(target=work, args=(r,)) for r in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    cache.check()
    assert wrong.tolist() == [0] * n and cache.lens.tolist() == [20] * n + [0] * n


def test_stack_refuses_a_cache_that_does_not_fit_and_keeps_lengths_on_bad_inputs():
    from kcapw_klcquant_b200 import PagedKvCache
    from kcapw_klcquant_b200.stack import MoeStack
    from tests.test_gpu_kv_cache import make_stack

    stack = make_stack(2, 20, layers=1)  # 2 key heads of 64, bf16
    kw = dict(attention=stack.attention, input_norm_weights=stack.input_norm_weights, cache=stack.cache, rope=stack.rope)
    size = dict(layers=1, pages=4, page_size=16, kv_heads=2, head_dim=64, rows=2, row_pages=2, device=DEV)
    for bad in (dict(dtype=HF), dict(kv_heads=1), dict(head_dim=128)):
        with pytest.raises(ValueError):
            MoeStack(stack.layers, stack.norm_weights, **dict(kw, cache=PagedKvCache(**dict(size, **bad))))
    cos, sin = stack.rope
    for rope in ((cos[:, :16], sin[:, :16]), (cos, sin[:9]), (cos,), (cos[0], sin[0])):
        with pytest.raises(ValueError):
            MoeStack(stack.layers, stack.norm_weights, **dict(kw, rope=rope))
    with pytest.raises(ValueError):
        MoeStack(stack.layers, stack.norm_weights, **dict(kw, input_norm_weights=[torch.ones(128, dtype=BF, device=DEV)]))
    for x in (torch.zeros(2, 256, device=DEV), torch.zeros(2, 128, dtype=BF, device=DEV), torch.zeros(512, dtype=BF, device=DEV),
              torch.zeros(2, 256, dtype=BF)):
        with pytest.raises(ValueError):
            stack.step(x)
        with pytest.raises(ValueError):
            stack.prompt(x, i32([0, 2]), i32([0]))
        assert stack.cache.lens.tolist() == [0, 0] and int(stack.cache.refs.sum()) == 0


@pytest.mark.parametrize("bad", [dict(qkv_bias=5), dict(o_bias=5), dict(sinks=3), dict(window=-1), dict(scale=0.0), dict(scale=float("nan")),
                                 dict(heads=130, kv_heads=2), dict(heads=0), dict(heads=7), dict(head_dim=80)])
def test_attention_layer_refuses_what_its_calls_would(bad):
    from kcapw_klcquant_b200 import AttentionLayer

    a = dict(heads=8, kv_heads=2, head_dim=64, **{k: torch.zeros(v, device=DEV) if k in ("qkv_bias", "o_bias", "sinks") else v for k, v in bad.items()
                                                 if k not in ("heads", "kv_heads", "head_dim")})
    a.update({k: v for k, v in bad.items() if k in ("heads", "kv_heads", "head_dim")})
    w = torch.zeros((a["heads"] + 2 * a["kv_heads"]) * a["head_dim"], 32, device=DEV)
    with pytest.raises(ValueError):
        AttentionLayer(w, torch.zeros(32, a["heads"] * a["head_dim"], device=DEV), **a)


# ---- shared prefixes -------------------------------------------------------------------


@pytest.mark.parametrize("dtype,heads,kv,d", [(BF, 8, 1, 64), (HF, 6, 2, 128)])
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("window,lens", [(300, [1350, 1313, 1400]), (300, [1281, 1280]), (0, [700, 33, 1000]), (5, [640, 700]), (100, [1400, 1390]),
                                         (0, [0, 1]), (300, [1350, 200, 0, 1300]), (40, list(range(3, 1400, 137)) * 8)])
def test_prefix_pages_without_a_visible_key_are_not_looked_up(dtype, heads, kv, d, ps, window, lens):
    """Entries before every row's window, between the windows of rows of different lengths, and past the longest of rows that end
    inside the prefix, may be anything."""
    from kcapw_klcquant_b200 import attn_decode, check_device_status

    prefix, n = 1280, max(1281, *lens)
    k, v = rnd((n, kv, d), dtype, 1), rnd((n, kv, d), dtype, 2)
    q, sinks = rnd((len(lens), heads, d), dtype, 3), torch.randn(heads, device=DEV)
    kp, vp, table = ref.paged([k] * len(lens), [v] * len(lens), ps)
    for e in range(prefix // ps):
        if not any(m > e * ps and (m - window if window else 0) < (e + 1) * ps for m in lens):
            table[:, e] = -1 if e % 2 else 10 ** 6
    out, lse = attn_decode(q, kp, vp, table, i32(lens), window=window, sinks=sinks, group_starts=i32([0, len(lens)]), prefix_lens=i32([prefix]),
                           return_lse=True)
    check_device_status(DEV)
    check_decode(q, [k[:m] for m in lens], [v[:m] for m in lens], window, sinks, out, lse)


@pytest.mark.parametrize("dtype,d", [(BF, 64), (HF, 64), (BF, 128)])
@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("bad", [None, "v", "k"])
def test_prefix_rows_that_see_none_of_it(dtype, d, window, bad):
    """Idle rows and rows whose window lies behind the prefix, between rows that see it; values and keys that are not finite reach
    the rows that see them only, from whichever share of the prefix they are in."""
    from kcapw_klcquant_b200 import attn_decode, check_device_status

    prefix, lens = 3200, [3300, 0, 3201, 4200, 3600, 0, 3200]
    pk, pv = rnd((prefix, 2, d), dtype, 1), rnd((prefix, 2, d), dtype, 2)
    ks = [torch.cat([pk, rnd((1000, 2, d), dtype, 10 + i)])[:n] for i, n in enumerate(lens)]
    vs = [torch.cat([pv, rnd((1000, 2, d), dtype, 50 + i)])[:n] for i, n in enumerate(lens)]
    q = rnd((len(lens), 16, d), dtype, 3)
    kw = dict(window=window, group_starts=i32([0, len(lens)]), prefix_lens=i32([prefix]), return_lse=True)
    clean, clean_lse = attn_decode(q, *ref.paged(ks, vs, 64, fill=0.0), i32(lens), **kw)
    check_device_status(DEV)
    check_decode(q, ks, vs, window, None, clean, clean_lse)
    if bad is None:
        return
    key = 2850  # seen by 3300, 3201, 3200 (and by 4200 and 3600 without a window)
    for t in ks if bad == "k" else vs:
        t[key:key + 1, 1, 9] = float("nan")
    out, lse = attn_decode(q, *ref.paged(ks, vs, 64, fill=0.0), i32(lens), **kw)
    want, want_lse = clean.clone(), clean_lse.clone()
    for i, n in enumerate(lens):
        if n > key and (window == 0 or key >= n - window):
            if bad == "k":
                want[i, 8:], want_lse[i, 8:] = float("nan"), float("nan")
            else:
                want[i, 8:, 9] = float("nan")
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))
    assert torch.equal(lse.isnan(), want_lse.isnan()) and torch.equal(lse.nan_to_num(nan=0.0), want_lse.nan_to_num(nan=0.0))


# ---- pages -----------------------------------------------------------------------------


def test_requests_behind_one_that_runs_out_of_pages():
    """Refused with it if they need pages, served if they do not; a request that is bad by itself touches no other."""
    from kcapw_klcquant_b200 import KlcError, PagedKvCache

    cache = PagedKvCache(layers=1, pages=6, page_size=16, kv_heads=1, head_dim=64, rows=5, row_pages=12, device=DEV)
    cache.reserve(i32([0, 0, 0, 10, 0]))  # one page, six more keys fit
    cache.check()
    cache.reserve(i32([160, 16, 1, 3, 0]))
    with pytest.raises(KlcError):
        cache.check()
    assert cache.lens.tolist() == [0, 0, 0, 13, 0] and int(cache.refs.sum()) == 1
    cache.reserve(i32([-1, 16, 10 ** 6, 3, 1]))
    with pytest.raises(KlcError):
        cache.check()
    assert cache.lens.tolist() == [0, 16, 0, 16, 1] and int(cache.refs.sum()) == 3
    cache.fork(i32([3, 9, 4, 1, 4]), i32([0, 2, 7, 2, 2]))  # a row twice: the first listing counts, and it is a bad one
    with pytest.raises(KlcError):
        cache.check()
    assert cache.lens.tolist() == [16, 16, 0, 16, 1]


def test_free_leaves_a_row_with_a_length_past_its_table():
    from kcapw_klcquant_b200 import KlcError, PagedKvCache

    cache = PagedKvCache(layers=1, pages=6, page_size=16, kv_heads=1, head_dim=64, rows=3, row_pages=2, device=DEV)
    cache.reserve(i32([20, 3, 0]))
    cache.lens[0] = 33  # two pages of 16
    cache.free(i32([0, 1, 2]))
    with pytest.raises(KlcError):
        cache.check()
    assert cache.lens.tolist() == [33, 0, 0] and cache.refs.tolist() == [1, 1, 0, 0, 0, 0]


def test_prompt_tokens_before_the_first_sequence_are_padding():
    from tests.test_gpu_kv_cache import make_stack

    stack, alone = make_stack(2, 20, layers=2), make_stack(2, 20, layers=2)
    x = rnd((30, 256), BF, 1)
    out = stack.prompt(x, i32([4, 4, 21]), i32([0, 1]))
    stack.cache.check()
    assert stack.cache.lens.tolist() == [0, 17]
    assert torch.equal(out[4:21], alone.prompt(x[4:21], i32([0, 17]), i32([1])))


@pytest.mark.parametrize("dtype,heads,kv,d", [(BF, 4, 2, 64), (HF, 34, 2, 128), (HF, 8, 1, 64)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("path", ["prompt", "decode", "prefix"])
def test_tiles_without_keys_do_not_hide_a_nan_seen_before(dtype, heads, kv, d, value, path):
    """A score that is not a number, then tiles of which the row (or, in decode, a warp's part of the row) sees nothing."""
    from kcapw_klcquant_b200 import attn_decode, attn_prompt

    key, q = 100, rnd((300, heads, d), dtype, 1).abs() + 0.1
    k, v = rnd((700, kv, d), dtype, 2), rnd((700, kv, d), dtype, 3)
    k[key, kv - 1, 5] = value
    if path == "prompt":  # rows of one item end in different tiles
        out, lse = attn_prompt(q, k[:300], v[:300], i32([0, 300]), return_lse=True)
        hit = torch.arange(300, device=DEV) >= key
    else:
        lens = [101 + i % 150 for i in range(300)] if path == "decode" else [90 + 2 * i for i in range(300)]
        kw = {} if path == "decode" else dict(group_starts=i32([0, 300]), prefix_lens=i32([640]))
        kp, vp, table = ref.paged([k], [v], 64)
        out, lse = attn_decode(q, kp, vp, table.expand(300, -1).contiguous(), i32(lens), return_lse=True, **kw)
        hit = i32(lens) > key
    group = heads // kv
    for got in (out, lse):
        assert got[hit, heads - group:].isnan().all()
        assert got[~hit].isfinite().all() and got[:, :heads - group].isfinite().all()


# ---- captured, large -------------------------------------------------------------------


def test_captured_prefix_decode_serves_other_groups_and_two_graphs_run_side_by_side():
    from kcapw_klcquant_b200 import attn_decode, check_device_status

    n, prefix = 6, 640
    k, v = rnd((1400, 2, 64), BF, 1), rnd((1400, 2, 64), BF, 2)
    kp, vp, table = ref.paged([k], [v], 32)
    table = table.expand(n, -1).contiguous()
    q = [rnd((n, 8, 64), BF, 3 + i) for i in range(2)]
    ln, gs, pl = i32([700] * n), i32([0, 3, 6]), i32([prefix, prefix])
    attn_decode(q[0], kp, vp, table, ln, group_starts=gs, prefix_lens=pl)
    graphs = []
    for x in q:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = attn_decode(x, kp, vp, table, ln, window=900, group_starts=gs, prefix_lens=pl)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for lens, starts, pres in (([700] * n, [0, 3, 6], [640, 640]), ([1400, 3, 0, 900, 640, 1280], [1, 1, 5], [32, 1248]),
                               ([641, 642, 643, 1, 1399, 33], [0, 6, 6], [640, 0]), ([1400] * n, [2, 2, 2], [64, 64])):
        ln.copy_(i32(lens))
        gs.copy_(i32(starts))
        pl.copy_(i32(pres))
        torch.cuda.synchronize()
        for _ in range(3):
            for s, (g, _) in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        check_device_status(DEV)
        for x, (_, out) in zip(q, graphs):
            check_decode(x, [k[:m] for m in lens], [v[:m] for m in lens], 900, None, out, None)


def test_pages_past_32_bits():
    """A pool of 5.2e9 elements whose last pages are the free ones: append, attend, fork with copies, compact."""
    from kcapw_klcquant_b200 import PagedKvCache, attn_decode, rope_append

    pages, ps, kv, d, n = 20000, 128, 8, 128, 300
    cache = PagedKvCache(layers=1, pages=pages, page_size=ps, kv_heads=kv, head_dim=d, rows=3, row_pages=4, device=DEV)
    cache.refs[:pages - 8] = 1
    cache.reserve(i32([n, 0, 0]))
    assert cache.block_table[0].tolist() == [pages - 8, pages - 7, pages - 6, -1]
    q, k, v = rnd((n, 8, d), BF, 1), rnd((n, kv, d), BF, 2), rnd((n, kv, d), BF, 3)
    ang = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * 0.01 * torch.arange(d // 2, device=DEV, dtype=torch.float64)
    q, k = rope_append(q, k, v, ang.cos().float(), ang.sin().float(), torch.arange(n, device=DEV, dtype=torch.int32),
                       torch.zeros(n, device=DEV, dtype=torch.int32), cache.k(0), cache.v(0), cache.block_table, return_k=True)
    cache.fork(i32([0, 0]), i32([1, 2]))
    cache.check()

    def attend():
        out = attn_decode(q[-3:], cache.k(0), cache.v(0), cache.block_table, cache.lens)
        check_decode(q[-3:], [k] * 3, [v] * 3, 0, None, out, None)

    attend()
    cache.refs[:pages - 8] = 0
    assert int(cache.compact()) == 5
    cache.check()
    assert sorted(set(cache.block_table.flatten().tolist())) == [-1, 0, 1, 2, 3, 4]
    attend()


def test_captured_prompt_serves_other_rows_and_offsets():
    from kcapw_klcquant_b200 import KlcError
    from tests.test_gpu_kv_cache import make_stack

    stack, eager = make_stack(4, 40, layers=2), make_stack(4, 40, layers=2)
    x, cu, rows = rnd((48, 256), BF, 1), i32([0, 20, 48]), i32([1, 3])
    stack.prompt(x, cu, rows)
    stack.cache.free(rows)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = stack.prompt(x, cu, rows)
    for offsets, into in (([0, 20, 48], [1, 3]), ([0, 48, 48], [2, 0]), ([3, 10, 40], [0, 2])):
        cu.copy_(i32(offsets))
        rows.copy_(i32(into))
        x.copy_(rnd((48, 256), BF, 7 + offsets[1]))
        g.replay()
        stack.cache.check()
        want = eager.prompt(x, cu, rows)
        a, b = offsets[0], offsets[-1]
        assert torch.equal(out[a:b], want[a:b]) and torch.equal(stack.cache.lens, eager.cache.lens)
        live = eager.cache.refs > 0
        assert torch.equal(stack.cache.refs, eager.cache.refs) and torch.equal(stack.cache.pool[:, :, live], eager.cache.pool[:, :, live])
        if offsets[0]:
            g.replay()  # the rows hold keys now
            with pytest.raises(KlcError):
                stack.cache.check()
            assert torch.equal(stack.cache.lens, eager.cache.lens)
        for s in (stack, eager):
            s.cache.free(rows)
