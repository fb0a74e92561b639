"""Attention over prompts and over the paged cache, and rotary append, against 64-bit references."""
from __future__ import annotations

import pytest
import torch

from tests import attention_ref as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
BF, HF = torch.bfloat16, torch.float16


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def cum(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV)


def check_prompt(q, k, v, lq, lk, window, sinks, out, lse, scale):
    aq = ak = 0
    for i, (n, m) in enumerate(zip(lq, lk)):
        pos = torch.arange(n, device=DEV) + (m - n)
        want, wl, bound = ref.attention(q[aq:aq + n], k[ak:ak + m], v[ak:ak + m], pos, scale, window, sinks)
        ref.assert_close(out[aq:aq + n], want, bound, f"sequence {i} ({n} rows, {m} keys)")
        if lse is not None:
            ref.assert_lse(lse[aq:aq + n], wl, f"sequence {i}")
        aq, ak = aq + n, ak + m


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,kv,d", [(8, 1, 64), (4, 4, 64), (6, 2, 128), (64, 1, 64), (10, 2, 128)])
@pytest.mark.parametrize("lens", [[1], [127, 1, 0, 130], [300, 17], [129, 128, 257]])
@pytest.mark.parametrize("window,sink", [(0, False), (0, True), (1, True), (50, False), (128, True)])
def test_prompt(dtype, heads, kv, d, lens, window, sink):
    from kcapw_klcquant_b200 import attn_prompt, check_device_status

    T = sum(lens)
    qkv = rnd((T + 3, heads + 2 * kv, d), dtype, 1)  # three rows of padding behind the last sequence
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    sinks = torch.randn(heads, device=DEV) if sink else None
    out = torch.full((T + 3, heads, d), 7.0, dtype=dtype, device=DEV)
    got, lse = attn_prompt(q, k, v, cum(lens), window=window, sinks=sinks, out=out, return_lse=True)
    check_device_status(DEV)
    assert got is out and (out[T:] == 7.0).all(), "rows behind the last sequence were written"
    check_prompt(q, k, v, lens, lens, window, sinks, out, lse, d ** -0.5)


@pytest.mark.parametrize("dtype,d", [(BF, 64), (HF, 128)])
@pytest.mark.parametrize("lq,lk", [([5, 130], [200, 700]), ([40], [3]), ([3, 9], [0, 9]), ([256, 1], [256, 1000])])
@pytest.mark.parametrize("window", [0, 64])
def test_prompt_other_keys(dtype, d, lq, lk, window):
    """More keys than queries (an earlier part of the sequence), fewer (rows that see nothing), none."""
    from kcapw_klcquant_b200 import attn_prompt, check_device_status

    q, k, v = rnd((sum(lq), 6, d), dtype, 2), rnd((sum(lk), 2, d), dtype, 3), rnd((sum(lk), 2, d), dtype, 4)
    out, lse = attn_prompt(q, k, v, cum(lq), cu_seqlens_k=cum(lk), window=window, return_lse=True, scale=0.2)
    check_device_status(DEV)
    check_prompt(q, k, v, lq, lk, window, None, out, lse, 0.2)


@pytest.mark.parametrize("window", [1 << 30, (1 << 31) - 1])
def test_largest_windows(window):
    """A window larger than any position is none, also for rows before the first key."""
    from kcapw_klcquant_b200 import attn_decode, attn_prompt

    q, k, v = rnd((200, 4, 64), BF, 2), rnd((70, 2, 64), BF, 3), rnd((70, 2, 64), BF, 4)
    a = attn_prompt(q, k, v, cum([200]), cu_seqlens_k=cum([70]))
    assert torch.equal(attn_prompt(q, k, v, cum([200]), cu_seqlens_k=cum([70]), window=window), a)
    kp, vp, table = ref.paged([k], [v], 16)
    ln = torch.tensor([70], dtype=torch.int32, device=DEV)
    a = attn_decode(q[:1], kp, vp, table, ln)
    assert torch.equal(attn_decode(q[:1], kp, vp, table, ln, window=window), a)


def test_prompt_output_over_the_queries_and_single_heads():
    from kcapw_klcquant_b200 import attn_prompt

    lens = [130, 61]
    q, k, v = rnd((191, 1, 128), HF, 2), rnd((191, 1, 128), HF, 3), rnd((191, 1, 128), HF, 4)
    want = attn_prompt(q, k, v, cum(lens))
    assert attn_prompt(q, k, v, cum(lens), out=q) is q and torch.equal(q, want)


def test_prompt_captured_serves_other_offsets():
    from kcapw_klcquant_b200 import attn_prompt

    q, k, v = rnd((300, 8, 64), BF, 2), rnd((300, 2, 64), BF, 3), rnd((300, 2, 64), BF, 4)
    cu = cum([100, 150, 50])
    attn_prompt(q, k, v, cu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = attn_prompt(q, k, v, cu)
    for lens in ([100, 150, 50], [1, 0, 299], [300, 0, 0]):
        cu.copy_(cum(lens))
        g.replay()
        check_prompt(q, k, v, lens, lens, 0, None, out, None, 0.125)


def test_calls_on_a_stream_that_is_not_current_at_creation():
    """Inputs made on one stream, used on another after an event; two prompts in flight at once."""
    from kcapw_klcquant_b200 import attn_prompt

    q, k, v = rnd((2000, 8, 128), BF, 2), rnd((2000, 2, 128), BF, 3), rnd((2000, 2, 128), BF, 4)
    want = attn_prompt(q, k, v, cum([1500, 500]))
    cu = cum([1500, 500])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(attn_prompt(q, k, v, cu))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_prompt_no_keys_at_all_and_no_rows():
    from kcapw_klcquant_b200 import attn_prompt

    q = rnd((5, 4, 64), BF, 5)
    e = torch.empty((0, 2, 64), dtype=BF, device=DEV)
    out, lse = attn_prompt(q, e, e, cum([5]), cu_seqlens_k=cum([0]), return_lse=True)
    assert (out == 0).all() and (lse == -float("inf")).all()
    assert attn_prompt(q[:0], e, e, cum([])).shape == (0, 4, 64)


@pytest.mark.parametrize("d", [64, 128])
def test_prompt_large_scores_and_growing_maxima(d):
    """Scores whose maximum grows along the keys by far more than the rescale threshold, and large negative ones."""
    from kcapw_klcquant_b200 import attn_prompt

    n = 900
    q, k, v = rnd((n, 2, d), HF, 6), rnd((n, 1, d), HF, 7), rnd((n, 1, d), HF, 8)
    q = q.abs()
    ramp = torch.linspace(-6, 6, n, device=DEV)[:, None, None]
    k = (k.abs() * ramp).to(HF)  # scores from about -200 to 200 along the keys
    out, lse = attn_prompt(q, k, v, cum([n]), return_lse=True)
    check_prompt(q, k, v, [n], [n], 0, None, out, lse, d ** -0.5)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_prompt_neighbours_do_not_reach_a_sequence(d, bad):
    """Not-a-number rows in padding and in other sequences leave a sequence's bits alone; one in its own query row stays there."""
    from kcapw_klcquant_b200 import attn_prompt

    lens = [70, 200, 33]
    mk = lambda s: rnd((sum(lens) + 9, 4, d), BF, s)  # noqa: E731
    q, k, v = mk(9), mk(10), mk(11)
    clean = attn_prompt(q, k, v, cum(lens))
    for t in (q, k, v):
        t[:70] = bad
        t[303:] = bad
    q[100, 1] = bad
    got = attn_prompt(q, k, v, cum(lens))
    keep = torch.ones(q.shape[0], 4, dtype=torch.bool, device=DEV)
    keep[:70] = False
    keep[303:] = False
    keep[100, 1] = False
    assert torch.equal(got[keep], clean[keep])
    assert got[100, 1].isnan().all()
    assert got[:70].isnan().any()


@pytest.mark.parametrize("d,heads", [(64, 8), (128, 1)])
@pytest.mark.parametrize("lq,lk,window", [([40], [500], 64), ([5, 300], [200, 700], 30), ([1, 1], [129, 127], 1)])
def test_prompt_keys_that_no_row_sees_may_hold_anything(d, heads, lq, lk, window):
    """Keys before every row's window (dropped by a cache, say) hold not-a-numbers."""
    from kcapw_klcquant_b200 import attn_prompt

    q, k, v = rnd((sum(lq), heads, d), BF, 9), rnd((sum(lk), 1, d), BF, 10), rnd((sum(lk), 1, d), BF, 11)
    clean = attn_prompt(q, k, v, cum(lq), cu_seqlens_k=cum(lk), window=window)
    check_prompt(q, k, v, lq, lk, window, None, clean, None, d ** -0.5)
    at = 0
    for n, m in zip(lq, lk):
        k[at:at + m - n - window + 1] = float("nan")
        v[at:at + m - n - window + 1] = float("inf")
        at += m
    assert torch.equal(attn_prompt(q, k, v, cum(lq), cu_seqlens_k=cum(lk), window=window), clean)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,kv,d", [(16, 2, 64), (2, 2, 64), (12, 4, 128), (1, 1, 128)])
@pytest.mark.parametrize("window", [0, 40, 150])
@pytest.mark.parametrize("lq,lk", [([400], [400]), ([60, 70], [300, 128]), ([50], [20])])
def test_prompt_values_that_are_not_finite_reach_the_rows_that_see_them(dtype, heads, kv, d, window, lq, lk):
    """Bad elements at the diagonal, at tile edges and at window edges: their column of the rows that see the key, nothing else."""
    from kcapw_klcquant_b200 import attn_prompt

    q, k, v = rnd((sum(lq), heads, d), dtype, 12), rnd((sum(lk), kv, d), dtype, 13), rnd((sum(lk), kv, d), dtype, 14)
    clean = attn_prompt(q, k, v, cum(lq), cu_seqlens_k=cum(lk), window=window)
    bad = [(lk[0] - 1, 3, float("nan")), (lk[0] // 2, 5, float("inf")), (lk[0] // 2, 40, float("-inf")), (0, 6, float("inf")),
           (min(127, lk[0] - 1), d - 1, float("nan")), (max(0, lk[0] - 20), 7, float("-inf")), (max(0, lk[0] - 45), 8, float("nan"))]
    for key, col, val in bad:
        v[key, kv - 1, col] = val
    got = attn_prompt(q, k, v, cum(lq), cu_seqlens_k=cum(lk), window=window)
    want = clean.clone()
    pos = torch.arange(lq[0], device=DEV) + lk[0] - lq[0]
    g = heads // kv
    for key, col, val in bad:
        see = (pos >= key) & ((pos < key + window) if window else True)
        want[:lq[0]][see, heads - g:, col] = val
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


@pytest.mark.parametrize("dtype,d", [(BF, 64), (HF, 128)])
def test_decode_prefix_values_that_are_not_finite(dtype, d):
    """In a shared prefix under a window, a bad value reaches the rows whose window holds its key."""
    from kcapw_klcquant_b200 import attn_decode

    prefix, window, tails = 320, 200, [1, 30, 90, 150, 199, 260]
    pk, pv = rnd((prefix, 2, d), dtype, 1), rnd((prefix, 2, d), dtype, 2)
    ks = [torch.cat([pk, rnd((t, 2, d), dtype, 10 + t)]) for t in tails]
    vs = [torch.cat([pv, rnd((t, 2, d), dtype, 500 + t)]) for t in tails]
    q = rnd((len(tails), 8, d), dtype, 3)
    ln = torch.tensor([prefix + t for t in tails], dtype=torch.int32, device=DEV)
    gs, pl = torch.tensor([0, len(tails)], dtype=torch.int32, device=DEV), torch.tensor([prefix], dtype=torch.int32, device=DEV)

    def run():
        kp, vp, table = ref.paged(ks, vs, 32)
        return attn_decode(q, kp, vp, table, ln, window=window, group_starts=gs, prefix_lens=pl)

    clean = run()
    want = clean.clone()
    for key, col, val in ((200, 4, float("nan")), (319, 9, float("inf")), (130, 11, float("nan")), (100, 20, float("inf"))):
        for i, t in enumerate(tails):
            vs[i][key, 0, col] = val
            if key >= prefix + t - window:
                want[i, :4, col] = val
    got = run()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


def test_prompt_nan_key_is_a_nan_row():
    from kcapw_klcquant_b200 import attn_prompt

    q, k, v = rnd((400, 2, 64), BF, 12), rnd((400, 2, 64), BF, 13), rnd((400, 2, 64), BF, 14)
    k[200] = float("nan")
    got = attn_prompt(q, k, v, cum([400]))
    assert got[200:].isnan().all() and not got[:200].isnan().any()


def test_prompt_bad_offsets_are_reported():
    from kcapw_klcquant_b200 import KlcError, attn_prompt, check_device_status

    q, k, v = rnd((100, 2, 64), BF, 15), rnd((100, 2, 64), BF, 16), rnd((100, 2, 64), BF, 17)
    for cu in ([0, 40, 200], [0, 40, 30], [-5, 40, 100]):
        attn_prompt(q, k, v, torch.tensor(cu, dtype=torch.int32, device=DEV))
        with pytest.raises(KlcError):
            check_device_status(DEV)
    check_device_status(DEV)  # reported once
    out = attn_prompt(q, k, v, cum([40, 60]))
    check_device_status(DEV)
    check_prompt(q, k, v, [40, 60], [40, 60], 0, None, out, None, 0.125)


def test_prompt_many_sequences_and_strided_inputs():
    """More sequences than lanes and CTAs, with keys in [heads, tokens] order and unaligned rows (copied)."""
    from kcapw_klcquant_b200 import attn_prompt

    lens = [(7 * i) % 23 for i in range(333)]
    T = sum(lens)
    q = rnd((4, T, 64), BF, 18).transpose(0, 1)
    k = rnd((2, T, 64), BF, 19).transpose(0, 1)
    v = rnd((T, 2, 67), BF, 20)[:, :, 3:]
    out = attn_prompt(q, k, v, cum(lens))
    check_prompt(q, k, v, lens, lens, 0, None, out, None, 0.125)


# ---- single tokens over the cache ------------------------------------------------


def decode_case(dtype, heads, kv, d, lens, ps, window, sink, seed=0, prefix=0, groups=None):
    ks = [rnd((n, kv, d), dtype, seed + 100 + i) for i, n in enumerate(lens)]
    vs = [rnd((n, kv, d), dtype, seed + 500 + i) for i, n in enumerate(lens)]
    q = rnd((len(lens), heads, d), dtype, seed + 1)
    sinks = torch.randn(heads, device=DEV) if sink else None
    return q, ks, vs, sinks


def check_decode(q, ks, vs, window, sinks, out, lse):
    d = q.shape[2]
    for i, (k, v) in enumerate(zip(ks, vs)):
        pos = torch.tensor([k.shape[0] - 1], device=DEV)
        want, wl, bound = ref.attention(q[i:i + 1], k, v, pos, d ** -0.5, window, sinks)
        ref.assert_close(out[i:i + 1], want, bound, f"row {i} ({k.shape[0]} keys)")
        if lse is not None:
            ref.assert_lse(lse[i:i + 1], wl, f"row {i}")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,kv,d", [(8, 1, 64), (4, 4, 128), (6, 2, 64), (40, 2, 128), (64, 1, 64)])
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("lens,window,sink", [([1], 0, False), ([0, 1, 63, 64, 65, 1000], 0, True), ([500, 2000, 3], 100, True),
                                              ([129, 127], 1, False)])
def test_decode(dtype, heads, kv, d, ps, lens, window, sink):
    """Unused parts of the pages hold NaN: nothing of them may reach a row."""
    from kcapw_klcquant_b200 import attn_decode, check_device_status

    q, ks, vs, sinks = decode_case(dtype, heads, kv, d, lens, ps, window, sink)
    kp, vp, table = ref.paged(ks, vs, ps)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if window:  # pages before the window may be gone
        for i, n in enumerate(lens):
            table[i, :max(0, n - window) // ps] = -1
    out, lse = attn_decode(q, kp, vp, table, ln, window=window, sinks=sinks, return_lse=True)
    check_device_status(DEV)
    check_decode(q, ks, vs, window, sinks, out, lse)


@pytest.mark.parametrize("dtype,heads,kv,d", [(BF, 8, 1, 64), (HF, 6, 2, 128), (BF, 16, 16, 64), (HF, 64, 1, 64)])
@pytest.mark.parametrize("ps,prefix", [(16, 48), (64, 256), (128, 1280)])
@pytest.mark.parametrize("window", [0, 300])
def test_decode_shared_prefix(dtype, heads, kv, d, ps, prefix, window):
    """Two groups with prefixes of their own, rows outside any group, a row that is all prefix, one shorter than it."""
    from kcapw_klcquant_b200 import attn_decode, check_device_status

    tails = [70, 0, 1, 200, 33, 500, 9, 64, 40]
    ga, gb = (1, 5), (5, 8)  # rows of the groups; rows 0 and 8 have no prefix
    pre = {0: 0, 8: 0}
    kpre = {g: (rnd((prefix * (1 + g), kv, d), dtype, 60 + g), rnd((prefix * (1 + g), kv, d), dtype, 70 + g)) for g in (0, 1)}
    ks, vs = [], []
    for i, t in enumerate(tails):
        k, v = rnd((t, kv, d), dtype, 200 + i), rnd((t, kv, d), dtype, 300 + i)
        if i not in pre:
            g = 0 if i < 5 else 1
            k, v = torch.cat([kpre[g][0], k]), torch.cat([kpre[g][1], v])
        ks.append(k)
        vs.append(v)
    kp, vp, table = ref.paged(ks, vs, ps)
    # the group's first row holds the prefix; the others' entries for it are not read
    for lo, hi, g in ((*ga, 0), (*gb, 1)):
        table[lo + 1:hi, :prefix * (1 + g) // ps] = -7
    q = rnd((len(tails), heads, d), dtype, 90)
    sinks = torch.randn(heads, device=DEV)
    ln = torch.tensor([k.shape[0] for k in ks], dtype=torch.int32, device=DEV)
    gs = torch.tensor([1, 5, 8], dtype=torch.int32, device=DEV)
    pl = torch.tensor([prefix, 2 * prefix], dtype=torch.int32, device=DEV)
    out, lse = attn_decode(q, kp, vp, table, ln, window=window, sinks=sinks, group_starts=gs, prefix_lens=pl, return_lse=True)
    check_device_status(DEV)
    check_decode(q, ks, vs, window, sinks, out, lse)
    # a row may end inside the prefix
    ln2 = ln.clone()
    ln2[3] = prefix - 5
    ks[3], vs[3] = ks[3][:prefix - 5], vs[3][:prefix - 5]
    out = attn_decode(q, kp, vp, table, ln2, window=window, sinks=sinks, group_starts=gs, prefix_lens=pl)
    check_device_status(DEV)
    check_decode(q, ks, vs, window, sinks, out, None)


def test_decode_large_group_spans_row_tiles():
    from kcapw_klcquant_b200 import attn_decode

    B, kv, d, ps, prefix = 70, 2, 64, 32, 640
    pk, pv = rnd((prefix, kv, d), BF, 1), rnd((prefix, kv, d), BF, 2)
    ks = [torch.cat([pk, rnd((i % 7, kv, d), BF, 10 + i)]) for i in range(B)]
    vs = [torch.cat([pv, rnd((i % 7, kv, d), BF, 110 + i)]) for i in range(B)]
    kp, vp, table = ref.paged(ks, vs, ps)
    q = rnd((B, 10, d), BF, 3)
    ln = torch.tensor([k.shape[0] for k in ks], dtype=torch.int32, device=DEV)
    gs, pl = torch.tensor([0, B], dtype=torch.int32, device=DEV), torch.tensor([prefix], dtype=torch.int32, device=DEV)
    out = attn_decode(q, kp, vp, table, ln, group_starts=gs, prefix_lens=pl)
    check_decode(q, ks, vs, 0, None, out, None)


def test_decode_results_do_not_depend_on_timing_or_company():
    """The same call gives the same bits, on two streams at once too."""
    from kcapw_klcquant_b200 import attn_decode

    q, ks, vs, sinks = decode_case(BF, 16, 2, 64, [3000, 17, 900, 4000, 1], 64, 0, True)
    kp, vp, table = ref.paged(ks, vs, 64)
    ln = torch.tensor([k.shape[0] for k in ks], dtype=torch.int32, device=DEV)
    first = attn_decode(q, kp, vp, table, ln, sinks=sinks)
    main = torch.cuda.current_stream()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        s.wait_stream(main)
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(attn_decode(q, kp, vp, table, ln, sinks=sinks))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


def test_decode_captured_serves_other_lengths_and_two_graphs_share_nothing():
    from kcapw_klcquant_b200 import attn_decode

    q, ks, vs, _ = decode_case(BF, 8, 2, 64, [800, 1500, 300], 64, 0, False)
    kp, vp, table = ref.paged(ks, vs, 64)
    ln = torch.tensor([800, 1500, 300], dtype=torch.int32, device=DEV)
    attn_decode(q, kp, vp, table, ln)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = attn_decode(q, kp, vp, table, ln)
        graphs.append((g, out))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for cur in ([800, 1500, 300], [5, 64, 299], [800, 0, 1]):
        ln.copy_(torch.tensor(cur, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            with torch.cuda.stream(s1):
                graphs[0][0].replay()
            with torch.cuda.stream(s2):
                graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            check_decode(q, [k[:n] for k, n in zip(ks, cur)], [v[:n] for v, n in zip(vs, cur)], 0, None, out, None)


def test_decode_bad_pages_and_lengths_are_reported():
    from kcapw_klcquant_b200 import KlcError, attn_decode, check_device_status

    lens = [300, 200, 100]
    q, ks, vs, _ = decode_case(BF, 8, 2, 64, lens, 64, 0, False)
    kp, vp, table = ref.paged(ks, vs, 64)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for row, col, val in ((1, 2, -1), (1, 0, 10 ** 6), (1, 3, kp.shape[0])):
        bad = table.clone()
        bad[row, col] = val
        out = attn_decode(q, kp, vp, bad, ln)
        with pytest.raises(KlcError):
            check_device_status(DEV)
        check_decode(q[::2], ks[::2], vs[::2], 0, None, out[::2], None)
    for val in (-3, 10 ** 6):
        bad = ln.clone()
        bad[1] = val
        out = attn_decode(q, kp, vp, table, bad)
        with pytest.raises(KlcError):
            check_device_status(DEV)
        check_decode(q[::2], ks[::2], vs[::2], 0, None, out[::2], None)


def test_decode_offsets_past_32_bits():
    """A pool of more than 2^31 elements whose last pages are the used ones."""
    from kcapw_klcquant_b200 import attn_decode

    ps, kv, d = 128, 8, 128
    pages = (1 << 31) // (ps * kv * d) + 8
    pool = torch.zeros((pages, kv, ps, d), dtype=BF, device=DEV)
    n = 300
    k = rnd((n, kv, d), BF, 5)
    ids = [pages - 1, pages - 5, pages - 2]
    for j, page in enumerate(ids):
        part = k[j * ps:(j + 1) * ps]
        pool[page, :, :part.shape[0]] = part.transpose(0, 1)
    q = rnd((1, 16, d), BF, 6)
    out = attn_decode(q, pool, pool, torch.tensor([ids], dtype=torch.int32, device=DEV), torch.tensor([n], dtype=torch.int32, device=DEV))
    check_decode(q, [k], [k], 0, None, out, None)


def test_decode_table_slices_and_page_strides():
    """The layers of one pool (pages far apart), a table that is a slice of a wider one, q a slice of a projection."""
    from kcapw_klcquant_b200 import attn_decode

    lens = [200, 77]
    q, ks, vs, _ = decode_case(BF, 6, 2, 64, lens, 32, 0, False)
    kp, vp, table = ref.paged(ks, vs, 32)
    pool = torch.full((kp.shape[0], 3, *kp.shape[1:]), float("nan"), dtype=BF, device=DEV)
    pool[:, 0], pool[:, 2] = kp, vp
    wide = torch.full((2, table.shape[1] + 9), -5, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + table.shape[1]] = table
    qkv = rnd((2, 10, 64), BF, 77)
    qkv[:, :6] = q
    out = attn_decode(qkv[:, :6], pool[:, 0], pool[:, 2], wide[:, 2:2 + table.shape[1]], torch.tensor(lens, dtype=torch.int32, device=DEV))
    check_decode(q, ks, vs, 0, None, out, None)


def test_decode_groups_cover_nothing_or_everything():
    """Zero-length prefixes, empty groups, no groups at all, and bad prefixes reported."""
    from kcapw_klcquant_b200 import KlcError, attn_decode, check_device_status

    lens = [100, 50, 300]
    q, ks, vs, _ = decode_case(BF, 8, 2, 64, lens, 16, 0, False)
    kp, vp, table = ref.paged(ks, vs, 16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    ln = i32(lens)
    for gs, pl in (([0, 3], [0]), ([0, 0, 1, 1], [16, 32, 16]), ([0], []), ([2, 3], [160])):
        out = attn_decode(q, kp, vp, table, ln, group_starts=i32(gs), prefix_lens=i32(pl))
        check_device_status(DEV)
        check_decode(q, ks, vs, 0, None, out, None)
    for gs, pl in (([0, 1], [15]), ([0, 1], [-16]), ([0, 1], [16 * 1000]), ([0, 9], [16]), ([2, 1], [16])):
        attn_decode(q, kp, vp, table, ln, group_starts=i32(gs), prefix_lens=i32(pl))
        with pytest.raises(KlcError):
            check_device_status(DEV)


def test_decode_long_context():
    from kcapw_klcquant_b200 import attn_decode

    q, ks, vs, sinks = decode_case(HF, 4, 1, 128, [70001], 16, 0, True)
    kp, vp, table = ref.paged(ks, vs, 16)
    out = attn_decode(q, kp, vp, table, torch.tensor([70001], dtype=torch.int32, device=DEV), sinks=sinks)
    check_decode(q, ks, vs, 0, sinks, out, None)


def test_decode_most_sequences():
    from kcapw_klcquant_b200 import attn_decode, check_device_status

    B, kv, d, ps = 4096, 1, 64, 16
    kp, vp = rnd((64, kv, ps, d), BF, 7), rnd((64, kv, ps, d), BF, 8)
    table = torch.randint(0, 64, (B, 2), dtype=torch.int32, device=DEV)
    ln = torch.randint(0, 33, (B,), dtype=torch.int32, device=DEV)
    q = rnd((B, 2, d), BF, 9)
    out = attn_decode(q, kp, vp, table, ln)
    check_device_status(DEV)
    for i in range(0, B, 97):
        n = int(ln[i])
        k = kp[table[i].long()].transpose(1, 2).reshape(-1, kv, d)[:n]
        v = vp[table[i].long()].transpose(1, 2).reshape(-1, kv, d)[:n]
        check_decode(q[i:i + 1], [k], [v], 0, None, out[i:i + 1], None)


# ---- rotary append -----------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,kv,d,ps", [(8, 2, 64, 16), (3, 1, 128, 64), (64, 8, 64, 128)])
def test_rope_append(dtype, heads, kv, d, ps):
    from kcapw_klcquant_b200 import check_device_status, rope_append

    T, rows, width, max_pos = 37, 5, 9, 8 * ps
    qkv = rnd((T, heads + 2 * kv, d), dtype, 1)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    pages = rows * width
    table = torch.randperm(pages, device=DEV, dtype=torch.int32).view(rows, width)
    slots = torch.randperm(rows * max_pos, device=DEV)[:T]
    row, pos = (slots // max_pos).to(torch.int32), (slots % max_pos).to(torch.int32)
    row[::9] = -1  # padding
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * 150000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    cos, sin = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
    kp = torch.full((pages, kv, ps, d), 5.0, dtype=dtype, device=DEV)
    vp = kp.clone()
    out = torch.full((T, heads, d), 5.0, dtype=dtype, device=DEV)
    got, ko = rope_append(q, k, v, cos, sin, pos, row, kp, vp, table, out=out, return_k=True)
    check_device_status(DEV)
    live = row >= 0
    c, s = cos[pos.long()], sin[pos.long()]
    u = ref.U[dtype]
    for x, y in ((q, got), (k, ko)):
        want = ref.rotate(x, c, s)
        # one rounding to the type (its subnormal step at worst), products and sum in fp32
        size = ref.rotate(x.abs(), c.abs(), -s.abs()).abs() + ref.rotate(x.abs(), c.abs(), s.abs()).abs()
        ref.assert_close(y[live], want[live], (u * want.abs() + 2.0 ** -22 * size + 2.0 ** -25)[live], "rotated")
    assert (got[~live] == 5.0).all()
    page = table[row.clamp(min=0).long(), (pos // ps).long()].long()
    at = (pos % ps).long()
    assert torch.equal(kp[page, :, at][live], ko[live]) and torch.equal(vp[page, :, at][live], v[live])
    used = torch.zeros((pages, ps), dtype=torch.bool, device=DEV)
    used[page[live], at[live]] = True
    assert (kp.transpose(1, 2)[~used] == 5.0).all() and (vp.transpose(1, 2)[~used] == 5.0).all()
    # in place
    q2 = q.contiguous()
    rope_append(q2, k, v, cos, sin, pos, row, kp, vp, table, out=q2)
    assert torch.equal(q2[live], got[live]) and torch.equal(q2[~live], q[~live])


def test_rope_append_reports_bad_places():
    from kcapw_klcquant_b200 import KlcError, check_device_status, rope_append

    q, k, v = rnd((1, 2, 64), BF, 1), rnd((1, 1, 64), BF, 2), rnd((1, 1, 64), BF, 3)
    cos = sin = torch.ones((32, 32), device=DEV)
    kp = torch.zeros((4, 1, 16, 64), dtype=BF, device=DEV)
    vp = kp.clone()
    for table, row, pos in (([[0, 1, 2]], 0, 32), ([[0, 1]], 1, 3), ([[0, 4]], 0, 20), ([[-1, 1]], 0, 5), ([[0]], 0, 17), ([[0, 1]], -2, 0),
                            ([[0, 1]], 0, -1)):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        rope_append(q, k, v, cos, sin, i32([pos]), i32([row]), kp, vp, i32(table))
        with pytest.raises(KlcError):
            check_device_status(DEV)
        assert (kp == 0).all() and (vp == 0).all()


def test_refusals_on_the_device():
    from kcapw_klcquant_b200 import KlcError, attn_decode, attn_prompt

    q, k = rnd((4, 4, 64), BF, 1), rnd((4, 2, 64), BF, 2)
    cu = cum([4])
    kp = torch.zeros((4, 2, 16, 64), dtype=BF, device=DEV)
    tb, ln = torch.zeros((4, 1), dtype=torch.int32, device=DEV), torch.ones(4, dtype=torch.int32, device=DEV)
    for exc, call in (
        (ValueError, lambda: attn_prompt(q.float(), k.float(), k.float(), cu)),
        (ValueError, lambda: attn_prompt(q, k.half(), k.half(), cu)),
        (ValueError, lambda: attn_prompt(q, k, k[:3], cu)),
        (ValueError, lambda: attn_prompt(q, k[:3], k[:3], cu)),
        (ValueError, lambda: attn_prompt(q, k, k, cu.long())),
        (ValueError, lambda: attn_prompt(q, k, k, cu, window=-1)),
        (ValueError, lambda: attn_prompt(q, k, k, cu, scale=0.0)),
        (ValueError, lambda: attn_prompt(q, k, k, cu, scale=float("inf"))),
        (ValueError, lambda: attn_prompt(q, k, k, cu, sinks=torch.zeros(3, device=DEV))),
        (ValueError, lambda: attn_prompt(q, k, k, cu, out=q[:3])),
        (ValueError, lambda: attn_prompt(q[:, :3], k, k, cu)),
        (KlcError, lambda: attn_prompt(q[..., :32].contiguous(), k[..., :32].contiguous(), k[..., :32].contiguous(), cu)),
        (ValueError, lambda: attn_decode(q, kp, kp, tb[:3], ln)),
        (ValueError, lambda: attn_decode(q, kp, kp, tb, ln[:3])),
        (ValueError, lambda: attn_decode(q, kp[:, :, :8].contiguous(), kp[:, :, :8].contiguous(), tb, ln)),
        (ValueError, lambda: attn_decode(q, kp.transpose(1, 2), kp.transpose(1, 2), tb, ln)),
        (ValueError, lambda: attn_decode(q, kp, kp, tb, ln, prefix_lens=ln[:1])),
        (ValueError, lambda: attn_decode(q, kp, kp, tb, ln, group_starts=ln, prefix_lens=ln)),
    ):
        with pytest.raises(exc):
            call()
