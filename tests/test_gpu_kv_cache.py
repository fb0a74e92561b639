"""Cache pages (reserve, fork, copy, free, compact) against a Python model, and the layer stack that uses them."""
from __future__ import annotations

import random

import pytest
import torch

from tests import attention_ref as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Model:
    """The cache's documented behaviour, one request at a time; a page's content is a number."""

    def __init__(self, pages, ps, rows, width):
        self.ps, self.width = ps, width
        self.refs, self.table, self.lens = [0] * pages, [[] for _ in range(rows)], [0] * rows
        self.content = [0] * pages
        self.fault = False

    def _take(self, n):
        free = [i for i, r in enumerate(self.refs) if r == 0]
        return free[:n] if len(free) >= n else None

    def reserve(self, add):
        out = False  # no page left for some row: later rows that need pages go without as well
        for r, a in enumerate(add):
            n = self.lens[r] + a
            if a < 0 or n > self.width * self.ps:
                self.fault = True
                continue
            need = -(-n // self.ps) - len(self.table[r])
            got = [] if need == 0 else (None if out else self._take(need))
            if got is None:
                out = self.fault = True
                continue
            for p in got:
                self.refs[p] = 1
            self.table[r] += got
            self.lens[r] = n

    def fork(self, parents, children, copy):
        rows = len(self.lens)
        lens, tables = list(self.lens), [list(t) for t in self.table]
        done, out = set(), False
        for par, ch in zip(parents, children):
            if not (0 <= par < rows and 0 <= ch < rows) or ch in done or lens[ch] != 0:
                self.fault = True
                if 0 <= ch < rows:
                    done.add(ch)
                continue
            done.add(ch)
            keep = 0 if copy else lens[par] // self.ps
            own = tables[par][keep:]
            got = [] if not own else (None if out else self._take(len(own)))
            if got is None:
                out = self.fault = True
                continue
            for p in tables[par][:keep]:
                self.refs[p] += 1
            for s, d in zip(own, got):
                self.refs[d] = 1
                self.content[d] = self.content[s]
            self.table[ch] = tables[par][:keep] + got
            self.lens[ch] = lens[par]

    def free(self, rows):
        for r in rows:
            if not 0 <= r < len(self.lens):
                self.fault = True
                continue
            for p in self.table[r]:
                self.refs[p] -= 1
            self.table[r], self.lens[r] = [], 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [i for i in range(live) if self.refs[i] == 0]
        movers = [i for i in range(live, len(self.refs)) if self.refs[i] > 0]
        to = dict(zip(movers, holes))
        for s, d in to.items():
            self.refs[d], self.refs[s], self.content[d] = self.refs[s], 0, self.content[s]
        self.table = [[to.get(p, p) for p in t] for t in self.table]
        return live


def make(pages, ps, rows, width, layers=2, kv=2, d=64):
    from kcapw_klcquant_b200 import PagedKvCache

    return PagedKvCache(layers=layers, pages=pages, page_size=ps, kv_heads=kv, head_dim=d, rows=rows, row_pages=width, device=DEV)


def paint(cache, model):
    """A number of its own in every live page, the same everywhere in the page but for the plane."""
    for p, r in enumerate(model.refs):
        if r > 0 and model.content[p] == 0:
            model.content[p] = paint.next = paint.next % 120 + 1
            planes = torch.arange(2 * cache.pool.shape[0], device=DEV).view(-1, 2, 1, 1, 1)
            cache.pool[:, :, p] = (model.content[p] + 128 * (planes % 2)).to(cache.pool.dtype)
        elif r == 0:
            model.content[p] = 0


paint.next = 0


def same(cache, model, what=""):
    from kcapw_klcquant_b200 import KlcError

    if model.fault:
        with pytest.raises(KlcError):
            cache.check()
        model.fault = False
    cache.check()
    assert cache.lens.tolist() == model.lens, what
    assert cache.refs.tolist() == model.refs, what
    table = [t + [-1] * (model.width - len(t)) for t in model.table]
    assert cache.block_table.tolist() == table, what
    first = cache.pool[:, :, :, 0, 0, 0].float().cpu()  # one value per page and plane, then whole pages
    for p, r in enumerate(model.refs):
        if r > 0 and model.content[p]:  # 0: taken in this step, not written yet
            assert first[0, 0, p] == model.content[p], f"{what}: page {p}"
            page = cache.pool[:, :, p].float()
            assert (page[:, 0] == model.content[p]).all() and (page[:, 1] == model.content[p] + 128).all(), f"{what}: page {p}"


@pytest.mark.parametrize("ps,pages,rows,width", [(16, 40, 8, 9), (128, 7, 5, 3), (64, 17, 12, 4), (32, 5000, 6, 40)])
@pytest.mark.parametrize("seed", range(3))
def test_random_walk(ps, pages, rows, width, seed):
    """Any order of requests, good and bad, leaves the state the documentation says."""
    rng = random.Random(seed)
    cache, model = make(pages, ps, rows, width), Model(pages, ps, rows, width)
    for step in range(40):
        op = rng.choice(["reserve", "reserve", "fork", "copy", "free", "compact"])
        if op == "reserve":
            add = [rng.choice([0, 0, 1, ps, rng.randrange(3 * ps)]) for _ in range(rows)]
            if rng.random() < 0.1:
                add[rng.randrange(rows)] = rng.choice([-1, 10 ** 6, 2 ** 31 - 1])
            cache.reserve(i32(add))
            model.reserve(add)
        elif op in ("fork", "copy"):
            n = rng.randrange(rows + 1)
            par = [rng.randrange(rows) for _ in range(n)]
            ch = [rng.randrange(rows) for _ in range(n)]
            if n and rng.random() < 0.2:
                (par if rng.random() < 0.5 else ch)[rng.randrange(n)] = rng.choice([-1, rows, 10 ** 6])
            cache.fork(i32(par), i32(ch), copy=op == "copy")
            model.fork(par, ch, op == "copy")
        elif op == "free":
            rs = [rng.randrange(rows) for _ in range(rng.randrange(3))]  # the same row twice at times
            cache.free(i32(rs))
            model.free(rs)
        else:
            assert int(cache.compact()) == model.compact()
        same(cache, model, f"step {step} {op}")
        paint(cache, model)


def test_large_pool():
    """More pages than one scan step, the free ones far back; rows by the thousand."""
    pages, rows = 70000, 3000
    cache = make(pages, 16, rows, 8, layers=1, kv=1)
    cache.refs[:60000] = 1
    cache.refs[60001] = 1
    cache.reserve(torch.full((rows,), 17, dtype=torch.int32, device=DEV))
    cache.check()
    want = [60000] + list(range(60002, 60002 + 2 * rows - 1))
    assert cache.block_table[:, :2].flatten().tolist() == want
    assert int(cache.compact()) == 60001 + 2 * rows
    assert cache.refs.max() == 1 and (cache.refs[:60001 + 2 * rows] == 1).all() and (cache.refs[60001 + 2 * rows:] == 0).all()


def test_ops_in_a_captured_graph():
    cache, model = make(30, 16, 6, 5), Model(30, 16, 6, 5)
    add = i32([1, 0, 1, 1, 0, 1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.reserve(add)
    for _ in range(40):
        g.replay()
        model.reserve(add.tolist())
    same(cache, model)


def test_snapshot_and_refusals():
    from kcapw_klcquant_b200 import PagedKvCache

    cache = make(30, 16, 6, 5)
    cache.reserve(i32([20, 3, 0, 0, 0, 0]))
    state = cache.snapshot()
    cache.reserve(i32([1] * 6))
    cache.restore(state)
    assert cache.lens.tolist() == [20, 3, 0, 0, 0, 0] and int(cache.refs.sum()) == 3
    for call in (lambda: cache.reserve(i32([1])), lambda: cache.reserve(torch.ones(6, device=DEV)), lambda: cache.fork(i32([0]), i32([1, 2])),
                 lambda: cache.fork(i32([0] * 7), i32([1] * 7)), lambda: cache.free(torch.zeros(1, dtype=torch.int32)),
                 lambda: PagedKvCache(layers=1, pages=4, page_size=24, kv_heads=1, head_dim=64, rows=1, row_pages=1),
                 lambda: PagedKvCache(layers=1, pages=4, page_size=16, kv_heads=1, head_dim=80, rows=1, row_pages=1),
                 lambda: PagedKvCache(layers=1, pages=4, page_size=16, kv_heads=1, head_dim=64, rows=1, row_pages=1, dtype=torch.float32)):
        with pytest.raises(ValueError):
            call()


# ---- the stack ------------------------------------------------------------------------


def make_stack(rows, pages, ps=16, layers=3, hidden=256, heads=8, kv=2, d=64):
    from kcapw_klcquant_b200 import AttentionLayer, MoeLayer, PagedKvCache
    from kcapw_klcquant_b200 import synthetic as syn
    from kcapw_klcquant_b200.stack import MoeStack

    g = torch.Generator(device=DEV).manual_seed(7)
    rnd = lambda *s, scale=0.05: (torch.randn(s, device=DEV, generator=g) * scale).to(torch.bfloat16)  # noqa: E731
    dims = syn.LayerDims(experts=16, hidden=hidden, intermediate=256, top_k=4)
    moe = [MoeLayer.from_tensors(0, syn.make_layer(dims, seed=30 + i, device=DEV), DEV, top_k=4) for i in range(layers)]
    attn = [AttentionLayer(rnd((heads + 2 * kv) * d, hidden), rnd(hidden, heads * d), heads, kv, d, qkv_bias=rnd((heads + 2 * kv) * d),
                           o_bias=rnd(hidden), sinks=rnd(heads, scale=1.0), window=20 if i % 2 else 0) for i in range(layers)]
    cache = PagedKvCache(layers=layers, pages=pages, page_size=ps, kv_heads=kv, head_dim=d, rows=rows, row_pages=pages // 2, device=DEV)
    ang = torch.arange(512, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    ones = [1 + rnd(hidden, scale=0.02) for _ in range(layers)]
    return MoeStack(moe, ones, precision="bf16", attention=attn, input_norm_weights=ones[::-1], cache=cache,
                    rope=(ang.cos().to(DEV), ang.sin().to(DEV)))


@pytest.mark.parametrize("layers", [1, 3])
def test_stack_is_its_parts(layers):
    """Prompts with padding, steps with a row that sits out, and captured steps: the same bits as the parts called by hand."""
    from kcapw_klcquant_b200 import attn_decode, attn_prompt, rope_append

    g = torch.Generator(device=DEV).manual_seed(3)
    rnd = lambda n: torch.randn(n, 256, device=DEV, generator=g).to(torch.bfloat16)  # noqa: E731
    stack, hand = make_stack(4, 40, layers=layers), make_stack(4, 40, layers=layers)

    def parts(x, attend):
        from kcapw_klcquant_b200 import rms_norm

        normed = rms_norm(x, hand.input_norm_weights[0], hand.eps)
        for li, (at, moe) in enumerate(zip(hand.attention, hand.layers)):
            x = x + at.output(attend(li, *at.project(normed)))
            nxt = (hand.input_norm_weights[li + 1], hand.eps) if li + 1 < layers else None
            x, rb = moe.forward(rms_norm(x, hand.norm_weights[li], hand.eps), precision=hand.precision, residual=x, next_norm=nxt)
            normed = rb.normed
        return x

    packed, cu, rows = rnd(65), i32([0, 19, 20, 60]), i32([2, 0, 3])
    out = stack.prompt(packed, cu, rows)
    stack.cache.check()
    assert stack.cache.lens.tolist() == [1, 0, 19, 40]
    hand.cache.reserve(i32([1, 0, 19, 40]))
    pos = torch.cat([torch.arange(n) for n in (19, 1, 40, 5)]).to(torch.int32).to(DEV)
    trow = i32([2] * 19 + [0] + [3] * 40 + [-1] * 5)

    def prompt(li, q, k, v):
        c, at = hand.cache, hand.attention[li]
        q, k = rope_append(q, k, v, *hand.rope, pos, trow, c.k(li), c.v(li), c.block_table, return_k=True)
        return attn_prompt(q, k, v, cu, window=at.window, sinks=at.sinks)

    want = parts(packed, prompt)
    assert torch.equal(out[:60], want[:60])
    live = stack.cache.refs > 0
    assert torch.equal(stack.cache.pool[:, :, live], hand.cache.pool[:, :, live])

    stack.set_active(torch.tensor([True, False, True, True], device=DEV))
    hrow, on = i32([0, -1, 2, 3]), [0, 2, 3]

    def one(x):
        before = hand.cache.lens.clone()
        hand.cache.reserve(i32([1, 0, 1, 1]))

        def attend(li, q, k, v):
            c, at = hand.cache, hand.attention[li]
            q = rope_append(q, k, v, *hand.rope, before, hrow, c.k(li), c.v(li), c.block_table)
            return attn_decode(q, c.k(li), c.v(li), c.block_table, c.lens, window=at.window, sinks=at.sinks)

        return parts(x, attend)

    xs = [rnd(4) for _ in range(30)]
    for x in xs[:2]:
        assert torch.equal(stack.step(x)[on], one(x)[on])
    before = stack.cache.lens.tolist()
    stack.capture(xs[2])
    assert stack.cache.lens.tolist() == before == [3, 0, 21, 42]
    for x in xs[2:]:  # past page ends
        assert torch.equal(stack.replay(x)[on], one(x)[on])
    stack.cache.check()
    assert stack.cache.lens.tolist() == [31, 0, 49, 70]


def test_run_together():
    """Prompt into the cache, beams forked from it, steps, a finished beam freed, the pool compacted, more steps: every output against
    the 64-bit definition over the keys the cache should hold."""
    from kcapw_klcquant_b200 import PagedKvCache, attn_decode, attn_prompt, rope_append

    H, hkv, d, ps, rows = 8, 2, 64, 16, 6
    cache = PagedKvCache(layers=1, pages=40, page_size=ps, kv_heads=hkv, head_dim=d, rows=rows, row_pages=12, device=DEV)
    ang = torch.arange(256, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    cos, sin = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
    g = torch.Generator(device=DEV).manual_seed(5)
    rnd = lambda n, h: torch.randn(n, h, d, device=DEV, generator=g).to(torch.bfloat16)  # noqa: E731
    sinks = torch.randn(H, device=DEV, generator=g)
    lens = [45, 32]
    T = sum(lens)
    q, k, v = rnd(T, H), rnd(T, hkv), rnd(T, hkv)
    cache.reserve(i32(lens + [0] * 4))
    q, k = rope_append(q, k, v, cos, sin, torch.cat([torch.arange(n) for n in lens]).to(torch.int32).to(DEV), i32([0] * 45 + [1] * 32), cache.k(0),
                       cache.v(0), cache.block_table, return_k=True)
    out = attn_prompt(q, k, v, i32([0, 45, 77]), sinks=sinks)
    held = {}
    for r, a, b in ((0, 0, 45), (1, 45, 77)):
        want, _, bound = ref.attention(q[a:b], k[a:b], v[a:b], torch.arange(b - a, device=DEV), d ** -0.5, 0, sinks)
        ref.assert_close(out[a:b], want, bound, f"prompt {r}")
        held[r] = (k[a:b], v[a:b])
    cache.fork(i32([0, 0, 1]), i32([2, 3, 4]))
    held[2], held[3], held[4] = held[0], held[0], held[1]
    groups, pre = i32([2, 4]), i32([32])  # rows 2 and 3 share row 0's full pages

    def steps(n):
        for _ in range(n):
            at = cache.lens.clone()
            live = [r for r in range(rows) if r in held]
            cache.reserve(i32([int(r in held) for r in range(rows)]))
            q, k, v = rnd(rows, H), rnd(rows, hkv), rnd(rows, hkv)
            q, k = rope_append(q, k, v, cos, sin, at, i32([r if r in held else -1 for r in range(rows)]), cache.k(0), cache.v(0),
                               cache.block_table, return_k=True)
            outs = [attn_decode(q, cache.k(0), cache.v(0), cache.block_table, cache.lens, sinks=sinks),
                    attn_decode(q, cache.k(0), cache.v(0), cache.block_table, cache.lens, sinks=sinks, group_starts=groups, prefix_lens=pre)]
            cache.check()
            for r in live:
                held[r] = (torch.cat([held[r][0], k[r:r + 1]]), torch.cat([held[r][1], v[r:r + 1]]))
                n_keys = held[r][0].shape[0]
                assert int(cache.lens[r]) == n_keys
                want, _, bound = ref.attention(q[r:r + 1], *held[r], torch.tensor([n_keys - 1], device=DEV), d ** -0.5, 0, sinks)
                for o in outs:
                    ref.assert_close(o[r:r + 1], want, bound, f"row {r}")
                    assert (o[5] == 0).all()  # an empty row

    steps(20)
    cache.free(i32([0, 4]))
    del held[0], held[4]
    n = int(cache.compact())
    assert n == int((cache.refs > 0).sum()) and (cache.refs[n:] == 0).all()
    steps(20)


def test_stack_refusals():
    from kcapw_klcquant_b200.stack import MoeStack

    stack = make_stack(2, 20, layers=1)
    kw = dict(attention=stack.attention, input_norm_weights=stack.input_norm_weights, cache=stack.cache, rope=stack.rope)
    for bad in (dict(kw, cache=None), dict(kw, rope=None), dict(kw, attention=[]), dict(kw, input_norm_weights=None), dict(kw, fuse_router=True)):
        with pytest.raises(ValueError):
            MoeStack(stack.layers, stack.norm_weights, **bad)
    x = torch.zeros(3, 256, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        stack.step(x)
    for cu, rows in ((i32([0, 3]), i32([0, 1])), (i32([0]), i32([])), (i32([0, 3]).long(), i32([0])), (i32([0, 3]), torch.zeros(1, device=DEV)),
                     (torch.tensor([0, 3], dtype=torch.int32), i32([0]))):
        with pytest.raises(ValueError):
            stack.prompt(x, cu, rows)
    from kcapw_klcquant_b200 import KlcError

    for rows in ([5], [-3], [2 ** 31 - 1]):  # rows that do not exist: reported, nothing written
        stack.prompt(x, i32([0, 3]), i32(rows))
        with pytest.raises(KlcError):
            stack.cache.check()
        assert stack.cache.lens.tolist() == [0, 0] and (stack.cache.pool == 0).all()
    with pytest.raises(RuntimeError):
        MoeStack(stack.layers, stack.norm_weights).prompt(x, i32([0, 3]), i32([0]))
