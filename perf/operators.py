"""Cases of the attention operators: prompts, single tokens over the paged cache, rotary append, cache pages.

``run`` computes each operator in plain torch (``own`` false) or through the
package's entry points (``own`` true); ``exact`` gives the outputs of the
definition in 64 bits.  Sizes follow the 64-query / 8-key head, 64-wide layout
that goes with the 2880-wide MoE layers (with a 128-key sliding window and
sinks on every second layer), and the 128-wide layout as the other common one.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _ragged(n, lo, hi, seed):
    """n lengths spread over the logarithm of [lo, hi], always the same for the same arguments."""
    rng = random.Random(seed)
    return [max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))) for _ in range(n)]


def listed():
    prompt = {"op": "prompt", "dtype": "bf16", "heads": 64, "kv_heads": 8, "dim": 64, "window": 0, "sinks": True}
    decode = {"op": "decode", "dtype": "bf16", "heads": 64, "kv_heads": 8, "dim": 64, "window": 0, "sinks": True,
              "page": 64, "prefix": 0}
    rope = {"op": "rope", "dtype": "bf16", "heads": 64, "kv_heads": 8, "dim": 64, "page": 64}
    return [
        # one short question: a latency case, less than one tile of keys
        dict(prompt, name="prompt_short", n=1, lo=37, hi=37, cached_lo=1, cached_hi=1, cached=False, seed=0),
        # a batch of prompts of mixed lengths in a sliding-window layer
        dict(prompt, name="prompt_window", n=12, lo=90, hi=2200, window=128, cached_lo=1, cached_hi=1, cached=False, seed=1),
        # chunks of prompts whose earlier chunks are already there (more keys than queries), half precision
        dict(prompt, name="prompt_chunk", dtype="f16", n=4, lo=700, hi=2048, cached_lo=300, cached_hi=6000, cached=True, seed=2),
        # one long document, 128-wide heads, odd length
        dict(prompt, name="prompt_long", heads=32, dim=128, sinks=False, n=1, lo=16221, hi=16221, cached_lo=1, cached_hi=1,
             cached=False, seed=3),
        # one user's chat turn: a latency case
        dict(decode, name="decode_one", n=1, lo=777, hi=777, seed=4),
        # the batched decode step: 32 sequences of mixed lengths
        dict(decode, name="decode_batch", n=32, lo=100, hi=9000, seed=5),
        # two very long contexts, 128-wide heads, small pages, half precision
        dict(decode, name="decode_long", dtype="f16", heads=32, dim=128, sinks=False, page=16, n=2, lo=90000, hi=131000, seed=6),
        # 64 requests behind one long system prompt
        dict(decode, name="decode_prefix", n=64, lo=5, hi=700, prefix=16384, seed=7),
        # the decode step's rotary embedding and cache write
        dict(rope, name="rope_step", n=32, lo=1, hi=1, max_pos=131072, seed=8),
        # the same for a batch of whole prompts
        dict(rope, name="rope_prompt", n=9, lo=300, hi=2500, max_pos=16384, seed=9),
        # beam search: children of a few parents share their pages (the partial last page is copied), then one token each
        {"name": "pages_fork", "op": "pages", "do": "fork", "dtype": "bf16", "layers": 8, "pages": 700, "page": 64, "kv_heads": 8,
         "dim": 64, "rows": 48, "n": 6, "children": 5, "lo": 200, "hi": 4000, "seed": 10},
        # finished sequences leave holes: free them, then move the live pages to the front
        {"name": "pages_compact", "op": "pages", "do": "compact", "dtype": "bf16", "layers": 8, "pages": 900, "page": 64,
         "kv_heads": 8, "dim": 64, "rows": 40, "n": 40, "children": 0, "lo": 300, "hi": 2500, "seed": 11},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    seed = rng.randrange(1 << 30)
    dtype = rng.choice(["bf16", "f16"])
    op = rng.choice(["prompt", "prompt", "decode", "decode", "rope", "pages"])
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 6, 8])
    heads = min(heads, 64 if dim == 64 else 32) // kv * kv
    if op == "prompt":
        n = _log_int(rng, 1, 24)
        hi = _log_int(rng, 2, max(2, min(12000, 24000 // n)))
        cached = rng.random() < 0.3
        return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv, "dim": dim, "window": rng.choice([0, 0, 1, 100, 128, 1000]),
                "sinks": rng.random() < 0.5, "n": n, "lo": max(1, hi // rng.choice([1, 4, 30])), "hi": hi, "cached": cached,
                "cached_lo": 1, "cached_hi": _log_int(rng, 1, 4000), "seed": seed}
    if op == "decode":
        n = _log_int(rng, 1, 96)
        hi = _log_int(rng, 1, max(2, min(60000, 300000 // n)))
        prefix = rng.choice([0, 0, 1]) * _log_int(rng, 1, 128) * 128
        return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv, "dim": dim, "window": rng.choice([0, 0, 0, 128, 5000]),
                "sinks": rng.random() < 0.5, "page": rng.choice([16, 32, 64, 128]), "prefix": prefix, "n": n,
                "lo": max(1, hi // rng.choice([1, 5, 50])), "hi": hi, "seed": seed}
    if op == "rope":
        n = _log_int(rng, 1, 32)
        hi = _log_int(rng, 1, 4000)
        return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv, "dim": dim, "page": rng.choice([16, 32, 64, 128]),
                "n": n, "lo": max(1, hi // 5), "hi": hi, "max_pos": rng.choice([8192, 131072]), "seed": seed}
    page = rng.choice([16, 32, 64, 128])
    pages = _log_int(rng, 120, 900)
    do = rng.choice(["fork", "clone", "compact"])
    n = rng.randint(2, 8)
    hi = max(2, pages * page // (4 * n))
    return {"op": op, "do": do, "dtype": dtype, "layers": rng.randint(1, 8), "pages": pages, "page": page, "kv_heads": kv, "dim": dim,
            "rows": 48, "n": n, "children": rng.randint(1, 2), "lo": max(1, hi // 10), "hi": hi, "seed": seed}


# ---- sizes ---------------------------------------------------------------


def _lens(case):
    lens = _ragged(case["n"], case["lo"], case["hi"], case["seed"])
    if case["op"] == "prompt":
        extra = _ragged(case["n"], case["cached_lo"], case["cached_hi"], case["seed"] + 1) if case["cached"] else [0] * case["n"]
        return lens, [a + b for a, b in zip(lens, extra)]
    return lens


def _cum(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _visible(first, last, window):
    """Sum over positions first..last (inclusive, 0-based) of the keys each sees."""
    if last < first:
        return 0
    if window <= 0:
        return (first + 1 + last + 1) * (last - first + 1) // 2
    full = max(first, window - 1)  # from here on every position sees `window` keys
    part = _visible(first, min(last, full - 1), 0)
    return part + max(0, last - full + 1) * window


def work(case):
    if case["op"] == "prompt":
        lq, lk = _lens(case)
        vis = sum(_visible(k - q, k - 1, case["window"]) for q, k in zip(lq, lk))
        byt = 2 * case["dim"] * (2 * sum(lq) * case["heads"] + 2 * sum(lk) * case["kv_heads"])
        return {"bytes": byt, "flops": 4 * case["dim"] * case["heads"] * vis}
    if case["op"] == "decode":
        w, pre = case["window"], case["prefix"]
        keys, vis, low = 0, 0, pre
        for t in _lens(case):
            n = pre + t
            lo = max(0, n - w) if w > 0 else 0
            vis += n - lo
            keys += n - max(lo, pre)
            low = min(low, lo)
        keys += pre - low
        byt = 2 * case["dim"] * (2 * keys * case["kv_heads"] + 2 * case["n"] * case["heads"])
        return {"bytes": byt, "flops": 4 * case["dim"] * case["heads"] * vis}
    if case["op"] == "rope":
        t = sum(_lens(case))
        d = case["dim"]
        return {"bytes": t * (2 * d * (2 * case["heads"] + 4 * case["kv_heads"]) + 4 * d), "flops": 3 * t * d * (case["heads"] + case["kv_heads"])}
    page_bytes = 2 * case["layers"] * 2 * case["kv_heads"] * case["page"] * case["dim"]
    return {"bytes": 2 * page_bytes * max(1, _moved_pages(case)), "flops": 0}


# ---- cache tables --------------------------------------------------------


def _ceil(a, b):
    return -(-a // b)


def _scattered(total, seed):
    ids = list(range(total))
    random.Random(seed).shuffle(ids)
    return ids


def _page_layout(case):
    """Rows' lengths and page lists of a pages case: the pages of the pool handed out in a scattered order."""
    lens = _lens(case)
    ids = _scattered(case["pages"], case["seed"] + 2)
    budget = case["pages"] * (1 if case["do"] == "compact" else 0.45)
    out_lens, tables, used = [], [], 0
    for n in lens:
        need = _ceil(n, case["page"])
        if used + need > budget:
            n, need = 0, 0
        tables.append(ids[used:used + need])
        out_lens.append(n)
        used += need
    return out_lens, tables


def _moved_pages(case):
    lens, tables = _page_layout(case)
    if case["do"] == "fork":
        return case["children"] * sum(1 for n in lens if n % case["page"])
    if case["do"] == "clone":
        return sum(len(t) for t in tables)
    live = [p for i, t in enumerate(tables) if i % 2 for p in t]
    return sum(1 for p in live if p >= len(live))


def _fork_lists(case):
    n, c = case["n"], (case["children"] if case["do"] == "fork" else 1)
    parents = [i for i in range(n) for _ in range(c)]
    return parents, [n + j for j in range(n * c)]


# ---- inputs --------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)


def _randn(shape, dtype, gen):
    return torch.randn(shape, device="cuda", dtype=torch.float32, generator=gen).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    dt = _DTYPES[case["dtype"]]
    g = _gen(seed)
    st = {"case": case}
    d, hkv = case["dim"], case["kv_heads"]
    if case["op"] == "prompt":
        lq, lk = _lens(case)
        # q, k and v are slices of one projection when no earlier chunk is there, as a layer has them
        h = case["heads"]
        if case["cached"]:
            st["q"] = _randn((sum(lq), h, d), dt, g)
            st["k"], st["v"] = (_randn((sum(lk), hkv, d), dt, g) for _ in range(2))
        else:
            qkv = _randn((sum(lq), h + 2 * hkv, d), dt, g)
            st["q"], st["k"], st["v"] = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
        st["lq"], st["lk"] = lq, lk
        st["cu_q"], st["cu_k"] = _i32(_cum(lq)), _i32(_cum(lk))
        st["sinks"] = torch.randn(h, device="cuda", generator=g) if case["sinks"] else None
        return st
    if case["op"] == "decode":
        ps, pre, tails = case["page"], case["prefix"], _lens(case)
        n = len(tails)
        shared = pre // ps
        need = [_ceil(t, ps) for t in tails]
        total = shared + sum(need) + 3
        ids = _scattered(total, case["seed"] + 3)
        width = shared + max(need)
        table, at = [], shared
        for m in need:
            table.append(ids[:shared] + ids[at:at + m] + [-1] * (width - shared - m))
            at += m
        st["q"] = _randn((n, case["heads"], d), dt, g)
        st["k"], st["v"] = (_randn((total, hkv, ps, d), dt, g) for _ in range(2))
        st["table"], st["lens"] = _i32(table), _i32([pre + t for t in tails])
        st["host_lens"] = [pre + t for t in tails]
        st["sinks"] = torch.randn(case["heads"], device="cuda", generator=g) if case["sinks"] else None
        st["groups"] = _i32([0, n]) if pre else None
        st["prefix_lens"] = _i32([pre]) if pre else None
        return st
    if case["op"] == "rope":
        ps, lens = case["page"], _lens(case)
        rng = random.Random(case["seed"] + 6)
        start = [rng.randrange(0, case["max_pos"] - n + 1) for n in lens]
        width = _ceil(case["max_pos"], ps)
        used = [(s // ps, (s + n - 1) // ps) for s, n in zip(start, lens)]
        ids = _scattered(sum(b - a + 1 for a, b in used), case["seed"] + 4)
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for i, (a, b) in enumerate(used):
            table[i, a:b + 1] = torch.tensor(ids[at:at + b - a + 1], dtype=torch.int32)
            at += b - a + 1
        t, h = sum(lens), case["heads"]
        qkv = _randn((t, h + 2 * hkv, d), dt, g)
        st["q"], st["k"], st["v"] = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
        st["kp"], st["vp"] = (torch.zeros((len(ids), hkv, ps, d), dtype=dt, device="cuda") for _ in range(2))
        st["table"] = table.cuda()
        st["pos"] = _i32([s + j for s, n in zip(start, lens) for j in range(n)])
        st["rows"] = _i32([i for i, n in enumerate(lens) for _ in range(n)])
        inv = 150000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        ang = torch.arange(case["max_pos"], dtype=torch.float64)[:, None] * inv
        st["cos"], st["sin"] = torch.cos(ang).float().cuda(), torch.sin(ang).float().cuda()
        return st
    lens, tables = _page_layout(case)
    rows = case["rows"]
    width = max(1, max(len(t) for t in tables) + 1)
    table = [t + [-1] * (width - len(t)) for t in tables] + [[-1] * width for _ in range(rows - len(tables))]
    refs = [0] * case["pages"]
    for t in tables:
        for p in t:
            refs[p] = 1
    shape = (case["layers"], 2, case["pages"], hkv, case["page"], d)
    if own:
        from kcapw_klcquant_b200 import PagedKvCache

        cache = PagedKvCache(layers=case["layers"], pages=case["pages"], page_size=case["page"], kv_heads=hkv, head_dim=d, rows=rows,
                             row_pages=width, dtype=dt, device="cuda")
        st["cache"] = cache
        st["pool"], st["table"], st["lens"], st["refs"] = cache.pool, cache.block_table, cache.lens, cache.refs
    else:
        st["pool"] = torch.empty(shape, dtype=dt, device="cuda")
        st["table"], st["lens"], st["refs"] = (torch.empty(s, dtype=torch.int32, device="cuda")
                                               for s in ((rows, width), (rows,), (case["pages"],)))
    for layer in range(case["layers"]):
        st["pool"][layer].copy_(_randn(shape[1:], dt, g))
    # the state before the step; every pass starts from it again
    st["table0"], st["lens0"], st["refs0"] = _i32(table), _i32(lens + [0] * (rows - len(lens))), _i32(refs)
    if case["do"] == "compact":
        st["finished"] = _i32(list(range(0, len(lens), 2)))
    else:
        parents, children = _fork_lists(case)
        st["parents"], st["children"] = _i32(parents), _i32(children)
        add = [0] * rows
        for c in children:
            add[c] = 1
        st["add"] = _i32(add)
    return st


# ---- one pass ------------------------------------------------------------


def run(st):
    op = st["case"]["op"]
    if op == "prompt":
        return _run_prompt(st)
    if op == "decode":
        return _run_decode(st)
    if op == "rope":
        return _run_rope(st)
    return _run_pages(st)


def _softmax_rows(s, sink):
    """Softmax numerators, denominators and row maxima of s fp32 [..., H, q, k] with an optional sink per head."""
    m = s.amax(-1, keepdim=True)
    if sink is not None:
        m = torch.maximum(m, sink[:, None, None])
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    den = p.sum(-1, keepdim=True)
    if sink is not None:
        den = den + torch.exp(sink[:, None, None] - m)
    return p, den


def _plain_attention(q, k, v, first, scale, window, sink):
    """q [n, H, D] at positions first.. over k, v [m, Hkv, D], in the inputs' type; rows in blocks that fit in memory."""
    n, h, d = q.shape
    m, hkv = k.shape[0], k.shape[1]
    grp = h // hkv
    kt = k.permute(1, 2, 0)  # [Hkv, D, m]
    vt = v.permute(1, 0, 2)
    out = torch.empty_like(q)
    step = max(1, min(n, (1 << 28) // max(1, h * m)))
    for a in range(0, n, step):
        b = min(n, a + step)
        hi = min(m, first + b)
        lo = max(0, first + a - window + 1) if window > 0 else 0
        qs = q[a:b].permute(1, 0, 2).reshape(hkv, grp * (b - a), d)
        s = torch.matmul(qs, kt[:, :, lo:hi]).view(h, b - a, hi - lo) * scale
        pos = torch.arange(first + a, first + b, device=q.device)[:, None]
        key = torch.arange(lo, hi, device=q.device)[None, :]
        hidden = key > pos
        if window > 0:
            hidden |= key <= pos - window
        s.masked_fill_(hidden, float("-inf"))
        p, den = _softmax_rows(s, sink)
        o = torch.matmul(p.view(hkv, grp * (b - a), hi - lo), vt[:, lo:hi]).view(h, b - a, d)
        out[a:b] = (o / den).permute(1, 0, 2)
    return out


def _run_prompt(st):
    c = st["case"]
    if own:
        from kcapw_klcquant_b200 import attn_prompt

        return attn_prompt(st["q"], st["k"], st["v"], st["cu_q"], cu_seqlens_k=st["cu_k"] if c["cached"] else None, window=c["window"],
                           sinks=st["sinks"])
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    out, aq, ak = [], 0, 0
    for n, m in zip(st["lq"], st["lk"]):
        out.append(_plain_attention(q[aq:aq + n], k[ak:ak + m], v[ak:ak + m], m - n, c["dim"] ** -0.5, c["window"], st["sinks"]))
        aq, ak = aq + n, ak + m
    return torch.cat(out).to(st["q"].dtype)


def _gather(pages, table_row, n):
    """The first n rows [n, Hkv, D] of a sequence from its pages."""
    hkv, ps, d = pages.shape[1:]
    got = pages[table_row[:_ceil(n, ps)].long()]
    return got.permute(0, 2, 1, 3).reshape(-1, hkv, d)[:n]


def _run_decode(st):
    c = st["case"]
    if own:
        from kcapw_klcquant_b200 import attn_decode

        return attn_decode(st["q"], st["k"], st["v"], st["table"], st["lens"], window=c["window"], sinks=st["sinks"],
                           group_starts=st["groups"], prefix_lens=st["prefix_lens"])
    out = []
    for i, n in enumerate(st["host_lens"]):
        k, v = _gather(st["k"], st["table"][i], n).float(), _gather(st["v"], st["table"][i], n).float()
        out.append(_plain_attention(st["q"][i:i + 1].float(), k, v, n - 1, c["dim"] ** -0.5, c["window"], st["sinks"]))
    return torch.cat(out).to(st["q"].dtype)


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _run_rope(st):
    if own:
        from kcapw_klcquant_b200 import rope_append

        q = rope_append(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["pos"], st["rows"], st["kp"], st["vp"], st["table"])
        return q, st["kp"], st["vp"]
    pos = st["pos"].long()
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    dt, ps = st["q"].dtype, st["kp"].shape[2]
    q = _rotate(st["q"].float(), cos, sin).to(dt)
    k = _rotate(st["k"].float(), cos, sin).to(dt)
    page = st["table"][st["rows"].long(), pos // ps].long()
    st["kp"][page, :, pos % ps] = k
    st["vp"][page, :, pos % ps] = st["v"]
    return q, st["kp"], st["vp"]


def _free_ids(refs):
    return torch.argsort((refs > 0).to(torch.int8), stable=True)


def _plain_fork(st, share):
    ps = st["case"]["page"]
    par, chi = st["parents"].long(), st["children"].long()
    table, lens, refs, pool = st["table"], st["lens"], st["refs"], st["pool"]
    n = lens[par].long()
    slot = torch.arange(table.shape[1], device="cuda")[None, :]
    held = slot < ((n + ps - 1) // ps)[:, None]
    fresh = held & (slot >= (n // ps)[:, None]) if share else held  # pages of the child's own
    order = (torch.cumsum(fresh.flatten().long(), 0) - 1).view_as(fresh)
    src = table[par]
    new = torch.where(fresh, _free_ids(refs)[order.clamp(min=0)].to(torch.int32), src)
    table[chi] = torch.where(held, new, torch.full_like(new, -1))
    lens[chi] = lens[par]
    refs.index_add_(0, new[held].long(), torch.ones_like(new[held]))
    pool[:, :, new[fresh].long()] = pool[:, :, src[fresh].long()]


def _plain_reserve(st, add):
    ps = st["case"]["page"]
    table, lens, refs = st["table"], st["lens"], st["refs"]
    slot = torch.arange(table.shape[1], device="cuda")[None, :]
    have, want = (lens + ps - 1) // ps, (lens + add + ps - 1) // ps
    fresh = (slot >= have[:, None]) & (slot < want[:, None])
    order = (torch.cumsum(fresh.flatten().long(), 0) - 1).view_as(fresh)
    new = _free_ids(refs)[order.clamp(min=0)].to(torch.int32)
    refs[new[fresh].long()] = 1
    table[fresh] = new[fresh]
    lens += add


def _plain_free(st, rows):
    rows = rows.long()
    table, refs = st["table"], st["refs"]
    gone = table[rows]
    gone = gone[gone >= 0]
    refs.index_add_(0, gone.long(), torch.full_like(gone, -1))
    table[rows] = -1
    st["lens"][rows] = 0


def _plain_compact(st):
    table, refs, pool = st["table"], st["refs"], st["pool"]
    live = refs > 0
    n = live.sum()
    ids = torch.arange(refs.numel(), device="cuda")
    dst, src = ids[~live & (ids < n)], ids[live & (ids >= n)]
    pool[:, :, dst] = pool[:, :, src]
    to = ids.clone()
    to[src] = dst
    st["table"].copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table))
    refs[dst] = refs[src]
    refs[src] = 0


def _run_pages(st):
    do = st["case"]["do"]
    for a, b in (("table", "table0"), ("lens", "lens0"), ("refs", "refs0")):
        st[a].copy_(st[b])
    if own:
        cache = st["cache"]
        if do == "compact":
            cache.free(st["finished"])
            cache.compact()
        else:
            cache.fork(st["parents"], st["children"], copy=do == "clone")
            cache.reserve(st["add"])
    elif do == "compact":
        _plain_free(st, st["finished"])
        _plain_compact(st)
    else:
        _plain_fork(st, share=do == "fork")
        _plain_reserve(st, st["add"])
    return st["table"], st["lens"], st["refs"], st["pool"]


# ---- the definition in 64 bits -------------------------------------------


def _exact_row_block(q, k, v, pos, scale, window, sink):
    """Attention of q [r, D] at positions pos over one key head's k, v [m, D], all float64, by sorted-key sums of exp."""
    logits = (q @ k.T) * scale
    key = torch.arange(k.shape[0], device=q.device)
    seen = (key[None] <= pos[:, None]) & ((key[None] > pos[:, None] - window) if window > 0 else True)
    logits = torch.where(seen, logits, torch.full_like(logits, -math.inf))
    if sink is not None:
        logits = torch.cat([logits, sink[:, None]], 1)
    lse = torch.logsumexp(logits, 1, keepdim=True)
    w = torch.exp(logits - lse)[:, :k.shape[0]]
    return torch.nan_to_num(w, nan=0.0) @ v


def _exact_attention(q, k, v, first, scale, window, sinks):
    n, h, d = q.shape
    grp = h // k.shape[1]
    out = torch.empty(n, h, d, dtype=torch.float64, device=q.device)
    kd, vd = k.double(), v.double()
    step = max(1, min(n, (1 << 26) // max(1, k.shape[0])))
    for head in range(h):
        kh, vh = kd[:, head // grp].contiguous(), vd[:, head // grp].contiguous()
        for a in range(0, n, step):
            b = min(n, a + step)
            hi = min(k.shape[0], first + b)
            pos = torch.arange(first + a, first + b, device=q.device)
            sink = None if sinks is None else sinks[head].double().expand(b - a)
            out[a:b, head] = _exact_row_block(q[a:b, head].double(), kh[:hi], vh[:hi], pos, scale, window, sink)
    return out


def exact(case, seed):
    if case["op"] == "pages":
        return None
    st = prepare(case, seed)
    scale = 1.0 / math.sqrt(case["dim"])
    if case["op"] == "prompt":
        parts, aq, ak = [], 0, 0
        for n, m in zip(st["lq"], st["lk"]):
            parts.append(_exact_attention(st["q"][aq:aq + n], st["k"][ak:ak + m], st["v"][ak:ak + m], m - n, scale, case["window"], st["sinks"]))
            aq, ak = aq + n, ak + m
        return torch.cat(parts)
    if case["op"] == "decode":
        parts = []
        for i, n in enumerate(st["host_lens"]):
            flat = torch.arange(n, device="cuda")
            page = st["table"][i].long()[flat // case["page"]]
            k, v = st["k"][page, :, flat % case["page"]], st["v"][page, :, flat % case["page"]]
            parts.append(_exact_attention(st["q"][i:i + 1], k, v, n - 1, scale, case["window"], st["sinks"]))
        return torch.cat(parts)
    pos = st["pos"].long()
    half = case["dim"] // 2
    c, s = st["cos"].double()[pos], st["sin"].double()[pos]

    def turn(x):
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * torch.complex(c, s)[:, None]
        return torch.cat([z.real, z.imag], -1)

    kp, vp = st["kp"].double(), st["vp"].double()
    where = st["table"].long()[st["rows"].long(), pos // case["page"]]
    kp[where, :, pos % case["page"]] = turn(st["k"])
    vp[where, :, pos % case["page"]] = st["v"].double()
    return turn(st["q"]), kp, vp
