"""Workloads of the operators around the INT2 attention of forked requests, for timing and
comparison: what a serving engine runs when it samples several continuations of one prompt.

A case is one call (or one step's calls) of one operator:

* ``qk``: norms of the queries and keys of each head and the position rotation in one pass, from
  rows inside the projection's output; optionally the rotation by R_k that the INT2 history wants
  (decode and chunk steps; a prefill does not need it).
* ``fork``: the free pages of the pool, then requests that continue a parent's tokens: whole pages
  shared, the first page (which holds the BF16 window) and an unfinished last page copied, in
  every layer's cache.
* ``compact``: live pages moved to the pool's start in every layer's cache, and the block tables
  that follow them.
* ``shared``: history attention of a batch whose requests share a long prefix, one step: the plan
  of the step, then every layer's attention.

Lengths and page ownership come from the case alone; rows, records and weights from the seed.
Records are Gaussian rows in the rotated basis, clipped at the default configuration's 96 % and
92 % quantiles; queries are scaled so that scores spread by about two nats. Head sizes, pages and
windows are the defaults of the package; batches and lengths those of ``bench.py`` (32 x 32768,
2048-token chunk, 4 x 4096 prefill) and generic ones around them.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DIM, PAGE, BLOCK, SLOT = 256, 768, 128, 160
PER = PAGE // BLOCK
DEV = "cuda"
EPS = 1e-6


# ------------------------------------------------------------------ the cases


def _qk(name, **over):
    case = dict(kind="qk", tokens=32, live=0, group=6, kv_heads=1, rotary=64, positions=32768,
                interleaved=False, unit_offset=True, rotate=True, fp32=False)
    case.update(over)
    case["live"] = case["live"] or case["tokens"]
    return dict(case, name=name) if name else case


def _cache(kind, name, **over):
    case = dict(kind=kind, requests=1, low=700, context=700, children=1, layers=4, kv_heads=1,
                sink=64, recent=256, spec=3, spare=0)
    case.update(over)
    return dict(case, name=name) if name else case


def _shared(name, **over):
    case = dict(kind="shared", groups=1, members=6, prefix=2000, low=300, tail=900, qlen=1, layers=4,
                group=6, kv_heads=1, sink=64, recent=256, spec=3)
    case.update(over)
    return dict(case, name=name) if name else case


def listed():
    return [
        # A decode batch on one tensor-parallel rank, queries rotated for the history in the call.
        _qk("qk 32 decode", tokens=32),
        # A prompt's chunk, two KV heads on the rank, a graph's padding behind the last token.
        _qk("qk 2048 chunk", tokens=2048, live=2041, kv_heads=2),
        # Prompts that arrive together: 4 x 4096 tokens, no history and so no rotation by R_k.
        _qk("qk 16384 prefill", tokens=16384, rotate=False),
        # One short conversation forked once: launches and latency.
        _cache("fork", "fork 1 short", layers=4),
        # Eight samples of one long prompt, all full-attention layers of a deep model.
        _cache("fork", "fork 1 to 8", low=32768, context=32768, children=8, layers=16),
        # A beam step of many users, ragged lengths.
        _cache("fork", "fork 48 ragged", requests=48, low=90, context=9001, children=2, layers=6),
        # A small server's pool after a few conversations have ended.
        _cache("compact", "compact 5 short", requests=5, low=300, context=3000, layers=4, spare=12),
        # A pool with holes after many requests have ended.
        _cache("compact", "compact 24", requests=24, low=500, context=14000, layers=8, spare=100),
        # A few samples of a short prompt.
        _shared("shared 6x2k", prefix=2000),
        # The headline decode batch as samples of one prompt.
        _shared("shared 32x32k", members=32, prefix=32000, tail=1500, sink=4, recent=128),
        # MTP verification of three prompts' samples, 4 query tokens each.
        _shared("shared mtp 3x9", groups=3, members=9, prefix=9011, tail=2000, qlen=4, layers=2),
        # A large agent batch over one long context.
        _shared("shared 256x32k", members=256, prefix=32500, tail=1200, layers=2, sink=4, recent=128),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["qk", "qk", "fork", "compact", "shared", "shared"])
    if kind == "qk":
        heads = rng.choice([1, 1, 2, 4])
        tokens = _log(rng, 1, 16384 // heads)
        return _qk("", tokens=tokens, live=tokens - (rng.randrange(tokens) // 8), kv_heads=heads,
                   group=rng.choice([1, 4, 5, 6, 6, 8]) if tokens < 8000 // heads else 4,
                   rotary=rng.choice([32, 64, 64, 96, 128, 256]),
                   positions=_log(rng, 512, 131072), interleaved=rng.random() < 0.3,
                   unit_offset=rng.random() < 0.5, rotate=rng.random() < 0.6,
                   fp32=rng.random() < 0.4)
    short = rng.random() < 0.4
    over = dict(kv_heads=rng.choice([1, 1, 1, 2]), sink=4 if short else 64,
                recent=128 if short else 256)
    if kind == "fork":
        requests = _log(rng, 1, 16)
        return _cache("fork", "", requests=requests, low=rng.choice([3, 70, 700]),
                      context=_log(rng, 701, 32768), layers=rng.choice([1, 3, 6]),
                      children=rng.choice([1, 2]) if requests > 6 else rng.choice([1, 2, 5]),
                      **over)
    if kind == "compact":
        requests = _log(rng, 1, 24)
        return _cache("compact", "", requests=requests, low=rng.choice([3, 70, 700]),
                      context=_log(rng, 701, 14000), layers=rng.choice([1, 2, 4]),
                      spare=_log(rng, 4, 100), **over)
    groups = rng.choice([1, 1, 2, 3])
    qlen = rng.choice([1, 1, 2, 3, 4])
    heads = over["kv_heads"]
    members = _log(rng, 2, 192 // (groups * qlen * heads))
    group = rng.choice([4, 5, 6, 6, 6, 8])
    most = 256 * 32000 * 6 // (groups * members * qlen * heads * group)
    prefix = _log(rng, 300, min(131072, most))
    return _shared("", groups=groups, members=members, prefix=prefix, qlen=qlen,
                   low=rng.choice([qlen, 150, 400]), tail=_log(rng, 401, 2000),
                   layers=rng.choice([1, 2]), group=group, **over)


def _spread(n, low, high):
    """n lengths spread over the logarithm from low to high, in a scattered order."""
    lengths = [int(round(low * (high / low) ** ((i + 0.5) / n))) for i in range(n)]
    return [lengths[i * 7 % n] if n % 7 else lengths[i] for i in range(n)]


def _pages(tokens):
    return -(-tokens // PAGE)


def _history(case, length):
    """History positions [begin, end) of a request of ``length`` tokens in this step."""
    prefix = length - case["qlen"]
    begin = min(case["sink"], prefix)
    return begin, max(begin, prefix - case["recent"])


def _shared_end(case, lengths):
    """End of the history positions that every member of a group shares."""
    return min([case["prefix"]] + [_history(case, n)[1] for n in lengths])


def _copied(case, length):
    """Bytes of one layer that a fork of a request of ``length`` tokens copies."""
    heads = case["kv_heads"]
    ring = case["recent"] + case["spec"] + 1
    slots = min(length, PAGE)
    if length > PAGE and length % PAGE:
        slots += length % PAGE
    return heads * (slots * SLOT + min(length, case["sink"] + ring) * 2 * DIM * 2)


def work(case):
    """What a pass cannot do without. ``qk``: each row read and written once (twice where it is
    rotated as well), the angles, R_k. ``fork``: each parent's copied rows read once, each child's
    written. ``compact``: each moved row read and written. ``shared``: 136 bytes per record read
    once (the shared ones once a group), queries, outputs and LSE; 4 operations per query row,
    visible key and dim."""
    if case["kind"] == "qk":
        n, hq, hk = case["live"], case["group"] * case["kv_heads"], case["kv_heads"]
        total = n * (hq + hk) * 1024 + n * (case["rotary"] * (4 if case["fp32"] else 2) + 8)
        total += (case["tokens"] - n) * (hq + hk) * 512
        flops = n * (hq + hk) * DIM * 6
        if case["rotate"]:
            total += case["tokens"] * hq * 512 + 2 * DIM * DIM
            flops += n * hq * 2 * DIM * DIM
        return {"bytes": total, "flops": flops}
    if case["kind"] == "fork":
        per = sum(_copied(case, n) for n in _spread(case["requests"], case["low"], case["context"]))
        return {"bytes": case["layers"] * per * (1 + case["children"]), "flops": 0}
    if case["kind"] == "compact":
        world, moved = _compact_world(case), {}
        ring = case["recent"] + case["spec"] + 1
        live = len({p for row in world.owned for p in row})
        for length, row in zip(world.lengths, world.owned):
            for j, page in enumerate(row):
                if page >= live:
                    moved[page] = min(PAGE, length - j * PAGE) * SLOT
                    moved[page] += min(length, case["sink"] + ring) * 1024 if j == 0 else 0
        total = sum(moved.values())
        return {"bytes": 2 * case["layers"] * case["kv_heads"] * total, "flops": 0}
    rows = case["group"] * case["kv_heads"]
    records = visible = 0
    for lengths in _shared_lengths(case):
        end = _shared_end(case, lengths)
        records += max(0, end - case["sink"])
        for n in lengths:
            begin, stop = _history(case, n)
            records += stop - max(begin, end)
            visible += (stop - begin) * case["qlen"]
    n = case["groups"] * case["members"] * case["qlen"]
    return {"bytes": case["layers"] * (136 * records * case["kv_heads"] + n * rows * (1024 + 4)),
            "flops": case["layers"] * 4 * DIM * rows * visible}


# ------------------------------------------------------------------ inputs


def _records(n, gen):
    """[n, 160] uint8 records of Gaussian rows: 2-bit codes, fp16 scale and zero, of K, then V."""
    out = torch.zeros(n, SLOT, dtype=torch.uint8, device=DEV)
    for at, clip in ((0, 2.05), (68, 1.75)):
        x = torch.randn(n, DIM, generator=gen, device=DEV)
        x.clamp_(-clip, clip)
        low = x.amin(1, keepdim=True)
        scale = ((x.amax(1, keepdim=True) - low) / 3).half()
        low = low.half()
        x.sub_(low.float()).div_(scale.float()).round_().clamp_(0, 3)
        codes = x.to(torch.uint8).view(n, DIM // 4, 4)
        out[:, at : at + 64] = (codes[..., 0] | codes[..., 1] << 2 | codes[..., 2] << 4
                                | codes[..., 3] << 6)
        out[:, at + 64 : at + 68] = torch.cat([scale, low], 1).view(torch.uint8)
    return out


def _layout(case):
    from oscar_new_amd.config import OscarConfig
    from oscar_new_amd.layout import CacheLayout

    config = OscarConfig(sink_tokens=case["sink"], recent_tokens=case["recent"],
                         speculative_tokens=case["spec"])
    return CacheLayout(PAGE, kv_heads=case["kv_heads"], config=config)


def _shuffle(items, salt):
    """A fixed scattered order of ``items`` (no random state: ownership belongs to the case)."""
    return sorted(items, key=lambda i: (i * 2654435761 + salt * 40503) % 4294967291)


def _table(rows, requests, columns):
    table = torch.full((requests, columns), -1, dtype=torch.int32)
    for r, own_pages in enumerate(rows):
        blocks = [p * PER + b for p in own_pages for b in range(PER)]
        table[r, : len(blocks)] = torch.tensor(blocks, dtype=torch.int32)
    return table


def _qk_inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    n, hk = case["tokens"], case["kv_heads"]
    hq = hk * case["group"]
    # One projection row per token: [query, gate] of each query head, then keys, then values.
    packed = torch.randn(n, (2 * hq + 2 * hk) * DIM, generator=gen, device=DEV)
    packed *= torch.rand(n, 1, generator=gen, device=DEV) * 3 + 0.2
    packed = packed.bfloat16()
    query = packed[:, : 2 * hq * DIM].view(n, hq, 2 * DIM)[..., :DIM]
    key = packed[:, 2 * hq * DIM : (2 * hq + hk) * DIM].view(n, hk, DIM)
    half = case["rotary"] // 2
    rate = 1e7 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    angle = torch.arange(case["positions"], device=DEV, dtype=torch.float64)[:, None] * rate
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1)
    cos_sin = cos_sin.float() if case["fp32"] else cos_sin.bfloat16()
    positions = torch.randint(case["positions"], (n,), generator=gen, device=DEV)
    weights = [0.3 * torch.randn(DIM, generator=gen, device=DEV) + (0 if case["unit_offset"] else 1)
               for _ in range(2)]
    if not case["fp32"]:
        weights = [w.bfloat16() for w in weights]
    rk = torch.linalg.qr(torch.randn(DIM, DIM, generator=gen, device=DEV))[0].bfloat16()
    counts = torch.tensor([1, case["live"]], dtype=torch.int32, device=DEV)
    return SimpleNamespace(case=case, query=query, key=key, weights=weights, cos_sin=cos_sin,
                           positions=positions, rk_t=rk.T.contiguous(), counts=counts)


def _fork_world(case):
    """Pages of the parents (none shared), the pool's size and the parent of each child."""
    lengths = _spread(case["requests"], case["low"], case["context"])
    need = sum(_pages(n) for n in lengths)
    children = case["requests"] * case["children"]
    pool = need + need // 6 + 2 * children + 2
    order = _shuffle(range(1, pool), 3)
    owned, at = [], 0
    for n in lengths:
        owned.append(order[at : at + _pages(n)])
        at += _pages(n)
    return SimpleNamespace(lengths=lengths, owned=owned, pool=pool, children=children,
                           parents=[i // case["children"] for i in range(children)])


def _compact_world(case):
    """Requests whose pages lie anywhere in the pool; every third one shares the inner pages of
    the one before, as forked requests do."""
    lengths = _spread(case["requests"], case["low"], case["context"])
    shared = [i % 3 == 2 for i in range(len(lengths))]
    for i, s in enumerate(shared):
        lengths[i] = lengths[i - 1] if s else lengths[i]
    pool = sum(_pages(n) for n in lengths) + case["spare"] + 1
    order = _shuffle(range(pool), 5)
    owned, at = [], 0
    for i, n in enumerate(lengths):
        need = _pages(n)
        row = order[at : at + need]
        if shared[i]:
            row = [row[0]] + owned[i - 1][1 : need - 1] + row[1:2]
        at += need
        owned.append(row[:need])
    return SimpleNamespace(lengths=lengths, owned=owned, pool=pool)


def _stripes(case, pool, gen):
    """Every layer's K and V cache views: random records and window rows in every page."""
    heads, caches = case["kv_heads"], []
    ring = case["recent"] + case["spec"] + 1
    rows = torch.randint(-1 << 62, 1 << 62, (pool, PAGE * heads * SLOT // 8), generator=gen,
                         device=DEV).view(torch.uint8).view(pool, -1)
    near = torch.randn(pool, (case["sink"] + ring) * 2 * heads * DIM, generator=gen, device=DEV)
    near = near.bfloat16()
    for layer in range(case["layers"]):
        k = torch.zeros(pool * PER, BLOCK, heads, DIM, dtype=torch.bfloat16, device=DEV)
        v = torch.zeros_like(k)
        k.view(torch.uint8).view(pool, -1)[:, : rows.shape[1]] = rows.roll(layer, 0)
        v.view(pool, -1)[:, : near.shape[1]] = near.roll(layer, 0)
        caches.append((k, v))
    return caches


def _cache_inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    fork = case["kind"] == "fork"
    w = _fork_world(case) if fork else _compact_world(case)
    requests = len(w.lengths)
    rows = requests + (w.children if fork else 0)
    columns = (max(_pages(n) for n in w.lengths) + 1) * PER
    s = SimpleNamespace(case=case, world=w, pool=w.pool, caches=_stripes(case, w.pool, gen))
    s.table = _table(w.owned, rows, columns).to(DEV)
    s.seq_lens = torch.tensor(w.lengths + [0] * (rows - requests), dtype=torch.int32, device=DEV)
    s.counts = torch.tensor([requests, requests], dtype=torch.int32, device=DEV)
    if fork:
        s.parents = torch.tensor(w.parents, dtype=torch.int32, device=DEV)
        s.children = torch.arange(requests, rows, dtype=torch.int32, device=DEV)
    return s


def _shared_lengths(case):
    """Token counts of each group's members in this step."""
    return [[case["prefix"] + n for n in _spread(case["members"], case["low"], case["tail"])]
            for _ in range(case["groups"])]


def _shared_inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    heads = case["kv_heads"]
    hq, whole = heads * case["group"], case["prefix"] // PAGE
    groups = _shared_lengths(case)
    lengths = [n for g in groups for n in g]
    pool = sum(whole + sum(_pages(n) - whole + 1 for n in g) for g in groups) + 1
    order = _shuffle(range(1, pool), 9)
    owned, copies, at = [], [], 0

    def take(count):
        nonlocal at
        at += count
        return order[at - count : at]

    for g in groups:
        leader = take(_pages(g[0]))
        owned.append(leader)
        for n in g[1:]:
            row = list(leader[:whole]) + take(_pages(n) - whole)
            if whole:  # the first page holds the request's window: a copy of its own
                row[0] = take(1)[0]
                copies.append((row[0], leader[0], PAGE))
            if case["prefix"] % PAGE:
                copies.append((row[whole], leader[whole], case["prefix"] % PAGE))
            owned.append(row)
    s = SimpleNamespace(case=case, lengths=lengths, layers=[])
    n = len(lengths) * case["qlen"]
    for _ in range(case["layers"]):
        history = torch.zeros(pool, PAGE * heads * DIM * 2, dtype=torch.uint8, device=DEV)
        for p0 in range(0, pool, 512):
            part = history[p0 : p0 + 512]
            part[:, : PAGE * heads * SLOT] = _records(part.shape[0] * PAGE * heads,
                                                      gen).view(part.shape[0], -1)
        for tokens in {c[2] for c in copies}:
            dst = torch.tensor([c[0] for c in copies if c[2] == tokens], device=DEV)
            src = torch.tensor([c[1] for c in copies if c[2] == tokens], device=DEV)
            end = tokens * heads * SLOT
            history[dst, :end] = history[src, :end]
        q = (2 * torch.randn(n, hq, DIM, generator=gen, device=DEV)).bfloat16()
        s.layers.append(SimpleNamespace(history=history.view(-1), q=q))
    columns = (max(_pages(x) for x in lengths) + 1) * PER
    s.table = _table(owned, len(lengths), columns).clamp_(min=0)
    return s


def prepare(case, seed):
    if case["kind"] == "qk":
        return _qk_inputs(case, seed)
    if case["kind"] in ("fork", "compact"):
        s = _cache_inputs(case, seed)
        if own:
            from oscar_new_amd import pages

            s.pages = pages.PageCaches(s.caches, _layout(case))
        return s
    s = _shared_inputs(case, seed)
    table, s.table = s.table, s.table.to(DEV)
    if not own:
        return s
    from oscar_new_amd.metadata import OscarMetadataBuilder

    s.layout = _layout(case)
    count, qlen = len(s.lengths), case["qlen"]
    starts = torch.arange(0, count * qlen + 1, qlen, dtype=torch.int32)
    seq = torch.tensor(s.lengths, dtype=torch.int32)
    common = SimpleNamespace(
        query_start_loc=starts.to(DEV), query_start_loc_cpu=starts, seq_lens=seq.to(DEV),
        seq_lens_cpu=seq, num_reqs=count, num_actual_tokens=count * qlen, max_query_len=qlen,
        max_seq_len=max(s.lengths), block_table_tensor=s.table, causal=True,
        slot_mapping=torch.full((count * qlen,), -1, dtype=torch.int64, device=DEV),
        attn_state="ChunkedPrefill")
    builder = OscarMetadataBuilder.standalone(s.layout, count, count * qlen,
                                              table.shape[1] * BLOCK, DEV)
    s.meta = builder.build(0, common)
    s.group_starts = torch.arange(0, count + 1, case["members"], dtype=torch.int32, device=DEV)
    s.prefix_tokens = torch.full((case["groups"],), case["prefix"], dtype=torch.int32, device=DEV)
    s.hq = case["kv_heads"] * case["group"]
    return s


# ------------------------------------------------------------------ the framework's calls


def _stripe_values(caches):
    """What the calls leave in the caches: the K stripes hold bytes, the V stripes window rows."""
    return [(k.view(torch.int16), v) for k, v in caches]


def _own(s):
    from oscar_new_amd import kernels, pages

    case = s.case
    if case["kind"] == "qk":
        return kernels.qk_norm_rope(
            s.query, s.key, *s.weights, s.cos_sin, s.positions, counts=s.counts, eps=EPS,
            unit_offset=case["unit_offset"], interleaved=case["interleaved"],
            rk_t=s.rk_t if case["rotate"] else None)
    if case["kind"] == "fork":
        free, _ = pages.free_pages(s.pages, s.table, s.seq_lens, s.counts)
        fresh = free[: 2 * s.parents.numel()].view(-1, 2)
        done = pages.fork_requests(s.pages, s.table, s.seq_lens, s.parents, s.children, fresh)
        return [s.table, s.seq_lens, done, free, _stripe_values(s.caches)]
    if case["kind"] == "compact":
        tables, live = pages.compact_pages(s.pages, s.table, s.seq_lens, s.counts)
        return [tables, live, _stripe_values(s.caches)]
    shared = kernels.prepare_shared(s.meta, s.layout, s.hq, s.group_starts, s.prefix_tokens)
    return [kernels.shared_history(layer.q, layer.history, s.meta, shared, s.layout, 1 / 16)
            for layer in s.layers]


# ------------------------------------------------------------------ the plain forms


def _plain_qk(s):
    case, half = s.case, s.case["rotary"] // 2
    angles = s.cos_sin[s.positions].float()[:, None]
    cos, sin = angles[..., :half], angles[..., half:]
    live = (torch.arange(case["tokens"], device=DEV) < s.counts[1])[:, None, None]
    out = []
    for x, w in zip((s.query, s.key), s.weights):
        x = x.float()
        w = w.float() + 1 if case["unit_offset"] else w.float()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        if case["interleaved"]:
            a, b = x[..., 0 : 2 * half : 2], x[..., 1 : 2 * half : 2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :half], x[..., half : 2 * half]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        x = torch.cat([turned, x[..., 2 * half :]], -1)
        out.append(torch.where(live, x, 0))
    if case["rotate"]:
        # The rotation reads the rounded query, as the attention's other branch does.
        out.append(out[0].bfloat16().float() @ s.rk_t.float().T)
    return [x.bfloat16() for x in out]


def _used_tokens(s, requests):
    """Tokens in use in every page, and the length of the request whose first page it is."""
    table = s.table[:requests, ::PER].long() // PER
    first = torch.arange(table.shape[1], device=DEV) * PAGE
    tokens = (s.seq_lens[:requests, None] - first).clamp(0, PAGE)
    page = torch.where(tokens > 0, table, 0).flatten()
    used = torch.zeros(s.pool, dtype=torch.int64, device=DEV)
    used.scatter_reduce_(0, page, tokens.flatten().long(), "amax")
    owner = torch.zeros_like(used)
    owner[table[:, 0]] = s.seq_lens[:requests].long()
    return used, owner


def _copy_rows(s, src, dst, slots, length):
    """Pages src -> dst of every layer: ``slots`` records, and the live window rows of a request
    of ``length`` tokens (0: none)."""
    case, heads = s.case, s.case["kv_heads"]
    sink, ring = case["sink"], case["recent"] + case["spec"] + 1
    at = torch.arange(PAGE, device=DEV)
    keep = at < slots[:, None]
    entry = torch.arange(sink + ring, device=DEV)
    # Window entry i < sink holds position i; entry sink + k the positions k modulo the ring.
    near = torch.where(entry < sink, entry < length[:, None],
                       (length[:, None] - sink >= ring)
                       | ((entry - sink - sink) % ring < length[:, None] - sink))
    for k, v in s.caches:
        rec = k.view(torch.uint8).view(s.pool, -1)[:, : PAGE * heads * SLOT]
        rec = rec.unflatten(1, (PAGE, heads * SLOT))
        rec[dst] = torch.where(keep[..., None], rec[src], rec[dst])
        win = v.view(s.pool, -1)[:, : (sink + ring) * 2 * heads * DIM]
        win = win.unflatten(1, (sink + ring, 2 * heads * DIM))
        win[dst] = torch.where(near[..., None], win[src], win[dst])


def _plain_fork(s):
    requests = s.case["requests"]
    used, _ = _used_tokens(s, requests)
    page = torch.arange(s.pool, device=DEV)
    order = torch.argsort(torch.where(used > 0, s.pool + page, page))
    free = torch.where(used[order] > 0, -1, order).int()
    parents, children = s.parents.long(), s.children.long()
    fresh = free[: 2 * parents.numel()].view(-1, 2).long()
    length = s.seq_lens[parents].long()
    count = (length + PAGE - 1) // PAGE
    row = s.table[parents, ::PER].long() // PER
    last = row.gather(1, (count - 1)[:, None])[:, 0]
    tail = length - (count - 1) * PAGE
    index = torch.arange(row.shape[1], device=DEV)
    extra = (count > 1) & (tail < PAGE)
    _copy_rows(s, row[:, 0], fresh[:, 0], length.clamp(max=PAGE), length)
    _copy_rows(s, torch.where(extra, last, row[:, 0]), torch.where(extra, fresh[:, 1], fresh[:, 0]),
               torch.where(extra, tail, 0), torch.zeros_like(length))
    row = torch.where(index == 0, fresh[:, :1], row)
    row = torch.where((index == (count - 1)[:, None]) & extra[:, None], fresh[:, 1:], row)
    blocks = (row[..., None] * PER + torch.arange(PER, device=DEV)).flatten(1).int()
    held = (index < count[:, None]).repeat_interleave(PER, 1)
    s.table[children] = torch.where(held, blocks, s.table[children])
    s.seq_lens[children] = s.seq_lens[parents]
    return [s.table, s.seq_lens, torch.ones_like(s.parents), free, _stripe_values(s.caches)]


def _plain_compact(s):
    requests = s.case["requests"]
    used, owner = _used_tokens(s, requests)
    page = torch.arange(s.pool, device=DEV)
    live = used > 0
    total = live.sum()
    holes = page[~live & (page < total)]
    movers = page[live & (page >= total)]
    place = page.clone()
    place[movers] = holes
    _copy_rows(s, movers, holes, used[movers], owner[movers])
    index = torch.arange(s.table.shape[1], device=DEV) // PER * PAGE
    held = index < s.seq_lens[:, None]
    block = s.table.long().clamp(min=0)
    moved = place[block // PER] * PER + block % PER
    return [torch.where(held, moved, s.table.long()).int(), total.int().view(1), _stripe_values(s.caches)]


def _rows_of(table, positions, heads):
    """Byte offsets of the records of ``positions`` ([..., tokens]) through rows of a block table."""
    block = table.gather(-1, positions // BLOCK).long()
    slot = block * BLOCK + positions % BLOCK
    return slot // PAGE * (PAGE * heads * DIM * 2) + slot % PAGE * (heads * SLOT)


def _values(history, offsets, at):
    """fp32 rows of the K (at 0) or V (at 68) half of the records at ``offsets``."""
    data = history[offsets[..., None] + torch.arange(at, at + 68, device=DEV)]
    codes = torch.stack([data[..., :64] >> s & 3 for s in (0, 2, 4, 6)], -1).flatten(-2).float()
    scale = data[..., 64:].contiguous().view(torch.float16).float()
    return codes * scale[..., :1] + scale[..., 1:]


def _plain_shared(s):
    case, answers = s.case, []
    heads, g, qlen, m = case["kv_heads"], case["group"], case["qlen"], case["members"]
    for layer in s.layers:
        n = layer.q.shape[0]
        out = torch.zeros(n, heads * g, DIM, device=DEV)
        lse = torch.full((n, heads * g), -math.inf, device=DEV)
        for i in range(case["groups"]):
            lengths = s.lengths[i * m : (i + 1) * m]
            table = s.table[i * m : (i + 1) * m].long()
            end = max(case["sink"], _shared_end(case, lengths))
            stop = [_history(case, x)[1] for x in lengths]
            common = torch.arange(case["sink"], end, device=DEV)
            common = _rows_of(table[0], common, heads)
            rest = torch.arange(end, max(stop + [end + 1]), device=DEV).expand(m, -1)
            seen = rest < torch.tensor(stop, device=DEV)[:, None]
            rest = _rows_of(table, rest.contiguous(), heads)
            tokens = slice(i * m * qlen, (i + 1) * m * qlen)
            for h in range(heads):
                q = layer.q[tokens, h * g : (h + 1) * g].float().reshape(m, qlen * g, DIM) / 16
                k0 = _values(layer.history, common + h * SLOT, 0)
                k1 = _values(layer.history, rest + h * SLOT, 0)
                a = (q.view(-1, DIM) @ k0.T).view(m, qlen * g, common.numel())
                b = torch.bmm(q, k1.transpose(1, 2).contiguous())
                b = torch.where(seen[:, None], b, -math.inf)
                top = b.amax(-1, keepdim=True)
                if a.shape[-1]:
                    top = torch.maximum(top, a.amax(-1, keepdim=True))
                top = torch.where(top == -math.inf, 0, top)
                a, b = torch.exp(a - top), torch.exp(b - top)
                total = a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True)
                v0 = _values(layer.history, common + h * SLOT, 68)
                x = (a.view(m * qlen * g, common.numel()) @ v0).view(m, qlen * g, DIM)
                x = x + torch.bmm(b, _values(layer.history, rest + h * SLOT, 68))
                x = torch.where(total > 0, x / total.clamp(min=1e-30), 0)
                out[tokens, h * g : (h + 1) * g] = x.view(m * qlen, g, DIM)
                lse[tokens, h * g : (h + 1) * g] = (top + torch.log(total)).view(m * qlen, g)
        answers.append((out.bfloat16(), lse))
    return answers


def run(state):
    if own:
        return _own(state)
    return {"qk": _plain_qk, "fork": _plain_fork, "compact": _plain_compact,
            "shared": _plain_shared}[state.case["kind"]](state)


# ------------------------------------------------------------------ 64-bit values


def _exact_qk(case, seed):
    s = _qk_inputs(case, seed)
    rotary = case["rotary"]
    table = s.cos_sin[s.positions].double()
    turn = torch.complex(table[:, : rotary // 2], table[:, rotary // 2 :])[:, None]
    results = []
    for x, w in ((s.query, s.weights[0]), (s.key, s.weights[1])):
        x = x.double()
        x = x * (x.square().sum(-1, keepdim=True) / DIM + EPS).rsqrt()
        x = x * (w.double() + (1.0 if case["unit_offset"] else 0.0))
        head = x[..., :rotary]
        head = (head.unflatten(-1, (rotary // 2, 2)) if case["interleaved"]
                else head.unflatten(-1, (2, rotary // 2)).transpose(-1, -2))
        head = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn)
        x[..., :rotary] = (head if case["interleaved"] else head.transpose(-1, -2)).flatten(-2)
        x[case["live"] :] = 0
        results.append(x)
    if case["rotate"]:
        results.append(results[0].bfloat16().double() @ s.rk_t.double().T)
    return results


def _copy_request(case, caches, src, dst, slots, length):
    heads = case["kv_heads"]
    sink, ring = case["sink"], case["recent"] + case["spec"] + 1
    entries = list(range(min(length, sink)))
    entries += sorted({sink + p % ring for p in range(max(sink, length - ring), length)})
    stripe, row = PAGE * heads * DIM, 2 * heads * DIM
    at = torch.tensor(entries, dtype=torch.long, device=DEV)
    for k, v in caches:
        rec, win = k.view(torch.uint8).view(-1, 2 * stripe), v.view(-1, stripe)
        rec[dst, : slots * heads * SLOT] = rec[src, : slots * heads * SLOT]
        if entries:
            win[dst, : (sink + ring) * row].view(-1, row)[at] = (
                win[src, : (sink + ring) * row].view(-1, row)[at])


def _exact_fork(case, seed):
    s = _cache_inputs(case, seed)
    w, table, lengths = s.world, s.table.cpu(), list(s.world.lengths)
    taken = {p for row in w.owned for p in row}
    free = [p for p in range(w.pool) if p not in taken]
    for i, parent in enumerate(w.parents):
        n, row = lengths[parent], list(w.owned[parent])
        _copy_request(case, s.caches, row[0], free[2 * i], min(n, PAGE), n)
        if n > PAGE and n % PAGE:
            _copy_request(case, s.caches, row[-1], free[2 * i + 1], n % PAGE, 0)
            row[-1] = free[2 * i + 1]
        row[0] = free[2 * i]
        for j, page in enumerate(row):
            for b in range(PER):
                table[case["requests"] + i, j * PER + b] = page * PER + b
        s.seq_lens[case["requests"] + i] = n
    order = torch.tensor(free + [-1] * len(taken), dtype=torch.int32, device=DEV)
    return [table.to(DEV), s.seq_lens, torch.ones_like(s.parents), order, _stripe_values(s.caches)]


def _exact_compact(case, seed):
    s = _cache_inputs(case, seed)
    w, table = s.world, s.table.cpu()
    slots, length = {}, {}
    for n, row in zip(w.lengths, w.owned):
        length[row[0]] = n
        for j, page in enumerate(row):
            slots[page] = max(slots.get(page, 0), min(PAGE, n - j * PAGE))
    holes = [p for p in range(len(slots)) if p not in slots]
    place = dict(zip(sorted(p for p in slots if p >= len(slots)), holes))
    for src, dst in place.items():
        _copy_request(case, s.caches, src, dst, slots[src], length.get(src, 0))
    for r, row in enumerate(w.owned):
        for j, page in enumerate(row):
            for b in range(PER):
                table[r, j * PER + b] = place.get(page, page) * PER + b
    live = torch.tensor([len(slots)], dtype=torch.int32, device=DEV)
    return [table.to(DEV), live, _stripe_values(s.caches)]


def _decoded(history, blocks, first, last, head, heads, at):
    """float64 rows of positions [first, last) of one request, found slot by slot."""
    position = torch.arange(first, last, device=DEV)
    block = blocks[position // BLOCK].long()
    inside = block % PER * BLOCK + position % BLOCK
    pages = history.view(-1, PAGE * heads * DIM * 2)[:, : PAGE * heads * SLOT]
    record = pages.unflatten(1, (PAGE, heads, SLOT))[block // PER, inside, head, at : at + 68]
    record = record.contiguous()
    low = [(record[:, :64] // 4**e % 4).double() for e in range(4)]
    pair = record[:, 64:].contiguous().view(torch.float16).double()
    return torch.stack(low, -1).view(-1, DIM) * pair[:, :1] + pair[:, 1:]


def _exact_shared(case, seed):
    s = _shared_inputs(case, seed)
    table, heads, g = s.table.to(DEV), case["kv_heads"], case["group"]
    answers = []
    for layer in s.layers:
        n = layer.q.shape[0]
        out = torch.zeros(n, heads * g, DIM, dtype=torch.float64, device=DEV)
        lse = torch.full((n, heads * g), -math.inf, dtype=torch.float64, device=DEV)
        for r, length in enumerate(s.lengths):
            begin, end = _history(case, length)
            if begin >= end:
                continue
            tokens = slice(r * case["qlen"], (r + 1) * case["qlen"])
            for h in range(heads):
                rows = slice(h * g, (h + 1) * g)
                q = layer.q[tokens, rows].double()
                key = _decoded(layer.history, table[r], begin, end, h, heads, 0)
                score = q.reshape(-1, DIM) @ key.T / 16
                lse[tokens, rows] = score.logsumexp(-1).view(-1, g)
                value = _decoded(layer.history, table[r], begin, end, h, heads, 68)
                out[tokens, rows] = (score.softmax(-1) @ value).view(-1, g, DIM)
        answers.append((out, lse))
    return answers


def exact(case, seed):
    return {"qk": _exact_qk, "fork": _exact_fork, "compact": _exact_compact,
            "shared": _exact_shared}[case["kind"]](case, seed)
