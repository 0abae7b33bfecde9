"""Workloads of the operators around a cache of 4-bit records, for timing and comparison: what a
serving engine runs when it keeps its history in 4 bits and its models place tokens on several axes.

A case is one call (or the calls of one use) of one operator:

* ``append``: rows of a packed projection on their way into the paged cache: norms of the queries
  and keys, the position rotation, the rotations by R_k and R_v, and the 4-bit records, in one call;
  then the appended records as values, as a check or a move of them reads them.
* ``axes``: norms and position rotation of queries and keys whose positions have several axes
  (time, height, width of images and video), without the cache.
* ``attend``: attention of one step over the 4-bit history of a batch, one layer: partial rows of
  the splits and their merge, by the partition that the layer chooses.

Lengths and page ownership come from the case alone; rows, records, positions and weights from the
seed. A record of one token and KV head is 272 bytes: K codes (dim d in nibble d % 2 of byte d / 2),
V codes, then fp16 K scale, K zero, V scale, V zero; the value of code c is zero + scale c. Queries
are scaled so that scores spread by about two nats. Head sizes, pages and windows are the defaults of
the package; batches and lengths those of ``bench.py`` (32 x 32768, 16 requests of 4 query tokens,
a 2048-token chunk, 4 x 4096 prefill) and generic ones around them.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DIM, PAGE, BLOCK, SLOT = 256, 768, 128, 272
PER = PAGE // BLOCK
STRIPE = PAGE * DIM * 2  # bytes of a page of one KV head's stripe
DEV = "cuda"
EPS = 1e-6
K_CLIP, V_CLIP = 0.99, 0.98


# ------------------------------------------------------------------ the cases


def _rows(kind, name, **over):
    case = dict(kind=kind, tokens=32, live=0, group=6, kv_heads=1, rotary=64, positions=32768,
                axes=1, cycle=False, interleaved=False, norm=True, unit_offset=True, rotate=True,
                fp32=False)
    case.update(over)
    case["live"] = case["live"] or case["tokens"]
    return dict(case, name=name) if name else case


def _attend(name, **over):
    case = dict(kind="attend", requests=1, low=900, context=900, qlen=1, group=6, kv_heads=1,
                sink=64, recent=256, spec=3)
    case.update(over)
    return dict(case, name=name) if name else case


def listed():
    return [
        # A decode batch on one tensor-parallel rank.
        _rows("append", "append 32 decode"),
        # A prompt's chunk with images in it, two KV heads, a graph's padding behind the last token.
        _rows("append", "append 2048 chunk", tokens=2048, live=2041, kv_heads=2, axes=3, rotary=128),
        # Prompts that arrive together, no history yet and so no queries rotated by R_k; a model
        # without norms of queries and keys.
        _rows("append", "append 16384 prefill", tokens=16384, rotate=False, norm=False, group=4),
        # A decode batch whose tokens carry three positions each, queries rotated in the call.
        _rows("axes", "axes 48 decode", tokens=48, axes=3, rotary=128, cycle=True),
        # One image's tokens, two axes, adjacent pairs.
        _rows("axes", "axes 1369 image", tokens=1369, axes=2, rotary=256, group=1, kv_heads=16,
              interleaved=True, rotate=False, positions=512, fp32=True),
        # Prompts with video.
        _rows("axes", "axes 16384 video", tokens=16384, axes=3, rotary=128, rotate=False),
        # One short conversation: launches and latency.
        _attend("attend 1x900"),
        # The headline decode batch.
        _attend("attend 32x32k", requests=32, low=32768, context=32768, sink=4, recent=128),
        # Ragged users, two KV heads.
        _attend("attend 24 ragged", requests=24, low=70, context=15011, kv_heads=2, group=5),
        # MTP verification, 4 query tokens a request.
        _attend("attend mtp 16", requests=16, low=1000, context=32000, qlen=4),
        # A continuation chunk of one long prompt.
        _attend("attend chunk 2048", low=32768, context=32768, qlen=2048),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "append", "axes", "attend", "attend"])
    heads = rng.choice([1, 1, 2, 4])
    if kind != "attend":
        tokens = _log(rng, 1, 16384 // heads)
        return _rows(kind, "", tokens=tokens, live=tokens - (rng.randrange(tokens) // 8),
                     kv_heads=heads, group=rng.choice([1, 4, 5, 6, 6, 8]) if tokens < 8000 // heads else 4,
                     rotary=rng.choice([32, 64, 64, 96, 128, 256]), positions=_log(rng, 512, 131072),
                     axes=rng.choice([1, 2, 3, 3, 4] if kind == "append" else [2, 3, 3, 4]),
                     cycle=rng.random() < 0.4, interleaved=rng.random() < 0.3,
                     norm=kind == "axes" or rng.random() < 0.7, unit_offset=rng.random() < 0.5,
                     rotate=rng.random() < 0.6, fp32=rng.random() < 0.4)
    short = rng.random() < 0.4
    group = rng.choice([1, 4, 5, 6, 6, 8])
    qlen = rng.choice([1, 1, 1, 2, 3, 4, 0])
    heads = min(heads, 2)
    over = dict(kv_heads=heads, group=group, sink=4 if short else 64, recent=128 if short else 256)
    if qlen == 0:  # a continuation chunk
        qlen = _log(rng, 17, 2048)
        return _attend("", qlen=qlen, low=qlen, context=qlen + _log(rng, 600, 180000 // (heads * group)) if group > 5
                       else qlen + _log(rng, 600, 30000 // heads), **over)
    requests = _log(rng, 1, 64 // heads)
    context = _log(rng, 400, min(131072, 1 << 20) if requests * heads < 8 else
                   (32 * 32768) // (requests * heads))
    return _attend("", qlen=qlen, requests=requests, low=rng.choice([qlen, 150, 399]),
                   context=context, **over)


def _lengths(case):
    """Token counts of the requests: spread over the logarithm, the longest first but scattered."""
    n, low, high = case["requests"], case["low"], case["context"]
    if n == 1:
        return [high]
    got = [int(round(low * (high / low) ** (i / (n - 1)))) for i in range(n)]
    return [got[i * 7 % n] for i in range(n)] if n % 7 else got


def _history(case, length):
    """History positions [begin, end) of a request of ``length`` tokens in this step."""
    prefix = length - case["qlen"]
    begin = min(case["sink"], prefix)
    return begin, max(begin, prefix - case["recent"])


def work(case):
    """What a pass cannot do without. ``append`` and ``axes``: each row read and written once (the
    queries twice where they are rotated as well), the angles and positions, R_k and R_v, the
    records of 264 bytes written, and read back as rows. ``attend``: 264 bytes per record, queries,
    outputs and LSE; 4 operations per query row, visible key and dim."""
    if case["kind"] == "attend":
        spans = [_history(case, n) for n in _lengths(case)]
        rows, heads = case["group"] * case["kv_heads"], case["kv_heads"]
        n = case["requests"] * case["qlen"]
        visible = sum(e - b for b, e in spans)
        return {"bytes": 264 * visible * heads + n * rows * (1024 + 4),
                "flops": 4 * DIM * rows * visible * case["qlen"]}
    n, hk = case["live"], case["kv_heads"]
    hq = hk * case["group"]
    total = n * (hq + hk) * 1024 + n * (case["rotary"] * (4 if case["fp32"] else 2) + 8 * case["axes"])
    total += (case["tokens"] - n) * (hq + hk) * 512
    flops = n * (hq + hk) * DIM * 6
    if case["rotate"]:
        total += case["tokens"] * hq * 512 + 2 * DIM * DIM
        flops += n * hq * 2 * DIM * DIM
    if case["kind"] == "append":
        total += 4 * DIM * DIM + n * hk * (512 + 2 * 264) + case["tokens"] * hk * 1024
        flops += n * hk * 4 * DIM * DIM
    return {"bytes": total, "flops": flops}


# ------------------------------------------------------------------ inputs


def _shuffle(items, salt):
    """A fixed scattered order of ``items`` (no random state: ownership belongs to the case)."""
    return sorted(items, key=lambda i: (i * 2654435761 + salt * 40503) % 4294967291)


def _pages(tokens):
    return -(-tokens // PAGE)


def _sections(case):
    """Pairs of every axis: the first about half as many as each of the others."""
    half, axes = case["rotary"] // 2, case["axes"]
    if axes == 1:
        return [half]
    rest = half * 2 // (2 * axes - 1)
    return [half - rest * (axes - 1)] + [rest] * (axes - 1)


def _pair_axes(case):
    """The axis of every pair: sections one after the other, or in turn while they last."""
    counts = _sections(case)
    if not case["cycle"]:
        return [a for a, c in enumerate(counts) for _ in range(c)]
    got = [0] * sum(counts)
    for a, c in enumerate(counts):
        if a:
            for i in range(c):
                if a + i * len(counts) < len(got):
                    got[a + i * len(counts)] = a
    return got


def _row_inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    n, hk, half = case["tokens"], case["kv_heads"], case["rotary"] // 2
    hq = hk * case["group"]
    # One projection row per token: [query, gate] of each query head, then keys, then values.
    packed = torch.randn(n, (2 * hq + 2 * hk) * DIM, generator=gen, device=DEV)
    packed *= torch.rand(n, 1, generator=gen, device=DEV) * 3 + 0.2
    packed = packed.bfloat16()
    query = packed[:, : 2 * hq * DIM].view(n, hq, 2 * DIM)[..., :DIM]
    key = packed[:, 2 * hq * DIM : (2 * hq + hk) * DIM].view(n, hk, DIM)
    value = packed[:, (2 * hq + hk) * DIM :].view(n, hk, DIM)
    rate = 1e7 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    angle = torch.arange(case["positions"], device=DEV, dtype=torch.float64)[:, None] * rate
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1)
    cos_sin = cos_sin.float() if case["fp32"] else cos_sin.bfloat16()
    positions = torch.randint(case["positions"], (case["axes"], n), generator=gen, device=DEV)
    # A quarter of the tokens are text: the same position on every axis.
    text = torch.rand(n, generator=gen, device=DEV) < 0.25
    positions = torch.where(text, positions[:1], positions)
    weights = [0.3 * torch.randn(DIM, generator=gen, device=DEV) + (0 if case["unit_offset"] else 1)
               for _ in range(2)]
    if not case["fp32"]:
        weights = [w.bfloat16() for w in weights]
    rk, rv = (torch.linalg.qr(torch.randn(DIM, DIM, generator=gen, device=DEV))[0].bfloat16()
              for _ in range(2))
    counts = torch.tensor([1, case["live"]], dtype=torch.int32, device=DEV)
    s = SimpleNamespace(case=case, query=query, key=key, value=value, weights=weights,
                        cos_sin=cos_sin, positions=positions, counts=counts,
                        rk_t=rk.T.contiguous(), rv_t=rv.T.contiguous(), axes=None)
    if case["axes"] > 1:
        s.axes = torch.tensor(_pair_axes(case), dtype=torch.int32, device=DEV)
    else:
        s.positions = positions[0].contiguous()
    if case["kind"] == "append":
        # Tokens go to pages of the pool in a scattered order, from the middle of a page on.
        start, pool = 300, _pages(n + 300) + 2
        page = torch.tensor(_shuffle(range(pool), 7), device=DEV)
        at = torch.arange(start, start + n, device=DEV)
        s.slots = page[at // PAGE] * PAGE + at % PAGE
        s.slots[case["live"] :] = -1
        s.history = torch.zeros(pool * hk * STRIPE, dtype=torch.uint8, device=DEV)
    return s


def _some_records(n, gen):
    """[n, 272] uint8 records of Gaussian rows, clipped at the quantiles of the configuration."""
    out = torch.zeros(n, SLOT, dtype=torch.uint8, device=DEV)
    for at, side, clip in ((0, 256, 2.576), (128, 260, 2.326)):
        x = torch.randn(n, DIM, generator=gen, device=DEV)
        x.clamp_(-clip, clip)
        low = x.amin(1, keepdim=True)
        scale = ((x.amax(1, keepdim=True) - low) / 15).half()
        low = low.half()
        x.sub_(low.float()).div_(scale.float()).round_().clamp_(0, 15)
        codes = x.to(torch.uint8).view(n, DIM // 2, 2)
        out[:, at : at + 128] = codes[..., 0] | codes[..., 1] << 4
        out[:, side : side + 4] = torch.cat([scale, low], 1).view(torch.uint8)
    return out


def _attend_inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    heads, lengths = case["kv_heads"], _lengths(case)
    pool = sum(_pages(n) for n in lengths) + 1
    order, at = _shuffle(range(1, pool), 9), 0
    columns = (max(_pages(n) for n in lengths) + 1) * PER
    table = torch.zeros(len(lengths), columns, dtype=torch.int32)
    for r, n in enumerate(lengths):
        row = order[at : at + _pages(n)]
        at += len(row)
        table[r, : len(row) * PER] = torch.tensor([p * PER + b for p in row for b in range(PER)],
                                                  dtype=torch.int32)
    history = torch.zeros(pool, heads * STRIPE, dtype=torch.uint8, device=DEV)
    for p0 in range(0, pool, 512):
        part = history[p0 : p0 + 512]
        part[:, : PAGE * heads * SLOT] = _some_records(part.shape[0] * PAGE * heads,
                                                       gen).view(part.shape[0], -1)
    n = len(lengths) * case["qlen"]
    query = (2 * torch.randn(n, heads * case["group"], DIM, generator=gen, device=DEV)).bfloat16()
    return SimpleNamespace(case=case, lengths=lengths, history=history.view(-1), query=query,
                           table=table.to(DEV))


def _layout(case):
    from oscar_new_amd.config import OscarConfig
    from oscar_new_amd.layout import CacheLayout

    config = OscarConfig(history_bits=4, sink_tokens=case.get("sink", 64),
                         recent_tokens=case.get("recent", 256), speculative_tokens=3,
                         k_clip_ratio=K_CLIP, v_clip_ratio=V_CLIP)
    return CacheLayout(PAGE, kv_heads=case["kv_heads"], config=config)


def prepare(case, seed):
    if case["kind"] != "attend":
        s = _row_inputs(case, seed)
        if own:
            s.layout = _layout(case)
        return s
    s = _attend_inputs(case, seed)
    if not own:
        return s
    from oscar_new_amd.backend import OscarAttentionImpl
    from oscar_new_amd.metadata import OscarMetadataBuilder

    s.layout = _layout(case)
    count, qlen, heads = len(s.lengths), case["qlen"], case["kv_heads"]
    starts = torch.arange(0, count * qlen + 1, qlen, dtype=torch.int32)
    seq = torch.tensor(s.lengths, dtype=torch.int32)
    common = SimpleNamespace(
        query_start_loc=starts.to(DEV), query_start_loc_cpu=starts, seq_lens=seq.to(DEV),
        seq_lens_cpu=seq, num_reqs=count, num_actual_tokens=count * qlen, max_query_len=qlen,
        max_seq_len=max(s.lengths), block_table_tensor=s.table, causal=True,
        slot_mapping=torch.full((count * qlen,), -1, dtype=torch.int64, device=DEV),
        attn_state="ChunkedPrefill")
    builder = OscarMetadataBuilder.standalone(s.layout, count, count * qlen,
                                              s.table.shape[1] * BLOCK, DEV)
    s.meta = builder.build(0, common)
    s.impl = OscarAttentionImpl.standalone(heads * case["group"], DIM, 1 / 16, heads,
                                           cfg=s.layout.config)
    return s


# ------------------------------------------------------------------ the framework's calls


def _own(s):
    from oscar_new_amd import kernels

    case = s.case
    if case["kind"] == "axes":
        return kernels.qk_norm_rope(
            s.query, s.key, *s.weights, s.cos_sin, s.positions, counts=s.counts, eps=EPS,
            unit_offset=case["unit_offset"], interleaved=case["interleaved"],
            rk_t=s.rk_t if case["rotate"] else None, axes=s.axes)
    if case["kind"] == "append":
        weights = s.weights if case["norm"] else (None, None)
        query, key, turned = kernels.rope_append(
            s.query, s.key, s.value, s.history, s.slots, s.counts, s.layout, s.rk_t, s.rv_t,
            cos_sin=s.cos_sin, positions=s.positions, axes=s.axes, q_weight=weights[0],
            k_weight=weights[1], eps=EPS, unit_offset=case["unit_offset"],
            interleaved=case["interleaved"], rotate_query=case["rotate"])
        kept = kernels.read_records(s.history, s.slots, s.layout)
        return [query, key, *kept] + ([turned] if case["rotate"] else [])
    splits, split_tokens = s.impl.partition_for(s.meta, s.query.shape[0])
    partials, lse = kernels.attention_partials(
        s.query, None, None, s.history, None, s.meta, s.layout, 1 / 16, splits, raw=False,
        split_tokens=split_tokens)
    return kernels.merge_splits(partials, lse, s.meta.counts)


# ------------------------------------------------------------------ the plain forms


def _plain_turn(s):
    """Queries and keys in fp32, normed and turned, zeros past the live tokens."""
    case, half = s.case, s.case["rotary"] // 2
    if s.axes is None:
        angles = s.cos_sin[s.positions].float()[:, None]
    else:
        pos = s.positions[s.axes.long()].T  # [tokens, half]
        pair = torch.arange(half, device=DEV)
        angles = torch.cat([s.cos_sin[pos, pair], s.cos_sin[pos, pair + half]], 1).float()[:, None]
    cos, sin = angles[..., :half], angles[..., half:]
    live = (torch.arange(case["tokens"], device=DEV) < s.counts[1])[:, None, None]
    out = []
    for x, w in zip((s.query, s.key), s.weights):
        x = x.float()
        if case["norm"]:
            w = w.float() + 1 if case["unit_offset"] else w.float()
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        if case["interleaved"]:
            a, b = x[..., 0 : 2 * half : 2], x[..., 1 : 2 * half : 2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :half], x[..., half : 2 * half]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        x = torch.cat([turned, x[..., 2 * half :]], -1)
        out.append(torch.where(live, x, 0).bfloat16())
    return out


def _plain_axes(s):
    query, key = _plain_turn(s)
    if s.case["rotate"]:
        return [query, key, (query.float() @ s.rk_t.float().T).bfloat16()]
    return [query, key]


def _quantile(magnitude, ratio):
    order = magnitude.sort(-1).values
    rank = ratio * (DIM - 1)
    low = math.floor(rank)
    a, b = order[..., low : low + 1], order[..., math.ceil(rank) : math.ceil(rank) + 1]
    return a + (rank - low) * (b - a)


def _plain_codes(x, ratio):
    """4-bit codes [.., 256], fp16 scale and zero of rows."""
    x = x.bfloat16().float()
    limit = _quantile(x.abs(), ratio)
    x = torch.minimum(torch.maximum(x, -limit), limit)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high - low) / 15).clamp(min=2.0**-14).half()
    zero = low.half()
    codes = ((x - zero.float()) / scale.float() + 0.5).clamp(0, 15).to(torch.uint8)
    return codes, scale, zero


def _decode(codes, side):
    """fp32 rows of packed codes [.., 128] and their scale and zero [.., 4] bytes."""
    pair = side.contiguous().view(torch.float16).float()
    values = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    return values * pair[..., :1] + pair[..., 1:]


def _plain_append(s):
    case, heads = s.case, s.case["kv_heads"]
    query, key = _plain_turn(s)
    pages = s.history.view(-1, heads * STRIPE)[:, : PAGE * heads * SLOT]
    pages = pages.unflatten(1, (PAGE, heads, SLOT))
    live = case["live"]
    page, inside = s.slots[:live] // PAGE, s.slots[:live] % PAGE
    for at, side, rows, turn, ratio in ((0, 256, key, s.rk_t, K_CLIP),
                                        (128, 260, s.value, s.rv_t, V_CLIP)):
        codes, scale, zero = _plain_codes(rows[:live].float() @ turn.float().T, ratio)
        pages[page, inside, :, at : at + 128] = codes[..., 0::2] | codes[..., 1::2] << 4
        pages[page, inside, :, side : side + 4] = torch.cat([scale, zero], -1).view(torch.uint8)
    record = pages[page, inside]
    kept = [torch.zeros_like(key), torch.zeros_like(key)]
    kept[0][:live] = _decode(record[..., :128], record[..., 256:260]).bfloat16()
    kept[1][:live] = _decode(record[..., 128:256], record[..., 260:264]).bfloat16()
    turned = [(query.float() @ s.rk_t.float().T).bfloat16()] if case["rotate"] else []
    return [query, key, *kept] + turned


def _plain_attend(s):
    case, heads, g, qlen = s.case, s.case["kv_heads"], s.case["group"], s.case["qlen"]
    spans = [_history(case, n) for n in s.lengths]
    m, longest = len(spans), max(max(e - b for b, e in spans), 1)
    begin = torch.tensor([b for b, _ in spans], device=DEV)[:, None]
    end = torch.tensor([e for _, e in spans], device=DEV)[:, None]
    at = begin + torch.arange(longest, device=DEV)
    seen = at < end
    at = torch.where(seen, at, 0)
    block = s.table.long().gather(1, at // BLOCK)
    pages = s.history.view(-1, heads * STRIPE)[:, : PAGE * heads * SLOT]
    pages = pages.unflatten(1, (PAGE, heads, SLOT))
    out = torch.zeros(m, qlen, heads, g, DIM, device=DEV)
    lse = torch.zeros(m, qlen, heads, g, device=DEV)
    for h in range(heads):
        record = pages[block // PER, block % PER * BLOCK + at % BLOCK, h]
        key = _decode(record[..., :128], record[..., 256:260])
        q = s.query.view(m, qlen, heads, g, DIM)[:, :, h].float().reshape(m, qlen * g, DIM) / 16
        score = torch.bmm(q, key.transpose(1, 2).contiguous())
        score = torch.where(seen[:, None], score, -math.inf)
        top = score.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, 0, top)
        score = torch.exp(score - top)
        total = score.sum(-1, keepdim=True)
        value = _decode(record[..., 128:256], record[..., 260:264])
        x = torch.bmm(score, value)
        x = torch.where(total > 0, x / total.clamp(min=1e-30), 0)
        out[:, :, h] = x.view(m, qlen, g, DIM)
        lse[:, :, h] = (top + torch.log(total)).view(m, qlen, g)
    n = m * qlen
    return out.view(n, heads * g, DIM).bfloat16(), lse.view(n, heads * g)


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "axes": _plain_axes, "attend": _plain_attend}[
        state.case["kind"]](state)


# ------------------------------------------------------------------ 64-bit values


def _exact_turn(case, s):
    half = case["rotary"] // 2
    table, tokens = s.cos_sin.double(), torch.arange(case["tokens"], device=DEV)
    turn = torch.empty(case["tokens"], half, dtype=torch.complex128, device=DEV)
    for j, axis in enumerate(_pair_axes(case)):
        row = s.positions if s.axes is None else s.positions[axis]
        turn[:, j] = torch.complex(table[row, j], table[row, half + j])
    results = []
    for x, w in ((s.query, s.weights[0]), (s.key, s.weights[1])):
        x = x.double()
        if case["norm"]:
            x = x * (x.square().sum(-1, keepdim=True) / DIM + EPS).rsqrt()
            x = x * (w.double() + (1.0 if case["unit_offset"] else 0.0))
        head = x[..., : 2 * half]
        head = (head.unflatten(-1, (half, 2)) if case["interleaved"]
                else head.unflatten(-1, (2, half)).transpose(-1, -2))
        head = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn[:, None])
        x = x.clone()
        x[..., : 2 * half] = (head if case["interleaved"] else head.transpose(-1, -2)).flatten(-2)
        x[tokens >= case["live"]] = 0
        results.append(x)
    return results


def _exact_values(rows, turn, ratio):
    """Values that the records of rows @ turn^T stand for; the rotated rows are bf16."""
    x = (rows.double() @ turn.double().T).bfloat16().double()
    order = x.abs().sort(-1).values
    rank = ratio * 255
    low = int(rank)
    limit = torch.lerp(order[..., low], order[..., min(low + 1, 255)], rank - low)[..., None]
    x = torch.maximum(torch.minimum(x, limit), -limit)
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    zero = low.half().double()
    scale = torch.clamp((high - low) / 15, min=2.0**-14).half().double()
    return torch.floor((x - zero) / scale + 0.5).clamp(0, 15) * scale + zero


def _exact_rows(case, seed):
    s = _row_inputs(case, seed)
    query, key = _exact_turn(case, s)
    turned = [query.bfloat16().double() @ s.rk_t.double().T] if case["rotate"] else []
    if case["kind"] == "axes":
        return [query, key] + turned
    kept = [_exact_values(key.bfloat16(), s.rk_t, K_CLIP), _exact_values(s.value, s.rv_t, V_CLIP)]
    for x in kept:
        x[case["live"] :] = 0
    return [query, key, *kept] + turned


def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    heads, g, qlen = case["kv_heads"], case["group"], case["qlen"]
    n = len(s.lengths) * qlen
    out = torch.zeros(n, heads * g, DIM, dtype=torch.float64, device=DEV)
    lse = torch.full((n, heads * g), -math.inf, dtype=torch.float64, device=DEV)
    pages = s.history.view(-1, PAGE * heads * DIM * 2)[:, : PAGE * heads * SLOT]
    pages = pages.unflatten(1, (PAGE, heads, SLOT))
    for r, length in enumerate(s.lengths):
        begin, end = _history(case, length)
        if begin >= end:
            continue
        at = torch.arange(begin, end, device=DEV)
        slot = s.table[r, at // BLOCK].long() * BLOCK + at % BLOCK
        tokens = slice(r * qlen, (r + 1) * qlen)
        for h in range(heads):
            record = pages[slot // PAGE, slot % PAGE, h]
            pair = record[:, 256:264].contiguous().view(torch.float16).double()
            rows = []
            for i in (0, 1):
                packed = record[:, 128 * i : 128 * i + 128]
                code = torch.empty(end - begin, DIM, dtype=torch.float64, device=DEV)
                code[:, 0::2], code[:, 1::2] = (packed % 16).double(), (packed // 16).double()
                rows.append(pair[:, 2 * i + 1 : 2 * i + 2] + pair[:, 2 * i : 2 * i + 1] * code)
            for h1 in range(h * g, (h + 1) * g):
                score = s.query[tokens, h1].double() @ rows[0].T / 16
                lse[tokens, h1] = score.logsumexp(-1)
                out[tokens, h1] = score.softmax(-1) @ rows[1]
    return out, lse


def exact(case, seed):
    return _exact_attend(case, seed) if case["kind"] == "attend" else _exact_rows(case, seed)
