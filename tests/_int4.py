"""Worlds of 4-bit records for the GPU tests: caches, metadata of a step, and attention in 64 bits."""

import math
from types import SimpleNamespace

import torch

from oscar_new_amd.config import OscarConfig, task_capacity
from oscar_new_amd.layout import CacheLayout

DEV = "cuda"
SLOT = 272


def layout_of(heads=1, page=768, block=128, bits=4, **config):
    config.setdefault("sink_tokens", 4)
    config.setdefault("recent_tokens", 32)
    config.setdefault("speculative_tokens", 3)
    return CacheLayout(page, heads, block, OscarConfig(history_bits=bits, **config))


def records(n, gen):
    """[n, 272] uint8: any codes, positive scales, zeros of either sign, NaN patterns in the padding."""
    out = torch.randint(256, (n, SLOT), generator=gen, device=DEV, dtype=torch.uint8)
    scale = torch.rand(n, 2, generator=gen, device=DEV) * 0.3 + 0.02
    zero = -7.5 * scale + torch.randn(n, 2, generator=gen, device=DEV) * 0.3
    side = torch.stack([scale, zero], 2).half().view(n, 4)
    out[:, 256:264] = side.view(torch.uint8)
    out[:, 264:] = 255
    return out


def world(lengths, qlens, layout, group, seed=1, extra_rows=0, extra_pages=1, high=False, poison=True):
    """A step of requests of ``lengths`` tokens with ``qlens`` query tokens each. Positions outside the
    history hold records of NaN scales. ``extra_rows``: padding rows behind the last token; ``high``: pages
    at the pool's end."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    heads, page, block = layout.kv_heads, layout.physical_block_tokens, layout.kernel_block_tokens
    per, cfg = layout.blocks_per_page, layout.config
    need = [-(-n // page) for n in lengths]
    pool = sum(need) + extra_pages
    order = torch.randperm(pool, generator=gen, device=DEV).tolist()
    if high:
        order = sorted(order, reverse=True)
    columns = max(max(need), 1) * per + 1
    table = torch.full((len(lengths), columns), -1, dtype=torch.int32)
    at = 0
    for r, c in enumerate(need):
        blocks = [p * per + b for p in order[at : at + c] for b in range(per)]
        table[r, : len(blocks)] = torch.tensor(blocks, dtype=torch.int32)
        at += c
    history = torch.zeros(pool, layout.stripe_page_bytes, dtype=torch.uint8, device=DEV)
    for p in order[:at]:
        history[p, : page * heads * SLOT] = records(page * heads, gen).view(-1)
    n = sum(qlens)
    s = SimpleNamespace(layout=layout, lengths=lengths, qlens=qlens, group=group, gen=gen, pool=pool,
                        history=history.view(-1), table_cpu=table, hq=heads * group)
    s.spans = []
    for length, q in zip(lengths, qlens):
        prefix = length - q
        sink = min(cfg.sink_tokens, prefix)
        s.spans.append((sink, max(sink, prefix - cfg.recent_tokens)))
    if poison:
        view = history[:, : page * heads * SLOT].view(pool, page, heads, SLOT)
        for r, (length, (lo, hi)) in enumerate(zip(lengths, s.spans)):
            for p0 in range(0, need[r] * page, page):
                inside = torch.arange(p0, p0 + page, device=DEV)
                bad = (inside < lo) | (inside >= hi)
                pg = int(table[r, p0 // block]) // per
                view[pg, bad, :, 256:264] = 255  # fp16 NaN
    s.query = (torch.randn(n + extra_rows, s.hq, 256, generator=gen, device=DEV) * 2).bfloat16()
    starts = [0]
    for q in qlens:
        starts.append(starts[-1] + q)
    tile = cfg.queries_per_tile
    tasks = [(r, q0) for r, q in enumerate(qlens) for q0 in range(0, q, tile)]
    rows = task_capacity(max(n + extra_rows, 1), max(len(lengths), 1), tile)
    listed = torch.full((max(rows, len(tasks), 1), 2), 77, dtype=torch.int32)
    if tasks:
        listed[: len(tasks)] = torch.tensor(tasks, dtype=torch.int32)
    s.meta = SimpleNamespace(
        query_start_loc=torch.tensor(starts, dtype=torch.int32, device=DEV),
        seq_lens=torch.tensor(lengths, dtype=torch.int32, device=DEV),
        block_tables=table.to(DEV), counts=torch.tensor([len(lengths), n], dtype=torch.int32, device=DEV),
        tasks=listed.to(DEV), task_count=torch.tensor([len(tasks)], dtype=torch.int32, device=DEV),
        max_num_reqs=len(lengths), num_reqs=len(lengths), max_query_len=max(qlens), layout=layout,
        num_actual_tokens=n)
    return s


def rows_of(s, r, head, positions):
    """float64 K and V values of positions of request r, and the codes and (scale, zero) of both."""
    page, per = s.layout.physical_block_tokens, s.layout.blocks_per_page
    block = s.layout.kernel_block_tokens
    heads = s.layout.kv_heads
    slot = s.meta.block_tables[r, positions // block].long() * block + positions % block
    view = s.history.view(s.pool, -1)[:, : page * heads * SLOT].unflatten(1, (page, heads, SLOT))
    rec = view[slot // page, slot % page, head]
    side = rec[:, 256:264].contiguous().view(torch.float16).double()
    out = []
    for i in (0, 1):
        packed = rec[:, 128 * i : 128 * (i + 1)]
        codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).double()
        out.append((codes, side[:, 2 * i : 2 * i + 1], side[:, 2 * i + 1 : 2 * i + 2]))
    return out


def exact(s, query, scale):
    """Per row: out and lse in 64 bits, and how far the kernel may be from them before its last rounding.

    The kernel's products of codes and queries are exact and summed in fp32 (256 terms and two more
    operations: at most 300 x 2^-24 of the sum of magnitudes), which moves a weight by e^d. The weights
    times V's scale are rounded to fp16 (2^-11, or 2^-24 of the largest scale where they are small); sums
    over L positions add at most L / 256 chunk sums of 32 terms in fp32 on a path, and the states' and
    splits' joins a few more, of the codes' part and the zeros' part each."""
    n = query.shape[0]
    out = torch.zeros(n, s.hq, 256, dtype=torch.float64, device=DEV)
    lse = torch.full((n, s.hq), -math.inf, dtype=torch.float64, device=DEV)
    slack, lse_slack = torch.zeros_like(out), torch.zeros_like(lse)
    t0, block = 0, s.layout.kernel_block_tokens
    for r, (q, (lo, hi)) in enumerate(zip(s.qlens, s.spans)):
        at = torch.arange(lo, hi, device=DEV)
        if hi > lo:
            at = at[s.meta.block_tables[r, at // block] >= 0]
        if len(at):
            for h in range(s.layout.kv_heads):
                rows = slice(h * s.group, (h + 1) * s.group)
                (kc, ks, kz), (vc, vs, vz) = rows_of(s, r, h, at)
                x = query[t0 : t0 + q, rows].double()
                score = x @ (kc * ks + kz).T * scale
                size = scale * (x.abs() @ kc.T * ks.T + x.abs().sum(-1, keepdim=True) * kz.abs().T)
                d = 300 * 2.0**-24 * size.amax(-1)
                w = score.softmax(-1)
                out[t0 : t0 + q, rows] = w @ (vc * vs + vz)
                lse[t0 : t0 + q, rows] = score.logsumexp(-1)
                codes = w @ (vs * vc)
                whole = codes + w @ vz.abs()
                sums = (64 + len(at) / 4) * 2.0**-24
                small = 15 * len(at) * 2.0**-24 * vs.amax()
                slack[t0 : t0 + q, rows] = 2.0**-11 * codes + small + (2 * d[..., None] + sums) * whole
                lse_slack[t0 : t0 + q, rows] = d + sums + 2.0**-21 * (1 + score.abs().amax(-1))
        t0 += q
    return out, lse, slack, lse_slack
