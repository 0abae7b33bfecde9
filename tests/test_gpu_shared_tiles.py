"""``kernels.shared_history`` where a plan takes tiles of 128 rows, several pieces of a row's
positions, or as many partial rows as a row may have, and values that are no numbers.

fp32 rows (``merged=False``) have no rounding of the output, so an element is off by the FP8 terms of
P alone: each of two terms rounds by at most 2^-4 of its value, 2^-8 of p s_v |c - 1.5| together (the
codes are used as 1.5 - c), and the scores' shift of tests/test_gpu_shared.py. The relative norm over
many rows is a statistic of that rounding. For p in [1, 2) the first term leaves a residual uniform
in +-2^-4, whose own step is 2^-8 in the upper half of that range (and half as much in each half
below): a variance of 2^-16 / 12 x (1/2 + 1/16 + 1/128 + ...) = 2^-16 / 12 x 4/7, over the mean p^2 of
2.16 that is (5.8e-4)^2. The bound allows 8.5e-4 of the norm of p s_v (c - 1.5), half as much again.
"""

import numpy as np
import pytest
import torch

from oscar_new_amd import kernels
from tests.test_gpu_shared import DEV, Batch, spread_requests

pytestmark = pytest.mark.gpu


def group(members, share, n, low=1, step=7):
    """One group of requests with tails of ``low``, ``low + step``, ... tokens."""
    return spread_requests((share, [low + step * (i % 61) for i in range(members)], n))


def planned(b):
    """The plan and its units as numpy [units, 8]: (block table row, first token, last row, first
    row, first position, end, slot, 16 rows)."""
    plan = kernels.prepare_shared(b.meta, b.layout, b.heads * b.g, b.starts, b.prefix)
    return plan, plan.units[: plan.unit_count.item()].cpu().numpy()


def check_cover(b, plan, units):
    """Every row's units hold each of its positions once, in slots of their own below the count that
    the merge reads. Returns the most partial rows of a row."""
    cfg = b.layout.config
    held, slots = {}, plan.token_slots.tolist()
    for req, token, end, base, lo, hi, slot, small in units.tolist():
        assert end - base <= (16 if small else 128)
        for row in range(base, end):
            held.setdefault((token + row // b.g, row % b.g), []).append((slot, lo, hi))
    at = 0
    for prefix, n in b.requests:
        begin = min(cfg.sink_tokens, prefix)
        stop = max(begin, prefix - cfg.recent_tokens)
        for token in range(at, at + n):
            assert slots[token] <= plan.slots
            for head in range(b.g):
                parts = sorted(held.get((token, head), []))
                assert [p[0] for p in parts] == list(range(slots[token]))
                spans = sorted(p[1:] for p in parts)
                ends = [begin] + [hi for _, hi in spans]
                assert [lo for lo, _ in spans] == ends[:-1] and ends[-1] == stop
        at += n
    return max(slots)


def check_rows(b, out, lse, drop=()):
    """fp32 rows against 64 bits: elements, LSE and the relative norm of all of them."""
    cfg, at = b.layout.config, 0
    far = allowed = 0.0
    for r, (prefix, n) in enumerate(b.requests):
        begin = min(cfg.sink_tokens, prefix)
        end = max(begin, prefix - cfg.recent_tokens)
        keep = np.setdiff1d(np.arange(begin, end), [p for lo, hi in drop for p in range(lo, hi)])
        rows = slice(at, at + n)
        at += n
        data = b.data[r].view(-1, b.heads, 160)[torch.from_numpy(keep).to(DEV)]
        for h in range(b.heads):
            half = []
            for o in (0, 68):
                d = data[:, h, o : o + 68]
                codes = torch.stack([d[:, :64] >> s & 3 for s in (0, 2, 4, 6)], -1).flatten(1)
                pair = d[:, 64:].contiguous().view(torch.float16).double()
                half.append((codes.double(), pair[:, :1], pair[:, 1:]))
            (kc, ks, kz), (vc, vs, vz) = half
            key, value, centred = kc * ks + kz, vc * vs + vz, (vc - 1.5).abs() * vs
            heads = slice(h * b.g, (h + 1) * b.g)
            q = b.q[rows, heads].double().reshape(-1, 256)
            score = q @ key.T.contiguous() / 16
            p = score.softmax(-1)
            want = p @ value
            shift = 2.0**-17 * q.abs().amax(-1) * key.abs().sum(1).max() / 16 + 2.0**-14
            bound = 2.0**-8 * (p @ centred) + 2 * shift[:, None] * (p @ value.abs())
            err = (out[rows, heads].double().reshape(-1, 256) - want).abs()
            assert bool((err <= bound).all()), (r, h, float((err / bound).max()))
            far += float(err.square().sum())
            allowed += float((p.square() @ centred.square()).sum())
            err = (lse[rows, heads].double().reshape(-1) - score.logsumexp(-1)).abs()
            assert bool((err <= shift).all()), (r, h, float((err / shift).max()))
    assert far**0.5 <= 8.5e-4 * allowed**0.5, (far / allowed) ** 0.5


def check_step(b, drop=()):
    rows, row_lse = b.run(merged=False)
    check_rows(b, rows[:, :, 0], row_lse[..., 0], drop)
    out, lse = b.run()
    assert torch.equal(rows[:, :, 0].bfloat16(), out) and torch.equal(row_lse[..., 0], lse)


def rewrite(b, at, values, share):
    """Bytes from ``at`` on of every record become ``values(tokens)``, the first ``share`` alike."""
    pages, bpp = b.history.view(-1, 768 * 512), b.layout.blocks_per_page
    for r, data in enumerate(b.data):
        new = values(data.shape[0])
        data[:, at : at + new.shape[1]] = new
        if r:
            data[:share] = b.data[0][:share]
        owned = b.meta.block_tables[r, ::bpp].tolist()
        for j in range(-(-data.shape[0] // 768)):
            part = data[768 * j : 768 * (j + 1)]
            pages[owned[j] // bpp, : part.numel()] = part.reshape(-1)


LARGE = {  # rows of the group's KV heads, all of more than 1024: 128-row tiles always
    "two heads, a partial last tile": dict(members=140, share=2500, n=2, heads=2, g=4),
    "a last tile that ends inside 16 rows": dict(members=211, share=3001, n=1, g=5, sink=4, recent=100),
    "no sink, one head, four tokens": dict(members=300, share=1291, n=4, g=1, sink=0, recent=97),
    "a whole chunk": dict(members=90, share=384, n=2, g=6, sink=128, recent=128),
    "32 heads": dict(members=35, share=9000, n=1, g=32),
}


@pytest.mark.parametrize("name", sorted(LARGE))
def test_tiles_of_128_rows(name):
    case = dict(LARGE[name])
    requests, groups = group(case.pop("members"), case.pop("share"), case.pop("n"), low=400)
    b = Batch(requests, groups, **case)
    plan, units = planned(b)
    shared = units[units[:, 5] <= groups[0][2]]
    assert len(shared) and not shared[:, 7].any()  # no 16-row tile holds a shared position
    assert check_cover(b, plan, units) > 1
    check_step(b)


def test_tiles_of_128_rows_of_a_group_that_may_take_either():
    requests, groups = group(128, 32000, 1, low=150, step=20)
    b = Batch(requests, groups, sink=4, recent=128)
    plan, units = planned(b)
    shared = units[units[:, 5] <= 32000]
    assert len(shared) and not shared[:, 7].any() and shared[:, 6].max() > 0  # in several pieces
    check_cover(b, plan, units)
    check_step(b)


def test_tiles_of_16_rows_of_more_rows_than_a_large_tile():
    requests, groups = spread_requests((2500, list(range(1, 400, 17)), 1))
    b = Batch(requests, groups)
    plan, units = planned(b)
    assert bool(units[:, 7].all()) and len(requests) * b.g > 128
    check_cover(b, plan, units)
    check_step(b)


@pytest.mark.parametrize("members", [8, 200])
def test_values_whose_codes_lie_close_to_their_middle(members):
    """Codes 1 and 2, as most of a row with outliers has: their own size is three times their distance
    from the middle, so the bound on the relative norm tells centred codes from the codes themselves."""
    requests, groups = group(members, 2000, 1, low=300)
    b = Batch(requests, groups)
    gen = torch.Generator(device=DEV).manual_seed(8)
    middle = torch.tensor([1, 2], dtype=torch.uint8, device=DEV)

    def codes(t):
        pick = middle[torch.randint(2, (t, 64, 4), generator=gen, device=DEV)]
        return pick[..., 0] | pick[..., 1] << 2 | pick[..., 2] << 4 | pick[..., 3] << 6

    rewrite(b, 68, codes, 2000)
    _, units = planned(b)
    assert bool(units[units[:, 5] <= 2000, 7].all()) == (members == 8)
    check_step(b)


@pytest.mark.parametrize("members", [8, 200])
def test_small_query_values_beside_large_ones(members):
    """Large values of either sign and, 2^-14 of them, small ones of one sign that add up to a seventh
    of a unit of the score: they are within the bound only if none is lost beside the large ones."""
    requests, groups = group(members, 2000, 1, low=300)
    b = Batch(requests, groups)
    gen = torch.Generator(device=DEV).manual_seed(9)

    def scale(t):  # keys of 0.8 times their codes
        return torch.tensor([0.8, 0.0], device=DEV).half().view(torch.uint8).expand(t, 4)

    rewrite(b, 64, scale, 2000)
    large = torch.randint(2, b.q.shape, generator=gen, device=DEV) * 2 - 1
    dim = torch.arange(256, device=DEV)
    b.q = torch.where(dim % 16 < 2, 128.0 * large, 2.0**-7 * (1 + dim % 2)).bfloat16()
    _, units = planned(b)
    assert bool(units[units[:, 5] <= 2000, 7].all()) == (members == 8)
    out, lse = b.run()
    b.check(out, lse)


def test_an_unmapped_block_of_a_shared_prefix():
    requests, groups = group(200, 2000, 1, low=300)
    b = Batch(requests, groups)
    b.meta.block_tables[:200, 7] = -1  # positions 896 .. 1023 of every member
    b.meta.block_tables[:200, 15] = -1  # the last shared ones, 1920 .. 1999, and 48 of their own
    _, units = planned(b)
    assert not units[units[:, 5] <= 1920, 7].any()
    check_step(b, drop=[(896, 1024), (1920, 2048)])


@pytest.mark.parametrize("slots", [4, 5, 6])
@pytest.mark.parametrize("members", [3, 175])  # tiles of 16 rows and of 128
def test_no_more_partial_rows_than_a_row_may_have(monkeypatch, slots, members):
    """Far fewer slots than the positions would fill: pieces as long as the slots ask for."""
    monkeypatch.setattr(kernels, "choose_shared_slots", lambda tokens, q_heads: slots)
    requests, groups = group(members, 40000, 1, low=400)
    b = Batch(requests, groups)
    plan, units = planned(b)
    assert plan.slots == slots
    held = check_cover(b, plan, units)
    # 312 shared chunks in slots - 2 equal pieces, and a request's own.
    assert held == slots - 1 if members == 175 else 2 <= held <= slots
    check_step(b)


def poison(b, request, position, at):
    """An infinite scale (at 64: K, at 132: V) of one record that a request reads."""
    bpp, blocks = b.layout.blocks_per_page, b.meta.block_tables[request]
    block = int(blocks[position // 128])
    row = block // bpp * (768 * b.heads * 512) + (block % bpp * 128 + position % 128) * b.heads * 160
    b.history[row + at : row + at + 2] = torch.tensor([0x00, 0x7C], dtype=torch.uint8, device=DEV)


@pytest.mark.parametrize("members", [3, 200])  # tiles of 16 rows and of 128
def test_infinite_queries_and_scales_stay_with_the_rows_that_see_them(members):
    """A score is s (q . c) + z sum q, so an infinite K scale is +inf (a NaN row) or -inf (a position of
    no weight) by the sign of q . c; an infinite V scale leaves nothing finite in a row that weighs
    it."""
    requests, groups = group(members, 1500, 1, low=700)
    b = Batch(requests, groups)
    clean, clean_lse = b.run()
    query, history = b.q.clone(), b.history.clone()
    for value in (float("inf"), float("-inf")):
        b.q[1, 2, 77] = value
        out, lse = b.run()
        assert bool(out[1, 2].isnan().all()) and not bool(lse[1, 2].isfinite())
        out[1, 2], lse[1, 2] = clean[1, 2], clean_lse[1, 2]
        assert torch.equal(out, clean) and torch.equal(lse, clean_lse)
        b.q.copy_(query)
    # Of request 2 alone, and a shared one: the leader's record is the one that is read.
    for request, position, rows in ((2, 1700, slice(2, 3)), (0, 700, slice(0, members))):
        codes = b.data[request][position, :64]
        codes = torch.stack([codes >> s & 3 for s in (0, 2, 4, 6)], -1).flatten().double()
        up = (b.q[rows].double() @ codes) > 0
        assert bool(up.any()) and not bool(up.all())
        poison(b, request, position, 64)
        out, lse = b.run()
        assert torch.equal(out[rows].isnan().all(-1), up) and torch.equal(lse[rows].isfinite(), ~up)
        assert bool(out[rows][~up].isfinite().all())
        out[rows], lse[rows] = clean[rows], clean_lse[rows]
        assert torch.equal(out, clean) and torch.equal(lse, clean_lse)
        b.history.copy_(history)
        poison(b, request, position, 132)
        out, lse = b.run()
        assert not bool(out[rows].isfinite().any()) and torch.equal(lse, clean_lse)
        out[rows] = clean[rows]
        assert torch.equal(out, clean)
        b.history.copy_(history)


def test_captured_plan_and_history_of_changing_requests():
    requests, groups = group(40, 3000, 2, low=300)
    b = Batch(requests, groups, pad=4)
    hq, m = b.heads * b.g, b.meta

    def step(q):
        plan = kernels.prepare_shared(m, b.layout, hq, b.starts, b.prefix, tokens=q.shape[0])
        return kernels.shared_history(q, b.history, m, plan, b.layout, 1 / 16)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(b.q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, lse = step(b.q)
    torch.cuda.current_stream().wait_stream(side)
    lengths = m.seq_lens.clone()
    for live, share, less in ((40, 3000, 0), (7, 3000, 0), (40, 700, 0), (33, 3000, 2500), (40, 3000, 0)):
        m.counts.copy_(torch.tensor([live, 2 * live], dtype=torch.int32))
        m.seq_lens[:40] = lengths[:40] - less
        b.prefix.fill_(share)
        b.requests = [(p - less, n) for p, n in requests]
        graph.replay()
        want, want_lse = step(b.q)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        b.check(out, lse, live=live)
