"""``kernels.shared_history`` against the softmax in 64 bits over each request's own positions.

Error bound of an output element, from the arithmetic: p s_v is two FP8 terms (each rounds by at most
2^-4 of its value, so 2^-8 of p s_v together), the output is rounded to bf16 (2^-8). The query is two
FP8 terms after scaling its largest value to [128, 256): exact but for parts below half of FP8's
smallest step, 2^-10, so at most 2^-17 of the row's largest value, which moves a score by at most
2^-17 max|q| sum|k| scale. fp32 sums and exponentials add under 2^-14 at these lengths and scores.
"""

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from oscar_new_amd import kernels
from oscar_new_amd.config import OscarConfig
from oscar_new_amd.layout import CacheLayout

pytestmark = pytest.mark.gpu
DEV = "cuda"


def records(n, gen):
    """[n, 160] records of random codes, scales of 0.2 to 0.9 and zeros about minus 1.5 of them."""
    out = torch.randint(0, 256, (n, 160), generator=gen, device=DEV, dtype=torch.uint8)
    for at in (64, 132):
        scale = torch.rand(n, 1, generator=gen, device=DEV) * 0.7 + 0.2
        zero = -1.5 * scale + 0.2 * torch.randn(n, 1, generator=gen, device=DEV)
        out[:, at : at + 4] = torch.cat([scale, zero], 1).half().view(torch.uint8)
    return out


class Batch:
    """Requests (cached tokens, query tokens) whose groups share prefixes: ``groups`` is a list of
    (first request, end, shared tokens). Slots that no request holds are 0xFF (NaN scales)."""

    def __init__(self, requests, groups, heads=1, g=6, sink=64, recent=256, page=768, seed=1,
                 pad=0, spare=2, spread=2.0):
        cfg = OscarConfig(sink_tokens=sink, recent_tokens=recent, speculative_tokens=3)
        self.layout = CacheLayout(page, kv_heads=heads, config=cfg)
        self.requests, self.heads, self.g = requests, heads, g
        gen = torch.Generator(device=DEV).manual_seed(seed)
        bpp = self.layout.blocks_per_page
        total = [p + n for p, n in requests]
        need = [-(-t // page) for t in total]
        pool = sum(need) + 1
        order = 1 + np.random.default_rng(seed).permutation(pool - 1)
        owned, at = [], 0
        for n in need:
            owned.append([int(p) for p in order[at : at + n]])
            at += n
        self.history = torch.full((pool, page * heads * 512), 0xFF, dtype=torch.uint8, device=DEV)
        row = heads * 160
        for r, t in enumerate(total):
            data = records(t * heads, gen).view(t, row)
            lead = next((a for a, b, s in groups if a < r < b), None)
            if lead is not None:  # the leader's first tokens, in shared pages or copies
                share = next(s for a, b, s in groups if a < r < b)
                share = max(0, min(share, t, total[lead]))
                data[:share] = self.data[lead][:share]
                for j in range(1, share // page):
                    owned[r][j] = owned[lead][j]
            if r == 0:
                self.data = []
            self.data.append(data)
            for j, p in enumerate(owned[r]):
                part = data[j * page : (j + 1) * page]
                self.history[p, : part.shape[0] * row] = part.reshape(-1)
        self.history = self.history.view(-1)
        count = len(requests)
        table = np.full((count + spare, bpp * (max(need) + 1)), -1, np.int32)
        for r, pages in enumerate(owned):
            for j, p in enumerate(pages):
                table[r, j * bpp : (j + 1) * bpp] = p * bpp + np.arange(bpp)
        starts = np.concatenate([[0], np.cumsum([n for _, n in requests])])
        tokens = int(starts[-1])
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        self.meta = SimpleNamespace(
            query_start_loc=i32(list(starts) + [tokens] * spare), seq_lens=i32(total + [0] * spare),
            block_tables=torch.from_numpy(table).to(DEV), counts=i32([count, tokens]),
            num_reqs=count, max_num_reqs=count + spare, num_actual_tokens=tokens + pad)
        self.q = (spread * torch.randn(tokens + pad, heads * g, 256, generator=gen, device=DEV)
                  ).bfloat16()
        bounds = sorted({a for a, _, _ in groups} | {b for _, b, _ in groups}) or [0]
        sizes = {(a, b): s for a, b, s in groups}
        self.starts = i32(bounds)
        self.prefix = i32([sizes.get(pair, 0) for pair in zip(bounds, bounds[1:])])

    def run(self, starts=None, prefix=None, **options):
        plan = kernels.prepare_shared(self.meta, self.layout, self.heads * self.g,
                                      self.starts if starts is None else starts,
                                      self.prefix if prefix is None else prefix)
        return kernels.shared_history(self.q, self.history, self.meta, plan, self.layout, 1 / 16,
                                      **options)

    def check(self, out, lse, live=None, drop=()):
        """``drop``: (request, first, end) positions whose blocks are unmapped."""
        cfg, at = self.layout.config, 0
        for r, (prefix, n) in enumerate(self.requests[:live]):
            begin = min(cfg.sink_tokens, prefix)
            end = max(begin, prefix - cfg.recent_tokens)
            keep = [p for p in range(begin, end)
                    if not any(r == d[0] and d[1] <= p < d[2] for d in drop)]
            rows = slice(at, at + n)
            at += n
            if not keep:
                assert not bool(out[rows].any()) and bool((lse[rows] == -torch.inf).all())
                continue
            data = self.data[r].view(-1, self.heads, 160)[keep]
            for h in range(self.heads):
                half = []
                for b in (0, 68):
                    d = data[:, h, b : b + 68]
                    codes = torch.stack([d[:, :64] >> s & 3 for s in (0, 2, 4, 6)], -1).flatten(1)
                    pair = d[:, 64:].contiguous().view(torch.float16).double()
                    half.append((codes.double(), pair[:, :1], pair[:, 1:]))
                (kc, ks, kz), (vc, vs, vz) = half
                key, value = kc * ks + kz, vc * vs + vz
                heads = slice(h * self.g, (h + 1) * self.g)
                q = self.q[rows, heads].double()
                score = torch.einsum("tgd,pd->tgp", q, key) / 16
                p = score.softmax(-1)
                want = p @ value
                shift = 2.0**-17 * q.abs().amax(-1) * key.abs().sum(1).max() / 16 + 2.0**-14
                bound = (2.0**-8 * (want.abs() + p @ (vc * vs)) + 2 * shift[..., None]
                         * (p @ value.abs()))
                err = (out[rows, heads].double() - want).abs()
                assert bool((err <= bound).all()), (r, h, float((err / bound).max()))
                err = (lse[rows, heads].double() - score.logsumexp(-1)).abs()
                assert bool((err <= shift).all()), (r, h, float((err / shift).max()))
        assert not bool(out[at:].any()) and bool((lse[at:] == -torch.inf).all())


def spread_requests(*parts):
    """(shared tokens, own token counts, query tokens) per group -> requests and groups."""
    requests, groups = [], []
    for share, own, n in parts:
        groups.append((len(requests), len(requests) + len(own), share))
        requests += [(share + o, n) for o in own]
    return requests, groups


CASES = {
    "two of a short prompt": [(500, [300, 301], 1)],
    "prefix inside the recent window": [(200, [10, 20, 30], 1)],
    "prefix below the sink": [(40, [900, 700], 1)],
    "one chunk": [(128, [600, 500, 800], 1)],
    "ragged": [(3001, [1, 255, 256, 257, 900, 2000, 5], 1)],
    "more rows than a tile": [(2500, list(range(1, 400, 17)), 1)],
    "mtp": [(2500, [300, 10, 555], 4), (1000, [1, 2, 1200], 4)],
    "a group of one and an empty request": [(1500, [700], 1), (0, [0, 0, 900], 2)],
    "long": [(40000, [1500, 90, 700], 1)],
}


@pytest.mark.parametrize("name", sorted(CASES))
@pytest.mark.parametrize("heads,g,sink,recent", [(1, 6, 64, 256), (2, 4, 4, 128), (1, 1, 0, 97)])
def test_rows_against_64_bits(name, heads, g, sink, recent):
    requests, groups = spread_requests(*CASES[name])
    b = Batch(requests, groups, heads=heads, g=g, sink=sink, recent=recent, pad=3)
    out, lse = b.run()
    b.check(out, lse)
    rows, row_lse = b.run(merged=False)
    assert rows.dtype == torch.float32 and tuple(rows.shape) == (*out.shape[:2], 1, 256)
    assert torch.equal(rows[:, :, 0].bfloat16(), out) and torch.equal(row_lse[..., 0], lse)


@pytest.mark.parametrize("g,page", [(8, 384), (3, 1536), (32, 768)])
def test_group_sizes_and_pages(g, page):
    requests, groups = spread_requests((2000, [400, 3, 1200], 2), (700, [50, 800], 2))
    b = Batch(requests, groups, g=g, page=page, sink=4, recent=100)
    b.check(*b.run())


def test_chunk_steps_of_many_query_tokens():
    requests = [(3000, 1), (3300, 57), (2900, 3), (500, 130), (0, 40)]
    b = Batch(requests, [(0, 3, 2800)], seed=4)
    b.check(*b.run())


def test_requests_outside_the_groups_share_nothing():
    requests = [(900, 1), (2000, 1), (2100, 1), (2500, 1), (700, 2), (3000, 1)]
    b = Batch(requests, [(1, 4, 1900)], seed=6)
    b.check(*b.run())


def test_starts_that_are_no_partition_share_nothing():
    requests, groups = spread_requests((1500, [300, 400, 500, 600], 1))
    b = Batch(requests, groups)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    for starts, prefix in (([0, 3, 1, 4], [1500] * 3), ([4, 0], [1500]),
                           ([-9, 2, 99], [1500, 1500]), ([0, 4], [-5]), ([0], []),
                           ([2, 2, 2], [1500, 1500])):
        b.check(*b.run(i32(starts), i32(prefix)))
    # A shared part is never longer than every member's history.
    b.check(*b.run(i32([0, 4]), i32([1500])))
    same = Batch([(1500, 1)] * 3, [(0, 3, 1500)])
    same.check(*same.run(i32([0, 3]), i32([1 << 30])))


def test_fewer_live_requests_and_tokens_than_rows():
    requests, groups = spread_requests((2000, [300, 400, 500, 600], 2))
    b = Batch(requests, groups)
    for live in (3, 1, 0):
        b.meta.counts.copy_(torch.tensor([live, 2 * live], dtype=torch.int32))
        out, lse = b.run()
        b.check(out, lse, live=live)


def test_an_unmapped_block_holds_no_tokens():
    requests, groups = spread_requests((2000, [900, 400], 1))
    b = Batch(requests, groups)
    b.meta.block_tables[0, 17] = -1  # positions 2176 .. 2303, behind the shared ones
    b.check(*b.run(), drop=[(0, 2176, 2304)])


@pytest.mark.parametrize("members", [3, 200])
def test_nan_in_a_query_stays_in_its_row(members):
    requests, groups = spread_requests((1500, [300] * members, 1))
    b = Batch(requests, groups)
    clean, clean_lse = b.run()
    b.q[1, 2, 77] = float("nan")
    out, lse = b.run()
    assert bool(out[1, 2].isnan().all()) and bool(lse[1, 2].isnan())
    out[1, 2], lse[1, 2] = clean[1, 2], clean_lse[1, 2]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


def test_agrees_with_the_unshared_launches():
    requests, groups = spread_requests((5000, [700] * 20, 1))
    b = Batch(requests, groups)
    out, lse = b.run()
    m = b.meta
    m.max_query_len = 1
    m.tasks = torch.zeros(64, 2, dtype=torch.int32, device=DEV)
    m.task_count = torch.zeros(1, dtype=torch.int32, device=DEV)
    kernels.prepare_tasks(m.query_start_loc, m.counts, m.tasks, m.task_count, m.max_num_reqs, 4)
    hp, hl = kernels.attention_partials(b.q, None, None, b.history, b.history, m, b.layout,
                                        1 / 16, 8, False)
    want, want_lse = kernels.merge_splits(hp, hl, m.counts)
    assert float((lse - want_lse).abs().max()) < 1e-4
    assert float((out.float() - want.float()).norm() / want.float().norm()) < 5e-3


def test_captured_step_with_a_plan_filled_again():
    requests, groups = spread_requests((2000, [300, 400, 500], 1), (900, [100, 800], 1))
    b = Batch(requests, groups)
    hq = b.heads * b.g
    plan = kernels.prepare_shared(b.meta, b.layout, hq, b.starts, b.prefix)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.shared_history(b.q, b.history, b.meta, plan, b.layout, 1 / 16)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, lse = kernels.shared_history(b.q, b.history, b.meta, plan, b.layout, 1 / 16)
    torch.cuda.current_stream().wait_stream(side)
    for share in ([2000, 900], [700, 0], [0, 300], [2000, 900]):
        b.prefix.copy_(torch.tensor(share, dtype=torch.int32))
        kernels.prepare_shared(b.meta, b.layout, hq, b.starts, b.prefix, out=plan)
        graph.replay()
        want, want_lse = kernels.shared_history(b.q, b.history, b.meta, plan, b.layout, 1 / 16)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        b.check(out, lse)


def test_two_streams_use_one_plan_at_once():
    requests, groups = spread_requests((3000, [300] * 30, 1), (900, [100, 800], 1))
    b = Batch(requests, groups)
    plan = kernels.prepare_shared(b.meta, b.layout, 6, b.starts, b.prefix)
    queries = [b.q, b.q.flip(0).contiguous()]
    want = [kernels.shared_history(q, b.history, b.meta, plan, b.layout, 1 / 16) for q in queries]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in queries]
    got = []
    for _ in range(5):
        for q, side in zip(queries, sides):
            with torch.cuda.stream(side):
                got.append(kernels.shared_history(q, b.history, b.meta, plan, b.layout, 1 / 16))
    torch.cuda.synchronize()
    for i, (out, lse) in enumerate(got):
        assert torch.equal(out, want[i % 2][0]) and torch.equal(lse, want[i % 2][1])


def test_tokens_of_no_request_hold_nothing():
    requests, groups = spread_requests((900, [300, 400], 1))
    b = Batch(requests, groups, pad=5)
    b.meta.counts[1] += 5  # live by the count, but behind the last request's
    out, lse = b.run()
    b.check(out, lse)
    b.meta.counts[0] = 0
    out, lse = b.run()
    assert not bool(out.any()) and bool((lse == -torch.inf).all())


@pytest.mark.parametrize("qlen,reqs", [(1, 600), (200, 100)])
def test_units_longer_than_their_offset_tables_far_in_a_pool(qlen, reqs):
    """Requests that map the same 300000 tokens in pages beyond 4 GB of records and declare nothing
    shared: more rows than the chip holds, so each unit is a whole row tile's positions. Either
    tile's lanes add a quarter of the positions one by one, each sum off by at most 2^-24 of it."""
    layout = CacheLayout(768, kv_heads=1, config=OscarConfig(sink_tokens=64, recent_tokens=256,
                                                             speculative_tokens=3))
    prefix, page = 300000, 768
    need, pool = -(-(prefix + qlen) // page), 12000
    gen = torch.Generator(device=DEV).manual_seed(3)
    data = records(need * page, gen)
    order = pool - 1 - torch.randperm(need, generator=gen, device=DEV)
    order[::5] = torch.arange(order[::5].numel(), device=DEV)  # and at the pool's start
    history = torch.empty(pool, page * 512, dtype=torch.uint8, device=DEV)
    history[order, : page * 160] = data.view(need, page * 160)
    bpp = layout.blocks_per_page
    row = (order[:, None] * bpp + torch.arange(bpp, device=DEV)).flatten().int()
    tokens = reqs * qlen
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    meta = SimpleNamespace(
        query_start_loc=i32(range(0, tokens + 1, qlen)), seq_lens=i32([prefix + qlen] * reqs),
        block_tables=row.expand(reqs, -1).contiguous(), counts=i32([reqs, tokens]), num_reqs=reqs,
        max_num_reqs=reqs, num_actual_tokens=tokens)
    q = (12 * torch.randn(tokens, 6, 256, generator=gen, device=DEV)).bfloat16()
    none = i32([])
    plan = kernels.prepare_shared(meta, layout, 6, i32([0]), none)
    units = plan.units[: plan.unit_count.item()]
    assert bool((units[:, 5] - units[:, 4] == prefix - 256 - 64).all())
    assert bool((units[:, 7] == (qlen == 1)).all())
    out, lse = kernels.shared_history(q, history.view(-1), meta, plan, layout, 1 / 16)
    half = []
    for b in (0, 68):
        d = data[64 : prefix - 256, b : b + 68]
        codes = torch.stack([d[:, :64] >> s & 3 for s in (0, 2, 4, 6)], -1).flatten(1).double()
        pair = d[:, 64:].contiguous().view(torch.float16).double()
        half.append((codes, pair[:, :1], pair[:, 1:]))
    (kc, ks, kz), (vc, vs, vz) = half
    key, value, spread = kc * ks + kz, vc * vs + vz, vc * vs
    rows = [0, tokens // 2, tokens - 1]
    picked = q[rows].double().view(-1, 256)
    score = picked @ key.T.contiguous() / 16
    p = score.softmax(-1)
    want = p @ value
    shift = (2.0**-17 * picked.abs().amax(-1) * key.abs().sum(1).max() / 16 + 2.0**-14
             + prefix / 4 * 2.0**-24)
    bound = 2.0**-8 * (want.abs() + p @ spread) + 2 * shift[:, None] * (p @ value.abs())
    err = (out[rows].double().view(-1, 256) - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    err = (lse[rows].double().view(-1) - score.logsumexp(-1)).abs()
    assert bool((err <= shift).all()), float((err / shift).max())


def test_refusals():
    requests, groups = spread_requests((600, [300, 400], 1))
    b = Batch(requests, groups)
    plan = kernels.prepare_shared(b.meta, b.layout, 6, b.starts, b.prefix)
    with pytest.raises(ValueError):
        kernels.prepare_shared(b.meta, b.layout, 6, b.starts, b.prefix[:0])
    with pytest.raises(ValueError):
        kernels.prepare_shared(b.meta, b.layout, 6, b.starts.long(), b.prefix)
    with pytest.raises(ValueError):
        kernels.prepare_shared(b.meta, b.layout, 0, b.starts, b.prefix)
    with pytest.raises(ValueError):
        kernels.prepare_shared(b.meta, b.layout, 12, b.starts, b.prefix, out=plan)
    with pytest.raises(ValueError):
        kernels.prepare_shared(b.meta, b.layout, 33, b.starts, b.prefix)
    for name in ("seq_lens", "counts", "query_start_loc"):
        good = getattr(b.meta, name)
        for bad, error in ((good.cpu(), RuntimeError), (good.long(), ValueError),
                           (good[:1], ValueError)):
            setattr(b.meta, name, bad)
            with pytest.raises(error):
                kernels.prepare_shared(b.meta, b.layout, 6, b.starts, b.prefix)
        setattr(b.meta, name, good)
    many = torch.zeros(9001, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        kernels.prepare_shared(b.meta, b.layout, 6, many, many[1:])
    call = kernels.shared_history
    with pytest.raises(ValueError):
        call(torch.cat([b.q, b.q]), b.history, b.meta, plan, b.layout, 1 / 16)
    with pytest.raises(ValueError):
        call(b.q[:, :3], b.history, b.meta, plan, b.layout, 1 / 16)
    with pytest.raises(ValueError):
        call(b.q, b.history.view(torch.int16), b.meta, plan, b.layout, 1 / 16)
    table = b.meta.block_tables
    for bad in (table[:3], table.T, table.long()):
        b.meta.block_tables = bad
        with pytest.raises(ValueError):
            call(b.q, b.history, b.meta, plan, b.layout, 1 / 16)
    b.meta.block_tables = table
    with pytest.raises(ValueError):
        call(b.q, b.history, b.meta, plan, CacheLayout(1536), 1 / 16)
    none = kernels.prepare_shared(b.meta, b.layout, 6, b.starts, b.prefix, tokens=0)
    with pytest.raises(ValueError):
        call(b.q[:1], b.history, b.meta, none, b.layout, 1 / 16)
    for scale in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            call(b.q, b.history, b.meta, plan, b.layout, scale)
    with pytest.raises(RuntimeError):
        call(b.q.cpu(), b.history, b.meta, plan, b.layout, 1 / 16)
    out, lse = call(b.q[:0], b.history, b.meta, plan, b.layout, 1 / 16)
    assert tuple(out.shape) == (0, 6, 256) and tuple(lse.shape) == (0, 6)
