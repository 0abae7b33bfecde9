"""Page forks and compaction (``oscar_new_amd.pages``) against a plain restatement, every byte of
every layer's stripes compared."""

import numpy as np
import pytest
import torch

from oscar_new_amd import pages
from oscar_new_amd.config import OscarConfig
from oscar_new_amd.layout import CacheLayout

pytestmark = pytest.mark.gpu
DEV = "cuda"


class World:
    """Caches of random bytes, requests whose pages lie anywhere, and the same state in numpy."""

    def __init__(self, lengths, pool=40, layers=2, page=768, heads=1, sink=64, recent=256, rows=None,
                 seed=5):
        cfg = OscarConfig(sink_tokens=sink, recent_tokens=recent, speculative_tokens=3)
        self.layout = CacheLayout(page, kv_heads=heads, config=cfg)
        self.bpp, self.pool, self.layers = self.layout.blocks_per_page, pool, layers
        gen = torch.Generator(device=DEV).manual_seed(seed)
        shape = (pool * self.bpp, 128, heads, 256)
        self.caches = []
        for _ in range(layers):
            pair = []
            for _ in range(2):
                raw = torch.randint(0, 256, (pool * self.layout.stripe_page_bytes,), generator=gen,
                                    device=DEV, dtype=torch.uint8)
                pair.append(raw.view(torch.bfloat16).view(shape))
            self.caches.append(tuple(pair))
        self.handle = pages.PageCaches(self.caches, self.layout)
        order = np.random.default_rng(seed).permutation(pool)
        rows = rows or len(lengths) + 4
        self.owned, at = [], 0
        table = np.full((rows, self.bpp * (max(self.need(n) for n in lengths) + 2)), -1, np.int32)
        for r, n in enumerate(lengths):
            self.owned.append([int(p) for p in order[at : at + self.need(n)]])
            at += self.need(n)
            self.map(table, r, self.owned[-1])
        self.table = torch.from_numpy(table).to(DEV)
        self.seq_lens = torch.tensor(list(lengths) + [0] * (rows - len(lengths)), dtype=torch.int32,
                                     device=DEV)
        self.counts = torch.tensor([len(lengths), 0], dtype=torch.int32, device=DEV)
        self.lengths = list(lengths)

    def need(self, n):
        return -(-n // self.layout.physical_block_tokens)

    def map(self, table, r, owned):
        for j, p in enumerate(owned):
            table[r, j * self.bpp : (j + 1) * self.bpp] = p * self.bpp + np.arange(self.bpp)

    def stripes(self):
        return [[t.reshape(-1).view(torch.uint8).cpu().numpy().reshape(self.pool, -1).copy()
                 for t in pair] for pair in self.caches]

    def copy(self, stripes, src, dst, slots, length):
        """The copy of one page in numpy: records, then the window rows of live positions."""
        lay, cfg = self.layout, self.layout.config
        row = lay.kv_heads * 1024
        for k, v in stripes:
            end = slots * lay.kv_heads * 160
            k[dst, :end] = k[src, :end]
            live = [p for p in range(length)
                    if p < cfg.sink_tokens or p >= max(cfg.sink_tokens, length - cfg.ring_tokens)]
            for e in {lay.window_index(p) for p in live}:
                v[dst, e * row : (e + 1) * row] = v[src, e * row : (e + 1) * row]

    def check(self, want):
        for got, exp in zip(self.stripes(), want):
            assert np.array_equal(got[0], exp[0]) and np.array_equal(got[1], exp[1])


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def fork(w, parents, children, fresh):
    return pages.fork_requests(w.handle, w.table, w.seq_lens, i32(parents), i32(children),
                               i32(fresh).view(-1, 2))


def expect_fork(w, stripes, table, seq, parent, child, fresh):
    n, row = w.lengths[parent], list(w.owned[parent])
    bp = w.layout.physical_block_tokens
    if row:
        w.copy(stripes, row[0], fresh[0], min(n, bp), n)
        if len(row) > 1 and n % bp:
            w.copy(stripes, row[-1], fresh[1], n % bp, 0)
            row[-1] = fresh[1]
        row[0] = fresh[0]
    w.map(table, child, row)
    seq[child] = n


LENGTHS = [1, 63, 64, 65, 300, 323, 324, 325, 767, 768, 769, 1536, 1537, 3000, 0]


@pytest.mark.parametrize("heads,page,sink,recent", [(1, 768, 64, 256), (2, 768, 4, 128),
                                                    (1, 256, 0, 97), (3, 1536, 64, 256)])
@pytest.mark.parametrize("length", LENGTHS)
def test_fork_copies_what_the_parent_holds(length, heads, page, sink, recent):
    w = World([length, 500], pool=32, page=page, heads=heads, sink=sink, recent=recent)
    free, count = pages.free_pages(w.handle, w.table, w.seq_lens, w.counts)
    taken = {p for row in w.owned for p in row}
    want = [p for p in range(w.pool) if p not in taken]
    assert free.tolist() == want + [-1] * len(taken) and count.item() == len(want)
    stripes, table, seq = w.stripes(), w.table.cpu().numpy(), w.seq_lens.cpu().numpy()
    table_before = table.copy()
    for i, child in enumerate((3, 2)):
        expect_fork(w, stripes, table, seq, 0, child, want[2 * i : 2 * i + 2])
    status = pages.fork_requests(w.handle, w.table, w.seq_lens, i32([0, 0]), i32([3, 2]),
                                 free[:4].view(2, 2))
    assert status.tolist() == [1, 1]
    assert np.array_equal(w.table.cpu().numpy(), table)
    assert np.array_equal(w.seq_lens.cpu().numpy(), seq)
    assert np.array_equal(table[:2], table_before[:2])
    w.check(stripes)


def test_fork_of_a_fork_and_free_pages_after_it():
    w = World([2000, 10], pool=20)
    free = pages.free_pages(w.handle, w.table, w.seq_lens, w.counts)[0].tolist()
    assert fork(w, [0], [2], [free[:2]]).tolist() == [1]
    w.owned.append([free[0], w.owned[0][1], free[1]])
    w.lengths.append(2000)
    w.counts[0] = 3
    free = pages.free_pages(w.handle, w.table, w.seq_lens, w.counts)[0].tolist()
    stripes, table, seq = w.stripes(), w.table.cpu().numpy(), w.seq_lens.cpu().numpy()
    expect_fork(w, stripes, table, seq, 2, 3, free[:2])
    assert fork(w, [2], [3], [free[:2]]).tolist() == [1]
    assert np.array_equal(w.table.cpu().numpy(), table)
    w.check(stripes)


def test_refused_forks_write_nothing():
    w = World([1000, 700, 769], pool=12, rows=8)
    free = pages.free_pages(w.handle, w.table, w.seq_lens, w.counts)[0].tolist()
    a, b, c, d = free[:4]
    own = w.owned[0]
    stripes, table, seq = w.stripes(), w.table.cpu().numpy(), w.seq_lens.cpu().numpy()
    calls = [  # every fork of these calls is refused but for the ones listed as done
        ([0], [3], [[-1, b]], [0]),
        ([0], [3], [[a, a]], [0]),
        ([0], [3], [[a, 12]], [0]),
        ([0], [3], [[a, own[1]]], [0]),
        ([0], [3], [[own[0], a]], [0]),
        ([8], [3], [[a, b]], [0]),
        ([-1], [3], [[a, b]], [0]),
        ([0], [8], [[a, b]], [0]),
        ([0], [-3], [[a, b]], [0]),
        ([0], [0], [[a, b]], [0]),
    ]
    for parents, children, fresh, want in calls:
        assert fork(w, parents, children, fresh).tolist() == want
    assert np.array_equal(w.table.cpu().numpy(), table)
    assert np.array_equal(w.seq_lens.cpu().numpy(), seq)
    w.check(stripes)
    # A child that is another fork's parent, a child twice, a page twice: the later entry (and the
    # fork whose parent changes) is refused, the others are carried out.
    status = fork(w, [1, 3, 2, 2, 2], [3, 4, 5, 5, 6], [[a, -1], [b, c], [c, d], [b, 11], [d, b]])
    assert status.tolist() == [1, 0, 0, 0, 0]
    expect_fork(w, stripes, table, seq, 1, 3, [a, -1])
    assert np.array_equal(w.table.cpu().numpy(), table)
    w.check(stripes)


def test_fork_refuses_a_parent_page_outside_the_pool():
    w = World([2000], pool=12, rows=4)
    w.table[0, w.bpp] = 12 * w.bpp
    free = [p for p in range(12) if p not in w.owned[0]]
    before = w.table.clone()
    assert fork(w, [0], [1], [free[:2]]).tolist() == [0]
    w.seq_lens[0] = 1 << 30  # more tokens than the table has columns for
    w.table[0] = before[0] % (12 * w.bpp)
    assert fork(w, [0], [1], [free[:2]]).tolist() == [0]
    assert torch.equal(w.table[1:], before[1:]) and w.seq_lens[1].item() == 0


def expect_compact(w, rows):
    bp = w.layout.physical_block_tokens
    slots, length = {}, {}
    for r in rows:
        for j, p in enumerate(w.owned[r]):
            slots[p] = max(slots.get(p, 0), min(bp, w.lengths[r] - j * bp))
            if j == 0:
                length[p] = w.lengths[r]
    holes = [p for p in range(len(slots)) if p not in slots]
    place = dict(zip(sorted(p for p in slots if p >= len(slots)), holes))
    stripes = w.stripes()
    for src, dst in place.items():
        w.copy(stripes, src, dst, slots[src], length.get(src, 0))
    table = w.table.cpu().numpy().copy()
    for r in rows:
        w.map(table, r, [place.get(p, p) for p in w.owned[r]])
    return stripes, table, len(slots)


@pytest.mark.parametrize("heads,page,sink,recent", [(1, 768, 64, 256), (2, 256, 4, 97)])
@pytest.mark.parametrize("lengths,live", [([3000, 1, 768, 769, 0, 324], 6), ([2500, 700], 1),
                                          ([90], 0), ([5], 1)])
def test_compaction(lengths, live, heads, page, sink, recent):
    w = World(lengths, pool=48, page=page, heads=heads, sink=sink, recent=recent)
    w.counts[0] = live
    stripes, table, total = expect_compact(w, range(live))
    before = w.table.clone()
    tables, count = pages.compact_pages(w.handle, w.table, w.seq_lens, w.counts)
    assert count.item() == total and np.array_equal(tables.cpu().numpy(), table)
    assert torch.equal(w.table, before)
    w.check(stripes)
    free = pages.free_pages(w.handle, tables, w.seq_lens, w.counts)[0]
    assert free[: 48 - total].tolist() == list(range(total, 48))


def test_compaction_keeps_shared_pages_shared():
    w = World([2000, 800], pool=30)
    w.owned.append([None, w.owned[0][1], None])
    w.lengths.append(2000)
    taken = set(w.owned[0] + w.owned[1])
    w.owned[2][0], w.owned[2][2] = [p for p in range(29, -1, -1) if p not in taken][:2]
    table = w.table.cpu().numpy()
    w.map(table, 2, w.owned[2])
    w.table.copy_(torch.from_numpy(table))
    w.seq_lens[2] = 2000
    w.counts[0] = 3
    stripes, table, total = expect_compact(w, range(3))
    tables, count = pages.compact_pages(w.handle, w.table, w.seq_lens, w.counts)
    assert count.item() == total == 7 and np.array_equal(tables.cpu().numpy(), table)
    w.check(stripes)


def test_large_pool_spans_several_scan_rounds():
    # One layer of small pages: 5000 pages, requests at both ends.
    w = World([700, 3000], pool=5000, layers=1, page=128, sink=0, recent=33)
    w.check(w.stripes())
    stripes, table, total = expect_compact(w, range(2))
    tables, count = pages.compact_pages(w.handle, w.table, w.seq_lens, w.counts)
    assert count.item() == total and np.array_equal(tables.cpu().numpy(), table)
    w.check(stripes)
    free, count = pages.free_pages(w.handle, w.table, w.seq_lens, w.counts)
    taken = {p for row in w.owned for p in row}
    assert free[: count.item()].tolist() == [p for p in range(5000) if p not in taken]


def test_pages_beyond_four_gigabytes():
    layout = CacheLayout(768, kv_heads=1, config=OscarConfig(speculative_tokens=3))
    pool, bpp, length = 12000, layout.blocks_per_page, 2 * 768 + 100
    assert pool * layout.stripe_page_bytes > 1 << 32
    stripes = [torch.empty(pool, layout.stripe_page_bytes, dtype=torch.uint8, device=DEV)
               for _ in range(2)]
    shape = (pool * bpp, 128, 1, 256)
    caches = pages.PageCaches([tuple(t.view(torch.bfloat16).view(shape) for t in stripes)], layout)
    owned = [11990, 11800, 11950]
    gen = torch.Generator(device=DEV).manual_seed(9)
    for t in stripes:
        t[owned] = torch.randint(0, 256, (3, t.shape[1]), generator=gen, device=DEV,
                                 dtype=torch.uint8)
    blocks = [p * bpp + b for p in owned for b in range(bpp)]
    table, seq = i32([blocks, [-1] * len(blocks)]), i32([length, 0])
    status = pages.fork_requests(caches, table, seq, i32([0]), i32([1]), i32([[11000, 11999]]))
    assert status.tolist() == [1] and seq.tolist() == [length] * 2
    assert table[1].tolist() == [p * bpp + b for p in (11000, 11800, 11999) for b in range(bpp)]
    (history, window), cfg = stripes, layout.config
    rows = (cfg.sink_tokens + cfg.ring_tokens) * 1024

    def alike(first, last):
        assert torch.equal(history[first, : 768 * 160], history[11990, : 768 * 160])
        assert torch.equal(window[first, :rows], window[11990, :rows])
        assert torch.equal(history[last, : 100 * 160], history[11950, : 100 * 160])

    alike(11000, 11999)
    # In use: 11000, 11800, 11950, 11990, 11999 -> pages 0 to 4 in that order.
    tables, live = pages.compact_pages(caches, table, seq, i32([2, 0]))
    assert live.item() == 5
    assert tables[0].tolist() == [p * bpp + b for p in (3, 1, 2) for b in range(bpp)]
    assert tables[1].tolist() == [p * bpp + b for p in (0, 1, 4) for b in range(bpp)]
    alike(0, 4)
    alike(3, 2)
    assert torch.equal(history[1, : 768 * 160], history[11800, : 768 * 160])


def test_captured_fork_replays_with_new_rows():
    w = World([1000, 700], pool=20, rows=6)
    parents, children = i32([0, 1]), i32([2, 3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        free, _ = pages.free_pages(w.handle, w.table, w.seq_lens, w.counts)
        return pages.fork_requests(w.handle, w.table, w.seq_lens, parents, children,
                                   free[:4].view(2, 2))

    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            status = step()
    torch.cuda.current_stream().wait_stream(side)
    free = [p for p in range(20) if p not in w.owned[0] + w.owned[1]]
    for kids in ([2, 3], [5, 4], [3, 5]):
        children.copy_(i32(kids))
        table, seq = w.table.cpu().numpy(), w.seq_lens.cpu().numpy()
        stripes = w.stripes()
        for i, child in enumerate(kids):
            expect_fork(w, stripes, table, seq, i, child, free[2 * i : 2 * i + 2])
        graph.replay()
        torch.cuda.synchronize()
        assert status.tolist() == [1, 1]
        assert np.array_equal(w.table.cpu().numpy(), table)
        w.check(stripes)


def test_captured_compaction_replays():
    w = World([1500, 300, 900], pool=30, rows=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pages.compact_pages(w.handle, w.table, w.seq_lens, w.counts)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            tables, live = pages.compact_pages(w.handle, w.table, w.seq_lens, w.counts)
    torch.cuda.current_stream().wait_stream(side)
    for count in (3, 1, 2, 3):
        w.counts[0] = count
        stripes, table, total = expect_compact(w, range(count))
        graph.replay()
        torch.cuda.synchronize()
        assert live.item() == total and np.array_equal(tables.cpu().numpy(), table)
        w.check(stripes)


def test_refusals():
    w = World([100], pool=4)
    other = World([100], pool=6)
    with pytest.raises(ValueError):
        pages.PageCaches([], w.layout)
    with pytest.raises(ValueError):
        pages.PageCaches([w.caches[0], other.caches[0]], w.layout)
    with pytest.raises(RuntimeError):
        pages.PageCaches([tuple(t.cpu() for t in w.caches[0])], w.layout)
    good = (w.handle, w.table, w.seq_lens, w.counts)
    for bad in ((w.handle, w.table.long(), *good[2:]), (w.handle, w.table.T, *good[2:]),
                (w.handle, w.table[0], *good[2:]), (w.handle, w.table, w.seq_lens[:2], w.counts),
                (w.handle, w.table, w.seq_lens.long(), w.counts),
                (w.handle, w.table, w.seq_lens, w.counts.long())):
        for call in (pages.free_pages, pages.compact_pages):
            with pytest.raises(ValueError):
                call(*bad)
    lists = [i32([0]), i32([1]), i32([[2, 3]])]
    for i, bad in ((0, i32([0, 1])), (1, i32([[1]])), (2, i32([2, 3])), (2, lists[2].long())):
        args = list(lists)
        args[i] = bad
        with pytest.raises(ValueError):
            pages.fork_requests(w.handle, w.table, w.seq_lens, *args)
    many = torch.zeros(5000, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        pages.fork_requests(w.handle, w.table, w.seq_lens, many, many,
                            torch.zeros(5000, 2, dtype=torch.int32, device=DEV))
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert pages.fork_requests(w.handle, w.table, w.seq_lens, none, none,
                               none.view(0, 2)).numel() == 0


def test_compaction_leaves_no_block_of_a_page_that_it_gave_away():
    """A row may map more pages than its tokens fill. Such a page is free: a moved page may lie in it,
    so the new table does not name it any more. A count that holds the reserved tokens keeps it."""
    w = World([2000, 900, 100], pool=24, rows=5)
    bpp, table = w.bpp, w.table.cpu().numpy()
    spare = [p for p in range(w.pool) if p not in sum(w.owned, [])]
    reserved = [w.owned[0] + spare[:1], w.owned[1], w.owned[2] + spare[1:3]]
    for r, owned in enumerate(reserved):
        w.map(table, r, owned)
    table[4, :bpp] = spare[3] * bpp + np.arange(bpp)  # a row that is not live keeps what it holds
    w.table.copy_(torch.from_numpy(table))
    stripes, want, total = expect_compact(w, range(3))
    for r, owned in enumerate(w.owned):
        want[r, bpp * len(owned) :] = -1
    w_before = [[t.clone() for t in pair] for pair in w.caches]
    tables, live = pages.compact_pages(w.handle, w.table, w.seq_lens, w.counts)
    assert live.item() == total == 6 and np.array_equal(tables.cpu().numpy(), want)
    w.check(stripes)
    for pair, before in zip(w.caches, w_before):
        for t, old in zip(pair, before):
            t.copy_(old)
    # The same with the reserved tokens counted: 2304 (three pages and one more), 1024, 2304.
    w.owned, w.lengths = reserved, [2305, 900, 2304]
    w.seq_lens[:3] = i32(w.lengths)
    free = pages.free_pages(w.handle, w.table, w.seq_lens, w.counts)[0].tolist()
    assert not set(free) & set(sum(reserved, []))
    stripes, want, total = expect_compact(w, range(3))
    tables, live = pages.compact_pages(w.handle, w.table, w.seq_lens, w.counts)
    assert live.item() == total == 9 and np.array_equal(tables.cpu().numpy(), want)
    w.check(stripes)


@pytest.mark.parametrize("length,columns,done", [(2000, 16, 1), (1920, 15, 1), (1921, 15, 0),
                                                 (2304, 18, 1), (100, 1, 1), (129, 1, 0)])
def test_forks_in_a_table_that_ends_inside_a_page(length, columns, done):
    """A table needs a column for every block that holds tokens, not for whole pages."""
    w = World([length, 50], pool=14, rows=4)
    whole = w.table.clone()
    w.table = w.table[:, :columns]
    free = [p for p in range(w.pool) if p not in sum(w.owned, [])]
    stripes, table, seq = w.stripes(), whole.cpu().numpy(), w.seq_lens.cpu().numpy()
    before = table.copy()
    if done:
        expect_fork(w, stripes, table, seq, 0, 3, free[:2])
    assert fork(w, [0], [3], [free[:2]]).tolist() == [done]
    assert np.array_equal(w.table.cpu().numpy(), table[:, :columns])
    assert np.array_equal(w.seq_lens.cpu().numpy(), seq)
    assert np.array_equal(w.table._base.cpu().numpy()[:, columns:], before[:, columns:])
    w.check(stripes)
