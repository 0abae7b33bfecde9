"""Layer steps of a cache with 4-bit records: prompt, chunk, MTP and decode steps through
``OscarAttentionImpl``, against the single launches (bit for bit) and against attention in 64 bits over
what the cache holds; captured steps; pages of such a cache."""

import math
from types import SimpleNamespace

import pytest
import torch

from oscar_new_amd import kernels, pages
from oscar_new_amd.backend import OscarAttentionImpl
from oscar_new_amd.metadata import OscarMetadataBuilder
from tests._int4 import DEV, layout_of

pytestmark = pytest.mark.gpu
SCALE = 1 / 16


class Served:
    """A layer, its cache and requests of growing lengths in pages of their own."""

    def __init__(self, requests, heads=1, group=6, most=4000, seed=2, bits=4):
        self.gen = torch.Generator(device=DEV).manual_seed(seed)
        self.layout = layout_of(heads, bits=bits, sink_tokens=4, recent_tokens=40, k_clip_ratio=0.99,
                                v_clip_ratio=0.99)
        self.heads, self.group, self.requests = heads, group, requests
        per = -(-most // 768)
        self.pool = requests * per + 3
        order = torch.randperm(self.pool, generator=self.gen, device=DEV)[: requests * per]
        blocks = order.view(requests, per, 1) * 6 + torch.arange(6, device=DEV)
        self.table = blocks.view(requests, per * 6).int().contiguous()
        shape = (self.pool * 6, 128, heads, 256)
        self.cache = tuple(torch.zeros(shape, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        self.lengths = [0] * requests
        self.impl = OscarAttentionImpl.standalone(heads * group, 256, SCALE, heads, cfg=self.layout.config)
        rand = lambda: torch.linalg.qr(torch.randn(256, 256, generator=self.gen, device=DEV))[0]  # noqa: E731
        self.impl.set_rotations(rand().bfloat16(), rand().bfloat16())
        self.builder = OscarMetadataBuilder.standalone(self.layout, requests, requests * 2100, most, DEV)
        self.kept = [[torch.zeros(0, heads, 256, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
                     for _ in range(requests)]

    def slots(self, r, positions):
        return self.table[r, positions // 128].long() * 128 + positions % 128

    def meta(self, counts, initial=False):
        """Metadata of a step with counts[r] new tokens of each request, the lengths after it."""
        starts = torch.zeros(len(counts) + 1, dtype=torch.int32)
        starts[1:] = torch.tensor(counts).cumsum(0)
        seq = torch.tensor([n + c for n, c in zip(self.lengths, counts)], dtype=torch.int32)
        at = [self.slots(r, torch.arange(n, n + c, device=DEV))
              for r, (n, c) in enumerate(zip(self.lengths, counts))]
        common = SimpleNamespace(
            query_start_loc=starts.to(DEV), query_start_loc_cpu=starts, seq_lens=seq.to(DEV),
            seq_lens_cpu=seq, num_reqs=len(counts), num_actual_tokens=int(starts[-1]),
            max_query_len=max(counts), max_seq_len=int(seq.max()), block_table_tensor=self.table,
            causal=True, slot_mapping=torch.cat(at), attn_state="PrefillNoCache" if initial else "X")
        return self.builder.build(0, common)

    def rows(self, n):
        rand = lambda h, s: (s * torch.randn(n, h, 256, generator=self.gen, device=DEV)).bfloat16()  # noqa: E731
        return rand(self.heads * self.group, 2), rand(self.heads, 1), rand(self.heads, 1)

    def step(self, counts, q, k, v, initial=False):
        meta = self.meta(counts, initial)
        out = torch.full((q.shape[0], q.shape[1] * 256), 7.0, dtype=torch.bfloat16, device=DEV)
        n = q.shape[0]
        self.impl.forward(None, q.view(n, -1), k.view(n, -1), v.view(n, -1), self.cache, meta, out)
        at = 0
        for r, c in enumerate(counts):
            for i, x in enumerate((k, v)):
                self.kept[r][i] = torch.cat([self.kept[r][i], x[at : at + c]])
            at += c
            self.lengths[r] += c
        return out, meta


def exact_step(w, counts, q, q_rot):
    """float64 outputs over the records' values in the history and the bf16 rows elsewhere, and each
    row's largest value magnitude."""
    cfg, outs, tops, t0 = w.layout.config, [], [], 0
    history = w.layout.tensor_views(w.cache)[0]
    rv = w.impl.rv.double()
    for r, c in enumerate(counts):
        length = w.lengths[r]
        prefix = length - c
        lo = min(cfg.sink_tokens, prefix)
        hi = max(lo, prefix - cfg.recent_tokens)
        key, value = (t.double() for t in w.kept[r])
        hk, hv = (t.double() for t in kernels.read_records(
            history, w.slots(r, torch.arange(lo, hi, device=DEV)), w.layout))
        near = torch.cat([torch.arange(lo, device=DEV), torch.arange(hi, length, device=DEV)])
        for t in range(c):
            seen = near[near <= prefix + t]
            for h in range(q.shape[1]):
                g = h // w.group
                score = torch.cat([hk[:, g] @ q_rot[t0 + t, h].double(),
                                   key[seen, g] @ q[t0 + t, h].double()]) * SCALE
                p = score.softmax(0)
                vals = torch.cat([hv[:, g] @ rv.T, value[seen, g]])
                outs.append(p @ vals)
                tops.append((p @ vals.abs()).amax() + vals.norm(dim=1).amax() / 16)
        t0 += c
    return torch.stack(outs).view(q.shape), torch.stack(tops).view(*q.shape[:2], 1)


def check(w, counts, out, q):
    """Roundings on the way: the records' values to bf16 (the oracle's reading), P of either branch, the
    merged history row, its rotation back and the output, each 2^-8 of the weighed values, and scores of
    rounded values: below 2^-5 of the row's weighed magnitude in all."""
    picked = [sum(counts[:r]) + t for r, c in enumerate(counts) for t in range(c)]
    assert len(picked) == q.shape[0]
    want, top = exact_step(w, counts, q, kernels.rotate(q, w.impl.rk))
    err = (out.view(q.shape).double() - want).abs()
    assert bool((err <= 2.0**-5 * top).all()), float((err / top).max())


def single_launches(w, counts, q, k, v, meta):
    """The step as single launches, on copies of the caches."""
    cache = tuple(t.clone() for t in w.cache)
    history, window = w.layout.tensor_views(cache)
    impl, lay = w.impl, w.layout
    kernels.rope_append(None, k, v, history, meta.slot_mapping, meta.counts, lay, impl.rk_t, impl.rv_t)
    splits, tokens = impl.partition_for(meta, q.shape[0])
    hp, hl = kernels.attention_partials(kernels.rotate(q, impl.rk), k, v, history, window, meta, lay, SCALE,
                                        splits, raw=False, split_tokens=tokens)
    merged, lse = kernels.merge_splits(hp, hl, meta.counts)
    rp, rl = kernels.attention_partials(q, k, v, history, window, meta, lay, SCALE, 1, raw=True)
    out = torch.empty(q.shape[0], q.shape[1] * 256, dtype=torch.bfloat16, device=DEV)
    kernels.merge_paths(kernels.rotate(merged, impl.rv.T), lse, rp, rl, meta.counts, out)
    kernels.store_windows(k, v, window, meta, lay)
    return out, cache


@pytest.mark.parametrize("heads,group", [(1, 6), (2, 4)])
def test_a_conversation(heads, group):
    w = Served(3, heads, group)
    counts = [300, 45, 900]
    q, k, v = w.rows(sum(counts))
    w.step(counts, q, k, v, initial=True)
    for counts in ([1, 1, 1], [4, 4, 4], [2, 1, 4], [70, 30, 1], [1, 200, 3], [1, 1, 1]):
        q, k, v = w.rows(sum(counts))
        meta = w.meta(counts)
        want, cache = single_launches(w, counts, q, k, v, meta)
        out, _ = w.step(counts, q, k, v)
        assert torch.equal(out, want)
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(cache, w.cache))
        check(w, counts, out, q)


def test_appended_rows_then_the_rest():
    """rope_append (norms, several position axes) and forward_appended: the layer step on turned rows."""
    a, b = Served(2, seed=9), Served(2, seed=9)
    gen = torch.Generator(device=DEV).manual_seed(1)
    cs = torch.randn(5000, 64, generator=gen, device=DEV)
    axes = kernels.rope_axes([8, 12, 12], device=DEV)
    weight = torch.rand(256, generator=gen, device=DEV) + 0.5
    for counts, initial in (([120, 500], True), ([1, 1], False), ([4, 3], False), ([90, 1], False)):
        n = sum(counts)
        q, k, v = a.rows(n)
        b.rows(n)
        pos = torch.randint(5000, (3, n), generator=gen, device=DEV)
        meta = b.meta(counts, initial)
        b.impl._bind_cache(b.cache, b.layout)
        rows = kernels.rope_append(q, k, v, b.impl.history, meta.slot_mapping, meta.counts, b.layout,
                                   b.impl.rk_t, b.impl.rv_t, cos_sin=cs, positions=pos, axes=axes,
                                   q_weight=weight, k_weight=weight, rotate_query=not initial)
        out = torch.empty(n, 6 * 256, dtype=torch.bfloat16, device=DEV)
        b.impl.forward_appended(rows[0], rows[1], v, rows[2], b.cache, meta, out)
        b.lengths = [x + c for x, c in zip(b.lengths, counts)]
        q, k = kernels.qk_norm_rope(q, k, weight, weight, cs, pos, axes=axes)
        want, _ = a.step(counts, q, k, v, initial)
        assert torch.equal(out, want)
        assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(a.cache, b.cache))


def test_a_captured_step():
    w = Served(3)
    counts = [300, 45, 900]
    w.step(counts, *w.rows(sum(counts)), initial=True)
    q, k, v = w.rows(3)
    out = torch.empty(3, 6 * 256, dtype=torch.bfloat16, device=DEV)

    def run(meta):
        w.impl.forward(None, q.view(3, -1), k.view(3, -1), v.view(3, -1), w.cache, meta, out)

    meta = w.meta([1, 1, 1])
    before = tuple(t.clone() for t in w.cache)
    run(meta)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(meta)
    for t, b in zip(w.cache, before):
        t.copy_(b)
    for _ in range(5):
        for x, fresh in zip((q, k, v), w.rows(3)):
            x.copy_(fresh)
        meta = w.meta([1, 1, 1])
        want, cache = single_launches(w, [1, 1, 1], q, k, v, meta)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(cache, w.cache))
        w.lengths = [n + 1 for n in w.lengths]


def test_layer_and_cache_must_agree():
    w = Served(1)
    other = Served(1, bits=2)
    q, k, v = w.rows(2)
    out = torch.empty(2, 6 * 256, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="records"):
        w.impl.forward(None, q, k, v, other.cache, other.meta([2], True), out)
    meta = w.meta([2])
    with pytest.raises(ValueError, match="R_k"):
        w.impl.forward_appended(q, k, v, None, w.cache, meta, out)
    with pytest.raises(ValueError, match="same tokens"):
        w.impl.forward_appended(q, k[:1], v, q, w.cache, meta, out)
    starts = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="layout"):
        kernels.prepare_shared(meta, w.layout, 6, starts, starts[1:])


def test_forked_and_moved_pages():
    """A fork's records and a compacted cache's are those of the parent: 4-bit records whole."""
    w = Served(2, heads=2, group=4, most=3000)
    counts = [2000, 100]
    w.step(counts, *w.rows(sum(counts)), initial=True)
    caches = pages.PageCaches([w.cache], w.layout)
    table = torch.full((3, w.table.shape[1]), -1, dtype=torch.int32, device=DEV)
    table[:2] = w.table
    seq = torch.tensor(w.lengths + [0], dtype=torch.int32, device=DEV)
    live = torch.tensor([2, 2], dtype=torch.int32, device=DEV)
    free, _ = pages.free_pages(caches, table, seq, live)
    i32 = dict(dtype=torch.int32, device=DEV)
    done = pages.fork_requests(caches, table, seq, torch.tensor([0], **i32), torch.tensor([2], **i32),
                               free[:2].view(1, 2))
    assert done.tolist() == [1] and seq.tolist() == [2000, 100, 2000]
    history = w.layout.tensor_views(w.cache)[0]
    at = torch.arange(2000, device=DEV)

    def values(t, r):
        return kernels.read_records(history, t[r, at // 128].long() * 128 + at % 128, w.layout)

    want = values(table, 0)
    assert bool(want[0].any()) and not bool(want[0].isnan().any())
    assert all(torch.equal(x, y) for x, y in zip(values(table, 2), want))
    live[:] = 3
    moved, count = pages.compact_pages(caches, table, seq, live)
    assert int(moved.max()) // 6 < int(count) and not torch.equal(moved, table)
    for r in (0, 2):
        assert all(torch.equal(x, y) for x, y in zip(values(moved, r), want))
