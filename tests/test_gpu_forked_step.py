"""Requests forked from one prompt through a decode step, as a server runs them: free pages, the
fork, norms and position rotation of the step's rows, the layer step with the prompt's shared
positions computed once, compaction, and another step. The layer step without the plan of shared
prefixes gives the same rows within rounding and the same cache bytes."""

from types import SimpleNamespace

import pytest
import torch

from oscar_new_amd import kernels, pages
from oscar_new_amd.backend import OscarAttentionImpl
from oscar_new_amd.config import OscarConfig
from oscar_new_amd.layout import CacheLayout
from oscar_new_amd.metadata import OscarMetadataBuilder

pytestmark = pytest.mark.gpu
DEV, HQ, LAYERS, POOL, ROWS = "cuda", 6, 2, 24, 5


class Server:
    def __init__(self, qlen, fused):
        self.gen = torch.Generator(device=DEV).manual_seed(11)
        self.layout = CacheLayout(768, config=OscarConfig(sink_tokens=4, recent_tokens=128))
        shape = (POOL * 6, 128, 1, 256)
        self.caches = [tuple(torch.zeros(shape, dtype=torch.bfloat16, device=DEV) for _ in range(2))
                       for _ in range(LAYERS)]
        self.handle = pages.PageCaches(self.caches, self.layout)
        self.impls = []
        for _ in range(LAYERS):
            impl = OscarAttentionImpl.standalone(HQ, 256, 1 / 16, 1, self.layout.config, fused=fused)
            impl.set_rotations(*(torch.linalg.qr(self.randn(256, 256))[0] for _ in range(2)))
            self.impls.append(impl)
        self.table = torch.full((ROWS, 36), -1, dtype=torch.int32, device=DEV)
        self.seq = torch.zeros(ROWS, dtype=torch.int32, device=DEV)
        self.builder = OscarMetadataBuilder.standalone(self.layout, ROWS, 4096, 36 * 128, DEV)
        angle = torch.arange(4096, device=DEV)[:, None] / 1e4 ** (torch.arange(32, device=DEV) / 32)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], 1)
        self.weights = [1 + 0.1 * self.randn(256) for _ in range(2)]
        self.qlen = qlen

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.gen, device=DEV)

    def step(self, rows, lengths, query, state, shared=None):
        """One step of every layer for the given table rows; their token counts after it."""
        starts = torch.zeros(len(rows) + 1, dtype=torch.int32)
        starts[1:] = torch.tensor(query).cumsum(0)
        n = int(starts[-1])
        positions = torch.cat([torch.arange(t - q, t) for t, q in zip(lengths, query)]).to(DEV)
        table = self.table[rows].contiguous()
        request = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(query)).to(DEV)
        slots = table[request, positions // 128].long() * 128 + positions % 128
        common = SimpleNamespace(
            query_start_loc=starts.to(DEV), query_start_loc_cpu=starts,
            seq_lens=torch.tensor(lengths, dtype=torch.int32, device=DEV),
            seq_lens_cpu=torch.tensor(lengths, dtype=torch.int32), num_reqs=len(rows),
            num_actual_tokens=n, max_query_len=max(query), max_seq_len=max(lengths),
            block_table_tensor=table, slot_mapping=slots, causal=True, attn_state=state)
        meta = self.builder.build(0, common)
        if shared is not None:
            meta.shared = kernels.prepare_shared(
                meta, self.layout, HQ, *(torch.tensor(v, dtype=torch.int32, device=DEV)
                                         for v in shared))
        outs = []
        for impl, cache in zip(self.impls, self.caches):
            q, k = kernels.qk_norm_rope(2 * self.randn(n, HQ, 256).bfloat16(),
                                        self.randn(n, 1, 256).bfloat16(), *self.weights,
                                        self.cos_sin, positions)
            out = torch.empty(n, HQ * 256, dtype=torch.bfloat16, device=DEV)
            impl.forward(None, q, k, self.randn(n, 1, 256).bfloat16(), cache, meta, out)
            outs.append(out)
        self.seq[rows] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        return outs

    def scenario(self, share):
        prompt, i32 = 2000, dict(dtype=torch.int32, device=DEV)
        self.table[0, :18] = torch.arange(60, 78, **i32)
        self.step([0], [prompt], [prompt], "PrefillNoCache")
        counts = torch.tensor([1, 0], **i32)
        free, _ = pages.free_pages(self.handle, self.table, self.seq, counts)
        kids = torch.arange(1, ROWS, **i32)
        done = pages.fork_requests(self.handle, self.table, self.seq, torch.zeros_like(kids), kids,
                                   free[: 2 * (ROWS - 1)].view(-1, 2))
        assert done.tolist() == [1] * (ROWS - 1)
        rows, outs = list(range(ROWS)), []
        for step in range(1, 4):
            lengths = [prompt + step * self.qlen] * ROWS
            outs += self.step(rows, lengths, [self.qlen] * ROWS, "ChunkedPrefill",
                              ([0, ROWS], [prompt]) if share else None)
            if step == 2:
                counts[0] = ROWS
                tables, live = pages.compact_pages(self.handle, self.table, self.seq, counts)
                assert live.item() == 1 + 2 * ROWS  # one shared page, a first and a last one each
                assert int(tables.max()) < 6 * live.item()
                self.table.copy_(tables)
        return outs


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("qlen", [1, 4, 70])
def test_forked_requests_decode_alike_with_and_without_the_plan(qlen, fused):
    with_plan, without = Server(qlen, fused), Server(qlen, fused)
    got, want = with_plan.scenario(True), without.scenario(False)
    for a, b in zip(got, want):
        # Two roundings of bf16 rows on either side (merge and output), and FP8 terms of P.
        assert float((a.float() - b.float()).norm() / b.float().norm()) < 1e-2
    for a, b in zip(with_plan.caches, without.caches):
        assert torch.equal(a[0].view(torch.int16), b[0].view(torch.int16))
        assert torch.equal(a[1].view(torch.int16), b[1].view(torch.int16))


@pytest.mark.parametrize("taken", [True, False])
@pytest.mark.parametrize("qlen", [1, 4, 70])
def test_steps_that_take_the_plan_and_steps_that_leave_it(monkeypatch, qlen, taken):
    calls, run = [], kernels.shared_history
    monkeypatch.setattr("oscar_new_amd.backend.shared_prefix_pays", lambda *args: taken)
    monkeypatch.setattr(kernels, "shared_history", lambda *a, **k: calls.append(1) or run(*a, **k))
    with_plan, without = Server(qlen, True), Server(qlen, True)
    got, want = with_plan.scenario(True), without.scenario(False)
    assert len(calls) == (3 * LAYERS if taken else 0)
    for a, b in zip(got, want):
        if taken:  # bounds as above
            assert float((a.float() - b.float()).norm() / b.float().norm()) < 1e-2
        else:
            assert torch.equal(a, b)
    for a, b in zip(with_plan.caches, without.caches):
        assert torch.equal(a[0].view(torch.int16), b[0].view(torch.int16))
        assert torch.equal(a[1].view(torch.int16), b[1].view(torch.int16))
