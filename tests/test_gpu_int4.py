"""``kernels.attention_partials`` over 4-bit records against attention in 64 bits (tests/_int4.py)."""

import pytest
import torch

from oscar_new_amd import kernels
from tests._int4 import DEV, exact, layout_of, world

pytestmark = pytest.mark.gpu
SCALE = 1 / 16


def attend(s, splits=8, split_tokens=-256, query=None, merged=True, chunk=None):
    query = s.query if query is None else query
    got = kernels.attention_partials(query, None, None, s.history, None, s.meta, s.layout, SCALE, splits,
                                     raw=False, split_tokens=split_tokens, chunk=chunk)
    return kernels.merge_splits(*got, s.meta.counts) if merged else got


def check(s, got, query=None, but=None):
    query = s.query if query is None else query
    out, lse = got
    n = sum(s.qlens)
    want, want_lse, slack, lse_slack = exact(s, query[:n], SCALE)
    if but is not None:  # rows that are not compared
        out, lse, want = out[~but][:, None], lse[~but][:, None], want[~but][:, None]
        want_lse, slack, lse_slack = (t[~but][:, None] for t in (want_lse, slack, lse_slack))
        n = out.shape[0]
    empty = want_lse == float("-inf")
    assert bool((out[:n].double() - want).abs().le(slack + 2.0**-8 * (want.abs() + slack)).all())
    assert bool((lse[:n][empty] == float("-inf")).all())
    assert bool((lse[:n].double() - want_lse)[~empty].abs().le(lse_slack[~empty]).all())


SHAPES = [
    ([1], [1]), ([2], [2]), ([36], [1]), ([37], [1]), ([38], [1]), ([69], [1]), ([133, 36, 300], [1, 1, 1]),
    ([1000], [4]), ([5000, 1, 37, 769], [1, 1, 1, 2]), ([900, 333, 64, 2049], [3, 4, 1, 2]),
    ([1500, 700], [7, 1]), ([1200], [33]),
]


@pytest.mark.parametrize("lengths,qlens", SHAPES)
@pytest.mark.parametrize("heads,group", [(1, 6), (2, 5), (4, 1), (1, 8), (3, 4)])
def test_lengths_and_heads(lengths, qlens, heads, group):
    s = world(lengths, qlens, layout_of(heads), group, seed=len(lengths) + heads)
    check(s, attend(s))


@pytest.mark.parametrize("splits,split_tokens", [(1, 0), (5, 0), (16, 0), (7, 256), (3, 64), (40, 128),
                                                 (64, -256), (2, -256), (8, -3), (16, -1000)])
@pytest.mark.parametrize("qlens", [[1, 1, 1], [4, 2, 4]])
def test_split_rules(splits, split_tokens, qlens):
    s = world([3000, 70, 1201], qlens, layout_of(2), 6, seed=splits)
    check(s, attend(s, splits, split_tokens))


@pytest.mark.parametrize("lengths,qlens", [([1], [1]), ([300], [300]), ([2000, 5, 40, 999], [31, 1, 2, 400]),
                                           ([700], [17]), ([900, 900], [64, 65]), ([129], [128])])
@pytest.mark.parametrize("heads,group", [(1, 6), (2, 5), (1, 1), (2, 8), (1, 32)])
@pytest.mark.parametrize("splits", [1, 3, 16])
def test_row_tiles(lengths, qlens, heads, group, splits):
    s = world(lengths, qlens, layout_of(heads, queries_per_tile=1 if group > 8 else 4), group,
              seed=splits, extra_rows=3)
    check(s, attend(s, splits, 0, chunk=True))
    s.meta.max_num_reqs = 700  # an engine's capacity: more tiles than there are
    assert all(torch.equal(a[: sum(qlens)], b[: sum(qlens)]) for a, b in zip(
        attend(s, splits, 0, chunk=True), attend(s, splits, 0, chunk=True)))
    check(s, attend(s, splits, 0, chunk=True))


def test_row_tiles_of_many_requests():
    lengths = [1 + (i * 97) % 700 for i in range(300)]
    qlens = [1 + (i * 31) % min(n, 40) for i, n in enumerate(lengths)]
    s = world(lengths, qlens, layout_of(1), 6)
    check(s, attend(s, 2, 0, chunk=True))


@pytest.mark.parametrize("page,block", [(384, 128), (1536, 128), (768, 64), (768, 32), (96, 32)])
def test_pages_and_blocks(page, block):
    s = world([1000, 97, 333], [1, 2, 1], layout_of(2, page, block, recent_tokens=17), 4)
    check(s, attend(s))


@pytest.mark.parametrize("group,qlen", [(16, 1), (32, 1), (16, 2), (17, 1), (10, 3)])
def test_many_heads(group, qlen):
    s = world([700, 40], [qlen, qlen], layout_of(1), group)
    check(s, attend(s))


def test_a_long_request():
    s = world([131072, 20], [1, 1], layout_of(1), 6)
    check(s, attend(s, 128))
    check(s, attend(s, 1, 0))  # one split: more kernel blocks than its table in LDS holds
    s = world([131072], [40], layout_of(1), 6)
    check(s, attend(s, 1, 0))


def test_unmapped_blocks_are_masked():
    s = world([2000, 900], [1, 4], layout_of(2), 6)
    s.meta.block_tables[0, 3:5] = -1
    s.meta.block_tables[1] = -1
    check(s, attend(s))
    s.meta.block_tables[0, 7] = 1 << 30  # outside the buffer: masked too
    got = attend(s)
    s.meta.block_tables[0, 7] = -1
    assert all(torch.equal(a, b) for a, b in zip(got, attend(s)))


def test_rows_past_the_live_tokens_stay_as_they_are():
    s = world([2000, 300], [1, 2], layout_of(1), 6, extra_rows=5)
    n, hq, splits = s.query.shape[0], s.hq, 8
    partials, lse = attend(s, splits, merged=False)
    out, out_lse = kernels.merge_splits(partials, lse, s.meta.counts)
    check(s, (out, out_lse))
    assert not bool(out[3:].any()) and bool((out_lse[3:] == float("-inf")).all())
    s.meta.counts[1] = 0
    s.meta.counts[0] = 0
    s.meta.task_count.zero_()
    out, out_lse = attend(s, splits)
    assert out.shape == (n, hq, 256) and not bool(out.any())


def test_strided_queries_and_infinite_ones():
    s = world([700, 800], [1, 1], layout_of(2), 4)
    packed = torch.zeros(2, 8, 520, dtype=torch.bfloat16, device=DEV)
    packed[..., 8:264] = s.query
    check(s, attend(s, query=packed[..., 8:264]))
    odd = torch.zeros(2, 8, 259, dtype=torch.bfloat16, device=DEV)
    odd[..., 1:257] = s.query
    check(s, attend(s, query=odd[..., 1:257]))
    query = s.query.clone()
    query[0, 3, 7], query[1, 0, 0], query[1, 5, 9] = float("nan"), float("inf"), float("-inf")
    out, lse = attend(s, query=query)
    bad = torch.zeros(2, 8, dtype=torch.bool, device=DEV)
    bad[0, 3] = bad[1, 0] = bad[1, 5] = True
    assert bool(out[bad].isnan().all())
    check(s, (out, lse), but=bad)
    # Of every split that is used (merge_splits takes a NaN LSE for an unused one).
    whole = attend(s, 1, 0, query=query, merged=False)
    assert bool(whole[0][bad].isnan().all()) and bool(whole[1][bad].isnan().all())


def test_small_values_beside_large_ones():
    s = world([900], [1], layout_of(1), 6)
    s.query[:, :, 17] *= 2.0**7
    s.query[:, :, 100:] *= 2.0**-9
    check(s, attend(s))


def test_scales_of_any_size():
    """Scales and zeros over fp16's range: no product leaves fp32's or loses its bits."""
    s = world([900], [1], layout_of(1), 6)
    view = s.history.view(s.pool, -1)[:, : 768 * 272].view(s.pool, 768, 272)
    side = view[..., 256:264].contiguous().view(torch.float16)
    at = torch.arange(768, device=DEV)
    side[..., 2] = torch.where(at % 2 == 0, 3000.0, 2.0**-14).half()  # V scales
    side[..., 3] = torch.where(at % 3 == 0, -6e4, 2e-5).half()
    view[..., 256:264] = side.view(torch.uint8)
    check(s, attend(s))


@pytest.mark.parametrize("qlen", [1, 4, 40])
def test_scores_and_scales_that_grow(qlen):
    """Weights are taken against a wavefront's first chunk: later ones far above it, far below it, and V
    scales that grow a thousandfold keep every row's accuracy."""
    for case in range(4):
        s = world([9000], [qlen], layout_of(1), 6, seed=case, poison=False)
        view = s.history.view(s.pool, -1)[:, : 768 * 272].view(s.pool, 768, 272)
        side = view[..., 256:264].contiguous().view(torch.float16)
        page = s.meta.block_tables[0, ::6][:12].long() // 6
        at = torch.arange(12 * 768, device=DEV).view(12, 768)
        if case == 0:  # a wavefront's first chunk tops the rest by 12 log2 units and more
            big = at < 260
            side[page, :, 0] = torch.where(big, 0.2, 0.002).half()
            side[page, :, 1] = 0.0
        elif case == 1:  # and lies below it, step by step
            side[page, :, 0] = (0.001 * 1.002 ** (at / 4).float()).half()
            side[page, :, 1] = 0.0
        elif case == 2:  # V scales
            side[page, :, 2] = (0.001 * 1.0008 ** at.float()).half()
            side[page, :, 3] = (-0.0075 * 1.0008 ** at.float()).half()
        else:  # the last position alone counts
            side[page, :, 0] = torch.where(at == 8950, 30.0, 0.01).half()
        view[..., 256:264] = side.view(torch.uint8)
        check(s, attend(s, split_tokens=0, splits=1))
        check(s, attend(s, split_tokens=0, splits=3, chunk=qlen > 16))


@pytest.mark.parametrize("qlen", [1, 4, 40])
def test_first_chunks_of_no_weight(qlen):
    """Positions of score -inf (keys of -inf, queries above zero) count nothing, a wavefront's first chunks
    among them, whose largest score is no reference then."""
    s = world([2000], [qlen], layout_of(1), 6, poison=False)
    s.query = s.query.abs() + 0.01
    lo, hi = s.spans[0]
    view = s.history.view(s.pool, -1)[:, : 768 * 272].view(s.pool, 768, 272)
    side = view[..., 256:264].contiguous().view(torch.float16)
    page = s.meta.block_tables[0, ::6][:3].long() // 6
    at = torch.arange(3 * 768, device=DEV).view(3, 768)
    side[page, :, 1] = torch.where(at < lo + 1000, -torch.inf, side[page, :, 1].float()).half()
    view[..., 256:264] = side.view(torch.uint8)
    got = [attend(s), attend(s, split_tokens=0, splits=1), attend(s, split_tokens=0, splits=3, chunk=qlen > 16)]
    s.spans = [(lo + 1000, hi)]
    for g in got:
        check(s, g)


def test_records_beyond_4_gb():
    layout = layout_of(2)
    s = world([3000, 800], [1, 1], layout, 6, extra_pages=5600, high=True, poison=False)
    assert s.history.numel() > 1 << 32 and int(s.meta.block_tables.max()) // 6 * 786432 > 1 << 32
    check(s, attend(s))


def test_a_captured_step_replays_with_new_lengths():
    s = world([3000, 900, 64], [1, 1, 1], layout_of(1), 6, poison=False)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    attend(s)
    with torch.cuda.graph(graph, stream=stream):
        got = attend(s)
    for lengths in ([3000, 900, 64], [37, 900, 1], [2999, 33, 64], [3000, 900, 64]):
        s.meta.seq_lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        s.lengths = lengths
        s.spans = [(min(4, n - 1), max(min(4, n - 1), n - 33)) for n in lengths]
        graph.replay()
        torch.cuda.synchronize()
        eager = attend(s)
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        check(s, got)


def test_two_streams_at_once():
    a = world([5000, 70], [1, 1], layout_of(1), 6, seed=3)
    b = world([4000, 900], [4, 2], layout_of(1), 6, seed=4)
    want = attend(a), attend(b)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(attend(s))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, y) for one in got[i] for x, y in zip(one, want[i]))
