"""A NaN in a history stays visible: the merged row and its LSE are NaN, in every merge and in a layer step.
Rows without one keep their bits, and rows of no weight their LSE of -inf."""

import pytest
import torch

from oscar_new_amd import kernels
from tests._int4 import DEV, layout_of, world
from tests.test_gpu_int4 import attend, check
from tests.test_gpu_int4_step import Served

pytestmark = pytest.mark.gpu


def parts(n, hq, splits, seed=3):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rows = torch.randn(n, hq, splits, 256, generator=gen, device=DEV)
    lse = torch.randn(n, hq, splits, generator=gen, device=DEV) * 3
    lse[2] = -float("inf")
    if splits > 1:
        lse[0, :, 1] = -float("inf")
    return rows, lse


@pytest.mark.parametrize("n", [7, 60])
@pytest.mark.parametrize("splits", [1, 2, 16, 17, 40, 130])
@pytest.mark.parametrize("everywhere", [False, True])
def test_split_merge(n, splits, everywhere):
    hq = 6
    rows, lse = parts(n, hq, splits)
    counts = torch.tensor([3, n - 1], dtype=torch.int32, device=DEV)
    want, want_lse = kernels.merge_splits(rows, lse, counts)
    bad = torch.zeros(n, hq, dtype=torch.bool, device=DEV)
    bad[1, 2] = bad[4, 0] = bad[n - 1, 3] = True  # the last token is padding
    at = slice(None) if everywhere else splits - 1
    rows, lse = rows.clone(), lse.clone()
    for t, h in bad.nonzero().tolist():
        rows[t, h, at], lse[t, h, at] = float("nan"), float("nan")
    out, logsum = kernels.merge_splits(rows, lse, counts)
    bad[n - 1] = False
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad)
    assert torch.equal(logsum.isnan(), bad)
    assert torch.equal(out[~bad], want[~bad]) and torch.equal(logsum[~bad], want_lse[~bad])
    assert bool(torch.isneginf(logsum[2]).all()) and bool(torch.isneginf(logsum[n - 1]).all())


@pytest.mark.parametrize("side", [0, 1])
def test_path_merge(side):
    n, hq = 5, 6
    gen = torch.Generator(device=DEV).manual_seed(4)
    a = torch.randn(n, hq, 256, generator=gen, device=DEV).bfloat16()
    b = torch.randn(n, hq, 1, 256, generator=gen, device=DEV)
    la, lb = (torch.randn(n, hq, generator=gen, device=DEV) for _ in range(2))
    la[3] = lb[3] = -float("inf")
    counts = torch.tensor([2, n - 1], dtype=torch.int32, device=DEV)

    def merged():
        out = torch.zeros(n, hq * 256, dtype=torch.bfloat16, device=DEV)
        lse = torch.zeros(n, hq, device=DEV)
        kernels.merge_paths(a, la, b, lb[..., None], counts, out, lse)
        return out.view(n, hq, 256), lse

    want, want_lse = merged()
    bad = torch.zeros(n, hq, dtype=torch.bool, device=DEV)
    bad[1, 2] = bad[2, 5] = True
    (la, lb)[side][bad] = float("nan")
    (a, b[:, :, 0])[side][bad] = float("nan")
    out, lse = merged()
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(lse.isnan(), bad)
    assert torch.equal(out[~bad], want[~bad]) and torch.equal(lse[~bad], want_lse[~bad])
    assert bool(torch.isneginf(lse[3]).all()) and bool(torch.isneginf(lse[4]).all())


@pytest.mark.parametrize("qlens,splits,split_tokens,chunk", [([1, 1, 2], 8, -256, None), ([1, 4, 1], 40, 128, None),
                                                             ([1, 1, 1], 1, 0, None), ([40, 17, 1], 3, 0, True)])
@pytest.mark.parametrize("value", [False, True])
def test_one_nan_record(qlens, splits, split_tokens, chunk, value):
    """The scale of one key (its scores are NaN) or value of the second request's."""
    s = world([900, 3000, 700], qlens, layout_of(2), 6)
    want, want_lse = attend(s, splits, split_tokens, chunk=chunk)
    slot = int(s.meta.block_tables[1, 1500 // 128]) * 128 + 1500 % 128
    side = s.history.view(s.pool, -1)[slot // 768, : 768 * 2 * 272].view(768, 2, 272)[slot % 768, 1, 256:264]
    side.view(torch.float16)[2 * value] = float("nan")
    out, lse = attend(s, splits, split_tokens, chunk=chunk)
    bad = torch.zeros_like(lse, dtype=torch.bool)
    bad[qlens[0] : qlens[0] + qlens[1], 6:] = True  # its rows of the second KV head
    assert torch.equal(out.isnan().all(-1), bad)
    assert torch.equal(out[~bad], want[~bad]) and torch.equal(lse[~bad], want_lse[~bad])
    assert torch.equal(lse.isnan(), bad & (not value))  # weights are whole where a value is not
    assert value is False or torch.equal(lse, want_lse)


@pytest.mark.parametrize("splits,split_tokens", [(8, -256), (40, 128), (1, 0)])
def test_queries_that_are_not_finite(splits, split_tokens):
    """An infinite score makes its wavefront take all of its rows against another reference: the others stay
    within rounding."""
    s = world([700, 3000], [1, 1], layout_of(2), 4)
    query = s.query.clone()
    query[0, 3, 7], query[1, 0, 0], query[1, 5, 9] = float("nan"), float("inf"), float("-inf")
    out, lse = attend(s, splits, split_tokens, query=query)
    bad = torch.zeros(2, 8, dtype=torch.bool, device=DEV)
    bad[0, 3] = bad[1, 0] = bad[1, 5] = True
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(lse.isnan(), bad)
    check(s, (out, lse), but=bad)


@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 1, 4], [40, 1, 2]])
def test_layer_step(counts):
    """With a NaN key in its history a request's outputs and LSEs are NaN, the other requests' are not."""
    w = Served(3, heads=1)
    q, k, v = w.rows(1500)
    w.step([500, 500, 500], q, k, v, initial=True)
    history = w.layout.tensor_views(w.cache)[0]
    slot = int(w.slots(1, torch.tensor([200], device=DEV)))
    at = w.layout.slot_offset(slot)
    history.view(-1)[at + 256 : at + 258] = 255  # the K scale
    n = sum(counts)
    q, k, v = w.rows(n)
    meta = w.meta(counts)
    meta.merged_lse = torch.zeros(n, 6, device=DEV)
    out = torch.zeros(n, 6 * 256, dtype=torch.bfloat16, device=DEV)
    w.impl.forward(None, q.view(n, -1), k.view(n, -1), v.view(n, -1), w.cache, meta, out)
    bad = torch.zeros(n, 6, dtype=torch.bool, device=DEV)
    bad[counts[0] : counts[0] + counts[1]] = True
    assert torch.equal(out.view(n, 6, 256).isnan().all(-1), bad)
    assert torch.equal(meta.merged_lse.isnan(), bad) and bool(meta.merged_lse[~bad].isfinite().all())
