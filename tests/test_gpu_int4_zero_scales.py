"""Attention over 4-bit records whose first chunks were never written (all zeros: no V scale to go by)."""

import pytest
import torch

from tests._int4 import DEV, layout_of, world
from tests.test_gpu_int4 import attend, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qlen", [1, 4, 40])
@pytest.mark.parametrize("scale", [0.05, 3.5, 4.0, 3000.0, 65504.0])
def test_zeros_ahead_of_values(qlen, scale):
    s = world([3000], [qlen], layout_of(1), 6, poison=False)
    lo, hi = s.spans[0]
    view = s.history.view(s.pool, -1)[:, : 768 * 272].view(s.pool, 768, 272)
    page = s.meta.block_tables[0, ::6][:4].long() // 6
    at = torch.arange(4 * 768, device=DEV).view(4, 768)
    record = view[page]
    side = record[..., 256:264].contiguous().view(torch.float16)
    side[..., 2], side[..., 3] = scale, -7.5 * min(scale, 8000.0)
    record[..., 256:264] = side.view(torch.uint8)
    record[at < lo + 400] = 0  # the first chunks of all wavefronts
    view[page] = record
    check(s, attend(s, split_tokens=0, splits=1))
    check(s, attend(s, split_tokens=0, splits=3, chunk=qlen > 16))
    check(s, attend(s) if qlen <= 16 else attend(s, split_tokens=0, splits=2))


@pytest.mark.parametrize("qlen", [1, 40])
def test_zeros_alone(qlen):
    s = world([1500], [qlen], layout_of(1), 6, poison=False)
    s.history.zero_()
    out, lse = attend(s, split_tokens=0, splits=2)
    lo, hi = s.spans[0]
    assert not bool(out.any())
    assert bool((lse.double() - torch.tensor(float(hi - lo), dtype=torch.float64).log()).abs().lt(2.0**-19).all())
