"""Rotation and codes of 4-bit records together, against the rotated rows in 64 bits.

Where a rotated value lies near a border of bf16 either neighbour is a right rounding, since sums of
another order end in another last bit of fp32; a step of bf16 can in turn move a value into the next of
the 16 codes, or its row's clip limit, scale and zero. So every code, scale and zero has a least and a
largest right value, and is held to them here. A sum of 256 exact products in fp32 is off by at most
256 x 2^-24 of the sum of magnitudes, the steps behind it by a few 2^-24 of their results."""

import pytest
import torch

from oscar_new_amd import kernels
from tests._int4 import DEV, layout_of


def rank_of(ratio):
    """The order statistic of the clip limit: the ratio is passed, and multiplied, in fp32."""
    return float(torch.tensor(ratio, dtype=torch.float32) * 255)


def bounds_of(rows, rotation, ratio):
    """Least and largest (codes, scale, zero) of the records of ``rows`` (bf16) times ``rotation``."""
    x, r = rows.double(), rotation.double()
    exact, off = x @ r, 256 * 2.0**-24 * (x.abs() @ r.abs())
    low, high = ((exact + s * off).float().bfloat16().double() for s in (-1, 1))
    # |x| of either end: the order statistics, and what is made of them, grow with every value.
    least = torch.where((low < 0) & (high > 0), 0.0, torch.minimum(low.abs(), high.abs()))
    most = torch.maximum(low.abs(), high.abs())
    rank = rank_of(ratio)
    at, slack = int(rank), 2.0**-20

    def limit(values):
        order = values.sort(-1).values
        a, b = order[..., at : at + 1], order[..., min(at + 1, 255) : min(at + 1, 255) + 1]
        return a + (rank - at) * (b - a)

    clip = limit(least) * (1 - slack), limit(most) * (1 + slack)

    def clipped(values, end):  # the limits' own ends: -limit is least where the limit is largest
        upper, lower = clip[end], -clip[1 - end]
        return torch.minimum(torch.maximum(values, lower), upper)

    ends = clipped(low, 0), clipped(high, 1)
    smallest = [e.amin(-1, keepdim=True) for e in ends]
    largest = [e.amax(-1, keepdim=True) for e in ends]
    zero = [z.float().half().double() for z in smallest]
    spread = [(largest[e] - smallest[1 - e]) / 15 * (1 + (slack if e else -slack)) for e in (0, 1)]
    scale = [s.clamp(min=2.0**-14).float().half().double() for s in spread]
    above = ends[0] - zero[1], ends[1] - zero[0]
    # A quotient is least over the larger scale where it is positive, over the smaller one elsewhere.
    first = torch.minimum(above[0] / scale[0], above[0] / scale[1]) - 1e-5
    last = torch.maximum(above[1] / scale[0], above[1] / scale[1]) + 1e-5
    codes = [torch.floor(y + 0.5).clamp(0, 15) for y in (first, last)]
    return codes, scale, zero


def within(values, ends):
    return bool(((values.double() >= ends[0]) & (values.double() <= ends[1])).all())


def rows_of_any_size(n, heads, gen, device):
    x = torch.randn(n, heads, 256, generator=gen, device=device)
    return (x * (torch.rand(n, 1, 1, generator=gen, device=device) * 3 + 0.2)).bfloat16()


def rotation_of(gen, device):
    return torch.linalg.qr(torch.randn(256, 256, generator=gen, device=device))[0].bfloat16()


@pytest.mark.parametrize("ratio", [0.99, 0.9])
def test_the_bounds(ratio):
    """They hold for a product in fp32, leave hardly a code open, and show a code that is one off."""
    gen = torch.Generator().manual_seed(11)
    rows, r = rows_of_any_size(2000, 1, gen, "cpu"), rotation_of(gen, "cpu")
    codes, scale, zero = bounds_of(rows, r, ratio)
    assert float((codes[0] != codes[1]).double().mean()) < 0.02
    x = (rows.float() @ r.float()).bfloat16().double()
    order = x.abs().sort(-1).values
    rank = rank_of(ratio)
    at = int(rank)
    limit = order[..., at : at + 1] + (rank - at) * (order[..., at + 1 : at + 2] - order[..., at : at + 1])
    x = torch.minimum(torch.maximum(x, -limit), limit)
    z = x.amin(-1, keepdim=True).half().double()
    s = ((x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True)) / 15).half().double()
    got = torch.floor((x - z) / s + 0.5).clamp(0, 15)
    assert within(got, codes) and within(s, scale) and within(z, zero)
    got[77, 0, 5] += 1 if got[77, 0, 5] < 15 else -1
    assert not within(got, codes)


@pytest.mark.gpu
@pytest.mark.parametrize("n,heads", [(5, 1), (150, 2), (1300, 2), (9000, 1)])
@pytest.mark.parametrize("rotary", [0, 64, 96])
def test_records_against_64_bits(n, heads, rotary):
    """Few rows, walking wavefronts (rotary 64) and blocks of 32 rows (96), without norms: rows of any size."""
    gen = torch.Generator(device=DEV).manual_seed(n + rotary)
    key, value = (rows_of_any_size(n, heads, gen, DEV) for _ in range(2))
    query = rows_of_any_size(n, 2 * heads, gen, DEV)
    rk, rv = rotation_of(gen, DEV), rotation_of(gen, DEV)
    turn = {}
    if rotary:
        angle = torch.rand(512, rotary // 2, generator=gen, device=DEV) * 6
        turn = dict(cos_sin=torch.cat([angle.cos(), angle.sin()], 1),
                    positions=torch.randint(512, (n,), generator=gen, device=DEV))
    layout = layout_of(heads, k_clip_ratio=0.99, v_clip_ratio=0.98)
    pages = n // 768 + 1
    history = torch.zeros(pages * layout.stripe_page_bytes, dtype=torch.uint8, device=DEV)
    slots = torch.randperm(pages * 768, generator=gen, device=DEV)[:n]
    counts = torch.tensor([1, n], dtype=torch.int32, device=DEV)
    turned = kernels.rope_append(query, key, value, history, slots, counts, layout, rk.T.contiguous(),
                                 rv.T.contiguous(), **turn)[1]
    view = history.view(pages, -1)[:, : 768 * heads * 272].unflatten(1, (768, heads, 272))
    record = view[slots // 768, slots % 768]
    side = record[..., 256:264].contiguous().view(torch.float16).double()
    back = kernels.read_records(history, slots, layout)
    for i, (rows, r, ratio) in enumerate(((turned, rk, 0.99), (value, rv, 0.98))):
        codes, scale, zero = bounds_of(rows, r, ratio)
        assert float((codes[0] != codes[1]).double().mean()) < 0.02
        packed = record[..., 128 * i : 128 * (i + 1)]
        got = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
        s, z = side[..., 2 * i, None], side[..., 2 * i + 1, None]
        assert within(got, codes) and within(s, scale) and within(z, zero)
        assert torch.equal(back[i], (got.float() * s.float() + z.float()).bfloat16())
