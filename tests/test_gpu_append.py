"""``kernels.rope_append``, ``read_records`` and the position axes of ``qk_norm_rope`` against the formulas
in 64 bits and against the single launches whose bits they keep.

Error bound of a turned row's element, from the arithmetic: one rounding to bf16 (2^-8 relative to the
value) after fp32 steps, which add at most 2^-18 of the row's largest normalized value (the sum of 256
squares, the root, two products, and the turn's two products and addition). Without norms the turn alone.
A record's codes, scale and zero follow from the rotated bf16 row in fp32, so they are compared bit for
bit with the same steps in torch."""

import pytest
import torch

from oscar_new_amd import kernels
from tests._int4 import DEV, SLOT, layout_of

pytestmark = pytest.mark.gpu


def make(n, hq, hk, rotary, axes=1, cycle=False, positions=977, table=torch.float32,
         weight=torch.float32, seed=3):
    gen = torch.Generator(device=DEV).manual_seed(seed + n + rotary + axes)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    packed = (rand(n, (2 * hq + 2 * hk) * 256) * (rand(n, 1).abs() + 0.1)).bfloat16()
    query = packed[:, : 2 * hq * 256].view(n, hq, 512)[..., :256]
    key = packed[:, 2 * hq * 256 : (2 * hq + hk) * 256].view(n, hk, 256)
    value = packed[:, (2 * hq + hk) * 256 :].view(n, hk, 256)
    angle = rand(positions, rotary // 2) * 3
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).to(table)
    pos = torch.randint(positions, (axes, n), generator=gen, device=DEV)
    pos[:, 0], pos[-1, -1] = 0, positions - 1
    order = torch.randint(axes, (rotary // 2,), generator=gen, device=DEV, dtype=torch.int32)
    weights = [(rand(256) * 0.4 + 1).to(weight) for _ in range(2)]
    rk, rv = (torch.linalg.qr(rand(256, 256))[0].bfloat16() for _ in range(2))
    return query, key, value, weights, cos_sin, pos, order, rk.T.contiguous(), rv.T.contiguous()


def formula(x, weight, cos_sin, pos, order, eps, unit_offset, interleaved):
    """float64 rows, and each row's largest magnitude ahead of the turn."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
        y = y * (weight.double() + (1.0 if unit_offset else 0.0))
    largest = y.abs().amax(-1, keepdim=True)
    half = cos_sin.shape[1] // 2
    at = pos[order.long()].T if order is not None else pos.view(-1, 1).expand(-1, half)
    pair = torch.arange(half, device=DEV)
    cos, sin = cos_sin.double()[at, pair][:, None], cos_sin.double()[at, pair + half][:, None]
    out = y.clone()
    if interleaved:
        a, b = y[..., 0 : 2 * half : 2], y[..., 1 : 2 * half : 2]
        out[..., 0 : 2 * half : 2], out[..., 1 : 2 * half : 2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = y[..., :half], y[..., half : 2 * half]
        out[..., :half], out[..., half : 2 * half] = a * cos - b * sin, b * cos + a * sin
    return out, largest


def check(got, *args):
    want, largest = formula(*args)
    assert got.is_contiguous() and got.dtype == torch.bfloat16
    assert bool(((got.double() - want).abs() <= want.abs() * 2.0**-8 + largest * 2.0**-18).all())


def codes_of(x, cfg, ratio, factor):
    """4-bit codes [.., 256] and the fp16 scale and zero of bf16 rows, in the kernel's fp32 steps."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)

    def quantize(limit):
        c = x if limit is None else torch.minimum(torch.maximum(x, -limit), limit)
        low, high = c.amin(-1, keepdim=True), c.amax(-1, keepdim=True)
        # By a tensor: torch multiplies by a scalar's reciprocal, which misses the ties of fp16, as
        # 6.0443115234375 / 15 = 1650.5 x 2^-12.
        scale = ((high - low) / torch.full_like(high, 15)).clamp(min=2.0**-14).half()
        zero = low.half()
        codes = ((c - zero.float()) / scale.float() + 0.5).trunc().clamp(0, 15)
        return codes, scale, zero

    if cfg.clip_mode == "factor":
        return quantize(top * torch.tensor(factor, dtype=torch.float32, device=DEV))
    if cfg.clip_mode == "percentile":
        if ratio == 0:
            return quantize(None)
        order = x.abs().sort(-1).values
        rank = torch.tensor(ratio, dtype=torch.float32) * 255
        low = int(rank.floor())
        a, b = order[..., low : low + 1], order[..., int(rank.ceil()) : int(rank.ceil()) + 1]
        return quantize(torch.addcmul(a.double(), (rank - low).double().to(DEV), (b - a).double()).float())
    raise AssertionError(cfg.clip_mode)


def record_parts(history, layout, slots):
    page, heads = layout.physical_block_tokens, layout.kv_heads
    view = history.view(-1, layout.stripe_page_bytes)[:, : page * heads * SLOT]
    rec = view.unflatten(1, (page, heads, SLOT))[slots // page, slots % page]
    side = rec[..., 256:264].contiguous().view(torch.float16)
    parts = []
    for i in (0, 1):
        packed = rec[..., 128 * i : 128 * (i + 1)]
        codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
        parts.append((codes, side[..., 2 * i], side[..., 2 * i + 1]))
    return parts, rec


def cache(n, layout, pages, seed=5):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    history = torch.full((pages * layout.stripe_page_bytes,), 171, dtype=torch.uint8, device=DEV)
    slots = torch.randperm(pages * layout.physical_block_tokens, generator=gen, device=DEV)[:n]
    return history, slots


def append(m, layout, history, slots, counts, norm=True, axes=True, **over):
    query, key, value, weights, cos_sin, pos, order, rk_t, rv_t = m
    w = weights if norm else (None, None)
    args = dict(cos_sin=cos_sin, positions=pos if axes else pos[0], axes=order if axes else None,
                q_weight=w[0], k_weight=w[1], eps=1e-5)
    args.update(over)
    return kernels.rope_append(query, key, value, history, slots, counts, layout, rk_t, rv_t, **args)


def counts_of(live):
    return torch.tensor([1, live], dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("n,hq,hk", [(1, 6, 1), (2, 1, 1), (17, 5, 2), (33, 16, 4), (700, 6, 1),
                                     (1031, 12, 2), (5, 40, 8)])
@pytest.mark.parametrize("rotary,interleaved", [(64, False), (96, False), (256, False), (64, True),
                                                (256, True), (20, False), (6, True), (2, False)])
def test_rows_of_several_axes(n, hq, hk, rotary, interleaved):
    for axes, table, weight, unit in ((3, torch.float32, torch.float32, False),
                                      (2, torch.bfloat16, torch.bfloat16, True),
                                      (4, torch.float32, torch.bfloat16, True)):
        q, k, _, w, cs, pos, order, rk_t, _ = make(n, hq, hk, rotary, axes, table=table, weight=weight)
        args = dict(eps=1e-5, unit_offset=unit, interleaved=interleaved, axes=order)
        got = kernels.qk_norm_rope(q, k, *w, cs, pos, **args)
        for x, y, weight_ in ((got[0], q, w[0]), (got[1], k, w[1])):
            check(x, y, weight_, cs, pos, order, 1e-5, unit, interleaved)
        turned = kernels.qk_norm_rope(q, k, *w, cs, pos, rk_t=rk_t, **args)
        assert torch.equal(turned[0], got[0]) and torch.equal(turned[1], got[1])
        assert torch.equal(turned[2], kernels.rotate(got[0], rk_t.T))


@pytest.mark.parametrize("rotary,interleaved", [(64, False), (128, False), (128, True), (32, False)])
@pytest.mark.parametrize("sections", [(16, 24, 24), (5, 6, 5), (7, 1, 8)])
@pytest.mark.parametrize("cycle", [False, True])
def test_sections(rotary, interleaved, sections, cycle):
    """Axes in sections (whole lanes of one axis, or borders inside them) and in turns, many rows."""
    total = sum(sections)
    counts = [c * (rotary // 2) // total for c in sections]
    counts[0] += rotary // 2 - sum(counts)
    if cycle and 3 * max(counts[1:]) > rotary // 2:  # more than their turns
        counts = [rotary // 2 - 2 * (rotary // 6)] + [rotary // 6] * 2
    for table in (torch.float32, torch.bfloat16):
        q, k, _, w, cs, pos, _, rk_t, _ = make(900, 5, 2, rotary, 3, table=table)
        order = kernels.rope_axes(counts, cycle, DEV)
        args = dict(eps=1e-5, interleaved=interleaved, axes=order)
        got = kernels.qk_norm_rope(q, k, *w, cs, pos, **args)
        for x, y, weight in ((got[0], q, w[0]), (got[1], k, w[1])):
            check(x, y, weight, cs, pos, order, 1e-5, False, interleaved)
        turned = kernels.qk_norm_rope(q, k, *w, cs, pos, rk_t=rk_t, **args)
        assert torch.equal(turned[0], got[0]) and torch.equal(turned[1], got[1])
        assert torch.equal(turned[2], kernels.rotate(got[0], rk_t.T))


@pytest.mark.parametrize("rotary,interleaved", [(64, False), (256, True), (20, False), (6, True), (0, False)])
@pytest.mark.parametrize("rotate", [False, True])
def test_one_axis_has_the_bits_of_the_plain_call(rotary, interleaved, rotate):
    q, k, _, w, cs, pos, _, rk_t, _ = make(317, 6, 2, rotary)
    args = dict(eps=1e-6, interleaved=interleaved, rk_t=rk_t if rotate else None, counts=counts_of(300))
    plain = kernels.qk_norm_rope(q, k, *w, cs, pos[0], **args)
    zero = torch.zeros(rotary // 2, dtype=torch.int32, device=DEV)
    assert all(torch.equal(a, b) for a, b in zip(
        kernels.qk_norm_rope(q, k, *w, cs, pos, axes=zero, **args), plain))
    same = pos.expand(3, -1)
    third = torch.arange(rotary // 2, device=DEV, dtype=torch.int32) % 3
    assert all(torch.equal(a, b) for a, b in zip(
        kernels.qk_norm_rope(q, k, *w, cs, same, axes=third, **args), plain))


def test_positions_and_axes_outside():
    q, k, _, w, cs, pos, order, rk_t, _ = make(40, 4, 2, 64, 3)
    pos[1, 5], pos[2, 6], pos[0, 7], pos[:, 30:] = -1, cs.shape[0], 1 << 40, 1 << 50
    got = kernels.qk_norm_rope(q, k, *w, cs, pos, axes=order, counts=counts_of(30), rk_t=rk_t)
    good = [t for t in range(30) if t not in (5, 6, 7)]
    for x in got:
        assert bool(x[[5, 6, 7]].isnan().all()) and not bool(x[30:].any())
        assert bool(x[good].isfinite().all())
    order = order.clone()
    order[3], order[9] = 3, -1  # pairs (3, 35) and (9, 41) belong to no axis
    wrong = kernels.qk_norm_rope(q, k, *w, cs, pos, axes=order, counts=counts_of(30), rk_t=rk_t)[:2]
    again = kernels.qk_norm_rope(q, k, *w, cs, pos, axes=order, counts=counts_of(30))
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(wrong, again))
    alone = kernels.qk_norm_rope(q, k, *w, cs, pos[:1], axes=order, counts=counts_of(30))
    assert bool(alone[0][good][..., [3, 35, 9, 41]].isnan().all())
    dims = torch.zeros(256, dtype=torch.bool, device=DEV)
    dims[[3, 35, 9, 41]] = True
    for x, y in zip(wrong, got):
        assert bool(x[good][..., dims].isnan().all())
        assert torch.equal(x[good][..., ~dims], y[good][..., ~dims])


@pytest.mark.parametrize("n,live,hq,hk", [(1, 1, 6, 1), (33, 30, 6, 1), (300, 300, 5, 2), (1500, 1400, 8, 2),
                                          (5, 0, 4, 4)])
@pytest.mark.parametrize("norm,rotary,interleaved", [(True, 64, False), (False, 64, True), (True, 0, False),
                                                     (False, 20, False)])
@pytest.mark.parametrize("bits", [2, 4])
def test_rows_and_records(n, live, hq, hk, norm, rotary, interleaved, bits):
    m = make(n, hq, hk, rotary, 3)
    q, k, v, w, cs, pos, order, rk_t, rv_t = m
    layout = layout_of(hk, bits=bits, k_clip_ratio=0.96, v_clip_ratio=0.99)
    history, slots = cache(n, layout, n // 768 + 2)
    slots[live // 2 : live // 2 + 1] = -1  # a token that is not kept
    before = history.clone()
    got = append(m, layout, history, slots, counts_of(live), norm=norm, interleaved=interleaved)
    for x, y, weight in ((got[0], q, w[0]), (got[1], k, w[1])):
        check(x[:live], y[:live], weight if norm else None, cs, pos[:, :live], order, 1e-5, False,
              interleaved)
        assert not bool(x[live:].any())
    assert torch.equal(got[2], kernels.rotate(got[0], rk_t.T))
    rotated = kernels.rotate(got[1], rk_t.T), kernels.rotate(v, rv_t.T)
    if bits == 2:
        want = before.clone()
        kernels.store_int2(*rotated, want, slots, counts_of(live), layout)
        assert torch.equal(history, want)
        return
    kept = torch.arange(live, device=DEV)[slots[:live] >= 0]
    parts, rec = record_parts(history, layout, slots[kept])
    for (codes, scale, zero), x, ratio in zip(parts, rotated, (0.96, 0.99)):
        want = codes_of(x[kept], layout.config, ratio, 1.0)
        assert torch.equal(scale, want[1][..., 0]) and torch.equal(zero, want[2][..., 0])
        assert torch.equal(codes, want[0].to(torch.uint8))
    # Nothing else of the buffer has changed.
    rec_view = rec.clone()
    rec_view[..., :264] = 171
    assert bool((rec_view == 171).all())
    touched = torch.ones(history.numel(), dtype=torch.bool, device=DEV)
    page = layout.physical_block_tokens
    view = touched.view(-1, layout.stripe_page_bytes)[:, : page * hk * SLOT].unflatten(1, (page, hk, SLOT))
    view[slots[kept] // page, slots[kept] % page] = False
    assert bool((history[touched] == 171).all())
    # And read_records gives the values they stand for.
    back = kernels.read_records(history, slots, layout)
    for got_rows, (codes, scale, zero) in zip(back, parts):
        value = codes.float() * scale.float()[..., None] + zero.float()[..., None]
        assert torch.equal(got_rows[kept], value.bfloat16())
        dead = slots < 0
        assert not bool(got_rows[dead].any())


@pytest.mark.parametrize("rotary,interleaved", [(64, False), (128, False), (192, False), (256, False), (0, False),
                                                (8, True), (96, True), (256, True), (32, False), (20, False)])
@pytest.mark.parametrize("n,live,hq,hk,axes", [(700, 700, 6, 1, 1), (1100, 1001, 3, 2, 3), (5000, 4999, 1, 1, 2)])
def test_many_rows(rotary, interleaved, n, live, hq, hk, axes):
    """The walk over many rows gives what few rows at a time give, bit for bit, NaN rows and all."""
    for table, weight, norm, rotate in ((torch.float32, torch.bfloat16, True, True),
                                        (torch.bfloat16, torch.float32, True, False),
                                        (torch.bfloat16, torch.float32, False, True)):
        m = list(make(n, hq, hk, rotary, axes, table=table, weight=weight))
        layout = layout_of(hk, k_clip_ratio=0.97, v_clip_ratio=0.99)
        history, slots = cache(n, layout, n // 768 + 2)
        slots[live // 3] = -1
        if rotary:
            m[5][axes - 1, 400], m[5][0, 90] = m[4].shape[0], -1
        if rotary == 0:
            m[4] = torch.zeros(1, 0, device=DEV)
        args = dict(norm=norm, axes=axes > 1, interleaved=interleaved, rotate_query=rotate)
        got = append(m, layout, history, slots, counts_of(live), **args)
        small = torch.full_like(history, 171)
        rows = [None if x is None else torch.empty_like(x) for x in got]
        step = 300
        for t0 in range(0, n, step):
            part = [x[t0 : t0 + step] for x in m[:3]] + m[3:5] + [m[5][:, t0 : t0 + step]] + m[6:]
            one = append(part, layout, small, slots[t0 : t0 + step].clone(),
                         counts_of(max(0, min(live - t0, step))), **args)
            for x, y in zip(rows, one):
                if x is not None:
                    x[t0 : t0 + step] = y
        for x, y in zip(got, rows):
            assert (x is None and y is None) or torch.equal(x.view(torch.int16), y.view(torch.int16))
        assert torch.equal(history, small)
        if rotary:
            assert bool(got[1][400].isnan().all()) and bool(got[1][90].isnan().all())
            key, value = kernels.read_records(history, slots, layout)
            assert bool(key[400].isnan().all()) and bool(value[400].isfinite().all())


@pytest.mark.parametrize("mode,k,v", [("factor", 0.8, 1.0), ("percentile", 0, 0.875), ("percentile", 1.0, 0.93)])
@pytest.mark.parametrize("n", [70, 1500])
def test_clip_modes(mode, k, v, n):
    m = make(n, 3, 1, 64)
    config = (dict(k_clip_factor=k, v_clip_factor=v) if mode == "factor"
              else dict(k_clip_ratio=k, v_clip_ratio=v))
    layout = layout_of(1, clip_mode=mode, **config)
    history, slots = cache(n, layout, 3)
    got = append(m, layout, history, slots, counts_of(n), axes=False)
    rotated = kernels.rotate(got[1], m[7].T), kernels.rotate(m[2], m[8].T)
    parts, _ = record_parts(history, layout, slots)
    for (codes, scale, zero), x, value in zip(parts, rotated, (k, v)):
        want = codes_of(x, layout.config, value, value)
        assert torch.equal(scale, want[1][..., 0]) and torch.equal(zero, want[2][..., 0])
        assert torch.equal(codes, want[0].to(torch.uint8))


def test_the_clip_search_takes_the_least_error():
    """The chosen factor's squared error in 64 bits is the least of the eight, but for the rounding of the
    kernel's fp32 sums (256 terms through a tree: 12 x 2^-24, and the terms' own steps, which are bounded
    by 2^-20 of the error and of the row's largest value times it)."""
    n = 200
    m = make(n, 1, 2, 64)
    layout = layout_of(2, clip_mode="search")
    history, slots = cache(n, layout, 2)
    got = append(m, layout, history, slots, counts_of(n), axes=False)
    rotated = kernels.rotate(got[1], m[7].T), kernels.rotate(m[2], m[8].T)
    parts, _ = record_parts(history, layout, slots)
    for (codes, scale, zero), x in zip(parts, rotated):
        x = x.double()
        decoded = codes.double() * scale.double()[..., None] + zero.double()[..., None]
        error = (decoded - x).square().sum(-1)
        best = torch.full_like(error, float("inf"))
        for i in range(8):
            cfg = layout_of(2, clip_mode="factor", k_clip_factor=1.0, v_clip_factor=1.0).config
            c, s, z = codes_of(x.float(), cfg, 0, 0.6 + 0.4 * i / 7)
            best = torch.minimum(best, (c.double() * s.double() + z.double() - x).square().sum(-1))
        top = x.abs().amax(-1)
        # |d(err^2)| <= 2 err 2^-21 top a value; summed over 256 by Cauchy-Schwarz.
        slack = best * 2.0**-19 + 2 * 16 * best.sqrt() * top * 2.0**-21
        assert bool((error <= best + slack).all())


def test_without_query_or_values():
    n = 50
    m = make(n, 4, 2, 64, 2)
    query, key, value, w, cs, pos, order, rk_t, rv_t = m
    layout = layout_of(2)
    whole, slots = cache(n, layout, 2)
    full = append(m, layout, whole, slots, counts_of(n))
    alone, _ = cache(n, layout, 2)
    got = kernels.rope_append(None, key, value, alone, slots, counts_of(n), layout, rk_t, rv_t, cos_sin=cs,
                              positions=pos, axes=order, k_weight=w[1], eps=1e-5)
    assert got[0] is None and got[2] is None and torch.equal(got[1], full[1])
    assert torch.equal(alone, whole)
    got = kernels.rope_append(query, key, None, None, None, None, None, rk_t, None, cos_sin=cs,
                              positions=pos, axes=order, q_weight=w[0], k_weight=w[1], eps=1e-5)
    assert all(torch.equal(a, b) for a, b in zip(got, full))
    # No position rotation and no norms: the rows themselves, rotated and stored.
    plain, _ = cache(n, layout, 2)
    got = kernels.rope_append(query, key, value, plain, slots, counts_of(n), layout, rk_t, rv_t,
                              rotate_query=False)
    assert torch.equal(got[0], query) and torch.equal(got[1], key) and got[2] is None
    parts, _ = record_parts(plain, layout, slots)
    want = codes_of(kernels.rotate(key, rk_t.T), layout.config, layout.config.k_clip_ratio, 1.0)
    assert torch.equal(parts[0][0], want[0].to(torch.uint8))
    empty = kernels.rope_append(query[:0], key[:0], value[:0], plain, slots, counts_of(0), layout, rk_t,
                                rv_t)
    assert all(t.shape[0] == 0 for t in empty)


def test_strides_and_slots_outside_the_buffer():
    n = 20
    m = list(make(n, 3, 1, 64))
    layout = layout_of(1)
    history, slots = cache(n, layout, 2)
    want = append(m, layout, history, slots, counts_of(n), axes=False)
    again, _ = cache(n, layout, 2)
    odd = [torch.zeros(n, t.shape[1], 259, dtype=torch.bfloat16, device=DEV) for t in m[:3]]
    for t, x in zip(odd, m[:3]):
        t[..., 1:257] = x
    got = append([t[..., 1:257] for t in odd] + m[3:], layout, again, slots, counts_of(n), axes=False)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(again, history)
    cut, _ = cache(n, layout, 2)
    far = slots.clone()
    far[3], far[4] = 2 * 768, (1 << 63) - 1
    append(m, layout, cut, far, counts_of(n), axes=False)
    inside = torch.ones(n, dtype=torch.bool, device=DEV)
    inside[3:5] = False
    mine, theirs = (record_parts(h, layout, slots[inside])[1] for h in (cut, history))
    assert torch.equal(mine, theirs)
    key, value = kernels.read_records(cut, far, layout)
    assert not bool(key[3:5].any()) and not bool(value[3:5].any())


@pytest.mark.parametrize("n", [8, 1400])
def test_extreme_rows(n):
    """Rows of zeros, equal values, tiny and huge ones: records of the same steps in torch."""
    m = list(make(n, 1, 1, 64))
    value = m[2].clone()
    value[0], value[1], value[2], value[3] = 0, 1.5, value[2] * 2.0**-30, value[3] * 2.0**12
    value[4], value[5, 0, 0] = -value[4].abs(), 3e4
    m[2] = value
    value[6] = 0  # nearly every value equal, a few far out: a threshold in the lowest bits
    value[6, 0, 3:9] = 2.0**20
    layout = layout_of(1)
    history, slots = cache(n, layout, 2)
    append(m, layout, history, slots, counts_of(n), axes=False)
    x = kernels.rotate(value, m[8].T)
    (_, (codes, scale, zero)), _ = record_parts(history, layout, slots)
    want = codes_of(x, layout.config, layout.config.v_clip_ratio, 1.0)
    assert torch.equal(scale, want[1][..., 0]) and torch.equal(zero, want[2][..., 0])
    assert torch.equal(codes, want[0].to(torch.uint8))
    m[2][7, 0, 17] = float("nan")
    append(m, layout, history, slots, counts_of(n), axes=False)
    assert bool(kernels.read_records(history, slots[7:8], layout)[1].isnan().all())


@pytest.mark.parametrize("n", [8, 1400, 2200])
@pytest.mark.parametrize("ratio", [1.0, 0.997, 0.99, 252 / 255, 0.985, 0.9, 0.875])
def test_order_statistics(n, ratio):
    """Rows of one sign, of few different values, of magnitudes over many powers of two, unturned."""
    m = list(make(n, 1, 1, 0))
    one = torch.eye(256, dtype=torch.bfloat16, device=DEV)
    x = m[2].float()
    x[0::8], x[1::8] = x[0::8].abs() + 0.01, -x[1::8].abs() - 0.01
    x[2::8] = (x[2::8] * 2).round() / 2  # many equal ones, zeros of either sign
    x[3::8] *= 2.0 ** torch.randint(-12, 3, x[3::8].shape, device=DEV)
    x[4::8] = x[4::8].sign() * 2.0**-100
    x[5::8, :, 5] = 1e30
    value = x.bfloat16()
    layout = layout_of(1, k_clip_ratio=ratio, v_clip_ratio=ratio)
    history, slots = cache(n, layout, n // 768 + 2)
    kernels.rope_append(None, value.flip(-1), value, history, slots, counts_of(n), layout, one, one)
    parts, _ = record_parts(history, layout, slots)
    for (codes, scale, zero), rows in zip(parts, (value.flip(-1), value)):
        want = codes_of(rows, layout.config, ratio, 1.0)
        # A zero point of zero is one of either sign.
        assert torch.equal(scale, want[1][..., 0]) and bool((zero == want[2][..., 0]).all())
        assert torch.equal(codes, want[0].to(torch.uint8))


@pytest.mark.parametrize("clip", [dict(v_clip_ratio=1.0), dict(v_clip_ratio=0.99), dict(v_clip_ratio=0.9),
                                  dict(v_clip_ratio=0), dict(clip_mode="factor", v_clip_factor=0.8)])
def test_rows_that_are_not_finite(clip):
    """Infinities, overflows and NaN: many rows at a time and few give the same bytes, and other rows keep
    theirs."""
    n = 2400
    m = list(make(n, 1, 1, 0))
    value = m[2].clone()
    value[0::7, 0, 3], value[1::7, 0, 5] = float("inf"), float("-inf")
    value[2::7, 0, 90:101:10], value[3::7], value[4::7, 0, 9] = 3e38, value[3::7] * 1e38, float("nan")
    layout = layout_of(1, **clip)
    for rv_t in (m[8], torch.eye(256, dtype=torch.bfloat16, device=DEV)):
        history, slots = cache(n, layout, n // 768 + 2)
        few = history.clone()
        finite = history.clone()
        kernels.rope_append(None, m[1], value, history, slots, counts_of(n), layout, m[7], rv_t)
        for a in range(0, n, 400):
            part = slice(a, a + 400)
            kernels.rope_append(None, m[1][part], value[part], few, slots[part].contiguous(), counts_of(400),
                                layout, m[7], rv_t)
        kernels.rope_append(None, m[1], m[2], finite, slots, counts_of(n), layout, m[7], rv_t)
        assert torch.equal(history, few)
        rows = [record_parts(h, layout, slots)[1][5::7] for h in (history, finite)]
        assert torch.equal(*rows)


@pytest.mark.parametrize("n", [40, 900])
def test_a_captured_append_replays(n):
    m = make(n, 6, 1, 64, 3)
    layout = layout_of(1)
    history, slots = cache(n, layout, 2)
    counts = counts_of(n)
    append(m, layout, history, slots, counts)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = append(m, layout, history, slots, counts)
    for live in (n, 1, 0, 33, n):
        counts[1] = live
        m[5].copy_(m[5].roll(1, 1))
        slots.copy_(slots.roll(3))
        history.fill_(171)
        graph.replay()
        torch.cuda.synchronize()
        fresh = torch.full_like(history, 171)
        eager = append(m, layout, fresh, slots, counts)
        assert all(torch.equal(a, b) for a, b in zip(got, eager)) and torch.equal(history, fresh)


def test_a_slot_beyond_4_gb():
    layout = layout_of(2)
    n, pages = 3, 5600
    m = make(n, 2, 2, 64)
    history = torch.zeros(pages * layout.stripe_page_bytes, dtype=torch.uint8, device=DEV)
    slots = torch.tensor([pages * 768 - 1, pages * 768 - 700, 5], device=DEV)
    append(m, layout, history, slots, counts_of(n), axes=False)
    small, near = cache(n, layout, 2)
    append(m, layout, small, near, counts_of(n), axes=False)
    for a, b in zip(kernels.read_records(history, slots, layout), kernels.read_records(small, near, layout)):
        assert torch.equal(a, b)


def test_refusals_on_the_device():
    m = make(6, 4, 2, 64, 3)
    q, k, v, w, cs, pos, order, rk_t, rv_t = m
    layout = layout_of(2)
    history, slots = cache(6, layout, 2)
    counts = counts_of(6)

    def call(q=q, k=k, v=v, slots=slots, counts=counts, layout=layout, rk_t=rk_t, rv_t=rv_t, cs=cs, pos=pos,
             order=order, qw=w[0], kw=w[1]):
        return kernels.rope_append(q, k, v, history, slots, counts, layout, rk_t, rv_t, cos_sin=cs,
                                   positions=pos, axes=order, q_weight=qw, k_weight=kw)

    bad = dict(q=q[:5], k=k[..., :128], v=v[:, :1], slots=slots[:5], counts=counts.long(), rk_t=None,
               rv_t=rv_t.float(), cs=cs[:, :63], pos=pos[:, :5], order=order[:31], qw=w[0][:128], kw=None,
               layout=layout_of(1))
    for name, value in bad.items():
        with pytest.raises(ValueError):
            call(**{name: value})
    for over in (dict(order=None), dict(cs=None), dict(pos=pos.int()), dict(counts=None),
                 dict(slots=slots.int()), dict(order=order.long())):
        with pytest.raises(ValueError):
            call(**over)
    with pytest.raises(ValueError):
        kernels.read_records(history, slots.int(), layout)
    with pytest.raises(ValueError, match="weights"):
        kernels.qk_norm_rope(q, k, None, None, cs, pos, axes=order)
    with pytest.raises(RuntimeError):
        call(pos=pos.cpu())
