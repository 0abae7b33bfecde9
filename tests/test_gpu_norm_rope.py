"""``kernels.qk_norm_rope`` against the formulas in 64 bits.

Error bound of an element, from the arithmetic: one rounding to bf16 (2^-8 relative to the value)
after fp32 steps. The sum of 256 squares has at most 13 additions on a path, so 13 x 2^-24, halved by
the square root; the root, the division, two products and the two products and the addition of the
turn add 7 x 2^-24 of |y| + |partner|: below 2^-19 of twice the row's largest normalized value.
"""

import pytest
import torch

from oscar_new_amd import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"


def formula(x, weight, cos_sin, positions, eps, unit_offset, interleaved):
    """float64 rows, and each row's largest normalized magnitude."""
    x = x.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    y = y * (weight.double() + (1.0 if unit_offset else 0.0))
    largest = y.abs().amax(-1, keepdim=True)
    half = cos_sin.shape[1] // 2
    angle = cos_sin[positions].double()[:, None]
    cos, sin = angle[..., :half], angle[..., half:]
    out = y.clone()
    if interleaved:
        a, b = y[..., 0 : 2 * half : 2], y[..., 1 : 2 * half : 2]
        out[..., 0 : 2 * half : 2] = a * cos - b * sin
        out[..., 1 : 2 * half : 2] = b * cos + a * sin
    else:
        a, b = y[..., :half], y[..., half : 2 * half]
        out[..., :half] = a * cos - b * sin
        out[..., half : 2 * half] = b * cos + a * sin
    return out, largest


def make(n, hq, hk, rotary, positions=977, table=torch.float32, weight=torch.float32, seed=3):
    gen = torch.Generator(device=DEV).manual_seed(seed + n + rotary)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    # Rows inside a packed projection output: [query, gate] per query head, keys behind them.
    packed = (rand(n, (2 * hq + hk) * 256) * (rand(n, 1).abs() + 0.1)).bfloat16()
    query = packed[:, : 2 * hq * 256].view(n, hq, 512)[..., :256]
    key = packed[:, 2 * hq * 256 :].view(n, hk, 256)
    angle = rand(positions, rotary // 2) * 3
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).to(table)
    pos = torch.randint(positions, (n,), generator=gen, device=DEV)
    if n > 1:
        pos[0], pos[1] = 0, positions - 1
    weights = [(rand(256) * 0.4 + 1).to(weight) for _ in range(2)]
    rk = torch.linalg.qr(rand(256, 256))[0].bfloat16().contiguous()
    return query, key, weights, cos_sin, pos, rk


def check(got, x, weight, cos_sin, pos, eps, unit_offset, interleaved):
    want, largest = formula(x, weight, cos_sin, pos, eps, unit_offset, interleaved)
    bound = want.abs() * 2.0**-8 + largest * 2.0**-18
    assert got.is_contiguous() and got.dtype == torch.bfloat16
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("n,hq,hk", [(1, 6, 1), (2, 1, 1), (17, 5, 2), (33, 16, 4), (700, 6, 1),
                                     (1031, 12, 2)])
@pytest.mark.parametrize("rotary,interleaved", [(64, False), (96, False), (256, False), (64, True),
                                                (256, True), (20, False), (6, True), (2, False),
                                                (0, False)])
def test_rows_against_64_bits(n, hq, hk, rotary, interleaved):
    for table, weight, unit in ((torch.float32, torch.float32, False),
                                (torch.bfloat16, torch.bfloat16, True)):
        q, k, w, cs, pos, rk = make(n, hq, hk, rotary, table=table, weight=weight)
        args = (q, k, *w, cs, pos)
        got = kernels.qk_norm_rope(*args, eps=1e-5, unit_offset=unit, interleaved=interleaved)
        check(got[0], q, w[0], cs, pos, 1e-5, unit, interleaved)
        check(got[1], k, w[1], cs, pos, 1e-5, unit, interleaved)
        turned = kernels.qk_norm_rope(*args, eps=1e-5, unit_offset=unit, interleaved=interleaved,
                                      rk_t=rk.T.contiguous())
        assert torch.equal(turned[0], got[0]) and torch.equal(turned[1], got[1])
        assert torch.equal(turned[2], kernels.rotate(got[0], rk))


@pytest.mark.parametrize("n,hq,hk,live", [(700, 6, 1, 700), (321, 6, 2, 300), (6001, 6, 1, 5500)])
@pytest.mark.parametrize("rotary,interleaved", [(64, False), (128, False), (192, False),
                                                (256, False), (0, False), (8, True), (96, True),
                                                (256, True), (32, False)])
def test_walks_of_many_rows(n, hq, hk, live, rotary, interleaved):
    """Each wavefront's rows by itself, one block or several, against the formulas and with the bits
    of the form without R_k and of ``rotate``."""
    for table, weight, unit in ((torch.float32, torch.bfloat16, False),
                                (torch.bfloat16, torch.float32, True)):
        q, k, w, cs, pos, rk = make(n, hq, hk, rotary, table=table, weight=weight)
        if live > 400 and rotary:
            pos[400], pos[live - 1] = cs.shape[0], -1
        counts = torch.tensor([1, live], dtype=torch.int32, device=DEV)
        args = dict(counts=counts, eps=1e-6, unit_offset=unit, interleaved=interleaved)
        got = kernels.qk_norm_rope(q, k, *w, cs, pos, **args)
        turned = kernels.qk_norm_rope(q, k, *w, cs, pos, rk_t=rk.T.contiguous(), **args)
        bad = [400, live - 1] if live > 400 and rotary else []
        good = [t for t in range(live) if t not in bad]
        for i, x in enumerate((q, k)):
            check(turned[i][good].contiguous(), x[good], w[i], cs, pos[good], 1e-6, unit,
                  interleaved)
        for t, plain in zip(turned, (*got, kernels.rotate(got[0], rk))):
            assert torch.equal(t[good], plain[good])
            assert bool(t[bad].isnan().all()) and not bool(t[live:].any())


@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("n,live", [(5, 3), (40, 0), (700, 511)])
def test_rows_past_the_live_tokens_are_zero(n, live, rotate):
    q, k, w, cs, pos, rk = make(n, 6, 1, 64)
    pos[live:] = 1 << 40  # a padded row's position is not read
    counts = torch.tensor([1, live], dtype=torch.int32, device=DEV)
    rk_t = rk.T.contiguous() if rotate else None
    got = kernels.qk_norm_rope(q, k, *w, cs, pos, counts=counts, rk_t=rk_t)
    for t in got:
        assert not bool(t[live:].any()) and bool(t[:live].isfinite().all())
    whole = kernels.qk_norm_rope(q[:live], k[:live], *w, cs, pos[:live], rk_t=rk_t)
    assert all(torch.equal(a[:live], b) for a, b in zip(got, whole))


def test_positions_outside_the_table_give_nan_rows():
    q, k, w, cs, pos, rk = make(9, 6, 1, 64)
    pos[2], pos[5] = -1, cs.shape[0]
    for t in kernels.qk_norm_rope(q, k, *w, cs, pos, rk_t=rk.T.contiguous()):
        bad = t.isnan().flatten(1)
        assert bool(bad[[2, 5]].all()) and not bool(bad[[0, 1, 3, 4, 6, 7, 8]].any())


def test_zero_and_infinite_rows():
    q, k, w, cs, pos, rk = make(4, 2, 1, 64)
    q, k = q.clone(), k.clone()
    q[0], k[1] = 0, 0
    q[2, 0, 100] = float("inf")  # outside the turned dims: 0 times its weight, NaN in its place
    q[3, 1, 7] = float("nan")
    got_q, got_k = kernels.qk_norm_rope(q, k, *w, cs, pos)
    assert not bool(got_q[0].any()) and not bool(got_k[1].any())
    assert got_q[2, 0].isnan().nonzero().flatten().tolist() == [100]
    assert bool(got_q[3, 1].isnan().all()) and bool(got_q[3, 0].isfinite().all())


def test_unaligned_rows_and_far_token_strides():
    q, k, w, cs, pos, rk = make(11, 6, 1, 64)
    want = kernels.qk_norm_rope(q, k, *w, cs, pos)
    odd = torch.empty(11 * 6 * 256 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(11, 6, 256)
    odd.copy_(q)
    wide = torch.empty(11, 1, 1 << 20, dtype=torch.bfloat16, device=DEV)[..., :256]
    wide.copy_(k)
    table = torch.empty(cs.shape[0], 67, device=DEV)[:, 1:65]  # neither aligned nor packed
    table.copy_(cs)
    got = kernels.qk_norm_rope(odd, wide, *w, table, pos)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_many_rows_far_apart_with_zero_infinite_and_nan_rows():
    q, k, w, cs, pos, rk = make(700, 6, 1, 64)
    q, k, rk_t = q.clone(), k.clone(), rk.T.contiguous()
    q[100], k[101] = 0, 0
    q[699, 0, 100] = float("inf")  # outside the turned dims: 0 times its weight, NaN in its place
    q[350, 1, 7] = float("nan")
    far = torch.empty(700, 1 << 22, dtype=torch.bfloat16, device=DEV)  # 5.9 GB from end to end
    wide_q, wide_k = far[:, : 6 * 256].view(700, 6, 256), far[:, 4096:4352].view(700, 1, 256)
    wide_q.copy_(q)
    wide_k.copy_(k)
    plain = kernels.qk_norm_rope(wide_q, wide_k, *w, cs, pos)
    got = kernels.qk_norm_rope(wide_q, wide_k, *w, cs, pos, rk_t=rk_t)
    for x, y in zip(got, (*plain, kernels.rotate(plain[0], rk))):
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num())
    assert not bool(got[0][100].any()) and not bool(got[1][101].any())
    assert got[0][699, 0].isnan().nonzero().flatten().tolist() == [100]
    nan = got[0].isnan().flatten(0, 1)
    assert bool(nan[350 * 6 + 1].all()) and int(nan.any(1).sum()) == 2
    compact = kernels.qk_norm_rope(q, k, *w, cs, pos, rk_t=rk_t)
    for x, y in zip(got, compact):
        assert torch.equal(x.nan_to_num(), y.nan_to_num())


def test_no_tokens():
    q, k, w, cs, pos, rk = make(3, 6, 1, 64)
    got = kernels.qk_norm_rope(q[:0], k[:0], *w, cs, pos[:0], rk_t=rk.T.contiguous())
    assert [tuple(t.shape) for t in got] == [(0, 6, 256), (0, 1, 256), (0, 6, 256)]


@pytest.mark.parametrize("n", [32, 700])
def test_captured_and_on_another_stream(n):
    q, k, w, cs, pos, rk = make(n, 6, 1, 64)
    q, k, rk_t = q.clone(), k.clone(), rk.T.contiguous()
    counts = torch.tensor([1, n], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.qk_norm_rope(q, k, *w, cs, pos, counts=counts, rk_t=rk_t)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = kernels.qk_norm_rope(q, k, *w, cs, pos, counts=counts, rk_t=rk_t)
    torch.cuda.current_stream().wait_stream(side)
    for live in (n, 9, n - 1):
        q.normal_()
        pos.random_(cs.shape[0])
        counts[1] = live
        graph.replay()
        want = kernels.qk_norm_rope(q, k, *w, cs, pos, counts=counts, rk_t=rk_t)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    q, k, w, cs, pos, rk = make(4, 6, 1, 64)
    call = kernels.qk_norm_rope
    for args in ((q, k[:3], *w, cs, pos), (q[..., :128], k[..., :128], *w, cs, pos),
                 (q, k, w[0][:128], w[1], cs, pos), (q, k, w[0].half(), w[1], cs, pos),
                 (q, k, *w, cs.half(), pos), (q, k, *w, cs[:, :33], pos), (q, k, *w, cs[:0], pos),
                 (q, k, *w, cs, pos.int()), (q, k, *w, cs, pos[:3])):
        with pytest.raises(ValueError):
            call(*args)
    for rk_t in (rk.T, rk.float(), rk[:128]):
        with pytest.raises(ValueError):
            call(q, k, *w, cs, pos, rk_t=rk_t)
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            call(q, k, *w, cs, pos, eps=eps)
    with pytest.raises(RuntimeError):
        call(q.cpu(), k, *w, cs, pos)


@pytest.mark.parametrize("n", [5, 700])  # blocks through LDS and wavefronts by themselves
@pytest.mark.parametrize("rotary,interleaved", [(64, False), (256, False), (64, True), (20, False)])
def test_finite_rows_whose_squares_leave_the_range_of_fp32(n, rotary, interleaved):
    """Rows are normalized wherever their squares, sum or mean overflow or vanish in fp32. The bound
    is the one above: every step but the scaling by a power of two is the same."""
    q, k, w, cs, pos, rk = make(n, 4, 2, rotary)
    q, k, rk_t = torch.randn(n, 4, 256, device=DEV), torch.randn(n, 2, 256, device=DEV), rk.T
    for x in (q, k):
        x[0] *= 1e19  # each square above the largest fp32 value, or their sum
        x[1, 0] *= 3e17
        x[1, 1, 100] = 3.3e38
        x[2, 0, :] = 3.3e38
        x[2, 1, 1:] = 0
        x[2, 1, 0] = -3e38
        x[3] *= 1e-24  # each square below the smallest
        x[4, 0] *= 1e-19
        x[4, 1] = 2.0**-133  # bf16's smallest
    q, k, rk_t = q.bfloat16(), k.bfloat16(), rk_t.contiguous()
    for eps in (0.0, 1e-32):
        args = dict(eps=eps, interleaved=interleaved)
        got = kernels.qk_norm_rope(q, k, *w, cs, pos, **args)
        turned = kernels.qk_norm_rope(q, k, *w, cs, pos, rk_t=rk_t, **args)
        for i, x in enumerate((q, k)):
            check(got[i], x, w[i], cs, pos, eps, False, interleaved)
        for t, plain in zip(turned, (*got, kernels.rotate(got[0], rk))):
            assert torch.equal(t, plain)
    # An eps that leaves the range with the mean: rows of tiny values, not zeros.
    large = kernels.qk_norm_rope(q[:3], k[:3], *w, cs, pos[:3], eps=3e38, interleaved=interleaved)
    for i, x in enumerate((q[:3], k[:3])):
        want, largest = formula(x, w[i], cs, pos[:3], 3e38, False, interleaved)
        bound = want.abs() * 2.0**-8 + largest * 2.0**-18 + 2.0**-134
        assert bool(((large[i].double() - want).abs() <= bound).all())
