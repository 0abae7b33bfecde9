"""Host-side refusals of the norm, page and shared-prefix entry points (no GPU: nothing is
launched; the addresses are fake, aligned and never dereferenced)."""

import torch
import pytest

from oscar_new_amd import _ext, kernels

A = 1 << 20


def layout(**over):
    fields = dict(head_dim=256, kv_heads=1, bp=768, bk=128, slot=160, vector=68, sink=4, recent=128,
                  ring=132, reserved=0, page=393216)
    fields.update(over)
    return _ext.OscarLayout(*fields.values())


def test_qk_norm_rope():
    def call(q=A, q_s0=1536, key=A, n=4, hq=6, hk=1, eps=1e-6, table=A, rows=100, stride=64,
             rotary=64, positions=A, out=A, rk_t=None, q_rot=None):
        return _ext.library().oscar_qk_norm_rope(q, q_s0, 256, key, 256, 256, n, hq, hk, A, A, 0, 0,
                                                 eps, table, rows, stride, 0, rotary, 0, positions,
                                                 None, out, A, rk_t, q_rot, None)

    assert call(n=0) == 0
    assert call(n=-1) == -2 and call(hq=0) == -2 and call(hk=0) == -2
    assert call(rotary=63) == -2 and call(rotary=258, stride=258) == -2 and call(rotary=-2) == -2
    assert call(stride=32) == -2 and call(rows=0) == -2
    assert call(n=1 << 31) == -2 and call(n=1 << 29) == -2
    assert call(n=1 << 27, hq=1) == -2  # more threads than a launch holds
    assert call(q=None) == -1 and call(table=None) == -1 and call(positions=None) == -1
    assert call(rk_t=A) == -1 and call(q_rot=A) == -1
    assert call(q=A + 2) == -4 and call(q_s0=1537) == -4 and call(out=A + 8) == -4
    assert call(rk_t=A + 2, q_rot=A) == -4
    assert call(eps=-1.0) == -5 and call(eps=float("nan")) == -5


def test_pages():
    lib = _ext.library()

    def free(num=10, table=A, stride=12, columns=12, rows=4, lay=layout(), used=A):
        return lib.oscar_free_pages(num, table, stride, columns, rows, A, A, lay, used, A, A, None)

    def fork(stripes=A, layers=2, num=10, table=A, stride=12, columns=12, rows=4, forks=2,
             lay=layout(), status=A):
        return lib.oscar_fork_requests(stripes, layers, num, table, stride, columns, rows, A, A, A,
                                       A, forks, lay, status, None)

    def compact(stripes=A, layers=2, num=10, table=A, stride=12, columns=12, rows=4, lay=layout(),
                scratch=A):
        return lib.oscar_compact_pages(stripes, layers, num, table, stride, columns, rows, A, A,
                                       lay, scratch, A, A, None)

    assert fork(forks=0) == 0
    for call in (free, fork, compact):
        assert call(num=0) == -2 and call(num=1 << 31) == -2 and call(rows=0) == -2
        assert call(stride=11) == -2 and call(columns=0) == -2
        assert call(table=None) == -1 and call(lay=layout(page=1)) == -3
    assert free(used=None) == -1 and compact(scratch=None) == -1 and fork(status=None) == -1
    for call in (fork, compact):
        assert call(stripes=None) == -1 and call(layers=0) == -2 and call(layers=65536) == -2
    assert fork(forks=-1) == -2 and fork(forks=4097) == -2


def test_shared_prefixes():
    lib = _ext.library()

    def plan(groups=2, reqs=8, tokens=8, hq=6, slots=64, lay=layout(), units=A, capacity=700,
             starts=A):
        return lib.oscar_shared_plan(A, A, A, starts, A, groups, reqs, tokens, hq, slots, lay,
                                     units, capacity, A, A, None)

    def attend(q=A, history=A, units=A, capacity=700, used=A, n=8, hq=6, slots=64, scale=1 / 16,
               lay=layout(), out=A, history_bytes=1 << 24):
        return lib.oscar_shared_history(q, 1536, 256, 1, history, history_bytes, A, 64, 64, A, units,
                                        capacity, A, used, n, hq, slots, scale, lay, A, A, 0, out,
                                        A, None)

    assert plan(groups=-1) == -2 and plan(reqs=0) == -2 and plan(tokens=-1) == -2
    assert plan(hq=0) == -2 and plan(slots=3) == -2 and plan(slots=257) == -2
    assert plan(groups=8000, reqs=200) == -5 and plan(hq=33) == -5
    least = lib.oscar_shared_capacity(8, 6, 2, 8, 1)
    assert plan(capacity=least - 1) == -2  # below what the plan may write
    assert lib.oscar_shared_capacity(8, 0, 2, 8, 1) == -1
    assert plan(units=None) == -1 and plan(starts=None) == -1 and plan(units=A + 4) == -4
    assert plan(lay=layout(page=1)) == -3
    assert attend(n=0) == 0
    assert attend(slots=3) == -2 and attend(slots=257) == -2 and attend(capacity=0) == -2
    assert attend(n=1 << 22) == -2 and attend(capacity=1 << 23) == -2  # threads of a launch
    assert attend(n=-1) == -2 and attend(hq=0) == -2 and attend(history_bytes=64) == -2
    assert attend(q=None) == -1 and attend(used=None) == -1 and attend(out=None) == -1
    assert attend(q=A + 2) == -4 and attend(out=A + 4) == -4 and attend(history=A + 4) == -4
    assert attend(scale=0.0) == -5 and attend(hq=33) == -5 and attend(lay=layout(bk=32)) == -5


def test_tensors_on_the_host_are_refused():
    q = torch.zeros(2, 6, 256, dtype=torch.bfloat16)
    w = torch.zeros(256)
    with pytest.raises(RuntimeError):
        kernels.qk_norm_rope(q, q[:, :1], w, w, torch.zeros(4, 64), torch.zeros(2, dtype=torch.int64))


def test_shared_history_takes_heads_of_256():
    plan = kernels.SharedPlan(None, 1, 4, 6, 1, 8, None, None)
    for d in (128, 512):
        with pytest.raises(ValueError, match="256"):
            kernels.shared_history(torch.zeros(2, 6, d), None, None, plan, None, 1 / 16)
