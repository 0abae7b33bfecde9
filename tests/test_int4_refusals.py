"""Host-side refusals of the entry points around 4-bit records and position axes (no GPU: nothing is
launched; the addresses are fake, aligned and never dereferenced)."""

import pytest
import torch

from oscar_new_amd import _ext, kernels
from oscar_new_amd.config import OscarConfig
from oscar_new_amd.layout import CacheLayout

A = 1 << 20
CLIP = _ext.OscarClip(0, 0.99, 0.98, 1.0, 1.0)


def layout(bits=4, **over):
    fields = dict(head_dim=256, kv_heads=1, bp=768, bk=128, slot=272 if bits == 4 else 160,
                  vector=132 if bits == 4 else 68, sink=4, recent=128, ring=132, reserved=0, page=393216)
    fields.update(over)
    return _ext.OscarLayout(*fields.values())


def test_configuration():
    cfg = OscarConfig(history_bits=4)
    assert (cfg.data_bytes, cfg.vector_bytes, cfg.slot_bytes) == (128, 132, 272)
    assert OscarConfig().slot_bytes == 160 and OscarConfig().vector_bytes == 68
    for bits in (0, 1, 3, 8):
        with pytest.raises(ValueError, match="2-bit or 4-bit"):
            OscarConfig(history_bits=bits)
    lay = CacheLayout(768, 2, config=cfg)
    assert lay.slot_offset(769, 1) == 2 * 393216 + 3 * 272
    assert kernels.layout_struct(lay).slot_bytes == 272


def test_environment(monkeypatch):
    for name in ("OSCAR_AMD_HISTORY_BITS", "VLLM_OSCAR_K_CLIP_RATIO", "VLLM_OSCAR_V_CLIP_RATIO"):
        monkeypatch.delenv(name, raising=False)
    cfg = OscarConfig.from_env()
    assert (cfg.history_bits, cfg.k_clip_ratio, cfg.v_clip_ratio) == (2, 0.96, 0.92)
    monkeypatch.setenv("OSCAR_AMD_HISTORY_BITS", "4")
    cfg = OscarConfig.from_env()
    assert (cfg.history_bits, cfg.k_clip_ratio, cfg.v_clip_ratio) == (4, 0.99, 0.99)
    monkeypatch.setenv("VLLM_OSCAR_K_CLIP_RATIO", "0.97")
    assert OscarConfig.from_env().k_clip_ratio == 0.97
    monkeypatch.setenv("OSCAR_AMD_HISTORY_BITS", "3")
    with pytest.raises(ValueError):
        OscarConfig.from_env()


def append(query=A, q_s0=1536, key=A, value=A, n=4, hq=6, hk=1, qw=A, kw=A, eps=1e-6, table=A,
           rows=100, stride=64, fp32=0, rotary=64, positions=A, pos_stride=4, count=3, axes=A, counts=A,
           q_out=A, k_out=A, rk_t=A, rv_t=A, q_rot=A, history=A, size=1 << 24, slots=A, lay=layout(),
           clip=CLIP):
    return _ext.library().oscar_rope_append(
        query, q_s0, 256, key, 256, 256, value, 256, 256, n, hq, hk, qw, kw, 0, 0, eps, table, rows,
        stride, fp32, rotary, 0, positions, pos_stride, count, axes, counts, q_out, k_out, rk_t, rv_t,
        q_rot, history, size, slots, lay, clip, None)


def test_append():
    assert append(n=0) == 0
    assert append(n=-1) == -2 and append(hq=-1) == -2 and append(hk=0) == -2
    assert append(rotary=63) == -2 and append(rotary=258, stride=258) == -2 and append(rotary=-2) == -2
    assert append(stride=32) == -2 and append(rows=0) == -2
    assert append(count=0) == -2 and append(count=33) == -2 and append(pos_stride=3) == -2
    assert append(hk=2) == -2 and append(size=-1) == -2  # another head count than the layout's
    assert append(n=1 << 24) == -2 and append(n=1, hq=1 << 27) == -2  # threads of a launch
    assert append(clip=_ext.OscarClip(3, 0.99, 0.98, 1.0, 1.0)) == -2
    for name in ("key", "positions", "table", "axes", "k_out", "rk_t", "rv_t", "history", "slots",
                 "counts", "q_out", "query", "clip", "qw", "kw"):
        assert append(**{name: None}) == -1, name
    assert append(hq=0) == -1  # a query of no heads
    assert append(lay=layout(slot=288)) == -3 and append(lay=layout(page=1)) == -3
    assert append(lay=layout(2, slot=272)) == -3
    for name in ("query", "key", "value", "history", "q_out", "k_out", "rk_t", "rv_t", "q_rot", "qw", "kw"):
        assert append(**{name: A + 8}) == -4, name
    assert append(q_s0=1537) == -4 and append(table=A + 1) == -4 and append(table=A + 2, fp32=1) == -4
    assert append(eps=-1.0) == -5 and append(eps=float("nan")) == -5


def test_history():
    def attend(q=A, q_s0=1536, history=A, size=1 << 24, table=A, n=8, hq=6, programs=8, splits=8, bn=32,
               qt=4, mql=1, scale=1 / 16, st=-256, lay=layout(), partials=A, lse=A, tasks=A, tiles=0, reqs=8):
        return _ext.library().oscar_history_int4(q, q_s0, 256, 1, history, size, A, A, table, 64, 64, A,
                                                 tasks, A, n, hq, programs, splits, bn, qt, mql, scale, st,
                                                 tiles, reqs, lay, partials, lse, None)

    assert attend(n=0) == 0
    assert attend(n=-1) == -2 and attend(hq=0) == -2 and attend(programs=0) == -2
    assert attend(splits=0) == -2 and attend(splits=65536) == -2 and attend(qt=0) == -2
    assert attend(size=32 * 272 - 1) == -2  # fewer bytes than a masked chunk reads
    assert attend(size=(1 << 36) + 1, n=0) == -5  # block offsets of 32 bits
    assert attend(q=None) == -1 and attend(history=None) == -1 and attend(tasks=None) == -1
    assert attend(partials=None) == -1 and attend(lse=None) == -1
    assert attend(lay=layout(2)) == -3 and attend(lay=layout(slot=264)) == -3
    assert attend(q=A + 2) == -4 and attend(history=A + 8) == -4 and attend(q_s0=1537) == -4
    assert attend(scale=0.0) == -5 and attend(hq=33) == -5 and attend(hq=9, mql=4) == -5
    assert attend(programs=16385) == -5  # task rows of the device rule
    assert attend(programs=1 << 24, st=0) == -2 and attend(st=-(1 << 30)) == -2
    assert attend(tiles=1) == -5 and attend(tiles=1, st=0, reqs=0) == -2
    assert attend(tiles=1, st=0, n=1 << 30) == -2 and attend(tiles=1, st=0, n=1 << 27, splits=64) == -2


def test_read():
    def read(history=A, size=1 << 24, slots=A, n=4, lay=layout(), key=A, value=A):
        return _ext.library().oscar_read_records(history, size, slots, n, lay, key, value, None)

    assert read(n=0) == 0 and read(n=-1) == -2 and read(size=-1) == -2 and read(n=1 << 28) == -2
    assert read(history=None) == -1 and read(slots=None) == -1 and read(key=None) == -1
    assert read(lay=layout(page=1)) == -3
    assert read(history=A + 2) == -4 and read(key=A + 8) == -4 and read(value=A + 8) == -4


def test_kernels_of_2_bit_records_refuse_4_bit_layouts():
    lib, lay = _ext.library(), layout()
    assert lib.oscar_store_int2(A, A, 4, A, 1 << 24, A, A, lay, CLIP, None) == -3
    assert lib.oscar_rotate_store_int2(A, 256, 256, A, 256, 256, 4, A, A, A, 1 << 24, A, A, lay, CLIP,
                                       None) == -3
    assert lib.oscar_unpack(A, 1 << 24, A, 4, lay, A, A, None) == -3
    assert lib.oscar_shared_plan(A, A, A, A, A, 2, 8, 8, 6, 64, lay, A, 700, A, A, None) == -3
    assert lib.oscar_attention_partials(A, 1536, 256, 1, None, 0, 0, 1, None, 0, 0, 1, A, 1 << 24, A,
                                        1 << 20, A, A, A, 64, 64, A, A, A, 8, 6, 8, 8, 32, 4, 1, 1 / 16,
                                        0, 0, lay, A, A, None, None) == -3


def test_axes_of_sections():
    assert kernels.rope_axes([2, 3, 1]).tolist() == [0, 0, 1, 1, 1, 2]
    assert kernels.rope_axes([2, 2, 2], interleaved=True).tolist() == [0, 1, 2, 0, 1, 2]
    assert kernels.rope_axes([4, 2, 1], interleaved=True).tolist() == [0, 1, 2, 0, 1, 0, 0]
    assert kernels.rope_axes([5]).tolist() == [0] * 5
    assert kernels.rope_axes([0, 2]).tolist() == [1, 1]
    for bad in ([], [3, -1]):
        with pytest.raises(ValueError, match="sections"):
            kernels.rope_axes(bad)
    with pytest.raises(ValueError, match="turns"):
        kernels.rope_axes([1, 5, 1], interleaved=True)


def test_tensors_on_the_host_are_refused():
    q = torch.zeros(2, 6, 256, dtype=torch.bfloat16)
    pos, w = torch.zeros(2, dtype=torch.int64), torch.zeros(256)
    lay = CacheLayout(768, config=OscarConfig(history_bits=4))
    with pytest.raises(RuntimeError):
        kernels.rope_append(q, q[:, :1], q[:, :1], torch.zeros(393216, dtype=torch.uint8), pos, pos.int(),
                            lay, None, None)
    with pytest.raises(RuntimeError):
        kernels.qk_norm_rope(q, q[:, :1], w, w, torch.zeros(4, 64), pos.view(1, 2),
                             axes=torch.zeros(32, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        kernels.read_records(torch.zeros(393216, dtype=torch.uint8), pos, lay)
