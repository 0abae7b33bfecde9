"""Clip percentiles that a configuration has by itself: 4-bit records want less clipping than 2-bit ones."""

from dataclasses import replace

import pytest

from oscar_new_amd.config import OscarConfig

RATIOS = {2: (0.96, 0.92), 4: (0.99, 0.99)}


def ratios(cfg):
    return cfg.k_clip_ratio, cfg.v_clip_ratio


@pytest.mark.parametrize("bits", [2, 4])
def test_by_the_bits_of_the_records(monkeypatch, bits):
    for name in ("VLLM_OSCAR_K_CLIP_RATIO", "VLLM_OSCAR_V_CLIP_RATIO"):
        monkeypatch.delenv(name, raising=False)
    monkeypatch.setenv("OSCAR_AMD_HISTORY_BITS", str(bits))
    made = OscarConfig(history_bits=bits)
    assert ratios(made) == RATIOS[bits] == ratios(OscarConfig.from_env())
    assert made == OscarConfig.from_env()
    assert made == OscarConfig(history_bits=bits, k_clip_ratio=RATIOS[bits][0], v_clip_ratio=RATIOS[bits][1])
    assert hash(made) == hash(OscarConfig.from_env())


@pytest.mark.parametrize("bits", [2, 4])
def test_given_ones_stay(monkeypatch, bits):
    assert ratios(OscarConfig(history_bits=bits, v_clip_ratio=0.0)) == (RATIOS[bits][0], 0.0)
    assert ratios(OscarConfig(history_bits=bits, k_clip_ratio=0.96)) == (0.96, RATIOS[bits][1])
    assert ratios(replace(OscarConfig(history_bits=bits), sink_tokens=8)) == RATIOS[bits]
    monkeypatch.setenv("OSCAR_AMD_HISTORY_BITS", str(bits))
    monkeypatch.setenv("VLLM_OSCAR_V_CLIP_RATIO", "0.9")
    assert OscarConfig.from_env().v_clip_ratio == 0.9
    with pytest.raises(ValueError):
        OscarConfig(history_bits=bits, k_clip_ratio=0.5)


def test_other_widths_are_refused():
    for bits in (3, 8):
        with pytest.raises(ValueError, match="2-bit or 4-bit"):
            OscarConfig(history_bits=bits)
