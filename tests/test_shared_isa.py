"""The direct-to-LDS loads of the shared-prefix and chunk tiles against the GFX9 hazard of
tests/test_isa_hazards.py (a VALU write of an SGPR five wait states before the load reads it), from
the ISA that hipcc emits (no GPU)."""

import subprocess
from pathlib import Path

import pytest

from tests.test_isa_hazards import HIPCC, ROOT, _late_sites


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc is not installed")
@pytest.mark.parametrize("source,loads", [("shared.hip", 20), ("history_chunk.hip", 6),
                                          ("norm_rope.hip", 16)])
def test_tiles_keep_five_wait_states_before_every_dma(tmp_path, source, loads):
    out = tmp_path / "kernels.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17",
                    "-fno-gpu-flush-denormals-to-zero", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", f"-I{ROOT / 'include'}", "--cuda-device-only", "-S",
                    str(ROOT / "oscar_new_amd" / "csrc" / source), "-o", str(out)],
                   check=True, capture_output=True, timeout=600)
    text = out.read_text()
    assert text.count("global_load_lds_dword") >= loads
    assert _late_sites(text) == []
