"""The kernels of 4-bit records in the ISA that hipcc emits (no GPU): their direct-to-LDS loads against the
GFX9 hazard of tests/test_isa_hazards.py, and no registers in scratch memory, on which their forms rest."""

import re
import subprocess
from pathlib import Path

import pytest

from tests.test_isa_hazards import HIPCC, ROOT, _late_sites


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc is not installed")
@pytest.mark.parametrize("source,loads,kernels", [("history4.hip", 27, "history4_"), ("append.hip", 16, "")])
def test_loads_and_registers(tmp_path, source, loads, kernels):
    out = tmp_path / "kernels.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17",
                    "-fno-gpu-flush-denormals-to-zero", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", f"-I{ROOT / 'include'}", "--cuda-device-only", "-S",
                    str(ROOT / "oscar_new_amd" / "csrc" / source), "-o", str(out)],
                   check=True, capture_output=True, timeout=600)
    text = out.read_text()
    assert text.count("global_load_lds_dword") >= loads
    assert _late_sites(text) == []
    bodies = re.findall(r"^_Z\S*%s\S*:.*?\.end_amdhsa_kernel" % kernels, text, re.S | re.M)
    assert bodies and not any("scratch_" in re.sub(r"\.amdhsa.*", "", body) for body in bodies)
