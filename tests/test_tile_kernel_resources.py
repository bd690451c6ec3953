"""The kernels of the norm, the tile products and the few rows keep everything in registers: a build that
spills is found here, without a GPU.  (Tiles of 256 x 256 hold 128 accumulators a lane and leave little room.)"""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "graphiler_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not (os.path.exists(HIPCC) or shutil.which("hipcc")), reason="no hipcc")
@pytest.mark.parametrize("source", ["norm", "gated", "gated_few", "gated_f32", "fp8_mm"])
def test_nothing_is_spilled(tmp_path, source):
    r = subprocess.run([HIPCC if os.path.exists(HIPCC) else "hipcc", "--offload-arch=gfx950", "-O3",
                        "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang",
                        "-packed-fp32-ops", "-Rpass-analysis=kernel-resource-usage", "--cuda-device-only", "-c",
                        source + ".hip", "-o", str(tmp_path / "kernel.o")],
                       cwd=CSRC, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "failed to meet occupancy" not in r.stderr
    spilled = [int(x) for x in re.findall(r"VGPRs Spill: (\d+)", r.stderr)]
    scratch = [int(x) for x in re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", r.stderr)]
    scalars = [int(x) for x in re.findall(r"SGPRs Spill: (\d+)", r.stderr)]
    assert spilled and len(spilled) == len(scratch) == len(scalars) and not any(scalars)
    assert not any(spilled) and not any(scratch), (spilled, scratch)
