"""The kernels of attention inside segments, of projections and of embedding rows keep nothing in memory that belongs in registers: a
build that spills is found here, without a GPU, and refused by the library's own build."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "graphiler_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc"
SOURCES = ["segment_attn", "segment_attn_grad", "linear_act", "linear_split", "embedding"]


@pytest.mark.parametrize("source", SOURCES)
def test_the_build_refuses_spills(source):
    with open(os.path.join(CSRC, "Makefile")) as f:
        lists = re.findall(r"^UNSPILLED(?:_VECTORS)? = (.*)$", f.read(), re.M)
    assert any(source in names.split() for names in lists)


def usage_of(source, where):
    """The compiler's report: the last build's where it is of these sources, else one made here."""
    kept = os.path.join(CSRC, "build", source + ".usage")
    made_of = [os.path.join(CSRC, n) for n in os.listdir(CSRC) if n.endswith(".h") or n in (source + ".hip", "Makefile")]
    if os.path.exists(kept) and all(os.path.getmtime(kept) > os.path.getmtime(n) for n in made_of):
        with open(kept) as f:
            return f.read()
    r = subprocess.run([HIPCC if os.path.exists(HIPCC) else "hipcc", "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang",
                        "-target-feature", "-Xclang", "-packed-fp32-ops", "-Rpass-analysis=kernel-resource-usage",
                        "--cuda-device-only", "-c", source + ".hip", "-o", str(where / "kernel.o")],
                       cwd=CSRC, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stderr


@pytest.mark.skipif(not (os.path.exists(HIPCC) or shutil.which("hipcc")), reason="no hipcc")
@pytest.mark.parametrize("source", SOURCES)
def test_nothing_is_spilled(tmp_path, source):
    said = usage_of(source, tmp_path)
    spilled, scratch = ([int(x) for x in re.findall(what + r": (\d+)", said)] for what in ("VGPRs Spill", r"ScratchSize \[bytes/lane\]"))
    assert spilled and len(spilled) == len(scratch)
    assert not any(spilled) and not any(scratch), (spilled, scratch)
