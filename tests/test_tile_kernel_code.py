"""What the tile products rely on in the code that the compiler makes of them, without a GPU."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "graphiler_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc" if os.path.exists("/opt/rocm/bin/hipcc") else shutil.which("hipcc")

pytestmark = pytest.mark.skipif(not HIPCC, reason="no hipcc")

# Three forms of an epilogue whose addresses are reckoned for every chunk: many uses of the tile's place in vector registers.
FORMS = """
#include "tile_mm.h"
namespace ga {
template <int F> struct Forms : Stored<float> {
  static constexpr int kOut = 1;
  float *out; int64_t ld; int form;
  __host__ __device__ Forms(float *o, int64_t l, int f) : out(o), ld(l), form(f) {}
  template <typename G> __device__ __forceinline__ void visit(G g) const {
    if (form == 0) g(Forms<0>(out, ld, form));
    else if (form == 1) g(Forms<1>(out, ld, form));
    else g(Forms<2>(out, ld, form));
  }
  __device__ __forceinline__ void make(const TileMm &, int64_t, int64_t, const floatx4 &g, const floatx4 &u,
                                       floatx4 (&o)[1]) const {
    for (int r = 0; r < 4; ++r) o[0][r] = gate_of(F, g[r]) * u[r];
  }
  __device__ __forceinline__ void store(const TileMm &p, int, int64_t row, int64_t col, const uintx4 &w, int64_t) const {
    store_chunk(out + row * ld + col, w, p.cols - col);
  }
};
template __global__ void tile_mm_kernel<false, false, true, true, 2, 4, 8, 4, 0, Forms<-1>>(TileMm, Forms<-1>);
}
"""


def assembly(source, cwd, out):
    r = subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature",
                        "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S", source, "-o", str(out)],
                       cwd=cwd, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    text = out.read_text()
    starts = list(re.finditer(r"^(_ZN2ga\S*kernel\S+):\s*;", text, re.M))
    assert starts
    return {m.group(1): text[m.end():text.index(".Lfunc_end", m.end())].split("\n") for m in starts}


def loops_around_loads(lines):
    return sum("s_and_saveexec" in line and any("buffer_" in x for x in lines[i + 1:i + 3]) for i, line in enumerate(lines))


def test_a_tile_s_place_is_scalar_whatever_the_epilogue(tmp_path):
    """A descriptor in vector registers is taken lane by lane, in a loop behind which no lane is active: what the compiler
    spills there is lost.  As the library is built, what hides the epilogue's lane happens to keep descriptors scalar; here
    they have to be so without it."""
    folder = tmp_path / "graphiler_amd" / "csrc"
    folder.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    shutil.copy(os.path.join(CSRC, "..", "..", "include", "graphiler_amd.h"), tmp_path / "include")
    for name in ("common.h", "vec8.h", "tile_mm.h"):
        shutil.copy(os.path.join(CSRC, name), folder)
    header = (folder / "tile_mm.h").read_text()
    hidden = '    asm volatile("" : "+v"(lane));\n'
    assert header.count(hidden) == 1
    (folder / "tile_mm.h").write_text(header.replace(hidden, ""))
    (folder / "forms.hip").write_text(FORMS)
    for lines in assembly("forms.hip", folder, tmp_path / "forms.s").values():
        assert sum("buffer_load_dwordx4" in line and " lds" in line for line in lines) > 0
        assert loops_around_loads(lines) == 0
        assert not any("scratch_store" in line for line in lines)


@pytest.fixture(scope="module", params=["gated", "fp8_mm"])
def tile_kernels(request, tmp_path_factory):
    kernels = assembly(request.param + ".hip", CSRC, tmp_path_factory.mktemp("code") / "kernels.s")
    tiles = {k: v for k, v in kernels.items() if "tile_mm_kernel" in k}
    assert tiles
    return tiles


def test_no_descriptor_is_taken_lane_by_lane(tile_kernels):
    for name, lines in tile_kernels.items():
        assert loops_around_loads(lines) == 0, name


def test_the_first_wait_leaves_only_moves_of_the_second_step(tile_kernels):
    """The wait in front of the first barrier counts: all loads but the youngest n have arrived.  The first step's tiles
    are whole only if those n are moves of the second step, with every move of the first in front of them."""
    for name, lines in tile_kernels.items():
        moves = [i for i, line in enumerate(lines) if "buffer_load_dwordx4" in line and " lds" in line]
        fence = [i for i, line in enumerate(lines) if "; moves of the second step" in line]
        assert len(fence) == 1, name
        barrier = next(i for i, line in enumerate(lines) if "s_barrier" in line)
        assert fence[0] < barrier, name
        counts = [re.search(r"vmcnt\((\d+)\)", line) for line in lines[fence[0]:barrier] if "s_waitcnt" in line]
        n = int([c for c in counts if c][-1].group(1))
        assert n > 0 and sum(fence[0] < i < barrier for i in moves) == n, name
        assert sum(i < fence[0] for i in moves) in (2 * n - 1, 2 * n), name


# 48 values that are all alive between two barriers, in 24 registers
SPILLS = """
#include "common.h"
__global__ __attribute__((amdgpu_num_vgpr(24))) void spilling_kernel(float *p) {
  float v[48];
#pragma unroll
  for (int i = 0; i < 48; ++i) v[i] = p[i * 64 + threadIdx.x];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 48; ++i) p[i * 64 + (threadIdx.x ^ 1)] = v[47 - i];
}
"""


@pytest.mark.parametrize("spills", [True, False])
def test_the_library_is_not_built_from_a_kernel_that_spills(tmp_path, spills):
    csrc = tmp_path / "graphiler_amd" / "csrc"
    shutil.copytree(CSRC, csrc, ignore=shutil.ignore_patterns("build"))
    shutil.copytree(os.path.join(CSRC, "..", "..", "include"), tmp_path / "include")
    (csrc / "gated_few.hip").write_text(SPILLS if spills else SPILLS.replace("amdgpu_num_vgpr(24)", "amdgpu_num_vgpr(128)"))
    r = subprocess.run(["make", "-C", str(csrc), "build/gated_few.o"], capture_output=True, text=True, timeout=900)
    assert (r.returncode != 0) == spills, r.stderr[-2000:]
    assert (csrc / "build" / "gated_few.o").exists() != spills
    assert ("gated_few.hip: a kernel spills" in r.stderr) == spills
