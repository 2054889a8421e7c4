"""The build's check of the compiler's register remarks."""
from __future__ import annotations

import pytest

from minivllm import _build


def remarks(name, scratch, spill, sgpr=0):
    lines = [f"Function Name: {name}", "    TotalSGPRs: 106", "    VGPRs: 128", "    AGPRs: 0",
             f"    ScratchSize [bytes/lane]: {scratch}", "    Dynamic Stack: False", "    Occupancy [waves/SIMD]: 4",
             f"    SGPRs Spill: {sgpr}", f"    VGPRs Spill: {spill}", "    LDS Size [bytes/block]: 0"]
    return "".join(f"/x/y.h:7:1: remark: {l} [-Rpass-analysis=kernel-resource-usage]\n    7 | void f() {{\n      | ^\n"
                   for l in lines)


def test_spills_are_found():
    text = "In file included from x.hip:2:\n" + remarks("_Za", 0, 0, 47) + remarks("_Zb", 68, 26) + remarks("_Zc", 16, 0)
    assert _build.spills(text) == {"_Zb": 26, "_Zc": 0}
    assert _build.spills("warning: something else\n") == {}
    _build.check_spills("x.hip", remarks("_Za", 0, 0, 47))
    for bad in (remarks("_Zb", 68, 26), remarks("_Zc", 16, 0)):
        with pytest.raises(RuntimeError, match="x.hip: kernel _Z[bc] spills"):
            _build.check_spills("x.hip", remarks("_Za", 0, 0) + bad)
    with pytest.raises(RuntimeError, match="no register counts"):
        _build.spills("x.h:1:1: remark: Function Name: _Zd [-R]\n")


def test_known_spills_are_allowed_as_they_are_alone():
    for part, count in _build.SPILLS.items():
        _build.check_spills("x.hip", remarks(f"_ZN3{part}Lb1E", 24, count))
        with pytest.raises(RuntimeError, match="spills"):
            _build.check_spills("x.hip", remarks(f"_ZN3{part}Lb1E", 28, count + 1))


def test_the_compiler_says_what_a_kernel_spills(tmp_path):
    """A kernel that cannot do without spilling, compiled (not run) as the build compiles."""
    src = tmp_path / "many.hip"
    src.write_text("""#include <hip/hip_runtime.h>
__global__ void __launch_bounds__(1024) many(float* p) {
  float x[200];
#pragma unroll
  for (int i = 0; i < 200; ++i) x[i] = p[i * 1024 + threadIdx.x];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 200; ++i) p[i * 1024 + threadIdx.x] = x[(i * 7) % 200] * x[199 - i];
}
""")
    said = _build._run([_build._hipcc(), *_build.HIP_FLAGS, *_build.REMARKS, "-c", str(src), "-o", str(tmp_path / "many.o")], False)
    (name, count), = _build.spills(said).items()
    assert "many" in name and count > 0
    with pytest.raises(RuntimeError, match="many"):
        _build.check_spills("many.hip", said)
