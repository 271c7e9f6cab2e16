"""The compiler's register report, for kernels that must not send registers to memory: a read back from there waits for every
request that the wave has in flight."""
import importlib.util
import re
import shutil
import subprocess
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parents[1] / "kernel-rsi_amd"


def scratch_and_waves(source):
    """{mangled kernel name: (bytes of scratch a lane, waves per SIMD)} of one kernel source, compiled as the library is."""
    spec = importlib.util.spec_from_file_location("krsi_build", PKG / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    cmd = [build._hipcc(), *build.HIP_FLAGS, *build.EXTRA_FLAGS.get(source, []), f"-I{build.INCLUDE}",
           f"-I{build.CSRC}", "-Rpass-analysis=kernel-resource-usage", "--offload-device-only", "-c",
           str(build.CSRC / source), "-o", "/dev/null"]
    report = subprocess.run(cmd, capture_output=True, text=True, check=True).stderr
    return {m[1]: (int(m[2]), int(m[3])) for m in
            re.finditer(r"Function Name: (\S+).*?ScratchSize[^:]*: (\d+).*?Occupancy[^:]*: (\d+)", report, re.S)}


@pytest.mark.skipif(not (Path("/opt/rocm/bin/hipcc").is_file() or shutil.which("hipcc")), reason="no hipcc")
@pytest.mark.parametrize("source,kernels", [("linear_8bit.hip", "linear_8bit_"), ("adamw.hip", "step"),
                                            ("add_rmsnorm.hip", "row_pass")])
def test_no_scratch(source, kernels):
    found = {k: v for k, v in scratch_and_waves(source).items() if kernels in k}
    assert found and not {k: v for k, v in found.items() if v[0]}


@pytest.mark.skipif(not (Path("/opt/rocm/bin/hipcc").is_file() or shutil.which("hipcc")), reason="no hipcc")
def test_two_waves_per_simd_of_the_large_tiles():
    """256 x 256 tiles by eight waves, which all of a CU's SIMDs have to hold two at a time."""
    found = scratch_and_waves("linear_8bit.hip")
    large = [v for k, v in found.items() if "linear_8bit_streamILi" in k and "ELi2ELi4ELi8ELi4ELi3ELi2E" in k]
    assert len(large) == 3 and all(waves >= 2 for _, waves in large)


@pytest.mark.skipif(not (Path("/opt/rocm/bin/hipcc").is_file() or shutil.which("hipcc")), reason="no hipcc")
def test_no_scratch_in_the_norms_backward():
    """Every width, with and without the stream's gradient, aligned and ragged: 6 widths in 16 bits and 7 in fp32."""
    found = {k: v[0] for k, v in scratch_and_waves("add_rmsnorm.hip").items() if "add_rms_bwd" in k}
    assert len([k for k in found if "short" not in k]) == (6 + 6 + 7) * 4
    assert not {k: v for k, v in found.items() if v}
