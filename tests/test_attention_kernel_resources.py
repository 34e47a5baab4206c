"""The attention operators' kernels at build time (no GPU needed: hipcc cross-compiles gfx950): no private arrays or spills in
scratch memory, the workgroups a CU that their launch bounds count on, and no packed fp32 instructions."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mint_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def _flags():
    """What build.sh compiles with."""
    text = open(os.path.join(CSRC, "build.sh")).read()
    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in text
    return ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


@pytest.mark.parametrize("unit,kernels", [("rel_attention", 45), ("qk_norm", 13)])
def test_kernels_keep_to_registers(unit, kernels, tmp_path):
    if not shutil.which(HIPCC) and not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    out = subprocess.run([HIPCC] + _flags() + ["-Rpass-analysis=kernel-resource-usage", "--save-temps=obj", "-c",
                                               os.path.join(CSRC, unit + ".hip"), "-o", str(tmp_path / (unit + ".o"))],
                         capture_output=True, text=True, timeout=900)
    assert out.returncode == 0, out.stderr[-3000:]
    use, name = {}, None
    for line in out.stderr.splitlines():
        m = re.search(r"Function Name: (\S+)", line)
        if m:
            name = m.group(1)
            use[name] = {}
        m = re.search(r"(VGPRs Spill|VGPRs|ScratchSize \[bytes/lane\]): (\d+)", line)
        if m and name:
            use[name].setdefault(m.group(1), int(m.group(2)))
    assert len(use) >= kernels, sorted(use)
    for n, u in use.items():
        assert u["ScratchSize [bytes/lane]"] == 0 and u["VGPRs Spill"] == 0, (n, u)
        m = re.search(r"rel_(dkdv|dq|fwd)_kernelILi(\d+)E", n)
        if m:
            slots = 4 if m.group(1) == "fwd" or int(m.group(2)) <= 96 else 3
            assert u["VGPRs"] <= 512 // slots // 8 * 8, (n, u)
    asm = [f for f in os.listdir(tmp_path) if f.endswith("gfx950.s")]
    assert asm and not re.search(r"v_pk_(add|mul|fma)_f32", (tmp_path / asm[0]).read_text())
