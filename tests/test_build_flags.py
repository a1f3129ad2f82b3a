"""What every device compilation of the library has to be given."""

import os
import subprocess

from conftest import PKG_DIR


def test_no_kernel_uses_packed_float32_instructions():
    """Every hipcc line that compiles for the GPU turns them off."""
    plan = subprocess.run(["make", "-n", "-B", "-C", os.path.join(PKG_DIR, "csrc"), "ARCH=gfx950"], check=True,
                          capture_output=True, text=True).stdout.replace("\\\n", " ")
    lines = [line for line in plan.splitlines() if "--offload-arch" in line and " -c " in line]
    sources = {word for line in lines for word in line.split() if word.endswith(".hip")}
    have = {f for f in os.listdir(os.path.join(PKG_DIR, "csrc")) if f.endswith(".hip")}
    assert sources == have
    for line in lines:
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, line
