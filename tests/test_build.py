"""The build: objects follow the flags that they were compiled with."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "myria3d_amd", "csrc")


@pytest.mark.skipif(not shutil.which("make"), reason="needs make")
def test_every_object_is_built_again_when_the_flags_change():
    """(-W: as if the file had just been written; -n: nothing is run)"""
    out = subprocess.run(["make", "-C", CSRC, "-n", "-W", "Makefile"], check=True, capture_output=True, text=True).stdout
    compiled = {line.split(" -c ")[1].split()[0] for line in out.splitlines() if " -c " in line}
    assert compiled == {f for f in os.listdir(CSRC) if f.endswith(".hip")}
    assert all("-packed-fp32-ops" in line for line in out.splitlines() if " -c " in line)
