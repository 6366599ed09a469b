"""What the compiler says of the layer norm kernels, without a GPU."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.mark.skipif(not (os.path.exists(HIPCC) or shutil.which("hipcc")), reason="needs hipcc (cross-compiles without a GPU)")
def test_no_layer_norm_kernel_goes_to_scratch_memory():
    """A row, its weights' gradients and the sums stay in registers, in every layout and type."""
    src = os.path.join(ROOT, "myria3d_amd", "csrc", "norm.hip")
    flags = re.search(r"^CXXFLAGS = (.*)$", open(os.path.join(os.path.dirname(src), "Makefile")).read(), re.M).group(1)
    text = subprocess.run([HIPCC, *flags.replace("$(ARCH)", "gfx950").split(), "-w", "--cuda-device-only", "-S", src, "-o", "-"], check=True,
                          capture_output=True, text=True, cwd=os.path.dirname(src)).stdout
    sizes = {m.group(1): (int(m.group(2)), int(m.group(3)))
             for m in re.finditer(r"\.name:\s+(_Z\w*layer_norm\w*).*?\.private_segment_fixed_size:\s+(\d+).*?\.vgpr_spill_count:\s+(\d+)", text, re.S)}
    assert sum("bwd" in name for name in sizes) > 60 and len(sizes) > 100
    assert not {name: s for name, s in sizes.items() if s != (0, 0)}
