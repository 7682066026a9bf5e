"""What the compiler says of kernels whose registers are close to full: no scratch."""
import os
import re
import shutil
import subprocess

import pytest

from auto_infer_amd.csrc import build


@pytest.mark.parametrize("source", ["kv_write_fp8.hip", "rope_append.hip"])
def test_cache_writes_spill_nothing(source, tmp_path):
    if not (os.path.exists(build.hipcc()) or shutil.which(build.hipcc())):
        pytest.skip("no hipcc")
    flags = [f for f in build.HIPCC_FLAGS if f != "-shared"]
    asm = tmp_path / "device.s"
    subprocess.run([build.hipcc(), *flags, "-I", os.path.join(build.ROOT, "include"), "-I", build.HERE, "--cuda-device-only",
                    "-S", os.path.join(build.HERE, source), "-o", str(asm)], check=True, capture_output=True, timeout=300)
    kernels = re.findall(r"\.name: +(_Z\S+)\n(?:.*\n)*?\s+\.private_segment_fixed_size: (\d+)\n(?:.*\n)*?\s+\.vgpr_spill_count: (\d+)",
                         asm.read_text())
    assert len(kernels) >= 12
    assert [k for k in kernels if k[1:] != ("0", "0")] == []
