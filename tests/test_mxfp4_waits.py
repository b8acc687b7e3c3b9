"""The few-token kernels of MXFP4 products whose activations are unaligned wait by hand as the others do, in a compilation of their own: nothing may
touch a register before the wait that releases it.  (The kernels of aligned rows and the tiles: test_norm_host.py.)"""
import os
import subprocess

import isa_wait_lint


def test_kernels_of_unaligned_activations(tmp_path):
    from frink_amd import build as fb
    out = tmp_path / "kernels.s"
    r = subprocess.run([fb.hipcc()] + fb.HIPCC_FLAGS + ["-x", "hip", "--cuda-device-only", "-S", os.path.join(fb.CSRC, "frk_mx4.hip"), "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    asm = out.read_text()
    kernels = [k for k in isa_wait_lint.kernels(asm) if "mx4_rows_kernel" in k and "ELb1ELb0E" in k]
    assert len(kernels) == 4, kernels  # (eight wavefronts of one, two and four strips, sixteen of one)
    for k in kernels:
        assert isa_wait_lint.violations(asm, k) == [], k
