"""aegis_torch where the 8-bit libraries were not built, or cannot be loaded."""
import os
import shutil
import subprocess
import sys

import pytest

from conftest import ROOT


@pytest.mark.parametrize("left", ["none", "broken"])
def test_matmul_without_the_8_bit_libraries(tmp_path, left):
    """matmul needs libaegis_capi.so alone; calls of the 8-bit operators then name what is missing."""
    pkg = tmp_path / "aegis-core_b200"
    (pkg / "build").mkdir(parents=True)
    src = os.path.join(ROOT, "aegis-core_b200")
    for f in os.listdir(src):
        if f.endswith(".py"):
            shutil.copy(os.path.join(src, f), pkg)
    os.symlink(os.path.join(src, "build", "libaegis_capi.so"), pkg / "build" / "libaegis_capi.so")
    if left == "broken":
        (pkg / "build" / "libaegis_torch_i8.so").write_bytes(b"not a library")
    code = """
import torch, aegis_torch
m = torch.empty(4, 8, dtype=torch.float16, device="meta")
assert torch.ops.aegis.matmul(m, m.t()).shape == (4, 4)
assert torch.ops.aegis.silu_mul_i8(m, m)[0].shape == (4, 8)
try:
    torch.ops.aegis.silu_mul_i8.default._op_dk(torch._C.DispatchKey.CUDA, m, m)
except RuntimeError as e:
    print(e)
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                       env={**os.environ, "PYTHONPATH": str(pkg)}, cwd=tmp_path)
    assert r.returncode == 0, r.stderr
    assert "aegis::silu_mul_i8" in r.stdout and "libaegis_torch_i8.so" in r.stdout
    assert ("not built" if left == "none" else "cannot be loaded") in r.stdout
