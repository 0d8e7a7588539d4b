"""The kernels' headers in one translation unit: they are linked into one library, so a name must be one thing in all of them.
No GPU needed."""
import glob
import os
import subprocess

from dfssm import build


def test_all_headers_together(tmp_path):
    headers = sorted(os.path.basename(p) for p in glob.glob(os.path.join(build.CSRC, "*.h")))
    assert "layer.h" in headers and "dfssm_kernels.h" in headers
    src = tmp_path / "all.hip"
    src.write_text("".join(f'#include "{h}"\n' for h in headers))
    r = subprocess.run([build.HIPCC, *build.FLAGS, "--cuda-host-only", "-fsyntax-only", str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
