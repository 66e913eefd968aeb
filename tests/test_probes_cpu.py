"""The stand-alone hardware probes compile for gfx950 with the flags of their build script."""
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-I", "pytorch_distributed_amd/csrc/kernels", "-I", "pytorch_distributed_amd/csrc"]


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="no hipcc")
def test_probes_compile(tmp_path):
    probes = sorted((ROOT / "tools" / "micro").glob("*.hip"))
    assert len(probes) >= 9

    def compile_one(src):
        out = tmp_path / (src.stem + ".s")
        run = subprocess.run(["hipcc", *FLAGS, "--cuda-device-only", "-S", str(src), "-o", str(out)], cwd=ROOT, capture_output=True, text=True)
        return src.name, run.returncode, run.stderr[-2000:], out.read_text() if out.exists() else ""

    with ThreadPoolExecutor(4) as pool:
        for name, code, err, text in pool.map(compile_one, probes):
            assert code == 0, f"{name}: {err}"
            assert "v_pk_mul_f32" not in text and "v_pk_add_f32" not in text and "v_pk_fma_f32" not in text, name
