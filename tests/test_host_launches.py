"""Entry points' host code run without a device: what they launch, recorded (tests/host)."""
import os
import shutil
import subprocess
from pathlib import Path

import pytest

HOST = Path(__file__).resolve().parent / "host"


def _hipcc():
    return next(c for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")) if c and Path(c).exists())


def _run(name, tmp_path):
    """The program's output; its kernels are host stubs, and nothing of the HIP runtime is linked."""
    program = tmp_path / name
    made = subprocess.run([_hipcc(), "--offload-host-only", "--offload-arch=gfx950", "-O1", "-std=c++17", "-w", "-no-hip-rt",
                           "-x", "hip", str(HOST / f"{name}.cpp"), "-o", str(program)], capture_output=True, text=True)
    assert made.returncode == 0, made.stderr[-3000:]
    ran = subprocess.run([str(program)], capture_output=True, text=True, timeout=300)
    assert ran.returncode == 0, ran.stdout[-3000:]
    return ran.stdout


@pytest.mark.parametrize("name", ["lora_order", "norm_rows"])
def test_launches(name, tmp_path):
    print(_run(name, tmp_path))
