"""How the library is compiled and imported: no GPU and no compiler run needed."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_source_is_compiled_with_packed_float32():
    lines = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "interflow_amd", "csrc")], check=True, capture_output=True, text=True).stdout.splitlines()
    compiles = [line for line in lines if " -c " in line]
    sources = [f for f in os.listdir(os.path.join(ROOT, "interflow_amd", "csrc")) if f.endswith(".hip")]
    assert len(compiles) == len(sources)
    for line in compiles:
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, line


def test_imports_without_a_gpu_build_of_torch():
    code = ("import torch\n"
            "del torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice\n"
            "import interflow_amd\n"
            "from interflow_amd import train_flow, train_ops\n"
            "interflow_amd.InterpFlow([2, 4])\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
