"""The search for a threshold among many equal candidates that the log probabilities'
best ids go by (csrc/kth_key.h), compiled for the host from the header that the kernel
includes (tests/c/kth_key.cpp): rows with ties of every extent, at zero and at powers of
two among them."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_thresholds(tmp_path):
    exe = str(tmp_path / "kth_key")
    rocm = os.environ.get("ROCM", "/opt/rocm")
    r = subprocess.run([rocm + "/llvm/bin/clang++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-o", exe,
                        os.path.join(ROOT, "tests", "c", "kth_key.cpp")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    print(r.stdout)
    rows, wrong = (int(x) for x in r.stdout.split("\n")[-2].replace(",", "").split()[::2])
    assert r.returncode == 0 and wrong == 0 and rows > 10000, r.stdout
