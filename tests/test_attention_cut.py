"""How attention's work is cut, by the functions that its launches and kernels use (csrc/lt_cut.h), on the CPU."""
import os
import subprocess

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "build", "test_attention_cut")


def test_cut_of_random_batches():
    out = subprocess.run([BIN], capture_output=True, text=True, timeout=120)
    print(out.stdout[-3000:])
    assert out.returncode == 0 and "ALL PASSED" in out.stdout, out.stdout + out.stderr
