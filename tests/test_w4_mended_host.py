"""What once went wrong around the products with 4-bit weights, as far as it needs no GPU."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_a_handle_and_a_models_matrices_have_the_same_limits(tmp_path):
    exe = tmp_path / "w4_weights_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", str(ROOT / "tests" / "cpp" / "w4_weights_test.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
