"""What once went wrong around the products with 4-bit weights, as far as it needs no GPU."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_a_handle_and_a_models_matrices_have_the_same_limits(tmp_path):
    exe = tmp_path / "w4_weights_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", str(ROOT / "tests" / "cpp" / "w4_weights_test.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


def test_a_thread_that_finds_the_type_table_filled_finds_the_rest(monkeypatch):
    """Calls skip the set-up when the table of element types is filled: everything else has to be there by then."""
    from retrograd_b200 import w4

    class Table(dict):
        def update(self, *args):
            assert w4._raw_stream is not None
            super().update(*args)

    monkeypatch.setattr(w4, "_TYPES", Table())
    monkeypatch.setattr(w4, "_raw_stream", None)
    w4._torch()
    assert len(w4._TYPES) == 3
