"""Q4_0 storage and the refusals of the products with 4-bit weights, without a GPU."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_every_refusal_of_the_products_is_decided_on_the_host(tmp_path):
    exe = tmp_path / "w4_checks_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", str(ROOT / "tests" / "cpp" / "w4_checks_test.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


@pytest.mark.parametrize("args,message", [
    ((8, 1, 64, 64, 1), b"the weights must be Q4_0 (2) or MXFP4 (39)"),
    ((2, 0, 64, 64, 1), b"rows are required"),
    ((2, 1, 0, 64, 1), b"n_in a multiple of 32"),
    ((2, 1, 64, 0, 1), b"n_in a multiple of 32"),
    ((39, 1, 64, 48, 1), b"n_in a multiple of 32"),
    ((2, 1, 64, 262144 + 32, 1), b"larger than 262144"),
    ((2, 1, 64, 64, 0), b"n_expert must be 1 to 256"),
    ((2, 1, 64, 64, 257), b"n_expert must be 1 to 256"),
    ((2, 1, 0xFFFFFFFF, 262144, 256), b"the bank is too large"),
])
def test_a_weight_handle_is_refused_before_anything_is_read(rb, args, message):
    lib = rb.load_library()
    kind, rows, n_out, n_in, n_expert = args
    assert not lib.retro_b200_w4_new(kind, 4096 if rows else None, n_out, n_in, n_expert)
    assert lib.retro_last_error().startswith(b"w4_new: ") and message in lib.retro_last_error()


def test_calls_without_a_handle_are_refused(rb):
    lib = rb.load_library()
    assert lib.retro_b200_w4_matvec(None, 4096, 0, 32, 1, None, 0.0, None, None, 0, 8192, 0, 32, None) == -3
    assert lib.retro_last_error() == b"w4_matvec: a weight handle is required"
    assert lib.retro_b200_w4_glu(None, None, 4096, 0, 32, 1, None, 0.0, 8192, 0, 32, None) == -3
    assert lib.retro_b200_w4_moe(4096, None, None, None, 4096, 0, 32, 1, 1, 0, None, 0.0, None, 0, 8192, 0, 32, None, None, 4096, 4096, None) == -3
    assert lib.retro_last_error() == b"w4_moe: a weight handle is required"
    n = C.c_size_t()
    assert lib.retro_b200_w4_moe_workspace(None, 1, 1, C.byref(n)) == -3
    assert lib.retro_b200_w4_info(None, None, None, None, None) == -3
    lib.retro_b200_w4_free(None)


def test_the_handle_checks_the_bytes_it_is_given(rb):
    with pytest.raises(rb.InvalidArgument, match="rows hold 17 bytes, the shape needs 18"):
        rb.W4Matrix(2, bytes(17), 1, 32)
    with pytest.raises(rb.InvalidArgument, match="rows hold 18 bytes, the shape needs 17"):
        rb.W4Matrix(39, bytes(18), 1, 32)
    with pytest.raises(rb.InvalidArgument, match="a size is negative"):
        rb.W4Matrix(2, bytes(18), -1, 32)
    with pytest.raises(rb.InvalidArgument, match="must be Q4_0"):
        rb.W4Matrix(12, bytes(144), 1, 256)


def test_q4_0_rows_are_the_published_quantiser_and_decode_like_gguf_py(rb, oracle):
    gguf = pytest.importorskip("gguf")
    rng = np.random.default_rng(4)
    x = (rng.normal(0, 0.02, 32 * 400) * np.repeat(np.exp2(rng.uniform(-6, 6, 400)), 32)).astype(np.float32)
    x[32 * 7:32 * 8] = 0
    raw = np.frombuffer(rb.quantize_row(2, x), dtype=np.uint8)
    want = gguf.quants.quantize(x.reshape(1, -1), gguf.GGMLQuantizationType.Q4_0).reshape(-1)
    assert np.array_equal(raw, want)
    decoded = gguf.quants.dequantize(want.reshape(-1, 18), gguf.GGMLQuantizationType.Q4_0).reshape(-1).astype(np.float32)
    assert np.array_equal(oracle.dequantize_row(oracle.T_Q4_0, raw, x.size), decoded)
