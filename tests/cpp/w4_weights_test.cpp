// Which weights the products with 4-bit weights hold: the same answer for a handle and for a model's matrices.
#include "../../retrograd_b200/csrc/w4_checks.hpp"

#include <cstdio>
#include <string>

using namespace rb200;

static int failures = 0;

static void expect(const char * what, const std::string & got, const std::string & want) {
    const bool ok = want.empty() ? got.empty() : got.find(want) != std::string::npos;
    if (!ok) {
        std::printf("%s: got '%s', expected '%s'\n", what, got.c_str(), want.c_str());
        ++failures;
    }
}

int main() {
    using w4::check_weights;
    expect("smallest", check_weights(GGML_Q4_0, 1, 32, 1), "");
    expect("largest row", check_weights(GGML_MXFP4, 7, 262144, 256), "");
    expect("longer row", check_weights(GGML_MXFP4, 7, 262144 + 32, 1), "larger than 262144");
    expect("another type", check_weights(GGML_Q8_0, 1, 32, 1), "must be Q4_0");
    expect("half a block", check_weights(GGML_Q4_0, 1, 48, 1), "multiple of 32");
    expect("no rows", check_weights(GGML_Q4_0, 0, 32, 1), "at least 1");
    expect("no columns", check_weights(GGML_Q4_0, 1, 0, 1), "at least 1");
    expect("no experts", check_weights(GGML_Q4_0, 1, 32, 0), "1 to 256");
    expect("many experts", check_weights(GGML_Q4_0, 1, 32, 257), "1 to 256");
    // 2048 units a row block: 2^20 - 1 of them fit a grid, 2^20 do not
    expect("a grid of units", check_weights(GGML_Q4_0, 32 * 1048575ull, 262144, 1), "");
    expect("more than a grid", check_weights(GGML_Q4_0, 32 * 1048575ull + 1, 262144, 1), "too large");
    expect("more in experts", check_weights(GGML_Q4_0, 32 * 4096ull, 262144, 256), "too large");
    expect("rows of an int", check_weights(GGML_Q4_0, 0x7fffffe0ull, 32, 1), "");
    expect("rows above an int", check_weights(GGML_Q4_0, 0x7fffffe1ull, 32, 1), "too large");
    expect("rows of 64 bits", check_weights(GGML_Q4_0, 1ull << 40, 32, 1), "too large");
    std::printf(failures ? "FAILED\n" : "ok\n");
    return failures != 0;
}
