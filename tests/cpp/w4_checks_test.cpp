// The refusals of the products with 4-bit weights: every one is decided on the host, from the arguments alone.
#include "../../retrograd_b200/csrc/w4_checks.hpp"

#include <cstdio>
#include <string>

using namespace rb200;
using namespace rb200::w4;

static int failures = 0;

static void expect(const char * what, const std::string & got, const std::string & want) {
    const bool ok = want.empty() ? got.empty() : got.find(want) != std::string::npos;
    if (!ok) {
        std::printf("%s: got '%s', expected '%s'\n", what, got.c_str(), want.c_str());
        ++failures;
    }
}

static const void * at(uintptr_t p) { return reinterpret_cast<const void *>(p); }

int main() {
    const ProductShape shape{3, 64, 32};
    const uintptr_t X = 0x100000, Y = 0x200000, R = 0x300000;
    const Rows none{"residual", nullptr, GGML_F32, 0};
    auto x = [&](uintptr_t p, uint32_t type = GGML_F32, int64_t ld = 64) { return Rows{"x", at(p), type, ld}; };
    auto y = [&](uintptr_t p, uint32_t type = GGML_F32, int64_t ld = 32) { return Rows{"y", at(p), type, ld}; };
    auto r = [&](uintptr_t p, uint32_t type = GGML_F32, int64_t ld = 32) { return Rows{"residual", at(p), type, ld}; };
    auto product = [&](const Rows & a, const Rows & b, const Rows & c, const float * norm = nullptr, float eps = 1e-5f, const float * bias = nullptr) {
        return check_product(shape, a, b, c, norm, eps, bias);
    };
    auto vec = [&](uintptr_t p) { return reinterpret_cast<const float *>(p); };

    expect("plain", product(x(X), y(Y), none), "");
    expect("no x", product(x(0), y(Y), none), "x is required");
    expect("no y", product(x(X), y(0), none), "y is required");
    expect("type", product(x(X, GGML_Q8_0), y(Y), none), "x must be f32");
    expect("y type", product(x(X), y(Y, 7), none), "y must be f32");
    expect("x alignment", product(x(X + 2), y(Y), none), "x must be aligned");
    expect("half alignment", product(x(X + 2, GGML_F16), y(Y), none), "");
    expect("odd half", product(x(X + 1, GGML_BF16), y(Y), none), "x must be aligned");
    expect("repeated row", product(x(X, GGML_F32, 0), y(Y), none), "");
    expect("narrow x rows", product(x(X, GGML_F32, 5), y(Y), none), "");
    expect("negative stride", product(x(X, GGML_F32, -64), y(Y), none), "negative");
    expect("huge stride", product(x(X, GGML_F32, (int64_t)1 << 40), y(Y), none), "too large");
    expect("narrow y rows", product(x(X), y(Y, GGML_F32, 31), none), "smaller than a row");
    expect("one y row", check_product({1, 64, 32}, x(X), y(Y, GGML_F32, 0), none, nullptr, 0.f, nullptr), "");
    expect("eps", product(x(X), y(Y), none, vec(R), -1.f), "eps");
    expect("eps nan", product(x(X), y(Y), none, vec(R), __builtin_nanf("")), "eps");
    expect("eps without norm", product(x(X), y(Y), none, nullptr, -1.f), "");
    expect("norm alignment", product(x(X), y(Y), none, vec(R + 2)), "norm must be 4-byte aligned");
    expect("bias alignment", product(x(X), y(Y), none, nullptr, 0.f, vec(R + 1)), "bias must be 4-byte aligned");
    expect("y on x", product(x(X), y(X), none), "y overlaps x");
    expect("y in x's last row", product(x(X), y(X + 3 * 256 - 4), none), "y overlaps x");
    expect("y behind x", product(x(X), y(X + 3 * 256), none), "");
    expect("columns of one buffer", product(x(X, GGML_F32, 96), y(X + 256, GGML_F32, 96), none), "");
    expect("columns that meet", product(x(X, GGML_F32, 96), y(X + 252, GGML_F32, 96), none), "y overlaps x");
    expect("columns, y in front", product(x(X + 128, GGML_F32, 96), y(X, GGML_F32, 96), none), "");
    expect("y on norm", product(x(X), y(Y), none, vec(Y + 8)), "y overlaps norm");
    expect("y on bias", product(x(X), y(Y), none, nullptr, 0.f, vec(Y + 3 * 128 - 4)), "y overlaps norm or bias");
    expect("residual", product(x(X), y(Y), r(R)), "");
    expect("in place", product(x(X), y(Y), r(Y)), "");
    expect("in place, other stride", product(x(X), y(Y), r(Y, GGML_F32, 64)), "without being it");
    expect("residual shifted", product(x(X), y(Y), r(Y + 4)), "without being it");
    expect("too many tokens", check_product({kMaxTokens + 1, 64, 32}, x(X), y(Y), none, nullptr, 0.f, nullptr), "too many");

    const MoeShape moe{3, 8, 2, 64, 32};
    const Rows my{"y", at(Y), GGML_F32, 64}, mx{"x", at(X), GGML_F32, 64};
    auto layer = [&](const Rows & a, const Rows & b, const Rows & c, MoeBuffers m) { return check_moe(moe, a, b, c, nullptr, 0.f, m); };
    const MoeBuffers good{vec(0x400000), nullptr, nullptr, (void *)at(0x500000), 4096, 4000};
    MoeBuffers m = good;
    expect("layer", layer(mx, my, none, m), "");
    expect("in place", layer(mx, Rows{"y", at(X), GGML_F32, 64}, none, m), "");
    expect("in place, shifted", layer(mx, Rows{"y", at(X + 4), GGML_F32, 64}, none, m), "without being it");
    expect("in place, type", layer(mx, Rows{"y", at(X), GGML_F16, 64}, none, m), "without being it");
    m.router = nullptr;
    expect("router", layer(mx, my, none, m), "router is required");
    m = good; m.router = vec(0x400002);
    expect("router alignment", layer(mx, my, none, m), "router must be 4-byte aligned");
    m = good; m.router = vec(Y);
    expect("y on router", layer(mx, my, none, m), "y overlaps norm or router");
    m = good; m.workspace_bytes = 3999;
    expect("small workspace", layer(mx, my, none, m), "the workspace needs 4000 bytes");
    m = good; m.workspace = nullptr;
    expect("no workspace", layer(mx, my, none, m), "the workspace needs");
    m = good; m.workspace = (void *)at(0x500008);
    expect("workspace alignment", layer(mx, my, none, m), "16-byte aligned");
    m = good; m.workspace = (void *)at(X + 512);
    expect("workspace on x", layer(mx, my, none, m), "overlap");
    m = good; m.ids = (int32_t *)at(0x500000 + 3996);
    expect("ids in the workspace", layer(mx, my, none, m), "overlap");
    m = good; m.ids = (int32_t *)at(0x500000 + 4000);
    expect("ids behind the workspace", layer(mx, my, none, m), "");
    m = good; m.ids = (int32_t *)at(Y + 4); m.weights = (float *)at(0x600000);
    expect("ids on y", layer(mx, my, none, m), "overlap");
    m = good; m.ids = (int32_t *)at(0x600000); m.weights = (float *)at(0x600000 + 20);
    expect("ids on weights", layer(mx, my, none, m), "overlap");
    m = good; m.weights = (float *)at(0x400000 + 4);
    expect("weights on router", layer(mx, my, none, m), "overlap");
    std::printf(failures ? "FAILED\n" : "ok\n");
    return failures != 0;
}
