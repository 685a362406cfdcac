// Products with 4-bit weights and group scales for few tokens: the device layout of the weights and the launch
// wrappers of w4.cu. Two stored formats, both with one scale per 32 columns: Q4_0 (w = d (q - 8), d an f16) and
// MXFP4 (w = 2^(s - 127) e2m1(q), s a byte).
#pragma once

#include "w4_checks.hpp"

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace rb200 {

constexpr int kW4PassTokens = 16;            // tokens one launch serves; longer calls run pass by pass
constexpr uint32_t kW4MaxUsed = 32;          // experts per token
constexpr uint32_t kW4MaxScaleByte = 207;    // MXFP4: weight scales up to 2^80, so that a row's scaled sum stays inside f32

// Device layout: units of 32 rows x 128 columns, a row block's units consecutive over the columns, row blocks consecutive,
// experts consecutive. A unit is, for each 64-column half and 16-row tile, 32 x 16 bytes, one 16-byte word per lane of the warp that
// multiplies it (the lane's share of the A fragments of four m16n8k16 products), then for each tile the 16 rows' four
// scales: 128 bytes of f16 or 64 bytes. Rows and columns beyond the matrix have scale zero. The bit order inside a word is described at
// w4_retile_kernel.
__host__ __device__ constexpr uint32_t w4_unit_bytes(bool mxfp4) { return mxfp4 ? 2176u : 2304u; }

struct W4View {
    const uint8_t * units = nullptr;
    uint32_t type = 0;              // GGML_Q4_0 or GGML_MXFP4
    uint32_t n_out = 0, n_in = 0;
    uint32_t n_expert = 1;
    uint32_t blocks = 0;            // 32-row blocks of one expert
    uint32_t steps = 0;             // 128-column steps
    size_t expert_bytes = 0;
};

size_t w4_bytes(uint32_t type, uint32_t n_out, uint32_t n_in, uint32_t n_expert);
// Lays GGUF rows [expert][row][blocks] (device memory) out as units. *max_scale (device, zeroed by the caller) becomes the
// largest MXFP4 scale byte; untouched for Q4_0. For shapes that w4::check_weights admits.
cudaError_t launch_w4_retile(const uint8_t * rows, uint32_t type, uint32_t n_out, uint32_t n_in, uint32_t n_expert, uint8_t * units, int * max_scale,
                             cudaStream_t stream);
W4View w4_view(const uint8_t * units, uint32_t type, uint32_t n_out, uint32_t n_in, uint32_t n_expert);

// Activations: f32, f16 or bf16 rows (GGML type codes); results: the same choice.
struct W4Product {
    W4View w;                       // the matrix; with `up`, the gate matrix
    const W4View * up = nullptr;    // y = silu(w x) * (up x)
    const void * x = nullptr;
    uint32_t x_type = 0;
    int64_t ld_x = 0;
    int n_tokens = 0;
    const float * norm = nullptr;   // RMSNorm weights: x is normalised first
    float eps = 0.f;
    const float * bias = nullptr;
    const void * residual = nullptr;    // of y's type; may be y itself
    int64_t ld_residual = 0;
    void * y = nullptr;
    uint32_t y_type = 0;
    int64_t ld_y = 0;
};
cudaError_t launch_w4_product(const W4Product & p, cudaStream_t stream);

struct W4Moe {
    W4View gate, up, down;
    const float * router = nullptr;     // [n_expert][n_in]
    const void * x = nullptr;
    uint32_t x_type = 0;
    int64_t ld_x = 0;
    int n_tokens = 0;
    int n_used = 0;
    bool normalise = false;             // divide the chosen probabilities by their sum
    const float * norm = nullptr;
    float eps = 0.f;
    const void * residual = nullptr;
    int64_t ld_residual = 0;
    void * y = nullptr;
    uint32_t y_type = 0;
    int64_t ld_y = 0;
    int32_t * ids = nullptr;            // [n_tokens][n_used], optional: the chosen experts, likeliest first
    float * weights = nullptr;          // [n_tokens][n_used], optional: their weights
    void * workspace = nullptr;
};
size_t w4_moe_workspace_bytes(uint32_t ff, uint32_t n_tokens, uint32_t n_used);
cudaError_t launch_w4_moe(const W4Moe & p, cudaStream_t stream);

} // namespace rb200
