// C entry points of the products with 4-bit weights (include/retro_b200.h, "products with 4-bit weights"): argument checks,
// the weight handle, and the switch to the handle's device. The kernels are in w4.cu.

#include "common.hpp"
#include "blocks.hpp"
#include "kernels.cuh"
#include "w4.cuh"
#include "w4_checks.hpp"

#include "../../include/retro_b200.h"

#include <memory>

using namespace rb200;

struct retro_b200_w4 {
    W4View view;
    int device = 0;
    uint8_t * units = nullptr;
    size_t bytes = 0;
    ~retro_b200_w4() { if (units) cudaFree(units); }
};

namespace {

// Makes `device` current for the call and puts the caller's back.
class DeviceScope {
public:
    explicit DeviceScope(int device) {
        RB_CUDA(cudaGetDevice(&before_));
        if (before_ != device) {
            RB_CUDA(cudaSetDevice(device));
            switched_ = true;
        }
    }
    ~DeviceScope() { if (switched_) cudaSetDevice(before_); }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope & operator=(const DeviceScope &) = delete;

private:
    int before_ = 0;
    bool switched_ = false;
};

int refuse(const char * op, const std::string & why) {
    set_error(std::string(op) + ": " + why);
    return STATUS_INVALID_ARGUMENT;
}

int launched(const char * op, cudaError_t status) {
    if (status == cudaSuccess) return STATUS_OK;
    cudaGetLastError();         // this call's own failure; one that the thread holds from elsewhere is no business of a launch that succeeded
    set_error(std::string(op) + ": launch failed: " + cudaGetErrorString(status));
    return STATUS_RUNTIME;
}

int product(const char * op, const retro_b200_w4 * w, const retro_b200_w4 * up, const void * d_x, uint32_t x_type, int64_t ld_x, uint32_t n_tokens,
            const float * d_norm, float eps, const float * d_bias, const void * d_residual, int64_t ld_residual, void * d_y, uint32_t y_type, int64_t ld_y,
            void * stream) {
    return boundary([&]() -> int {
        if (!w) return refuse(op, "a weight handle is required");
        if (w->view.n_expert != 1) return refuse(op, "the handle holds a bank of experts");
        if (up) {
            if (up->view.n_expert != 1) return refuse(op, "the handle holds a bank of experts");
            if (up->view.type != w->view.type || up->view.n_out != w->view.n_out || up->view.n_in != w->view.n_in)
                return refuse(op, "gate and up must have one type and shape");
            if (up->device != w->device) return refuse(op, "gate and up are on different devices");
        }
        const w4::ProductShape shape{n_tokens, w->view.n_in, w->view.n_out};
        const w4::Rows x{"x", d_x, x_type, ld_x}, y{"y", d_y, y_type, ld_y}, residual{"residual", d_residual, y_type, ld_residual};
        const std::string why = w4::check_product(shape, x, y, residual, d_norm, eps, d_bias);
        if (!why.empty()) return refuse(op, why);
        if (n_tokens == 0) return STATUS_OK;
        const DeviceScope scope(w->device);
        W4Product p;
        p.w = w->view;
        p.up = up ? &up->view : nullptr;
        p.x = d_x;
        p.x_type = x_type;
        p.ld_x = ld_x;
        p.n_tokens = (int)n_tokens;
        p.norm = d_norm;
        p.eps = eps;
        p.bias = d_bias;
        p.residual = d_residual;
        p.ld_residual = ld_residual;
        p.y = d_y;
        p.y_type = y_type;
        p.ld_y = ld_y;
        return launched(op, launch_w4_product(p, static_cast<cudaStream_t>(stream)));
    });
}

} // namespace

extern "C" {

retro_b200_w4 * retro_b200_w4_new(uint32_t ggml_type, const void * rows, uint32_t n_out, uint32_t n_in, uint32_t n_expert) {
    retro_b200_w4 * made = nullptr;
    boundary([&]() -> int {
        const char * op = "w4_new";
        if (!rows) return refuse(op, "rows are required");
        const std::string why = w4::check_weights(ggml_type, n_out, n_in, n_expert);
        if (!why.empty()) return refuse(op, why);
        auto w = std::make_unique<retro_b200_w4>();
        RB_CUDA(cudaGetDevice(&w->device));
        w->bytes = w4_bytes(ggml_type, n_out, n_in, n_expert);
        RB_CUDA(cudaMalloc(&w->units, w->bytes + sizeof(int)));
        w->view = w4_view(w->units, ggml_type, n_out, n_in, n_expert);
        int * d_max = reinterpret_cast<int *>(w->units + w->bytes);     // the largest scale byte, behind the units
        struct Raw { uint8_t * p = nullptr; ~Raw() { if (p) cudaFree(p); } } raw;
        const cudaStream_t stream = cudaStreamPerThread;        // (making one and taking it down is 0.09 ms)
        // Rows that are in this device's memory are read where they are, others are copied there first. (128256 x 4096, Q4_0, rows on
        // the device: 1.0 ms the call, 0.42 ms of it the layout kernel, 0.35 ms the allocation; 1.9 ms with a copy of them. The same rows on the host: 29 ms.)
        const size_t n_raw = (size_t)n_expert * n_out * (n_in / 32) * (ggml_type == GGML_Q4_0 ? 18 : 17);
        cudaPointerAttributes from{};
        RB_CUDA(cudaPointerGetAttributes(&from, rows));
        const uint8_t * d_rows = static_cast<const uint8_t *>(rows);
        RB_CUDA(cudaDeviceSynchronize());       // rows that some stream is still writing
        if (from.type != cudaMemoryTypeDevice || from.device != w->device) {
            RB_CUDA(cudaMalloc(&raw.p, n_raw));
            RB_CUDA(cudaMemcpyAsync(raw.p, rows, n_raw, cudaMemcpyDefault, stream));
            d_rows = raw.p;
        }
        RB_CUDA(cudaMemsetAsync(d_max, 0, sizeof(int), stream));
        RB_CUDA(launch_w4_retile(d_rows, ggml_type, n_out, n_in, n_expert, w->units, d_max, stream));
        int h_max = 0;
        RB_CUDA(cudaMemcpyAsync(&h_max, d_max, sizeof h_max, cudaMemcpyDeviceToHost, stream));
        RB_CUDA(cudaStreamSynchronize(stream));
        if (h_max > (int)kW4MaxScaleByte) return refuse(op, "an MXFP4 scale byte is above 207 (2^80)");
        made = w.release();
        return STATUS_OK;
    });
    return made;
}

void retro_b200_w4_free(retro_b200_w4 * w) {
    if (!w) return;
    boundary([&]() -> int {
        std::unique_ptr<retro_b200_w4> owned(w);
        const DeviceScope scope(w->device);
        owned.reset();
        return STATUS_OK;
    });
}

int retro_b200_w4_info(const retro_b200_w4 * w, uint32_t * out_type, uint32_t * out_shape_3, uint64_t * out_bytes, int * out_device) {
    return boundary([&]() -> int {
        if (!w) return refuse("w4_info", "a weight handle is required");
        if (out_type) *out_type = w->view.type;
        if (out_shape_3) {
            out_shape_3[0] = w->view.n_expert;
            out_shape_3[1] = w->view.n_out;
            out_shape_3[2] = w->view.n_in;
        }
        if (out_bytes) *out_bytes = w->bytes;
        if (out_device) *out_device = w->device;
        return STATUS_OK;
    });
}

int retro_b200_w4_matvec(const retro_b200_w4 * w, const void * d_x, uint32_t x_type, int64_t ld_x, uint32_t n_tokens, const float * d_norm, float eps,
                         const float * d_bias, const void * d_residual, int64_t ld_residual, void * d_y, uint32_t y_type, int64_t ld_y, void * stream) {
    return product("w4_matvec", w, nullptr, d_x, x_type, ld_x, n_tokens, d_norm, eps, d_bias, d_residual, ld_residual, d_y, y_type, ld_y, stream);
}

int retro_b200_w4_glu(const retro_b200_w4 * gate, const retro_b200_w4 * up, const void * d_x, uint32_t x_type, int64_t ld_x, uint32_t n_tokens,
                      const float * d_norm, float eps, void * d_y, uint32_t y_type, int64_t ld_y, void * stream) {
    if (!up) return boundary([&]() -> int { return refuse("w4_glu", "a weight handle is required"); });
    return product("w4_glu", gate, up, d_x, x_type, ld_x, n_tokens, d_norm, eps, nullptr, nullptr, 0, d_y, y_type, ld_y, stream);
}

int retro_b200_w4_moe_workspace(const retro_b200_w4 * gate, uint32_t n_tokens, uint32_t n_used, size_t * out_bytes) {
    return boundary([&]() -> int {
        if (!gate || !out_bytes) return refuse("w4_moe_workspace", "a weight handle and a place for the result are required");
        if (n_used == 0 || n_used > kW4MaxUsed) return refuse("w4_moe_workspace", "n_used must be 1 to 32");
        *out_bytes = w4_moe_workspace_bytes(gate->view.n_out, n_tokens, n_used);
        return STATUS_OK;
    });
}

int retro_b200_w4_moe(const float * d_router, const retro_b200_w4 * gate, const retro_b200_w4 * up, const retro_b200_w4 * down, const void * d_x,
                      uint32_t x_type, int64_t ld_x, uint32_t n_tokens, uint32_t n_used, int normalise, const float * d_norm, float eps,
                      const void * d_residual, int64_t ld_residual, void * d_y, uint32_t y_type, int64_t ld_y, int32_t * d_ids, float * d_weights,
                      void * d_workspace, size_t workspace_bytes, void * stream) {
    return boundary([&]() -> int {
        const char * op = "w4_moe";
        if (!gate || !up || !down) return refuse(op, "a weight handle is required");
        const W4View & g = gate->view, & u = up->view, & d = down->view;
        if (u.type != g.type || u.n_out != g.n_out || u.n_in != g.n_in || u.n_expert != g.n_expert)
            return refuse(op, "gate and up must have one type and shape");
        if (d.n_expert != g.n_expert || d.n_in != g.n_out || d.n_out != g.n_in) return refuse(op, "down must be the transpose of gate in shape");
        if (up->device != gate->device || down->device != gate->device) return refuse(op, "the banks are on different devices");
        if (n_used == 0 || n_used > g.n_expert || n_used > kW4MaxUsed) return refuse(op, "n_used must be 1 to n_expert, at most 32");
        const w4::MoeShape shape{n_tokens, g.n_expert, n_used, g.n_in, g.n_out};
        const w4::Rows x{"x", d_x, x_type, ld_x}, y{"y", d_y, y_type, ld_y}, residual{"residual", d_residual, y_type, ld_residual};
        const w4::MoeBuffers buffers{d_router, d_ids, d_weights, d_workspace, workspace_bytes, w4_moe_workspace_bytes(g.n_out, n_tokens, n_used)};
        const std::string why = w4::check_moe(shape, x, y, residual, d_norm, eps, buffers);
        if (!why.empty()) return refuse(op, why);
        if (n_tokens == 0) return STATUS_OK;
        const DeviceScope scope(gate->device);
        W4Moe p;
        p.gate = g;
        p.up = u;
        p.down = d;
        p.router = d_router;
        p.x = d_x;
        p.x_type = x_type;
        p.ld_x = ld_x;
        p.n_tokens = (int)n_tokens;
        p.n_used = (int)n_used;
        p.normalise = normalise != 0;
        p.norm = d_norm;
        p.eps = eps;
        p.residual = d_residual;
        p.ld_residual = ld_residual;
        p.y = d_y;
        p.y_type = y_type;
        p.ld_y = ld_y;
        p.ids = d_ids;
        p.weights = d_weights;
        p.workspace = d_workspace;
        return launched(op, launch_w4_moe(p, static_cast<cudaStream_t>(stream)));
    });
}

} // extern "C"
