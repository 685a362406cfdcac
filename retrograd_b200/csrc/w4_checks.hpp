// The argument checks of the products with 4-bit weights, free of CUDA calls: every refusal is decided from the
// arguments alone, before anything is enqueued.
#pragma once

#include "blocks.hpp"

#include <cmath>
#include <cstdint>
#include <string>

namespace rb200 {

constexpr uint32_t kW4MaxColumns = 262144;   // longest row: one token's activations of an eighth of it fit in shared memory
constexpr uint32_t kW4MaxExperts = 256;

namespace w4 {

// What the kernels hold as weights: an empty text, or why not. (A grid counts the units of a bank, an int its rows.)
inline std::string check_weights(uint32_t ggml_type, uint64_t n_out, uint64_t n_in, uint64_t n_expert) {
    if (ggml_type != GGML_Q4_0 && ggml_type != GGML_MXFP4) return "the weights must be Q4_0 (2) or MXFP4 (39)";
    if (n_out == 0 || n_in == 0 || n_in % 32 != 0) return "n_out must be at least 1 and n_in a multiple of 32";
    if (n_in > kW4MaxColumns) return "n_in is larger than 262144";
    if (n_expert == 0 || n_expert > kW4MaxExperts) return "n_expert must be 1 to 256";
    if (n_out > 0x7fffffe0ull || n_expert * ((n_out + 31) / 32) * ((n_in + 127) / 128) > 0x7fffffffull) return "the bank is too large";
    return "";
}

constexpr uint32_t kMaxTokens = 1u << 24;

inline bool element_type(uint32_t type) { return type == GGML_F32 || type == GGML_F16 || type == GGML_BF16; }
inline size_t element_bytes(uint32_t type) { return type == GGML_F32 ? 4 : 2; }

// A caller's rows: first element, element type, row stride in elements.
struct Rows {
    const char * name;
    const void * p;
    uint32_t type;
    int64_t ld;
};

// `rows` rows of `width` bytes, `stride` bytes apart.
struct Region {
    uintptr_t at;
    size_t rows, width, stride;
    size_t bytes() const { return rows ? (rows - 1) * stride + width : 0; }
};

inline Region region(const Rows & r, size_t rows, size_t width) {
    const size_t es = element_bytes(r.type);
    return {reinterpret_cast<uintptr_t>(r.p), r.p ? rows : 0, width * es, (size_t)r.ld * es};
}
inline Region flat(const void * p, size_t bytes) { return {reinterpret_cast<uintptr_t>(p), p ? (size_t)1 : 0, bytes, bytes}; }

// Whether the two regions share a byte. Rows of one stride may interleave, as column ranges of one buffer do.
inline bool overlap(const Region & a, const Region & b) {
    if (!a.bytes() || !b.bytes() || a.at + a.bytes() <= b.at || b.at + b.bytes() <= a.at) return false;
    if (a.rows == 1 || b.rows == 1 || a.stride != b.stride || a.stride < a.width || a.stride < b.width) {
        if (a.rows == 1 && b.rows == 1) return true;
        // one row against many: it may lie in the gap behind one of them
        const Region & one = a.rows == 1 ? a : b;
        const Region & many = a.rows == 1 ? b : a;
        if (one.rows != 1 || many.stride < many.width || one.at < many.at) return true;
        const size_t shift = (one.at - many.at) % many.stride;
        return shift < many.width || shift + one.width > many.stride;
    }
    const size_t s = a.stride;
    const size_t shift = b.at >= a.at ? (b.at - a.at) % s : (s - (a.at - b.at) % s) % s;
    return shift < a.width || shift + b.width > s;
}

// An empty text when the rows can be read (or, `written`, written).
inline std::string check_rows(const Rows & r, size_t rows, size_t width, bool written) {
    const std::string n = r.name;
    if (!r.p) return n + " is required";
    if (!element_type(r.type)) return n + " must be f32 (0), f16 (1) or bf16 (30)";
    if (reinterpret_cast<uintptr_t>(r.p) % element_bytes(r.type) != 0) return n + " must be aligned to its element type";
    if (r.ld < 0 || r.ld > (int64_t)1 << 36) return n + ": the row stride is negative or too large";
    if (written && rows > 1 && r.ld < (int64_t)width) return n + ": the row stride is smaller than a row";
    return "";
}

inline std::string check_vector(const char * name, const void * p) {
    return reinterpret_cast<uintptr_t>(p) % 4 != 0 ? std::string(name) + " must be 4-byte aligned" : std::string();
}

inline std::string check_norm(const float * norm, float eps) {
    if (norm && !(eps >= 0.f && std::isfinite(eps))) return "eps must be finite and not negative";
    return check_vector("norm", norm);
}

// A residual may be y itself; anything else y is not allowed to touch.
inline std::string check_residual(const Rows & y, const Rows & residual, size_t rows, size_t width) {
    if (!residual.p) return "";
    const std::string why = check_rows(residual, rows, width, false);
    if (!why.empty()) return why;
    if (residual.p == y.p && (residual.ld == y.ld || rows <= 1)) return "";
    return overlap(region(y, rows, width), region(residual, rows, width)) ? "y overlaps residual without being it" : "";
}

struct ProductShape {
    uint32_t tokens, n_in, n_out;
};

inline std::string check_product(const ProductShape & s, const Rows & x, const Rows & y, const Rows & residual, const float * norm, float eps, const float * bias) {
    if (s.tokens > kMaxTokens) return "too many tokens";
    std::string why = check_rows(x, s.tokens, s.n_in, false);
    if (why.empty()) why = check_rows(y, s.tokens, s.n_out, true);
    if (why.empty()) why = check_norm(norm, eps);
    if (why.empty()) why = check_vector("bias", bias);
    if (!why.empty()) return why;
    const Region out = region(y, s.tokens, s.n_out);
    if (overlap(out, region(x, s.tokens, s.n_in))) return "y overlaps x";
    if (overlap(out, flat(norm, 4 * (size_t)s.n_in)) || overlap(out, flat(bias, 4 * (size_t)s.n_out))) return "y overlaps norm or bias";
    return check_residual(y, residual, s.tokens, s.n_out);
}

struct MoeShape {
    uint32_t tokens, n_expert, n_used, d, ff;
};

struct MoeBuffers {
    const float * router;
    int32_t * ids;
    float * weights;
    void * workspace;
    size_t workspace_bytes, workspace_needed;
};

inline std::string check_moe(const MoeShape & s, const Rows & x, const Rows & y, const Rows & residual, const float * norm, float eps, const MoeBuffers & m) {
    if (s.tokens > kMaxTokens) return "too many tokens";
    std::string why = check_rows(x, s.tokens, s.d, false);
    if (why.empty()) why = check_rows(y, s.tokens, s.d, true);
    if (why.empty()) why = check_norm(norm, eps);
    if (why.empty() && !m.router) why = "router is required";
    if (why.empty()) why = check_vector("router", m.router);
    if (why.empty()) why = check_vector("ids", m.ids);
    if (why.empty()) why = check_vector("weights", m.weights);
    if (!why.empty()) return why;
    if (!m.workspace || m.workspace_bytes < m.workspace_needed)
        return "the workspace needs " + std::to_string(m.workspace_needed) + " bytes";
    if (reinterpret_cast<uintptr_t>(m.workspace) % 16 != 0) return "the workspace must be 16-byte aligned";
    // everything that is written, against what is read and against one another; x may be y itself
    const Region out = region(y, s.tokens, s.d), in = region(x, s.tokens, s.d), work = flat(m.workspace, m.workspace_needed);
    const Region norms = flat(norm, 4 * (size_t)s.d), route = flat(m.router, 4 * (size_t)s.d * s.n_expert);
    const size_t picks = 4 * (size_t)s.tokens * s.n_used;
    const Region ids = flat(m.ids, picks), weights = flat(m.weights, picks), res = region(residual, s.tokens, s.d);
    const bool in_place = x.p == y.p && x.type == y.type && (x.ld == y.ld || s.tokens <= 1);
    if (!in_place && overlap(out, in)) return "y overlaps x without being it";
    for (const Region & w : {work, ids, weights})
        for (const Region & r : {out, in, norms, route, res})
            if (overlap(w, r)) return "the workspace, ids or weights overlap another operand";
    if (overlap(work, ids) || overlap(work, weights) || overlap(ids, weights)) return "the workspace, ids or weights overlap another operand";
    if (overlap(out, norms) || overlap(out, route)) return "y overlaps norm or router";
    return check_residual(y, residual, s.tokens, s.d);
}

} // namespace w4
} // namespace rb200
