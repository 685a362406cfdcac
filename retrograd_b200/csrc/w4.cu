// Products with 4-bit weights for at most sixteen tokens, bound by the weight stream.
//
// Mathematics. A unit of 16 rows x 64 columns is the A operand of four m16n8k16 products; the tokens are the columns
// of B. The weights enter as exact f16 values that cost no arithmetic beyond masks and shifts:
//   Q4_0   the nibble q in the low bits of an f16 is the subnormal q 2^-24, in the next four bits 16 q 2^-24; the
//          columns whose nibbles sit there get their activations divided by 16. The offset is the product chain's start
//          value, -8 2^-24 times the group's sum of activations.
//   MXFP4  sign and e2m1 magnitude placed at an f16's sign bit and bits 9..11 are the value times 2^-14.
// A token's activations are scaled by a power of two that brings the largest of them into [2^13, 2^14) and split into
// hi + lo f16 (22 bits); activations that are f16 or bf16 themselves need no lo. A 32-column group is exactly two
// products, so its f32 sum comes out on its own, is multiplied by the group's scale and added in f32.
//
// Split. A cluster of up to eight CTAs owns a range of row tiles; each CTA takes a range of the columns for all of them, so
// it converts only its share of the activations. Its warps take (pair of row tiles, part of the CTA's columns) items, and
// the partial sums meet in shared memory, are added over the cluster's shared memories in a fixed order (no workspace, no
// atomics: results are the same in every run), and get bias, residual or the gate's activation there. Every warp keeps
// kDepth units of two tiles in flight in registers.

#include "kernels.cuh"
#include "blocks.hpp"
#include "w4.cuh"

#include <algorithm>
#include <cuda_bf16.h>

namespace rb200 {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kDepth = 4;           // units in flight per warp and row tile
constexpr int kSlotCol = 36;        // floats per (partial slot, token): 32 rows, padded so that a warp's stores meet no bank twice
constexpr int kMaxSegs = 16;
constexpr int kRowList = kW4PassTokens;

struct Act {
    const void * p;
    int64_t ld;
    uint32_t type;
    bool vec;       // four elements may be read at once
};

__device__ __forceinline__ float load1(const Act & a, int64_t row, int k) {
    const int64_t i = row * a.ld + k;
    if (a.type == GGML_F32) return static_cast<const float *>(a.p)[i];
    const uint16_t h = static_cast<const uint16_t *>(a.p)[i];
    return a.type == GGML_F16 ? __half2float(__ushort_as_half(h)) : __uint_as_float((uint32_t)h << 16);
}

// Elements k .. k + 3 of a row.
__device__ __forceinline__ void load4(const Act & a, int64_t row, int k, float (&v)[4]) {
    if (!a.vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = load1(a, row, k + i);
        return;
    }
    const int64_t at = row * a.ld + k;
    if (a.type == GGML_F32) {
        const float4 f = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.p) + at);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
        const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.p) + at);
        if (a.type == GGML_F16) {
            const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)), hi = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
            v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
        } else {
            v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
            v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
        }
    }
}

__device__ __forceinline__ void store1(void * p, uint32_t type, int64_t i, float v) {
    if (type == GGML_F32) static_cast<float *>(p)[i] = v;
    else if (type == GGML_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// ---- cluster

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t smem_address(const void * p) { return (uint32_t)__cvta_generic_to_shared(p); }
// Shared-memory float `index` behind `base` of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t remote_address(uint32_t base, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(base), "r"(rank));
    return a;
}
__device__ __forceinline__ float remote_load(uint32_t address) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(address) : "memory");
    return v;
}

// ---- weights

template <bool MX> struct Unit {
    uint4 q;
    uint2 s;        // MXFP4 uses .x only
};

template <bool MX> __device__ __forceinline__ void load_unit(Unit<MX> & u, const uint8_t * p, int lane) {
    // weights are never written while a handle lives, so the read-only path holds even while earlier kernels still run
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(u.q.x), "=r"(u.q.y), "=r"(u.q.z), "=r"(u.q.w) : "l"(p + lane * 16));
    if constexpr (MX) {
        asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(u.s.x) : "l"(p + 512 + (lane >> 2) * 4));
    } else {
        asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(u.s.x), "=r"(u.s.y) : "l"(p + 512 + (lane >> 2) * 8));
    }
}

// A registers of product S of group H from the lane's four words.
template <bool MX, int H, int S> __device__ __forceinline__ void decode(const uint4 & q, uint32_t (&a)[4]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (!MX) {
            a[j] = (S ? w[j] >> 8 : w[j]) & (H ? 0x00f000f0u : 0x000f000fu);
        } else if constexpr (H == 0 && S == 0) {
            a[j] = w[j] & 0x8e008e00u;
        } else if constexpr (H == 0) {
            a[j] = (w[j] << 3) & 0x8e008e00u;
        } else if constexpr (S == 0) {
            // sign at bit 14, magnitude at 5..3: one multiplication moves both
            a[j] = ((w[j] & 0x40384038u) * 66u) & 0x8e008e00u;
        } else {
            // sign at bit 13, magnitude at 2..0
            a[j] = ((w[j] & 0x20072007u) * 516u) & 0x8e008e00u;
        }
    }
}

// Scales of rows g and g + 8 for group H.
template <bool MX, int H> __device__ __forceinline__ void scales(const uint2 & s, float & d0, float & d1) {
    if constexpr (MX) {
        d0 = __uint_as_float((H ? s.x << 15 : s.x << 23) & 0x7f800000u);
        d1 = __uint_as_float((H ? s.x >> 1 : s.x << 7) & 0x7f800000u);
    } else {
        const __half2 a = *reinterpret_cast<const __half2 *>(&s.x), b = *reinterpret_cast<const __half2 *>(&s.y);
        d0 = H ? __high2float(a) : __low2float(a);
        d1 = H ? __high2float(b) : __low2float(b);
    }
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// How many tokens a product chain serves. PACK: up to four, MMA column c is token c's hi part and column c + 4 its lo part.
enum Mode { PACK = 0, ONE = 1, TWO = 2 };
__device__ __forceinline__ int mode_of(int n, int parts) { return n > 8 ? TWO : parts == 2 && n <= 4 ? PACK : ONE; }

// ---- activations in shared memory
//
// x   [step][group][part][token][32] f16, c [step][group][token] f32: the start value of the group's products (Q4_0).
struct Staged {
    uint8_t * x;
    float * c;
    int n;          // tokens held
};
__host__ __device__ inline int staged_x_bytes(int steps, int parts, int n) { return steps * 2 * parts * n * 64; }
__host__ __device__ inline int staged_c_bytes(bool mx, int steps, int n) { return mx ? 0 : steps * 2 * n * 4; }

struct Scratch {
    float f1[kMaxSegs][kRowList], f2[kMaxSegs][kRowList];   // a token's sums times f1 times f2 are in the activations' own scale
    float ss[kRowList];                                     // sum of squares of the CTA's columns
    float red[2][kWarps];
};

// Converts columns [k0, k0 + 64 steps) of `n` rows. row_of(i) is the row of token i; columns at and behind n_in are zero.
template <bool MX, int PARTS, class RowOf>
__device__ void stage(const Act & act, RowOf row_of, int n, int k0, int steps, int n_in, const float * norm, const Staged & out, Scratch & sc, int seg) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_token = n > 4 ? 1 : n > 2 ? 2 : n > 1 ? 4 : 8;      // warps that share a token
    const int stride = kWarps / per_token;
    const int part = warp % per_token;
    const int count = steps * 16;                                     // chunks of four columns
    for (int t0 = 0; t0 < n; t0 += stride) {
        const int t = t0 + warp / per_token;
        const bool live = t < n;
        const int64_t row = live ? row_of(t) : 0;
        float top = 0.f, squares = 0.f;
        bool finite = true;
        for (int i = part * 32 + lane; live && i < count; i += per_token * 32) {
            const int k = k0 + 4 * i;
            if (k >= n_in) break;
            float v[4];
            load4(act, row, k, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                squares += v[e] * v[e];
                if (norm) v[e] *= norm[k + e];
                top = fmaxf(top, fabsf(v[e]));
                finite = finite && fabsf(v[e]) < INFINITY;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            squares += __shfl_xor_sync(0xffffffffu, squares, o);
        }
        if (!__all_sync(0xffffffffu, finite)) top = INFINITY;
        if (per_token > 1) {
            if (lane == 0) { sc.red[0][warp] = top; sc.red[1][warp] = squares; }
            __syncthreads();
            const int first = warp - part;
            top = 0.f;
            squares = 0.f;
            for (int i = 0; i < per_token; ++i) { top = fmaxf(top, sc.red[0][first + i]); squares += sc.red[1][first + i]; }
        }
        // 2^shift brings the largest magnitude into [2^13, 2^14); in two factors, so that none leaves f32. A row with an
        // infinity or a NaN is left as it is: its own sums become NaN, those of the other tokens stay what they are.
        const int shift = top > 0.f && top < INFINITY ? 13 - ilogbf(top) : 0;
        const float up1 = scalbnf(1.f, shift / 2), up2 = scalbnf(1.f, shift - shift / 2);
        if (live && part == 0 && lane == 0) {
            const int down = (MX ? 6 : 24) - shift;
            sc.f1[seg][t] = scalbnf(1.f, down / 2);
            sc.f2[seg][t] = scalbnf(1.f, down - down / 2);
            sc.ss[t] = squares;
        }
        // the trip count is the warp's, not the lane's: the group sums below are taken by the whole warp
        const int trips = live ? (count + per_token * 32 - 1) / (per_token * 32) : 0;
        for (int it = 0; it < trips; ++it) {
            const int i = it * per_token * 32 + part * 32 + lane;
            const int k = k0 + 4 * i;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (i < count && k < n_in) {
                load4(act, row, k, v);
                if (norm) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] *= norm[k + e];
                }
            }
            const int step = i >> 4, group = (i >> 3) & 1, at = (i & 7) * 4;
            const float lower = !MX && group ? 0.0625f : 1.f;
            __half hi[4], lo[4];
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float f = v[e] * up1 * up2 * lower;
                hi[e] = __float2half_rn(f);
                sum += __half2float(hi[e]);
                if constexpr (PARTS == 2) {
                    lo[e] = __float2half_rn(f - __half2float(hi[e]));
                    sum += __half2float(lo[e]);
                }
            }
            if (i < count) {
                uint8_t * dst = out.x + ((size_t)((step * 2 + group) * PARTS) * out.n + t) * 64 + at * 2;
                *reinterpret_cast<uint2 *>(dst) = make_uint2((uint32_t)__half_as_ushort(hi[0]) | (uint32_t)__half_as_ushort(hi[1]) << 16,
                                                             (uint32_t)__half_as_ushort(hi[2]) | (uint32_t)__half_as_ushort(hi[3]) << 16);
                if constexpr (PARTS == 2)
                    *reinterpret_cast<uint2 *>(dst + (size_t)out.n * 64) =
                        make_uint2((uint32_t)__half_as_ushort(lo[0]) | (uint32_t)__half_as_ushort(lo[1]) << 16,
                                   (uint32_t)__half_as_ushort(lo[2]) | (uint32_t)__half_as_ushort(lo[3]) << 16);
            }
            if constexpr (!MX) {
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (i < count && (lane & 7) == 0) out.c[(step * 2 + group) * out.n + t] = sum * (group ? -128.f : -8.f) * 5.9604644775390625e-8f;
            }
        }
        if (per_token > 1) __syncthreads();     // sc.red is written again for the next tokens
    }
}

// ---- the product chain

// A run: consecutive 64-column steps of two row tiles against one set of tokens.
struct Run {
    const uint8_t * p0, * p1;   // the tiles' first units
    int len;                    // steps
    Staged x;                   // activations, from the run's first step on
    const uint8_t * list;       // token (place in x) of each MMA column
    int n;                      // how many
};

// Where a lane finds its B fragments and start values of one run.
struct Lane {
    const uint8_t * b[2];
    const float * c[2][2];
    int b_step, b_part, b_group, c_step, c_group;
};

template <bool MX, int PARTS>
__device__ __forceinline__ void begin_run(const Run & r, int mode, int lane, Lane & l) {
    const int g = lane >> 2, t4 = lane & 3;
    l.b_part = r.x.n * 64;
    l.b_group = PARTS * l.b_part;
    l.b_step = 2 * l.b_group;
    l.c_step = 2 * r.x.n;
    l.c_group = r.x.n;
    if (mode == PACK) {
        const int tok = r.list[min(g & 3, r.n - 1)];
        l.b[0] = r.x.x + (size_t)tok * 64 + t4 * 16 + (g >= 4 ? l.b_part : 0);
    } else {
        l.b[0] = r.x.x + (size_t)r.list[min(g, r.n - 1)] * 64 + t4 * 16;
    }
    l.b[1] = mode == TWO ? r.x.x + (size_t)r.list[min(g + 8, r.n - 1)] * 64 + t4 * 16 : l.b[0];
    if constexpr (!MX) {
#pragma unroll
        for (int nc = 0; nc < 2; ++nc)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = mode == PACK ? (2 * t4 + e) & 3 : 8 * nc + 2 * t4 + e;
                l.c[nc][e] = r.x.c + r.list[min(col, r.n - 1)];
            }
    }
}

template <bool MX, int PARTS, int MODE>
__device__ __forceinline__ void do_step(const Unit<MX> (&u)[2], Lane & l, int lane, float (&acc)[2][2][4]) {
    constexpr int NC = MODE == TWO ? 2 : 1;
    constexpr int NP = MODE == PACK ? 1 : PARTS;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint4 b[NC][NP];
        float start[NC][2];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
#pragma unroll
            for (int p = 0; p < NP; ++p) b[nc][p] = *reinterpret_cast<const uint4 *>(l.b[nc] + h * l.b_group + p * l.b_part);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                start[nc][e] = 0.f;
                if constexpr (!MX) {
                    start[nc][e] = l.c[nc][e][h * l.c_group];
                    if (MODE == PACK && (lane & 2)) start[nc][e] = 0.f;      // the lo columns carry no offset
                }
            }
        }
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
            float c[NC][4];
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) { c[nc][0] = c[nc][2] = start[nc][0]; c[nc][1] = c[nc][3] = start[nc][1]; }
            uint32_t a[4];
            if (h == 0) decode<MX, 0, 0>(u[tile].q, a); else decode<MX, 1, 0>(u[tile].q, a);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc)
#pragma unroll
                for (int p = 0; p < NP; ++p) mma(c[nc], a, b[nc][p].x, b[nc][p].y);
            if (h == 0) decode<MX, 0, 1>(u[tile].q, a); else decode<MX, 1, 1>(u[tile].q, a);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc)
#pragma unroll
                for (int p = 0; p < NP; ++p) mma(c[nc], a, b[nc][p].z, b[nc][p].w);
            float d0, d1;
            if (h == 0) scales<MX, 0>(u[tile].s, d0, d1); else scales<MX, 1>(u[tile].s, d0, d1);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) {
                acc[tile][nc][0] += d0 * c[nc][0];
                acc[tile][nc][1] += d0 * c[nc][1];
                acc[tile][nc][2] += d1 * c[nc][2];
                acc[tile][nc][3] += d1 * c[nc][3];
            }
        }
    }
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
        l.b[nc] += l.b_step;
        if constexpr (!MX) { l.c[nc][0] += l.c_step; l.c[nc][1] += l.c_step; }
    }
}

// Calls put(row 0..31 of the pair, column, sum) for every column of the run this lane holds.
template <class Put>
__device__ __forceinline__ void end_run(int mode, int n, int lane, float (&acc)[2][2][4], Put put) {
    const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
#pragma unroll
        for (int nc = 0; nc < 2; ++nc) {
            if (nc == 1 && mode != TWO) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = acc[tile][nc][i];
                if (mode == PACK) v += __shfl_xor_sync(0xffffffffu, v, 2);      // hi column + lo column
                const int col = 8 * nc + 2 * t4 + (i & 1);
                if (col < n && !(mode == PACK && t4 >= 2)) put(tile * 16 + g + (i >> 1) * 8, col, v);
            }
        }
#pragma unroll
        for (int nc = 0; nc < 2; ++nc)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[tile][nc][i] = 0.f;
    }
}

// A warp's sequence of runs: items warp, warp + kWarps, ... below n_items, each with n_segs runs (some may be empty).
// Source: int len(item, seg); Run run(item, seg); put(item, seg, row, column, sum). MODES: the modes that occur.
template <bool MX, int PARTS, int MODES, class Source>
struct Stream {
    Source & src;
    const int n_items, n_segs, lane;
    Unit<MX> buf[kDepth][2];
    struct Cursor { int item, seg, rem; } ld, cp;
    const uint8_t * p0, * p1;

    __device__ __forceinline__ Stream(Source & s, int items, int segs) : src(s), n_items(items), n_segs(segs), lane(threadIdx.x & 31) {
        ld = {(int)(threadIdx.x >> 5), -1, 0};
        next(ld);
        cp = ld;
        if (ld.item < n_items) point();
    }
    __device__ __forceinline__ void next(Cursor & c) {
        do {
            if (++c.seg == n_segs) { c.seg = 0; c.item += kWarps; }
            if (c.item >= n_items) return;
            c.rem = src.len(c.item, c.seg);
        } while (c.rem == 0);
    }
    __device__ __forceinline__ void point() {
        const Run r = src.run(ld.item, ld.seg);
        p0 = r.p0;
        p1 = r.p1;
    }
    __device__ __forceinline__ void fetch(int d) {
        if (ld.item >= n_items) return;
        load_unit<MX>(buf[d][0], p0, lane);
        load_unit<MX>(buf[d][1], p1, lane);
        p0 += w4_unit_bytes(MX);
        p1 += w4_unit_bytes(MX);
        if (--ld.rem == 0) {
            next(ld);
            if (ld.item < n_items) point();
        }
    }
    // The first units of the sequence; needs nothing but the weights.
    __device__ __forceinline__ void prefetch() {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) fetch(d);
    }
    __device__ __forceinline__ void work() {
        if (cp.item >= n_items) return;
        float acc[2][2][4] = {};
        Lane l;
        Run r = src.run(cp.item, cp.seg);
        int mode = mode_of(r.n, PARTS);
        begin_run<MX, PARTS>(r, mode, lane, l);
        while (cp.item < n_items) {
#pragma unroll
            for (int d = 0; d < kDepth; ++d) {
                if (cp.item >= n_items) break;
                if constexpr (MODES & (1 << PACK)) if (MODES == (1 << PACK) || mode == PACK) do_step<MX, PARTS, PACK>(buf[d], l, lane, acc);
                if constexpr (MODES & (1 << ONE)) if (MODES == (1 << ONE) || mode == ONE) do_step<MX, PARTS, ONE>(buf[d], l, lane, acc);
                if constexpr (MODES & (1 << TWO)) if (MODES == (1 << TWO) || mode == TWO) do_step<MX, PARTS, TWO>(buf[d], l, lane, acc);
                fetch(d);
                if (--cp.rem == 0) {
                    end_run(mode, r.n, lane, acc, [&](int row, int col, float v) { src.put(cp.item, cp.seg, row, col, v); });
                    next(cp);
                    if (cp.item < n_items) {
                        r = src.run(cp.item, cp.seg);
                        mode = mode_of(r.n, PARTS);
                        begin_run<MX, PARTS>(r, mode, lane, l);
                    }
                }
            }
        }
    }
};

// Parts of the columns the warps split an item into: as few as keep the warps evenly loaded. The cost counts steps of the
// busiest warp and two steps' time for every partial sum it writes.
__host__ __device__ inline int split_columns(int jobs, int steps) {
    int best = 1, best_cost = 0x7fffffff;
    for (int ks = 1; ks <= kWarps; ks *= 2) {
        if (ks > 1 && ks > steps) break;
        const int rounds = (jobs * ks + kWarps - 1) / kWarps;
        const int cost = rounds * ((steps + ks - 1) / ks + 2);
        if (cost < best_cost) { best_cost = cost; best = ks; }
    }
    return best;
}

// Range `part` of `parts` nearly equal ranges of [0, n).
__host__ __device__ inline int part_begin(int n, int part, int parts) { return (int)((int64_t)n * part / parts); }

// ---- y = W x, and y = silu(W x) * (U x)

struct ProductArgs {
    const uint8_t * w, * u;
    Act x;
    int T, n_in, n_out, tiles, steps;
    const float * norm;
    float eps;
    const float * bias;
    const void * residual;
    int64_t ld_residual;
    void * y;
    uint32_t y_type;
    int64_t ld_y;
    int jobs, clusters;             // a job is a pair of row tiles; with the gate, one tile of each matrix
    int x_bytes, c_bytes, slots;    // shared memory: staged activations, start values, partial slots of T * kSlotCol floats
};

template <bool MX, bool GLU> struct ProductSource {
    const ProductArgs & a;
    const uint8_t * list;
    Staged x;
    float * partial;
    const Scratch & sc;
    int job0, s0, n_steps, ks;

    __device__ __forceinline__ int len(int item, int) const {
        const int sub = item % ks;
        return part_begin(n_steps, sub + 1, ks) - part_begin(n_steps, sub, ks);
    }
    __device__ __forceinline__ Run run(int item, int) const {
        const int job = job0 + item / ks, sub = item % ks;
        const int s = part_begin(n_steps, sub, ks);
        const int t0 = GLU ? job : 2 * job, t1 = GLU ? job : min(2 * job + 1, a.tiles - 1);
        Run r;
        r.p0 = a.w + ((size_t)t0 * a.steps + s0 + s) * w4_unit_bytes(MX);
        r.p1 = (GLU ? a.u : a.w) + ((size_t)t1 * a.steps + s0 + s) * w4_unit_bytes(MX);
        r.len = 0;
        r.x = {x.x + (size_t)s * (x.n * 64) * b_rows, MX ? nullptr : x.c + (size_t)s * 2 * x.n, x.n};
        r.list = list;
        r.n = a.T;
        return r;
    }
    int b_rows;     // 2 * PARTS
    __device__ __forceinline__ void put(int item, int, int row, int col, float v) const {
        partial[((size_t)item * a.T + col) * kSlotCol + row] = v * sc.f1[0][col] * sc.f2[0][col];
    }
};

template <bool MX, int PARTS, bool GLU, int MODE>
__global__ void __launch_bounds__(kThreads, 2) w4_product_kernel(ProductArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Scratch sc;
    __shared__ uint8_t list[kRowList];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), C = (int)cluster_size();
    const int cluster = blockIdx.x / C;
    const int s0 = part_begin(a.steps, rank, C), n_steps = part_begin(a.steps, rank + 1, C) - s0;
    const int j_begin = part_begin(a.jobs, cluster, a.clusters), j_end = part_begin(a.jobs, cluster + 1, a.clusters);
    const int ks = min(split_columns(j_end - j_begin, a.steps / C), a.slots);
    const int per_round = max(1, a.slots / ks);
    Staged x{smem, reinterpret_cast<float *>(smem + a.x_bytes), a.T};
    float * partial = reinterpret_cast<float *>(smem + a.x_bytes + a.c_bytes);
    if (threadIdx.x < kRowList) list[threadIdx.x] = (uint8_t)threadIdx.x;

    for (int j0 = j_begin; j0 < j_end; j0 += per_round) {
        const int jobs = min(per_round, j_end - j0);
        ProductSource<MX, GLU> src{a, list, x, partial, sc, j0, s0, n_steps, ks, 2 * PARTS};
        Stream<MX, PARTS, 1 << MODE, ProductSource<MX, GLU>> stream(src, jobs * ks, 1);
        stream.prefetch();
        if (j0 == j_begin) {
            // the weights above are the library's own; everything below is the caller's
            pdl_trigger();
            pdl_wait();
            stage<MX, PARTS>(a.x, [](int t) { return (int64_t)t; }, a.T, s0 * 64, n_steps, a.n_in, a.norm, x, sc, 0);
            __syncthreads();
        }
        stream.work();
        cluster_sync();
        // 32 rows of one token at a time: the cluster's partial sums in the order of the columns
        const uint32_t base = smem_address(partial);
        for (int u = rank + C * warp; u < jobs * a.T; u += C * kWarps) {
            const int job = u / a.T, t = u % a.T;
            float v = 0.f;
            for (int c = 0; c < C; ++c) {
                const uint32_t at = remote_address(base, c) + (((size_t)job * ks * a.T + t) * kSlotCol + lane) * 4;
                for (int i = 0; i < ks; ++i) v += remote_load(at + (uint32_t)(i * a.T * kSlotCol * 4));
            }
            if (a.norm) {
                float ss = lane < C ? remote_load(remote_address(smem_address(&sc.ss[t]), lane)) : 0.f;
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                ss = __shfl_sync(0xffffffffu, ss, 0);
                v *= rsqrtf(ss / (float)a.n_in + a.eps);
            }
            int row;
            if constexpr (GLU) {
                const float up = __shfl_down_sync(0xffffffffu, v, 16);
                v = v / (1.f + expf(-v)) * up;
                row = lane < 16 ? (j0 + job) * 16 + lane : a.n_out;
            } else {
                row = (j0 + job) * 32 + lane;
            }
            if (row < a.n_out) {
                if (a.bias) v += a.bias[row];
                if (a.residual) v += load1(Act{a.residual, a.ld_residual, a.y_type, false}, t, row);
                store1(a.y, a.y_type, t * a.ld_y + row, v);
            }
        }
        cluster_sync();     // nobody reuses or leaves the slots that others still read
    }
    if (j_begin >= j_end) {
        pdl_trigger();
        pdl_wait();
    }
}

// ---- a mixture-of-experts layer
//
// Two kernels. The first: every cluster normalises and routes all tokens for itself (the router is a few hundred
// kilobytes that the L2 cache holds; one CTA reads an eighth of it) instead of waiting for one place to do it, then multiplies its share of the chosen
// experts' (gate tile, up tile) pairs and writes h = w_e silu(a) b for each (token, expert) pair. The second treats the chosen
// experts' down matrices as one long reduction: a cluster owns a range of y's rows, its CTAs divide the experts' concatenated columns,
// and the sum over experts is part of the sum over the cluster.

struct MoeMeta {                        // in the workspace, in front of h
    int32_t n;                          // chosen experts
    int32_t pad[3];
    uint16_t expert[kW4MaxExperts];     // ascending
    uint16_t count[kW4MaxExperts];      // their tokens
    uint16_t pair[kW4MaxExperts][kRowList];     // token * n_used + rank of the expert among the token's
};

struct MoeArgs {
    const uint8_t * gate, * up, * down;
    size_t gate_expert, up_expert, down_expert;     // bytes of one expert
    const float * router;
    Act x;
    int T, E, k, d, ff;
    int tiles_ff, steps_d, tiles_d, steps_ff;
    bool normalise;
    const float * norm;
    float eps;
    const void * residual;
    int64_t ld_residual;
    void * y;
    uint32_t y_type;
    int64_t ld_y;
    int32_t * ids;
    float * weights;
    MoeMeta * meta;
    float * h;
    int64_t ld_h;
    int clusters, x_bytes, c_bytes, logit_bytes, partial_floats;
};

struct Picks {
    uint16_t expert[kRowList * kW4MaxUsed];
    float weight[kRowList * kW4MaxUsed];
    float rstd[kRowList];
    uint16_t unique[kW4MaxExperts];
    uint8_t count[kW4MaxExperts];                   // of unique[i]
    uint8_t token[kW4MaxExperts][kRowList];
    int warp_unique[kWarps];
    int n, most;                                    // unique experts, largest count
};

// The CTA's columns' part of every (token, expert) logit.
__device__ void partial_logits(const MoeArgs & a, int k0, int k1, float * out) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int EB = 4, TB = 4;       // experts and tokens a warp takes at once
    const Act router{a.router, a.d, GGML_F32, (uintptr_t)a.router % 16 == 0};
    for (int e0 = warp * EB; e0 < a.E; e0 += kWarps * EB) {
        for (int t0 = 0; t0 < a.T; t0 += TB) {
            float acc[EB][TB] = {};
            for (int k = k0 + lane * 4; k < k1; k += 128) {
                float g[4] = {1.f, 1.f, 1.f, 1.f};
                if (a.norm) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) g[i] = a.norm[k + i];
                }
                float r[EB][4];
#pragma unroll
                for (int e = 0; e < EB; ++e) load4(router, min(e0 + e, a.E - 1), k, r[e]);
#pragma unroll
                for (int t = 0; t < TB; ++t) {
                    if (t0 + t >= a.T) break;
                    float v[4];
                    load4(a.x, t0 + t, k, v);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float f = v[i] * g[i];
#pragma unroll
                        for (int e = 0; e < EB; ++e) acc[e][t] += r[e][i] * f;
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                if (t0 + t >= a.T) break;
#pragma unroll
                for (int e = 0; e < EB; ++e) {
                    float v = acc[e][t];
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                    if (lane == 0 && e0 + e < a.E) out[(t0 + t) * a.E + e0 + e] = v;
                }
            }
        }
    }
}

// Softmax over the experts and the n_used likeliest of one token, by one warp. Ties go to the lowest index; whatever the
// logits hold, n_used different experts are chosen (a NaN makes the weights NaN).
__device__ void pick_experts(const float * logits, int E, int k, bool normalise, uint16_t * expert, float * weight) {
    const int lane = threadIdx.x & 31;
    constexpr int PER = kW4MaxExperts / 32;
    float p[PER];
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = lane + 32 * j;
        p[j] = e < E ? logits[e] : -INFINITY;
        mx = fmaxf(mx, p[j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        p[j] = lane + 32 * j < E ? expf(p[j] - mx) : 0.f;
        sum += p[j];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    uint32_t taken = 0;
    float chosen = 0.f;
    for (int pick = 0; pick < k; ++pick) {
        float best = -2.f, value = 0.f;
        int at = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int e = lane + 32 * j;
            if (e >= E || (taken >> j & 1)) continue;
            const float v = p[j] / sum;
            const float key = v >= 0.f ? v : -1.f;      // NaN behind every number
            if (key > best) { best = key; value = v; at = e; }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ob = __shfl_xor_sync(0xffffffffu, best, o), ov = __shfl_xor_sync(0xffffffffu, value, o);
            const int oa = __shfl_xor_sync(0xffffffffu, at, o);
            if (ob > best || (ob == best && oa < at)) { best = ob; value = ov; at = oa; }
        }
        if ((at & 31) == lane) taken |= 1u << (at >> 5);
        if (lane == 0) { expert[pick] = (uint16_t)at; weight[pick] = value; }
        chosen += value;
    }
    if (normalise) {
        __syncwarp();
        for (int i = lane; i < k; i += 32) weight[i] /= chosen;
    }
}

// The chosen experts in ascending order with their tokens, from the picks of all tokens.
__device__ void group_picks(const MoeArgs & a, Picks & p, MoeMeta * meta) {
    const int e = threadIdx.x, warp = e >> 5, lane = e & 31;
    uint32_t mask = 0;                  // tokens that chose expert e
    if (e < a.E) {
        for (int i = 0; i < a.T * a.k; ++i)
            if (p.expert[i] == e) mask |= 1u << (i / a.k);
    }
    const uint32_t chosen = __ballot_sync(0xffffffffu, mask != 0);
    if (lane == 0) p.warp_unique[warp] = __popc(chosen);
    if (e == 0) p.most = 1;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += p.warp_unique[w];
        all += p.warp_unique[w];
    }
    if (mask) {
        const int u = before + __popc(chosen & ((1u << lane) - 1u));
        const int n = __popc(mask);
        p.unique[u] = (uint16_t)e;
        p.count[u] = (uint8_t)n;
        atomicMax(&p.most, n);
        int at = 0;
        for (uint32_t m = mask; m; m &= m - 1) p.token[u][at++] = (uint8_t)(__ffs(m) - 1);
        if (meta) {
            meta->expert[u] = (uint16_t)e;
            meta->count[u] = (uint16_t)n;
            for (int i = 0; i < n; ++i) {
                const int t = p.token[u][i];
                int j = 0;
                while (j < a.k - 1 && p.expert[t * a.k + j] != e) ++j;
                meta->pair[u][i] = (uint16_t)(t * a.k + j);
            }
        }
    }
    if (e == 0) {
        p.n = all;
        if (meta) meta->n = all;
    }
    __syncthreads();
}

template <bool MX, int PARTS> struct GateUpSource {
    const MoeArgs & a;
    const Picks & p;
    Staged x;
    float * partial;
    const Scratch & sc;
    int job0, s0, n_steps, ks, most;

    __device__ __forceinline__ int len(int item, int) const {
        const int sub = item % ks;
        return part_begin(n_steps, sub + 1, ks) - part_begin(n_steps, sub, ks);
    }
    __device__ __forceinline__ Run run(int item, int) const {
        const int job = job0 + item / ks, s = part_begin(n_steps, item % ks, ks);
        const int u = job / a.tiles_ff, tile = job % a.tiles_ff;
        const size_t at = ((size_t)tile * a.steps_d + s0 + s) * w4_unit_bytes(MX);
        const int e = p.unique[u];
        Run r;
        r.p0 = a.gate + e * a.gate_expert + at;
        r.p1 = a.up + e * a.up_expert + at;
        r.x = {x.x + (size_t)s * (2 * PARTS * 64) * x.n, MX ? nullptr : x.c + (size_t)s * 2 * x.n, x.n};
        r.list = p.token[u];
        r.n = p.count[u];
        return r;
    }
    __device__ __forceinline__ void put(int item, int, int row, int col, float v) const {
        const int tok = p.token[(job0 + item / ks) / a.tiles_ff][col];
        partial[((size_t)item * most + col) * kSlotCol + row] = v * sc.f1[0][tok] * sc.f2[0][tok];
    }
};

template <bool MX, int PARTS, int MODES>
__global__ void __launch_bounds__(kThreads, 2) w4_moe_gate_up_kernel(MoeArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Scratch sc;
    __shared__ Picks picks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), C = (int)cluster_size();
    const int cluster = blockIdx.x / C;
    const int s0 = part_begin(a.steps_d, rank, C), n_steps = part_begin(a.steps_d, rank + 1, C) - s0;
    Staged x{smem, reinterpret_cast<float *>(smem + a.x_bytes), a.T};
    float * mine = reinterpret_cast<float *>(smem + a.x_bytes + a.c_bytes);         // this CTA's part of the logits
    float * logits = mine + a.logit_bytes / 4;
    float * partial = logits + a.logit_bytes / 4;

    pdl_trigger();
    pdl_wait();
    stage<MX, PARTS>(a.x, [](int t) { return (int64_t)t; }, a.T, s0 * 64, n_steps, a.d, a.norm, x, sc, 0);
    partial_logits(a, s0 * 64, min(a.d, (s0 + n_steps) * 64), mine);
    cluster_sync();
    if (threadIdx.x < a.T) {
        float ss = 0.f;
        for (int c = 0; c < C; ++c) ss += remote_load(remote_address(smem_address(&sc.ss[threadIdx.x]), c));
        picks.rstd[threadIdx.x] = a.norm ? rsqrtf(ss / (float)a.d + a.eps) : 1.f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.T * a.E; i += kThreads) {
        float v = 0.f;
        for (int c = 0; c < C; ++c) v += remote_load(remote_address(smem_address(mine), c) + i * 4);
        logits[i] = v * picks.rstd[i / a.E];
    }
    __syncthreads();
    for (int t = warp; t < a.T; t += kWarps) pick_experts(logits + t * a.E, a.E, a.k, a.normalise, picks.expert + t * a.k, picks.weight + t * a.k);
    __syncthreads();
    const bool first = blockIdx.x == 0;
    group_picks(a, picks, first ? a.meta : nullptr);
    if (first) {
        for (int i = threadIdx.x; i < a.T * a.k; i += kThreads) {
            if (a.ids) a.ids[i] = picks.expert[i];
            if (a.weights) a.weights[i] = picks.weight[i];
        }
    }

    const int total = picks.n * a.tiles_ff, most = picks.most;
    const int j_begin = part_begin(total, cluster, a.clusters), j_end = part_begin(total, cluster + 1, a.clusters);
    const int slots = a.partial_floats / (most * kSlotCol);
    const int ks = min(split_columns(j_end - j_begin, a.steps_d / C), slots);
    const int per_round = slots / ks;
    for (int j0 = j_begin; j0 < j_end; j0 += per_round) {
        const int jobs = min(per_round, j_end - j0);
        GateUpSource<MX, PARTS> src{a, picks, x, partial, sc, j0, s0, n_steps, ks, most};
        Stream<MX, PARTS, MODES, GateUpSource<MX, PARTS>> stream(src, jobs * ks, 1);
        stream.prefetch();
        stream.work();
        cluster_sync();
        const uint32_t base = smem_address(partial);
        for (int i = rank + C * warp; i < jobs * most; i += C * kWarps) {
            const int job = i / most, col = i % most;
            const int u = (j0 + job) / a.tiles_ff, tile = (j0 + job) % a.tiles_ff;
            if (col >= picks.count[u]) continue;
            float v = 0.f;
            for (int c = 0; c < C; ++c) {
                const uint32_t at = remote_address(base, c) + (((size_t)job * ks * most + col) * kSlotCol + lane) * 4;
                for (int s = 0; s < ks; ++s) v += remote_load(at + (uint32_t)(s * most * kSlotCol * 4));
            }
            const int t = picks.token[u][col];
            v *= picks.rstd[t];
            const float b = __shfl_down_sync(0xffffffffu, v, 16);
            int j = 0;
            while (j < a.k - 1 && picks.expert[t * a.k + j] != picks.unique[u]) ++j;
            const int pair = t * a.k + j, row = tile * 16 + lane;
            if (lane < 16 && row < a.ff) a.h[pair * a.ld_h + row] = picks.weight[pair] * (v / (1.f + expf(-v)) * b);
        }
        cluster_sync();
    }
    cluster_sync();     // nobody leaves while its logits are read
}

struct Seg {
    int u, s0, len, x_off, c_off, n;
};
struct DownTable {
    Seg seg[kMaxSegs];
    int n;
    int next;           // the step behind the chunk
};

template <bool MX> struct DownSource {
    const MoeArgs & a;
    const DownTable & table;
    uint8_t * smem;
    float * partial;
    const Scratch & sc;
    const uint8_t * identity;
    int job0, ks;

    __device__ __forceinline__ int len(int item, int seg) const {
        const int n = table.seg[seg].len, sub = item % ks;
        return part_begin(n, sub + 1, ks) - part_begin(n, sub, ks);
    }
    __device__ __forceinline__ Run run(int item, int seg) const {
        const Seg & g = table.seg[seg];
        const int job = job0 + item / ks, s = part_begin(g.len, item % ks, ks);
        const uint8_t * e = a.down + a.meta->expert[g.u] * a.down_expert;
        Run r;
        r.p0 = e + ((size_t)(2 * job) * a.steps_ff + g.s0 + s) * w4_unit_bytes(MX);
        r.p1 = e + ((size_t)min(2 * job + 1, a.tiles_d - 1) * a.steps_ff + g.s0 + s) * w4_unit_bytes(MX);
        r.x = {smem + g.x_off + (size_t)s * (2 * 2 * 64) * g.n, MX ? nullptr : reinterpret_cast<float *>(smem + g.c_off) + (size_t)s * 2 * g.n, g.n};
        r.list = identity;
        r.n = g.n;
        return r;
    }
    __device__ __forceinline__ void put(int item, int seg, int row, int col, float v) const {
        const int tok = a.meta->pair[table.seg[seg].u][col] / a.k;
        partial[((size_t)item * a.T + tok) * kSlotCol + row] += v * sc.f1[seg][col] * sc.f2[seg][col];
    }
};

template <bool MX, int MODES>
__global__ void __launch_bounds__(kThreads, 2) w4_moe_down_kernel(MoeArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Scratch sc;
    __shared__ DownTable table;
    __shared__ uint8_t identity[kRowList];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), C = (int)cluster_size();
    const int cluster = blockIdx.x / C;
    float * partial = reinterpret_cast<float *>(smem + a.x_bytes);
    if (threadIdx.x < kRowList) identity[threadIdx.x] = (uint8_t)threadIdx.x;
    pdl_trigger();
    pdl_wait();
    const int total = a.meta->n * a.steps_ff;       // the chosen experts' columns, one behind the other
    const int begin = part_begin(total, rank, C), end = part_begin(total, rank + 1, C);
    const int jobs_all = (a.tiles_d + 1) / 2;
    const int j_begin = part_begin(jobs_all, cluster, a.clusters), j_end = part_begin(jobs_all, cluster + 1, a.clusters);
    const int slots = a.partial_floats / (a.T * kSlotCol);
    const int ks = min(split_columns(j_end - j_begin, max(1, total / C)), slots);
    const int per_round = slots / ks;
    const Act h{a.h, a.ld_h, GGML_F32, true};
    for (int j0 = j_begin; j0 < j_end; j0 += per_round) {
        const int jobs = min(per_round, j_end - j0);
        for (int i = threadIdx.x; i < jobs * ks * a.T * kSlotCol; i += kThreads) partial[i] = 0.f;
        for (int p = begin; p < end;) {
            if (threadIdx.x == 0) {
                // as many steps as fit into the shared memory for activations
                int n = 0, used = 0, at = p;
                while (at < end && n < kMaxSegs) {
                    const int u = at / a.steps_ff, off = at % a.steps_ff, tokens = a.meta->count[u];
                    const int each = staged_x_bytes(1, 2, tokens) + staged_c_bytes(MX, 1, tokens);
                    const int len = min(min(a.steps_ff - off, end - at), (a.x_bytes - used - 16) / each);
                    if (len <= 0) break;
                    const int x_bytes = staged_x_bytes(len, 2, tokens);
                    table.seg[n] = {u, off, len, used, used + x_bytes, tokens};
                    used += (x_bytes + staged_c_bytes(MX, len, tokens) + 15) / 16 * 16;
                    at += len;
                    ++n;
                }
                table.n = n;
                table.next = at;
            }
            __syncthreads();
            DownSource<MX> src{a, table, smem, partial, sc, identity, j0, ks};
            Stream<MX, 2, MODES, DownSource<MX>> stream(src, jobs * ks, table.n);
            stream.prefetch();
            for (int i = 0; i < table.n; ++i) {
                const Seg & g = table.seg[i];
                const uint16_t * pair = a.meta->pair[g.u];
                stage<MX, 2>(h, [pair](int t) { return (int64_t)pair[t]; }, g.n, g.s0 * 64, g.len, a.ff, nullptr,
                             Staged{smem + g.x_off, reinterpret_cast<float *>(smem + g.c_off), g.n}, sc, i);
            }
            __syncthreads();
            stream.work();
            p = table.next;
            __syncthreads();
        }
        cluster_sync();
        const uint32_t base = smem_address(partial);
        for (int u = rank + C * warp; u < jobs * a.T; u += C * kWarps) {
            const int job = u / a.T, t = u % a.T;
            float v = 0.f;
            for (int c = 0; c < C; ++c) {
                const uint32_t at = remote_address(base, c) + (((size_t)job * ks * a.T + t) * kSlotCol + lane) * 4;
                for (int i = 0; i < ks; ++i) v += remote_load(at + (uint32_t)(i * a.T * kSlotCol * 4));
            }
            const int row = (j0 + job) * 32 + lane;
            if (row < a.d) {
                if (a.residual) v += load1(Act{a.residual, a.ld_residual, a.y_type, false}, t, row);
                store1(a.y, a.y_type, t * a.ld_y + row, v);
            }
        }
        cluster_sync();
    }
}

// ---- retiling
//
// Word j (0..3) of lane (g, t) holds row g + 8 (j & 1), columns 8 t + 4 s + 2 (j >> 1) + e of group h, for the products
// s = 0, 1, groups h = 0, 1 and halves e = 0, 1 of the word. Q4_0: the nibble at bit 16 e + 8 s + 4 h. MXFP4: inside half
// e, (sign, magnitude) at bits (15, 11..9), (12, 8..6), (14, 5..3), (13, 2..0) for (h, s) = (0,0), (0,1), (1,0), (1,1).
template <bool MX>
__global__ void w4_retile_kernel(const uint8_t * rows, uint32_t n_out, uint32_t n_in, uint32_t tiles, uint32_t steps, uint8_t * units, int * max_scale) {
    constexpr uint32_t kBlock = MX ? 17 : 18;
    const uint32_t blocks = n_in / 32;
    const size_t unit = blockIdx.x;
    const uint32_t step = (uint32_t)(unit % steps);
    const size_t tile_of_all = unit / steps;
    const uint32_t tile = (uint32_t)(tile_of_all % tiles);
    const size_t expert = tile_of_all / tiles;
    uint8_t * dst = units + unit * w4_unit_bytes(MX);
    const uint32_t lane = threadIdx.x >> 2, j = threadIdx.x & 3;
    const uint32_t g = lane >> 2, t = lane & 3;
    const uint32_t row = tile * 16 + g + 8 * (j & 1);
    uint32_t word = 0;
    for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t block = step * 2 + h;
        if (row >= n_out || block >= blocks) continue;
        const uint8_t * q = rows + ((expert * n_out + row) * blocks + block) * kBlock + (MX ? 1 : 2);
        for (uint32_t s = 0; s < 2; ++s)
            for (uint32_t e = 0; e < 2; ++e) {
                const uint32_t k = 8 * t + 4 * s + 2 * (j >> 1) + e;
                const uint32_t n = (q[k & 15] >> (k >= 16 ? 4 : 0)) & 15u;
                if (!MX) {
                    word |= n << (16 * e + 8 * s + 4 * h);
                } else {
                    const uint32_t sign = n >> 3, mag = n & 7;
                    const uint32_t half = h == 0 ? (s == 0 ? sign << 15 | mag << 9 : sign << 12 | mag << 6) : (s == 0 ? sign << 14 | mag << 3 : sign << 13 | mag);
                    word |= half << (16 * e);
                }
            }
    }
    *reinterpret_cast<uint32_t *>(dst + lane * 16 + j * 4) = word;
    if (threadIdx.x < 32) {
        // scales of (g, group), then of (g + 8, group), for g = 0..7
        const uint32_t sg = threadIdx.x >> 2, upper = (threadIdx.x >> 1) & 1, h = threadIdx.x & 1;
        const uint32_t srow = tile * 16 + sg + 8 * upper, block = step * 2 + h;
        const bool live = srow < n_out && block < blocks;
        const uint8_t * b = rows + ((expert * n_out + srow) * blocks + block) * kBlock;
        if (MX) {
            // kept as s + 8, so that the smallest scale 2^-127 is a normal f32 as well; 2^-8 is part of the rows' final factor
            const int s = live ? b[0] : 0;
            if (live) atomicMax(max_scale, s);
            dst[512 + sg * 4 + upper * 2 + h] = live ? (uint8_t)min(s + 8, 255) : 0;
        } else {
            reinterpret_cast<uint16_t *>(dst + 512)[sg * 4 + upper * 2 + h] = live ? (uint16_t)(b[0] | b[1] << 8) : 0;
        }
    }
}

// ---- launch plans

int device_sms() {
    static int sms[256] = {};
    int device = 0;
    cudaGetDevice(&device);
    int & n = sms[device & 255];
    if (!n) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
    return n;
}

constexpr int kMaxSmem = 200 * 1024;

template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), int grid, int cluster, size_t smem, cudaStream_t stream, Args &&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

template <bool MX, int PARTS, bool GLU, int MODE>
cudaError_t launch_product(const ProductArgs & a, int C, size_t smem, cudaStream_t stream) {
    static PerDeviceOnce once;
    if (once.first()) {
        const cudaError_t e = cudaFuncSetAttribute(w4_product_kernel<MX, PARTS, GLU, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
        if (e != cudaSuccess) return e;
    }
    return launch_cluster(w4_product_kernel<MX, PARTS, GLU, MODE>, a.clusters * C, C, smem, stream, a);
}

template <bool MX, bool GLU>
cudaError_t launch_product_of(const ProductArgs & a, int parts, int C, size_t smem, cudaStream_t stream) {
    if (parts == 2) {
        if (a.T <= 4) return launch_product<MX, 2, GLU, PACK>(a, C, smem, stream);
        if (a.T <= 8) return launch_product<MX, 2, GLU, ONE>(a, C, smem, stream);
        return launch_product<MX, 2, GLU, TWO>(a, C, smem, stream);
    }
    if (a.T <= 8) return launch_product<MX, 1, GLU, ONE>(a, C, smem, stream);
    return launch_product<MX, 1, GLU, TWO>(a, C, smem, stream);
}

size_t type_bytes(uint32_t type) { return type == GGML_F32 ? 4 : 2; }

Act make_act(const void * p, int64_t ld, uint32_t type) {
    const size_t es = type_bytes(type);
    return {p, ld, type, (uintptr_t)p % (4 * es) == 0 && (ld * (int64_t)es) % (int64_t)(4 * es) == 0};
}

const void * row_at(const void * p, uint32_t type, int64_t ld, int64_t row) {
    return p ? static_cast<const uint8_t *>(p) + row * ld * (int64_t)type_bytes(type) : nullptr;
}

template <bool MX, int PARTS, int MODES> cudaError_t launch_gate_up(const MoeArgs & a, int C, size_t smem, cudaStream_t stream) {
    static PerDeviceOnce once;
    if (once.first()) {
        const cudaError_t e = cudaFuncSetAttribute(w4_moe_gate_up_kernel<MX, PARTS, MODES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
        if (e != cudaSuccess) return e;
    }
    return launch_cluster(w4_moe_gate_up_kernel<MX, PARTS, MODES>, a.clusters * C, C, smem, stream, a);
}

template <bool MX, int MODES> cudaError_t launch_down(const MoeArgs & a, int C, size_t smem, cudaStream_t stream) {
    static PerDeviceOnce once;
    if (once.first()) {
        const cudaError_t e = cudaFuncSetAttribute(w4_moe_down_kernel<MX, MODES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
        if (e != cudaSuccess) return e;
    }
    return launch_cluster(w4_moe_down_kernel<MX, MODES>, a.clusters * C, C, smem, stream, a);
}

// The kernels are built for the modes that calls of up to 4, 8 and 16 tokens reach.
template <bool MX> cudaError_t launch_gate_up_of(const MoeArgs & a, int parts, int C, size_t smem, cudaStream_t stream) {
    if (parts == 2) {
        if (a.T <= 4) return launch_gate_up<MX, 2, 1 << PACK>(a, C, smem, stream);
        if (a.T <= 8) return launch_gate_up<MX, 2, 1 << PACK | 1 << ONE>(a, C, smem, stream);
        return launch_gate_up<MX, 2, 1 << PACK | 1 << ONE | 1 << TWO>(a, C, smem, stream);
    }
    if (a.T <= 8) return launch_gate_up<MX, 1, 1 << ONE>(a, C, smem, stream);
    return launch_gate_up<MX, 1, 1 << ONE | 1 << TWO>(a, C, smem, stream);
}

template <bool MX> cudaError_t launch_down_of(const MoeArgs & a, int C, size_t smem, cudaStream_t stream) {
    if (a.T <= 4) return launch_down<MX, 1 << PACK>(a, C, smem, stream);
    if (a.T <= 8) return launch_down<MX, 1 << PACK | 1 << ONE>(a, C, smem, stream);
    return launch_down<MX, 1 << PACK | 1 << ONE | 1 << TWO>(a, C, smem, stream);
}

int64_t moe_ld_h(uint32_t ff) { return ((int64_t)ff + 3) / 4 * 4; }

} // namespace

size_t w4_bytes(uint32_t type, uint32_t n_out, uint32_t n_in, uint32_t n_expert) {
    return (size_t)n_expert * ((n_out + 15) / 16) * ((n_in + 63) / 64) * w4_unit_bytes(type == GGML_MXFP4);
}

W4View w4_view(const uint8_t * units, uint32_t type, uint32_t n_out, uint32_t n_in, uint32_t n_expert) {
    W4View v;
    v.units = units;
    v.type = type;
    v.n_out = n_out;
    v.n_in = n_in;
    v.n_expert = n_expert;
    v.tiles = (n_out + 15) / 16;
    v.steps = (n_in + 63) / 64;
    v.expert_bytes = (size_t)v.tiles * v.steps * w4_unit_bytes(type == GGML_MXFP4);
    return v;
}

void launch_w4_retile(const uint8_t * rows, uint32_t type, uint32_t n_out, uint32_t n_in, uint32_t n_expert, uint8_t * units, int * max_scale,
                      cudaStream_t stream) {
    const W4View v = w4_view(units, type, n_out, n_in, n_expert);
    const size_t n = (size_t)n_expert * v.tiles * v.steps;
    if (type == GGML_MXFP4) w4_retile_kernel<true><<<(unsigned)n, 128, 0, stream>>>(rows, n_out, n_in, v.tiles, v.steps, units, max_scale);
    else w4_retile_kernel<false><<<(unsigned)n, 128, 0, stream>>>(rows, n_out, n_in, v.tiles, v.steps, units, max_scale);
}

cudaError_t launch_w4_product(const W4Product & p, cudaStream_t stream) {
    const bool mx = p.w.type == GGML_MXFP4, glu = p.up != nullptr;
    const int parts = p.x_type == GGML_F32 || p.norm ? 2 : 1;
    const int sms = device_sms();
    const int jobs = glu ? (int)p.w.tiles : ((int)p.w.tiles + 1) / 2;
    const int steps = (int)p.w.steps;
    for (int t0 = 0, n = 0; t0 < p.n_tokens; t0 += n) {
        n = std::min(kW4PassTokens, p.n_tokens - t0);
        // the smallest cluster that fills the GPU, and whose share of the activations is small beside its share of the weights
        int C = 1;
        auto staged = [&](int c) { const int s = (steps + c - 1) / c; return staged_x_bytes(s, parts, n) + staged_c_bytes(mx, s, n); };
        while (C < 8 && 2 * C <= steps && ((int64_t)jobs * C < 2 * sms || (int64_t)n * sms * 8 > (int64_t)jobs * C * C * 4)) C *= 2;
        while (C < 8 && 2 * C <= steps && staged(C) > 96 * 1024) C *= 2;
        while (n > 1 && staged(C) > 160 * 1024) n = (n + 1) / 2;
        ProductArgs a{};
        a.w = p.w.units;
        a.u = glu ? p.up->units : nullptr;
        a.x = make_act(row_at(p.x, p.x_type, p.ld_x, t0), p.ld_x, p.x_type);
        a.T = n;
        a.n_in = (int)p.w.n_in;
        a.n_out = (int)p.w.n_out;
        a.tiles = (int)p.w.tiles;
        a.steps = steps;
        a.norm = p.norm;
        a.eps = p.eps;
        a.bias = p.bias;
        a.residual = row_at(p.residual, p.y_type, p.ld_residual, t0);
        a.ld_residual = p.ld_residual;
        a.y = const_cast<void *>(row_at(p.y, p.y_type, p.ld_y, t0));
        a.y_type = p.y_type;
        a.ld_y = p.ld_y;
        a.jobs = jobs;
        const int most = std::max(1, 2 * sms / C);
        const int per = (jobs + most - 1) / most;
        a.clusters = (jobs + per - 1) / per;
        const int s = (steps + C - 1) / C;
        a.x_bytes = (staged_x_bytes(s, parts, n) + 127) / 128 * 128;
        a.c_bytes = (staged_c_bytes(mx, s, n) + 127) / 128 * 128;
        a.jobs = jobs;
        const int slot = n * kSlotCol * 4;
        const int wanted = per * split_columns(per, steps / C);
        const int room = std::max(kWarps * slot, std::min(100 * 1024 - a.x_bytes - a.c_bytes, kMaxSmem - a.x_bytes - a.c_bytes));
        a.slots = std::max(1, std::min(wanted, room / slot));
        const size_t smem = (size_t)a.x_bytes + a.c_bytes + (size_t)a.slots * slot;
        cudaError_t e;
        if (mx) e = glu ? launch_product_of<true, true>(a, parts, C, smem, stream) : launch_product_of<true, false>(a, parts, C, smem, stream);
        else e = glu ? launch_product_of<false, true>(a, parts, C, smem, stream) : launch_product_of<false, false>(a, parts, C, smem, stream);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

size_t w4_moe_workspace_bytes(uint32_t ff, uint32_t n_tokens, uint32_t n_used) {
    const size_t pairs = (size_t)std::min<uint32_t>(n_tokens, kW4PassTokens) * n_used;
    return (sizeof(MoeMeta) + 255) / 256 * 256 + pairs * (size_t)moe_ld_h(ff) * 4;
}

cudaError_t launch_w4_moe(const W4Moe & p, cudaStream_t stream) {
    const bool mx = p.gate.type == GGML_MXFP4, mx_down = p.down.type == GGML_MXFP4;
    const int parts = p.x_type == GGML_F32 || p.norm ? 2 : 1;
    const int sms = device_sms();
    const int E = (int)p.gate.n_expert, d = (int)p.gate.n_in, ff = (int)p.gate.n_out;
    const int steps_d = (int)p.gate.steps, steps_ff = (int)p.down.steps;
    auto up_to = [](int x, int unit) { return (x + unit - 1) / unit * unit; };
    for (int t0 = 0, n = 0; t0 < p.n_tokens; t0 += n) {
        n = std::min(kW4PassTokens, p.n_tokens - t0);
        int C = 8;
        while (C > steps_d) C /= 2;
        auto staged = [&] { const int s = (steps_d + C - 1) / C; return staged_x_bytes(s, parts, n) + staged_c_bytes(mx, s, n); };
        while (n > 1 && staged() > 120 * 1024) n = (n + 1) / 2;
        MoeArgs a{};
        a.gate = p.gate.units;
        a.up = p.up.units;
        a.down = p.down.units;
        a.gate_expert = p.gate.expert_bytes;
        a.up_expert = p.up.expert_bytes;
        a.down_expert = p.down.expert_bytes;
        a.router = p.router;
        a.x = make_act(row_at(p.x, p.x_type, p.ld_x, t0), p.ld_x, p.x_type);
        a.T = n;
        a.E = E;
        a.k = p.n_used;
        a.d = d;
        a.ff = ff;
        a.tiles_ff = (int)p.gate.tiles;
        a.steps_d = steps_d;
        a.tiles_d = (int)p.down.tiles;
        a.steps_ff = steps_ff;
        a.normalise = p.normalise;
        a.norm = p.norm;
        a.eps = p.eps;
        a.residual = row_at(p.residual, p.y_type, p.ld_residual, t0);
        a.ld_residual = p.ld_residual;
        a.y = const_cast<void *>(row_at(p.y, p.y_type, p.ld_y, t0));
        a.y_type = p.y_type;
        a.ld_y = p.ld_y;
        a.ids = p.ids ? p.ids + (size_t)t0 * p.n_used : nullptr;
        a.weights = p.weights ? p.weights + (size_t)t0 * p.n_used : nullptr;
        a.meta = static_cast<MoeMeta *>(p.workspace);
        a.h = reinterpret_cast<float *>(static_cast<uint8_t *>(p.workspace) + (sizeof(MoeMeta) + 255) / 256 * 256);
        a.ld_h = moe_ld_h((uint32_t)ff);

        // first kernel: at most `reach` experts are chosen
        const int reach = std::min(E, n * p.n_used);
        const int s = (steps_d + C - 1) / C;
        a.x_bytes = up_to(staged_x_bytes(s, parts, n), 128);
        a.c_bytes = up_to(staged_c_bytes(mx, s, n), 128);
        a.logit_bytes = up_to(n * E * 4, 128);
        a.clusters = std::max(1, (int)std::min<int64_t>(2 * sms / C, (int64_t)reach * a.tiles_ff));
        const int fixed = a.x_bytes + a.c_bytes + 2 * a.logit_bytes;
        a.partial_floats = std::max(kWarps * n * kSlotCol, (88 * 1024 - fixed) / 4);
        cudaError_t e = mx ? launch_gate_up_of<true>(a, parts, C, (size_t)fixed + a.partial_floats * 4, stream)
                           : launch_gate_up_of<false>(a, parts, C, (size_t)fixed + a.partial_floats * 4, stream);
        if (e != cudaSuccess) return e;

        // second kernel
        C = 8;
        while (C > steps_ff * p.n_used) C /= 2;
        const int jobs = (a.tiles_d + 1) / 2;
        const int most = std::max(1, 2 * sms / C), per = (jobs + most - 1) / most;
        a.clusters = (jobs + per - 1) / per;
        a.x_bytes = 64 * 1024;
        a.c_bytes = a.logit_bytes = 0;
        a.partial_floats = std::max(kWarps * n * kSlotCol, std::min(per * kWarps * n * kSlotCol, (100 * 1024 - a.x_bytes) / 4));
        e = mx_down ? launch_down_of<true>(a, C, (size_t)a.x_bytes + a.partial_floats * 4, stream)
                    : launch_down_of<false>(a, C, (size_t)a.x_bytes + a.partial_floats * 4, stream);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

} // namespace rb200
