// Products with 4-bit weights for at most sixteen tokens, bound by the weight stream.
//
// Mathematics. 16 rows x 64 columns are the A operands of four m16n8k16 products; the tokens are the columns
// of B. The weights enter as exact f16 values that cost no arithmetic beyond masks and shifts:
//   Q4_0   the nibble q in the low bits of an f16 is the subnormal q 2^-24, in the next four bits 16 q 2^-24; the
//          columns whose nibbles sit there get their activations divided by 16. The offset is the product chain's start
//          value, -8 2^-24 times the group's sum of activations.
//   MXFP4  sign and e2m1 magnitude placed at an f16's sign bit and bits 9..11 are the value times 2^-14.
// A token's activations are scaled by a power of two that brings the largest of them into [2^13, 2^14) and split into
// hi + lo f16 (22 bits); activations that are f16 or bf16 themselves need no lo. A 32-column group is exactly two
// products, so its f32 sum comes out on its own, is multiplied by the group's scale and added in f32.
//
// Split. A cluster of up to eight CTAs owns a range of row blocks (32 rows); each CTA takes a range of the columns for all of them, so
// it converts only its share of the activations. Its warps take (row block, part of the CTA's columns) runs, and
// write every (row block, token)'s sums into the shared memory of the CTA that owns it, which adds them in a fixed order after one
// cluster barrier (no workspace, no atomics: results are the same in every run) and applies bias, residual or the gate's
// activation. Every warp streams its units through a ring of its own in shared memory by asynchronous copies, three or five units
// ahead, so that no registers are held by loads in flight and three CTAs fit on an SM.

#include "kernels.cuh"
#include "blocks.hpp"
#include "w4.cuh"

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cuda_bf16.h>

namespace rb200 {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kSlotCol = 36;        // floats per (partial slot, token): 32 rows, padded so that a warp's stores meet no bank twice
constexpr int kMaxSegs = 16;
constexpr int kMaxCluster = 8;
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

__device__ __forceinline__ void scale4(float (&v)[4], const float * by) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= by[e];
}

__device__ __forceinline__ void store1(void * p, uint32_t type, int64_t i, float v) {
    if (type == GGML_F32) static_cast<float *>(p)[i] = v;
    else if (type == GGML_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// ---- cluster

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t smem_address(const void * p) { return (uint32_t)__cvta_generic_to_shared(p); }
// The address of `at` (this CTA's shared memory) in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t remote_address(uint32_t at, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at), "r"(rank));
    return a;
}
__device__ __forceinline__ float remote_load(uint32_t address) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ void remote_store(uint32_t address, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(address), "f"(v) : "memory");
}
// The CTAs of a cluster have started: required before the first access to another's shared memory. Arrive early, wait late.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
}

// ---- weights

// The lane's share of a unit: A words and scales of its two row tiles.
template <bool MX> struct Unit {
    uint4 q[2];
    uint2 s[2];     // MXFP4 uses .x only
};

// Units in a warp's ring; fewer beside the activations of many tokens.
__host__ __device__ constexpr int stages_for(int n) { return n > 4 ? 4 : 6; }
__host__ __device__ constexpr int ring_bytes(bool mx, int n) { return kWarps * stages_for(n) * (int)w4_unit_bytes(mx); }

__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t * src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 shared_u4(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ uint2 shared_u2(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}
__device__ __forceinline__ uint32_t shared_u1(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}

template <bool MX> __device__ __forceinline__ void read_unit(uint32_t words, uint32_t scales, Unit<MX> & u) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        u.q[i] = shared_u4(words + i * 512);
        if constexpr (MX) u.s[i].x = shared_u1(scales + i * 32);
        else u.s[i] = shared_u2(scales + i * 64);
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

// c = a b + (s0, s1, s0, s1), and c += a b.
__device__ __forceinline__ void mma_start(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float s0, float s1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};\n"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(s0), "f"(s1));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// How many tokens a product chain serves. PACK: up to four, MMA column c is token c's hi part and column c + 4 its lo part.
enum Mode { PACK = 0, ONE = 1, TWO = 2 };
__host__ __device__ constexpr int mode_of(int n, int parts) { return n > 8 ? TWO : parts == 2 && n <= 4 ? PACK : ONE; }

// ---- activations in shared memory
//
// x   [step][group][part][NT tokens][32] f16, then (Q4_0) c [step][group][NT tokens] f32: the start values of the group's products. NT,
// the tokens there is room for, is a template argument wherever they are read, so that the offsets inside a step are immediates.
__host__ __device__ constexpr int step_x_bytes(int parts, int nt) { return 2 * parts * nt * 64; }
__host__ __device__ constexpr int step_c_bytes(bool mx, int nt) { return mx ? 0 : 2 * nt * 4; }
__host__ __device__ constexpr int step_bytes(bool mx, int parts, int nt) { return step_x_bytes(parts, nt) + step_c_bytes(mx, nt); }
struct Staged {
    uint8_t * x;
    float * c;
};

struct Scratch {
    float f1[kMaxSegs][kRowList], f2[kMaxSegs][kRowList];   // a token's sums times f1 times f2 are in the activations' own scale
    float ss[kMaxCluster][kRowList];                        // sums of squares of each CTA's columns
    uint32_t top[kWarps];
    float squares[kWarps];
    uint64_t zero;                                          // start values of PACK's lo columns
};

// One token's row of activations, or the part of it a CTA needs, and where it goes.
struct StageRow {
    int64_t row;
    int k0, steps;              // columns k0 .. k0 + 64 steps - 1; those at and behind n_in are zero
    int nt, place;              // room of the token set, the token's place in it
    int seg;                    // row of Scratch::f1, f2
    Staged out;
};

template <bool MX, int PARTS> __device__ __forceinline__ void stage_chunk(const StageRow & r, int i, float (&v)[4], float up) {
    const int step = i >> 4, group = (i >> 3) & 1, at = (i & 7) * 4;
    const bool inside = i < r.steps * 16;
    const float factor = !MX && group ? up * 0.0625f : up;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= factor;
    if constexpr (!MX) {
        float sum = (v[0] + v[1]) + (v[2] + v[3]);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (inside && (threadIdx.x & 7) == 0) r.out.c[(step * 2 + group) * r.nt + r.place] = sum * (group ? -128.f : -8.f) * 5.9604644775390625e-8f;
    }
    if (inside) {
        const __half2 h0 = __floats2half2_rn(v[0], v[1]), h1 = __floats2half2_rn(v[2], v[3]);
        uint8_t * dst = r.out.x + ((step * 2 + group) * PARTS * r.nt + r.place) * 64 + at * 2;
        *reinterpret_cast<uint2 *>(dst) = make_uint2(*reinterpret_cast<const uint32_t *>(&h0), *reinterpret_cast<const uint32_t *>(&h1));
        if constexpr (PARTS == 2) {
            const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
            const __half2 l0 = __floats2half2_rn(v[0] - f0.x, v[1] - f0.y), l1 = __floats2half2_rn(v[2] - f1.x, v[3] - f1.y);
            *reinterpret_cast<uint2 *>(dst + r.nt * 64) = make_uint2(*reinterpret_cast<const uint32_t *>(&l0), *reinterpret_cast<const uint32_t *>(&l1));
        }
    }
}

// Converts n rows; row_of(i) describes them. Each is one warp's work, or with few rows that of several warps. NORM: rows
// are multiplied by `norm`, and put_squares(row, sum) gets the row's sum of squares. Every thread takes part; a barrier follows at the caller's.
template <bool MX, int PARTS, bool NORM, class RowOf, class PutSquares>
__device__ void stage_rows(const Act & act, int n, int n_in, const float * norm, Scratch & sc, RowOf row_of, PutSquares put_squares) {
    constexpr int kHeld = 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int shared = n > 4 ? 1 : n > 2 ? 2 : n > 1 ? 4 : 8;      // warps that share a row
    const int part = warp % shared;
    for (int i0 = warp / shared; i0 < n || shared > 1; i0 += kWarps / shared) {
        const bool live = i0 < n;
        const StageRow r = row_of(live ? i0 : 0);
        const int count = live ? min(r.steps * 16, (n_in - r.k0) / 4) : 0;     // chunks of four columns that exist, whole groups
        const int trips = live ? (r.steps * 16 + shared * 32 - 1) / (shared * 32) : 0;
        const int first = part * 32 + lane;
        // the largest magnitude as bits: a NaN is above infinity, infinity above every number
        uint32_t top = 0;
        float squares = 0.f;
        float held[kHeld][4];
        // loads of kHeld chunks are in flight together; a row that is no longer than them is read once
        auto load = [&](int it0) {
#pragma unroll
            for (int it = 0; it < kHeld; ++it) {
                const int i = first + (it0 + it) * shared * 32;
                held[it][0] = held[it][1] = held[it][2] = held[it][3] = 0.f;
                if (it0 + it < trips && i < count) load4(act, r.row, r.k0 + 4 * i, held[it]);
            }
        };
        auto weigh = [&](int it0) {
            if constexpr (NORM) {
#pragma unroll
                for (int it = 0; it < kHeld; ++it) {
                    const int i = first + (it0 + it) * shared * 32;
                    if (it0 + it < trips && i < count) scale4(held[it], norm + r.k0 + 4 * i);
                }
            }
        };
        for (int it0 = 0; it0 < trips; it0 += kHeld) {
            load(it0);
            if constexpr (NORM) {
#pragma unroll
                for (int it = 0; it < kHeld; ++it)
#pragma unroll
                    for (int e = 0; e < 4; ++e) squares += held[it][e] * held[it][e];
            }
            weigh(it0);
#pragma unroll
            for (int it = 0; it < kHeld; ++it)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(held[it][e]) & 0x7fffffffu);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if constexpr (NORM) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
        }
        if (shared > 1) {
            if (lane == 0) { sc.top[warp] = top; sc.squares[warp] = squares; }
            __syncthreads();
            top = 0;
            squares = 0.f;
            for (int i = 0; i < shared; ++i) { top = max(top, sc.top[warp - part + i]); squares += sc.squares[warp - part + i]; }
        }
        // 2^shift brings the largest magnitude into [2^13, 2^14), as far as it is an f32 itself (below 2^-113 the values only
        // come near). A row with an infinity or a NaN is left as it is: its own sums become NaN, those of the other tokens
        // stay what they are.
        const int shift = top > 0 && top < 0x7f800000u ? min(126, 13 - ((int)(top >> 23) - 127)) : 0;
        const float up = __uint_as_float((uint32_t)(shift + 127) << 23);
        if (live && part == 0 && lane == 0) {
            const int down = (MX ? 6 : 24) - shift;
            sc.f1[r.seg][r.place] = __uint_as_float((uint32_t)(down / 2 + 127) << 23);
            sc.f2[r.seg][r.place] = __uint_as_float((uint32_t)(down - down / 2 + 127) << 23);
            if constexpr (NORM) put_squares(i0, squares);
        }
        for (int it0 = 0; it0 < trips; it0 += kHeld) {
            if (trips > kHeld) {
                load(it0);
                weigh(it0);
            }
#pragma unroll
            for (int it = 0; it < kHeld; ++it) if (it0 + it < trips) stage_chunk<MX, PARTS>(r, first + (it0 + it) * shared * 32, held[it], up);
        }
        if (shared > 1) break;      // that many warps share a row only when one round holds all rows
    }
}

// The rows of a call's tokens, normalised by its weights when it has any. A row's squares go to every CTA of the cluster.
template <bool MX, int PARTS>
__device__ __forceinline__ void stage_tokens(const Act & act, int n, int nt, int s0, int steps, int n_in, const float * norm, const Staged & out, Scratch & sc,
                                             int rank, int C) {
    auto row_of = [&](int t) { return StageRow{(int64_t)t, s0 * 64, steps, nt, t, 0, out}; };
    if (norm) {
        cluster_wait();
        stage_rows<MX, PARTS, true>(act, n, n_in, norm, sc, row_of, [&](int t, float squares) {
            for (int c = 0; c < C; ++c) remote_store(remote_address(smem_address(&sc.ss[rank][t]), c), squares);
        });
    } else {
        stage_rows<MX, PARTS, false>(act, n, n_in, nullptr, sc, row_of, [](int, float) {});
        cluster_wait();
    }
}

// 1 / sqrt(mean of squares + eps) of token t, once the cluster has met after stage_tokens.
__device__ __forceinline__ float rms_factor(const Scratch & sc, int t, int C, int n_in, float eps) {
    float ss = 0.f;
    for (int c = 0; c < C; ++c) ss += sc.ss[c][t];
    return rsqrtf(ss / (float)n_in + eps);
}

// ---- the product chain

// A warp works through runs: the units of a row block against one set of tokens. Consecutive runs with the same tokens and
// columns are a group. What a group needs of the activations:
struct Group {
    Staged x;                   // from the group's first step on
    const uint8_t * list;       // token (place in x) of each MMA column; unused where the places are the columns
    int n;                      // how many
    int seg;                    // row of Scratch::f1, f2
};

// Where a lane finds its B fragments and start values, and the factors of its columns' sums.
struct Lane {
    uint32_t b[2], c[2][2];             // shared-memory addresses at the group's first step
    uint32_t c_step;
    float f1[2][2], f2[2][2];
};

template <bool MX, int PARTS, int MODE, int NT, bool LIST>
__device__ __forceinline__ void begin_group(const Group & r, int lane, const Scratch & sc, Lane & l) {
    constexpr int NC = MODE == TWO ? 2 : 1;
    const int g = lane >> 2, t4 = lane & 3;
    const bool lo = MODE == PACK;
    const uint32_t x = smem_address(r.x.x), c = MX ? 0 : smem_address(r.x.c);
    auto place = [&](int col) { const int i = min(col, r.n - 1); return LIST ? (int)r.list[i] : i; };
    l.b[0] = x + place(lo ? g & 3 : g) * 64 + t4 * 16 + (lo && g >= 4 ? NT * 64 : 0);
    if constexpr (NC == 2) l.b[1] = x + place(g + 8) * 64 + t4 * 16;
    l.c_step = step_c_bytes(MX, NT);
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int tok = place(lo ? (2 * t4 + e) & 3 : 8 * nc + 2 * t4 + e);
            if constexpr (!MX) l.c[nc][e] = c + tok * 4;
            l.f1[nc][e] = sc.f1[r.seg][tok];
            l.f2[nc][e] = sc.f2[r.seg][tok];
        }
    if constexpr (!MX && lo) {
        if (t4 >= 2) {
            l.c[0][0] = l.c[0][1] = smem_address(&sc.zero);
            l.c_step = 0;
        }
    }
}

// One unit. NT == 1: every MMA column is the one token, and only the even ones are kept.
template <bool MX, int PARTS, int MODE, int NT, bool LIST>
__device__ __forceinline__ void do_step(uint32_t words, uint32_t scale_at, uint32_t b_at, uint32_t c_at, const Lane & l, float (&acc)[2][2][4]) {
    constexpr int NC = MODE == TWO ? 2 : 1;
    constexpr int NP = MODE == PACK ? 1 : PARTS;
    Unit<MX> u;
    read_unit<MX>(words, scale_at, u);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint4 b[NC][NP];
        float start[NC][2];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
#pragma unroll
            for (int p = 0; p < NP; ++p) b[nc][p] = shared_u4(l.b[nc] + b_at + (h * PARTS + p) * (NT * 64));
            start[nc][0] = start[nc][1] = 0.f;
            if constexpr (!MX) {
                const int c_group = MODE == PACK ? 0 : h * NT * 4;      // PACK: the zero has no groups, so h is part of c_at there
                const uint32_t hh = MODE == PACK ? h * (l.c_step >> 1) : 0;
                start[nc][0] = __uint_as_float(shared_u1(l.c[nc][0] + c_at + c_group + hh));
                start[nc][1] = NT == 1 ? start[nc][0] : __uint_as_float(shared_u1(l.c[nc][1] + c_at + c_group + hh));
            }
        }
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
            float c[NC][4];
            uint32_t a[4];
            if (h == 0) decode<MX, 0, 0>(u.q[tile], a); else decode<MX, 1, 0>(u.q[tile], a);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) {
                mma_start(c[nc], a, b[nc][0].x, b[nc][0].y, start[nc][0], start[nc][1]);
                if constexpr (NP == 2) mma(c[nc], a, b[nc][NP - 1].x, b[nc][NP - 1].y);
            }
            if (h == 0) decode<MX, 0, 1>(u.q[tile], a); else decode<MX, 1, 1>(u.q[tile], a);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc)
#pragma unroll
                for (int p = 0; p < NP; ++p) mma(c[nc], a, b[nc][p].z, b[nc][p].w);
            float d0, d1;
            if (h == 0) scales<MX, 0>(u.s[tile], d0, d1); else scales<MX, 1>(u.s[tile], d0, d1);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) {
                acc[tile][nc][0] += d0 * c[nc][0];
                acc[tile][nc][2] += d1 * c[nc][2];
                if constexpr (NT > 1) {
                    acc[tile][nc][1] += d0 * c[nc][1];
                    acc[tile][nc][3] += d1 * c[nc][3];
                }
            }
        }
    }
}

// Hands a run's sums to put(row 0..31 of the block, column, sum) and clears them.
template <int MODE, int NT, class Put>
__device__ __forceinline__ void end_run(int n, int lane, const Lane & l, float (&acc)[2][2][4], Put put) {
    const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int tile = 0; tile < 2; ++tile)
#pragma unroll
        for (int nc = 0; nc < (MODE == TWO ? 2 : 1); ++nc)
#pragma unroll
            for (int i = 0; i < 4; i += NT > 1 ? 1 : 2) {
                float v = acc[tile][nc][i];
                if constexpr (MODE == PACK) v += __shfl_xor_sync(0xffffffffu, v, 2);      // hi column + lo column
                const int col = 8 * nc + 2 * t4 + (i & 1);
                if (col < n && !(MODE == PACK && t4 >= 2)) put(tile * 16 + g + (i >> 1) * 8, col, v * l.f1[nc][i & 1] * l.f2[nc][i & 1]);
                acc[tile][nc][i] = 0.f;
            }
}

// Where a warp is in its sequence of runs.
struct Cursor {
    const uint8_t * p;          // the next unit
    int rem;                    // units left in the run
    int group, job;             // the Source's
    bool live;
};

// Runs a warp's sequence. Source: first(Cursor &) and next(Cursor &) move to a run (never an empty one) and set everything;
// group(const Cursor &) describes the activations; put(const Cursor &, row, column, sum) takes the sums.
template <bool MX, int STAGES, class Source> struct Stream {
    const Source & src;
    const int lane;
    const uint32_t ring;
    Cursor ld, cp;
    uint32_t fill, at;          // ring offsets of the stage to fill and the stage to multiply

    __device__ __forceinline__ Stream(const Source & s, uint8_t * rings)
        : src(s), lane(threadIdx.x & 31), ring(smem_address(rings) + (threadIdx.x >> 5) * (STAGES * w4_unit_bytes(MX))), fill(0), at(0) {
        src.first(ld);
        cp = ld;
    }
    __device__ __forceinline__ void fetch() {
        if (ld.live) {
            const uint32_t dst = ring + fill + lane * 16;
            const uint8_t * p = ld.p + lane * 16;
            copy16(dst, p);
            copy16(dst + 512, p + 512);
            if (lane < (MX ? 4 : 8)) copy16(dst + 1024, p + 1024);
            ld.p += w4_unit_bytes(MX);
            if (--ld.rem == 0) src.next(ld);
        }
        fill = fill == (STAGES - 1) * w4_unit_bytes(MX) ? 0 : fill + w4_unit_bytes(MX);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // The first units of the sequence; needs nothing but the weights. The ring must be free: a barrier lies between its last reads and this.
    __device__ __forceinline__ void prefetch() {
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) fetch();
    }
    // All runs of the cursor's group whose job is below `limit`.
    template <int PARTS, int MODE, int NT, bool LIST> __device__ __forceinline__ void work_group(const Group & r, const Scratch & sc, int limit = 0x7fffffff) {
        float acc[2][2][4] = {};
        Lane l;
        begin_group<MX, PARTS, MODE, NT, LIST>(r, lane, sc, l);
        const int group = cp.group;
        const uint32_t words = ring + lane * 16, scale_at = ring + 1024 + (lane >> 2) * (MX ? 4 : 8);
        do {
            uint32_t b_at = 0, c_at = 0;
            for (int n = cp.rem; n > 0; --n) {
                asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
                __syncwarp();           // every lane's copies of this unit have landed, and the stage read last is free
                fetch();
                do_step<MX, PARTS, MODE, NT, LIST>(words + at, scale_at + at, b_at, c_at, l, acc);
                at = at == (STAGES - 1) * w4_unit_bytes(MX) ? 0 : at + w4_unit_bytes(MX);
                b_at += step_x_bytes(PARTS, NT);
                c_at += l.c_step;
            }
            end_run<MODE, NT>(r.n, lane, l, acc, [&](int row, int col, float v) { src.put(cp, row, col, v); });
            src.next(cp);
        } while (cp.live && cp.group == group && cp.job < limit);
    }
    // The runs of jobs below `limit`. Token sets staged with room for NT tokens, whose groups hold up to `NT` of them.
    template <int PARTS, int NT, bool LIST> __device__ __forceinline__ void work(const Scratch & sc, int limit) {
        while (cp.live && cp.job < limit) {
            const Group r = src.group(cp);
            if constexpr (!LIST) work_group<PARTS, mode_of(NT, PARTS), NT, LIST>(r, sc, limit);
            else {
                const int mode = mode_of(r.n, PARTS);
                if (PARTS == 2 && mode == PACK) work_group<PARTS, PARTS == 2 ? PACK : ONE, NT, LIST>(r, sc, limit);
                if constexpr (NT > (PARTS == 2 ? 4 : 0)) if (mode == ONE) work_group<PARTS, ONE, NT, LIST>(r, sc, limit);
                if constexpr (NT > 8) if (mode == TWO) work_group<PARTS, TWO, NT, LIST>(r, sc, limit);
            }
        }
    }
    // Token sets staged with room for 1, 2, 4, 8 or 16, whichever holds them; none above MOST.
    template <int PARTS, int MOST> __device__ __forceinline__ void work_sized(const Scratch & sc) {
        while (cp.live) {
            const Group r = src.group(cp);
            if (r.n == 1) work_group<PARTS, mode_of(1, PARTS), 1, false>(r, sc);
            if constexpr (MOST > 1) if (r.n == 2) work_group<PARTS, mode_of(2, PARTS), 2, false>(r, sc);
            if constexpr (MOST > 2) if (r.n > 2 && r.n <= 4) work_group<PARTS, mode_of(4, PARTS), 4, false>(r, sc);
            if constexpr (MOST > 4) if (r.n > 4 && r.n <= 8) work_group<PARTS, mode_of(8, PARTS), 8, false>(r, sc);
            if constexpr (MOST > 8) if (r.n > 8) work_group<PARTS, mode_of(16, PARTS), 16, false>(r, sc);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
};

// Room a set of n tokens is staged with.
__host__ __device__ constexpr int room_for(int n) { return n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : n <= 8 ? 8 : 16; }

// Parts (a power of two) the warps split the columns of a job into: as few as keep the warps evenly loaded, and at most `most`.
// Warp w takes part w % ks of jobs w / ks, w / ks + kWarps / ks, ... The cost counts steps of the busiest warp and two steps' time
// for every partial sum it writes.
__host__ __device__ inline int split_columns(int jobs, int steps, int most) {
    int best = 1, best_cost = 0x7fffffff;
    for (int ks = 1; ks <= kWarps && ks <= most; ks *= 2) {
        if (ks > 1 && ks > steps) break;
        const int rounds = (jobs * ks + kWarps - 1) / kWarps;
        const int cost = rounds * ((steps + ks - 1) / ks + 2);
        if (cost < best_cost) { best_cost = cost; best = ks; }
    }
    return best;
}

// Range `part` of `parts` nearly equal ranges of [0, n).
__host__ __device__ inline int part_begin(int n, int part, int parts) {
    const unsigned each = (unsigned)n / (unsigned)parts, more = (unsigned)n - each * parts;
    return (int)(part * each + min((unsigned)part, more));
}

// The same for 2^log_parts parts.
__device__ __forceinline__ int part_begin2(int n, int part, int log_parts) {
    return part * (n >> log_parts) + min(part, n & ((1 << log_parts) - 1));
}

// ---- y = W x, and y = silu(W x) * (U x)

// The inbox of a CTA: for each (row block, token) it owns, the sums of 32 rows from every (CTA, part of the columns) of the
// cluster; with the gate, of gate and of up. Unit u of a round, block * tokens + token, belongs to CTA u % C. Rounds use two
// inboxes in turn: whoever writes round r + 2's has met everyone after they read round r's.
struct Inbox {
    uint32_t base;              // shared-memory address
    int bytes;                  // of one of the two
    int rank, log_c, ks, per;   // per: matrices of a block

    __device__ __forceinline__ void put(int round, int unit, int which, int sub, int row, float v) const {
        const int from = (((unit >> log_c) * per + which) << log_c | rank) * ks + sub;
        remote_store(remote_address(base + (round & 1) * bytes + (from * 32 + row) * 4, unit & ((1 << log_c) - 1)), v);
    }
    // Row `lane` of the sum over the cluster for the CTA's own unit number `mine`, in the order of the columns.
    __device__ __forceinline__ float sum(int round, int mine, int which) const {
        const int n = ks << log_c;
        const uint32_t at = base + (round & 1) * bytes + ((mine * per + which) * n * 32 + (threadIdx.x & 31)) * 4;
        float v = 0.f;
#pragma unroll 8
        for (int i = 0; i < n; ++i) v += __uint_as_float(shared_u1(at + i * 128));
        return v;
    }
};
// Bytes of one inbox for `units` units of a round.
__host__ __device__ inline int64_t inbox_bytes(int64_t units, int C, int ks, int per) { return (units + C - 1) / C * per * C * ks * 128; }
// Row blocks a round can take with `room` bytes for one inbox; at least one.
__host__ __device__ inline int blocks_per_round(int room, int tokens, int C, int ks, int per) {
    const int units = room / (per * C * ks * 128) * C;      // whole units in every CTA
    return max(1, units / tokens);
}

struct ProductArgs {
    const uint8_t * w, * u;
    Act x;
    int T, n_in, n_out, steps;
    const float * norm;
    float eps;
    const float * bias;
    const void * residual;
    int64_t ld_residual;
    void * y;
    uint32_t y_type;
    int64_t ld_y;
    int each, more, clusters;       // row blocks of a cluster (one more in the first `more`), of gate and up together as of one matrix
    int x_bytes, c_bytes, inbox;    // shared memory: staged activations, start values, one inbox
    int ks, per_round;              // parts of the columns and blocks of a round, the same in every cluster: one inbox may have to do
};

// Jobs: a row block; with the gate, block j of gate and of up are jobs 2 j and 2 j + 1.
template <bool MX, int PARTS, bool GLU, int NT> struct ProductSource {
    const ProductArgs & a;
    Staged x;                   // from this warp's columns on
    Inbox inbox;
    int job0, jobs, ks;         // jobs job0 .. job0 + jobs - 1
    int sub, step, len;         // this warp's columns
    int round, round0;          // the round, and its first job

    __device__ __forceinline__ void point(Cursor & c) const {
        c.live = c.job < jobs;
        const int job = job0 + c.job;
        const size_t block = GLU ? job >> 1 : job;
        c.p = (GLU && (job & 1) ? a.u : a.w) + (block * a.steps + step) * w4_unit_bytes(MX);
        c.rem = len;
    }
    __device__ __forceinline__ void first(Cursor & c) const {
        c.group = 0;
        c.job = (threadIdx.x >> 5) >> (__ffs(ks) - 1);
        point(c);
    }
    __device__ __forceinline__ void next(Cursor & c) const {
        c.job += kWarps >> (__ffs(ks) - 1);
        point(c);
    }
    __device__ __forceinline__ Group group(const Cursor &) const { return {x, nullptr, a.T, 0}; }
    __device__ __forceinline__ void put(const Cursor & c, int row, int col, float v) const {
        const int job = c.job - round0;
        inbox.put(round, (GLU ? job >> 1 : job) * a.T + col, GLU ? job & 1 : 0, sub, row, v);
    }
};

template <bool MX, int PARTS, bool GLU, int NT>
__global__ void __launch_bounds__(kThreads, NT > 8 ? 2 : 3) w4_product_kernel(ProductArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Scratch sc;
    constexpr int kPer = GLU ? 2 : 1;           // jobs of a row block
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), C = (int)cluster_size();
    const int cluster = blockIdx.x / C;
    cluster_arrive();
    const int log_c = __ffs(C) - 1;
    const int s0 = part_begin2(a.steps, rank, log_c), n_steps = part_begin2(a.steps, rank + 1, log_c) - s0;
    const int b_begin = cluster * a.each + min(cluster, a.more), blocks = a.each + (cluster < a.more);
    const int ks = a.ks, log_ks = __ffs(ks) - 1;
    const int per_round = a.per_round;
    uint8_t * const rings = smem + a.x_bytes + a.c_bytes;
    const Staged x{smem, reinterpret_cast<float *>(smem + a.x_bytes)};
    const Inbox inbox{smem_address(rings + ring_bytes(MX, NT)), a.inbox, rank, log_c, ks, kPer};
    const int sub = warp & (ks - 1), step = part_begin2(n_steps, sub, log_ks), len = part_begin2(n_steps, sub + 1, log_ks) - step;
    const Staged x_warp{x.x + step * step_x_bytes(PARTS, NT), x.c + step * step_c_bytes(MX, NT) / 4};
    if (threadIdx.x == 0) sc.zero = 0;

    ProductSource<MX, PARTS, GLU, NT> src{a, x_warp, inbox, b_begin * kPer, blocks * kPer, ks, sub, s0 + step, len, 0, 0};
    Stream<MX, stages_for(NT), ProductSource<MX, PARTS, GLU, NT>> stream(src, rings);
    stream.prefetch();
    // the weights above are the library's own; everything below is the caller's
    pdl_trigger();
    pdl_wait();
    stage_tokens<MX, PARTS>(a.x, a.T, NT, s0, n_steps, a.n_in, a.norm, x, sc, rank, C);
    __syncthreads();
    for (int b0 = 0; b0 < blocks; b0 += per_round, ++src.round) {
        const int now = min(per_round, blocks - b0);
        src.round0 = b0 * kPer;
        stream.template work<PARTS, NT, false>(sc, (b0 + now) * kPer);
        cluster_sync();
        // 32 rows of one token at a time
        for (int i = warp; i * C + rank < now * a.T; i += kWarps) {
            const int unit = i * C + rank, b = unit / a.T, t = unit - b * a.T;
            float v = inbox.sum(src.round, i, 0);
            const float factor = a.norm ? rms_factor(sc, t, C, a.n_in, a.eps) : 1.f;
            v *= factor;
            if constexpr (GLU) v = v / (1.f + expf(-v)) * (inbox.sum(src.round, i, 1) * factor);
            const int row = (b_begin + b0 + b) * 32 + lane;
            if (row < a.n_out) {
                if (a.bias) v += a.bias[row];
                if (a.residual) v += load1(Act{a.residual, a.ld_residual, a.y_type, false}, t, row);
                store1(a.y, a.y_type, t * a.ld_y + row, v);
            }
        }
    }
}

// ---- a mixture-of-experts layer
//
// Two kernels. The first: every cluster normalises and routes all tokens for itself (the router is a few hundred
// kilobytes that the L2 cache holds; one CTA reads an eighth of it) instead of waiting for one place to do it, then multiplies its share of the chosen
// experts' (gate tile, up tile) pairs and writes h = w_e silu(a) b for each (token, expert) pair. The second treats the chosen
// experts' down matrices as one long reduction: a cluster owns a range of y's rows, its CTAs divide the experts' concatenated columns,
// and the sum over experts is part of the sum over the cluster.

struct alignas(16) MoeMeta {                     // in the workspace, in front of h
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
    bool router_vec;            // sixteen bytes of it may be read at once
    Act x;
    int T, E, k, d, ff;
    int blocks_ff, steps_d, blocks_d, steps_ff;
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
    int clusters, x_bytes, c_bytes, logit_bytes, inbox, partial;        // shared memory, in bytes
};

struct Picks {
    uint16_t expert[kRowList * kW4MaxUsed];
    float weight[kRowList * kW4MaxUsed];
    float rstd[kRowList];
    uint16_t unique[kW4MaxExperts];
    uint8_t count[kW4MaxExperts];                   // of unique[i]
    uint8_t token[kW4MaxExperts][kRowList];
    uint32_t mask[kW4MaxExperts];                   // by expert: the tokens that chose it
    uint8_t rank[kW4MaxExperts][kRowList];          // of the expert among the token's
    int warp_unique[kWarps], warp_most[kWarps];
    int n, most;                                    // unique experts, largest count
};

// Sums each of the 16 values of a lane over the warp; lane i ends up with value i >> 1 (lanes 2 i and 2 i + 1 alike).
__device__ __forceinline__ float warp_sums16(float (&v)[16]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int half = 8; half > 0; half >>= 1) {
        const bool upper = lane & (2 * half);
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float send = upper ? v[i] : v[i + half], keep = upper ? v[i + half] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, 2 * half);
        }
    }
    return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1);
}

// Columns of the router that fit into `room` bytes for all experts: whole groups of 32.
__device__ __forceinline__ int router_columns(int E, int room) { return room / (E * 128) * 32; }

// Copies columns [k, k + n) of all router rows to shared memory, row e at e * n. The caller commits, waits and synchronises.
__device__ __forceinline__ void fetch_router(const MoeArgs & a, int k, int n, uint8_t * to) {
    const uint32_t dst = smem_address(to);
    if (a.router_vec) {
        const int chunks = n / 4;
        for (int i = threadIdx.x; i < a.E * chunks; i += kThreads) {
            const int e = i / chunks, c = i - e * chunks;
            copy16(dst + i * 16, reinterpret_cast<const uint8_t *>(a.router + (size_t)e * a.d + k + c * 4));
        }
    } else {
        for (int i = threadIdx.x; i < a.E * n; i += kThreads) {
            const int e = i / n, c = i - e * n;
            reinterpret_cast<float *>(to)[i] = a.router[(size_t)e * a.d + k + c];
        }
    }
}

// The CTA's columns' part of every (token, expert) logit, from the staged activations and, piece by piece, the router in
// `room` (the first piece is already on its way). The sums are in the staged activations' scale.
template <bool MX, int PARTS, int NT> __device__ void partial_logits(const MoeArgs & a, int k0, int k1, const Staged & x, uint8_t * room, int room_bytes, float * out) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int EB = 4, TB = NT == 1 ? 1 : 4;         // experts and tokens a warp takes at once
    const int width = router_columns(a.E, room_bytes);
    const int groups_t = (a.T + TB - 1) / TB, items = (a.E + EB - 1) / EB * groups_t;
    for (int k = k0; k < k1; k += width) {
        const int n = min(width, k1 - k);
        if (k > k0) {
            __syncthreads();
            fetch_router(a, k, n, room);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        const float * r = reinterpret_cast<const float *>(room);
        for (int item = warp; item < items; item += kWarps) {
            const int e0 = item / groups_t * EB, t0 = (item - item / groups_t * groups_t) * TB;
            float acc[16] = {};
            for (int c = lane * 4; c < n; c += 128) {
                const int at = k - k0 + c, step = at >> 6, group = (at >> 5) & 1;
                float4 w[EB];
#pragma unroll
                for (int e = 0; e < EB; ++e) w[e] = *reinterpret_cast<const float4 *>(r + min(e0 + e, a.E - 1) * n + c);
                const float factor = !MX && group ? 16.f : 1.f;
#pragma unroll
                for (int t = 0; t < TB; ++t) {
                    const uint8_t * p = x.x + ((step * 2 + group) * PARTS * NT + min(t0 + t, a.T - 1)) * 64 + (at & 31) * 2;
                    const uint2 h = *reinterpret_cast<const uint2 *>(p);
                    float2 v0 = __half22float2(*reinterpret_cast<const __half2 *>(&h.x)), v1 = __half22float2(*reinterpret_cast<const __half2 *>(&h.y));
                    if constexpr (PARTS == 2) {
                        const uint2 l = *reinterpret_cast<const uint2 *>(p + NT * 64);
                        const float2 l0 = __half22float2(*reinterpret_cast<const __half2 *>(&l.x)), l1 = __half22float2(*reinterpret_cast<const __half2 *>(&l.y));
                        v0.x += l0.x; v0.y += l0.y; v1.x += l1.x; v1.y += l1.y;
                    }
#pragma unroll
                    for (int e = 0; e < EB; ++e)
                        acc[e * TB + t] += factor * (w[e].x * v0.x + w[e].y * v0.y + w[e].z * v1.x + w[e].w * v1.y);
                }
            }
            const float sum = warp_sums16(acc);
            const int i = lane >> 1, e = e0 + i / TB, t = t0 + i % TB;
            if (!(lane & 1) && i < EB * TB && e < a.E && t < a.T) {
                if (k == k0) out[t * a.E + e] = sum;
                else out[t * a.E + e] += sum;
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
        if (32 * j < E) mx = fmaxf(mx, p[j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (32 * j >= E) break;
        p[j] = lane + 32 * j < E ? expf(p[j] - mx) : 0.f;
        sum += p[j];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // key: the probability's bits, which order like the probabilities, plus one; a NaN behind every number, taken ones at zero
    uint32_t key[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        key[j] = 0;
        if (32 * j >= E) continue;
        p[j] /= sum;
        key[j] = lane + 32 * j < E ? (p[j] >= 0.f ? __float_as_uint(p[j]) + 2u : 1u) : 0u;
    }
    float chosen = 0.f;
    for (int pick = 0; pick < k; ++pick) {
        uint32_t best = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) if (32 * j < E) best = max(best, key[j]);
        best = __reduce_max_sync(0xffffffffu, best);
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int j = PER - 1; j >= 0; --j) if (32 * j < E && key[j] == best) at = lane + 32 * j;
        at = __reduce_min_sync(0xffffffffu, at);
        float value = 0.f;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (32 * j < E && at == (uint32_t)(lane + 32 * j)) {
                value = p[j];
                key[j] = 0;
            }
        }
        value = __shfl_sync(0xffffffffu, value, at & 31);
        if (lane == 0) { expert[pick] = (uint16_t)at; weight[pick] = value; }
        chosen += value;
    }
    if (normalise) {
        __syncwarp();
        for (int i = lane; i < k; i += 32) weight[i] /= chosen;
    }
}

// The chosen experts in ascending order with their tokens, from the picks of all tokens. Picks::mask is zero before.
__device__ void group_picks(const MoeArgs & a, Picks & p, MoeMeta * meta) {
    const int e = threadIdx.x, warp = e >> 5, lane = e & 31;
    for (int i = e; i < a.T * a.k; i += kThreads) {
        const int t = i / a.k, expert = p.expert[i];
        atomicOr(&p.mask[expert], 1u << t);
        p.rank[expert][t] = (uint8_t)(i - t * a.k);
    }
    __syncthreads();
    const uint32_t mask = p.mask[e];                // tokens that chose expert e
    const uint32_t chosen = __ballot_sync(0xffffffffu, mask != 0);
    const int n = __popc(mask);
    const uint32_t most = __reduce_max_sync(0xffffffffu, (uint32_t)n);
    if (lane == 0) { p.warp_unique[warp] = __popc(chosen); p.warp_most[warp] = (int)most; }
    __syncthreads();
    int before = 0, all = 0, top = 1;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += p.warp_unique[w];
        all += p.warp_unique[w];
        top = max(top, p.warp_most[w]);
    }
    if (mask) {
        const int u = before + __popc(chosen & ((1u << lane) - 1u));
        p.unique[u] = (uint16_t)e;
        p.count[u] = (uint8_t)n;
        int i = 0;
        for (uint32_t m = mask; m; m &= m - 1, ++i) {
            const int t = __ffs(m) - 1;
            p.token[u][i] = (uint8_t)t;
            if (meta) meta->pair[u][i] = (uint16_t)(t * a.k + p.rank[e][t]);
        }
        if (meta) {
            meta->expert[u] = (uint16_t)e;
            meta->count[u] = (uint16_t)n;
        }
    }
    if (e == 0) {
        p.n = all;
        p.most = top;
        if (meta) meta->n = all;
    }
    __syncthreads();
}

// Jobs: block j of an expert's gate and of its up matrix are jobs 2 j and 2 j + 1, experts one behind the other.
template <bool MX, int PARTS, int NT> struct GateUpSource {
    const MoeArgs & a;
    const Picks & p;
    Staged x;
    Inbox inbox;
    int job0, jobs, ks, most;
    int sub, step, len;
    int round, round0;

    // Cursor::group is the expert's place among the chosen ones.
    __device__ __forceinline__ void point(Cursor & c) const {
        c.live = c.job < jobs;
        if (!c.live) return;
        const int job = job0 + c.job, block = job >> 1;
        c.group = block / a.blocks_ff;
        const int e = p.unique[c.group];
        c.p = (job & 1 ? a.up + e * a.up_expert : a.gate + e * a.gate_expert) + ((size_t)(block - c.group * a.blocks_ff) * a.steps_d + step) * w4_unit_bytes(MX);
        c.rem = len;
    }
    __device__ __forceinline__ void first(Cursor & c) const {
        c.job = (threadIdx.x >> 5) >> (__ffs(ks) - 1);
        point(c);
    }
    __device__ __forceinline__ void next(Cursor & c) const {
        c.job += kWarps >> (__ffs(ks) - 1);
        point(c);
    }
    __device__ __forceinline__ Group group(const Cursor & c) const { return {x, p.token[c.group], p.count[c.group], 0}; }
    __device__ __forceinline__ void put(const Cursor & c, int row, int col, float v) const {
        const int job = c.job - round0;
        inbox.put(round, (job >> 1) * most + col, job & 1, sub, row, v);
    }
};

template <bool MX, int PARTS, int NT>
__global__ void __launch_bounds__(kThreads, NT > 8 ? 2 : 3) w4_moe_gate_up_kernel(MoeArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Scratch sc;
    __shared__ Picks picks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), C = (int)cluster_size();
    const int cluster = blockIdx.x / C;
    cluster_arrive();
    const int log_c = __ffs(C) - 1;
    const int s0 = part_begin2(a.steps_d, rank, log_c), n_steps = part_begin2(a.steps_d, rank + 1, log_c) - s0;
    const Staged x{smem, reinterpret_cast<float *>(smem + a.x_bytes)};
    float * mine = reinterpret_cast<float *>(smem + a.x_bytes + a.c_bytes);         // this CTA's part of the logits
    float * logits = mine + a.logit_bytes / 4;
    uint8_t * const rings = smem + a.x_bytes + a.c_bytes + 2 * a.logit_bytes;
    if (threadIdx.x == 0) sc.zero = 0;
    picks.mask[threadIdx.x] = 0;

    pdl_trigger();
    pdl_wait();
    const int k0 = s0 * 64, k1 = min(a.d, (s0 + n_steps) * 64);
    fetch_router(a, k0, min(k1 - k0, router_columns(a.E, ring_bytes(MX, NT))), rings);      // the rings are idle until the experts are known
    asm volatile("cp.async.commit_group;" ::: "memory");
    stage_tokens<MX, PARTS>(a.x, a.T, NT, s0, n_steps, a.d, a.norm, x, sc, rank, C);
    __syncthreads();
    partial_logits<MX, PARTS, NT>(a, k0, k1, x, rings, ring_bytes(MX, NT), mine);
    // out of the activations' scale: a token's factors without the weights' constant
    __syncthreads();
    for (int i = threadIdx.x; i < a.T * a.E; i += kThreads) mine[i] = mine[i] * sc.f1[0][i / a.E] * sc.f2[0][i / a.E] * (MX ? 0.015625f : 5.9604644775390625e-8f);
    cluster_sync();
    for (int i = threadIdx.x; i < a.T * a.E; i += kThreads) {
        float part[kMaxCluster];
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) part[c] = c < C ? remote_load(remote_address(smem_address(mine + i), c)) : 0.f;
        float v = 0.f;
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) v += part[c];
        logits[i] = a.norm ? v * rms_factor(sc, i / a.E, C, a.d, a.eps) : v;
    }
    if (threadIdx.x < a.T) picks.rstd[threadIdx.x] = a.norm ? rms_factor(sc, threadIdx.x, C, a.d, a.eps) : 1.f;
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

    const int total = picks.n * a.blocks_ff, most = picks.most;
    const int b_begin = part_begin(total, cluster, a.clusters), blocks = part_begin(total, cluster + 1, a.clusters) - b_begin;
    const int ks = split_columns(blocks * 2, a.steps_d / C, (int)(a.inbox / inbox_bytes(most, C, 1, 2)));
    const int per_round = blocks_per_round(a.inbox, most, C, ks, 2);
    const int log_ks = __ffs(ks) - 1;
    const int sub = warp & (ks - 1), step = part_begin2(n_steps, sub, log_ks), len = part_begin2(n_steps, sub + 1, log_ks) - step;
    const Staged x_warp{x.x + step * step_x_bytes(PARTS, NT), x.c + step * step_c_bytes(MX, NT) / 4};
    const Inbox inbox{smem_address(rings + ring_bytes(MX, NT)), a.inbox, rank, log_c, ks, 2};
    GateUpSource<MX, PARTS, NT> src{a, picks, x_warp, inbox, 2 * b_begin, 2 * blocks, ks, most, sub, s0 + step, len, 0, 0};
    Stream<MX, stages_for(NT), GateUpSource<MX, PARTS, NT>> stream(src, rings);
    stream.prefetch();
    for (int b0 = 0; b0 < blocks; b0 += per_round, ++src.round) {
        const int now = min(per_round, blocks - b0);
        src.round0 = 2 * b0;
        stream.template work<PARTS, NT, (NT > 1)>(sc, 2 * (b0 + now));
        cluster_sync();
        for (int i = warp; i * C + rank < now * most; i += kWarps) {
            const int unit = i * C + rank, b = unit / most, col = unit - b * most;
            const int u = (b_begin + b0 + b) / a.blocks_ff, row = ((b_begin + b0 + b) - u * a.blocks_ff) * 32 + lane;
            if (col >= picks.count[u]) continue;
            const int t = picks.token[u][col], pair = t * a.k + picks.rank[picks.unique[u]][t];
            const float v = inbox.sum(src.round, i, 0) * picks.rstd[t], up = inbox.sum(src.round, i, 1) * picks.rstd[t];
            if (row < a.ff) a.h[pair * a.ld_h + row] = picks.weight[pair] * (v / (1.f + expf(-v)) * up);
        }
    }
    if (blocks == 0) cluster_sync();        // nobody leaves while its logits are read
}

// Consecutive steps of one chosen expert.
struct Seg {
    int u, expert, s0, len, x_off, c_off, n, row0;      // row0: tokens of the segments before
};
struct DownTable {
    Seg seg[kMaxSegs];
    uint8_t token[kMaxSegs][kRowList];
    int n, rows;
    int next;           // the step behind the chunk
};

// The segments from step p on, as many as `room` bytes of shared memory for activations hold. By one warp.
template <bool MX> __device__ void cut_segments(const MoeArgs & a, const MoeMeta & meta, int p, int end, int room, DownTable & table) {
    const int lane = threadIdx.x & 31;
    const int u = p / a.steps_ff + lane;
    const int from = max(p, u * a.steps_ff), whole = lane < kMaxSegs ? max(0, min(end, (u + 1) * a.steps_ff) - from) : 0;
    const int tokens = whole > 0 ? meta.count[u] : 0, nt = room_for(tokens);
    const int bytes = (whole * step_bytes(MX, 2, nt) + 15) / 16 * 16;
    int used = bytes, rows = tokens;        // inclusive sums over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int b = __shfl_up_sync(0xffffffffu, used, o), r = __shfl_up_sync(0xffffffffu, rows, o);
        if (lane >= o) { used += b; rows += r; }
    }
    used -= bytes;
    rows -= tokens;
    const int len = max(0, min(whole, (room - used) / step_bytes(MX, 2, nt)));
    // the first segment that does not fit ends the chunk; room for one step of the first is always there
    const uint32_t cut = __ballot_sync(0xffffffffu, len < whole);
    const int last = cut ? __ffs(cut) - 1 : 31;
    const uint32_t kept = __ballot_sync(0xffffffffu, len > 0 && lane <= last);
    const int n = __popc(kept);
    if (kept >> lane & 1) {
        const int x_bytes = len * step_x_bytes(2, nt);
        table.seg[lane] = {u, meta.expert[u], from - u * a.steps_ff, len, used, used + x_bytes, tokens, rows};
        for (int i = 0; i < tokens; ++i) table.token[lane][i] = (uint8_t)(meta.pair[u][i] / a.k);
        if (lane == n - 1) {
            table.n = n;
            table.rows = rows + tokens;
            table.next = from + len;
        }
    }
}

template <bool MX> struct DownSource {
    const MoeArgs & a;
    const DownTable & table;
    uint8_t * smem;
    float * partial;
    int job0, jobs, ks, sub;

    // Cursor::group is the segment: all jobs of one, then the next.
    __device__ __forceinline__ void point(Cursor & c) const {
        while (true) {
            c.live = c.group < table.n;
            if (!c.live) return;
            const Seg & g = table.seg[c.group];
            const int log_ks = __ffs(ks) - 1, s = part_begin2(g.len, sub, log_ks);
            c.rem = part_begin2(g.len, sub + 1, log_ks) - s;
            if (c.job < jobs && c.rem > 0) {
                c.p = a.down + g.expert * a.down_expert + ((size_t)(job0 + c.job) * a.steps_ff + g.s0 + s) * w4_unit_bytes(MX);
                return;
            }
            ++c.group;
            c.job = (threadIdx.x >> 5) >> (__ffs(ks) - 1);
        }
    }
    __device__ __forceinline__ void first(Cursor & c) const {
        c.group = 0;
        c.job = (threadIdx.x >> 5) >> (__ffs(ks) - 1);
        point(c);
    }
    __device__ __forceinline__ void next(Cursor & c) const {
        c.job += kWarps >> (__ffs(ks) - 1);
        point(c);
    }
    __device__ __forceinline__ Group group(const Cursor & c) const {
        const Seg & g = table.seg[c.group];
        const int s = part_begin2(g.len, sub, __ffs(ks) - 1), nt = room_for(g.n);
        return {{smem + g.x_off + s * step_x_bytes(2, nt), reinterpret_cast<float *>(smem + g.c_off + s * step_c_bytes(MX, nt))}, nullptr, g.n, c.group};
    }
    __device__ __forceinline__ void put(const Cursor & c, int row, int col, float v) const {
        partial[((c.job * ks + sub) * a.T + table.token[c.group][col]) * kSlotCol + row] += v;
    }
};

template <bool MX, int MOST>
__global__ void __launch_bounds__(kThreads, MOST > 8 ? 2 : 3) w4_moe_down_kernel(MoeArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Scratch sc;
    __shared__ DownTable table;
    __shared__ MoeMeta meta;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), C = (int)cluster_size();
    const int cluster = blockIdx.x / C;
    cluster_arrive();
    uint8_t * const rings = smem + a.x_bytes;
    float * partial = reinterpret_cast<float *>(rings + ring_bytes(MX, MOST));
    const Inbox inbox{smem_address(rings + ring_bytes(MX, MOST) + a.partial), a.inbox, rank, __ffs(C) - 1, 1, 1};
    const int j_begin = part_begin(a.blocks_d, cluster, a.clusters), j_end = part_begin(a.blocks_d, cluster + 1, a.clusters);
    if (threadIdx.x == 0) sc.zero = 0;
    pdl_trigger();
    pdl_wait();
    {
        const int4 * from = reinterpret_cast<const int4 *>(a.meta);
        int4 * to = reinterpret_cast<int4 *>(&meta);
        const int reach = min(a.E, a.T * a.k);
        for (int i = threadIdx.x; i < (int)((offsetof(MoeMeta, pair) + sizeof(meta.pair[0]) * reach) / 16); i += kThreads) to[i] = from[i];
    }
    cluster_wait();
    __syncthreads();
    const int total = meta.n * a.steps_ff;          // the chosen experts' columns, one behind the other
    const int begin = part_begin2(total, rank, __ffs(C) - 1), end = part_begin2(total, rank + 1, __ffs(C) - 1);
    const int slot = a.T * kSlotCol * 4;
    const int ks = split_columns(j_end - j_begin, max(1, total / C), a.partial / slot);
    const int per_round = min(a.partial / (slot * ks), blocks_per_round(a.inbox, a.T, C, 1, 1));
    const Act h{a.h, a.ld_h, GGML_F32, true};
    int round = 0;
    for (int j0 = j_begin; j0 < j_end; j0 += per_round, ++round) {
        const int jobs = min(per_round, j_end - j0);
        for (int i = threadIdx.x; i < jobs * ks * a.T * kSlotCol; i += kThreads) partial[i] = 0.f;
        for (int p = begin; p < end; p = table.next) {
            __syncthreads();            // the table, the activations and the slots are free (or cleared)
            if (warp == 0) cut_segments<MX>(a, meta, p, end, a.x_bytes - 16, table);
            __syncthreads();
            const DownSource<MX> src{a, table, smem, partial, j0, jobs, ks, warp % ks};
            Stream<MX, stages_for(MOST), DownSource<MX>> stream(src, rings);
            stream.prefetch();
            stage_rows<MX, 2, false>(h, table.rows, a.ff, nullptr, sc, [&](int i) {
                int n = 0;
                while (n + 1 < table.n && i >= table.seg[n + 1].row0) ++n;
                const Seg & g = table.seg[n];
                return StageRow{(int64_t)meta.pair[g.u][i - g.row0], g.s0 * 64, g.len, room_for(g.n), i - g.row0, n,
                                Staged{smem + g.x_off, reinterpret_cast<float *>(smem + g.c_off)}};
            }, [](int, float) {});
            __syncthreads();
            stream.template work_sized<2, MOST>(sc);
        }
        __syncthreads();
        for (int unit = warp; unit < jobs * a.T; unit += kWarps) {
            const int job = unit / a.T, t = unit - job * a.T;
            float v = 0.f;
            for (int i = 0; i < ks; ++i) v += partial[((job * ks + i) * a.T + t) * kSlotCol + lane];
            inbox.put(round, unit, 0, 0, lane, v);
        }
        cluster_sync();
        for (int i = warp; i * C + rank < jobs * a.T; i += kWarps) {
            const int unit = i * C + rank, job = unit / a.T, t = unit - job * a.T;
            float v = inbox.sum(round, i, 0);
            const int row = (j0 + job) * 32 + lane;
            if (row < a.d) {
                if (a.residual) v += load1(Act{a.residual, a.ld_residual, a.y_type, false}, t, row);
                store1(a.y, a.y_type, t * a.ld_y + row, v);
            }
        }
    }
}

// ---- retiling
//
// Word j (0..3) of lane (g, t) holds row g + 8 (j & 1), columns 8 t + 4 s + 2 (j >> 1) + e of group h, for the products
// s = 0, 1, groups h = 0, 1 and halves e = 0, 1 of the word. Q4_0: the nibble at bit 16 e + 8 s + 4 h. MXFP4: inside half
// e, (sign, magnitude) at bits (15, 11..9), (12, 8..6), (14, 5..3), (13, 2..0) for (h, s) = (0,0), (0,1), (1,0), (1,1).
template <bool MX>
__global__ void w4_retile_kernel(const uint8_t * rows, uint32_t n_out, uint32_t n_in, uint32_t row_blocks, uint32_t steps, uint8_t * units, int * max_scale) {
    constexpr uint32_t kBlock = MX ? 17 : 18;
    const uint32_t blocks = n_in / 32;
    const size_t unit = blockIdx.x;
    const uint32_t step = (uint32_t)(unit % steps);
    const size_t block_of_all = unit / steps;
    const uint32_t row_block = (uint32_t)(block_of_all % row_blocks);
    const size_t expert = block_of_all / row_blocks;
    uint8_t * dst = units + unit * w4_unit_bytes(MX);
    const uint32_t tile = threadIdx.x >> 7, lane = (threadIdx.x & 127) >> 2, j = threadIdx.x & 3;
    const uint32_t g = lane >> 2, t = lane & 3;
    const uint32_t row = row_block * 32 + tile * 16 + g + 8 * (j & 1);
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
    *reinterpret_cast<uint32_t *>(dst + tile * 512 + lane * 16 + j * 4) = word;
    if (threadIdx.x < 64) {
        // scales of (g, group), then of (g + 8, group), for g = 0..7, of each tile
        const uint32_t st = threadIdx.x >> 5, sg = (threadIdx.x & 31) >> 2, upper = (threadIdx.x >> 1) & 1, h = threadIdx.x & 1;
        const uint32_t srow = row_block * 32 + st * 16 + sg + 8 * upper, block = step * 2 + h;
        const bool live = srow < n_out && block < blocks;
        const uint8_t * b = rows + ((expert * n_out + srow) * blocks + block) * kBlock;
        if (MX) {
            // kept as s + 8, so that the smallest scale 2^-127 is a normal f32 as well; 2^-8 is part of the rows' final factor
            const int s = live ? b[0] : 0;
            const uint32_t warp_max = __reduce_max_sync(0xffffffffu, (uint32_t)s);
            if ((threadIdx.x & 31) == 0) atomicMax(max_scale, (int)warp_max);
            dst[1024 + st * 32 + sg * 4 + upper * 2 + h] = live ? (uint8_t)min(s + 8, 255) : 0;
        } else {
            reinterpret_cast<uint16_t *>(dst + 1024 + st * 64)[sg * 4 + upper * 2 + h] = live ? (uint16_t)(b[0] | b[1] << 8) : 0;
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

template <typename... KArgs> cudaError_t allow_smem(PerDeviceOnce & once, void (*kernel)(KArgs...)) {
    return once.first() ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) : cudaSuccess;
}

template <bool MX, int PARTS, bool GLU, int NT> cudaError_t launch_product(const ProductArgs & a, int C, size_t smem, cudaStream_t stream) {
    static PerDeviceOnce once;
    const cudaError_t e = allow_smem(once, w4_product_kernel<MX, PARTS, GLU, NT>);
    return e != cudaSuccess ? e : launch_cluster(w4_product_kernel<MX, PARTS, GLU, NT>, a.clusters * C, C, smem, stream, a);
}

// Room the kernels that take whole calls of n tokens stage them with: those sizes they are built for.
int product_room(int n, int parts) { return n == 1 ? 1 : n <= 4 && parts == 2 ? 4 : n <= 8 ? 8 : 16; }

template <bool MX, bool GLU>
cudaError_t launch_product_of(const ProductArgs & a, int parts, int C, size_t smem, cudaStream_t stream) {
    const int nt = product_room(a.T, parts);
    if (parts == 2) {
        if (nt == 1) return launch_product<MX, 2, GLU, 1>(a, C, smem, stream);
        if (nt == 4) return launch_product<MX, 2, GLU, 4>(a, C, smem, stream);
        if (nt == 8) return launch_product<MX, 2, GLU, 8>(a, C, smem, stream);
        return launch_product<MX, 2, GLU, 16>(a, C, smem, stream);
    }
    if (nt == 1) return launch_product<MX, 1, GLU, 1>(a, C, smem, stream);
    if (nt == 8) return launch_product<MX, 1, GLU, 8>(a, C, smem, stream);
    return launch_product<MX, 1, GLU, 16>(a, C, smem, stream);
}

size_t type_bytes(uint32_t type) { return type == GGML_F32 ? 4 : 2; }

Act make_act(const void * p, int64_t ld, uint32_t type) {
    const size_t es = type_bytes(type);
    return {p, ld, type, (uintptr_t)p % (4 * es) == 0 && (ld * (int64_t)es) % (int64_t)(4 * es) == 0};
}

const void * row_at(const void * p, uint32_t type, int64_t ld, int64_t row) {
    return p ? static_cast<const uint8_t *>(p) + row * ld * (int64_t)type_bytes(type) : nullptr;
}

template <bool MX, int PARTS, int NT> cudaError_t launch_gate_up(const MoeArgs & a, int C, size_t smem, cudaStream_t stream) {
    static PerDeviceOnce once;
    const cudaError_t e = allow_smem(once, w4_moe_gate_up_kernel<MX, PARTS, NT>);
    return e != cudaSuccess ? e : launch_cluster(w4_moe_gate_up_kernel<MX, PARTS, NT>, a.clusters * C, C, smem, stream, a);
}

template <bool MX, int MOST> cudaError_t launch_down(const MoeArgs & a, int C, size_t smem, cudaStream_t stream) {
    static PerDeviceOnce once;
    const cudaError_t e = allow_smem(once, w4_moe_down_kernel<MX, MOST>);
    return e != cudaSuccess ? e : launch_cluster(w4_moe_down_kernel<MX, MOST>, a.clusters * C, C, smem, stream, a);
}

template <bool MX> cudaError_t launch_gate_up_of(const MoeArgs & a, int parts, int C, size_t smem, cudaStream_t stream) {
    const int nt = product_room(a.T, parts);
    if (parts == 2) {
        if (nt == 1) return launch_gate_up<MX, 2, 1>(a, C, smem, stream);
        if (nt == 4) return launch_gate_up<MX, 2, 4>(a, C, smem, stream);
        if (nt == 8) return launch_gate_up<MX, 2, 8>(a, C, smem, stream);
        return launch_gate_up<MX, 2, 16>(a, C, smem, stream);
    }
    if (nt == 1) return launch_gate_up<MX, 1, 1>(a, C, smem, stream);
    if (nt == 8) return launch_gate_up<MX, 1, 8>(a, C, smem, stream);
    return launch_gate_up<MX, 1, 16>(a, C, smem, stream);
}

template <bool MX> cudaError_t launch_down_of(const MoeArgs & a, int C, size_t smem, cudaStream_t stream) {
    if (a.T == 1) return launch_down<MX, 1>(a, C, smem, stream);
    if (a.T <= 4) return launch_down<MX, 4>(a, C, smem, stream);
    if (a.T <= 8) return launch_down<MX, 8>(a, C, smem, stream);
    return launch_down<MX, 16>(a, C, smem, stream);
}

int up_to(int x, int unit) { return (x + unit - 1) / unit * unit; }

int64_t moe_ld_h(uint32_t ff) { return ((int64_t)ff + 3) / 4 * 4; }

} // namespace

size_t w4_bytes(uint32_t type, uint32_t n_out, uint32_t n_in, uint32_t n_expert) {
    return (size_t)n_expert * ((n_out + 31) / 32) * ((n_in + 63) / 64) * w4_unit_bytes(type == GGML_MXFP4);
}

W4View w4_view(const uint8_t * units, uint32_t type, uint32_t n_out, uint32_t n_in, uint32_t n_expert) {
    W4View v;
    v.units = units;
    v.type = type;
    v.n_out = n_out;
    v.n_in = n_in;
    v.n_expert = n_expert;
    v.blocks = (n_out + 31) / 32;
    v.steps = (n_in + 63) / 64;
    v.expert_bytes = (size_t)v.blocks * v.steps * w4_unit_bytes(type == GGML_MXFP4);
    return v;
}

void launch_w4_retile(const uint8_t * rows, uint32_t type, uint32_t n_out, uint32_t n_in, uint32_t n_expert, uint8_t * units, int * max_scale,
                      cudaStream_t stream) {
    const W4View v = w4_view(units, type, n_out, n_in, n_expert);
    const size_t n = (size_t)n_expert * v.blocks * v.steps;
    if (type == GGML_MXFP4) w4_retile_kernel<true><<<(unsigned)n, 256, 0, stream>>>(rows, n_out, n_in, v.blocks, v.steps, units, max_scale);
    else w4_retile_kernel<false><<<(unsigned)n, 256, 0, stream>>>(rows, n_out, n_in, v.blocks, v.steps, units, max_scale);
}

// Clusters of a size that are on the GPU together, with `resident` CTAs on an SM: a cluster lies within one of the GPU's processing
// clusters, whose SM counts are no multiples of it. Asked once per device.
int resident_clusters(int log_c, int resident) {
    struct Table { std::atomic<int> n[4][3]; };
    static Table tables[64];
    int device = 0;
    cudaGetDevice(&device);
    std::atomic<int> & known = tables[device & 63].n[log_c][resident - 1];
    int n = known.load();
    if (n) return n;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << log_c;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(1u << log_c);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = std::min(kMaxSmem, 226 * 1024 / resident - 4096);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    static PerDeviceOnce once;
    auto kernel = w4_product_kernel<false, 2, false, 1>;
    if (allow_smem(once, kernel) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = std::max(1, resident * device_sms() >> log_c);
    }
    known.store(n);
    return n;
}

// How a product is cut: CTAs of a cluster, clusters, and the shared memory of a CTA.
struct Cut {
    int C = 0, clusters = 0, resident = 0;
    double cost = 0;
};

// Chooses the cluster size for `blocks` row blocks of `per` matrices and `steps` column steps whose activations take `each` bytes of
// shared memory a step. The estimate is in clocks: the weight stream at the SM's share of the memory bandwidth, but no faster
// than the copies in flight of the CTAs on the busiest SM allow; the conversion of the CTA's share of the activations; and the sums it
// receives; `step_clocks` is what else a column step costs a CTA.
Cut choose_cut(int blocks, int per, int steps, int n, int each, int ring, int fixed, double step_clocks, int unit, int sms) {
    Cut best;
    for (int C = 1; C <= kMaxCluster && C <= steps; C *= 2) {
        const int s = (steps + C - 1) / C;
        const int64_t inbox = 2 * inbox_bytes(n, C, 1, per);
        const int64_t smem = s * each + ring + fixed + inbox + 4096;
        if (smem > kMaxSmem) continue;
        Cut c;
        c.C = C;
        c.resident = (int)std::min<int64_t>(n > 8 ? 2 : 3, 226 * 1024 / smem);
        if (const char * e = std::getenv("W4_RES")) c.resident = std::min(c.resident, atoi(e));
        if (const char * e = std::getenv("W4_C")) if (C != atoi(e)) continue;
        const int log_c = C == 1 ? 0 : C == 2 ? 1 : C == 4 ? 2 : 3;
        const int most = resident_clusters(log_c, c.resident), blocks_each = (blocks + most - 1) / most;
        c.clusters = (blocks + blocks_each - 1) / blocks_each;
        const int busy = (c.clusters * C + sms - 1) / sms;
        const double in_flight = (double)busy * ring * (stages_for(n) - 1) / stages_for(n);
        const double stream = std::max((double)blocks * per * steps * unit / (23.5 * sms), (double)busy * blocks_each * per * s * unit / std::min(46.0, in_flight / 1600.0));
        const double convert = busy * s * (n * 64 * 0.12 + step_clocks) + 800, sums = busy * (double)blocks_each * per * n * 8;
        c.cost = stream + convert + sums;
        if (!best.C || c.cost < best.cost) best = c;
    }
    return best;
}

cudaError_t launch_w4_product(const W4Product & p, cudaStream_t stream) {
    const bool mx = p.w.type == GGML_MXFP4, glu = p.up != nullptr;
    const int parts = p.x_type == GGML_F32 || p.norm ? 2 : 1;
    const int sms = device_sms();
    const int blocks = (int)p.w.blocks, per = glu ? 2 : 1, steps = (int)p.w.steps;
    for (int t0 = 0, n = 0; t0 < p.n_tokens; t0 += n) {
        n = std::min(kW4PassTokens, p.n_tokens - t0);
        Cut cut;
        for (;; n = (n + 1) / 2) {
            cut = choose_cut(blocks, per, steps, n, step_bytes(mx, parts, product_room(n, parts)), ring_bytes(mx, product_room(n, parts)), 0, 0, (int)w4_unit_bytes(mx), sms);
            if (cut.C || n == 1) break;
        }
        if (!cut.C) return cudaErrorInvalidValue;       // rows this long are refused when the handle is made
        const int C = cut.C, nt = product_room(n, parts), s = (steps + C - 1) / C;
        ProductArgs a{};
        a.w = p.w.units;
        a.u = glu ? p.up->units : nullptr;
        a.x = make_act(row_at(p.x, p.x_type, p.ld_x, t0), p.ld_x, p.x_type);
        a.T = n;
        a.n_in = (int)p.w.n_in;
        a.n_out = (int)p.w.n_out;
        a.steps = steps;
        a.norm = p.norm;
        a.eps = p.eps;
        a.bias = p.bias;
        a.residual = row_at(p.residual, p.y_type, p.ld_residual, t0);
        a.ld_residual = p.ld_residual;
        a.y = const_cast<void *>(row_at(p.y, p.y_type, p.ld_y, t0));
        a.y_type = p.y_type;
        a.ld_y = p.ld_y;
        a.each = blocks / cut.clusters;
        a.more = blocks % cut.clusters;
        a.clusters = cut.clusters;
        a.x_bytes = up_to(s * step_x_bytes(parts, nt), 128);
        a.c_bytes = up_to(s * step_c_bytes(mx, nt), 128);
        // two inboxes in what is left of the CTA's share of the shared memory; one, if everything fits into it
        const int fixed = a.x_bytes + a.c_bytes + ring_bytes(mx, nt);
        const int blocks_each = (blocks + cut.clusters - 1) / cut.clusters;
        const int room = std::min(226 * 1024 / cut.resident - 4096, kMaxSmem) - fixed;
        a.ks = split_columns(blocks_each * per, steps / C, (int)std::max<int64_t>(1, room / 2 / inbox_bytes(n, C, 1, per)));
        const int64_t whole = inbox_bytes((int64_t)blocks_each * n, C, a.ks, per);
        a.inbox = (int)(whole <= room ? whole : std::max<int64_t>(room / 2 / 128 * 128, inbox_bytes(n, C, a.ks, per)));
        a.per_round = blocks_per_round(a.inbox, n, C, a.ks, per);
        const size_t smem = (size_t)fixed + (whole <= room ? 1 : 2) * (size_t)a.inbox;
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
    for (int t0 = 0, n = 0; t0 < p.n_tokens; t0 += n) {
        n = std::min(kW4PassTokens, p.n_tokens - t0);
        // first kernel: n tokens choose at most `reach` experts, a little fewer if they choose independently
        int reach = 0;
        Cut cut;
        for (;; n = (n + 1) / 2) {
            reach = (int)std::ceil(E * (1.0 - std::pow(1.0 - (double)p.n_used / E, n)));
            cut = choose_cut(reach * (int)p.gate.blocks, 2, steps_d, n, step_bytes(mx, parts, product_room(n, parts)), ring_bytes(mx, product_room(n, parts)),
                             2 * up_to(n * E * 4, 128) + 16 * 1024, n * E * 0.65 + E * 8, (int)w4_unit_bytes(mx), sms);
            if (cut.C || n == 1) break;
        }
        if (!cut.C) return cudaErrorInvalidValue;
        int C = cut.C;
        MoeArgs a{};
        a.gate = p.gate.units;
        a.up = p.up.units;
        a.down = p.down.units;
        a.gate_expert = p.gate.expert_bytes;
        a.up_expert = p.up.expert_bytes;
        a.down_expert = p.down.expert_bytes;
        a.router = p.router;
        a.router_vec = (uintptr_t)p.router % 16 == 0;
        a.x = make_act(row_at(p.x, p.x_type, p.ld_x, t0), p.ld_x, p.x_type);
        a.T = n;
        a.E = E;
        a.k = p.n_used;
        a.d = d;
        a.ff = ff;
        a.blocks_ff = (int)p.gate.blocks;
        a.steps_d = steps_d;
        a.blocks_d = (int)p.down.blocks;
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

        const int s = (steps_d + C - 1) / C, nt = product_room(n, parts);
        a.x_bytes = up_to(s * step_x_bytes(parts, nt), 128);
        a.c_bytes = up_to(s * step_c_bytes(mx, nt), 128);
        a.logit_bytes = up_to(n * E * 4, 128);
        a.clusters = cut.clusters;
        int fixed = a.x_bytes + a.c_bytes + 2 * a.logit_bytes + ring_bytes(mx, nt);
        a.inbox = (int)std::max<int64_t>((std::min(226 * 1024 / cut.resident - 20 * 1024, kMaxSmem) - fixed) / 2 / 128 * 128, inbox_bytes(n, C, 1, 2));
        cudaError_t e = mx ? launch_gate_up_of<true>(a, parts, C, (size_t)fixed + 2 * a.inbox, stream) : launch_gate_up_of<false>(a, parts, C, (size_t)fixed + 2 * a.inbox, stream);
        if (e != cudaSuccess) return e;

        // second kernel
        C = kMaxCluster;
        while (C > steps_ff * p.n_used) C /= 2;
        const int resident = 2;
        const int most = resident_clusters(C == 1 ? 0 : C == 2 ? 1 : C == 4 ? 2 : 3, resident), per = (a.blocks_d + most - 1) / most;
        a.clusters = (a.blocks_d + per - 1) / per;
        a.x_bytes = (n > 8 ? 24 : n > 1 ? 20 : 12) * 1024;
        a.c_bytes = a.logit_bytes = 0;
        const int slot = n * kSlotCol * 4, down_fixed = a.x_bytes + ring_bytes(mx_down, n == 1 ? 1 : n <= 4 ? 4 : 8);
        a.inbox = (int)inbox_bytes(std::min(per, kWarps) * n, C, 1, 1);
        a.partial = std::max(kWarps * slot, std::min(per * kWarps * slot, 226 * 1024 / resident - 18 * 1024 - down_fixed - 2 * a.inbox) / slot * slot);
        const size_t smem = (size_t)down_fixed + a.partial + 2 * a.inbox;
        e = mx_down ? launch_down_of<true>(a, C, smem, stream) : launch_down_of<false>(a, C, smem, stream);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

} // namespace rb200
