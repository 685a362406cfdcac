// Products with 4-bit weights for at most sixteen tokens, bound by the weight stream.
//
// Mathematics. 16 rows x 64 columns are the A operands of four m16n8k16 products; the tokens are the columns
// of B. The weights enter as exact f16 values that cost little arithmetic:
//   Q4_0   the nibble q in the top four mantissa bits of an f16 is the subnormal q 2^-18: a rotation and a mask. (In the
//          low bits it would save the rotation, but the tensor cores align products by the operands' exponents and dropped up to ten
//          bits of such products: 1.6e-6 of the result. As the difference q - 8 it costs an addition, 63.5 us instead of 56 for
//          128256 x 4096 at one token.) The offset is the product chain's start value, -8 2^-18 times the group's sum of activations.
//   MXFP4  the conversion instruction for pairs of e2m1 values.
// A token's activations are scaled by a power of two that brings the largest of them into [2^13, 2^14) and split into
// hi + lo f16 (22 bits); activations that are f16 or bf16 themselves need no lo. A 32-column group is exactly two
// products, so its f32 sum comes out on its own, is multiplied by the group's scale and added in f32.
//
// Split. A cluster of up to eight CTAs owns a range of row blocks (32 rows); each CTA takes a range of the columns for all of them, so
// it converts only its share of the activations. Its warps take (row block, part of the CTA's columns) runs, and
// write every (row block, token)'s sums into the shared memory of the CTA that owns it, which adds them in a fixed order after one
// cluster barrier (no workspace, no atomics: results are the same in every run) and applies bias, residual or the gate's
// activation. Every warp streams its units through a ring of its own in shared memory by asynchronous copies, one or two units
// ahead, so that no registers are held by loads in flight. Up to four tokens run as three CTAs of eight warps on an SM; more
// as one of sixteen, because all warps of a CTA share its activations.
//
// Measured (replayed in a graph, weights larger than the L2 cache; a call by itself is longer by up to 7 us), Q4_0: 128256 x 4096 at one token 56 us, 5.24 TB/s, bound by the integer pipe that
// unpacks (63 us a call); 14336 x 4096 gated pair 18.7 us at one token (3.5 TB/s), 36 us at sixteen, where mma.sync with hi and lo parts is the busiest unit of the product loop
// and staging takes 6 us; 4096 x 14336 at one token 11.4 us (2.9 TB/s), a third of it staging and the launch. MXFP4, 201088 x 2880, sixteen
// bf16 tokens: 96 us, 3.2 TB/s. A layer of 32 experts of 2880 x 2880 (MXFP4, four used): 31 us at one token, 114 us at sixteen.

#include "kernels.cuh"
#include "blocks.hpp"
#include "w4.cuh"

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cuda_bf16.h>

namespace rb200 {

namespace {

constexpr int kSlotCol = 36;        // floats per (partial slot, token) of the second expert kernel: 32 rows, padded against bank conflicts
constexpr int kRowList = kW4PassTokens;
constexpr int kMaxCluster = 8;
// Warps of a CTA that serves up to n tokens, and its CTAs on an SM. (Two to four tokens on eight: 14336 x 4096
// gated pair 21.8 to 22.2 us, where sixteen take 17.5 to 17.9 us; expert layer of 32 x 2880 x 2880 at three tokens 69 us, where they take 51 us.)
__host__ __device__ constexpr int warps_for(int n) { return n > 4 ? 16 : 8; }
__host__ __device__ constexpr int resident_for(int n) { return n > 4 ? 1 : 3; }
// Units in the ring of each of its warps. For products of more than eight f32 tokens the activations and the sums need the room more (14336 x
// 4096 gated pair, sixteen tokens: 50 us with three, whose sums took seven rounds, 36 us with two); where the activations are
// halves two is slower (4096 x 14336, eleven f16 tokens: 25 us and 20 us), and so it is for the expert layer (163 us and 147 us).
__host__ __device__ constexpr int stages_for(int n, int parts) { return n > 8 && parts == 2 ? 2 : 3; }
constexpr int kMoeStages = 3;

struct Act {
    const void * p;
    int64_t ld;
    uint32_t type;
    bool vec;       // rows may be read sixteen bytes at a time
};

__device__ __forceinline__ float load1(const Act & a, int64_t row, int k) {
    const int64_t i = row * a.ld + k;
    if (a.type == GGML_F32) return static_cast<const float *>(a.p)[i];
    const uint16_t h = static_cast<const uint16_t *>(a.p)[i];
    return a.type == GGML_F16 ? __half2float(__ushort_as_half(h)) : __uint_as_float((uint32_t)h << 16);
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

// One 64-column half of a unit: the lane's A words of its two row tiles.
struct Words {
    uint4 q[2];
};
// The lane's scales, rows g and g + 8 of the two tiles, four groups each.
template <bool MX> struct Scales {
    uint4 s[2];     // MXFP4 uses .x and .y only
};

__host__ __device__ constexpr int ring_bytes(bool mx, int n, int stages) { return warps_for(n) * stages * (int)w4_unit_bytes(mx); }

__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t * src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
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
__device__ __forceinline__ void store_u4(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ float shared_f1(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
    return v;
}

// A registers of product S of group H of a 64-column half, from the lane's four words.
template <bool MX, int H, int S> __device__ __forceinline__ void decode(const uint4 & q, uint32_t (&a)[4]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (!MX) {
            a[j] = __funnelshift_r(w[j], w[j], 4 * (2 * H + S)) & 0x03c003c0u;
        } else {
            // byte 2 H + S of the word
            asm("{\n.reg .b8 b<4>;\nmov.b32 {b0, b1, b2, b3}, %1;\ncvt.rn.f16x2.e2m1x2 %0, b%2;\n}" : "=r"(a[j]) : "r"(w[j]), "n"(2 * H + S));
        }
    }
}

// Scales of rows g and g + 8 for group G of a unit.
template <bool MX, int G> __device__ __forceinline__ void scales(const uint4 & s, float & d0, float & d1) {
    if constexpr (MX) {
        constexpr uint32_t kExponent = 0x7f800000u;
        d0 = __uint_as_float((G == 0 ? s.x << 23 : G == 1 ? s.x << 15 : G == 2 ? s.x << 7 : s.x >> 1) & kExponent);
        d1 = __uint_as_float((G == 0 ? s.y << 23 : G == 1 ? s.y << 15 : G == 2 ? s.y << 7 : s.y >> 1) & kExponent);
    } else {
        const uint32_t a = G < 2 ? s.x : s.y, b = G < 2 ? s.z : s.w;
        const __half2 ha = *reinterpret_cast<const __half2 *>(&a), hb = *reinterpret_cast<const __half2 *>(&b);
        d0 = G & 1 ? __high2float(ha) : __low2float(ha);
        d1 = G & 1 ? __high2float(hb) : __low2float(hb);
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
// x   [step][group][part][NT tokens][32] f16, and c [step][group][NT tokens] f32: the start values of the group's products (Q4_0). NT,
// the tokens there is room for, is a template argument wherever they are read, so that the offsets inside a step are immediates.
// Activations with a scale of their own in every group (the experts' hidden rows) have, instead of c, f [step][group][NT tokens]
// (factor, start value) behind each step's x.
__host__ __device__ constexpr int step_x_bytes(int parts, int nt) { return 4 * parts * nt * 64; }
__host__ __device__ constexpr int step_c_bytes(bool mx, int nt) { return mx ? 0 : 4 * nt * 4; }
__host__ __device__ constexpr int step_bytes(bool mx, int parts, int nt) { return step_x_bytes(parts, nt) + step_c_bytes(mx, nt); }
__host__ __device__ constexpr int step_h_bytes(int nt) { return step_x_bytes(2, nt) + 4 * nt * 8; }
struct Staged {
    uint8_t * x;
    float * c;
};

template <int WARPS> struct Scratch {
    float factor[kRowList];                     // a token's sums times it are in the activations' own scale
    float ss[kMaxCluster][kRowList];            // sums of squares of each CTA's columns
    uint32_t top[WARPS];
    float squares[WARPS];
    uint64_t zero;                              // start values of PACK's lo columns
};

// 2^shift brings the magnitude with these bits into [2^13, 2^14), as far as it and the factor that takes it back (2^-8 - shift for MXFP4) are
// normal f32: below 2^-104 the values only come near, and are off by 2^-143 at most; above 2^113 the shift stays at -100, and from 65520 2^100 on, what an f16 rounds to
// infinity, they count as infinite. Rows with an infinity or a NaN are left as they are: their own
// sums become NaN, those of the other tokens stay what they are.
__device__ __forceinline__ int shift_for(uint32_t top) { return top > 0 && top < 0x7f800000u ? max(-100, min(118, 140 - (int)(top >> 23))) : 0; }
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// The power of two a sum is short of: of the weights' f16 form, and of MXFP4's scale bytes (kept plus 8).
__host__ __device__ constexpr int weight_shift(bool mx) { return mx ? -8 : 18; }
constexpr float kStart = -8.f * 3.814697265625e-6f;        // Q4_0's offset, in units of 2^-18

__device__ __forceinline__ uint32_t bits(const __half2 & h) { return *reinterpret_cast<const uint32_t *>(&h); }

// Four neighbouring scaled values as f16 (hi, and what it leaves) at `dst` and `dst + lo_at`.
template <int PARTS> __device__ __forceinline__ void put_split(uint8_t * dst, int lo_at, const float (&v)[4]) {
    const __half2 h0 = __floats2half2_rn(v[0], v[1]), h1 = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2 *>(dst) = make_uint2(bits(h0), bits(h1));
    if constexpr (PARTS == 2) {
        const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
        *reinterpret_cast<uint2 *>(dst + lo_at) = make_uint2(bits(__floats2half2_rn(v[0] - f0.x, v[1] - f0.y)), bits(__floats2half2_rn(v[2] - f1.x, v[3] - f1.y)));
    }
}

// Where a call's norm weights wait for its rows: 512 bytes for every step, four steps in each of `count` places `stride` bytes apart.
struct NormRoom {
    uint32_t base;
    int stride, count;
    __device__ __forceinline__ uint32_t at(int step) const { return base + (step >> 2) * stride + (step & 3) * 512; }
};

// Sixteen bytes of `from` (element size ES) to shared memory, asynchronously where their alignment allows it. Through the L2 cache only.
template <int ES> __device__ __forceinline__ void fetch16(uint32_t dst, const void * from, bool vec) {
    if (vec) {
        copy16(dst, static_cast<const uint8_t *>(from));
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (ES == 4) w[j] = __ldcg(static_cast<const unsigned *>(from) + j);
        else w[j] = __ldcg(static_cast<const unsigned short *>(from) + 2 * j) | (uint32_t)__ldcg(static_cast<const unsigned short *>(from) + 2 * j + 1) << 16;
    }
    store_u4(dst, w[0], w[1], w[2], w[3]);
}

// Four columns of a row as they are stored: f32 in .x to .w, halves in .x and .y.
__device__ __forceinline__ void widen4(const uint4 & u, uint32_t type, float (&v)[4]) {
    if (type == GGML_F32) {
        v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
    } else if (type == GGML_F16) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    } else {
        v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
        v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
    }
}
template <int PARTS> __device__ __forceinline__ uint32_t type_of(const Act & act) { return PARTS == 2 ? act.type : act.type == GGML_F16 ? GGML_F16 : GGML_BF16; }

// Columns k .. k + 3 of a row, through the L2 cache only.
__device__ __forceinline__ uint4 load4(const Act & act, uint32_t type, int64_t row, int k) {
    uint4 u = {};
    if (type == GGML_F32) {
        const unsigned * from = static_cast<const unsigned *>(act.p) + row * act.ld + k;
        if (act.vec) u = __ldcg(reinterpret_cast<const uint4 *>(from));
        else u = make_uint4(__ldcg(from), __ldcg(from + 1), __ldcg(from + 2), __ldcg(from + 3));
    } else {
        const unsigned short * from = static_cast<const unsigned short *>(act.p) + row * act.ld + k;
        if (act.vec) {
            const uint2 w = __ldcg(reinterpret_cast<const uint2 *>(from));
            u.x = w.x;
            u.y = w.y;
        } else {
            u.x = __ldcg(from) | (uint32_t)__ldcg(from + 1) << 16;
            u.y = __ldcg(from + 2) | (uint32_t)__ldcg(from + 3) << 16;
        }
    }
    return u;
}

// The largest magnitude (as bits: a NaN is above infinity, infinity above every number) and the sum of squares of a row that
// `shared` warps share. Every thread takes part.
template <int WARPS> __device__ __forceinline__ void row_totals(Scratch<WARPS> & sc, int shared, int part, uint32_t & top, float & squares) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    top = __reduce_max_sync(0xffffffffu, top);
    {
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
}

// Converts columns [k0, k0 + 128 steps) of n rows into the layout of nt tokens; columns at and behind n_in are zero. A row is one warp's
// work, or with few rows that of several warps, a step at a time. Up to kHeld steps a warp are held in registers. For more, all rows
// are first copied as they are, every 32 columns to where their converted form belongs (f32 fill the places of hi and lo, halves that of hi), so
// that the copies are in flight together; the largest magnitude and the conversion are two passes over shared memory. (Sixteen f32 tokens,
// 14336 x 4096 gated pair: 36 us; 38.6 us with registers in two batches and a second reading. One token, 4096 x 14336: 11.4 us in registers,
// 12.0 us through shared memory.) A function of its own, so that the product loops' registers do not depend on it. With `norm`, rows are multiplied by it,
// and put_squares(row, sum) gets the row's sum of squares. Every thread takes part; a barrier follows at the caller's.
template <bool MX, int PARTS, int WARPS, class PutSquares>
__device__ __noinline__ void stage_rows(const Act act, int n, int nt, int k0, int steps, int n_in, const float * norm, const NormRoom room, const Staged out,
                           Scratch<WARPS> & sc, PutSquares put_squares) {
    constexpr int kHeld = 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int shared = 1, log_shared = 0;     // warps that share a row
    while (2 * shared * n <= WARPS) { shared *= 2; ++log_shared; }
    const int part = warp & (shared - 1), row = warp >> log_shared;
    const int columns = min(steps * 128, n_in - k0);
    const bool live = row < n;          // there are as many warps as tokens, or more
    const uint32_t type = type_of<PARTS>(act);
    const int group_bytes = PARTS * nt * 64, lo = nt * 64;
    const bool norm_vec = norm && (reinterpret_cast<uintptr_t>(norm) & 15) == 0;
    uint32_t top = 0;
    float squares = 0.f, up = 1.f;
    auto count = [&](const float (&v)[4]) {
        if (norm) {
#pragma unroll
            for (int e = 0; e < 4; ++e) squares += v[e] * v[e];
        }
    };
    auto compare = [&](const float (&v)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    };
    auto totals = [&] {
        row_totals<WARPS>(sc, shared, part, top, squares);
        const int shift = shift_for(top);
        up = power(shift);
        if (live && part == 0 && lane == 0) {
            sc.factor[row] = power(weight_shift(MX) - shift);
            if (norm) put_squares(row, squares);
        }
    };
    // the lane's columns of a step in their final form; every lane has read what it needs of the place they go to
    auto put = [&](int step, float (&v)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= up;
        if constexpr (!MX) {
            float sum = (v[0] + v[1]) + (v[2] + v[3]);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if ((lane & 7) == 0) out.c[(step * 4 + (lane >> 3)) * nt + row] = sum * kStart;
        }
        put_split<PARTS>(out.x + (step * 4 + (lane >> 3)) * group_bytes + row * 64 + (lane & 7) * 8, lo, v);
    };

    if (steps <= kHeld << log_shared) {
        uint4 raw[kHeld], by[kHeld];
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int c = (part + (i << log_shared)) * 128 + lane * 4;
            raw[i] = by[i] = make_uint4(0, 0, 0, 0);
            if (live && c < columns) {
                raw[i] = load4(act, type, row, k0 + c);
                if (norm) by[i] = load4(Act{norm, 0, GGML_F32, norm_vec}, GGML_F32, 0, k0 + c);
            }
        }
        float v[kHeld][4];
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            widen4(raw[i], type, v[i]);
            count(v[i]);
            if (norm) {
                v[i][0] *= __uint_as_float(by[i].x); v[i][1] *= __uint_as_float(by[i].y); v[i][2] *= __uint_as_float(by[i].z); v[i][3] *= __uint_as_float(by[i].w);
            }
            compare(v[i]);
        }
        totals();
        if (!live) return;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int step = part + (i << log_shared);
            if (step >= steps) break;
            put(step, v[i]);
        }
        return;
    }

    const uint32_t slot = smem_address(out.x) + row * 64;
    const bool norm_staged = norm && steps <= 4 * room.count;
    if (norm_staged) {
        for (int i = threadIdx.x; i < steps * 32; i += WARPS * 32) {
            const uint32_t dst = room.at(i >> 5) + (i & 31) * 16;
            if (4 * i < columns) fetch16<4>(dst, norm + k0 + 4 * i, norm_vec);
            else store_u4(dst, 0, 0, 0, 0);
        }
    }
    if (live) {
        if (type == GGML_F32) {
            const float * from = static_cast<const float *>(act.p) + row * act.ld + k0;
            for (int step = part; step < steps; step += shared) {
                const uint32_t dst = slot + (step * 4 + (lane >> 3)) * group_bytes + (lane & 4 ? lo : 0) + (lane & 3) * 16;
                const int c = step * 128 + lane * 4;
                if (c < columns) fetch16<4>(dst, from + c, act.vec);
                else store_u4(dst, 0, 0, 0, 0);
            }
        } else {                        // two of the warp's steps at a time
            const uint16_t * from = static_cast<const uint16_t *>(act.p) + row * act.ld + k0;
            for (int step = part + ((lane >> 4) << log_shared); step < steps; step += 2 * shared) {
                const uint32_t dst = slot + (step * 4 + ((lane & 15) >> 2)) * group_bytes + (lane & 3) * 16;
                const int c = step * 128 + (lane & 15) * 8;
                if (c < columns) fetch16<2>(dst, from + c, act.vec);
                else store_u4(dst, 0, 0, 0, 0);
            }
        }
    }
    copies_commit();
    copies_wait<0>();
    __syncthreads();

    auto read = [&](int step, float (&v)[4]) {
        const uint32_t at = slot + (step * 4 + (lane >> 3)) * group_bytes;
        uint4 u = {};
        if (type == GGML_F32) {
            u = shared_u4(at + (lane & 4 ? lo : 0) + (lane & 3) * 16);
        } else {
            const uint2 w = shared_u2(at + (lane & 7) * 8);
            u.x = w.x;
            u.y = w.y;
        }
        widen4(u, type, v);
    };
    auto weigh = [&](int step, float (&v)[4]) {
        if (norm) {
            uint4 by = {};
            const int c = step * 128 + lane * 4;
            if (norm_staged) by = shared_u4(room.at(step) + lane * 16);
            else if (c < columns) by = load4(Act{norm, 0, GGML_F32, norm_vec}, GGML_F32, 0, k0 + c);
            v[0] *= __uint_as_float(by.x); v[1] *= __uint_as_float(by.y); v[2] *= __uint_as_float(by.z); v[3] *= __uint_as_float(by.w);
        }
    };
    if (live) {
#pragma unroll 2
        for (int step = part; step < steps; step += shared) {
            float v[4];
            read(step, v);
            count(v);
            weigh(step, v);
            compare(v);
        }
    }
    totals();
    if (!live) return;
#pragma unroll 2
    for (int step = part; step < steps; step += shared) {
        float v[4];
        read(step, v);
        weigh(step, v);
        __syncwarp();
        put(step, v);
    }
}

// The rows of a call's tokens, normalised by its weights when it has any. A row's squares go to every CTA of the cluster.
template <bool MX, int PARTS, int WARPS>
__device__ __forceinline__ void stage_tokens(const Act & act, int n, int nt, int k0, int steps, int n_in, const float * norm, const NormRoom & room,
                                             const Staged & out, Scratch<WARPS> & sc, int rank, int C) {
    cluster_wait();
    stage_rows<MX, PARTS, WARPS>(act, n, nt, k0, steps, n_in, norm, room, out, sc, [&](int t, float squares) {
        for (int c = 0; c < C; ++c) remote_store(remote_address(smem_address(&sc.ss[rank][t]), c), squares);
    });
}

// 1 / sqrt(mean of squares + eps) of token t, once the cluster has met after stage_tokens.
template <int WARPS> __device__ __forceinline__ float rms_factor(const Scratch<WARPS> & sc, int t, int C, int n_in, float eps) {
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
};

// Where a lane finds its B fragments and start values, and the factors of its columns' sums.
struct Lane {
    uint32_t b[2], c[2][2];             // shared-memory addresses at the group's first step
    uint32_t c_step, c_group;
    float factor[2][2];
};

// OWN: every group of columns has factors of its own (see Staged).
template <bool MX, int PARTS, int MODE, int NT, bool LIST, bool OWN, class S>
__device__ __forceinline__ void begin_group(const Group & r, int lane, const S & sc, Lane & l) {
    constexpr int NC = MODE == TWO ? 2 : 1;
    const int g = lane >> 2, t4 = lane & 3;
    constexpr bool lo = MODE == PACK;
    const uint32_t x = smem_address(r.x.x), c = OWN ? x + step_x_bytes(PARTS, NT) : MX ? 0 : smem_address(r.x.c);
    auto place = [&](int col) { const int i = min(col, r.n - 1); return LIST ? (int)r.list[i] : i; };
    l.b[0] = x + place(lo ? g & 3 : g) * 64 + t4 * 16 + (lo && g >= 4 ? NT * 64 : 0);
    if constexpr (NC == 2) l.b[1] = x + place(g + 8) * 64 + t4 * 16;
    l.c_step = OWN ? step_h_bytes(NT) : step_c_bytes(MX, NT);
    l.c_group = NT * (OWN ? 8 : 4);
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int tok = place(lo ? (2 * t4 + e) & 3 : 8 * nc + 2 * t4 + e);
            l.c[nc][e] = c + tok * (OWN ? 8 : 4);
            if constexpr (!OWN) l.factor[nc][e] = sc.factor[tok];
        }
    if constexpr (!MX && lo && !OWN) {
        if (t4 >= 2) {              // the lo columns carry no offset
            l.c[0][0] = l.c[0][1] = smem_address(&sc.zero);
            l.c_step = l.c_group = 0;
        }
    }
}

// Products of group G of a unit. NT == 1: every MMA column is the one token, and only the even ones are kept.
template <bool MX, int PARTS, int MODE, int NT, bool OWN, int G>
__device__ __forceinline__ void do_group(const Words & u, const Scales<MX> & sc, uint32_t b_at, uint32_t c_at, const Lane & l, int lane, float (&acc)[2][2][4]) {
    constexpr int NC = MODE == TWO ? 2 : 1;
    constexpr int NP = MODE == PACK ? 1 : PARTS;
    uint4 b[NC][NP];
    float start[NC][2], factor[NC][2];
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
#pragma unroll
        for (int p = 0; p < NP; ++p) b[nc][p] = shared_u4(l.b[nc] + b_at + (G * PARTS + p) * (NT * 64));
        start[nc][0] = start[nc][1] = 0.f;
        if constexpr (OWN) {
#pragma unroll
            for (int e = 0; e < (NT == 1 ? 1 : 2); ++e) {
                const uint2 fs = shared_u2(l.c[nc][e] + c_at + G * (NT * 8));
                factor[nc][e] = __uint_as_float(fs.x);
                if constexpr (!MX) start[nc][e] = MODE == PACK && (lane & 2) ? 0.f : __uint_as_float(fs.y);
            }
            if constexpr (NT == 1) start[nc][1] = start[nc][0];
        } else if constexpr (!MX) {
            const uint32_t at = c_at + (MODE == PACK ? G * l.c_group : G * (NT * 4));      // PACK: the zero has no groups
            start[nc][0] = shared_f1(l.c[nc][0] + at);
            start[nc][1] = NT == 1 ? start[nc][0] : shared_f1(l.c[nc][1] + at);
        }
    }
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
        float c[NC][4];
        uint32_t a[4];
        decode<MX, G & 1, 0>(u.q[tile], a);
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            mma_start(c[nc], a, b[nc][0].x, b[nc][0].y, start[nc][0], start[nc][1]);
            if constexpr (NP == 2) mma(c[nc], a, b[nc][NP - 1].x, b[nc][NP - 1].y);
        }
        decode<MX, G & 1, 1>(u.q[tile], a);
#pragma unroll
        for (int nc = 0; nc < NC; ++nc)
#pragma unroll
            for (int p = 0; p < NP; ++p) mma(c[nc], a, b[nc][p].z, b[nc][p].w);
        float d0, d1;
        scales<MX, G>(sc.s[tile], d0, d1);
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            if constexpr (OWN) {
                c[nc][0] *= factor[nc][0];
                c[nc][2] *= factor[nc][0];
                if constexpr (NT > 1) { c[nc][1] *= factor[nc][1]; c[nc][3] *= factor[nc][1]; }
            }
            acc[tile][nc][0] += d0 * c[nc][0];
            acc[tile][nc][2] += d1 * c[nc][2];
            if constexpr (NT > 1) {
                acc[tile][nc][1] += d0 * c[nc][1];
                acc[tile][nc][3] += d1 * c[nc][3];
            }
        }
    }
}

// One unit, whose words and scales the lane finds at `words` and `scale_at`.
template <bool MX, int PARTS, int MODE, int NT, bool OWN>
__device__ __forceinline__ void do_step(uint32_t words, uint32_t scale_at, uint32_t b_at, uint32_t c_at, const Lane & l, int lane, float (&acc)[2][2][4]) {
    Scales<MX> sc;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        if constexpr (MX) {
            const uint2 v = shared_u2(scale_at + t * 64);
            sc.s[t].x = v.x;
            sc.s[t].y = v.y;
        } else {
            sc.s[t] = shared_u4(scale_at + t * 128);
        }
    }
    Words u;
    u.q[0] = shared_u4(words);
    u.q[1] = shared_u4(words + 512);
    do_group<MX, PARTS, MODE, NT, OWN, 0>(u, sc, b_at, c_at, l, lane, acc);
    do_group<MX, PARTS, MODE, NT, OWN, 1>(u, sc, b_at, c_at, l, lane, acc);
    u.q[0] = shared_u4(words + 1024);
    u.q[1] = shared_u4(words + 1536);
    do_group<MX, PARTS, MODE, NT, OWN, 2>(u, sc, b_at, c_at, l, lane, acc);
    do_group<MX, PARTS, MODE, NT, OWN, 3>(u, sc, b_at, c_at, l, lane, acc);
}

// Hands on a run's sums and clears them: begin(column), then put(row - lane / 4, sum) for the lane's four rows of the block.
template <int MODE, int NT, bool OWN, class Begin, class Put>
__device__ __forceinline__ void end_run(int n, int lane, const Lane & l, float (&acc)[2][2][4], Begin begin, Put put) {
    const int t4 = lane & 3;
#pragma unroll
    for (int nc = 0; nc < (MODE == TWO ? 2 : 1); ++nc)
#pragma unroll
        for (int e = 0; e < (NT > 1 ? 2 : 1); ++e) {
            const int col = 8 * nc + 2 * t4 + e;
            const bool mine = col < n && !(MODE == PACK && t4 >= 2);
            if constexpr (MODE == PACK) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float & a = acc[i >> 1][nc][e + 2 * (i & 1)];
                    a += __shfl_xor_sync(0xffffffffu, a, 2);        // hi column + lo column
                }
            }
            if (mine) {
                begin(col);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = acc[i >> 1][nc][e + 2 * (i & 1)];
                    put(i * 8, OWN ? a : a * l.factor[nc][e]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i >> 1][nc][e + 2 * (i & 1)] = 0.f;
        }
}

// Where a warp is in its sequence of runs.
struct Cursor {
    const uint8_t * p;          // the lane's part of the next unit
    int rem;                    // units left in the run
    int group, job;             // the Source's
    bool live;
};

// Runs a warp's sequence. Source: first(Cursor &) and next(Cursor &) move to a run (never an empty one) and set everything;
// group(const Cursor &) describes the activations; column(const Cursor &, column) is the cluster address that takes 32 rows' sums.
// LIST: groups name their tokens.
template <bool MX, int STAGES, class Source> struct Stream {
    static constexpr int kStages = STAGES;
    static constexpr uint32_t kUnit = w4_unit_bytes(MX);
    const Source & src;
    const int lane;
    const uint32_t ring;        // the lane's first word in the warp's ring
    Cursor ld, cp;
    uint32_t fill, at;          // ring offsets of the stage to fill and the stage to multiply

    __device__ __forceinline__ Stream(const Source & s, uint8_t * rings)
        : src(s), lane(threadIdx.x & 31), ring(smem_address(rings) + (threadIdx.x >> 5) * (kStages * kUnit) + lane * 16), fill(0), at(0) {
        src.first(ld);
        cp = ld;
    }
    __device__ __forceinline__ void fetch() {
        if (ld.live) {
            const uint32_t dst = ring + fill;
#pragma unroll
            for (int i = 0; i < 4; ++i) copy16(dst + i * 512, ld.p + i * 512);
            if (lane < (MX ? 8 : 16)) copy16(dst + 2048, ld.p + 2048);
            ld.p += kUnit;
            if (--ld.rem == 0) src.next(ld);
        }
        fill = fill == (kStages - 1) * kUnit ? 0 : fill + kUnit;
        copies_commit();
    }
    // The first units of the sequence; needs nothing but the weights. The ring must be free: a barrier lies between its last reads and this.
    __device__ __forceinline__ void prefetch() {
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) fetch();
    }
    // All runs of the cursor's group whose job is below `limit`.
    template <int PARTS, int MODE, int NT, bool LIST, bool OWN, class S> __device__ __forceinline__ void work_group(const Group & r, const S & sc, int limit) {
        float acc[2][2][4] = {};
        Lane l;
        begin_group<MX, PARTS, MODE, NT, LIST, OWN>(r, lane, sc, l);
        const int group = cp.group;
        const uint32_t scale_at = ring - lane * 16 + 2048 + (lane >> 2) * (MX ? 8 : 16);
        do {
            uint32_t b_at = 0, c_at = 0;
            for (int n = cp.rem; n > 0; --n) {
                copies_wait<kStages - 2>();
                __syncwarp();           // every lane's copies of this unit have landed, and the stage read last is free
                fetch();
                do_step<MX, PARTS, MODE, NT, OWN>(ring + at, scale_at + at, b_at, c_at, l, lane, acc);
                at = at == (kStages - 1) * kUnit ? 0 : at + kUnit;
                b_at += OWN ? step_h_bytes(NT) : step_x_bytes(PARTS, NT);
                c_at += l.c_step;
            }
            uint32_t to = 0;
            end_run<MODE, NT, OWN>(r.n, lane, l, acc, [&](int col) { to = src.column(cp, col) + (lane >> 2) * 4; }, [&](int row, float v) { remote_store(to + row * 4, v); });
            src.next(cp);
        } while (cp.live && cp.group == group && cp.job < limit);
    }
    // The runs of jobs below `limit`. Token sets staged with room for NT tokens, whose groups hold up to NT of them.
    template <int PARTS, int NT, bool LIST, class S> __device__ __forceinline__ void work(const S & sc, int limit) {
        while (cp.live && cp.job < limit) {
            const Group r = src.group(cp);
            if constexpr (!LIST) work_group<PARTS, mode_of(NT, PARTS), NT, LIST, false>(r, sc, limit);
            else {
                const int mode = mode_of(r.n, PARTS);
                if (PARTS == 2 && mode == PACK) work_group<PARTS, PARTS == 2 ? PACK : ONE, NT, LIST, false>(r, sc, limit);
                if constexpr (NT > (PARTS == 2 ? 4 : 0)) if (mode == ONE) work_group<PARTS, ONE, NT, LIST, false>(r, sc, limit);
                if constexpr (NT > 8) if (mode == TWO) work_group<PARTS, TWO, NT, LIST, false>(r, sc, limit);
            }
        }
    }
};

// Parts (a power of two) the warps split the columns of a job into: as few as keep the warps evenly loaded, and at most `most`.
// Warp w takes part w % ks of jobs w / ks, w / ks + warps / ks, ... The cost counts steps of the busiest warp and one and a half steps' time
// for every sum it hands on.
__host__ __device__ inline int split_columns(int jobs, int steps, int warps, int most) {
    int best = 1, best_cost = 0x7fffffff;
    for (int ks = 1; ks <= warps && ks <= most; ks *= 2) {
        if (ks > 1 && ks > steps) break;
        const int rounds = (jobs * ks + warps - 1) / warps;
        const int cost = rounds * (2 * ((steps + ks - 1) / ks) + 3);
        if (cost < best_cost) { best_cost = cost; best = ks; }
    }
    return best;
}

// The same with any number of parts, where warps / ks jobs run side by side; and its cost.
inline int divide_columns(int jobs, int steps, int warps, int most, int & cost) {
    int best = 1;
    cost = 0x7fffffff;
    for (int ks = 1; ks <= warps && ks <= most && (ks == 1 || ks <= steps); ++ks) {
        const int abreast = warps / ks, rounds = (jobs + abreast - 1) / abreast;
        const int c = rounds * (2 * ((steps + ks - 1) / ks) + 3);
        if (c < cost) { cost = c; best = ks; }
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

    // The cluster address of 32 rows' sums.
    __device__ __forceinline__ uint32_t slot(int round, int unit, int which, int sub) const {
        const int from = (((unit >> log_c) * per + which) << log_c | rank) * ks + sub;
        return remote_address(base + (round & 1) * bytes + from * 128, unit & ((1 << log_c) - 1));
    }
    // Row `lane` of the sum over the cluster for the CTA's own unit number `mine`, in the order of the columns.
    __device__ __forceinline__ float sum(int round, int mine, int which) const {
        const int n = ks << log_c;
        const uint32_t at = base + (round & 1) * bytes + ((mine * per + which) * n * 32 + (threadIdx.x & 31)) * 4;
        float v = 0.f;
#pragma unroll 8
        for (int i = 0; i < n; ++i) v += shared_f1(at + i * 128);
        return v;
    }
};
// Bytes of one inbox for `units` units of a round.
__host__ __device__ inline int64_t inbox_bytes(int64_t units, int C, int ks, int per) { return (units + C - 1) / C * per * C * ks * 128; }
// Row blocks a round takes with `room` bytes for one inbox: at least one, and where possible so many that every warp has the same number of runs.
__host__ __device__ inline int blocks_per_round(int64_t room, int tokens, int C, int ks, int per, int warps) {
    const int units = (int)(room / (per * C * ks * 128)) * C;       // whole units in every CTA
    const int blocks = units / tokens, even = (warps + ks * per - 1) / (ks * per);
    return blocks < 1 ? 1 : blocks > even ? blocks - blocks % even : blocks;
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
    int each, more;                 // row blocks of a cluster (one more in the first `more`), of gate and up together as of one matrix
    int x_bytes, c_bytes, inbox;    // shared memory: staged activations, start values, one inbox
    int ks, per_round;              // parts of the columns and blocks of a round, the same in every cluster: one inbox may have to do
};

// Jobs: a row block; with the gate, block j of gate and of up are jobs 2 j and 2 j + 1.
template <bool MX, int PARTS, bool GLU, int NT> struct ProductSource {
    const ProductArgs & a;
    Staged x;                   // from this warp's columns on
    Inbox inbox;
    int job0, jobs;             // jobs job0 .. job0 + jobs - 1
    int first_job, stride;      // this warp's
    int sub, step, len;         // its columns
    int round, round0;          // the round, and its first job

    __device__ __forceinline__ void point(Cursor & c) const {
        c.live = c.job < jobs;
        const int job = job0 + c.job;
        const size_t block = GLU ? job >> 1 : job;
        c.p = (GLU && (job & 1) ? a.u : a.w) + (block * a.steps + step) * w4_unit_bytes(MX) + (threadIdx.x & 31) * 16;
        c.rem = len;
    }
    __device__ __forceinline__ void first(Cursor & c) const {
        c.group = 0;
        c.job = first_job;
        point(c);
    }
    __device__ __forceinline__ void next(Cursor & c) const {
        c.job += stride;
        point(c);
    }
    __device__ __forceinline__ Group group(const Cursor &) const { return {x, nullptr, a.T}; }
    __device__ __forceinline__ uint32_t column(const Cursor & c, int col) const {
        const int job = c.job - round0;
        return inbox.slot(round, (GLU ? job >> 1 : job) * a.T + col, GLU ? job & 1 : 0, sub);
    }
};

template <bool MX, int PARTS, bool GLU, int NT>
__global__ void __launch_bounds__(warps_for(NT) * 32, resident_for(NT)) w4_product_kernel(ProductArgs a) {
    constexpr int kWarps = warps_for(NT);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Scratch<kWarps> sc;
    constexpr int kPer = GLU ? 2 : 1;           // jobs of a row block
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), C = (int)cluster_size(), log_c = __ffs(C) - 1;
    const int cluster = blockIdx.x >> log_c;
    cluster_arrive();
    const int s0 = part_begin2(a.steps, rank, log_c), n_steps = part_begin2(a.steps, rank + 1, log_c) - s0;
    const int b_begin = cluster * a.each + min(cluster, a.more), blocks = a.each + (cluster < a.more);
    const int ks = a.ks, log_ks = __ffs(ks) - 1;
    uint8_t * const rings = smem + a.x_bytes + a.c_bytes;
    const Staged x{smem, reinterpret_cast<float *>(smem + a.x_bytes)};
    const Inbox inbox{smem_address(rings + ring_bytes(MX, NT, stages_for(NT, PARTS))), a.inbox, rank, log_c, ks, kPer};
    const int sub = warp & (ks - 1), step = part_begin2(n_steps, sub, log_ks), len = part_begin2(n_steps, sub + 1, log_ks) - step;
    const Staged x_warp{x.x + step * step_x_bytes(PARTS, NT), x.c + step * step_c_bytes(MX, NT) / 4};
    if (threadIdx.x == 0) sc.zero = 0;

    ProductSource<MX, PARTS, GLU, NT> src{a, x_warp, inbox, b_begin * kPer, blocks * kPer, warp >> log_ks, kWarps >> log_ks, sub, s0 + step, len, 0, 0};
    Stream<MX, stages_for(NT, PARTS), ProductSource<MX, PARTS, GLU, NT>> stream(src, rings);
    stream.prefetch();
    // the weights above are the library's own; everything below is the caller's
    pdl_trigger();
    pdl_wait();
    // the norm's weights wait in the last stage of every warp's ring, which the first units leave free
    using Ring = Stream<MX, stages_for(NT, PARTS), ProductSource<MX, PARTS, GLU, NT>>;
    const NormRoom room{smem_address(rings) + (Ring::kStages - 1) * Ring::kUnit, (int)(Ring::kStages * Ring::kUnit), kWarps};
    stage_tokens<MX, PARTS>(a.x, a.T, NT, s0 * 128, n_steps, a.n_in, a.norm, room, x, sc, rank, C);
    __syncthreads();
    for (int b0 = 0; b0 < blocks; b0 += a.per_round, ++src.round) {
        const int now = min(a.per_round, blocks - b0);
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
// kilobytes that the L2 cache holds; a CTA reads its columns of it), then multiplies its share of the chosen
// experts' gate and up blocks and writes h = w_e silu(a) b for each (token, expert) pair, split into hi + lo f16 with a power of two for every
// 32 columns: what the second kernel's products take. That one treats the chosen experts' down matrices as one long reduction: a cluster
// owns a range of y's rows, its CTAs and their warps divide the experts' concatenated columns, every unit of weights arrives
// in a warp's ring together with the hidden columns it multiplies, and the sum over experts is part of the sum over the cluster. An
// expert of more than three tokens is visited once per three of them (its weights then come from the L2 cache).

constexpr int kSet = 3;                 // tokens of an expert the second kernel takes at once
constexpr int kMaxPairs = kRowList * kW4MaxUsed;

// The routing's result, in shared memory and for the second kernel in the workspace in front of the hidden columns: a header {chosen experts, sets, -, -}, then arrays
// at these bytes, each long enough for `experts` chosen experts and `pairs` (token, expert) pairs.
struct RouteAt {
    int expert, before, cost;               // of the chosen experts, ascending: u16 id; u16 pairs before it; i32 cost of the blocks before it (one more of the latter two)
    int weight, token;                      // of the pairs, by expert: f32, u8
    int set_expert, set_first, set_count;   // up to kSet tokens of an expert: u16 id, u16 first pair, u8 count
    int bytes;
};
__host__ __device__ constexpr RouteAt route_at(int experts, int pairs) {
    RouteAt r{};
    const auto up16 = [](int n) { return (n + 15) / 16 * 16; };
    r.expert = 16;
    r.before = r.expert + up16(2 * experts);
    r.cost = r.before + up16(2 * (experts + 1));
    r.weight = r.cost + up16(4 * (experts + 1));
    r.token = r.weight + up16(4 * pairs);
    r.set_expert = r.token + up16(pairs);
    r.set_first = r.set_expert + up16(2 * pairs);
    r.set_count = r.set_first + up16(2 * pairs);
    r.bytes = r.set_count + up16(pairs);
    return r;
}
constexpr int kRouteBytes = route_at(kW4MaxExperts, kMaxPairs).bytes;

// A copy of it in shared memory.
struct Route {
    const uint8_t * p;
    RouteAt at;
    __device__ __forceinline__ int experts() const { return reinterpret_cast<const int *>(p)[0]; }
    __device__ __forceinline__ int sets() const { return reinterpret_cast<const int *>(p)[1]; }
    __device__ __forceinline__ int expert(int u) const { return reinterpret_cast<const uint16_t *>(p + at.expert)[u]; }
    __device__ __forceinline__ int before(int u) const { return reinterpret_cast<const uint16_t *>(p + at.before)[u]; }
    __device__ __forceinline__ int count(int u) const { return before(u + 1) - before(u); }
    __device__ __forceinline__ int cost(int u) const { return reinterpret_cast<const int *>(p + at.cost)[u]; }
    __device__ __forceinline__ float weight(int pair) const { return reinterpret_cast<const float *>(p + at.weight)[pair]; }
    __device__ __forceinline__ const uint8_t * tokens(int pair) const { return p + at.token + pair; }
    __device__ __forceinline__ int set_expert(int i) const { return reinterpret_cast<const uint16_t *>(p + at.set_expert)[i]; }
    __device__ __forceinline__ int set_first(int i) const { return reinterpret_cast<const uint16_t *>(p + at.set_first)[i]; }
    __device__ __forceinline__ int set_count(int i) const { return p[at.set_count + i]; }
    // Units are the (block, token) results of the chosen experts' blocks, one behind the other: the first of a block.
    __device__ __forceinline__ int unit(int u, int block, int blocks) const { return before(u) * blocks + block * count(u); }
};

// Copies the header and bytes [from, to) of a route, through the L2 cache only. A barrier follows at the caller's.
__device__ __forceinline__ void copy_route(const uint8_t * route, uint8_t * copy, int from, int to) {
    for (int i = threadIdx.x; i < 1 + (to - from) / 16; i += blockDim.x) {
        const int at = i == 0 ? 0 : from + 16 * (i - 1);
        *reinterpret_cast<uint4 *>(copy + at) = __ldcg(reinterpret_cast<const uint4 *>(route + at));
    }
}

// What a block of an expert with n tokens costs, in parts of the time its weights take: 0.63 us for the two matrices' blocks of 32 x 2880 in a cluster
// of four, 0.045 us more for each token's sums, 0.2 us more where the tokens' hi and lo are products of their own.
__device__ __forceinline__ int block_cost(int n, int parts) { return 14 + n + (n > 8 ? 5 * parts : n > 4 && parts == 2 ? 5 : 0); }

// Hidden columns: by set, by 128-column step, [group][part][token][32] f16, then [group][token] (factor, start value).
constexpr int kHiddenBytes = 544;       // of one token and step
static_assert(step_h_bytes(1) == kHiddenBytes && step_h_bytes(kSet) == kSet * kHiddenBytes, "a set's bytes are its tokens'");

struct MoeArgs {
    const uint8_t * gate, * up, * down;
    size_t gate_expert, up_expert, down_expert;     // bytes of one expert
    const float * router;
    bool router_vec;            // sixteen bytes of it may be read at once
    bool down_mx;
    int parts;
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
    uint8_t * route;
    RouteAt at;
    uint8_t * hidden;
    int clusters, x_bytes, c_bytes, logit_bytes, inbox, partial;        // shared memory, in bytes
    int ks, per_round;          // of the second kernel: parts of the columns, blocks of a round
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
        for (int i = threadIdx.x; i < a.E * chunks; i += blockDim.x) {
            const int e = i / chunks, c = i - e * chunks;
            copy16(dst + i * 16, reinterpret_cast<const uint8_t *>(a.router + (size_t)e * a.d + k + c * 4));
        }
    } else {
        for (int i = threadIdx.x; i < a.E * n; i += blockDim.x) {
            const int e = i / n, c = i - e * n;
            reinterpret_cast<float *>(to)[i] = a.router[(size_t)e * a.d + k + c];
        }
    }
}

// The CTA's columns' part of every (token, expert) logit, from the staged activations and, piece by piece, the router in
// `room` (the first piece is already on its way). The sums are in the staged activations' scale.
template <bool MX, int PARTS, int NT, int WARPS>
__device__ void partial_logits(const MoeArgs & a, int k0, int k1, const Staged & x, uint8_t * room, int room_bytes, float * out) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int EB = 4, TB = NT == 1 ? 1 : 4;         // experts and tokens a warp takes at once
    const int width = router_columns(a.E, room_bytes);
    const int groups_t = (a.T + TB - 1) / TB, items = (a.E + EB - 1) / EB * groups_t;
    for (int k = k0; k < k1; k += width) {
        const int n = min(width, k1 - k);
        if (k > k0) {
            __syncthreads();
            fetch_router(a, k, n, room);
            copies_commit();
        }
        copies_wait<0>();
        __syncthreads();
        const float * r = reinterpret_cast<const float *>(room);
        for (int item = warp; item < items; item += WARPS) {
            const int e0 = item / groups_t * EB, t0 = (item - item / groups_t * groups_t) * TB;
            float acc[16] = {};
            for (int c = lane * 4; c < n; c += 128) {
                const int at = k - k0 + c, step = at >> 7, group = (at >> 5) & 3;
                float4 w[EB];
#pragma unroll
                for (int e = 0; e < EB; ++e) w[e] = *reinterpret_cast<const float4 *>(r + min(e0 + e, a.E - 1) * n + c);
#pragma unroll
                for (int t = 0; t < TB; ++t) {
                    const uint8_t * p = x.x + ((step * 4 + group) * PARTS * NT + min(t0 + t, a.T - 1)) * 64 + (at & 31) * 2;
                    const uint2 h = *reinterpret_cast<const uint2 *>(p);
                    float2 v0 = __half22float2(*reinterpret_cast<const __half2 *>(&h.x)), v1 = __half22float2(*reinterpret_cast<const __half2 *>(&h.y));
                    if constexpr (PARTS == 2) {
                        const uint2 l = *reinterpret_cast<const uint2 *>(p + NT * 64);
                        const float2 l0 = __half22float2(*reinterpret_cast<const __half2 *>(&l.x)), l1 = __half22float2(*reinterpret_cast<const __half2 *>(&l.y));
                        v0.x += l0.x; v0.y += l0.y; v1.x += l1.x; v1.y += l1.y;
                    }
#pragma unroll
                    for (int e = 0; e < EB; ++e)
                        acc[e * TB + t] += w[e].x * v0.x + w[e].y * v0.y + w[e].z * v1.x + w[e].w * v1.y;
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

// Softmax over the experts and the n_used likeliest of one token, by one warp: pick i is lane i's. Ties go to the lowest index; whatever the
// logits hold, k different experts are chosen (a NaN makes the weights NaN). PER: experts of a lane.
template <int PER, class Logit> __device__ __forceinline__ void pick_experts(Logit logit, int E, int k, bool normalise, int & expert, float & weight) {
    const int lane = threadIdx.x & 31;
    float p[PER];
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = lane + 32 * j;
        p[j] = e < E ? logit(e) : -INFINITY;
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
    // key: the probability's bits, which order like the probabilities, plus two; a NaN behind every number, taken ones at zero
    uint32_t key[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        p[j] /= sum;
        key[j] = lane + 32 * j < E ? (p[j] >= 0.f ? __float_as_uint(p[j]) + 2u : 1u) : 0u;
    }
    float chosen = 0.f;
    expert = 0;
    weight = 0.f;
    for (int pick = 0; pick < k; ++pick) {
        uint32_t best = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) best = max(best, key[j]);
        best = __reduce_max_sync(0xffffffffu, best);
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int j = PER - 1; j >= 0; --j) if (key[j] == best) at = lane + 32 * j;
        at = __reduce_min_sync(0xffffffffu, at);
        float value = 0.f;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (at == (uint32_t)(lane + 32 * j)) {
                value = p[j];
                key[j] = 0;
            }
        }
        value = __shfl_sync(0xffffffffu, value, at & 31);
        if (lane == pick) { expert = (int)at; weight = value; }
        chosen += value;
    }
    if (normalise) weight /= chosen;
}

// What the lists are made from.
struct Picks {
    uint32_t expert[kMaxPairs];                 // of all tokens, likeliest first
    float weight[kMaxPairs];
    uint32_t mask[kW4MaxExperts];               // by expert: the tokens that chose it
    uint16_t before[kW4MaxExperts];             // pairs of the experts before
    int totals[4][8];
};

// Writes the lists of the chosen experts, ascending, from the picks of all tokens. Picks::mask is zero before; a barrier follows at the caller's.
__device__ void write_route(const MoeArgs & a, Picks & p, uint8_t * route) {
    const int e = threadIdx.x, warp = e >> 5, lane = e & 31;
    const int pairs = a.T * a.k;
    for (int i = e; i < pairs; i += blockDim.x) atomicOr(&p.mask[p.expert[i]], 1u << (i / a.k));
    __syncthreads();
    const uint32_t mask = e < (int)kW4MaxExperts ? p.mask[e] : 0;      // tokens that chose expert e
    const int n = __popc(mask), sets = (n + kSet - 1) / kSet;
    // chosen experts, pairs, sets and cost before this one: inside the warp, then over the eight warps that hold experts
    const int own[4] = {n > 0 ? 1 : 0, n, sets, n > 0 ? a.blocks_ff * block_cost(n, a.parts) : 0};
    int sum[4] = {own[0], own[1], own[2], own[3]};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int v = __shfl_up_sync(0xffffffffu, sum[i], o);
            if (lane >= o) sum[i] += v;
        }
    }
    if (warp < 8 && lane == 31) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p.totals[i][warp] = sum[i];
    }
    __syncthreads();
    int before[4], all[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        before[i] = sum[i] - own[i];
        all[i] = 0;
        for (int w = 0; w < 8; ++w) {
            if (w < warp) before[i] += p.totals[i][w];
            all[i] += p.totals[i][w];
        }
    }
    if (mask) {
        const int u = before[0];
        reinterpret_cast<uint16_t *>(route + a.at.expert)[u] = (uint16_t)e;
        reinterpret_cast<uint16_t *>(route + a.at.before)[u] = (uint16_t)before[1];
        reinterpret_cast<int *>(route + a.at.cost)[u] = before[3];
        p.before[e] = (uint16_t)before[1];
        for (int j = 0; j < sets; ++j) {
            reinterpret_cast<uint16_t *>(route + a.at.set_expert)[before[2] + j] = (uint16_t)e;
            reinterpret_cast<uint16_t *>(route + a.at.set_first)[before[2] + j] = (uint16_t)(before[1] + kSet * j);
            route[a.at.set_count + before[2] + j] = (uint8_t)min(kSet, n - kSet * j);
        }
    }
    if (e == 0) {
        reinterpret_cast<uint16_t *>(route + a.at.before)[all[0]] = (uint16_t)all[1];
        reinterpret_cast<int *>(route + a.at.cost)[all[0]] = all[3];
        *reinterpret_cast<int4 *>(route) = make_int4(all[0], all[2], 0, 0);
    }
    __syncthreads();
    for (int i = e; i < pairs; i += blockDim.x) {               // an expert's tokens ascend
        const int t = i / a.k, at = p.before[p.expert[i]] + __popc(p.mask[p.expert[i]] & ((1u << t) - 1));
        route[a.at.token + at] = (uint8_t)t;
        reinterpret_cast<float *>(route + a.at.weight)[at] = p.weight[i];
    }
}

// Jobs: block j of an expert's gate and of its up matrix are jobs 2 j and 2 j + 1, experts one behind the other.
template <bool MX, int PARTS, int NT> struct GateUpSource {
    const MoeArgs & a;
    const Route & r;
    Staged x;
    Inbox inbox;
    int job0, jobs;
    int first_job, stride;
    int sub, step, len;
    int round, unit0;           // the round, and its first unit

    // Cursor::group is the expert's place among the chosen ones.
    __device__ __forceinline__ void point(Cursor & c) const {
        c.live = c.job < jobs;
        if (!c.live) return;
        const int job = job0 + c.job, block = job >> 1;
        c.group = block / a.blocks_ff;
        const int e = r.expert(c.group);
        c.p = (job & 1 ? a.up + e * a.up_expert : a.gate + e * a.gate_expert) +
              ((size_t)(block - c.group * a.blocks_ff) * a.steps_d + step) * w4_unit_bytes(MX) + (threadIdx.x & 31) * 16;
        c.rem = len;
    }
    __device__ __forceinline__ void first(Cursor & c) const {
        c.job = first_job;
        point(c);
    }
    __device__ __forceinline__ void next(Cursor & c) const {
        c.job += stride;
        point(c);
    }
    __device__ __forceinline__ Group group(const Cursor & c) const { return {x, r.tokens(r.before(c.group)), r.count(c.group)}; }
    __device__ __forceinline__ uint32_t column(const Cursor & c, int col) const {
        const int job = job0 + c.job;
        return inbox.slot(round, r.unit(c.group, (job >> 1) - c.group * a.blocks_ff, a.blocks_ff) - unit0 + col, job & 1, sub);
    }
};

// Writes one token's hidden value of column block * 32 + lane (and, behind the last block, zeros up to a whole step).
__device__ __forceinline__ void put_hidden(const MoeArgs & a, const Route & r, int u, int col, int block, float v) {
    const int lane = threadIdx.x & 31;
    const int set = col / kSet, place = col - set * kSet, nt = min(kSet, r.count(u) - set * kSet);
    uint8_t * at = a.hidden + ((size_t)(r.before(u) + set * kSet) * a.steps_ff + (size_t)(block >> 2) * nt) * kHiddenBytes;
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu);
    const int shift = shift_for(top);
    const int last = block == a.blocks_ff - 1 ? 3 : block & 3;
    for (int group = block & 3; group <= last; ++group) {
        if (group != (block & 3)) v = 0.f;
        const float s = v * power(shift);
        const __half hi = __float2half_rn(s), lo = __float2half_rn(s - __half2float(hi));
        __half * x = reinterpret_cast<__half *>(at + (group * 2 * nt + place) * 64) + lane;
        x[0] = hi;
        x[nt * 32] = lo;
        float sum = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0)
            *reinterpret_cast<float2 *>(at + step_x_bytes(2, nt) + (group * nt + place) * 8) =
                make_float2(power(weight_shift(a.down_mx) - shift), sum * kStart);
    }
}

template <bool MX, int PARTS, int NT>
__global__ void __launch_bounds__(warps_for(NT) * 32, NT > 4 ? 1 : 2) w4_moe_gate_up_kernel(MoeArgs a) {
    constexpr int kWarps = warps_for(NT);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Scratch<kWarps> sc;
    __shared__ Picks picks;
    __shared__ __align__(16) uint8_t route_copy[kRouteBytes];
    __shared__ int range[2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), C = (int)cluster_size(), log_c = __ffs(C) - 1;
    const int cluster = blockIdx.x >> log_c;
    cluster_arrive();
    const int s0 = part_begin2(a.steps_d, rank, log_c), n_steps = part_begin2(a.steps_d, rank + 1, log_c) - s0;
    const Staged x{smem, reinterpret_cast<float *>(smem + a.x_bytes)};
    float * mine = reinterpret_cast<float *>(smem + a.x_bytes + a.c_bytes);         // this CTA's part of the logits
    float * logits = mine + a.logit_bytes / 4;
    uint8_t * const rings = smem + a.x_bytes + a.c_bytes + 2 * a.logit_bytes;
    if (threadIdx.x == 0) sc.zero = 0;
    if (threadIdx.x < kW4MaxExperts) picks.mask[threadIdx.x] = 0;

    pdl_trigger();
    pdl_wait();
    const int k0 = s0 * 128, k1 = min(a.d, (s0 + n_steps) * 128);
    // the rings and the first inbox are idle until the experts are known
    const int idle = ring_bytes(MX, NT, kMoeStages) + a.inbox;
    fetch_router(a, k0, min(k1 - k0, router_columns(a.E, idle)), rings);
    copies_commit();
    stage_tokens<MX, PARTS>(a.x, a.T, NT, k0, n_steps, a.d, a.norm, NormRoom{0, 0, 0}, x, sc, rank, C);
    __syncthreads();
    partial_logits<MX, PARTS, NT, kWarps>(a, k0, k1, x, rings, idle, mine);
    // Out of the activations' scale (a token's factor without the weights' constant) and to every CTA of the cluster: into its second
    // inbox, which nobody else writes before the cluster has met after the first round, where that has room.
    __syncthreads();
    const int n_logits = a.T * a.E;
    const uint32_t mail = smem_address(rings) + ring_bytes(MX, NT, kMoeStages) + a.inbox;
    const bool posted = C * n_logits * 4 <= a.inbox;
    for (int i = threadIdx.x; i < n_logits; i += kWarps * 32) {
        const float v = mine[i] * (sc.factor[i / a.E] * power(-weight_shift(MX)));
        if (posted) {
            for (int c = 0; c < C; ++c) remote_store(remote_address(mail + (rank * n_logits + i) * 4, c), v);
        } else {
            mine[i] = v;
        }
    }
    cluster_sync();
    for (int i = threadIdx.x; i < n_logits; i += kWarps * 32) {
        float v = 0.f;
        for (int c = 0; c < C; ++c) v += posted ? shared_f1(mail + (c * n_logits + i) * 4) : remote_load(remote_address(smem_address(mine + i), c));
        logits[i] = a.norm ? v * rms_factor(sc, i / a.E, C, a.d, a.eps) : v;
    }
    __syncthreads();
    for (int t = warp; t < a.T; t += kWarps) {
        auto logit = [&](int e) { return logits[t * a.E + e]; };
        int expert;
        float weight;
        if (a.E <= 32) pick_experts<1>(logit, a.E, a.k, a.normalise, expert, weight);
        else if (a.E <= 128) pick_experts<4>(logit, a.E, a.k, a.normalise, expert, weight);
        else pick_experts<kW4MaxExperts / 32>(logit, a.E, a.k, a.normalise, expert, weight);
        if (lane < a.k) {
            const int i = t * a.k + lane;
            picks.expert[i] = (uint32_t)expert;
            picks.weight[i] = weight;
            if (blockIdx.x == 0 && a.ids) a.ids[i] = expert;
            if (blockIdx.x == 0 && a.weights) a.weights[i] = weight;
        }
    }
    if (threadIdx.x < 2) range[threadIdx.x] = 0;
    __syncthreads();
    write_route(a, picks, route_copy);
    __syncthreads();
    const Route route{route_copy, a.at};
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < a.at.bytes / 16; i += kWarps * 32) reinterpret_cast<uint4 *>(a.route)[i] = reinterpret_cast<const uint4 *>(route_copy)[i];
    }
    // The cluster's blocks: those whose cost begins in its share of the whole cost.
    if (threadIdx.x < 2) range[threadIdx.x] = 0;
    __syncthreads();
    {
        const int u = threadIdx.x, n = route.experts();
        if (u < n) {
            const int64_t all = route.cost(n);
            const int from = route.cost(u), to = route.cost(u + 1), each = (to - from) / a.blocks_ff;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int point = (int)(all * (cluster + i) / a.clusters);
                if (from < point && point <= to) range[i] = u * a.blocks_ff + (point - from + each - 1) / each;
            }
        }
    }
    __syncthreads();
    const int b_begin = range[0], blocks = range[1] - b_begin;
    // parts of the columns: no more than the inbox has room for with every token at one expert
    const int ks = split_columns(blocks * 2, a.steps_d >> log_c, kWarps, (int)(a.inbox / inbox_bytes(a.T, C, 1, 2))), log_ks = __ffs(ks) - 1;
    const int room = (a.inbox >> (log_c + log_ks + 8)) << log_c;        // units of a round
    const int sub = warp & (ks - 1), step = part_begin2(n_steps, sub, log_ks), len = part_begin2(n_steps, sub + 1, log_ks) - step;
    const Staged x_warp{x.x + step * step_x_bytes(PARTS, NT), x.c + step * step_c_bytes(MX, NT) / 4};
    const Inbox inbox{smem_address(rings + ring_bytes(MX, NT, kMoeStages)), a.inbox, rank, log_c, ks, 2};
    GateUpSource<MX, PARTS, NT> src{a, route, x_warp, inbox, 2 * b_begin, 2 * blocks, warp >> log_ks, kWarps >> log_ks, sub, s0 + step, len, 0, 0};
    Stream<MX, kMoeStages, GateUpSource<MX, PARTS, NT>> stream(src, rings);
    stream.prefetch();
    int u = b_begin / a.blocks_ff, block = b_begin - u * a.blocks_ff;       // where the round begins
    for (int b0 = 0; b0 < blocks; ++src.round) {
        // as many blocks as the inbox has room for
        const int u0 = u, block0 = block;
        int now = 0, units = 0;
        while (b0 + now < blocks) {
            const int n = route.count(u), more = min(min(a.blocks_ff - block, blocks - b0 - now), (room - units) / n);
            now += more;
            units += more * n;
            block += more;
            if (block < a.blocks_ff) break;
            ++u;
            block = 0;
        }
        src.unit0 = route.unit(u0, block0, a.blocks_ff);
        stream.template work<PARTS, NT, (NT > 1)>(sc, 2 * (b0 + now));
        cluster_sync();
        int v_u = u0;
        for (int i = warp; i * C + rank < units; i += kWarps) {
            const int unit = src.unit0 + i * C + rank;
            while (v_u + 1 < route.experts() && unit >= route.unit(v_u + 1, 0, a.blocks_ff)) ++v_u;
            const int n = route.count(v_u), at = unit - route.unit(v_u, 0, a.blocks_ff), b = at / n, col = at - b * n, pair = route.before(v_u) + col;
            const float rstd = a.norm ? rms_factor(sc, *route.tokens(pair), C, a.d, a.eps) : 1.f;
            const float v = inbox.sum(src.round, i, 0) * rstd, up = inbox.sum(src.round, i, 1) * rstd;
            put_hidden(a, route, v_u, col, b, route.weight(pair) * (v / (1.f + expf(-v)) * up));
        }
        b0 += now;
    }
    if (blocks == 0) cluster_sync();        // nobody leaves while its logits are read
}

// The second kernel's stream: as Stream, but a unit comes with the hidden columns it multiplies. Weights run two units ahead, hidden
// columns one.
template <bool MX, int MOST> struct DownStream {
    static constexpr int kWarps = MOST > 1 ? 16 : 8, kStages = 3;
    static constexpr uint32_t kUnit = w4_unit_bytes(MX), kHidden = MOST * kHiddenBytes;
    static constexpr int kRingBytes = kWarps * (kStages * (int)kUnit + 2 * (int)kHidden);
    const MoeArgs & a;
    const Route & r;
    const int lane;
    const uint32_t weights;             // the warp's rings
    uint8_t * const hidden;
    // this warp: steps [from, to) of the sets' concatenated columns, of jobs first, first + stride, ...
    const int from, to, job0, jobs, stride;
    struct Place {
        const uint8_t * p;
        int set, left, job, at;         // at: step of the concatenated columns
        bool live;
    } w, h, c;
    uint32_t fill, h_fill, at, h_at;

    __device__ __forceinline__ DownStream(const MoeArgs & args, const Route & route, uint8_t * rings, int f, int t, int j0, int j, int first, int step)
        : a(args), r(route), lane(threadIdx.x & 31), weights(smem_address(rings) + (threadIdx.x >> 5) * (kStages * kUnit)),
          hidden(rings + kWarps * kStages * kUnit + (threadIdx.x >> 5) * (2 * kHidden)), from(f), to(t), job0(j0), jobs(j), stride(step),
          fill(0), h_fill(0), at(0), h_at(0) {
        w.live = from < to && first < jobs;
        w.job = first;
        w.at = from;
        w.set = from / a.steps_ff;
        h = w;
        c = w;
        if (w.live) {
            point_weights();
            point_hidden();
            c.left = left(c);
        }
    }
    __device__ __forceinline__ int left(const Place & p) const { return min(to, (p.set + 1) * a.steps_ff) - p.at; }
    __device__ __forceinline__ void point_weights() {
        w.p = a.down + r.set_expert(w.set) * a.down_expert + ((size_t)(job0 + w.job) * a.steps_ff + (w.at - w.set * a.steps_ff)) * kUnit + lane * 16;
        w.left = left(w);
    }
    __device__ __forceinline__ void point_hidden() {
        h.p = a.hidden + ((size_t)r.set_first(h.set) * a.steps_ff + (size_t)(h.at - h.set * a.steps_ff) * r.set_count(h.set)) * kHiddenBytes + lane * 16;
        h.left = left(h);
    }
    // To the next run: the next set of the job, or the next job from the beginning.
    __device__ __forceinline__ void next(Place & p) const {
        ++p.set;
        p.at = p.set * a.steps_ff;
        if (p.at >= to) {
            p.job += stride;
            p.at = from;
            p.set = from / a.steps_ff;
            p.live = p.job < jobs;
        }
    }
    __device__ __forceinline__ void fetch_weights() {
        if (w.live) {
            const uint32_t dst = weights + fill + lane * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i) copy16(dst + i * 512, w.p + i * 512);
            if (lane < (MX ? 8 : 16)) copy16(dst + 2048, w.p + 2048);
            w.p += kUnit;
            if (--w.left == 0) {
                next(w);
                if (w.live) point_weights();
            }
        }
        fill = fill == (kStages - 1) * kUnit ? 0 : fill + kUnit;
        copies_commit();
    }
    __device__ __forceinline__ void fetch_hidden() {
        if (h.live) {
            const uint32_t dst = smem_address(hidden) + h_fill + lane * 16;
            const int chunks = r.set_count(h.set) * (kHiddenBytes / 16);
#pragma unroll
            for (int i = 0; i < (MOST * (kHiddenBytes / 16) + 31) / 32; ++i) if (lane + 32 * i < chunks) copy16(dst + i * 512, h.p + i * 512);
            h.p += chunks * 16;
            if (--h.left == 0) {
                next(h);
                if (h.live) point_hidden();
            }
        }
        h_fill ^= kHidden;              // one stage or the other
        copies_commit();
    }
    __device__ __forceinline__ void prefetch() {
        fetch_weights();
        fetch_hidden();
        fetch_weights();
    }
    template <int NT, class Column> __device__ __forceinline__ void work_run(Column column) {
        float acc[2][2][4] = {};
        Lane l;
        const Group g{{hidden, nullptr}, nullptr, NT};
        begin_group<MX, 2, PACK, NT, false, true>(g, lane, 0, l);
        const uint32_t at0 = weights + lane * 16, scale_at = weights + 2048 + (lane >> 2) * (MX ? 8 : 16);
        for (int n = c.left; n > 0; --n) {
            copies_wait<1>();           // this unit's weights and hidden columns have landed, the next unit's weights may be on their way
            __syncwarp();
            fetch_hidden();
            fetch_weights();
            do_step<MX, 2, PACK, NT, true>(at0 + at, scale_at + at, h_at, h_at, l, lane, acc);
            at = at == (kStages - 1) * kUnit ? 0 : at + kUnit;
            h_at ^= kHidden;
        }
        float * to = nullptr;
        end_run<PACK, NT, true>(NT, lane, l, acc, [&](int col) { to = column(col) + (lane >> 2); }, [&](int row, float v) { to[row] += v; });
    }
    // slot(job, token): where 32 rows' sums are added up
    template <class Slot> __device__ __forceinline__ void work(Slot slot) {
        while (c.live) {
            const int n = r.set_count(c.set);
            auto column = [&](int col) { return slot(c.job, *r.tokens(r.set_first(c.set) + col)); };
            if (n == 1) work_run<1>(column);
            if constexpr (MOST > 1) if (n == 2) work_run<2>(column);
            if constexpr (MOST > 2) if (n == 3) work_run<3>(column);
            next(c);
            if (c.live) c.left = left(c);
        }
    }
};

template <bool MX, int MOST>
__global__ void __launch_bounds__(DownStream<MX, MOST>::kWarps * 32, MOST > 1 ? 1 : 3) w4_moe_down_kernel(MoeArgs a) {
    constexpr int kWarps = DownStream<MX, MOST>::kWarps;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(16) uint8_t route_copy[kRouteBytes];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), C = (int)cluster_size(), log_c = __ffs(C) - 1;
    const int cluster = blockIdx.x >> log_c;
    cluster_arrive();
    float * partial = reinterpret_cast<float *>(smem + DownStream<MX, MOST>::kRingBytes);
    const Inbox inbox{smem_address(partial) + a.partial, a.inbox, rank, log_c, 1, 1};
    const int j_begin = part_begin(a.blocks_d, cluster, a.clusters), j_end = part_begin(a.blocks_d, cluster + 1, a.clusters);
    pdl_trigger();
    pdl_wait();
    const Route route{route_copy, a.at};
    copy_route(a.route, route_copy, a.at.token, a.at.bytes);
    cluster_wait();
    __syncthreads();
    const int total = route.sets() * a.steps_ff;    // the sets' columns, one behind the other
    const int begin = part_begin2(total, rank, log_c), n = part_begin2(total, rank + 1, log_c) - begin;
    const int ks = a.ks, first = warp / ks, sub = warp - first * ks, stride = kWarps / ks;
    int round = 0;
    for (int j0 = j_begin; j0 < j_end; j0 += a.per_round, ++round) {
        const int jobs = min(a.per_round, j_end - j0);
        DownStream<MX, MOST> stream(a, route, smem, begin + part_begin(n, sub, ks), begin + part_begin(n, sub + 1, ks), j0,
                                    first < stride ? jobs : 0, first, stride);
        stream.prefetch();
        for (int i = threadIdx.x; i < jobs * ks * a.T * kSlotCol; i += kWarps * 32) partial[i] = 0.f;
        __syncthreads();
        stream.work([&](int job, int token) { return partial + ((job * ks + sub) * a.T + token) * kSlotCol; });
        __syncthreads();
        for (int unit = warp; unit < jobs * a.T; unit += kWarps) {
            const int job = unit / a.T, t = unit - job * a.T;
            float v = 0.f;
            for (int i = 0; i < ks; ++i) v += partial[((job * ks + i) * a.T + t) * kSlotCol + lane];
            remote_store(inbox.slot(round, unit, 0, 0) + lane * 4, v);
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
// Word j (0..3) of lane (g, t) and half w (0, 1) of a unit's row tile holds row g + 8 (j & 1), columns 8 t + 4 s + 2 (j >> 1) + e of
// group 2 w + h, for the products s = 0, 1, groups h = 0, 1 and e = 0, 1. Q4_0: the nibble at bit 6 + 16 e + 4 (2 h + s), modulo 32. MXFP4: the
// nibble at bit 8 (2 h + s) + 4 e, a pair for the conversion to every byte.
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
    for (uint32_t i = threadIdx.x; i < 512; i += blockDim.x) {
        const uint32_t w = i >> 8, tile = (i >> 7) & 1, lane = (i & 127) >> 2, j = i & 3;
        const uint32_t g = lane >> 2, t = lane & 3;
        const uint32_t row = row_block * 32 + tile * 16 + g + 8 * (j & 1);
        uint32_t word = 0;
        for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t block = step * 4 + w * 2 + h;
            if (row >= n_out || block >= blocks) continue;
            const uint8_t * q = rows + ((expert * n_out + row) * blocks + block) * kBlock + (MX ? 1 : 2);
            for (uint32_t s = 0; s < 2; ++s)
                for (uint32_t e = 0; e < 2; ++e) {
                    const uint32_t k = 8 * t + 4 * s + 2 * (j >> 1) + e;
                    const uint32_t n = (q[k & 15] >> (k >= 16 ? 4 : 0)) & 15u;
                    word |= MX ? n << (8 * (2 * h + s) + 4 * e) : __funnelshift_l(n << (6 + 16 * e), n << (6 + 16 * e), 4 * (2 * h + s));
                }
        }
        *reinterpret_cast<uint32_t *>(dst + i * 4) = word;
    }
    if (threadIdx.x < 128) {
        // scales of the four groups of row g, then of row g + 8, for g = 0..7, of each tile
        const uint32_t tile = threadIdx.x >> 6, g = (threadIdx.x & 63) >> 3, upper = (threadIdx.x >> 2) & 1, group = threadIdx.x & 3;
        const uint32_t row = row_block * 32 + tile * 16 + g + 8 * upper, block = step * 4 + group;
        const bool live = row < n_out && block < blocks;
        const uint8_t * b = rows + ((expert * n_out + row) * blocks + block) * kBlock;
        if (MX) {
            // kept as s + 8, so that the smallest scale 2^-127 is a normal f32 as well; 2^-8 is part of the rows' final factor
            const int s = live ? b[0] : 0;
            const uint32_t warp_max = __reduce_max_sync(0xffffffffu, (uint32_t)s);
            if ((threadIdx.x & 31) == 0) atomicMax(max_scale, (int)warp_max);
            dst[2048 + tile * 64 + g * 8 + upper * 4 + group] = live ? (uint8_t)min(s + 8, 255) : 0;
        } else {
            reinterpret_cast<uint16_t *>(dst + 2048 + tile * 128)[g * 8 + upper * 4 + group] = live ? (uint16_t)(b[0] | b[1] << 8) : 0;
        }
    }
}

// ---- launch plans

int device_sms() {
    static std::atomic<int> sms[64] = {};
    int device = 0;
    cudaGetDevice(&device);
    int n = sms[device & 63].load();
    if (!n) {
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
        sms[device & 63].store(n);
    }
    return n;
}

constexpr int kMaxSmem = 200 * 1024;            // dynamic shared memory of a CTA
constexpr int kSmShare = 226 * 1024;            // what the CTAs of an SM have together

int log2_of(int C) { return C == 1 ? 0 : C == 2 ? 1 : C == 4 ? 2 : 3; }
int up_to(int x, int unit) { return (x + unit - 1) / unit * unit; }

template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), int grid, int threads, int cluster, size_t smem, cudaStream_t stream, Args &&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
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

// Devices on which a kernel has been given its shared memory. Set behind the call that does it: of threads that come at once, each does.
struct Prepared {
    std::atomic<uint64_t> done[4] = {};
};
template <typename... KArgs> cudaError_t allow_smem(Prepared & prepared, void (*kernel)(KArgs...)) {
    int device = 0;
    cudaGetDevice(&device);
    std::atomic<uint64_t> & done = prepared.done[(device >> 6) & 3];
    const uint64_t bit = 1ull << (device & 63);
    if (done.load() & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
    if (e == cudaSuccess) done.fetch_or(bit);
    return e;
}

template <bool MX, int PARTS, bool GLU, int NT> cudaError_t launch_product(const ProductArgs & a, int clusters, int C, size_t smem, cudaStream_t stream) {
    static Prepared once;
    const cudaError_t e = allow_smem(once, w4_product_kernel<MX, PARTS, GLU, NT>);
    return e != cudaSuccess ? e : launch_cluster(w4_product_kernel<MX, PARTS, GLU, NT>, clusters * C, warps_for(NT) * 32, C, smem, stream, a);
}

// Room the kernels that take whole calls of n tokens stage them with: those sizes they are built for. (14336 x 4096 gated pair, one token: 18.7 us, 21.3 us with
// room for four; six tokens: 24.8 us, 30.4 us with room for sixteen. Expert layer of 32 x 2880 x 2880: 30.1 and 32.2 us, 67.5 and 69.9 us.)
int product_room(int n) { return n == 1 ? 1 : n <= 4 ? 4 : n <= 8 ? 8 : 16; }

// Calls f with the room as a constant.
template <class F> cudaError_t with_room(int nt, F f) {
    if (nt == 1) return f(std::integral_constant<int, 1>{});
    if (nt == 4) return f(std::integral_constant<int, 4>{});
    if (nt == 8) return f(std::integral_constant<int, 8>{});
    return f(std::integral_constant<int, 16>{});
}

template <bool MX, bool GLU> cudaError_t launch_product_of(const ProductArgs & a, int parts, int clusters, int C, size_t smem, cudaStream_t stream) {
    const int nt = product_room(a.T);
    if (parts == 2) return with_room(nt, [&](auto n) { return launch_product<MX, 2, GLU, decltype(n)::value>(a, clusters, C, smem, stream); });
    return with_room(nt, [&](auto n) { return launch_product<MX, 1, GLU, decltype(n)::value>(a, clusters, C, smem, stream); });
}

template <bool MX, int PARTS, int NT> cudaError_t launch_gate_up(const MoeArgs & a, int C, size_t smem, cudaStream_t stream) {
    static Prepared once;
    const cudaError_t e = allow_smem(once, w4_moe_gate_up_kernel<MX, PARTS, NT>);
    return e != cudaSuccess ? e : launch_cluster(w4_moe_gate_up_kernel<MX, PARTS, NT>, a.clusters * C, warps_for(NT) * 32, C, smem, stream, a);
}

template <bool MX> cudaError_t launch_gate_up_of(const MoeArgs & a, int parts, int C, size_t smem, cudaStream_t stream) {
    const int nt = product_room(a.T);
    if (parts == 2) return with_room(nt, [&](auto n) { return launch_gate_up<MX, 2, decltype(n)::value>(a, C, smem, stream); });
    return with_room(nt, [&](auto n) { return launch_gate_up<MX, 1, decltype(n)::value>(a, C, smem, stream); });
}

template <bool MX, int MOST> cudaError_t launch_down(const MoeArgs & a, int C, size_t smem, cudaStream_t stream) {
    static Prepared once;
    const cudaError_t e = allow_smem(once, w4_moe_down_kernel<MX, MOST>);
    return e != cudaSuccess ? e : launch_cluster(w4_moe_down_kernel<MX, MOST>, a.clusters * C, DownStream<MX, MOST>::kWarps * 32, C, smem, stream, a);
}

const void * row_at(const void * p, uint32_t type, int64_t ld, int64_t row) {
    return p ? static_cast<const uint8_t *>(p) + row * ld * (type == GGML_F32 ? 4 : 2) : nullptr;
}

Act make_act(const void * p, int64_t ld, uint32_t type) {
    const size_t es = type == GGML_F32 ? 4 : 2;
    return {p, ld, type, (uintptr_t)p % 16 == 0 && ld * (int64_t)es % 16 == 0};
}

// Clusters of 2^log_c CTAs that are on the GPU together, with `resident` CTAs on an SM: a cluster lies within one of the GPU's processing
// clusters, whose SM counts are no multiples of it. Asked once per device and kind.
int resident_clusters(int log_c, int resident, int threads) {
    struct Table { std::atomic<int> n[4][4]; };
    static Table tables[64];
    int device = 0;
    cudaGetDevice(&device);
    std::atomic<int> & known = tables[device & 63].n[log_c][threads > 256 ? 3 : resident - 1];
    int n = known.load();
    if (n) return n;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << log_c;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(1u << log_c);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = std::min(kMaxSmem, kSmShare / resident - 4096);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto ask = [&](auto kernel) {
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
        return cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
    };
    const cudaError_t e = threads > 256 ? ask(w4_product_kernel<false, 2, false, 16>) : ask(w4_product_kernel<false, 2, false, 1>);
    if (e != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = std::max(1, resident * device_sms() >> log_c);
    }
    known.store(n);
    return n;
}

// How a product is cut: CTAs of a cluster, clusters, and CTAs on an SM.
struct Cut {
    int C = 0, clusters = 0, resident = 0;
    double cost = 0;
};

// Chooses the cluster size for `blocks` row blocks of `per` matrices and `steps` column steps whose activations take `each` bytes of
// shared memory a step. The estimate is in clocks: the weight stream at the SM's share of the memory bandwidth, but no faster
// than the busiest SM's warps get through it or than its copies in flight allow; the conversion of the CTA's share of the activations; the sums it
// receives; and a barrier for every round its inbox allows. 23.5 bytes a clock and SM and 13 MB in flight are 6.6 TB/s for two microseconds; the clocks of a unit, a
// conversion, a sum and a barrier are fitted to measured times, not derived. `fixed` is other dynamic shared memory, `statics` the kernel's static one.
Cut choose_cut(int blocks, int per, int steps, int n, int each, bool mx, int stages, int most_resident, int least_c, int most_c, int fixed, int statics, int sms) {
    Cut best;
    const int warps = warps_for(n), ring = ring_bytes(mx, n, stages), unit = (int)w4_unit_bytes(mx);
    for (int C = least_c; C <= most_c && C <= steps; C *= 2) {
        const int s = (steps + C - 1) / C;
        const int64_t smem = (int64_t)s * each + ring + fixed + statics + 2 * inbox_bytes(n, C, 1, per) + 4096;
        if (smem - statics - 4096 + 256 > kMaxSmem || smem > kSmShare) continue;    // the parts are rounded up
        Cut c;
        c.C = C;
        c.resident = (int)std::min<int64_t>(most_resident, kSmShare / smem);
        // as few clusters as keep their size: the places they leave free are where the next kernel of the stream begins
        const int most = resident_clusters(log2_of(C), c.resident, warps * 32), blocks_each = (blocks + most - 1) / most;
        c.clusters = (blocks + blocks_each - 1) / blocks_each;
        const int busy = (c.clusters * C + sms - 1) / sms;
        const int ks = split_columns(blocks_each * per, steps / C, warps, warps);
        const int runs = (blocks_each * per * ks + warps - 1) / warps;           // of the busiest warp
        const double unit_clocks = n > 8 ? 150 : n > 4 ? 120 : 80;
        const double in_flight = (double)c.clusters * C * warps * (stages - 1) * unit;
        const double stream = std::max({(double)blocks * per * steps * unit / (23.5 * sms) * std::max(1.0, 13e6 / in_flight),     // two microseconds of latency under load
                                        (double)busy * runs * warps * ((s + ks - 1) / ks + (n > 8 ? 0.6 : 0.3)) * unit_clocks});
        const double convert = busy * s * n * 128 * 0.1 + 800, sums = busy * (double)blocks_each * per * n * (6 + 2 * C * ks);
        const int64_t room = std::min(kSmShare / c.resident - statics - 4096, kMaxSmem) - fixed - ring - (int64_t)s * each;
        const double rounds = std::ceil((double)inbox_bytes((int64_t)blocks_each * n, C, ks, per) / std::max<int64_t>(room, 1024));
        c.cost = stream + convert + sums / 4 + (rounds > 1 ? 2 * rounds : 1) * 1500;
        if (!best.C || c.cost < best.cost) best = c;
    }
    return best;
}

// choose_cut for a product of n tokens (in passes of fewer, where rows are too long for them): remembered by the sizes it depends on.
Cut product_cut(int blocks, int per, int steps, bool mx, int parts, int & n) {
    struct Known {
        int key[7] = {};
        int n = 0;
        Cut cut;
    };
    thread_local Known known[16];
    int device = 0;
    cudaGetDevice(&device);
    const int key[7] = {blocks, per, steps, mx, parts, n, device + 1};
    Known & k = known[((unsigned)blocks * 31 + (unsigned)steps * 7 + (unsigned)n * 3 + (unsigned)per) % 16];
    if (!std::equal(key, key + 7, k.key)) {
        for (k.n = n;; k.n = (k.n + 1) / 2) {
            const int room = product_room(k.n);
            k.cut = choose_cut(blocks, per, steps, k.n, step_bytes(mx, parts, room), mx, stages_for(k.n, parts), resident_for(room), 1, kMaxCluster, 0, 0, device_sms());
            if (k.cut.C || k.n == 1) break;
        }
        std::copy(key, key + 7, k.key);
    }
    n = k.n;
    return k.cut;
}

} // namespace

size_t w4_bytes(uint32_t type, uint32_t n_out, uint32_t n_in, uint32_t n_expert) {
    return (size_t)n_expert * ((n_out + 31) / 32) * ((n_in + 127) / 128) * w4_unit_bytes(type == GGML_MXFP4);
}

W4View w4_view(const uint8_t * units, uint32_t type, uint32_t n_out, uint32_t n_in, uint32_t n_expert) {
    W4View v;
    v.units = units;
    v.type = type;
    v.n_out = n_out;
    v.n_in = n_in;
    v.n_expert = n_expert;
    v.blocks = (n_out + 31) / 32;
    v.steps = (n_in + 127) / 128;
    v.expert_bytes = (size_t)v.blocks * v.steps * w4_unit_bytes(type == GGML_MXFP4);
    return v;
}

cudaError_t launch_w4_retile(const uint8_t * rows, uint32_t type, uint32_t n_out, uint32_t n_in, uint32_t n_expert, uint8_t * units, int * max_scale,
                             cudaStream_t stream) {
    const W4View v = w4_view(units, type, n_out, n_in, n_expert);
    const size_t n = (size_t)n_expert * v.blocks * v.steps;
    if (type == GGML_MXFP4) w4_retile_kernel<true><<<(unsigned)n, 256, 0, stream>>>(rows, n_out, n_in, v.blocks, v.steps, units, max_scale);
    else w4_retile_kernel<false><<<(unsigned)n, 256, 0, stream>>>(rows, n_out, n_in, v.blocks, v.steps, units, max_scale);
    return cudaGetLastError();
}

cudaError_t launch_w4_product(const W4Product & p, cudaStream_t stream) {
    const bool mx = p.w.type == GGML_MXFP4, glu = p.up != nullptr;
    const int parts = p.x_type == GGML_F32 || p.norm ? 2 : 1;
    const int blocks = (int)p.w.blocks, per = glu ? 2 : 1, steps = (int)p.w.steps;
    for (int t0 = 0, n = 0; t0 < p.n_tokens; t0 += n) {
        n = std::min(kW4PassTokens, p.n_tokens - t0);
        const Cut cut = product_cut(blocks, per, steps, mx, parts, n);
        if (!cut.C) return cudaErrorInvalidValue;       // rows this long are refused when the handle is made
        const int C = cut.C, nt = product_room(n), warps = warps_for(n), s = (steps + C - 1) / C;
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
        a.x_bytes = up_to(s * step_x_bytes(parts, nt), 128);
        a.c_bytes = up_to(s * step_c_bytes(mx, nt), 128);
        // two inboxes in what is left of the CTA's share of the shared memory; one, if everything fits into it
        const int fixed = a.x_bytes + a.c_bytes + ring_bytes(mx, nt, stages_for(nt, parts));
        const int blocks_each = a.each + (a.more > 0);
        const int64_t room = std::min(kSmShare / cut.resident - 4096, kMaxSmem) - fixed;
        a.ks = split_columns(blocks_each * per, steps / C, warps, (int)std::max<int64_t>(1, room / 2 / inbox_bytes(n, C, 1, per)));
        const int64_t whole = inbox_bytes((int64_t)blocks_each * n, C, a.ks, per);
        a.inbox = (int)(whole <= room ? whole : std::max<int64_t>(room / 2 / 128 * 128, inbox_bytes(n, C, a.ks, per)));
        a.per_round = whole <= room ? blocks_each : blocks_per_round(a.inbox, n, C, a.ks, per, warps);
        size_t smem = (size_t)fixed + (whole <= room ? 1 : 2) * (size_t)a.inbox;
        // no more CTAs on an SM than an even spread needs: clusters are packed densely otherwise, and leave SMs idle
        const int spread = (cut.clusters * C + device_sms() - 1) / device_sms();
        if (spread < cut.resident) smem = std::max(smem, (size_t)(kSmShare / (spread + 1)));
        cudaError_t e;
        if (mx) e = glu ? launch_product_of<true, true>(a, parts, cut.clusters, C, smem, stream) : launch_product_of<true, false>(a, parts, cut.clusters, C, smem, stream);
        else e = glu ? launch_product_of<false, true>(a, parts, cut.clusters, C, smem, stream) : launch_product_of<false, false>(a, parts, cut.clusters, C, smem, stream);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// Workspace in front of the hidden columns.
static size_t route_room(size_t pairs) { return (route_at((int)std::min<size_t>(pairs, kW4MaxExperts), (int)pairs).bytes + 255) / 256 * 256; }

size_t w4_moe_workspace_bytes(uint32_t ff, uint32_t n_tokens, uint32_t n_used) {
    const size_t pairs = (size_t)std::min<uint32_t>(n_tokens, kW4PassTokens) * n_used;
    return route_room(pairs) + pairs * ((ff + 127) / 128) * kHiddenBytes;
}

namespace {

constexpr int kMoeStatic = 15 * 1024;       // static shared memory of the first kernel, rounded up: picks, route and what stage_tokens needs

// How the two kernels of a pass over n tokens are cut.
struct MoePlan {
    int n = 0;
    Cut cut;
    int C = 0, clusters = 0, ks = 0, per_round = 0, inbox = 0, partial = 0;
    size_t smem = 0;
};

MoePlan make_moe_plan(int E, int used, int blocks_ff, int steps_d, int blocks_d, int steps_ff, bool mx, bool mx_down, int parts, int n) {
    MoePlan m;
    // First kernel: n tokens that choose independently choose about `reach` experts. It runs in clusters of four (one token, 32 experts of
    // 2880 x 2880: 31 us the layer, 38 us with eight; 64 experts of 1024 x 2048, six tokens: 50 us, 55 us with two), of more where rows are so long
    // that four cannot hold them.
    for (;; n = (n + 1) / 2) {
        const int reach = std::max(1, (int)std::ceil(E * (1.0 - std::pow(1.0 - (double)used / E, n)))), room = product_room(n);
        const int least_c = steps_d < 2 ? 1 : steps_d < 4 ? 2 : 4;
        for (int C = least_c; !m.cut.C && C <= kMaxCluster; C *= 2)
            m.cut = choose_cut(reach * blocks_ff, 2, steps_d, n, step_bytes(mx, parts, room), mx, kMoeStages, room > 4 ? 1 : 2, C, C, 2 * up_to(n * E * 4, 128), kMoeStatic, device_sms());
        if (m.cut.C || n == 1) break;
    }
    m.n = n;
    if (!m.cut.C) return m;
    // Second kernel, in clusters of four: eight would leave a warp two units of a run at one token. One token: three CTAs of eight warps on an SM;
    // several: one of sixteen, whose partial sums share the room better (sixteen tokens, 32 experts of 2880 x 2880: 11 us of 135 less).
    m.C = 4;
    while (m.C > steps_ff * used) m.C /= 2;
    const int resident = n > 1 ? 1 : 3, warps = n > 1 ? 16 : 8;
    const int most = resident_clusters(log2_of(m.C), resident, warps * 32), per = (blocks_d + most - 1) / most;
    m.clusters = (blocks_d + per - 1) / per;
    const int slot = n * kSlotCol * 4;
    const int rings = mx_down ? (n > 1 ? DownStream<true, kSet>::kRingBytes : DownStream<true, 1>::kRingBytes)
                              : (n > 1 ? DownStream<false, kSet>::kRingBytes : DownStream<false, 1>::kRingBytes);
    // A slot for every (block, part of the columns) of a round, and an inbox for its blocks, two where there are several rounds. A
    // round's end costs about as much as five steps.
    const int left = std::min(kSmShare / resident - 8 * 1024, kMaxSmem) - rings, steps = std::max(1, n * used * steps_ff / m.C);
    int64_t least = INT64_MAX;
    for (int rounds = 1, found = 0; found < 4 && rounds <= per; ++rounds) {
        const int blocks = (per + rounds - 1) / rounds, many = rounds > 1 ? 2 : 1;
        const int64_t inbox = inbox_bytes((int64_t)blocks * n, m.C, 1, 1), fit = (left - many * inbox) / ((int64_t)blocks * slot);
        if (fit < 1) continue;
        int cost;
        const int ks = divide_columns(blocks, steps, warps, (int)std::min<int64_t>(fit, warps), cost);
        ++found;
        if ((int64_t)rounds * (cost + 10) < least) {
            least = (int64_t)rounds * (cost + 10);
            m.per_round = blocks;
            m.ks = ks;
            m.inbox = (int)inbox;
            m.partial = blocks * ks * slot;
            m.smem = (size_t)rings + m.partial + many * (size_t)inbox;
        }
    }
    if (!m.smem) m.cut.C = 0;
    return m;
}

// The same, remembered by the sizes it depends on.
MoePlan moe_plan(const W4Moe & p, bool mx, bool mx_down, int parts, int n) {
    struct Known {
        int key[11] = {};
        MoePlan plan;
    };
    thread_local Known known[16];
    int device = 0;
    cudaGetDevice(&device);
    const int key[11] = {(int)p.gate.n_expert, p.n_used, (int)p.gate.blocks, (int)p.gate.steps, (int)p.down.blocks, (int)p.down.steps, mx, mx_down, parts, n, device + 1};
    Known & k = known[((unsigned)key[0] + (unsigned)key[2] * 31 + (unsigned)key[3] * 7 + (unsigned)n * 3) % 16];
    if (!std::equal(key, key + 11, k.key)) {
        k.plan = make_moe_plan(key[0], key[1], key[2], key[3], key[4], key[5], mx, mx_down, parts, n);
        std::copy(key, key + 11, k.key);
    }
    return k.plan;
}

} // namespace

cudaError_t launch_w4_moe(const W4Moe & p, cudaStream_t stream) {
    const bool mx = p.gate.type == GGML_MXFP4, mx_down = p.down.type == GGML_MXFP4;
    const int parts = p.x_type == GGML_F32 || p.norm ? 2 : 1;
    const int E = (int)p.gate.n_expert, d = (int)p.gate.n_in, ff = (int)p.gate.n_out;
    const int steps_d = (int)p.gate.steps, steps_ff = (int)p.down.steps;
    for (int t0 = 0, n = 0; t0 < p.n_tokens; t0 += n) {
        n = std::min(kW4PassTokens, p.n_tokens - t0);
        const MoePlan plan = moe_plan(p, mx, mx_down, parts, n);
        if (!plan.cut.C) return cudaErrorInvalidValue;      // rows this long are refused when the handle is made
        n = plan.n;
        const Cut & cut = plan.cut;
        MoeArgs a{};
        a.gate = p.gate.units;
        a.up = p.up.units;
        a.down = p.down.units;
        a.gate_expert = p.gate.expert_bytes;
        a.up_expert = p.up.expert_bytes;
        a.down_expert = p.down.expert_bytes;
        a.router = p.router;
        a.router_vec = (uintptr_t)p.router % 16 == 0;
        a.down_mx = mx_down;
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
        a.parts = parts;
        a.at = route_at(std::min(E, n * p.n_used), n * p.n_used);
        a.route = static_cast<uint8_t *>(p.workspace);
        a.hidden = a.route + route_room((size_t)n * p.n_used);

        const int nt = product_room(n), s = (steps_d + cut.C - 1) / cut.C;
        a.x_bytes = up_to(s * step_x_bytes(parts, nt), 128);
        a.c_bytes = up_to(s * step_c_bytes(mx, nt), 128);
        a.logit_bytes = up_to(n * E * 4, 128);
        a.clusters = cut.clusters;
        const int fixed = a.x_bytes + a.c_bytes + 2 * a.logit_bytes + ring_bytes(mx, nt, kMoeStages);
        a.inbox = (int)std::max<int64_t>((std::min(kSmShare / cut.resident - kMoeStatic - 4096, kMaxSmem) - fixed) / 2 / 128 * 128, inbox_bytes(n, cut.C, 1, 2));
        cudaError_t e = mx ? launch_gate_up_of<true>(a, parts, cut.C, (size_t)fixed + 2 * a.inbox, stream)
                           : launch_gate_up_of<false>(a, parts, cut.C, (size_t)fixed + 2 * a.inbox, stream);
        if (e != cudaSuccess) return e;

        a.clusters = plan.clusters;
        a.ks = plan.ks;
        a.per_round = plan.per_round;
        a.inbox = plan.inbox;
        a.partial = plan.partial;
        const int C = plan.C;
        const size_t smem = plan.smem;
        if (mx_down) e = n > 1 ? launch_down<true, kSet>(a, C, smem, stream) : launch_down<true, 1>(a, C, smem, stream);
        else e = n > 1 ? launch_down<false, kSet>(a, C, smem, stream) : launch_down<false, 1>(a, C, smem, stream);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

} // namespace rb200
