// AdamW over many tensors at once, moments in 32 or in 8 bits, and the global gradient norm (include/sr_amd.h "optimizer").
//
// One step of a tensor, every operation rounded once to float32 (this file is compiled without contraction, so that the
// results are those of the formulas, bit for bit):
//   g  = grad * factor                         factor: 1, or min(1, max_norm / (norm + 1e-6)) from device memory
//   m' = b1 m + (1 - b1) g                     v' = b2 v + (1 - b2) (g g)
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * (m' / (sqrt(v') * (1 - b2^t)^-1/2 + eps))
//   e' = d e + (1 - d) p'                      the weight average, if there is one
//
// Moments in 8 bits.  256 consecutive values of a tensor (a block) share an exponent E, that of the block's largest value (one
// more if its mantissa is above 1.875, so that no value rounds out of range).  A code is the top of the float that holds
// x * 2^-(E + 112) (m) or x * 2^-(E + 96) (v): those floats have an exponent field of at most 15 or 31, so bits 20 and up are a
// 4-bit exponent and 3 mantissa bits, or a 5-bit exponent and 3 mantissa bits, subnormals included; m has its sign in bit 7.
// Both reach down to 2^-17 of the block's largest gradient (2^-33 of the largest v).  Adding 20 random bits before the cut is
// stochastic rounding: with b2 = 0.999 v moves by a thousandth a step, a hundredth of the distance of two codes, and rounded
// to nearest it would never move; rounded so, its mean is right.  v' > 0 does not round to 0 (m' / (sqrt(0) + eps) would be a
// step of 1 / eps).  bfloat16 weights are rounded the same way for the same reason.  The random bits are a hash of (seed, step,
// number of the element): no state, no order, the same on every run.  A scale that is a power of two decodes exactly, and what
// was decoded encodes to itself, so a checkpoint in float32 resumes where it was.  A block with a NaN, an infinity or a magnitude
// above 1.875 * 2^127 (whose exponent would be 255) has the exponent byte 255 and decodes to NaN as a whole.
//
// What bounds it: memory.  Every value is read and written once: 28 bytes with float32 moments, 16 with 8-bit ones.  256 M float32
// values take 1.39 ms, 5.15 TB/s; four arrays read and three written at once is what costs against the 5.9 TB/s of one array scaled
// in place (5.65 for three read and one written): with the arithmetic taken out the time is the same.  8-bit moments: 128 M float32
// values 0.40 ms, 5.15 TB/s; with bfloat16 weights (10 bytes, 76 vector instructions a value) 96 M take 0.20 to 0.24 ms, and their
// instructions alone 0.19 to issue.
// Work is split into pieces of 1024 consecutive values of one tensor, one per WAVE: most of RRDBNet-FDConv's 8380 tensors are
// smaller than a piece, and a workgroup each would leave three of its four waves idle.  A wave issues the loads of its four groups
// of 256 values (16 bytes per lane and tensor) before it computes, and stores group by group.  Measured against that, on 256 M
// values: pieces of 512 +4 %, of 2048 +1 % (8 bits: +6 %, with bfloat16 +40 %), all loads of one array together +4 %, all stores
// at the end +5 %, nontemporal loads +7 %, stores +1 %, a contiguous eighth per XCD -2 % but +5 to 8 % with 8 bits or bfloat16.
#include "common.h"

#include <math.h>
#include <string.h>

#include <new>
#include <vector>

#pragma clang fp contract(off)

namespace sr {

constexpr int PIECE = 1024;              // values of one wave
constexpr int QBLOCK = SR_ADAMW_BLOCK;   // values that share an exponent
static_assert(QBLOCK == 256, "a wave of 64 lanes holds four values each of a block");
constexpr int NORM_WG = 2048;            // workgroups (= partial sums) of the norm per list: 8 per CU
constexpr uint32_t GOLDEN = 0x9E3779B1u;

struct Rec {  // one tensor, 64 bytes: one scalar load
    void* p;
    void *m, *v;
    uint8_t *me, *ve;
    float* ema;
    int64_t n, index;
};
struct Piece {
    uint32_t tensor, number;  // the number-th PIECE values of the tensor
};

// The gradients' addresses: they are new tensors every step, and a kernel cannot follow a host list.  Short lists travel in the
// kernel's arguments (no copy, no second launch: 8 us of a step of 53 tensors), long ones lie on the device.
struct GradsAt {
    const void* const* at;
    __device__ __forceinline__ const void* operator[](uint32_t i) const { return at[i]; }
};
struct GradsByValue {
    const void* at[SR_ADAMW_BY_VALUE];
    __device__ __forceinline__ const void* operator[](uint32_t i) const { return at[i]; }
};

struct Scalars {
    float b1, c1, b2, c2, decay, step_size, rbc2, eps, d, cd;
    uint32_t k0, k1;
};

__host__ __device__ inline void make_key(uint64_t seed, int64_t step, Scalars& s) {  // splitmix64
    // (G. Steele, D. Lea, C. Flood, "Fast splittable pseudorandom number generators", 2014)
    uint64_t z = seed + (uint64_t)step * 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    z ^= z >> 31;
    s.k0 = (uint32_t)z;
    s.k1 = (uint32_t)(z >> 32);
}
__host__ __device__ inline Scalars make_scalars(const sr_adamw_hyper& h, double lr, int64_t step) {
    Scalars s;
    s.b1 = (float)h.beta1;
    s.c1 = (float)(1.0 - h.beta1);
    s.b2 = (float)h.beta2;
    s.c2 = (float)(1.0 - h.beta2);
    s.decay = (float)(1.0 - lr * h.weight_decay);
    s.step_size = (float)(lr / (1.0 - pow(h.beta1, (double)step)));
    s.rbc2 = (float)pow(1.0 - pow(h.beta2, (double)step), -0.5);
    s.eps = (float)h.eps;
    s.d = (float)h.ema_decay;
    s.cd = (float)(1.0 - h.ema_decay);
    make_key(h.seed, step, s);
    return s;
}

// 32 random bits for element (hi, lo) of a step; hi_c = hi * GOLDEN.  The two odd constants and the shifts are those of the mixer of
// 32-bit words with the least bias that Christopher Wellons found by search and published in 2018; k1 enters between them so that steps whose k0 differ in few bits do not share values.
__device__ __forceinline__ uint32_t mix(uint32_t lo, uint32_t hi_c, uint32_t k0, uint32_t k1) {
    uint32_t x = (lo ^ k0) + hi_c;
    x = (x ^ (x >> 16)) * 0x7FEB352Du + k1;
    x = (x ^ (x >> 15)) * 0x846CA68Bu;
    return x ^ (x >> 16);
}

// pointers that come out of a table are of no known address space, and FLAT instructions (which also wait for LDS) would follow
#define GLOBAL __attribute__((address_space(1)))
template <typename T>
__device__ __forceinline__ GLOBAL T* global(const void* p) {
    return (GLOBAL T*)const_cast<void*>(p);
}

// vectors with the alignment of their elements: tensors are views at any offset (the gradients of one layer are pieces of one
// buffer); the hardware loads and stores 16 bytes at any address
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h4u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint8_t b4u __attribute__((ext_vector_type(4), aligned(1)));

// 4 values at p, of which the first cnt exist (the others: 0)
__device__ __forceinline__ void load4(const GLOBAL float* p, int cnt, float (&r)[4]) {
    if (cnt >= 4) {
        const f4u x = *(const GLOBAL f4u*)p;
        r[0] = x.x, r[1] = x.y, r[2] = x.z, r[3] = x.w;
    } else {
        r[0] = cnt > 0 ? p[0] : 0.f, r[1] = cnt > 1 ? p[1] : 0.f, r[2] = cnt > 2 ? p[2] : 0.f, r[3] = 0.f;
    }
}
__device__ __forceinline__ void load4(const GLOBAL bf16_t* p, int cnt, float (&r)[4]) {
    if (cnt >= 4) {
        const h4u x = *(const GLOBAL h4u*)p;
        r[0] = bf16_to_f32(x.x), r[1] = bf16_to_f32(x.y), r[2] = bf16_to_f32(x.z), r[3] = bf16_to_f32(x.w);
    } else {
        r[0] = cnt > 0 ? bf16_to_f32(p[0]) : 0.f, r[1] = cnt > 1 ? bf16_to_f32(p[1]) : 0.f, r[2] = cnt > 2 ? bf16_to_f32(p[2]) : 0.f, r[3] = 0.f;
    }
}
__device__ __forceinline__ void store4(GLOBAL float* p, int cnt, const float (&r)[4]) {
    if (cnt >= 4) {
        const f4u x = {r[0], r[1], r[2], r[3]};
        *(GLOBAL f4u*)p = x;
    } else {
        if (cnt > 0) p[0] = r[0];
        if (cnt > 1) p[1] = r[1];
        if (cnt > 2) p[2] = r[2];
    }
}
__device__ __forceinline__ void store4(GLOBAL bf16_t* p, int cnt, const uint16_t (&r)[4]) {
    if (cnt >= 4) {
        const h4u x = {r[0], r[1], r[2], r[3]};
        *(GLOBAL h4u*)p = x;
    } else {
        if (cnt > 0) p[0] = r[0];
        if (cnt > 1) p[1] = r[1];
        if (cnt > 2) p[2] = r[2];
    }
}
__device__ __forceinline__ uint32_t load4b(const GLOBAL uint8_t* p, int cnt) {  // byte j of the result: code j
    if (cnt >= 4) return __builtin_bit_cast(uint32_t, *(const GLOBAL b4u*)p);
    uint32_t r = 0;
    if (cnt > 0) r = p[0];
    if (cnt > 1) r |= (uint32_t)p[1] << 8;
    if (cnt > 2) r |= (uint32_t)p[2] << 16;
    return r;
}
__device__ __forceinline__ void store4b(GLOBAL uint8_t* p, int cnt, uint32_t x) {
    if (cnt >= 4) {
        *(GLOBAL b4u*)p = __builtin_bit_cast(b4u, x);
    } else {
        if (cnt > 0) p[0] = (uint8_t)x;
        if (cnt > 1) p[1] = (uint8_t)(x >> 8);
        if (cnt > 2) p[2] = (uint8_t)(x >> 16);
    }
}

// the largest of 64 lanes' unsigned values, in all lanes (every lane must be active): rows of 16, then across the rows
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
    return x > y ? x : y;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = dpp_max<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
    x = dpp_max<0x112, 0xf>(x);
    x = dpp_max<0x114, 0xf>(x);
    x = dpp_max<0x118, 0xf>(x);
    x = dpp_max<0x142, 0xa>(x);  // row_bcast 15
    x = dpp_max<0x143, 0xc>(x);  // row_bcast 31
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

// the exponent byte of a block from the bits of its largest magnitude (as integers, NaN > infinity > numbers)
__device__ __forceinline__ uint32_t block_exponent(uint32_t top) {
    const uint32_t e = (top + 0x0FFFFFu) >> 23;
    return e < 1 ? 1 : e > 254 ? 255 : e;
}
constexpr int M_BIAS = 112, V_BIAS = 96;  // where the exponent field of the block's largest value lies: 127 - 15, 127 - 31

// the four codes in a word -> values
__device__ __forceinline__ void decode4_m(uint32_t c, uint32_t eb, float (&m)[4]) {
    const int e = (int)eb - 127 + M_BIAS;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int t = (int)(c << (24 - 8 * j)) >> 4;  // sign in 27 .. 31, the other bits in 20 .. 26, other codes below
        m[j] = ldexpf(__uint_as_float((uint32_t)t & 0x87F00000u), e);
    }
    if (eb == 255) m[0] = m[1] = m[2] = m[3] = __uint_as_float(0x7FC00000u);
}
__device__ __forceinline__ void decode4_v(uint32_t c, uint32_t eb, float (&v)[4]) {
    const int e = (int)eb - 127 + V_BIAS;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = ldexpf(__uint_as_float((c >> 8 * j & 0xFF) << 20), e);
    if (eb == 255) v[0] = v[1] = v[2] = v[3] = __uint_as_float(0x7FC00000u);
}
__device__ __forceinline__ uint32_t top_bytes(const uint32_t (&w)[4]) {
    return __builtin_amdgcn_perm(w[1], w[0], 0x0C0C0703u) | __builtin_amdgcn_perm(w[3], w[2], 0x07030C0Cu);
}
// the largest magnitude of a wave's 4 * 64 values, as bits
__device__ __forceinline__ uint32_t block_top(const float (&x)[4]) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = max(top, __float_as_uint(x[j]) << 1);
    return wave_max(top) >> 1;
}
// Values -> codes (byte j: value j).  The float of a code's place in the format, shifted left by four, has the code in its top
// byte; below it come 16 random bits and the middle of what is finer.  Nothing carries out: block_exponent left room.
__device__ __forceinline__ uint32_t encode4_m(const float (&m)[4], uint32_t eb, const uint32_t (&h)[4]) {
    const int e = 127 - M_BIAS - (int)eb;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t y = (__float_as_uint(ldexpf(fabsf(m[j]), e)) << 4) + __builtin_amdgcn_perm(h[j], 0x80u, 0x0C050400u);
        w[j] = (y & 0x7FFFFFFFu) | (__float_as_uint(m[j]) & 0x80000000u);
    }
    return eb == 255 ? 0 : top_bytes(w);
}
__device__ __forceinline__ uint32_t encode4_v(const float (&v)[4], uint32_t eb, const uint32_t (&h)[4]) {
    const int e = 127 - V_BIAS - (int)eb;
    uint32_t w[4], least = ~0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        w[j] = (__float_as_uint(ldexpf(fabsf(v[j]), e)) << 4) + __builtin_amdgcn_perm(h[j], 0x80u, 0x0C070600u);
        least = min(least, w[j]);
    }
    if (least < 1u << 24) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (w[j] < 1u << 24 && v[j] > 0.f) w[j] = 1u << 24;
    }
    return eb == 255 ? 0 : top_bytes(w);
}
__device__ __forceinline__ void hash4(uint64_t at, const Scalars& s, uint32_t (&h)[4]) {
    const uint32_t lo = (uint32_t)at, c = (uint32_t)(at >> 32) * GOLDEN;
    if (lo < 0xFFFFFFFCu) {
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = mix(lo + j, c, s.k0, s.k1);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = mix((uint32_t)(at + j), (uint32_t)((at + j) >> 32) * GOLDEN, s.k0, s.k1);
    }
}
// stochastic rounding to bfloat16; infinities and (quiet) NaN as they are
__device__ __forceinline__ uint16_t round_bf16(float x, uint32_t h) {
    const uint32_t noise = __builtin_isfinite(x) ? (h * GOLDEN) >> 16 : 0;
    return (uint16_t)((__float_as_uint(x) + noise) >> 16);
}

// Square root and quotient, correctly rounded as sqrtf and `/` are, without their handling of the ends of the range: half the
// instructions, which is what bounds the step with 8-bit moments.  rsq / rcp are good to one ulp; one correction by the exact
// residual rounds the root correctly (checked for all 2^24 significands) and the reciprocal (all 2^23), and with a correctly
// rounded reciprocal the same correction rounds the quotient correctly (Markstein's theorem).  The ranges below keep every
// residual exact: 0 <= x < 2^124, no subnormals but 0; |a| 0 or in [2^-85, 2^84], b in [2^-40, 2^57].
__device__ __forceinline__ float root(float x) {
    const float y = __builtin_amdgcn_rsqf(fmaxf(x, 0x1p-100f));
    const float r = x * y;
    return fmaf(fmaf(-r, r, x), 0.5f * y, r);
}
__device__ __forceinline__ float quotient(float a, float b) {
    float r = __builtin_amdgcn_rcpf(b);
    r = fmaf(fmaf(-b, r, 1.f), r, r);
    const float q = a * r;
    return fmaf(fmaf(-b, q, a), r, q);
}

__device__ __forceinline__ void moments4(const Scalars& s, float factor, const float (&g)[4], float (&m)[4], float (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float gj = g[j] * factor;
        m[j] = m[j] * s.b1 + gj * s.c1;
        v[j] = v[j] * s.b2 + (gj * gj) * s.c2;
    }
}
__device__ __forceinline__ void weights4(const Scalars& s, float (&p)[4], const float (&m)[4], const float (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = p[j] * s.decay - (m[j] / (sqrtf(v[j]) * s.rbc2 + s.eps)) * s.step_size;
}
// The same for v < 2^60 and |m| < 2^20, as a block's exponents tell, and for constants in_range().  v and m are raised by 2^64 first
// (which keeps subnormals in range) and the constants that follow take it back: exact, so the results are the same bits unless the
// quotient itself is subnormal, where this one does not round it and the update is below 2^-126.
__device__ __forceinline__ bool in_range(const Scalars& s) {
    // the divisor between 2^-40 and 2^57 (1 - b2 is 2^-53 at least), and step_size * 2^-64 normal
    return s.eps >= 0x1p-40f && s.eps <= 0x1p40f && s.step_size >= 0x1p-60f;
}
__device__ __forceinline__ void weights4_in_range(const Scalars& s, float (&p)[4], const float (&m)[4], const float (&v)[4]) {
    const float rbc2 = s.rbc2 * 0x1p-32f, step_size = s.step_size * 0x1p-64f;
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = p[j] * s.decay - quotient(m[j] * 0x1p64f, root(v[j] * 0x1p64f) * rbc2 + s.eps) * step_size;
}

template <typename P, int BITS, bool FULL>
__device__ __forceinline__ void step_piece(const Rec& r, const void* grad, const Scalars& s, float factor, int64_t off, int left, int lane) {
    constexpr int GROUPS = PIECE / 256;
    GLOBAL P* pp = global<P>(r.p) + off;
    const GLOBAL P* gp = global<P>(grad) + off;
    GLOBAL float* ep = global<float>(r.ema) + off;
    GLOBAL float *m32 = global<float>(r.m) + off, *v32 = global<float>(r.v) + off;
    GLOBAL uint8_t *m8 = global<uint8_t>(r.m) + off, *v8 = global<uint8_t>(r.v) + off;
    GLOBAL uint8_t *me = global<uint8_t>(r.me) + off / QBLOCK, *ve = global<uint8_t>(r.ve) + off / QBLOCK;
    float p[GROUPS][4], g[GROUPS][4], m[GROUPS][4], v[GROUPS][4], e[GROUPS][4];
    uint32_t mc[GROUPS], vc[GROUPS], meb[GROUPS], veb[GROUPS];
    if (BITS == 8 && FULL) {  // four exponents at once
        const uint32_t a = __builtin_amdgcn_readfirstlane(load4b(me, 4)), b = __builtin_amdgcn_readfirstlane(load4b(ve, 4));
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) meb[k] = a >> 8 * k & 0xFF, veb[k] = b >> 8 * k & 0xFF;
    }
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        if (!FULL && k * 256 >= left) break;
        const int at = k * 256 + lane * 4, cnt = FULL ? 4 : left - at;
        load4(pp + at, cnt, p[k]);
        load4(gp + at, cnt, g[k]);
        if (BITS == 32) {
            load4(m32 + at, cnt, m[k]);
            load4(v32 + at, cnt, v[k]);
        } else {
            mc[k] = load4b(m8 + at, cnt);
            vc[k] = load4b(v8 + at, cnt);
            if (!FULL) meb[k] = __builtin_amdgcn_readfirstlane(me[k]), veb[k] = __builtin_amdgcn_readfirstlane(ve[k]);
        }
        if (r.ema) load4(ep + at, cnt, e[k]);
    }
    uint32_t em = 0, ev = 0;  // the new exponents
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        if (!FULL && k * 256 >= left) break;
        const int at = k * 256 + lane * 4, cnt = FULL ? 4 : left - at;
        if (BITS == 8) {
            decode4_m(mc[k], meb[k], m[k]);
            decode4_v(vc[k], veb[k], v[k]);
        }
        moments4(s, factor, g[k], m[k], v[k]);
        uint32_t a = 0, b = 0;
        if (BITS == 8) {
            if (!FULL) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // a lane past the end must not take part in the block's maximum
                    m[k][j] = j < cnt ? m[k][j] : 0.f;
                    v[k][j] = j < cnt ? v[k][j] : 0.f;
                }
            }
            a = block_exponent(block_top(m[k]));
            b = block_exponent(block_top(v[k]));
            em |= a << 8 * k;
            ev |= b << 8 * k;
        }
        if (BITS == 8 && a < 127 + 20 && b < 127 + 60 && in_range(s))
            weights4_in_range(s, p[k], m[k], v[k]);
        else
            weights4(s, p[k], m[k], v[k]);
        if (r.ema) {
#pragma unroll
            for (int j = 0; j < 4; ++j) e[k][j] = e[k][j] * s.d + p[k][j] * s.cd;
            store4(ep + at, cnt, e[k]);
        }
        uint32_t h[4];
        if (BITS == 8 || sizeof(P) == 2) hash4((uint64_t)(r.index + off + at), s, h);
        if constexpr (sizeof(P) == 2) {
            uint16_t q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = round_bf16(p[k][j], h[j]);
            store4(pp + at, cnt, q);
        } else {
            store4(pp + at, cnt, p[k]);
        }
        if (BITS == 32) {
            store4(m32 + at, cnt, m[k]);
            store4(v32 + at, cnt, v[k]);
        } else {
            store4b(m8 + at, cnt, encode4_m(m[k], a, h));
            store4b(v8 + at, cnt, encode4_v(v[k], b, h));
        }
    }
    if (BITS == 8 && lane == 0) {
        const int blocks = FULL ? GROUPS : (left + QBLOCK - 1) / QBLOCK;
        store4b(me, blocks, em);
        store4b(ve, blocks, ev);
    }
}

__device__ __forceinline__ uint32_t wave_number() {
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * (blockDim.x / 64) + threadIdx.x / 64));
}

template <typename P, int BITS, typename G>
__global__ __launch_bounds__(256) void adamw_step_kernel(const Rec* __restrict__ recs, const Piece* __restrict__ pieces, uint32_t npieces,
                                                         const float* __restrict__ factor_at, const Scalars* __restrict__ scalars_at,
                                                         Scalars scalars, G grads) {
    const uint32_t w = wave_number();
    const int lane = threadIdx.x & 63;
    if (w >= npieces) return;
    const Piece c = pieces[w];
    const void* gp = grads[c.tensor];
    if (gp == (const void*)SR_ADAMW_SKIP) return;
    const Rec r = recs[c.tensor];
    if (!gp && !r.ema) return;
    Scalars s = scalars;
    if (scalars_at) s = *scalars_at;
    float factor = 1.f;
    if (factor_at) factor = *factor_at;
    const int64_t off = (int64_t)c.number * PIECE;
    const int left = r.n - off < PIECE ? (int)(r.n - off) : PIECE;
    if (!gp) {  // no gradient: the weights stay, their average goes on
        GLOBAL float* e = global<float>(r.ema) + off;
        const GLOBAL P* p = global<P>(r.p) + off;
        for (int at = lane; at < left; at += 64) {
            float w;
            if constexpr (sizeof(P) == 2)
                w = bf16_to_f32(p[at]);
            else
                w = p[at];
            e[at] = e[at] * s.d + w * s.cd;
        }
        return;
    }
    if (left == PIECE)
        step_piece<P, BITS, true>(r, gp, s, factor, off, left, lane);
    else
        step_piece<P, BITS, false>(r, gp, s, factor, off, left, lane);
}

// step counter and scalars of a captured step: the host's values are fixed at capture, these move with every replay
__global__ void adamw_tick_kernel(sr_adamw_hyper h, const float* lr, int64_t* step, Scalars* out) {
    const int64_t t = *step + 1;
    *step = t;
    *out = make_scalars(h, lr ? (double)*lr : h.lr, t);
}

// Moments as the values they stand for, at the tensors' places in one flat pair of arrays.  Four values a lane and group, all
// groups' loads first.
template <typename TO>
__device__ __forceinline__ void put4(GLOBAL TO* to, int cnt, const float (&x)[4]) {
    if constexpr (sizeof(TO) == 2) {
        uint16_t y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = f32_to_bf16(x[j]);
        store4(to, cnt, y);
    } else {
        store4(to, cnt, x);
    }
}
template <typename TO, int BITS, bool FULL>
__device__ __forceinline__ void moments_piece(const Rec& r, int64_t off, int left, int lane, TO* mo, TO* vo) {
    constexpr int GROUPS = PIECE / 256;
    float m[GROUPS][4], v[GROUPS][4];
    uint32_t mc[GROUPS], vc[GROUPS], a[GROUPS], b[GROUPS];
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        if (!FULL && k * 256 >= left) break;
        const int at = k * 256 + lane * 4, cnt = FULL ? 4 : left - at;
        if (BITS == 32) {
            load4(global<float>(r.m) + off + at, cnt, m[k]);
            load4(global<float>(r.v) + off + at, cnt, v[k]);
        } else {
            mc[k] = load4b(global<uint8_t>(r.m) + off + at, cnt);
            vc[k] = load4b(global<uint8_t>(r.v) + off + at, cnt);
            a[k] = global<uint8_t>(r.me)[off / QBLOCK + k];
            b[k] = global<uint8_t>(r.ve)[off / QBLOCK + k];
        }
    }
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        if (!FULL && k * 256 >= left) break;
        const int at = k * 256 + lane * 4, cnt = FULL ? 4 : left - at;
        if (BITS == 8) {
            decode4_m(mc[k], __builtin_amdgcn_readfirstlane(a[k]), m[k]);
            decode4_v(vc[k], __builtin_amdgcn_readfirstlane(b[k]), v[k]);
        }
        put4(global<TO>(mo) + r.index + off + at, cnt, m[k]);
        put4(global<TO>(vo) + r.index + off + at, cnt, v[k]);
    }
}
template <typename TO, int BITS>
__global__ __launch_bounds__(256) void adamw_moments_kernel(const Rec* __restrict__ recs, const Piece* __restrict__ pieces, uint32_t npieces,
                                                            TO* __restrict__ mo, TO* __restrict__ vo) {
    const uint32_t w = wave_number();
    const int lane = threadIdx.x & 63;
    if (w >= npieces) return;
    const Piece c = pieces[w];
    const Rec r = recs[c.tensor];
    const int64_t off = (int64_t)c.number * PIECE;
    const int left = r.n - off < PIECE ? (int)(r.n - off) : PIECE;
    if (left == PIECE)
        moments_piece<TO, BITS, true>(r, off, left, lane, mo, vo);
    else
        moments_piece<TO, BITS, false>(r, off, left, lane, mo, vo);
}

template <int BITS>
__global__ __launch_bounds__(256) void adamw_set_moments_kernel(const Rec* __restrict__ recs, const Piece* __restrict__ pieces, uint32_t npieces,
                                                                const float* __restrict__ mi, const float* __restrict__ vi, Scalars s) {
    const uint32_t w = wave_number();
    const int lane = threadIdx.x & 63;
    if (w >= npieces) return;
    const Piece c = pieces[w];
    const Rec r = recs[c.tensor];
    const int64_t off = (int64_t)c.number * PIECE;
    const int left = r.n - off < PIECE ? (int)(r.n - off) : PIECE;
#pragma unroll
    for (int k = 0; k < PIECE / 256; ++k) {
        if (k * 256 >= left) return;
        const int at = k * 256 + lane * 4, cnt = left - at;
        float m[4], v[4];
        load4(global<float>(mi) + r.index + off + at, cnt, m);
        load4(global<float>(vi) + r.index + off + at, cnt, v);
        if (BITS == 32) {
            store4(global<float>(r.m) + off + at, cnt, m);
            store4(global<float>(r.v) + off + at, cnt, v);
        } else {
            uint32_t h[4];
            hash4((uint64_t)(r.index + off + at), s, h);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = v[j] >= 0.f ? v[j] : __uint_as_float(0x7FC00000u);  // no second moment: as sqrt has it
            const uint32_t a = block_exponent(block_top(m)), b = block_exponent(block_top(v));
            store4b(global<uint8_t>(r.m) + off + at, cnt, encode4_m(m, a, h));
            store4b(global<uint8_t>(r.v) + off + at, cnt, encode4_v(v, b, h));
            if (lane == 0) {
                global<uint8_t>(r.me)[off / QBLOCK + k] = (uint8_t)a;
                global<uint8_t>(r.ve)[off / QBLOCK + k] = (uint8_t)b;
            }
        }
    }
}

// ---- global gradient norm ---------------------------------------------------------------------------------------------
// Squares are added in float64 (a float32 square overflows from 1.8e19 on, and 1e8 of them lose three digits; float64 multiply-adds
// run at the float32 rate here), in an order that the shapes alone determine.  Work items are runs of consecutive values; waves
// take them in turn, four 16-byte loads of every lane in flight.  256 M bfloat16 values: norm 0.10 ms, 5 TB/s; scaling 0.18 ms, 5.8
// TB/s (0.21 with one 8-byte load at a time); both 0.27, and 0.29 if the scaling does not go backwards.  Right after a step the
// norm of 48 M bfloat16 values takes 37 us instead of 25: the memory-side cache is full of what the step wrote, and every line read
// pushes one out.  Two or four pieces at a time did not change that.
template <typename G>
struct PieceSource {  // the pieces of an optimizer's list, gradients by tensor
    const Rec* recs;
    const Piece* pieces;
    G grads;
    template <typename T>
    __device__ __forceinline__ const T* run(uint32_t i, int64_t& n) const {
        const Piece c = pieces[i];
        const T* g = (const T*)grads[c.tensor];
        n = 0;
        if (!g || g == (const T*)SR_ADAMW_SKIP) return g;
        const int64_t off = (int64_t)c.number * PIECE, left = recs[c.tensor].n - off;
        n = left < PIECE ? left : PIECE;
        return g + off;
    }
};
struct SpansAt {
    const sr_grad_span* at;
    __device__ __forceinline__ sr_grad_span operator[](uint32_t i) const { return at[i]; }
};
struct SpansByValue {
    sr_grad_span at[SR_GRAD_SPANS_BY_VALUE];
    __device__ __forceinline__ sr_grad_span operator[](uint32_t i) const { return at[i]; }
};
template <typename S>
struct SpanSource {
    S spans;
    template <typename T>
    __device__ __forceinline__ const T* run(uint32_t i, int64_t& n) const {
        const sr_grad_span s = spans[i];
        n = s.n;
        return (const T*)s.g;
    }
};

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int k = 32; k; k >>= 1) x += __shfl_xor(x, k, 64);
    return x;
}

// 16 bytes of gradients
template <typename T>
constexpr int W16 = 16 / (int)sizeof(T);
typedef uint32_t w4u __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ void load16(const GLOBAL float* p, float (&x)[4]) { load4(p, 4, x); }
__device__ __forceinline__ void load16(const GLOBAL bf16_t* p, float (&x)[8]) {
    const w4u w = *(const GLOBAL w4u*)p;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[2 * j] = lo_f(w[j]), x[2 * j + 1] = hi_f(w[j]);
}
__device__ __forceinline__ void store16(GLOBAL float* p, const float (&x)[4]) { store4(p, 4, x); }
__device__ __forceinline__ void store16(GLOBAL bf16_t* p, const float (&x)[8]) {
    w4u w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack2(x[2 * j], x[2 * j + 1]);
    *(GLOBAL w4u*)p = w;
}

// U loads in flight, as long as there are U more for every lane
template <int U, typename T>
__device__ __forceinline__ void add_squares(const GLOBAL T* g, int64_t& at, int64_t whole, double (&acc)[4]) {
    constexpr int W = W16<T>;
    for (; at + (U - 1) * 64 * W < whole; at += U * 64 * W) {
        float x[U][W];
#pragma unroll
        for (int k = 0; k < U; ++k) load16(g + at + k * 64 * W, x[k]);
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
            for (int j = 0; j < W; ++j) acc[j & 3] = fma((double)x[k][j], (double)x[k][j], acc[j & 3]);
    }
}
template <int U, typename T>
__device__ __forceinline__ void scale_by(GLOBAL T* g, int64_t& at, int64_t whole, float factor) {
    constexpr int W = W16<T>;
    for (; at + (U - 1) * 64 * W < whole; at += U * 64 * W) {
        float x[U][W];
#pragma unroll
        for (int k = 0; k < U; ++k) load16(g + at + k * 64 * W, x[k]);
#pragma unroll
        for (int k = 0; k < U; ++k) {
#pragma unroll
            for (int j = 0; j < W; ++j) x[k][j] *= factor;
            store16(g + at + k * 64 * W, x[k]);
        }
    }
}

template <typename T, typename S>
__global__ __launch_bounds__(256) void grad_norm_kernel(S src, uint32_t items, double* __restrict__ partial) {
    constexpr int W = W16<T>;
    __shared__ double sums[4];
    const int lane = threadIdx.x & 63;
    double acc[4] = {0, 0, 0, 0};
    for (uint32_t i = wave_number(); i < items; i += gridDim.x * 4) {
        int64_t n;
        const GLOBAL T* g = global<T>(src.template run<T>(i, n));
        const int64_t whole = n / (64 * W) * (64 * W);  // full loads of all lanes
        int64_t at = lane * W;
        add_squares<4>(g, at, whole, acc);
        add_squares<2>(g, at, whole, acc);
        add_squares<1>(g, at, whole, acc);
#pragma unroll
        for (int k = 0; k < W; ++k) {  // what is left, one value a lane
            const int64_t rest = whole + k * 64 + lane;
            const float x = rest < n ? Elem<T>::ld((const T*)(g + rest)) : 0.f;
            acc[k & 3] = fma((double)x, (double)x, acc[k & 3]);
        }
    }
    const double sum = wave_sum((acc[0] + acc[1]) + (acc[2] + acc[3]));
    if (lane == 0) sums[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

struct Partials {
    int32_t n[SR_GRAD_MAX_LISTS];
    int32_t lists;
};
__global__ __launch_bounds__(256) void grad_norm_finish_kernel(Partials parts, const double* __restrict__ partial, double max_norm, float* __restrict__ out) {
    __shared__ double sums[4];
    double acc = 0;
    for (int l = 0; l < parts.lists; ++l)
        for (int i = threadIdx.x; i < parts.n[l]; i += 256) acc += partial[l * NORM_WG + i];
    acc = wave_sum(acc);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x / 64] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        const double norm = sqrt((sums[0] + sums[1]) + (sums[2] + sums[3]));
        const double f = max_norm / (norm + 1e-6);
        out[0] = (float)norm;
        out[1] = f >= 1.0 ? 1.f : (float)f;  // NaN stays
    }
}

template <typename T, typename S>
__global__ __launch_bounds__(256) void grad_scale_kernel(S spans, uint32_t items, const float* __restrict__ factor_at) {
    constexpr int W = W16<T>;
    const float factor = *factor_at;
    if (factor == 1.f) return;
    const int lane = threadIdx.x & 63;
    for (uint32_t i = wave_number(); i < items; i += gridDim.x * 4) {
        const sr_grad_span span = spans[items - 1 - i];  // backwards: what the norm read last is still in the memory-side cache
        GLOBAL T* g = global<T>(span.g);
        const int64_t n = span.n, whole = n / (64 * W) * (64 * W);
        int64_t at = lane * W;
        scale_by<4>(g, at, whole, factor);
        scale_by<2>(g, at, whole, factor);
        scale_by<1>(g, at, whole, factor);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const int64_t rest = whole + k * 64 + lane;
            if (rest < n) Elem<T>::st((T*)(g + rest), Elem<T>::ld((const T*)(g + rest)) * factor);
        }
    }
}

// ---- small host -> device copies through kernel arguments ---------------------------------------------------------------
constexpr int UPLOAD = 3840;  // bytes per launch: kernel arguments are 4 KB
struct UploadArgs {
    uint64_t dst;
    int32_t bytes;
    int32_t pad;
    uint32_t data[UPLOAD / 4];
};
__global__ __launch_bounds__(256) void upload_kernel(UploadArgs a) {
    for (int i = threadIdx.x; i < a.bytes / 4; i += 256) ((uint32_t*)a.dst)[i] = a.data[i];
}

// A word per workgroup, written behind its barrier, tells that it has read its part: no counter that would have to be cleared.
// 128 KB of reads across the host link in flight (one workgroup alone: 67 KB in 9 us instead of 4).
constexpr uint32_t PINNED_WG = 1024, PINNED_ALL = PINNED_WG * SR_UPLOAD_WORDS;
__global__ __launch_bounds__(PINNED_WG) void upload_pinned_kernel(const uint32_t* __restrict__ src, uint32_t* __restrict__ dst, uint32_t words,
                                                                  int64_t* done, int64_t ticket) {
    const uint32_t quads = words / 4, me = blockIdx.x * PINNED_WG + threadIdx.x;
    for (uint32_t i = me; i < quads; i += PINNED_ALL) ((uint4*)dst)[i] = ((const uint4*)src)[i];
    if (me < (words & 3)) dst[quads * 4 + me] = src[quads * 4 + me];
    __syncthreads();
    if (threadIdx.x == 0) __hip_atomic_store(done + blockIdx.x, ticket, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
}

}  // namespace sr

using namespace sr;

struct sr_adamw {
    int dtype, bits, count, device;
    uint32_t npieces;
    bool ema;
    void* tables;  // Rec[count], Piece[npieces]
    const Rec* recs() const { return (const Rec*)tables; }
    const Piece* pieces() const { return (const Piece*)((const char*)tables + sizeof(Rec) * (size_t)count); }
};

namespace {
int build_tables(const sr_adamw_tensor* t, int count, int dtype, int bits, std::vector<Rec>& recs, std::vector<Piece>& pieces, bool& ema) {
    int with_ema = 0;
    uint64_t total = 0;
    for (int i = 0; i < count; ++i) {
        const sr_adamw_tensor& x = t[i];
        SR_REQUIRE(x.n >= 0 && x.n <= ((int64_t)1 << 40) && x.index >= 0 && x.index <= ((int64_t)1 << 50));
        SR_REQUIRE(x.n == 0 || (x.p && x.m && x.v && (bits == 32 || (x.me && x.ve))));
        const uintptr_t align = dtype == SR_F32 ? 4 : 2;
        SR_REQUIRE((uintptr_t)x.p % align == 0 && (uintptr_t)x.ema % 4 == 0);
        SR_REQUIRE(bits == 8 || ((uintptr_t)x.m % 4 == 0 && (uintptr_t)x.v % 4 == 0));
        if (x.n) with_ema |= x.ema ? 1 : 2;
        total += (uint64_t)(x.n + PIECE - 1) / PIECE;
    }
    SR_REQUIRE(with_ema != 3 && total <= 0x7FFFFFFFu);
    ema = with_ema == 1;
    recs.resize(count);
    pieces.reserve(total);
    for (int i = 0; i < count; ++i) {
        recs[i] = {t[i].p, t[i].m, t[i].v, t[i].me, t[i].ve, t[i].ema, t[i].n, t[i].index};
        const uint32_t k = (uint32_t)((t[i].n + PIECE - 1) / PIECE);
        for (uint32_t j = 0; j < k; ++j) pieces.push_back({(uint32_t)i, j});
    }
    return SR_OK;
}
int on_device(const sr_adamw* l) {
    int dev = 0;
    SR_HIP(hipGetDevice(&dev));
    return dev == l->device ? SR_OK : SR_ERR_STATE;
}
uint32_t waves_to_wgs(uint32_t waves) { return (waves + 3) / 4; }
int check_hyper(const sr_adamw_hyper* h, int64_t step) {
    SR_REQUIRE(h);
    SR_REQUIRE(h->lr >= 0 && h->beta1 >= 0 && h->beta1 < 1 && h->beta2 >= 0 && h->beta2 < 1 && h->eps >= 0 && h->weight_decay >= 0);
    SR_REQUIRE(h->ema_decay >= 0 && h->ema_decay <= 1 && step >= 1);
    return SR_OK;
}
}  // namespace

extern "C" int sr_adamw_create(int dtype, int bits, int count, const sr_adamw_tensor* tensors, sr_adamw** out) {
    SR_REQUIRE(out && count > 0 && tensors && (dtype == SR_F32 || dtype == SR_BF16) && (bits == 32 || bits == 8));
    *out = nullptr;
    try {
        std::vector<Rec> recs;
        std::vector<Piece> pieces;
        bool ema = false;
        const int rc = build_tables(tensors, count, dtype, bits, recs, pieces, ema);
        if (rc) return rc;
        int dev = 0;
        SR_HIP(hipGetDevice(&dev));
        sr_adamw* l = new sr_adamw{dtype, bits, count, dev, (uint32_t)pieces.size(), ema, nullptr};
        const size_t rb = sizeof(Rec) * recs.size(), pb = sizeof(Piece) * pieces.size();
        hipError_t e = hipMalloc(&l->tables, rb + pb);
        if (e == hipSuccess) e = hipMemcpy(l->tables, recs.data(), rb, hipMemcpyHostToDevice);
        if (e == hipSuccess && pb) e = hipMemcpy((char*)l->tables + rb, pieces.data(), pb, hipMemcpyHostToDevice);
        if (e != hipSuccess) {
            sr_adamw_destroy(l);
            return hip_fail(e);
        }
        *out = l;
        return SR_OK;
    } catch (...) {  // no memory for the tables
        return SR_ERR_STATE;
    }
}

extern "C" void sr_adamw_destroy(sr_adamw* l) {
    if (!l) return;
    if (l->tables) (void)hipFree(l->tables);
    delete l;
}

namespace {
GradsByValue by_value(const sr_adamw* l, const void* const* grads) {
    GradsByValue g;
    memcpy(g.at, grads, sizeof(void*) * (size_t)l->count);
    memset(g.at + l->count, 0, sizeof(void*) * (size_t)(SR_ADAMW_BY_VALUE - l->count));
    return g;
}
template <typename G>
void launch_step(const sr_adamw* l, const G& g, const Scalars* at, const Scalars& s, const float* factor, hipStream_t st) {
    const dim3 grid(waves_to_wgs(l->npieces));
#define SR_STEP(P, BITS) adamw_step_kernel<P, BITS, G><<<grid, 256, 0, st>>>(l->recs(), l->pieces(), l->npieces, factor, at, s, g)
    if (l->dtype == SR_F32) {
        if (l->bits == 32)
            SR_STEP(float, 32);
        else
            SR_STEP(float, 8);
    } else {
        if (l->bits == 32)
            SR_STEP(bf16_t, 32);
        else
            SR_STEP(bf16_t, 8);
    }
#undef SR_STEP
}
SpansByValue by_value(const sr_grad_span* spans, int64_t n) {
    SpansByValue s;
    memset(&s, 0, sizeof(s));
    memcpy(s.at, spans, sizeof(sr_grad_span) * (size_t)n);
    return s;
}
template <typename S>
void launch_scale(int dtype, uint32_t wgs, const S& spans, uint32_t items, const float* factor, hipStream_t st) {
    if (dtype == SR_F32)
        grad_scale_kernel<float><<<wgs, 256, 0, st>>>(spans, items, factor);
    else
        grad_scale_kernel<bf16_t><<<wgs, 256, 0, st>>>(spans, items, factor);
}
template <typename S>
void launch_norm(int dtype, uint32_t wgs, const S& src, uint32_t items, double* out, hipStream_t st) {
    if (dtype == SR_F32)
        grad_norm_kernel<float><<<wgs, 256, 0, st>>>(src, items, out);
    else
        grad_norm_kernel<bf16_t><<<wgs, 256, 0, st>>>(src, items, out);
}
}  // namespace

extern "C" int sr_adamw_step(const sr_adamw* l, const sr_adamw_hyper* h, int64_t step, const void* scalars, const void* const* grads, int on_host,
                             const float* factor, void* stream) {
    SR_REQUIRE(l && grads && (!on_host || l->count <= SR_ADAMW_BY_VALUE));
    Scalars s = {};
    if (!scalars) {
        const int rc = check_hyper(h, step);
        if (rc) return rc;
        s = make_scalars(*h, h->lr, step);
    }
    const int rc = on_device(l);
    if (rc) return rc;
    if (!l->npieces) return SR_OK;
    if (on_host)
        launch_step(l, by_value(l, grads), (const Scalars*)scalars, s, factor, (hipStream_t)stream);
    else
        launch_step(l, GradsAt{grads}, (const Scalars*)scalars, s, factor, (hipStream_t)stream);
    SR_LAUNCH_CHECK();
    return SR_OK;
}

extern "C" int sr_adamw_tick(const sr_adamw_hyper* h, const float* lr, int64_t* step, void* scalars, void* stream) {
    SR_REQUIRE(step && scalars);
    static_assert(sizeof(Scalars) <= SR_ADAMW_SCALARS_BYTES, "size in the header");
    const int rc = check_hyper(h, 1);
    if (rc) return rc;
    adamw_tick_kernel<<<1, 1, 0, (hipStream_t)stream>>>(*h, lr, step, (Scalars*)scalars);
    SR_LAUNCH_CHECK();
    return SR_OK;
}

extern "C" int sr_adamw_moments(const sr_adamw* l, int dtype, void* m, void* v, void* stream) {
    SR_REQUIRE(l && m && v && (dtype == SR_F32 || dtype == SR_BF16));
    const int rc = on_device(l);
    if (rc) return rc;
    if (!l->npieces) return SR_OK;
    const dim3 grid(waves_to_wgs(l->npieces));
    hipStream_t st = (hipStream_t)stream;
#define SR_MOMENTS(T, BITS) adamw_moments_kernel<T, BITS><<<grid, 256, 0, st>>>(l->recs(), l->pieces(), l->npieces, (T*)m, (T*)v)
    if (dtype == SR_F32) {
        if (l->bits == 32)
            SR_MOMENTS(float, 32);
        else
            SR_MOMENTS(float, 8);
    } else {
        if (l->bits == 32)
            SR_MOMENTS(bf16_t, 32);
        else
            SR_MOMENTS(bf16_t, 8);
    }
#undef SR_MOMENTS
    SR_LAUNCH_CHECK();
    return SR_OK;
}

extern "C" int sr_adamw_set_moments(const sr_adamw* l, const float* m, const float* v, uint64_t seed, void* stream) {
    SR_REQUIRE(l && m && v);
    const int rc = on_device(l);
    if (rc) return rc;
    if (!l->npieces) return SR_OK;
    Scalars s = {};
    make_key(seed, 0, s);
    const dim3 grid(waves_to_wgs(l->npieces));
    if (l->bits == 32)
        adamw_set_moments_kernel<32><<<grid, 256, 0, (hipStream_t)stream>>>(l->recs(), l->pieces(), l->npieces, m, v, s);
    else
        adamw_set_moments_kernel<8><<<grid, 256, 0, (hipStream_t)stream>>>(l->recs(), l->pieces(), l->npieces, m, v, s);
    SR_LAUNCH_CHECK();
    return SR_OK;
}

extern "C" size_t sr_grad_norm_workspace_bytes(int nlists) { return nlists > 0 ? (size_t)nlists * NORM_WG * sizeof(double) : 0; }

extern "C" int sr_grad_norm(int nlists, const sr_grad_list* lists, double max_norm, float* out, void* workspace, size_t workspace_bytes,
                            void* stream) {
    SR_REQUIRE(nlists >= 0 && nlists <= SR_GRAD_MAX_LISTS && (lists || !nlists) && out && max_norm >= 0);
    for (int i = 0; i < nlists; ++i) {
        const sr_grad_list& l = lists[i];
        if (l.list) {
            SR_REQUIRE(l.grads && (!l.on_host || l.list->count <= SR_ADAMW_BY_VALUE));
            const int rc = on_device(l.list);
            if (rc) return rc;
        } else {
            SR_REQUIRE((l.dtype == SR_F32 || l.dtype == SR_BF16) && l.nspans >= 0 && l.nspans <= (l.on_host ? SR_GRAD_SPANS_BY_VALUE : 0x7FFFFFFF) &&
                       (l.spans || !l.nspans));
        }
    }
    if (nlists && (!workspace || workspace_bytes < sr_grad_norm_workspace_bytes(nlists))) return SR_ERR_WORKSPACE;
    SR_REQUIRE((uintptr_t)workspace % 8 == 0);
    hipStream_t st = (hipStream_t)stream;
    Partials parts = {};
    parts.lists = nlists;
    for (int i = 0; i < nlists; ++i) {
        const sr_grad_list& l = lists[i];
        const uint32_t items = l.list ? l.list->npieces : (uint32_t)l.nspans;
        if (!items) continue;
        const uint32_t want = waves_to_wgs(items), wgs = want < NORM_WG ? want : NORM_WG;
        parts.n[i] = (int32_t)wgs;
        double* out_i = (double*)workspace + (size_t)i * NORM_WG;
        if (!l.list && l.on_host)
            launch_norm(l.dtype, wgs, SpanSource<SpansByValue>{by_value(l.spans, l.nspans)}, items, out_i, st);
        else if (!l.list)
            launch_norm(l.dtype, wgs, SpanSource<SpansAt>{{l.spans}}, items, out_i, st);
        else if (l.on_host)
            launch_norm(l.list->dtype, wgs, PieceSource<GradsByValue>{l.list->recs(), l.list->pieces(), by_value(l.list, l.grads)}, items, out_i, st);
        else
            launch_norm(l.list->dtype, wgs, PieceSource<GradsAt>{l.list->recs(), l.list->pieces(), {l.grads}}, items, out_i, st);
        SR_LAUNCH_CHECK();
    }
    grad_norm_finish_kernel<<<1, 256, 0, st>>>(parts, (const double*)workspace, max_norm, out);
    SR_LAUNCH_CHECK();
    return SR_OK;
}

extern "C" int sr_grad_scale(int dtype, int64_t nspans, const sr_grad_span* spans, int on_host, const float* factor, void* stream) {
    SR_REQUIRE((dtype == SR_F32 || dtype == SR_BF16) && nspans >= 0 && nspans <= (on_host ? SR_GRAD_SPANS_BY_VALUE : 0x7FFFFFFF));
    SR_REQUIRE((spans || !nspans) && factor);
    if (!nspans) return SR_OK;
    const uint32_t want = waves_to_wgs((uint32_t)nspans), wgs = want < NORM_WG ? want : NORM_WG;
    if (on_host)
        launch_scale(dtype, wgs, by_value(spans, nspans), (uint32_t)nspans, factor, (hipStream_t)stream);
    else
        launch_scale(dtype, wgs, SpansAt{spans}, (uint32_t)nspans, factor, (hipStream_t)stream);
    SR_LAUNCH_CHECK();
    return SR_OK;
}

extern "C" int sr_upload(const void* src_host, void* dst, size_t bytes, void* stream) {
    SR_REQUIRE(bytes % 4 == 0 && (uintptr_t)dst % 4 == 0 && ((src_host && dst) || !bytes));
    for (size_t at = 0; at < bytes; at += UPLOAD) {
        UploadArgs a;
        a.dst = (uint64_t)(uintptr_t)dst + at;
        a.bytes = (int32_t)(bytes - at < UPLOAD ? bytes - at : UPLOAD);
        a.pad = 0;
        memcpy(a.data, (const char*)src_host + at, a.bytes);
        upload_kernel<<<1, 256, 0, (hipStream_t)stream>>>(a);
        SR_LAUNCH_CHECK();
    }
    return SR_OK;
}

extern "C" int sr_upload_pinned(const void* src_pinned, void* dst, size_t bytes, int64_t* done, int64_t ticket, void* stream) {
    SR_REQUIRE(bytes % 4 == 0 && bytes > 0 && bytes <= ((size_t)1 << 30) && src_pinned && dst && done);
    SR_REQUIRE((uintptr_t)dst % 16 == 0 && (uintptr_t)src_pinned % 16 == 0 && (uintptr_t)done % 8 == 0);
    upload_pinned_kernel<<<SR_UPLOAD_WORDS, PINNED_WG, 0, (hipStream_t)stream>>>((const uint32_t*)src_pinned, (uint32_t*)dst, (uint32_t)(bytes / 4), done, ticket);
    SR_LAUNCH_CHECK();
    return SR_OK;
}
