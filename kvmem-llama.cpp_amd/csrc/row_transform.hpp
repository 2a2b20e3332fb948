// Device code shared by the kernels that bring fp32 rows into the cache's form
// (the stage-in transform and the rows of new tokens): ggml's quantizers, the
// rotary angles' sin and cos, the Walsh-Hadamard butterflies, all for lanes
// that hold 8 consecutive elements of a row.  Files that include it are
// compiled without FP contraction: products and sums are separate IEEE
// operations, as in ggml's quantize_row_*_ref.
#pragma once

#include "kvmem_internal.hpp"

#pragma clang fp contract(off)

namespace kvmem_hip {

template <int TYPE> struct Fmt;
template <> struct Fmt<KVMEM_TYPE_Q8_0> { static constexpr int GB = 34; };
template <> struct Fmt<KVMEM_TYPE_Q4_0> { static constexpr int GB = 18; };
template <> struct Fmt<KVMEM_TYPE_Q5_0> { static constexpr int GB = 22; };
template <> struct Fmt<KVMEM_TYPE_F16> { static constexpr int GB = 64; };

// ---------------------------------------------------------------- lanes

// Quad exchange through DPP: lane i of each 4-lane quad reads lane i^1 / i^2.
__device__ inline uint32_t quad_xor1(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true));
}
__device__ inline uint32_t quad_xor2(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, true));
}

__device__ inline float half_bits_to_float(uint32_t h) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
}

__device__ inline uint32_t float_to_half_bits(float f) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));  // v_cvt_f16_f32, RNE
}

__device__ inline void unpack8(const uint4 &v, uint32_t h[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[2 * i] = w[i] & 0xffffu;
        h[2 * i + 1] = w[i] >> 16;
    }
}

__device__ inline void store_u16(uint8_t *p, uint32_t v) {
    *reinterpret_cast<uint16_t *>(p) = static_cast<uint16_t>(v);
}

// Eight bytes packed in two words -> four 2-byte LDS stores (the group
// layouts only guarantee 2-byte alignment).
__device__ inline void store_8bytes(uint8_t *p, uint32_t lo, uint32_t hi) {
    store_u16(p + 0, lo & 0xffffu);
    store_u16(p + 2, lo >> 16);
    store_u16(p + 4, hi & 0xffffu);
    store_u16(p + 6, hi >> 16);
}

// The quantizers' scale arithmetic without the IEEE division sequence.
// scale_div127(a) = a / 127 for every non-negative float a: the product with
// the rounded reciprocal of 127 corrected by one exact residual (two FMAs);
// scale_recip(d) = 1 / d for every normal |d| <= 2^126 (q8_0/q4_0/q5_0 scales
// never exceed 2^125): the hardware reciprocal refined by one Newton step.
// Both equal the correctly rounded quotients over their whole ranges (checked
// exhaustively by kvmem_hip_check_scale_arith on the device).
__device__ inline float scale_div127(float a) {
    constexpr float r127 = 1.0f / 127.0f;
    const float q0 = a * r127;
    return __builtin_fmaf(__builtin_fmaf(-q0, 127.0f, a), r127, q0);
}

__device__ inline float scale_recip(float d) {
    const float r0 = __builtin_amdgcn_rcpf(d);
    return __builtin_fmaf(__builtin_fmaf(-d, r0, 1.0f), r0, r0);
}

// roundf (half away from zero) of |s| < 128.5, the range of q8_0's x*id:
// truncation of s + copysign(0.49999997f, s) (the float below 0.5) equals
// roundf for every float in that range (checked exhaustively over all of
// them), in three instructions instead of roundf's compare-and-fix.
__device__ inline int round_q8(float s) {
    return static_cast<int>(s + copysignf(0x1.fffffep-2f, s));
}

template <int TOP>
__device__ inline uint32_t trunc_code(float x, float id, float bias) {
    const float s = x * id;     // rounded product
    const float t = s + bias;   // rounded sum (separate operation)
    const int c = static_cast<int>(t);
    return static_cast<uint32_t>(c < TOP ? c : TOP);
}

// Bit 4 of each of the 4 bytes of w, as a 4-bit value (byte i -> bit i).
__device__ inline uint32_t bit4_of_bytes(uint32_t w) {
    const uint32_t x = (w >> 4) & 0x01010101u;
    return (x * 0x01020408u) >> 24;  // bits 0, 8, 16, 24 -> 24..27, no carries
}

// ------------------------------------------------- transformed (fp32) rows

// sin and cos of an fp32 angle.  The angle is reduced by pi/2 in double
// (Cody-Waite: k = rint(a * 2/pi), r = a - k*pi/2 with pi/2 split into two
// doubles, one fused multiply-add each), the Taylor series of sin (to r^17)
// and cos (to r^16) are summed by Horner's rule on |r| <= pi/4 (truncation
// below 1e-17), and each result is rounded once to fp32.  Every step is one
// correctly rounded IEEE operation, so a C restatement of the same steps
// reproduces the same bits.  Angles are finite with |a| < 2^40 (a RoPE
// angle is an int32 position times a frequency of at most one).
__device__ inline void rope_sincos(float a, float &sn, float &cs) {
    const double x = static_cast<double>(a);
    const double k = __builtin_rint(x * 0x1.45f306dc9c883p-1);
    double r = x;  // |a| < pi/4: no reduction (keeps the sign of zero)
    if (k != 0.0) {
        r = __builtin_fma(-k, 0x1.921fb54442d18p+0, x);
        r = __builtin_fma(-k, 0x1.1a62633145c07p-54, r);
    }
    const double r2 = r * r;
    double ps = 0x1.952c77030ad4ap-49;
    ps = __builtin_fma(ps, r2, -0x1.ae7f3e733b81fp-41);
    ps = __builtin_fma(ps, r2, 0x1.6124613a86d09p-33);
    ps = __builtin_fma(ps, r2, -0x1.ae64567f544e4p-26);
    ps = __builtin_fma(ps, r2, 0x1.71de3a556c734p-19);
    ps = __builtin_fma(ps, r2, -0x1.a01a01a01a01ap-13);
    ps = __builtin_fma(ps, r2, 0x1.1111111111111p-7);
    ps = __builtin_fma(ps, r2, -0x1.5555555555555p-3);
    double pc = 0x1.ae7f3e733b81fp-45;
    pc = __builtin_fma(pc, r2, -0x1.93974a8c07c9dp-37);
    pc = __builtin_fma(pc, r2, 0x1.1eed8eff8d898p-29);
    pc = __builtin_fma(pc, r2, -0x1.27e4fb7789f5cp-22);
    pc = __builtin_fma(pc, r2, 0x1.a01a01a01a01ap-16);
    pc = __builtin_fma(pc, r2, -0x1.6c16c16c16c17p-10);
    pc = __builtin_fma(pc, r2, 0x1.5555555555555p-5);
    pc = __builtin_fma(pc, r2, -0.5);
    const double sr = r == 0.0 ? r : __builtin_fma(r * r2, ps, r);  // sin(+-0) = +-0
    const double cr = __builtin_fma(r2, pc, 1.0);
    const int quadrant = static_cast<int>(k - 4.0 * __builtin_floor(k * 0.25));  // k mod 4, exact
    const double sv = (quadrant & 1) ? cr : sr;
    const double cv = (quadrant & 1) ? sr : cr;
    sn = static_cast<float>((quadrant & 2) ? -sv : sv);
    cs = static_cast<float>(((quadrant + 1) & 2) ? -cv : cv);
}

// One butterfly stage of span 8*M across lanes: the lane whose bit M is set
// holds the upper element and keeps partner - own, the other own + partner
// (p + (-x) is the IEEE subtraction p - x).
template <uint32_t M>
__device__ inline void butterfly_lanes(float x[8], uint32_t lane) {
    const uint32_t flip = (lane & M) ? 0x80000000u : 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float p = lane_xor<M>(x[i]);
        x[i] = p + __uint_as_float(__float_as_uint(x[i]) ^ flip);
    }
}

// Walsh-Hadamard rotation of runs of `width` elements, in the order of the
// reference's fwht_kernel: scale every element, then butterflies of span
// 1, 2, 4 (inside the lane) and 8 .. width/2 (partner lane ^ span/8).
__device__ inline void fwht_lanes(float x[8], uint32_t width, float scale, uint32_t lane) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = x[i] * scale;
    }
#pragma unroll
    for (int h = 1; h < 8; h <<= 1) {
#pragma unroll
        for (int i = 0; i < 8; i += 2 * h) {
#pragma unroll
            for (int j = 0; j < h; ++j) {
                const float a = x[i + j];
                const float b = x[i + j + h];
                x[i + j] = a + b;
                x[i + j + h] = a - b;
            }
        }
    }
    // width is uniform: whole stages are skipped together
    butterfly_lanes<1>(x, lane);
    butterfly_lanes<2>(x, lane);
    butterfly_lanes<4>(x, lane);
    if (width > 64u) {
        butterfly_lanes<8>(x, lane);
    }
    if (width > 128u) {
        butterfly_lanes<16>(x, lane);
    }
    if (width > 256u) {
        butterfly_lanes<32>(x, lane);
    }
}

// Partner values of a RoPE pair: lane ^ (n_rot/16) when that is a power of
// two (a head's first-half lanes then differ from their partners in exactly
// that bit), else lane +- n_rot/16 through a general lane permute.
__device__ inline void rope_partners(const float x[8], float p[8], uint32_t n_rot, uint32_t lane,
                                     bool rot, bool first) {
    const uint32_t d = n_rot / 16u;
#define KVMEM_XOR_CASE(M)                     \
    case M:                                   \
        for (int i = 0; i < 8; ++i) {         \
            p[i] = lane_xor<M>(x[i]);         \
        }                                     \
        return;
    switch (d) {
        KVMEM_XOR_CASE(1)
        KVMEM_XOR_CASE(2)
        KVMEM_XOR_CASE(4)
        KVMEM_XOR_CASE(8)
        KVMEM_XOR_CASE(16)
        KVMEM_XOR_CASE(32)
        default: break;
    }
#undef KVMEM_XOR_CASE
    const int src = static_cast<int>(rot ? (first ? lane + d : lane - d) : lane);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        p[i] = __shfl(x[i], src, 64);
    }
}

// vmax of ggml's q4_0/q5_0 over fp32 values: the first element of largest
// magnitude (NaNs never win, as in the reference's strict `amax < |v|`);
// an all-zero group keeps the initial vmax = +0.
__device__ inline float quad_vmax_f(const float x[8], uint32_t q) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        amax = fmaxf(amax, fabsf(x[i]));
    }
    amax = fmaxf(amax, __uint_as_float(quad_xor1(__float_as_uint(amax))));
    amax = fmaxf(amax, __uint_as_float(quad_xor2(__float_as_uint(amax))));
    uint32_t key = 0xffffffffu;  // (element << 1) | sign of the first maximum
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        if (fabsf(x[i]) == amax) {
            key = ((8u * q + i) << 1) | (__float_as_uint(x[i]) >> 31);
        }
    }
    uint32_t o = quad_xor1(key);
    key = o < key ? o : key;
    o = quad_xor2(key);
    key = o < key ? o : key;
    return amax == 0.0f ? 0.0f : ((key & 1u) ? -amax : amax);
}

template <int TYPE>
__device__ inline void quant_quarter_f(const float x[8], uint32_t q, uint8_t *g, bool valid);

template <>
__device__ inline void quant_quarter_f<KVMEM_TYPE_Q8_0>(const float x[8], uint32_t q, uint8_t *g,
                                                         bool valid) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        amax = fmaxf(amax, fabsf(x[i]));
    }
    amax = fmaxf(amax, __uint_as_float(quad_xor1(__float_as_uint(amax))));
    amax = fmaxf(amax, __uint_as_float(quad_xor2(__float_as_uint(amax))));
    const float d = scale_div127(amax);
    const float id = d != 0.0f ? scale_recip(d) : 0.0f;
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = round_q8(x[i] * id);
        w[i >> 2] |= (static_cast<uint32_t>(c) & 0xffu) << (8 * (i & 3));
    }
    if (valid) {
        if (q == 0) {
            store_u16(g, float_to_half_bits(d));
        }
        store_8bytes(g + 2 + 8 * q, w[0], w[1]);
    }
}

template <int TOP>
__device__ inline void trunc_codes_f(const float x[8], float id, float bias, uint32_t &w0,
                                     uint32_t &w1) {
    w0 = 0u;
    w1 = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w0 |= trunc_code<TOP>(x[i], id, bias) << (8 * i);
        w1 |= trunc_code<TOP>(x[i + 4], id, bias) << (8 * i);
    }
}

template <>
__device__ inline void quant_quarter_f<KVMEM_TYPE_Q4_0>(const float x[8], uint32_t q, uint8_t *g,
                                                         bool valid) {
    const float vmax = quad_vmax_f(x, q);
    const float d = vmax * -0.125f;        // == vmax / -8 (exact scaling)
    const float id = d != 0.0f ? scale_recip(d) : 0.0f;
    uint32_t w0, w1;
    trunc_codes_f<15>(x, id, 8.5f, w0, w1);
    const uint32_t p0 = quad_xor2(w0);
    const uint32_t p1 = quad_xor2(w1);
    if (valid) {
        if (q == 0) {
            store_u16(g, float_to_half_bits(d));
        }
        if (q < 2) {
            store_8bytes(g + 2 + 8 * q, w0 | (p0 << 4), w1 | (p1 << 4));
        }
    }
}

template <>
__device__ inline void quant_quarter_f<KVMEM_TYPE_Q5_0>(const float x[8], uint32_t q, uint8_t *g,
                                                         bool valid) {
    const float vmax = quad_vmax_f(x, q);
    const float d = vmax * -0.0625f;       // == vmax / -16 (exact scaling)
    const float id = d != 0.0f ? scale_recip(d) : 0.0f;
    uint32_t w0, w1;
    trunc_codes_f<31>(x, id, 16.5f, w0, w1);
    uint32_t qh = (bit4_of_bytes(w0) | (bit4_of_bytes(w1) << 4)) << (8 * q);
    qh |= quad_xor1(qh);
    qh |= quad_xor2(qh);
    w0 &= 0x0f0f0f0fu;
    w1 &= 0x0f0f0f0fu;
    const uint32_t p0 = quad_xor2(w0);
    const uint32_t p1 = quad_xor2(w1);
    if (valid) {
        if (q == 0) {
            store_u16(g, float_to_half_bits(d));
            store_u16(g + 2, qh & 0xffffu);
            store_u16(g + 4, qh >> 16);
        }
        if (q < 2) {
            store_8bytes(g + 6 + 8 * q, w0 | (p0 << 4), w1 | (p1 << 4));
        }
    }
}

template <>
__device__ inline void quant_quarter_f<KVMEM_TYPE_F16>(const float x[8], uint32_t q, uint8_t *g,
                                                        bool valid) {
    if (valid) {
        uint4 v;
        v.x = float_to_half_bits(x[0]) | (float_to_half_bits(x[1]) << 16);
        v.y = float_to_half_bits(x[2]) | (float_to_half_bits(x[3]) << 16);
        v.z = float_to_half_bits(x[4]) | (float_to_half_bits(x[5]) << 16);
        v.w = float_to_half_bits(x[6]) | (float_to_half_bits(x[7]) << 16);
        *reinterpret_cast<uint4 *>(g + 16 * q) = v;
    }
}

}  // namespace kvmem_hip
