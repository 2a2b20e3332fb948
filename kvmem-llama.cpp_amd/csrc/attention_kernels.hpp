// Kernels of kvmem_hip_attention (attention.hip); one translation unit per key
// type instantiates them.
#pragma once

#include "attention.hpp"

#include <algorithm>
#include <cmath>

namespace kvmem_hip {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// ------------------------------------------------------- cached formats

// A head's slice of a row, moved in units of D/16 bytes (16 for f16): its
// address is a multiple of that.
template <int TYPE, int D>
struct Slice {
    static constexpr uint32_t GB = TYPE == KVMEM_TYPE_Q8_0 ? 34 : TYPE == KVMEM_TYPE_Q5_0 ? 22
                                   : TYPE == KVMEM_TYPE_Q4_0 ? 18 : 64;
    static constexpr uint32_t bytes = D / 32 * GB;
    static constexpr uint32_t unit = TYPE == KVMEM_TYPE_F16 ? 16 : D / 16;
    static constexpr uint32_t units = bytes / unit;
    // LDS bytes between keys: f16 rows are padded so that 16 keys' reads
    // spread over the banks
    static constexpr uint32_t stride = TYPE == KVMEM_TYPE_F16 ? bytes + 16 : bytes;
    // a wave's load moves whole slices, one lane a unit (the last lanes idle):
    // the addresses of its loads then differ by constants
    static constexpr uint32_t per_load = 64 / units;
};

template <uint32_t UNIT> struct UnitOf;
template <> struct UnitOf<4> { typedef uint32_t type; };
template <> struct UnitOf<8> { typedef u32x2_t type; };
template <> struct UnitOf<16> { typedef u32x4_t type; };

__device__ inline uint32_t lds_half(const uint8_t *p) { return *reinterpret_cast<const uint16_t *>(p); }

// N words of LDS from an even address.  Groups of 18, 22 and 34 bytes put every
// other group's codes 2 bytes off a word; the LDS answers such reads at a
// fraction of its rate (stalls were three quarters of a step's time), so words are
// read where they are aligned and shifted together.  The word after the last is
// read too.
template <int N>
__device__ inline void lds_words(const uint8_t *p, uint32_t shift, uint32_t out[N]) {
    const uint32_t *q = reinterpret_cast<const uint32_t *>(p - shift);
    uint32_t w[N + 1];
#pragma unroll
    for (int i = 0; i <= N; ++i) {
        w[i] = q[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        out[i] = __builtin_amdgcn_alignbyte(w[i + 1], w[i], shift);
    }
}
// The same where the address is known to be a word's.
struct Aligned {};
template <int N>
__device__ inline void lds_words(const uint8_t *p, Aligned, uint32_t out[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        out[i] = reinterpret_cast<const uint32_t *>(p)[i];
    }
}

// Key operand of one group of 32 dims: the 8 elements a lane (key, chunk c of
// 4) feeds the matrix instruction, as f16.  Quantized codes stay integers:
// an f16 whose bits are the code n is the subnormal n * 2^-24, which the
// matrix cores multiply exactly, so a masked word is an operand already.
// A code in the upper nibble is 16 times its value there; the query element
// that meets it is divided by 16.  The code's offset (8, 16, 128) comes off
// through the accumulator's start, the group's scale is multiplied into the
// fp32 sum: keys enter the scores unrounded.
// shift: the bytes that the group's codes lie off a word (2 in groups of even
// number, Aligned where that is known).
// Element e is dim piece(c, i) + l % 4 of the group, l = order(e) and i = l / 4:
// a lane's 8 dims are two runs of four.
template <int TYPE> struct KeyOp;

template <> struct KeyOp<KVMEM_TYPE_Q4_0> {
    static constexpr float offset = 8.0f;
    static constexpr bool codes = true;
    template <class Shift>
    __device__ static inline u32x4_t load(const uint8_t *g, uint32_t c, Shift shift) {
        uint32_t w;
        lds_words<1>(g + 2 + 4 * c, shift, &w);
        u32x4_t r;
        r[0] = w & 0x000F000Fu;
        r[1] = w & 0x00F000F0u;
        r[2] = (w >> 8) & 0x000F000Fu;
        r[3] = (w >> 8) & 0x00F000F0u;
        return r;
    }
    __device__ static inline uint32_t piece(uint32_t c, uint32_t i) { return 4 * c + 16 * i; }
    __device__ static constexpr uint32_t order(uint32_t e) { return 2 * (e & 2u) + 2 * (e & 1u) + (e >> 2); }
    // the operand's element is this many times the code
    __device__ static constexpr float times(uint32_t e) { return (e & 2u) ? 16.0f : 1.0f; }
};

template <> struct KeyOp<KVMEM_TYPE_Q5_0> {
    static constexpr float offset = 16.0f;
    static constexpr bool codes = true;
    template <class Shift>
    __device__ static inline u32x4_t load(const uint8_t *g, uint32_t c, Shift shift) {
        uint32_t h, w;
        lds_words<1>(g + 2, shift, &h);
        lds_words<1>(g + 6 + 4 * c, shift, &w);
        h >>= 4 * c;
        // bits 0 and 2 of a 4-bit field to bits 4 and 20 (8 and 24 for the
        // upper nibbles): two shifted copies in one product, no carries
        const uint32_t lo = (h & 15u) * 0x00040010u;
        const uint32_t hi = ((h >> 16) & 15u) * 0x00400100u;
        u32x4_t r;
        r[0] = (w & 0x000F000Fu) | (lo & 0x00100010u);
        r[1] = (w & 0x00F000F0u) | (hi & 0x01000100u);
        r[2] = ((w >> 8) & 0x000F000Fu) | ((lo >> 1) & 0x00100010u);
        r[3] = ((w >> 8) & 0x00F000F0u) | ((hi >> 1) & 0x01000100u);
        return r;
    }
    __device__ static inline uint32_t piece(uint32_t c, uint32_t i) { return 4 * c + 16 * i; }
    __device__ static constexpr uint32_t order(uint32_t e) { return 2 * (e & 2u) + 2 * (e & 1u) + (e >> 2); }
    __device__ static constexpr float times(uint32_t e) { return (e & 2u) ? 16.0f : 1.0f; }
};

template <> struct KeyOp<KVMEM_TYPE_Q8_0> {
    static constexpr float offset = 128.0f;
    static constexpr bool codes = true;
    template <class Shift>
    __device__ static inline u32x4_t load(const uint8_t *g, uint32_t c, Shift shift) {
        uint32_t w[2];
        lds_words<2>(g + 2 + 8 * c, shift, w);
        const uint32_t a = w[0] ^ 0x80808080u;
        const uint32_t b = w[1] ^ 0x80808080u;
        u32x4_t r;
        r[0] = a & 0x00FF00FFu;
        r[1] = (a >> 8) & 0x00FF00FFu;
        r[2] = b & 0x00FF00FFu;
        r[3] = (b >> 8) & 0x00FF00FFu;
        return r;
    }
    __device__ static inline uint32_t piece(uint32_t c, uint32_t i) { return 8 * c + 4 * i; }
    __device__ static constexpr uint32_t order(uint32_t e) { return (e & 4u) + 2 * (e & 1u) + ((e >> 1) & 1u); }
    __device__ static constexpr float times(uint32_t) { return 1.0f; }
};

template <> struct KeyOp<KVMEM_TYPE_F16> {
    static constexpr float offset = 0.0f;
    static constexpr bool codes = false;
    template <class Shift>
    __device__ static inline u32x4_t load(const uint8_t *g, uint32_t c, Shift) {
        return *reinterpret_cast<const u32x4_t *>(g + 16 * c);
    }
    __device__ static inline uint32_t piece(uint32_t c, uint32_t i) { return 8 * c + 4 * i; }
    __device__ static constexpr uint32_t order(uint32_t e) { return e; }
    __device__ static constexpr float times(uint32_t) { return 1.0f; }
};

__device__ inline half2_t as_half2(uint32_t w) { return __builtin_bit_cast(half2_t, w); }
__device__ inline uint32_t as_word(half2_t h) { return __builtin_bit_cast(uint32_t, h); }

// (low halves, high halves) of a key pair's words: a in the lower 16 bits.
__device__ inline uint32_t pair_lo(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ inline uint32_t pair_hi(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// The same value, of which the compiler knows nothing: what is derived from it is
// computed anew where it is used instead of being kept in registers.
__device__ inline uint32_t anew(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// The bits of 1024 and of 64 in both halves of a word.
struct Magic {
    uint32_t low, high;
};
// Constants; in registers (decode, which has some to spare) a mask and these
// are one instruction: nothing but one scalar register fits in it otherwise.
constexpr Magic kMagic{0x64006400u, 0x54005400u};

// f16 values of a pair of codes in bits 0..9 of each half: 1024 + n by the
// bits of 1024, less 1024 + offset (both exact), times the scales (the one
// rounding).
__device__ inline uint32_t pair_value(uint32_t codes, uint32_t magic, float offset, uint32_t scales) {
    const _Float16 o = static_cast<_Float16>(-(1024.0f + offset));
    return as_word((as_half2(codes | magic) + half2_t{o, o}) * as_half2(scales));
}
// The same for codes in bits 4..9: 64 + n by the bits of 64.
__device__ inline uint32_t pair_value_hi(uint32_t codes, uint32_t magic, float offset, uint32_t scales) {
    const _Float16 o = static_cast<_Float16>(-(64.0f + offset));
    return as_word((as_half2(codes | magic) + half2_t{o, o}) * as_half2(scales));
}

// Value operand: lane n owns VD dims of a key's slice.  Rows
// hold consecutive dims of one key and the matrix instruction wants
// consecutive keys of one dim, so a lane reads its dims of 8 keys and pairs
// keys with byte permutes, still in packed codes (a nibble permute moves 8
// elements).  raw(): the keys' words and scales; emit(keep, f): f(t,
// operands of dims t .. t + 3) over the VD dims, keys cleared in `keep` (16 bits a
// key, pairs as the operand's words) as zeros;  dim(n, t): which dim t is.
template <int TYPE, int VD> struct ValueOp;

template <int VD>
struct ValueOp<KVMEM_TYPE_Q4_0, VD> {
    // dims nth(t) .. nth(t + RUN - 1), t a multiple of RUN, are neighbours: the lower
    // nibbles' first, then the upper ones'
    static constexpr int RUN = VD / 2 < 4 ? VD / 2 : 4;
    static constexpr int nth(int t) { return t < VD / 2 ? 2 * t : 2 * (t - VD / 2) + 1; }
    static constexpr int NB = VD / 2;  // bytes of codes
    static constexpr int NW = NB < 4 ? 1 : NB / 4;
    static constexpr float offset = 8.0f;
    uint32_t w[8][NW];
    uint32_t d[4];
    __device__ static inline uint32_t dim(uint32_t n, uint32_t t) {
        constexpr uint32_t per = 32 / VD;  // lanes of a group
        return 32 * (n / per) + NB * (n % per) + (t >> 1) + 16 * (t & 1u);
    }
    template <class RowOf>
    __device__ inline void raw(uint32_t n, RowOf row) {
        constexpr uint32_t per = 32 / VD;
        const uint32_t off = 2u * (~(n / per) & 1u);  // of the lane's group's codes in a word
        uint32_t s[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const uint8_t *g = row(e) + (n / per) * 18u;
            s[e] = lds_half(g);
            const uint8_t *b = g + 2 + NB * (n % per);
            if constexpr (NB >= 4) {
                lds_words<NW>(b, off, w[e]);
            } else {
                w[e][0] = lds_half(b);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            d[i] = s[2 * i] | (s[2 * i + 1] << 16);
        }
    }
    template <class F>
    __device__ inline void emit(const u32x4_t &keep, const Magic &magic, F f) const {
        const u32x4_t ds{d[0] & keep[0], d[1] & keep[1], d[2] & keep[2], d[3] & keep[3]};
#pragma unroll
        for (int i = 0; i < NW; ++i) {
#pragma unroll
            for (int h = 0; h < (NB < 4 ? 1 : 2); ++h) {
                u32x4_t a[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t t = h ? pair_hi(w[2 * j][i], w[2 * j + 1][i]) : pair_lo(w[2 * j][i], w[2 * j + 1][i]);
                    a[0][j] = pair_value(t & 0x000F000Fu, magic.low, offset, ds[j]);
                    a[1][j] = pair_value_hi(t & 0x00F000F0u, magic.high, offset, ds[j]);
                    a[2][j] = pair_value((t >> 8) & 0x000F000Fu, magic.low, offset, ds[j]);
                    a[3][j] = pair_value_hi((t >> 8) & 0x00F000F0u, magic.high, offset, ds[j]);
                }
                f(8 * i + 4 * h, a);
            }
        }
    }
};

template <int VD>
struct ValueOp<KVMEM_TYPE_Q5_0, VD> {
    // dims nth(t) .. nth(t + RUN - 1), t a multiple of RUN, are neighbours: the lower
    // nibbles' first, then the upper ones'
    static constexpr int RUN = VD / 2 < 4 ? VD / 2 : 4;
    static constexpr int nth(int t) { return t < VD / 2 ? 2 * t : 2 * (t - VD / 2) + 1; }
    static constexpr int NB = VD / 2;
    static constexpr int NW = NB < 4 ? 1 : NB / 4;
    static constexpr float offset = 16.0f;
    uint32_t w[8][NW];  // lower four bits, as Q4_0's
    uint32_t h[8];      // fifth bits: of the lower nibbles from bit 0, of the upper from bit 16
    uint32_t d[4];
    __device__ static inline uint32_t dim(uint32_t n, uint32_t t) { return ValueOp<KVMEM_TYPE_Q4_0, VD>::dim(n, t); }
    template <class RowOf>
    __device__ inline void raw(uint32_t n, RowOf row) {
        constexpr uint32_t per = 32 / VD;
        const uint32_t off = 2u * (~(n / per) & 1u);  // of the lane's group's codes in a word
        uint32_t s[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const uint8_t *g = row(e) + (n / per) * 22u;
            s[e] = lds_half(g);
            lds_words<1>(g + 2, off, &h[e]);
            h[e] >>= NB * (n % per);
            const uint8_t *b = g + 6 + NB * (n % per);
            if constexpr (NB >= 4) {
                lds_words<NW>(b, off, w[e]);
            } else {
                w[e][0] = lds_half(b);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            d[i] = s[2 * i] | (s[2 * i + 1] << 16);
        }
    }
    template <class F>
    __device__ inline void emit(const u32x4_t &keep, const Magic &magic, F f) const {
        const u32x4_t ds{d[0] & keep[0], d[1] & keep[1], d[2] & keep[2], d[3] & keep[3]};
        // the fifth bits of a key pair, in the halves of one word
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            lo[j] = pair_lo(h[2 * j], h[2 * j + 1]);
            hi[j] = pair_hi(h[2 * j], h[2 * j + 1]);
        }
#pragma unroll
        for (int i = 0; i < NW; ++i) {
#pragma unroll
            for (int q = 0; q < (NB < 4 ? 1 : 2); ++q) {
                u32x4_t a[4];
                const int b0 = 4 * i + 2 * q;  // byte of the lane's codes
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t t = q ? pair_hi(w[2 * j][i], w[2 * j + 1][i]) : pair_lo(w[2 * j][i], w[2 * j + 1][i]);
                    a[0][j] = pair_value((t & 0x000F000Fu) | (((lo[j] >> b0) & 0x00010001u) << 4), magic.low, offset, ds[j]);
                    a[1][j] = pair_value_hi((t & 0x00F000F0u) | (((hi[j] >> b0) & 0x00010001u) << 8), magic.high, offset, ds[j]);
                    a[2][j] = pair_value(((t >> 8) & 0x000F000Fu) | (((lo[j] >> (b0 + 1)) & 0x00010001u) << 4), magic.low, offset,
                                      ds[j]);
                    a[3][j] = pair_value_hi(((t >> 8) & 0x00F000F0u) | (((hi[j] >> (b0 + 1)) & 0x00010001u) << 8), magic.high, offset,
                                         ds[j]);
                }
                f(8 * i + 4 * q, a);
            }
        }
    }
};

template <int VD>
struct ValueOp<KVMEM_TYPE_Q8_0, VD> {
    static constexpr int RUN = 4;
    static constexpr int nth(int t) { return t; }
    static constexpr int NW = VD / 4;
    uint32_t w[8][NW];
    uint32_t d[4];
    __device__ static inline uint32_t dim(uint32_t n, uint32_t t) { return VD * n + t; }
    template <class RowOf>
    __device__ inline void raw(uint32_t n, RowOf row) {
        constexpr uint32_t per = 32 / VD;
        const uint32_t off = 2u * (~(n / per) & 1u);  // of the lane's group's codes in a word
        uint32_t s[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const uint8_t *g = row(e) + (n / per) * 34u;
            s[e] = lds_half(g);
            lds_words<NW>(g + 2 + VD * (n % per), off, w[e]);
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                w[e][i] ^= 0x80808080u;
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            d[i] = s[2 * i] | (s[2 * i + 1] << 16);
        }
    }
    template <class F>
    __device__ inline void emit(const u32x4_t &keep, const Magic &magic, F f) const {
        const u32x4_t ds{d[0] & keep[0], d[1] & keep[1], d[2] & keep[2], d[3] & keep[3]};
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            u32x4_t a[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                // byte b of both keys, zero-extended to 16 bits
                const uint32_t sel = 0x0c000c00u | static_cast<uint32_t>(b) | (static_cast<uint32_t>(4 + b) << 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    a[b][j] = pair_value(__builtin_amdgcn_perm(w[2 * j + 1][i], w[2 * j][i], sel), magic.low, 128.0f, ds[j]);
                }
            }
            f(4 * i, a);
        }
    }
};

template <int VD>
struct ValueOp<KVMEM_TYPE_F16, VD> {
    static constexpr int RUN = 4;
    static constexpr int nth(int t) { return t; }
    static constexpr int NW = VD / 2;
    uint32_t w[8][NW];
    __device__ static inline uint32_t dim(uint32_t n, uint32_t t) { return VD * n + t; }
    template <class RowOf>
    __device__ inline void raw(uint32_t n, RowOf row) {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const uint8_t *b = row(e) + 2u * VD * n;
            if constexpr (NW == 2) {
                const u32x2_t x = *reinterpret_cast<const u32x2_t *>(b);
                w[e][0] = x[0];
                w[e][1] = x[1];
            } else {
#pragma unroll
                for (int i = 0; i < NW; i += 4) {
                    const u32x4_t x = *reinterpret_cast<const u32x4_t *>(b + 4 * i);
                    w[e][i] = x[0];
                    w[e][i + 1] = x[1];
                    w[e][i + 2] = x[2];
                    w[e][i + 3] = x[3];
                }
            }
        }
    }
    template <class F>
    __device__ inline void emit(const u32x4_t &keep, const Magic &magic, F f) const {
#pragma unroll
        for (int i = 0; i < NW; i += 2) {
            u32x4_t a[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a[0][j] = pair_lo(w[2 * j][i], w[2 * j + 1][i]) & keep[j];
                a[1][j] = pair_hi(w[2 * j][i], w[2 * j + 1][i]) & keep[j];
                a[2][j] = pair_lo(w[2 * j][i + 1], w[2 * j + 1][i + 1]) & keep[j];
                a[3][j] = pair_hi(w[2 * j][i + 1], w[2 * j + 1][i + 1]) & keep[j];
            }
            f(2 * i, a);
        }
    }
};

// ------------------------------------------------------------ wave helpers

// The value of lane ^ 16 (lanes swapped between row pairs) and lane ^ 32.
__device__ inline float lane_xor16(float v) {
    return __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), 0x1F | (16 << 10)));
}
__device__ inline float lane_xor32(float v) { return __shfl_xor(v, 32, 64); }

__device__ inline float lane_xor8(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xF, 0xF, true));  // row_ror:8
}

// Of a block of 32 keys, those that exist and lie below `limit` (both from the
// block's first key), for a lane whose element e of the block's operand is key
// GAP (e / 4) + first + e % 4: bit GAP (e / 4) + e % 4.
__device__ inline uint32_t seen_keys(uint32_t have, int32_t limit, uint32_t first) {
    const int32_t left = limit - static_cast<int32_t>(first);
    const uint32_t below = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u;
    return (have >> first) & below;
}

// Operand masks of those keys: 16 bits a key, pairs as the operand's words.
template <uint32_t GAP>
__device__ inline u32x4_t keep_keys(uint32_t seen) {
    u32x4_t keep;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t two = seen >> (GAP * (j >> 1) + 2u * (j & 1u));
        keep[j] = (two & 1u) * 0x0000ffffu + ((two >> 1) & 1u) * 0xffff0000u;
    }
    return keep;
}

// Values that are not finite, where some rows of a workgroup do not attend their
// key: a weight of zero would still hand those rows the NaN.  Such a value enters
// the product as zero, its key is noted for its dim (first[dim], the lowest such
// key), and rows that attend that key get NaN for the dim at the end.  `a`: the
// operand of one dim for 8 keys, element e key at(e).
template <class At>
__device__ inline void clear_odd(u32x4_t &a, uint32_t *first, At at) {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        const bool lo = (a[j] & 0x7C00u) == 0x7C00u;
        const bool hi = (a[j] & 0x7C000000u) == 0x7C000000u;
        if (lo) {
            atomicMin(first, at(2 * j));
        }
        if (hi) {
            atomicMin(first, at(2 * j + 1));
        }
        a[j] &= (lo ? 0u : 0x0000ffffu) | (hi ? 0u : 0xffff0000u);
    }
}

// A wave's LDS writes become visible to its own later reads, in order.
__device__ inline void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A lane's 8 query elements of a group as they lie in memory (f16 or bf16 bits).
template <class KO>
__device__ inline u32x4_t load_query(const uint8_t *q, uint32_t g, uint32_t c) {
    const u32x2_t a = *reinterpret_cast<const u32x2_t *>(q + 64u * g + 2u * KO::piece(c, 0));
    const u32x2_t b = *reinterpret_cast<const u32x2_t *>(q + 64u * g + 2u * KO::piece(c, 1));
    return u32x4_t{a[0], a[1], b[0], b[1]};
}

// The larger magnitudes of two pairs (bits: both formats order as integers).
__device__ inline uint32_t max_magnitude(uint32_t a, uint32_t b) {
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a & 0x7fff7fffu),
                                                                  __builtin_bit_cast(u16x2_t, b)));
}

template <bool BF16>
__device__ inline float query_value(uint32_t bits) {
    return BF16 ? __uint_as_float(bits << 16)
                : static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
}

// f16 queries in the key operand's order, times `up`.
template <class KO, bool BF16>
__device__ inline half8_t query_operand(const u32x4_t &w, float up) {
    half8_t r;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
        const uint32_t l = KO::order(e);
        r[e] = static_cast<_Float16>(query_value<BF16>((l & 1u) ? w[l >> 1] >> 16 : w[l >> 1] & 0xffffu) * up);
    }
    return r;
}

// Exponent of the power of two that brings a row's largest query magnitude to
// at most 2^9: f16 then holds the row whatever its exponents.
__device__ inline int query_shift(float top) {
    int ex = 0;
    if (top > 0.0f && top < INFINITY) {
        (void) frexpf(top, &ex);
        ex = min(9 - ex, 120);  // the power itself stays a normal float
    }
    return ex;
}

// Scores (log2 units) up to which a fused product less the rounded maximum is as good
// as the rounded product less the maximum: the rounding is at most 2^-4 there, which a
// row's weights and their sum have in common.
constexpr float kFarScore = 0x1p20f;
__device__ inline bool is_far(float top) { return fabsf(top) > kFarScore && top != -INFINITY; }

// What brings the operands' products back to scores in log2 units: scale * log2(e) *
// 2^e, which may pass fp32 (queries from 2^112 on, large scales) although the scores
// do not.  Where a row's does, `more`, a power of two, is split off for all rows of
// the wave, and 1 nearly always: x * fac * more then passes fp32 only where the score
// does (a product is 0 or at least 2^-72, so what `more` cannot hold would be
// infinite anyway).
struct ScoreFactor {
    float fac, more;
};
__device__ inline ScoreFactor score_factor(float scale, int e) {
    int ex = 0;
    const float m = frexpf(scale, &ex) * kLog2e;
    ex += e;
    int k = 0;
    if (__any(ex > 126)) {
        float most = static_cast<float>(ex);
        most = fmaxf(most, lane_xor<1>(most));
        most = fmaxf(most, lane_xor<2>(most));
        most = fmaxf(most, lane_xor<4>(most));
        most = fmaxf(most, lane_xor<8>(most));
        most = fmaxf(most, lane_xor<16>(most));
        most = fmaxf(most, lane_xor<32>(most));
        k = min(__builtin_amdgcn_readfirstlane(static_cast<int>(most)) - 126, 127);
    }
    // (2^k from its bits: in a scalar register, as k is)
    return {ldexpf(m, min(ex - k, 126)),
            __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(127 + k)) << 23)};
}

// ------------------------------------------------------------ few queries

template <int TK, int TV, int D>
constexpr uint32_t decode_wave_bytes() {
    return step_keys(D) * (Slice<TK, D>::stride + Slice<TV, D>::stride + (KeyOp<TK>::codes ? D / 16 : 0));
}

// Rows of one KV head's queries over one part of a request's keys: up to 16
// (token, head) rows, keys split over the workgroup's four waves.  Scores are
// held transposed (keys by rows) so that a lane owns one query row: S^T = K Q^T,
// O^T = V^T P^T, and a lane's weights of S^T are its operand of the second
// product as they stand.  With up to 8 rows the other 8 columns of the second
// product take what the weights lost to f16.
//
// Bound for few keys by the way to them (lengths, table, rows, then the joining:
// 9 us for a single key, 14 us for 2011), for many by vector instructions, mostly
// values made f16, and the waits between them: q4_0, 24/4 heads of 256, 32768 keys
// 22 us (vector instructions 33 % busy), 131072 47 us = 3.2 TB/s; f16 105 us = 5.1
// TB/s; q8_0 76 us = 3.8 TB/s.  32 ragged requests up to 16384 keys, 32/8 heads of
// 128, q4_0: 123 us = 2.5 TB/s, vector instructions 57 % busy where a compute unit is
// (they are for 72 % of the time: requests are cut by the longest one's keys).
// Above 8 rows a weight is f16 alone, 2^-11 of itself: a second product for the
// digits it lost would take as long as the first, and the values beside it are
// rounded as much.
template <int TK, int TV, int D>
__global__ __launch_bounds__(256, decode_waves(TK, TV, D)) void attn_decode_kernel(AttnParams p) {
    using SK = Slice<TK, D>;
    using SV = Slice<TV, D>;
    using KO = KeyOp<TK>;
    constexpr int NG = D / 32;
    constexpr int VD = D / 16;
    using VO = ValueOp<TV, VD>;
    constexpr uint32_t KT = step_keys(D);
    constexpr int NT = KT / 16;  // key tiles of a step
    constexpr uint32_t NC = KT > 64 ? KT / 64 : 1;  // keys a lane finds the cells of
    constexpr uint32_t NLK = (KT + SK::per_load - 1) / SK::per_load;  // loads of a step
    constexpr uint32_t NLV = (KT + SV::per_load - 1) / SV::per_load;
    typedef typename UnitOf<SK::unit>::type UK;
    typedef typename UnitOf<SV::unit>::type UV;
    typedef uint16_t scales_t __attribute__((ext_vector_type(NG)));
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float2 wave_ml[kWaves][kRowTile];
    __shared__ uint32_t first_odd[D];

    const uint32_t unit = blockIdx.x % p.units;
    const uint32_t y = blockIdx.x / p.units;
    // part by part, each starting one request further: a request's parts, and the
    // parts that only long requests have, fall on all XCDs
    const uint32_t part = unit / p.n_seq;
    const uint32_t s = (unit + part) % p.n_seq;
    if (part >= p.n_parts) {
        return;
    }
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t c0 = part * p.chunk;
    const uint32_t *table = p.table + static_cast<uint64_t>(s) * p.table_stride;
    constexpr uint32_t step = kWaves * KT;
    uint32_t j0 = c0 + wave * KT;
    // Their table entries are read a step before they are looked at: a value of a
    // load that is waited for here would wait for the rows requested before it.
    struct Slots {
        uint32_t of[NC];
    };
    auto slots_of = [&](uint32_t j0) {
        Slots r;
#pragma unroll
        for (uint32_t i = 0; i < NC; ++i) {
            // within the table, whatever the request's length
            r.of[i] = table[block_of(p, min(j0 + (lane & (KT - 1u)) + 64u * i, p.room - 1u))];
        }
        return r;
    };
    const Slots first_slots = slots_of(j0);  // on its way with the request's length

    const uint32_t hk = y % p.n_head_kv;
    const uint32_t tile = y / p.n_head_kv;
    const Span r = request_span(p, s);
    const uint32_t m = min(r.m, p.max_q);
    const uint32_t row0 = tile * kRowTile;
    if (row0 >= m * p.group) {
        return;
    }
    const uint32_t rows = min(kRowTile, m * p.group - row0);
    const uint32_t tok0 = row0 / p.group;  // first and last token of the rows
    const uint32_t tok1 = (row0 + rows - 1u) / p.group;
    const uint32_t n = key_limit(p, r, tok1);      // keys any of them attends
    const uint32_t n_all = key_limit(p, r, tok0);  // keys all of them attend
    const uint32_t n_parts = max(1u, (n + p.chunk - 1u) / p.chunk);
    if (part >= n_parts) {
        return;
    }
    const uint32_t nl = lane & 15u;   // query row; dim lane of the values
    const uint32_t c = lane >> 4;     // chunk of the contraction
    const uint32_t c1 = min(n, c0 + p.chunk);
    const uint8_t *k_head = p.k + static_cast<uint64_t>(hk) * SK::bytes;
    const uint8_t *v_head = p.v + static_cast<uint64_t>(hk) * SV::bytes;

    // The cells of this lane's keys of the step at j0, and which keys exist
    // (bit = key); one that does not has cell 0, and is masked where it matters.
    struct Cells {
        uint32_t at[NC];
        uint64_t have[NC];
    };
    auto cells_of = [&](const Slots &slots, uint32_t j0) {
        Cells r;
#pragma unroll
        for (uint32_t i = 0; i < NC; ++i) {
            const uint32_t j = j0 + (lane & (KT - 1u)) + 64u * i;
            const uint32_t slot = slots.of[i];
            const bool in = j < c1 && slot < p.n_slots;
            r.at[i] = in ? slot * p.T + (j - block_of(p, j) * p.T) : 0u;
            r.have[i] = __ballot(in);
        }
        return r;
    };
    auto cell_at = [&](const Cells &cells, uint32_t key) {
        uint32_t at = __shfl(cells.at[0], key & (KT - 1u) & 63u, 64);
        if constexpr (NC == 2) {
            const uint32_t hi = __shfl(cells.at[1], key & 63u, 64);
            at = key < 64u ? at : hi;
        }
        return at;
    };
    const uint32_t kk = lane / SK::units;  // this lane's key and unit of a load
    const uint32_t ku = min(kk, SK::per_load - 1u) == kk ? lane - kk * SK::units : 0u;
    const uint32_t vk = lane / SV::units;
    const uint32_t vu = min(vk, SV::per_load - 1u) == vk ? lane - vk * SV::units : 0u;
    UK rk[NLK];
    UV rv[NLV];
    auto load_tile = [&](const Cells &cells) {
#pragma unroll
        for (uint32_t i = 0; i < NLK; ++i) {
            const uint32_t at = cell_at(cells, kk + i * SK::per_load);
            rk[i] = *reinterpret_cast<const UK *>(k_head + static_cast<uint64_t>(at) * p.row_k + ku * SK::unit);
        }
#pragma unroll
        for (uint32_t i = 0; i < NLV; ++i) {
            const uint32_t at = cell_at(cells, vk + i * SV::per_load);
            rv[i] = *reinterpret_cast<const UV *>(v_head + static_cast<uint64_t>(at) * p.row_v + vu * SV::unit);
        }
    };
    const bool uneven = tok0 != tok1 && c1 > n_all;  // some rows do not attend all the keys
    if (uneven) {
        if (threadIdx.x < D) {
            first_odd[threadIdx.x] = ~0u;
        }
        __syncthreads();
    }

    // up to 8 rows: each stands in two columns, for the upper and the lower
    // digits of its weights
    const bool twice = rows <= 8u;
    const uint32_t my_row = row0 + min(twice ? (nl & 7u) : nl, rows - 1u);
    const uint32_t my_tok = my_row / p.group;
    const uint32_t my_head = hk * p.group + (my_row - my_tok * p.group);
    const uint32_t limit = key_limit(p, r, my_tok);

    // The row's queries, scaled into f16's range.  Codes carry an offset: the
    // sum of a group's queries times it comes off each score, as one more product
    // of the groups' scales with those sums (in two f16 pieces, 22 bits).
    Cells cells;
    Slots next;
    half8_t qf[NG];
    half8_t q_off;
    float fac, more;
    {
        const uint8_t *q = p.q + static_cast<uint64_t>(r.first + my_tok) * p.q_nb2 + my_head * p.q_nb1;
        u32x4_t x[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            x[g] = load_query<KO>(q, g, c);
        }
        cells = cells_of(first_slots, j0);
        load_tile(cells);
        next = slots_of(j0 + step);
        uint32_t bits = 0;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bits = max_magnitude(x[g][i], bits);
            }
        }
        bits = max(bits & 0xffffu, bits >> 16);
        float most = p.q_bf16 ? query_value<true>(bits) : query_value<false>(bits);
        most = fmaxf(most, lane_xor16(most));
        most = fmaxf(most, lane_xor32(most));
        const int ex = query_shift(most);
        const float up = ldexpf(1.0f, ex);
        if (p.q_bf16) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                qf[g] = query_operand<KO, true>(x[g], up);
            }
        } else {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                qf[g] = query_operand<KO, false>(x[g], up);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            q_off[e] = 0;
        }
        if constexpr (KO::codes) {
            // a group's sum is its product with a key of ones; its upper and lower
            // f16 digits stand in chunks 0 and 1 of the contraction
            half8_t ones;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                ones[e] = static_cast<_Float16>(KO::times(e));
            }
            const _Float16 pick_hi = static_cast<_Float16>(c == 0 ? 1.0f : 0.0f);
            const _Float16 pick_lo = static_cast<_Float16>(c == 1 ? 1.0f : 0.0f);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    qf[g][e] *= static_cast<_Float16>(1.0f / KO::times(e));
                }
                const float all = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                      ones, qf[g], float4_t{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0)[0] *
                                  (-KO::offset * 0x1p-10f);
                const _Float16 hi = static_cast<_Float16>(all);
                const _Float16 lo = static_cast<_Float16>(all - static_cast<float>(hi));
                q_off[g] = hi * pick_hi + lo * pick_lo;
            }
        }
        const ScoreFactor f = score_factor(p.scale, (KO::codes ? 24 : 0) - ex);
        fac = f.fac;
        more = f.more;
    }

    uint8_t *kt = lds + wave * decode_wave_bytes<TK, TV, D>();
    uint8_t *vt = kt + KT * SK::stride;
    scales_t *ks = reinterpret_cast<scales_t *>(vt + KT * SV::stride);  // [key] scales of its groups

    float top = -INFINITY;  // of the row, log2 units
    float sum = 0.0f;       // of this lane's weights
    float4_t o[VD];
#pragma unroll
    for (int t = 0; t < VD; ++t) {
        o[t] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // where registers are to spare
    constexpr bool kSpare = D < 256 || (TK == KVMEM_TYPE_Q4_0 && TV == KVMEM_TYPE_Q4_0);
    const Magic magic = kSpare ? Magic{anew(kMagic.low), anew(kMagic.high)} : kMagic;
    for (; j0 < c1; j0 += step) {
        const Cells now = cells;
        bool whole = true;
#pragma unroll
        for (uint32_t i = 0; i < NC; ++i) {
            whole = whole && now.have[i] == ~0ull;
        }
        wave_lds_sync();  // the last step's reads are done
        if (kk < SK::per_load) {
#pragma unroll
            for (uint32_t i = 0; i < NLK; ++i) {
                const uint32_t key = kk + i * SK::per_load;
                if ((i + 1) * SK::per_load <= KT || key < KT) {
                    *reinterpret_cast<UK *>(kt + key * SK::stride + ku * SK::unit) = rk[i];
                }
            }
        }
        if (vk < SV::per_load) {
#pragma unroll
            for (uint32_t i = 0; i < NLV; ++i) {
                const uint32_t key = vk + i * SV::per_load;
                if ((i + 1) * SV::per_load <= KT || key < KT) {
                    *reinterpret_cast<UV *>(vt + key * SV::stride + vu * SV::unit) = rv[i];
                }
            }
        }
        wave_lds_sync();
        cells = cells_of(next, j0 + step);
        load_tile(cells);
        next = slots_of(j0 + 2u * step);
        if constexpr (KO::codes) {
            // a key's scales side by side: 256 of a step, four a lane
            constexpr uint32_t per = NG < 4 ? NG : 4;
            typedef uint16_t some_t __attribute__((ext_vector_type(per)));
#pragma unroll
            for (uint32_t i = 0; i < 4u / per; ++i) {
                const uint32_t key = (lane + 64u * i) % KT;
                const uint32_t g0 = (lane + 64u * i) / KT * per;
                some_t d;
#pragma unroll
                for (uint32_t g = 0; g < per; ++g) {
                    d[g] = static_cast<uint16_t>(lds_half(kt + key * SK::stride + (g0 + g) * SK::GB));
                }
                *reinterpret_cast<some_t *>(reinterpret_cast<uint16_t *>(ks + key) + g0) = d;
            }
            wave_lds_sync();
        }
        float x[NT][4];
#pragma unroll
        for (uint32_t a0 = 0; a0 < NT; a0 += 2) {  // two tiles' products wait for one another's
            const uint8_t *kr[2];
            float4_t sc[2];
            scales_t d[2][4];
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                kr[i] = kt + (16u * (a0 + i) + nl) * SK::stride;
                sc[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (KO::codes) {
                    half8_t kd;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        kd[e] = 0;
                    }
                    const scales_t mine = ks[16u * (a0 + i) + nl];
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        kd[g] = __builtin_bit_cast(_Float16, static_cast<uint16_t>(mine[g]));
                    }
                    sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kd, q_off, sc[i], 0, 0, 0);
                    sc[i] *= 0x1p-14f;
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        d[i][j] = ks[16u * (a0 + i) + 4u * c + j];
                    }
                }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float4_t acc[2];
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    const uint8_t *gp = kr[i] + g * SK::GB;
                    const half8_t kf = __builtin_bit_cast(
                        half8_t, (g & 1) ? KO::load(gp, c, Aligned{}) : KO::load(gp, c, 2u));
                    if constexpr (KO::codes) {
                        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[g], float4_t{0.0f, 0.0f, 0.0f, 0.0f}, 0,
                                                                        0, 0);
                    } else {
                        sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[g], sc[i], 0, 0, 0);
                    }
                }
                if constexpr (KO::codes) {
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            sc[i][j] = __builtin_fmaf(
                                static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(d[i][j][g]))),
                                acc[i][j], sc[i][j]);
                        }
                    }
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[a0 + i][j] = sc[i][j] * fac;
                }
            }
        }
        if (more != 1.0f) {
#pragma unroll
            for (uint32_t a = 0; a < NT; ++a) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    x[a][i] *= more;
                }
            }
        }
        if (!whole || j0 + KT > n_all) {
#pragma unroll
            for (uint32_t h = 0; h < NT / 2; ++h) {
                const uint32_t seen = seen_keys(static_cast<uint32_t>(now.have[h >> 1] >> (32u * (h & 1u))),
                                                static_cast<int32_t>(limit - j0) - static_cast<int32_t>(32u * h), 4u * c);
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    float &v = x[2 * h + (e >> 2)][e & 3u];
                    v = (seen & (1u << (16u * (e >> 2) + (e & 3u)))) ? v : -INFINITY;
                }
            }
        }
        float most = -INFINITY;
#pragma unroll
        for (uint32_t a = 0; a < NT; ++a) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                most = fmaxf(most, x[a][i]);
            }
        }
        most = fmaxf(most, lane_xor16(most));
        most = fmaxf(most, lane_xor32(most));
        if (__any(most > top + kTopSlack)) {
            // each row by its own maximum: a row's sums do not depend on its neighbours
            const float higher = most > top + kTopSlack ? most : top;
            const float fade = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - higher);
            sum *= fade;
#pragma unroll
            for (int t = 0; t < VD; ++t) {
                o[t] *= fade;
            }
            top = higher;
        }
        const float base = (top == -INFINITY ? 0.0f : top) - kWeightShift;
        half8_t w[NT / 2];
#pragma unroll
        for (uint32_t a = 0; a < NT; ++a) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const float pe = __builtin_amdgcn_exp2f(x[a][i] - base);
                sum += pe;
                const _Float16 hi = static_cast<_Float16>(pe);
                w[a >> 1][4u * (a & 1u) + i] =
                    twice && (nl & 8u) ? static_cast<_Float16>(pe - static_cast<float>(hi)) : hi;
            }
        }
#pragma unroll
        for (uint32_t h = 0; h < NT / 2; ++h) {  // 32 keys each
            VO vo;
            vo.raw(nl, [&](uint32_t e) {
                return vt + (32u * h + 16u * (e >> 2) + 4u * c + (e & 3u)) * SV::stride;
            });
            u32x4_t keep{~0u, ~0u, ~0u, ~0u};
            if (!whole) {  // rows of keys that do not exist are not even finite
                keep = keep_keys<16>(static_cast<uint32_t>(now.have[h >> 1] >> (32u * (h & 1u))) >> (4u * c));
            }
            vo.emit(keep, magic, [&](int t0, u32x4_t *a) {
                if (uneven && j0 + KT > n_all) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        clear_odd(a[t], first_odd + VO::dim(nl, t0 + t),
                                  [&](uint32_t e) { return j0 + 32u * h + 16u * (e >> 2) + 4u * c + (e & 3u); });
                    }
                }
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    o[t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a[t]), w[h],
                                                                       o[t0 + t], 0, 0, 0);
                }
            });
        }
    }

    // join the chunks' sums and the two columns of a row
    sum += lane_xor16(sum);
    sum += lane_xor32(sum);
    if (twice) {
#pragma unroll
        for (int t = 0; t < VD; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[t][i] += lane_xor8(o[t][i]);
            }
        }
    }
    if (c == 0) {
        wave_ml[wave][nl] = make_float2(top, sum);
    }
    __syncthreads();  // every wave has left its tiles
    float all = wave_ml[0][nl].x;
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) {
        all = fmaxf(all, wave_ml[w][nl].x);
    }
    float *ow = reinterpret_cast<float *>(lds) + wave * rows * D;  // [row][dim]
    const float fade = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - all);
    if (nl < rows) {
        constexpr int RUN = VO::RUN;  // neighbouring dims among a lane's
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
#pragma unroll
            for (int t = 0; t < VD; t += RUN) {
                typedef float run_t __attribute__((ext_vector_type(RUN)));
                run_t v;
#pragma unroll
                for (int u = 0; u < RUN; ++u) {
                    v[u] = o[VO::nth(t + u)][i] * fade;
                }
                *reinterpret_cast<run_t *>(ow + nl * D + VO::dim(4u * c + i, VO::nth(t))) = v;
            }
        }
    }
    __syncthreads();
    // a wave takes 256 elements of the rows, a lane four
    const float *ol = reinterpret_cast<const float *>(lds);
    for (uint32_t e0 = wave * 256u; e0 < rows * D; e0 += 1024u) {
        const uint32_t e = min(e0 + 4u * lane, rows * D - 4u);
        const bool in = e == e0 + 4u * lane;
        const uint32_t row = e / D;
        const uint32_t d = e & (D - 1u);
        const uint32_t tok = (row0 + row) / p.group;
        const uint32_t head = hk * p.group + (row0 + row - tok * p.group);
        const uint64_t at = static_cast<uint64_t>(r.first + tok) * p.n_head + head;
        float mx = -INFINITY, total = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            mx = fmaxf(mx, wave_ml[w][row].x);
        }
        float4_t x{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            const float2 ml = wave_ml[w][row];
            total += ml.y * (ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mx));
            x += *reinterpret_cast<const float4_t *>(ol + w * rows * D + e);
        }
        if (uneven) {
            const uint32_t limit = key_limit(p, r, tok);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = first_odd[d + i] < limit ? NAN : x[i];
            }
        }
        if (n_parts > 1) {
            if (in) {
                const uint64_t pe = static_cast<uint64_t>(part) * p.n_tokens * p.n_head + at;
                *reinterpret_cast<float4_t *>(p.part_o + pe * D + d) = x;
                if (d == 0) {
                    p.part_ml[pe] = make_float2(mx, total);
                }
            }
            continue;
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
        if (p.hadamard) {
            rotate_lanes<4>(y, p.hadamard, lane);
        }
        if (in) {
            store_elems<4>(p.out, p.out_type, at * D + d, y);
            if (d == 0 && p.lse) {
                p.lse[at] = total == 0.0f ? -INFINITY : (mx - kWeightShift) / kLog2e + logf(total);
            }
        }
    }
}

// A group's scale with which some code passes f16 (an infinite scale too).
template <class KO>
__device__ inline bool beyond_f16(uint32_t scale) {
    const _Float16 d = __builtin_bit_cast(_Float16, static_cast<uint16_t>(scale));
    return __builtin_fabsf16(d) > static_cast<_Float16>(65504.0f / KO::offset);
}

// f16 values of a key operand's codes, scaled (rounded once).
template <class KO>
__device__ inline u32x4_t key_values(u32x4_t codes, uint32_t scale) {
    if constexpr (!KO::codes) {
        return codes;
    } else {
        u32x4_t r;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            r[j] = KO::times(2 * j) == 1.0f ? pair_value(codes[j], kMagic.low, KO::offset, scale)
                                            : pair_value_hi(codes[j], kMagic.high, KO::offset, scale);
        }
        return r;
    }
}

// ------------------------------------------------------------ many queries

typedef float float16_t __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void_t;

template <int TK, int TV, int D>
struct PrefillLds {
    static constexpr uint32_t KT = step_keys(D);
    static constexpr uint32_t raw_k = KT * Slice<TK, D>::bytes;  // rows as cached
    static constexpr uint32_t raw = raw_k + KT * Slice<TV, D>::bytes;
    static constexpr uint32_t key_stride = 2 * D + 16;           // padded against bank conflicts
    static constexpr uint32_t keys = KT * key_stride;            // keys as f16 [key][D]
    // values as f16 [octet of keys][D] operands; one operand's room after each 32
    // keeps the writing lanes (dims of neighbouring groups) on different banks
    static constexpr uint32_t octet = (D + D / 32) * 16;
    static constexpr uint32_t values = KT / 8 * octet;
    // two of each: one in use while the next is made; 16 bytes behind the
    // last row, whose last word is read with the next one
    static constexpr uint32_t bytes = 2 * (raw + keys + values) + 16;
};

// Where operand `dim` of an octet stands.
__device__ inline uint32_t value_slot(uint32_t dim) { return dim + (dim >> 5); }

// 256 rows of one KV head's queries over one part of a request's keys, 32 a wave.
// Steps of step_keys(D) keys: their rows come into LDS two steps ahead, are made
// f16 one step ahead (8 keys of 4 value dims for each thread of four waves, and 4
// octets of key dims for each of the others), and every wave multiplies its rows
// (transposed products as in the decode kernel, on 32x32 tiles).  One barrier a
// step.  Two waves per SIMD cover each other's LDS reads and softmax; 128 rows in
// four waves take as long for 126 rows (118 and 116 us over 32768 keys) and twice
// as long for many, since making f16 is done twice.
//
// Bound by the matrix units and what stands between their products.  512 tokens
// over 32768 keys, 24/4 heads of 256, q4_0: 469-491 us = 835-872 TFLOP/s, the
// matrix units 41 % busy, vector instructions 50 % (nine for each matrix
// instruction); f16 521 us; 32/8 heads of 128: f16 328 us, q8_0 370 us.  A workgroup
// takes about 15 us beside its steps (table, first rows and queries in, sums out),
// which short prompts feel.  Keys and weights are f16 because the matrix units take
// that: 2^-11 of each, which averages over a row's keys (against 64 bits this call is
// off by 1.7e-3 in bf16, as the same arithmetic in fp32 is).
template <int TK, int TV, int D>
__global__ __launch_bounds__(64 * kPrefillWaves, 2) void attn_prefill_kernel(AttnParams p) {
    constexpr uint32_t NW = kPrefillWaves;
    using SK = Slice<TK, D>;
    using SV = Slice<TV, D>;
    using KO = KeyOp<TK>;
    using VO = ValueOp<TV, 4>;
    using L = PrefillLds<TK, TV, D>;
    constexpr uint32_t KT = L::KT;
    constexpr int NT = KT / 32;    // key tiles of a step
    constexpr int QS = D / 16;     // products of a key tile's scores
    constexpr int NB = D / 32;     // blocks of value dims
    constexpr uint32_t NC = KT > 64 ? KT / 64 : 1;
    constexpr uint32_t NTH = 64 * NW;
    constexpr uint32_t NK = (KT * SK::units + NTH - 1u) / NTH;
    constexpr uint32_t NV = (KT * SV::units + NTH - 1u) / NTH;
    constexpr uint32_t kRows = kPrefillRows;
    typedef typename UnitOf<SK::unit>::type UK;
    typedef typename UnitOf<SV::unit>::type UV;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ uint32_t first_odd[D];
    // Of the two steps of f16 keys in LDS: the step whose key has a group beyond f16
    // and is held times 2^-7 (its elements are then rounded to 2^-18 at the finest, far
    // below what rounds its largest ones), and the step that has any such key.
    __shared__ __attribute__((aligned(16))) uint32_t beyond[2][KT];
    __shared__ uint32_t any_beyond[2];

    // Workgroups go to the 8 XCDs in turn.  A unit (request, part, KV head) stays on
    // one of them, whose L2 then holds its rows for all row tiles; units that do
    // not make a round of eight are spread.  Tiles with the most keys come first.
    const uint32_t xcd = blockIdx.x & 7u;
    const uint32_t turn_of = blockIdx.x >> 3;
    const uint32_t per_xcd = p.units >> 3;
    const uint32_t even = per_xcd * p.row_tiles;
    uint32_t unit, tile;
    if (turn_of < even) {
        unit = (turn_of % per_xcd) * 8u + xcd;
        tile = turn_of / per_xcd;
    } else {
        const uint32_t rest = p.units & 7u;
        const uint32_t w = (turn_of - even) * 8u + xcd;
        unit = per_xcd * 8u + w % max(rest, 1u);
        tile = w / max(rest, 1u);
    }
    if (unit >= p.units || tile >= p.row_tiles) {
        return;
    }
    tile = p.row_tiles - 1u - tile;
    const uint32_t hk = unit % p.n_head_kv;
    const uint32_t sp = unit / p.n_head_kv;
    const uint32_t s = sp / p.n_parts;
    const uint32_t part = sp - s * p.n_parts;
    if (s >= p.n_seq) {
        return;
    }
    const Span r = request_span(p, s);
    const uint32_t m = min(r.m, p.max_q);
    const uint32_t row0 = tile * kRows;
    if (row0 >= m * p.group) {
        return;
    }
    const uint32_t rows = min(kRows, m * p.group - row0);
    const uint32_t n = key_limit(p, r, (row0 + rows - 1u) / p.group);
    const uint32_t n_all = key_limit(p, r, row0 / p.group);
    const uint32_t n_parts = max(1u, (n + p.chunk - 1u) / p.chunk);
    if (part >= n_parts) {
        return;
    }
    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t nl = lane & 31u;  // query row of a tile
    const uint32_t hh = lane >> 5;   // half of the contraction
    const uint32_t c0 = part * p.chunk;
    const uint32_t c1 = min(n, c0 + p.chunk);
    const uint8_t *k_head = p.k + static_cast<uint64_t>(hk) * SK::bytes;
    const uint8_t *v_head = p.v + static_cast<uint64_t>(hk) * SV::bytes;
    const uint32_t *table = p.table + static_cast<uint64_t>(s) * p.table_stride;

    // as in the decode kernel: cells of a step's keys, and which keys exist
    struct Cells {
        uint32_t at[NC];
        uint64_t have[NC];
    };
    // Their table entries are read a step before they are looked at: a value of a
    // load that is waited for here would wait for the rows requested before it.
    struct Slots {
        uint32_t of[NC];
    };
    auto slots_of = [&](uint32_t j0) {
        Slots r;
#pragma unroll
        for (uint32_t i = 0; i < NC; ++i) {
            // within the table, whatever the request's length
            r.of[i] = table[block_of(p, min(j0 + (lane & (KT - 1u)) + 64u * i, p.room - 1u))];
        }
        return r;
    };
    auto cells_of = [&](const Slots &slots, uint32_t j0) {
        Cells r;
#pragma unroll
        for (uint32_t i = 0; i < NC; ++i) {
            const uint32_t j = j0 + (lane & (KT - 1u)) + 64u * i;
            const uint32_t slot = slots.of[i];
            const bool in = j < c1 && slot < p.n_slots;
            r.at[i] = in ? slot * p.T + (j - block_of(p, j) * p.T) : 0u;
            r.have[i] = __ballot(in);
        }
        return r;
    };
    auto cell_at = [&](const Cells &cells, uint32_t key) {
        uint32_t at = __shfl(cells.at[0], key & (KT - 1u) & 63u, 64);
        if constexpr (NC == 2) {
            const uint32_t hi = __shfl(cells.at[1], key & 63u, 64);
            at = key < 64u ? at : hi;
        }
        return at;
    };
    // A step's rows on their way to `raw`.  Slices of 256 dims are whole 16-byte
    // units: those go straight to LDS (fetch_tile; there are no registers to spare),
    // narrower ones through registers (load here, store in put_tile).
    constexpr bool kDirect = D == 256;
    constexpr uint32_t KU = KT * SK::units;
    constexpr uint32_t NU = KU + KT * SV::units;
    UK rk[kDirect ? 1 : NK];
    UV rv[kDirect ? 1 : NV];
    auto fetch_tile = [&](const Cells &cells, uint8_t *raw) {
        if constexpr (kDirect) {
            const uint32_t t = anew(tid);
#pragma unroll
            for (uint32_t i = 0; i < (NU + NTH - 1u) / NTH; ++i) {
                const uint32_t u = i * NTH + t;
                const bool is_v = u >= KU;
                const uint32_t w = is_v ? u - KU : u;
                const uint32_t key = is_v ? w / SV::units : w / SK::units;
                const uint32_t off = (w - key * (is_v ? SV::units : SK::units)) * 16u;
                const uint64_t row = static_cast<uint64_t>(cell_at(cells, key)) * (is_v ? p.row_v : p.row_k);
                const uint8_t *src = (is_v ? v_head : k_head) + row + off;
                if ((i + 1) * NTH <= NU || u < NU) {
                    __builtin_amdgcn_global_load_lds(src, (lds_void_t *) (raw + (i * NTH + wave * 64u) * 16u), 16, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < NK; ++i) {
                const uint32_t u = i * NTH + tid;
                const uint32_t key = u / SK::units;
                const uint32_t at = cell_at(cells, key);
                rk[i] = *reinterpret_cast<const UK *>(k_head + static_cast<uint64_t>(at) * p.row_k +
                                                      (u - key * SK::units) * SK::unit);
            }
#pragma unroll
            for (uint32_t i = 0; i < NV; ++i) {
                const uint32_t u = i * NTH + tid;
                const uint32_t key = u / SV::units;
                const uint32_t at = cell_at(cells, key);
                rv[i] = *reinterpret_cast<const UV *>(v_head + static_cast<uint64_t>(at) * p.row_v +
                                                      (u - key * SV::units) * SV::unit);
            }
        }
    };
    // The fetched step is in `raw` once the barrier behind this call is passed.
    auto put_tile = [&](uint8_t *raw) {
        if constexpr (kDirect) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        } else {
#pragma unroll
            for (uint32_t i = 0; i < NK; ++i) {
                const uint32_t u = i * NTH + tid;
                if ((i + 1) * NTH <= KT * SK::units || u < KT * SK::units) {
                    *reinterpret_cast<UK *>(raw + u * SK::unit) = rk[i];
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < NV; ++i) {
                const uint32_t u = i * NTH + tid;
                if ((i + 1) * NTH <= KT * SV::units || u < KT * SV::units) {
                    *reinterpret_cast<UV *>(raw + L::raw_k + u * SV::unit) = rv[i];
                }
            }
        }
    };
    uint8_t *const raw0 = lds;
    uint8_t *const keys0 = lds + 2 * L::raw;
    uint8_t *const values0 = keys0 + 2 * L::keys;

    // Making f16 of a step's rows, in pieces.  Values: this thread's octet of
    // keys (keys 16 (q / 2) + 8 (e / 4) + 4 (q % 2) + e % 4, as a lane of the
    // scores holds them) and its 4 dims.
    const bool for_values = wave < 4u;  // four waves make values, four keys
    const bool for_keys = !for_values;
    const bool mixed = c1 > n_all;  // some rows do not attend all the keys
    auto make_values = [&](const uint8_t *raw, uint8_t *values, const uint64_t *have, uint32_t j0, uint32_t mt) {
        const uint32_t oct = mt / (D / 4);
        const uint32_t dl = mt % (D / 4);
        VO vo;
        vo.raw(dl, [&](uint32_t e) {
            return raw + L::raw_k + (16u * (oct >> 1) + 8u * (e >> 2) + 4u * (oct & 1u) + (e & 3u)) * SV::bytes;
        });
        const uint32_t in = static_cast<uint32_t>(have[oct >> 3] >> (16u * ((oct >> 1) & 3u) + 4u * (oct & 1u)));
        vo.emit(keep_keys<8>(in), kMagic, [&](int, u32x4_t *a) {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint32_t dim = VO::dim(dl, t);
                if (mixed && j0 + KT > n_all) {
                    clear_odd(a[t], first_odd + dim, [&](uint32_t e) {
                        return j0 + 16u * (oct >> 1) + 8u * (e >> 2) + 4u * (oct & 1u) + (e & 3u);
                    });
                }
                *reinterpret_cast<u32x4_t *>(values + oct * L::octet + value_slot(dim) * 16u) = a[t];
            }
        });
    };
    // Keys: octet i of 4 of this thread.
    u32x4_t codes;
    uint32_t key_scale = 0;
    auto key_read = [&](const uint8_t *raw, uint32_t i, uint32_t mt) {
        const uint32_t u = i * 256u + mt;
        const uint32_t key = u / (D / 8);
        const uint32_t o = u % (D / 8);
        const uint8_t *g = raw + key * SK::bytes + (o >> 2) * SK::GB;
        if constexpr (KO::codes) {
            key_scale = lds_half(g) * 0x00010001u;
        }
        codes = KO::load(g, o & 3u, 2u * (~(o >> 2) & 1u));
    };
    auto key_write = [&](uint8_t *keys, uint32_t i, uint32_t mt, uint32_t which, uint32_t j0) {
        const uint32_t u = i * 256u + mt;
        const uint32_t key = u / (D / 8);
        const uint32_t o = u % (D / 8);
        if constexpr (KO::codes) {
            // a key's octets are D / 8 neighbouring lanes
            const uint64_t big = __ballot(beyond_f16<KO>(key_scale));
            if (__builtin_expect(big != 0, 0)) {
                const uint32_t at = anew(lane);
                if ((big >> (at & ~(D / 8u - 1u))) & ((1ull << (D / 8)) - 1u)) {
                    key_scale = as_word(as_half2(key_scale) * half2_t{0x1p-7f16, 0x1p-7f16});
                    beyond[which][key] = j0;
                    any_beyond[which] = j0;
                }
            }
        }
        *reinterpret_cast<u32x4_t *>(keys + key * L::key_stride + o * 16u) = key_values<KO>(codes, key_scale);
    };

    const Slots slots0 = slots_of(c0);
    const Slots slots1 = slots_of(c0 + KT);
    Slots next = slots_of(c0 + 2u * KT);

    // The first rows are on their way while the queries are made.
    const Cells cells0 = cells_of(slots0, c0);
    const Cells cells1 = cells_of(slots1, c0 + KT);
    fetch_tile(cells0, raw0);
    if constexpr (kDirect) {
        fetch_tile(cells1, raw0 + L::raw);
    }

    // This wave's queries, scaled into f16's range row by row: made operands in
    // LDS, where the steps' f16 rows will stand.
    half8_t qf[QS];
    // token and query head of a lane's row (rows behind the last one repeat it)
    auto tok_of = [&](uint32_t l) { return (row0 + min(wave * 32u + (l & 31u), rows - 1u)) / p.group; };
    auto head_of = [&](uint32_t l) { return hk * p.group + (row0 + min(wave * 32u + (l & 31u), rows - 1u)) % p.group; };
    float fac, more;
    {
        constexpr uint32_t TURNS = NW * QS * 1024u <= 2 * (L::keys + L::values) ? 1 : 2;
        constexpr uint32_t PER = NW / TURNS;  // waves whose queries fit at a time
        u32x4_t *ql = reinterpret_cast<u32x4_t *>(lds + 2 * L::raw) + (wave % PER) * QS * 64u + lane;
        const uint8_t *q = p.q + static_cast<uint64_t>(r.first + tok_of(lane)) * p.q_nb2 + head_of(lane) * p.q_nb1;
        int ex = 0;
#pragma unroll
        for (uint32_t turn = 0; turn < TURNS; ++turn) {
            if (wave / PER == turn) {
                uint32_t bits = 0;
#pragma unroll 4
                for (uint32_t st = 0; st < QS; ++st) {
                    const u32x4_t x = load_query<KO>(q, st >> 1, 2u * (st & 1u) + hh);
                    ql[st * 64u] = x;
                    bits = max_magnitude(x[0], max_magnitude(x[1], max_magnitude(x[2], max_magnitude(x[3], bits))));
                }
                bits = max(bits & 0xffffu, bits >> 16);
                float most = p.q_bf16 ? query_value<true>(bits) : query_value<false>(bits);
                most = fmaxf(most, lane_xor32(most));
                ex = query_shift(most);
                const float up = ldexpf(1.0f, ex);
#pragma unroll 1
                for (uint32_t st = 0; st < QS; ++st) {
                    const u32x4_t x = ql[st * 64u];
                    const half8_t h = p.q_bf16 ? query_operand<KO, true>(x, up) : query_operand<KO, false>(x, up);
                    ql[st * 64u] = __builtin_bit_cast(u32x4_t, h);
                }
#pragma unroll
                for (uint32_t st = 0; st < QS; ++st) {
                    qf[st] = __builtin_bit_cast(half8_t, ql[st * 64u]);
                }
            }
            __syncthreads();  // the queries have left the step buffers
        }
        const ScoreFactor f = score_factor(p.scale, -ex);
        fac = fmaxf(f.fac, 0x1p-126f);
        more = f.more;
    }

    float top = -INFINITY;
    float sum = 0.0f;
    bool far = more != 1.0f;  // some row's scores have passed kFarScore (or its factor fp32)
    float16_t o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            o[b][i] = 0.0f;
        }
    }
    if (tid < D) {
        first_odd[tid] = ~0u;
    }
    if constexpr (KO::codes) {
        if (tid < KT) {
            beyond[0][tid] = beyond[1][tid] = ~0u;
        }
        if (tid < 2u) {
            any_beyond[tid] = ~0u;
        }
    }
    put_tile(raw0);
    if constexpr (!kDirect) {
        fetch_tile(cells1, raw0 + L::raw);
        put_tile(raw0 + L::raw);
    }
    uint64_t have[NC], have1[NC];
#pragma unroll
    for (uint32_t i = 0; i < NC; ++i) {
        have[i] = cells0.have[i];
        have1[i] = cells1.have[i];
    }
    __syncthreads();
    if (for_values) {
        make_values(raw0, values0, have, c0, tid & 255u);
    }
    if (for_keys) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            key_read(raw0, i, tid & 255u);
            key_write(keys0, i, tid & 255u, 0u, c0);
        }
    }
    __syncthreads();

    uint32_t buf = 0;  // step modulo 2
    for (uint32_t j0 = c0; j0 < c1; j0 += KT) {
        uint64_t have2[NC];
        const Cells cells = cells_of(next, j0 + 2u * KT);
        fetch_tile(cells, raw0 + buf * L::raw);  // (its rows were made f16 in the last step)
        next = slots_of(j0 + 3u * KT);
#pragma unroll
        for (uint32_t i = 0; i < NC; ++i) {
            have2[i] = cells.have[i];
        }
        const uint32_t mt = anew(tid & 255u);
        const uint8_t *raw1 = raw0 + (buf ^ 1u) * L::raw;
        uint8_t *keys1 = keys0 + (buf ^ 1u) * L::keys;
        uint8_t *values1 = values0 + (buf ^ 1u) * L::values;

        if (for_keys) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                key_read(raw1, i, mt);
                key_write(keys1, i, mt, buf ^ 1u, j0 + KT);
            }
        }
        uint32_t far_keys = 0;
        if constexpr (KO::codes) {
            far_keys = any_beyond[buf];
        }
        float16_t sc[NT];
        const uint8_t *kr = keys0 + buf * L::keys + nl * L::key_stride + hh * 16u;
        auto key_operand = [&](int z) {
            return *reinterpret_cast<const half8_t *>(kr + z / QS * 32 * L::key_stride + z % QS * 32);
        };
        half8_t ring[4];  // operands are read four products ahead
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            ring[z] = key_operand(z);
        }
#pragma unroll
        for (int z = 0; z < NT * QS; ++z) {
            const int a = z / QS;
            if (z % QS == 0) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sc[a][i] = 0.0f;
                }
            }
            sc[a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[z & 3], qf[z % QS], sc[a], 0, 0, 0);
            if (z + 4 < NT * QS) {
                ring[z & 3] = key_operand(z + 4);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (KO::codes) {
            if (__builtin_expect(__builtin_amdgcn_readfirstlane(far_keys) == j0, 0)) {
                const uint32_t *of = &beyond[buf][4 * (anew(lane) >> 5)];
#pragma unroll
                for (int a = 0; a < NT; ++a) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        sc[a][i] *= of[32 * a + 2 * (i & ~3) + (i & 3)] == j0 ? 0x1p7f : 1.0f;
                    }
                }
            }
        }
        bool whole = j0 + KT <= n_all;
#pragma unroll
        for (uint32_t i = 0; i < NC; ++i) {
            whole = whole && have[i] == ~0ull;
        }
        if (!whole) {
            const uint32_t limit = key_limit(p, r, tok_of(anew(lane)));
#pragma unroll
            for (uint32_t a = 0; a < NT; ++a) {
                const uint32_t seen =
                    seen_keys(static_cast<uint32_t>(have[a >> 1] >> (32u * (a & 1u))),
                              static_cast<int32_t>(limit - j0) - static_cast<int32_t>(32u * a), 4u * hh);
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i) {
                    sc[a][i] = (seen & (1u << (8u * (i >> 2) + (i & 3u)))) ? sc[a][i] : -INFINITY;
                }
            }
        }
        float most = -INFINITY;
#pragma unroll
        for (int a = 0; a < NT; ++a) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                most = fmaxf(most, sc[a][i]);
            }
        }
        most *= fac;
        most = fmaxf(most * more, lane_xor32(most * more));
        if (__any(most > top + kTopSlack)) {
            // each row by its own maximum: a row's sums do not depend on its neighbours
            const float higher = most > top + kTopSlack ? most : top;
            const float fade = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - higher);
            sum *= fade;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                o[b] *= fade;
            }
            top = higher;
            far = far || __any(is_far(top));
        }
        const float base = (top == -INFINITY ? 0.0f : top) - kWeightShift;
        half8_t w[2 * NT];
        // The maximum is a rounded product.  Beyond kFarScore what its rounding took
        // off is no longer small against a weight's exponent: products are rounded
        // there as the maximum's was (row by row, for rows that have come so far).
        float times = fac, less = base;
        if (__builtin_expect(far, 0)) {
            const float all = fac * more;
            const bool rounded = is_far(top) || all == INFINITY;
#pragma unroll
            for (int a = 0; a < NT; ++a) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sc[a][i] = rounded ? sc[a][i] * fac * more - base : __builtin_fmaf(sc[a][i], all, -base);
                }
            }
            times = 1.0f;
            less = 0.0f;
        }
#pragma unroll
        for (int a = 0; a < NT; ++a) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float pe = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[a][i], times, -less));
                sum += pe;
                w[2 * a + (i >> 3)][i & 7] = static_cast<_Float16>(pe);
            }
        }
        const uint8_t *vr = values0 + buf * L::values + hh * L::octet + nl * 16u;
        auto value_operand = [&](int z) {
            return *reinterpret_cast<const half8_t *>(vr + 2 * (z / NB) * L::octet + 33 * (z % NB) * 16);
        };
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            ring[z] = value_operand(z);
        }
#pragma unroll
        for (int z = 0; z < 2 * NT * NB; ++z) {
            o[z % NB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[z & 3], w[z / NB], o[z % NB], 0, 0, 0);
            if (z + 4 < 2 * NT * NB) {
                ring[z & 3] = value_operand(z + 4);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (for_values) {
            make_values(raw1, values1, have1, j0 + KT, mt);
        }
        put_tile(raw0 + buf * L::raw);
#pragma unroll
        for (uint32_t i = 0; i < NC; ++i) {
            have[i] = have1[i];
            have1[i] = have2[i];
        }
        buf ^= 1u;
        __syncthreads();
    }

    // a lane holds dims 32 b + 8 (i / 4) + 4 hh + i % 4 of its row
    const bool uneven = mixed && __syncthreads_or(tid < D && first_odd[tid] != ~0u);
    sum += lane_xor32(sum);
    const uint32_t end_lane = anew(lane);
    const uint32_t tok = tok_of(end_lane);
    const uint32_t head = head_of(end_lane);
    const uint32_t limit = key_limit(p, r, tok);
    const bool mine = wave * 32u + (end_lane & 31u) < rows;
    // parts, and sums that still have to be rotated, go to the joining kernel
    const bool joined = n_parts > 1 || p.hadamard;
    const uint64_t at = static_cast<uint64_t>(r.first + tok) * p.n_head + head;
    const uint64_t to = (joined ? static_cast<uint64_t>(part) * p.n_tokens * p.n_head : 0u) + at;
    const float f = joined ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
    uint8_t *out = joined ? reinterpret_cast<uint8_t *>(p.part_o) : p.out;
    const int type = joined ? static_cast<int>(KVMEM_TYPE_F32) : p.out_type;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const uint32_t dim = 32 * b + 2 * i + 4 * hh;
            float x[4] = {o[b][i] * f, o[b][i + 1] * f, o[b][i + 2] * f, o[b][i + 3] * f};
            if (uneven) {
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    x[d] = first_odd[dim + d] < limit ? NAN : x[d];
                }
            }
            if (mine) {
                store_elems<4>(out, type, to * D + dim, x);
            }
        }
    }
    if (mine && hh == 0) {
        if (joined) {
            p.part_ml[to] = make_float2(top, sum);
        } else if (p.lse) {
            p.lse[at] = sum == 0.0f ? -INFINITY : (top - kWeightShift) / kLog2e + logf(sum);
        }
    }
}

// -------------------------------------------------------------------- launch

template <int TK, int TV, int D>
static void launch_types(hipStream_t stream, const AttnPlan &pl, const AttnParams &p) {
    const uint32_t grid = static_cast<uint32_t>(pl.grid);
    if (pl.prefill) {
        attn_prefill_kernel<TK, TV, D><<<grid, 64 * kPrefillWaves, PrefillLds<TK, TV, D>::bytes, stream>>>(p);
    } else {
        const uint32_t rows = std::min(kRowTile, p.max_q * p.group);
        // 16 bytes behind the last slice: its last word is read with the next one
        const uint32_t lds = std::max<uint32_t>(kWaves * decode_wave_bytes<TK, TV, D>() + 16u,
                                                std::max<uint32_t>(kWaves * rows * D * 4u, 1024u));
        attn_decode_kernel<TK, TV, D><<<grid, 256, lds, stream>>>(p);
    }
}

template <int TK, int TV>
static void launch_dims(hipStream_t stream, uint32_t d, const AttnPlan &pl, const AttnParams &p) {
    if (d == 64) {
        launch_types<TK, TV, 64>(stream, pl, p);
    } else if (d == 128) {
        launch_types<TK, TV, 128>(stream, pl, p);
    } else {
        launch_types<TK, TV, 256>(stream, pl, p);
    }
}

template <int TK>
void launch_attention(hipStream_t stream, int type_v, uint32_t d, const AttnPlan &pl, const AttnParams &p) {
    switch (type_v) {
        case KVMEM_TYPE_Q4_0: launch_dims<TK, KVMEM_TYPE_Q4_0>(stream, d, pl, p); break;
        case KVMEM_TYPE_Q5_0: launch_dims<TK, KVMEM_TYPE_Q5_0>(stream, d, pl, p); break;
        case KVMEM_TYPE_Q8_0: launch_dims<TK, KVMEM_TYPE_Q8_0>(stream, d, pl, p); break;
        default: launch_dims<TK, KVMEM_TYPE_F16>(stream, d, pl, p); break;
    }
}

template <int TK>
bool load_attention() {
    return load_kernel_object(&attn_decode_kernel<TK, KVMEM_TYPE_Q4_0, 64>);
}

}  // namespace kvmem_hip
