// Attention of new tokens over the pool's rows (kvmem_hip_attention).
#include "kvmem_internal.hpp"

#include <algorithm>
#include <cmath>

namespace kvmem_hip {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

constexpr uint32_t kTileKeys = 32;   // keys of one prefill step
constexpr uint32_t kRowTile = 16;    // query rows of a workgroup
constexpr uint32_t kWaves = 4;
constexpr uint32_t kNoCell = 0xffffffffu;
// Softmax weights are 2^(x - top + shift) before they are rounded to f16.  A
// row's `top` follows its maximum only when that has grown by more than
// kTopSlack (log2), so the sums are rarely scaled down again; weights then stay
// below 2^15, and those down to 2^-20 of 2^top are normal f16 numbers.
constexpr float kWeightShift = 6.0f;
constexpr float kTopSlack = 9.0f;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
    const uint8_t *q;
    uint64_t q_nb1, q_nb2;
    uint8_t *out;
    float *lse;
    const uint8_t *k;
    const uint8_t *v;
    const uint32_t *q_start;
    const uint32_t *kv_len;
    const uint32_t *table;
    float *part_o;              // [part][token][head][D] sums of weighted values
    float2 *part_ml;            // [part][token][head] maximum (log2), sum of weights
    uint32_t row_k, row_v;      // bytes of a cached row
    uint32_t n_tokens, n_seq, max_q, max_kv, n_head, n_head_kv, group, T, n_slots, table_stride;
    uint32_t chunk;             // keys of one part
    uint32_t n_parts;           // parts of the longest request
    uint32_t row_tile;          // rows of one workgroup
    uint32_t row_tiles;         // of the longest request
    uint32_t units;             // of the grid's fast index, a multiple of 8
    int32_t causal;
    int32_t q_bf16;
    int32_t out_type;
    uint32_t hadamard;
    float scale;
};

// A request's share of the call: its first token, tokens, keys in range.
struct Span {
    uint32_t first, m, len, keys;
};

__device__ inline Span request_span(const AttnParams &p, uint32_t s) {
    Span r;
    const uint32_t a = p.q_start ? min(p.q_start[s], p.n_tokens) : s;
    const uint32_t b = p.q_start ? min(p.q_start[s + 1], p.n_tokens) : s + 1;
    r.first = a;
    r.m = b > a ? b - a : 0u;
    r.len = p.kv_len[s];
    const uint64_t room = static_cast<uint64_t>(p.table_stride) * p.T;
    r.keys = static_cast<uint32_t>(min<uint64_t>(min(r.len, p.max_kv), room));
    return r;
}

// Keys token i attends: [0, limit).
__device__ inline uint32_t key_limit(const AttnParams &p, const Span &r, uint32_t i) {
    if (!p.causal) {
        return r.keys;
    }
    const int64_t last = static_cast<int64_t>(r.len) - r.m + i + 1;
    return last <= 0 ? 0u : static_cast<uint32_t>(min<int64_t>(r.keys, last));
}

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
// The same where the shift is known: 2 bytes (OFF) or none.
template <int N, bool OFF>
__device__ inline void lds_words(const uint8_t *p, uint32_t out[N]) {
    if constexpr (OFF) {
        lds_words<N>(p, 2u, out);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            out[i] = reinterpret_cast<const uint32_t *>(p)[i];
        }
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
// OFF: the group's codes lie 2 bytes off a word (groups of even number).
// Element e is dim piece(c, i) + l % 4 of the group, l = order(e) and i = l / 4:
// a lane's 8 dims are two runs of four.
template <int TYPE> struct KeyOp;

template <> struct KeyOp<KVMEM_TYPE_Q4_0> {
    static constexpr float offset = 8.0f;
    static constexpr bool codes = true;
    template <bool OFF>
    __device__ static inline u32x4_t load(const uint8_t *g, uint32_t c) {
        uint32_t w;
        lds_words<1, OFF>(g + 2 + 4 * c, &w);
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
    template <bool OFF>
    __device__ static inline u32x4_t load(const uint8_t *g, uint32_t c) {
        uint32_t h, w;
        lds_words<1, OFF>(g + 2, &h);
        lds_words<1, OFF>(g + 6 + 4 * c, &w);
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
    template <bool OFF>
    __device__ static inline u32x4_t load(const uint8_t *g, uint32_t c) {
        uint32_t w[2];
        lds_words<2, OFF>(g + 2 + 8 * c, w);
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
    template <bool OFF>
    __device__ static inline u32x4_t load(const uint8_t *g, uint32_t c) {
        return *reinterpret_cast<const u32x4_t *>(g + 16 * c);
    }
    __device__ static inline uint32_t piece(uint32_t c, uint32_t i) { return 8 * c + 4 * i; }
    __device__ static constexpr uint32_t order(uint32_t e) { return e; }
    __device__ static constexpr float times(uint32_t) { return 1.0f; }
};

// The operand of group g of a key's slice (an unrolled g).
template <class KO, uint32_t GB>
__device__ inline u32x4_t load_key(const uint8_t *slice, int g, uint32_t c) {
    return (g & 1) ? KO::template load<false>(slice + g * GB, c) : KO::template load<true>(slice + g * GB, c);
}

__device__ inline half2_t as_half2(uint32_t w) { return __builtin_bit_cast(half2_t, w); }
__device__ inline uint32_t as_word(half2_t h) { return __builtin_bit_cast(uint32_t, h); }

// (low halves, high halves) of a key pair's words: a in the lower 16 bits.
__device__ inline uint32_t pair_lo(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ inline uint32_t pair_hi(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// f16 values of a pair of codes in bits 0..9 of each half: 1024 + n by the
// bits of 1024, less 1024 + offset (both exact), times the scales (the one
// rounding).
__device__ inline uint32_t pair_value(uint32_t codes, float offset, uint32_t scales) {
    const _Float16 o = static_cast<_Float16>(-(1024.0f + offset));
    return as_word((as_half2(codes | 0x64006400u) + half2_t{o, o}) * as_half2(scales));
}
// The same for codes in bits 4..9: 64 + n by the bits of 64.
__device__ inline uint32_t pair_value_hi(uint32_t codes, float offset, uint32_t scales) {
    const _Float16 o = static_cast<_Float16>(-(64.0f + offset));
    return as_word((as_half2(codes | 0x54005400u) + half2_t{o, o}) * as_half2(scales));
}

// Value operand: lane n of 16 owns VD = D/16 dims of a key's slice.  Rows
// hold consecutive dims of one key and the matrix instruction wants
// consecutive keys of one dim, so a lane reads its dims of 8 keys and pairs
// keys with byte permutes, still in packed codes (a nibble permute moves 8
// elements).  raw(): the keys' words and scales; emit(keep, f): f(t,
// operands of dims t .. t + 3) over the VD dims, keys cleared in `keep` (16 bits a
// key, pairs as the operand's words) as zeros;  dim(n, t): which dim t is.
template <int TYPE, int D> struct ValueOp;

template <int D>
struct ValueOp<KVMEM_TYPE_Q4_0, D> {
    static constexpr int VD = D / 16;
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
    __device__ inline void emit(const u32x4_t &keep, F f) const {
        const u32x4_t ds{d[0] & keep[0], d[1] & keep[1], d[2] & keep[2], d[3] & keep[3]};
#pragma unroll
        for (int i = 0; i < NW; ++i) {
#pragma unroll
            for (int h = 0; h < (NB < 4 ? 1 : 2); ++h) {
                u32x4_t a[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t t = h ? pair_hi(w[2 * j][i], w[2 * j + 1][i]) : pair_lo(w[2 * j][i], w[2 * j + 1][i]);
                    a[0][j] = pair_value(t & 0x000F000Fu, offset, ds[j]);
                    a[1][j] = pair_value_hi(t & 0x00F000F0u, offset, ds[j]);
                    a[2][j] = pair_value((t >> 8) & 0x000F000Fu, offset, ds[j]);
                    a[3][j] = pair_value_hi((t >> 8) & 0x00F000F0u, offset, ds[j]);
                }
                f(8 * i + 4 * h, a);
            }
        }
    }
};

template <int D>
struct ValueOp<KVMEM_TYPE_Q5_0, D> {
    static constexpr int VD = D / 16;
    static constexpr int NB = VD / 2;
    static constexpr int NW = NB < 4 ? 1 : NB / 4;
    static constexpr float offset = 16.0f;
    uint32_t w[8][NW];  // lower four bits, as Q4_0's
    uint32_t h[8];      // fifth bits: of the lower nibbles from bit 0, of the upper from bit 16
    uint32_t d[4];
    __device__ static inline uint32_t dim(uint32_t n, uint32_t t) { return ValueOp<KVMEM_TYPE_Q4_0, D>::dim(n, t); }
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
    __device__ inline void emit(const u32x4_t &keep, F f) const {
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
                    a[0][j] = pair_value((t & 0x000F000Fu) | (((lo[j] >> b0) & 0x00010001u) << 4), offset, ds[j]);
                    a[1][j] = pair_value_hi((t & 0x00F000F0u) | (((hi[j] >> b0) & 0x00010001u) << 8), offset, ds[j]);
                    a[2][j] = pair_value(((t >> 8) & 0x000F000Fu) | (((lo[j] >> (b0 + 1)) & 0x00010001u) << 4), offset,
                                      ds[j]);
                    a[3][j] = pair_value_hi(((t >> 8) & 0x00F000F0u) | (((hi[j] >> (b0 + 1)) & 0x00010001u) << 8), offset,
                                         ds[j]);
                }
                f(8 * i + 4 * q, a);
            }
        }
    }
};

template <int D>
struct ValueOp<KVMEM_TYPE_Q8_0, D> {
    static constexpr int VD = D / 16;
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
    __device__ inline void emit(const u32x4_t &keep, F f) const {
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
                    a[b][j] = pair_value(__builtin_amdgcn_perm(w[2 * j + 1][i], w[2 * j][i], sel), 128.0f, ds[j]);
                }
            }
            f(4 * i, a);
        }
    }
};

template <int D>
struct ValueOp<KVMEM_TYPE_F16, D> {
    static constexpr int VD = D / 16;
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
    __device__ inline void emit(const u32x4_t &keep, F f) const {
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

// The keys of a block of 32 that exist and lie below `limit` (counted from the
// block's first key), for a lane whose element e of the block's operand is key
// 16 (e / 4) + first + e % 4: bit 16 (e / 4) + e % 4.
__device__ inline uint32_t seen_keys(uint32_t have, int32_t limit, uint32_t first) {
    const int32_t left = limit - static_cast<int32_t>(first);
    const uint32_t below = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u;
    return (have >> first) & below;
}

// Operand masks of those keys: 16 bits a key, pairs as the operand's words.
__device__ inline u32x4_t keep_keys(uint32_t seen) {
    u32x4_t keep;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t two = seen >> (16u * (j >> 1) + 2u * (j & 1u));
        keep[j] = (two & 1u) * 0x0000ffffu + ((two >> 1) & 1u) * 0xffff0000u;
    }
    return keep;
}

// A wave's LDS writes become visible to its own later reads, in order.
__device__ inline void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ inline void store_elem(uint8_t *out, int type, uint64_t i, float x) {
    if (type == KVMEM_TYPE_F32) {
        reinterpret_cast<float *>(out)[i] = x;
    } else if (type == KVMEM_TYPE_F16) {
        reinterpret_cast<_Float16 *>(out)[i] = static_cast<_Float16>(x);
    } else {
        reinterpret_cast<__bf16 *>(out)[i] = static_cast<__bf16>(x);
    }
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

// Walsh-Hadamard rotation of an output element (dim d of a row, one thread per
// dim, every thread of the workgroup calls): butterflies of span 1 .. width/2
// through LDS.
__device__ inline float rotate_back(float x, uint32_t width, uint32_t d, float *row) {
    x *= 1.0f / sqrtf(static_cast<float>(width));
    for (uint32_t s = 1; s < width; s <<= 1) {
        __syncthreads();
        row[d] = x;
        __syncthreads();
        const float y = row[d ^ s];
        x = (d & s) ? y - x : x + y;
    }
    return x;
}

// ------------------------------------------------------------ few queries

// Keys of a wave's step: about the same bytes for every head size (9 KiB of
// q4_0 keys and values), enough in flight per compute unit to stream.
template <int D>
constexpr uint32_t decode_keys() { return 32u * (256 / D); }

template <int TK, int TV, int D>
constexpr uint32_t decode_wave_bytes() {
    return decode_keys<D>() * (Slice<TK, D>::stride + Slice<TV, D>::stride + (KeyOp<TK>::codes ? D / 16 : 0));
}

// Rows of one KV head's queries over one part of a request's keys: up to 16
// (token, head) rows, keys split over the workgroup's four waves.  Scores are
// held transposed (keys by rows) so that a lane owns one query row: S^T = K Q^T,
// O^T = V^T P^T, and a lane's weights of S^T are its operand of the second
// product as they stand.
// Two waves per SIMD, but for 16-bit rows of 256: their step's rows take half the
// registers, and one wave has as many bytes in flight.
constexpr int decode_occupancy(int tk, int tv, int d) {
    return d == 256 && (tk == KVMEM_TYPE_F16 || tv == KVMEM_TYPE_F16) ? 1 : 2;
}

template <int TK, int TV, int D>
__global__ __launch_bounds__(256, decode_occupancy(TK, TV, D)) void attn_decode_kernel(AttnParams p) {
    using SK = Slice<TK, D>;
    using SV = Slice<TV, D>;
    using KO = KeyOp<TK>;
    using VO = ValueOp<TV, D>;
    constexpr int NG = D / 32;
    constexpr int VD = D / 16;
    constexpr uint32_t KT = decode_keys<D>();
    constexpr int NT = KT / 16;  // key tiles of a step
    constexpr uint32_t NC = KT > 64 ? KT / 64 : 1;  // keys a lane finds the cells of
    constexpr uint32_t NLK = (KT + SK::per_load - 1) / SK::per_load;  // loads of a step
    constexpr uint32_t NLV = (KT + SV::per_load - 1) / SV::per_load;
    typedef typename UnitOf<SK::unit>::type UK;
    typedef typename UnitOf<SV::unit>::type UV;
    typedef uint16_t scales_t __attribute__((ext_vector_type(NG)));
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float2 wave_ml[kWaves][kRowTile];

    const uint32_t unit = blockIdx.x % p.units;
    const uint32_t y = blockIdx.x / p.units;
    const uint32_t s = unit / p.n_parts;
    const uint32_t part = unit - s * p.n_parts;
    if (s >= p.n_seq) {
        return;
    }
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
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t nl = lane & 15u;   // query row; dim lane of the values
    const uint32_t c = lane >> 4;     // chunk of the contraction
    const uint32_t c0 = part * p.chunk;
    const uint32_t c1 = min(n, c0 + p.chunk);
    const uint8_t *k_head = p.k + static_cast<uint64_t>(hk) * SK::bytes;
    const uint8_t *v_head = p.v + static_cast<uint64_t>(hk) * SV::bytes;
    const uint32_t *table = p.table + static_cast<uint64_t>(s) * p.table_stride;

    // The cells of this lane's keys of the step at j0, and which keys exist
    // (bit = key); one that does not has cell 0, and is masked where it matters.
    struct Cells {
        uint32_t at[NC];
        uint64_t have[NC];
    };
    auto cells_of = [&](uint32_t j0) {
        Cells r;
#pragma unroll
        for (uint32_t i = 0; i < NC; ++i) {
            const uint32_t j = j0 + (lane & (KT - 1u)) + 64u * i;
            uint32_t slot = KVMEM_HIP_NO_SLOT;
            const uint32_t b = j / p.T;
            if (j < c1) {
                slot = table[b];
            }
            r.at[i] = slot < p.n_slots ? slot * p.T + (j - b * p.T) : 0u;
            r.have[i] = __ballot(slot < p.n_slots);
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
    constexpr uint32_t step = kWaves * KT;
    uint32_t j0 = c0 + wave * KT;
    Cells cells = cells_of(j0);

    // up to 8 rows: each stands in two columns, for the upper and the lower
    // digits of its weights
    const bool twice = rows <= 8u;
    const uint32_t my_row = row0 + min(twice ? (nl & 7u) : nl, rows - 1u);
    const uint32_t my_tok = my_row / p.group;
    const uint32_t my_head = hk * p.group + (my_row - my_tok * p.group);
    const uint32_t limit = key_limit(p, r, my_tok);

    // The row's queries, scaled into f16's range.  Codes carry an offset: the
    // sum of a group's queries times it comes off each score, as one more product
    // of the groups' scales with those sums (in three f16 pieces, 33 bits).
    half8_t qf[NG];
    half8_t q_off;
    float fac;
    {
        const uint8_t *q = p.q + static_cast<uint64_t>(r.first + my_tok) * p.q_nb2 + my_head * p.q_nb1;
        u32x4_t x[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            x[g] = load_query<KO>(q, g, c);
        }
        load_tile(cells);
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
            // piece c of the sum stands in chunk c of the contraction
            const _Float16 pick[3] = {static_cast<_Float16>(c == 0 ? 1.0f : 0.0f),
                                      static_cast<_Float16>(c == 1 ? 1.0f : 0.0f),
                                      static_cast<_Float16>(c == 2 ? 1.0f : 0.0f)};
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float all = 0.0f;
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    all += static_cast<float>(qf[g][e]);
                    qf[g][e] *= static_cast<_Float16>(1.0f / KO::times(e));
                }
                all += lane_xor16(all);
                all += lane_xor32(all);
                all *= -KO::offset * 0x1p-10f;
                const _Float16 hi = static_cast<_Float16>(all);
                const float left = all - static_cast<float>(hi);
                const _Float16 mid = static_cast<_Float16>(left);
                const _Float16 lo = static_cast<_Float16>(left - static_cast<float>(mid));
                q_off[g] = hi * pick[0] + mid * pick[1] + lo * pick[2];
            }
        }
        fac = ldexpf(p.scale * kLog2e, (KO::codes ? 24 : 0) - ex);
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

    Cells next = cells_of(j0 + step);
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
        cells = next;
        load_tile(cells);
        next = cells_of(j0 + 2u * step);
        if constexpr (KO::codes) {
            // a key's scales side by side
            for (uint32_t key = lane % KT; key < KT; key += 64u) {
                constexpr uint32_t per = KT < 64u ? NG * KT / 64u : NG;  // groups of a lane
                const uint32_t g0 = KT < 64u ? lane / KT * per : 0u;
#pragma unroll
                for (uint32_t g = 0; g < per; ++g) {
                    reinterpret_cast<uint16_t *>(ks + key)[g0 + g] =
                        static_cast<uint16_t>(lds_half(kt + key * SK::stride + (g0 + g) * SK::GB));
                }
            }
            wave_lds_sync();
        }
        float x[NT][4];
#pragma unroll
        for (uint32_t a = 0; a < NT; ++a) {
            const uint8_t *kr = kt + (16u * a + nl) * SK::stride;
            float4_t sc{0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (KO::codes) {
                half8_t kd;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    kd[e] = 0;
                }
                const scales_t mine = ks[16u * a + nl];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    kd[g] = __builtin_bit_cast(_Float16, static_cast<uint16_t>(mine[g]));
                }
                sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kd, q_off, sc, 0, 0, 0);
                sc *= 0x1p-14f;
                scales_t d[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    d[i] = ks[16u * a + 4u * c + i];
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const half8_t kf = __builtin_bit_cast(half8_t, load_key<KO, SK::GB>(kr, g, c));
                    const float4_t acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        kf, qf[g], float4_t{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sc[i] = __builtin_fmaf(
                            static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(d[i][g]))), acc[i],
                            sc[i]);
                    }
                }
            } else {
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const half8_t kf = __builtin_bit_cast(half8_t, load_key<KO, SK::GB>(kr, g, c));
                    sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[g], sc, 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[a][i] = sc[i] * fac;
            }
        }
        const bool split = j0 + KT > n_all && tok0 != tok1;  // some rows do not attend all these keys
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
            const float higher = fmaxf(top, most);
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
            // A zero weight would still hand a row a NaN or infinity: keys that do
            // not exist are cleared, and where some rows do not attend all the
            // others, each token's rows take the product with their later keys
            // cleared.
            for (uint32_t tk = split ? tok0 : tok1; tk <= tok1; ++tk) {
                wave_lds_sync();  // the values are read (and unpacked) once a pass, not kept for all
                VO vo;
                vo.raw(nl, [&](uint32_t e) {
                    return vt + (32u * h + 16u * (e >> 2) + 4u * c + (e & 3u)) * SV::stride;
                });
                u32x4_t keep{~0u, ~0u, ~0u, ~0u};
                if (split || !whole) {
                    keep = keep_keys(seen_keys(
                        static_cast<uint32_t>(now.have[h >> 1] >> (32u * (h & 1u))),
                        static_cast<int32_t>(key_limit(p, r, tk) - j0) - static_cast<int32_t>(32u * h), 4u * c));
                }
                vo.emit(keep, [&](int t0, const u32x4_t *a) {
                    if (split) {
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            const float4_t y = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                __builtin_bit_cast(half8_t, a[t]), w[h], o[t0 + t], 0, 0, 0);
                            o[t0 + t] = my_tok == tk ? y : o[t0 + t];
                        }
                    } else {
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            o[t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a[t]), w[h],
                                                                               o[t0 + t], 0, 0, 0);
                        }
                    }
                });
            }
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
#pragma unroll
        for (int t = 0; t < VD; ++t) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                ow[nl * D + VO::dim(4u * c + i, t)] = o[t][i] * fade;
            }
        }
    }
    __syncthreads();
    const float *ol = reinterpret_cast<const float *>(lds);
    const bool last = n_parts == 1;
    float *turn = reinterpret_cast<float *>(lds);
    for (uint32_t e0 = 0; e0 < rows * D; e0 += 256u) {
        const uint32_t e = e0 + threadIdx.x;
        const bool in = e < rows * D;
        const uint32_t row = min(e / D, rows - 1u);
        const uint32_t d = e & (D - 1u);
        const uint32_t tok = (row0 + row) / p.group;
        const uint32_t head = hk * p.group + (row0 + row - tok * p.group);
        const uint64_t at = static_cast<uint64_t>(r.first + tok) * p.n_head + head;
        float total = 0.0f, mx = -INFINITY, x = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            mx = fmaxf(mx, wave_ml[w][row].x);
        }
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            const float2 ml = wave_ml[w][row];
            total += ml.x == -INFINITY ? 0.0f * ml.y : ml.y * __builtin_amdgcn_exp2f(ml.x - mx);
            x += in ? ol[w * rows * D + e] : 0.0f;
        }
        if (!last) {
            if (in) {
                const uint64_t pe = (static_cast<uint64_t>(part) * p.n_tokens * p.n_head) + at;
                p.part_o[pe * D + d] = x;
                if (d == 0) {
                    p.part_ml[pe] = make_float2(mx, total);
                }
            }
            continue;
        }
        x = total == 0.0f ? 0.0f : x / total;
        if (p.hadamard) {
            // this round's own 256 elements of the LDS rows (read above by these threads only)
            x = rotate_back(x, p.hadamard, e & (p.hadamard - 1u), turn + (e - (e & (p.hadamard - 1u))));
        }
        if (in) {
            store_elem(p.out, p.out_type, at * D + d, x);
            if (d == 0 && p.lse) {
                p.lse[at] = total == 0.0f ? -INFINITY : (mx - kWeightShift) / kLog2e + logf(total);
            }
        }
    }
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
            r[j] = KO::times(2 * j) == 1.0f ? pair_value(codes[j], KO::offset, scale)
                                            : pair_value_hi(codes[j], KO::offset, scale);
        }
        return r;
    }
}

// ------------------------------------------------------------ many queries

constexpr uint32_t kPrefillRows = 128;  // rows of a workgroup, 32 a wave
typedef float float16_t __attribute__((ext_vector_type(16)));

template <int TK, int TV, int D>
constexpr uint32_t prefill_bytes() {
    return kTileKeys * (Slice<TK, D>::bytes + Slice<TV, D>::bytes)  // the rows as cached
           + kTileKeys * (2 * D + 16)                               // keys as f16
           + kTileKeys * 2 * D;                                     // values as f16
}

// 128 rows of one KV head's queries over one part of a request's keys: steps
// of 32 keys, made f16 once for the workgroup in LDS, each wave multiplying
// its 32 rows (transposed products as in the decode kernel, on 32x32 tiles).
template <int TK, int TV, int D>
__global__ __launch_bounds__(256) void attn_prefill_kernel(AttnParams p) {
    using SK = Slice<TK, D>;
    using SV = Slice<TV, D>;
    using KO = KeyOp<TK>;
    using VO = ValueOp<TV, D>;
    constexpr int NB = D / 32;
    constexpr uint32_t NK = (kTileKeys * SK::units + 255u) / 256u;
    constexpr uint32_t NV = (kTileKeys * SV::units + 255u) / 256u;
    typedef typename UnitOf<SK::unit>::type UK;
    typedef typename UnitOf<SV::unit>::type UV;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];

    const uint32_t unit = blockIdx.x % p.units;
    const uint32_t tile = p.row_tiles - 1u - blockIdx.x / p.units;  // long rows first
    const uint32_t hk = unit % p.n_head_kv;
    const uint32_t sp = unit / p.n_head_kv;
    const uint32_t s = sp / p.n_parts;
    const uint32_t part = sp - s * p.n_parts;
    if (s >= p.n_seq) {
        return;
    }
    const Span r = request_span(p, s);
    const uint32_t m = min(r.m, p.max_q);
    const uint32_t row0 = tile * kPrefillRows;
    if (row0 >= m * p.group) {
        return;
    }
    const uint32_t rows = min(kPrefillRows, m * p.group - row0);
    const uint32_t n = key_limit(p, r, (row0 + rows - 1u) / p.group);
    const uint32_t n_all = key_limit(p, r, row0 / p.group);
    const uint32_t n_parts = max(1u, (n + p.chunk - 1u) / p.chunk);
    if (part >= n_parts) {
        return;
    }
    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t nl = lane & 31u;  // query row of the wave
    const uint32_t hh = lane >> 5;   // half of the contraction
    const uint32_t in_tile = wave * 32u + nl;
    const uint32_t my_row = row0 + min(in_tile, rows - 1u);
    const uint32_t my_tok = my_row / p.group;
    const uint32_t my_head = hk * p.group + (my_row - my_tok * p.group);
    const uint32_t limit = key_limit(p, r, my_tok);
    const uint32_t tok0 = (row0 + min(wave * 32u, rows - 1u)) / p.group;
    const uint32_t tok1 = (row0 + min(wave * 32u + 31u, rows - 1u)) / p.group;

    half8_t qf[D / 16];
    float fac;
    {
        const uint8_t *q = p.q + static_cast<uint64_t>(r.first + my_tok) * p.q_nb2 + my_head * p.q_nb1;
        u32x4_t x[D / 16];
#pragma unroll
        for (uint32_t st = 0; st < D / 16; ++st) {
            x[st] = load_query<KO>(q, st >> 1, 2u * (st & 1u) + hh);
        }
        uint32_t bits = 0;
#pragma unroll
        for (uint32_t st = 0; st < D / 16; ++st) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bits = max_magnitude(x[st][i], bits);
            }
        }
        bits = max(bits & 0xffffu, bits >> 16);
        float most = p.q_bf16 ? query_value<true>(bits) : query_value<false>(bits);
        most = fmaxf(most, lane_xor32(most));
        const int ex = query_shift(most);
        const float up = ldexpf(1.0f, ex);
        if (p.q_bf16) {
#pragma unroll
            for (uint32_t st = 0; st < D / 16; ++st) {
                qf[st] = query_operand<KO, true>(x[st], up);
            }
        } else {
#pragma unroll
            for (uint32_t st = 0; st < D / 16; ++st) {
                qf[st] = query_operand<KO, false>(x[st], up);
            }
        }
        fac = ldexpf(p.scale * kLog2e, -ex);
    }

    uint8_t *raw_k = lds;
    uint8_t *raw_v = raw_k + kTileKeys * SK::bytes;
    uint8_t *kt = raw_v + kTileKeys * SV::bytes;    // [key][D] f16, rows padded by 16 bytes
    uint8_t *vt = kt + kTileKeys * (2 * D + 16);    // [octet of keys][D] operands of 8 f16

    const uint32_t c0 = part * p.chunk;
    const uint32_t c1 = min(n, c0 + p.chunk);
    const uint8_t *k_head = p.k + static_cast<uint64_t>(hk) * SK::bytes;
    const uint8_t *v_head = p.v + static_cast<uint64_t>(hk) * SV::bytes;
    const uint32_t *table = p.table + static_cast<uint64_t>(s) * p.table_stride;

    auto cell_of = [&](uint32_t j0) {
        const uint32_t j = j0 + nl;
        if (j >= c1) {
            return kNoCell;
        }
        const uint32_t b = j / p.T;
        const uint32_t slot = table[b];
        return slot < p.n_slots ? slot * p.T + (j - b * p.T) : kNoCell;
    };
    UK rk[NK];
    UV rv[NV];
    auto load_tile = [&](uint32_t cell) {
#pragma unroll
        for (uint32_t i = 0; i < NK; ++i) {
            const uint32_t u = i * 256u + tid;
            const uint32_t key = u / SK::units;
            const uint32_t at = __shfl(cell, key & 31u, 64);
            rk[i] = UK{};
            if (key < kTileKeys && at != kNoCell) {
                rk[i] = *reinterpret_cast<const UK *>(k_head + static_cast<uint64_t>(at) * p.row_k +
                                                      (u - key * SK::units) * SK::unit);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i) {
            const uint32_t u = i * 256u + tid;
            const uint32_t key = u / SV::units;
            const uint32_t at = __shfl(cell, key & 31u, 64);
            rv[i] = UV{};
            if (key < kTileKeys && at != kNoCell) {
                rv[i] = *reinterpret_cast<const UV *>(v_head + static_cast<uint64_t>(at) * p.row_v +
                                                      (u - key * SV::units) * SV::unit);
            }
        }
    };

    float top = -INFINITY;
    float sum = 0.0f;
    float16_t o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            o[b][i] = 0.0f;
        }
    }

    uint32_t cell = cell_of(c0);
    load_tile(cell);
    uint32_t next = cell_of(c0 + kTileKeys);
    for (uint32_t j0 = c0; j0 < c1; j0 += kTileKeys) {
        const uint32_t have = static_cast<uint32_t>(__ballot(cell != kNoCell));
#pragma unroll
        for (uint32_t i = 0; i < NK; ++i) {
            const uint32_t u = i * 256u + tid;
            if (u < kTileKeys * SK::units) {
                *reinterpret_cast<UK *>(raw_k + u * SK::unit) = rk[i];
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i) {
            const uint32_t u = i * 256u + tid;
            if (u < kTileKeys * SV::units) {
                *reinterpret_cast<UV *>(raw_v + u * SV::unit) = rv[i];
            }
        }
        __syncthreads();  // rows in place; the last step's operands are used
        cell = next;
        load_tile(cell);
        next = cell_of(j0 + 2u * kTileKeys);
        // keys: a thread makes 8 dims of a key
        for (uint32_t u = tid; u < kTileKeys * (D / 8); u += 256u) {
            const uint32_t key = u / (D / 8);
            const uint32_t oct = u - key * (D / 8);
            const uint8_t *g = raw_k + key * SK::bytes + (oct >> 2) * SK::GB;
            uint32_t scale = 0;
            if constexpr (KO::codes) {
                scale = lds_half(g) * 0x00010001u;
            }
            *reinterpret_cast<u32x4_t *>(kt + key * (2 * D + 16) + oct * 16u) =
                key_values<KO>((oct & 4u) ? KO::template load<false>(g, oct & 3u) : KO::template load<true>(g, oct & 3u), scale);
        }
        // values: a thread makes 8 keys of D/16 dims; octet q holds keys
        // 16 (q / 2) + 8 (e / 4) + 4 (q % 2) + e % 4, as a lane of the scores does
        const bool partial = j0 + kTileKeys > n_all;
        uint32_t bad = 0;
        if (tid < 16u * (kTileKeys / 8u)) {
            const uint32_t q = tid >> 4;
            const uint32_t dl = tid & 15u;
            VO vo;
            vo.raw(dl, [&](uint32_t e) {
                return raw_v + (16u * (q >> 1) + 8u * (e >> 2) + 4u * (q & 1u) + (e & 3u)) * SV::bytes;
            });
            vo.emit(u32x4_t{~0u, ~0u, ~0u, ~0u}, [&](int t0, const u32x4_t *a) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    *reinterpret_cast<u32x4_t *>(vt + (q * D + VO::dim(dl, t0 + t)) * 16u) = a[t];
                    if (partial) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            bad |= ((a[t][j] & 0x7C00u) == 0x7C00u) | ((a[t][j] & 0x7C000000u) == 0x7C000000u);
                        }
                    }
                }
            });
        }
        bool clear = false;
        if (partial) {
            clear = __syncthreads_or(bad);
        } else {
            __syncthreads();
        }

        float16_t sc;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            sc[i] = 0.0f;
        }
        const uint8_t *kr = kt + nl * (2 * D + 16) + hh * 16u;
#pragma unroll
        for (int st = 0; st < D / 16; ++st) {
            const half8_t kf = *reinterpret_cast<const half8_t *>(kr + st * 32);
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[st], sc, 0, 0, 0);
        }
        float most = -INFINITY;
        if (have != 0xffffffffu || partial) {
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
                const uint32_t key = 8u * (i >> 2) + 4u * hh + (i & 3u);
                sc[i] = ((have >> key) & 1u) && j0 + key < limit ? sc[i] * fac : -INFINITY;
                most = fmaxf(most, sc[i]);
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
                sc[i] *= fac;
                most = fmaxf(most, sc[i]);
            }
        }
        most = fmaxf(most, lane_xor32(most));
        if (__any(most > top + kTopSlack)) {
            const float now = fmaxf(top, most);
            const float fade = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - now);
            sum *= fade;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                o[b] *= fade;
            }
            top = now;
        }
        const float base = (top == -INFINITY ? 0.0f : top) - kWeightShift;
        half8_t w[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float pe = __builtin_amdgcn_exp2f(sc[i] - base);
            sum += pe;
            w[i >> 3][i & 7] = static_cast<_Float16>(pe);
        }
        const uint8_t *vr = vt + (hh * D + nl) * 16u;
        if (!clear) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const half8_t vf = *reinterpret_cast<const half8_t *>(vr + (2 * ks * D + 32 * b) * 16);
                    o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, w[ks], o[b], 0, 0, 0);
                }
            }
        } else {
            // a NaN or infinity among values that some rows do not attend: each
            // token's rows take the product with its own later keys cleared
            for (uint32_t tk = tok0; tk <= tok1; ++tk) {
                const uint32_t lim = key_limit(p, r, tk);
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    u32x4_t keep;
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint32_t key = j0 + 16u * ks + 8u * (j >> 1) + 4u * hh + 2u * (j & 1u);
                        keep[j] = (key < lim ? 0x0000ffffu : 0u) | (key + 1u < lim ? 0xffff0000u : 0u);
                    }
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const u32x4_t vf = *reinterpret_cast<const u32x4_t *>(vr + (2 * ks * D + 32 * b) * 16);
                        const float16_t x = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                            __builtin_bit_cast(half8_t, vf & keep), w[ks], o[b], 0, 0, 0);
                        o[b] = my_tok == tk ? x : o[b];
                    }
                }
            }
        }
    }

    sum += lane_xor32(sum);
    const uint64_t at = static_cast<uint64_t>(r.first + my_tok) * p.n_head + my_head;
    const bool mine = in_tile < rows;
    // a lane holds dims 32 b + 8 (i / 4) + 4 hh + i % 4 of its row
    if (n_parts > 1) {
        if (mine) {
            const uint64_t pe = static_cast<uint64_t>(part) * p.n_tokens * p.n_head + at;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    *reinterpret_cast<float4_t *>(p.part_o + pe * D + 32 * b + 2 * i + 4 * hh) =
                        float4_t{o[b][i], o[b][i + 1], o[b][i + 2], o[b][i + 3]};
                }
            }
            if (hh == 0) {
                p.part_ml[pe] = make_float2(top, sum);
            }
        }
        return;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        o[b] *= inv;
    }
    if (p.hadamard) {
        // spans 1, 2, 8, 16 inside a block's registers, 4 with lane ^ 32, 32 and up between blocks
        const float f = 1.0f / sqrtf(static_cast<float>(p.hadamard));
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            o[b] *= f;
#pragma unroll
            for (int sp = 1; sp < 16; sp <<= 1) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (!(i & sp)) {
                        const float u = o[b][i];
                        const float v = o[b][i + sp];
                        o[b][i] = u + v;
                        o[b][i + sp] = u - v;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float v = lane_xor32(o[b][i]);
                o[b][i] = hh ? v - o[b][i] : o[b][i] + v;
            }
        }
#pragma unroll
        for (int sp = 1; sp < NB; sp <<= 1) {
            if (32u * sp < p.hadamard) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (!(b & sp)) {
                        const float16_t u = o[b];
                        const float16_t v = o[b + sp];
                        o[b] = u + v;
                        o[b + sp] = u - v;
                    }
                }
            }
        }
    }
    if (mine) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const uint64_t e = at * D + 32 * b + 2 * i + 4 * hh;
                if (p.out_type == KVMEM_TYPE_F32) {
                    *reinterpret_cast<float4_t *>(p.out + 4 * e) =
                        float4_t{o[b][i], o[b][i + 1], o[b][i + 2], o[b][i + 3]};
                } else if (p.out_type == KVMEM_TYPE_F16) {
                    *reinterpret_cast<half4_t *>(p.out + 2 * e) =
                        half4_t{static_cast<_Float16>(o[b][i]), static_cast<_Float16>(o[b][i + 1]),
                                static_cast<_Float16>(o[b][i + 2]), static_cast<_Float16>(o[b][i + 3])};
                } else {
                    typedef __bf16 bf4_t __attribute__((ext_vector_type(4)));
                    *reinterpret_cast<bf4_t *>(p.out + 2 * e) =
                        bf4_t{static_cast<__bf16>(o[b][i]), static_cast<__bf16>(o[b][i + 1]),
                              static_cast<__bf16>(o[b][i + 2]), static_cast<__bf16>(o[b][i + 3])};
                }
            }
        }
        if (hh == 0 && p.lse) {
            p.lse[at] = sum == 0.0f ? -INFINITY : (top - kWeightShift) / kLog2e + logf(sum);
        }
    }
}

// ------------------------------------------------------------- joining parts

// One workgroup per (token, head): the parts' sums, each weighted by its
// maximum.  Each wave adds the parts k = wave, wave + 4, ... in order, a lane its
// D/64 dims, then the waves' sums are added in order.
template <int D>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnParams p) {
    constexpr int E = D / 64;
    typedef float dims_t __attribute__((ext_vector_type(E)));
    __shared__ float sums[kWaves][D];
    __shared__ float turn[256];
    const uint32_t h = blockIdx.x % p.n_head;
    const uint32_t tok = blockIdx.x / p.n_head;
    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the request this token belongs to
    uint32_t s = tok;
    if (p.q_start) {
        uint32_t lo = 0, hi = p.n_seq;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (p.q_start[mid] <= tok) {
                lo = mid;
            } else {
                hi = mid;
            }
        }
        s = lo;
    }
    if (s >= p.n_seq) {
        return;
    }
    const Span r = request_span(p, s);
    if (tok < r.first || tok - r.first >= min(r.m, p.max_q)) {
        return;
    }
    const uint32_t i = tok - r.first;
    // the part count of the row tile this row was in
    const uint32_t row = i * p.group + h % p.group;
    const uint32_t row0 = row / p.row_tile * p.row_tile;
    const uint32_t rows = min(p.row_tile, min(r.m, p.max_q) * p.group - row0);
    const uint32_t n = key_limit(p, r, (row0 + rows - 1u) / p.group);
    const uint32_t n_parts = (n + p.chunk - 1u) / p.chunk;
    if (n_parts <= 1) {
        return;
    }
    const uint64_t at = static_cast<uint64_t>(tok) * p.n_head + h;
    const uint64_t stride = static_cast<uint64_t>(p.n_tokens) * p.n_head;
    float top = -INFINITY;
    for (uint32_t k = lane; k < n_parts; k += 64u) {
        top = fmaxf(top, p.part_ml[k * stride + at].x);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        top = fmaxf(top, __shfl_xor(top, d, 64));
    }
    const float *po = p.part_o + at * D + lane * E;
    float total = 0.0f;
    dims_t x = {};
#pragma unroll 8
    for (uint32_t k = wave; k < n_parts; k += kWaves) {
        const float2 ml = p.part_ml[k * stride + at];
        const float f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - top);
        total += ml.y * f;
        x += *reinterpret_cast<const dims_t *>(po + k * stride * D) * f;
    }
    *reinterpret_cast<dims_t *>(&sums[wave][lane * E]) = x;
    if (lane == 0) {
        turn[wave] = total;
    }
    __syncthreads();
    total = (turn[0] + turn[1]) + (turn[2] + turn[3]);
    const uint32_t d = tid & (D - 1u);  // D < 256: more than one thread a dim, the first one stores
    float y = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
    y = total == 0.0f ? 0.0f : y / total;
    if (p.hadamard) {
        y = rotate_back(y, p.hadamard, tid & (p.hadamard - 1u), turn + (tid - (tid & (p.hadamard - 1u))));
    }
    if (tid < D) {
        store_elem(p.out, p.out_type, at * D + d, y);
    }
    if (tid == 0 && p.lse) {
        p.lse[at] = total == 0.0f ? -INFINITY : (top - kWeightShift) / kLog2e + logf(total);
    }
}

// How a call is laid out on the chip.
struct AttnPlan {
    bool prefill;
    uint32_t row_tile, row_tiles, chunk, n_parts, units;
    uint64_t grid;
    size_t o_bytes, ml_bytes;  // workspace: sums, then maxima and weights
};

// Query rows of a request above which the prefill kernel takes the call.
constexpr uint32_t kDecodeRows = 16;
// Workgroups a launch is split up to.
constexpr uint32_t kDecodeGroups = 512;
constexpr uint32_t kPrefillGroups = 512;

static AttnPlan plan_attention(const kvmem_hip_pool *pool, const kvmem_hip_attn_args *a) {
    AttnPlan pl{};
    const uint32_t max_q = a->q_start ? std::min(a->max_q, a->n_tokens) : 1u;
    const uint32_t group = a->n_head / a->n_head_kv;
    const uint64_t rows = static_cast<uint64_t>(max_q) * group;
    pl.prefill = rows > kDecodeRows;
    pl.row_tile = pl.prefill ? kPrefillRows : kRowTile;
    pl.row_tiles = static_cast<uint32_t>((rows + pl.row_tile - 1) / pl.row_tile);
    const uint32_t quantum = pl.prefill ? kTileKeys : 32u * (256u / a->head_dim) * kWaves;
    const uint64_t room = static_cast<uint64_t>(a->table_stride) * pool->block_tokens;
    const uint64_t keys = std::max<uint64_t>(1, std::min<uint64_t>(a->max_kv, room));
    const uint64_t groups = static_cast<uint64_t>(a->n_seq) * a->n_head_kv * pl.row_tiles;
    const uint64_t want = pl.prefill ? kPrefillGroups : kDecodeGroups;
    uint64_t parts = std::max<uint64_t>(1, want / groups);
    parts = std::min<uint64_t>(parts, (keys + quantum - 1) / quantum);
    uint64_t chunk = (keys + parts - 1) / parts;
    chunk = (chunk + quantum - 1) / quantum * quantum;
    pl.chunk = static_cast<uint32_t>(chunk);
    pl.n_parts = static_cast<uint32_t>((keys + chunk - 1) / chunk);
    const uint64_t units = (static_cast<uint64_t>(a->n_seq) * pl.n_parts * (pl.prefill ? a->n_head_kv : 1u) + 7) / 8 * 8;
    pl.units = static_cast<uint32_t>(units);
    pl.grid = units * pl.row_tiles * (pl.prefill ? 1u : a->n_head_kv);
    if (pl.n_parts > 1) {
        const size_t heads = static_cast<size_t>(a->n_tokens) * a->n_head * pl.n_parts;
        pl.o_bytes = heads * a->head_dim * sizeof(float);
        pl.ml_bytes = heads * sizeof(float2);
    }
    return pl;
}

template <int TK, int TV, int D>
static void launch_attention(hipStream_t stream, const AttnPlan &pl, const AttnParams &p) {
    if (pl.prefill) {
        attn_prefill_kernel<TK, TV, D><<<static_cast<uint32_t>(pl.grid), 256, prefill_bytes<TK, TV, D>(), stream>>>(p);
    } else {
        const uint32_t rows = std::min(kRowTile, p.max_q * p.group);
        // 16 bytes behind the last slice: its last word is read with the next one
        const uint32_t lds = std::max<uint32_t>(kWaves * decode_wave_bytes<TK, TV, D>() + 16u,
                                                std::max<uint32_t>(kWaves * rows * D * 4u, 1024u));
        attn_decode_kernel<TK, TV, D><<<static_cast<uint32_t>(pl.grid), 256, lds, stream>>>(p);
    }
    if (pl.n_parts > 1) {
        attn_join_kernel<D><<<p.n_tokens * p.n_head, 256, 0, stream>>>(p);
    }
}

template <int TK, int TV>
static void launch_attention_d(hipStream_t stream, uint32_t d, const AttnPlan &pl, const AttnParams &p) {
    if (d == 64) {
        launch_attention<TK, TV, 64>(stream, pl, p);
    } else if (d == 128) {
        launch_attention<TK, TV, 128>(stream, pl, p);
    } else {
        launch_attention<TK, TV, 256>(stream, pl, p);
    }
}

template <int TK>
static void launch_attention_v(hipStream_t stream, int tv, uint32_t d, const AttnPlan &pl, const AttnParams &p) {
    switch (tv) {
        case KVMEM_TYPE_Q4_0: launch_attention_d<TK, KVMEM_TYPE_Q4_0>(stream, d, pl, p); break;
        case KVMEM_TYPE_Q5_0: launch_attention_d<TK, KVMEM_TYPE_Q5_0>(stream, d, pl, p); break;
        case KVMEM_TYPE_Q8_0: launch_attention_d<TK, KVMEM_TYPE_Q8_0>(stream, d, pl, p); break;
        default: launch_attention_d<TK, KVMEM_TYPE_F16>(stream, d, pl, p); break;
    }
}

bool load_attention_kernels() {
    return load_kernel_object(&attn_join_kernel<64>);
}

static bool cache_type(int t) {
    return t == KVMEM_TYPE_Q4_0 || t == KVMEM_TYPE_Q5_0 || t == KVMEM_TYPE_Q8_0 || t == KVMEM_TYPE_F16;
}

// nullptr, or what is wrong with a call's arguments (code receives the status).
static const char *check_attention(const kvmem_hip_pool *pool, const kvmem_hip_attn_args *a, int &code) {
    code = KVMEM_HIP_ERR_INVALID;
    if (!pool || !a) {
        return "attention: null arguments";
    }
    const uint32_t D = a->head_dim;
    if (a->n_seq == 0 || a->n_tokens == 0 || a->max_q == 0) {
        return nullptr;  // nothing to attend: no array is looked at
    }
    if (a->n_head == 0 || a->n_head_kv == 0 || a->n_head % a->n_head_kv != 0 || a->n_head > 4096) {
        return "attention: n_head must be a multiple of n_head_kv, at most 4096";
    }
    if (!a->q || !a->out || !a->kv_len || !a->table || a->table_stride == 0) {
        return "attention: null array";
    }
    if (!a->q_start && a->n_seq > a->n_tokens) {
        return "attention: fewer tokens than requests";
    }
    if ((reinterpret_cast<uintptr_t>(a->q) | a->q_nb1 | a->q_nb2 | reinterpret_cast<uintptr_t>(a->out)) & 15u) {
        return "attention: q, its strides and out must be 16-byte aligned";
    }
    if ((reinterpret_cast<uintptr_t>(a->q_start) | reinterpret_cast<uintptr_t>(a->kv_len) |
         reinterpret_cast<uintptr_t>(a->table) | reinterpret_cast<uintptr_t>(a->lse)) & 3u) {
        return "attention: arrays must be 4-byte aligned";
    }
    if (a->n_seq > 65535u || static_cast<uint64_t>(a->n_tokens) * a->n_head > (1u << 23) || a->max_kv > 0x7fffffffu) {
        return "attention: at most 65535 requests, 2^23 (token, head) rows and 2^31 keys";
    }
    if (!(a->scale >= 0.0f) || std::isinf(a->scale)) {
        return "attention: scale must be finite and not negative";
    }
    if (pool->block_tokens == 0 || pool->n_slots == 0 || static_cast<uint64_t>(pool->n_slots) * pool->block_tokens > 0x7fffffffu) {
        return "attention: the pool's rows must fit 31 bits";
    }
    if (pool->n_embd_k != static_cast<uint64_t>(a->n_head_kv) * D || pool->n_embd_v != pool->n_embd_k) {
        return "attention: the pool's rows have another width";
    }
    const kvmem_hip_transform *xf = pool->xf;
    if (xf && xf->hadamard_v &&
        (xf->head_dim != D || (xf->hadamard_v & (xf->hadamard_v - 1)) || xf->hadamard_v < 64 || xf->hadamard_v > D)) {
        return "attention: hadamard_v must be a power of two from 64 to head_dim";
    }
    code = KVMEM_HIP_ERR_UNSUPPORTED;
    if (D != 64 && D != 128 && D != 256) {
        return "attention: head_dim must be 64, 128 or 256";
    }
    if (a->q_type != KVMEM_TYPE_F16 && a->q_type != KVMEM_TYPE_BF16) {
        return "attention: queries must be F16 or BF16";
    }
    if (a->out_type != KVMEM_TYPE_F32 && a->out_type != KVMEM_TYPE_F16 && a->out_type != KVMEM_TYPE_BF16) {
        return "attention: output must be F32, F16 or BF16";
    }
    if (!cache_type(pool->type_k) || !cache_type(pool->type_v)) {
        return "attention: unsupported cache type";
    }
    code = KVMEM_HIP_OK;
    return nullptr;
}

static bool nothing_to_attend(const kvmem_hip_attn_args *a) {
    return a->n_seq == 0 || a->n_tokens == 0 || a->max_q == 0;
}

}  // namespace kvmem_hip

using namespace kvmem_hip;

extern "C" {

size_t kvmem_hip_attention_workspace(const kvmem_hip_pool *pool, const kvmem_hip_attn_args *a) {
    int code = 0;
    if (check_attention(pool, a, code) || nothing_to_attend(a)) {
        return 0;
    }
    const AttnPlan pl = plan_attention(pool, a);
    return pl.o_bytes + pl.ml_bytes;
}

int kvmem_hip_attention(kvmem_hip_ctx *ctx, const kvmem_hip_pool *pool, uint32_t layer,
                        const kvmem_hip_attn_args *a) {
    if (!ctx) {
        return KVMEM_HIP_ERR_INVALID;
    }
    int code = 0;
    if (const char *why = check_attention(pool, a, code)) {
        return fail(ctx, code, why);
    }
    if (nothing_to_attend(a)) {
        return KVMEM_HIP_OK;
    }
    if (layer >= pool->n_layers || !pool->k_layers || !pool->v_layers) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "attention: no such pool layer");
    }
    const void *k = pool->k_layers[layer];
    const void *v = pool->v_layers[layer];
    if (!k || !v || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u)) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "attention: layer pointer null or not 16-byte aligned");
    }
    AttnParams p{};
    p.q = static_cast<const uint8_t *>(a->q);
    p.q_nb1 = a->q_nb1;
    p.q_nb2 = a->q_nb2;
    p.out = static_cast<uint8_t *>(a->out);
    p.lse = a->lse;
    p.k = static_cast<const uint8_t *>(k);
    p.v = static_cast<const uint8_t *>(v);
    p.q_start = a->q_start;
    p.kv_len = a->kv_len;
    p.table = a->table;
    p.row_k = static_cast<uint32_t>(kvmem_hip_row_size(pool->type_k, pool->n_embd_k));
    p.row_v = static_cast<uint32_t>(kvmem_hip_row_size(pool->type_v, pool->n_embd_v));
    p.n_tokens = a->n_tokens;
    p.n_seq = a->n_seq;
    p.max_q = a->q_start ? std::min(a->max_q, a->n_tokens) : 1u;
    p.max_kv = a->max_kv;
    p.n_head = a->n_head;
    p.n_head_kv = a->n_head_kv;
    p.group = a->n_head / a->n_head_kv;
    p.T = pool->block_tokens;
    p.n_slots = pool->n_slots;
    p.table_stride = a->table_stride;
    p.causal = a->causal != 0;
    p.q_bf16 = a->q_type == KVMEM_TYPE_BF16;
    p.out_type = a->out_type;
    p.hadamard = pool->xf ? pool->xf->hadamard_v : 0;
    p.scale = a->scale > 0.0f ? a->scale : 1.0f / sqrtf(static_cast<float>(a->head_dim));
    const AttnPlan pl = plan_attention(pool, a);
    if (pl.grid >= 1u << 24) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "attention: too many requests of max_q tokens for one launch");
    }
    p.chunk = pl.chunk;
    p.n_parts = pl.n_parts;
    p.row_tile = pl.row_tile;
    p.row_tiles = pl.row_tiles;
    p.units = pl.units;
    (void) hipSetDevice(ctx->device);
    const size_t need = pl.o_bytes + pl.ml_bytes;
    if (need) {
        uint8_t *ws = static_cast<uint8_t *>(a->workspace);
        if (ws) {
            if ((reinterpret_cast<uintptr_t>(ws) & 15u) || a->workspace_bytes < need) {
                return fail(ctx, KVMEM_HIP_ERR_INVALID, "attention: workspace too small or not 16-byte aligned");
            }
        } else {
            hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
            if (!hip_ok(ctx, hipStreamIsCapturing(ctx->stream, &capture), "attention capture state")) {
                return KVMEM_HIP_ERR_RUNTIME;
            }
            if (capture != hipStreamCaptureStatusNone) {
                return fail(ctx, KVMEM_HIP_ERR_INVALID, "attention: a captured call needs a workspace of its own");
            }
            if (!ensure_dev(ctx, ctx->attn_scratch, need, "attention workspace")) {
                return KVMEM_HIP_ERR_NOMEM;
            }
            ws = static_cast<uint8_t *>(ctx->attn_scratch.ptr);
        }
        p.part_o = reinterpret_cast<float *>(ws);
        p.part_ml = reinterpret_cast<float2 *>(ws + pl.o_bytes);
    }
    if (injected_fail(ctx, KVMEM_HIP_FAIL_LAUNCH, "attention launch")) {
        return KVMEM_HIP_ERR_RUNTIME;
    }
    switch (pool->type_k) {
        case KVMEM_TYPE_Q4_0: launch_attention_v<KVMEM_TYPE_Q4_0>(ctx->stream, pool->type_v, a->head_dim, pl, p); break;
        case KVMEM_TYPE_Q5_0: launch_attention_v<KVMEM_TYPE_Q5_0>(ctx->stream, pool->type_v, a->head_dim, pl, p); break;
        case KVMEM_TYPE_Q8_0: launch_attention_v<KVMEM_TYPE_Q8_0>(ctx->stream, pool->type_v, a->head_dim, pl, p); break;
        default: launch_attention_v<KVMEM_TYPE_F16>(ctx->stream, pool->type_v, a->head_dim, pl, p); break;
    }
    return hip_ok(ctx, hipGetLastError(), "attention launch") ? KVMEM_HIP_OK : KVMEM_HIP_ERR_RUNTIME;
}

}  // extern "C"
