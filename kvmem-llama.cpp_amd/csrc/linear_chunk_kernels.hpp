// Linear attention by chunks of 64 tokens, for prompts (the formulas are those of
// linear.hip; a_t = exp(log_decay_t), G_i the chunk's sum of log_decay up to token i).
// With S the state before the chunk, D the chunk's rows d_i, and
//     A_ij = beta_i (k_i . k_j) e^(G_i - G_j)   j < i
//     P_ij = scale (q_i . k_j) e^(G_i - G_j)    j <= i
// the recurrence is, in products of matrices,
//     D  = (1 + A)^-1 diag(beta) (V - diag(e^G) K S)      (V itself without beta)
//     O  = scale diag(e^G) Q S + P D
//     S' = e^(G_last) S + K^T diag(e^(G_last - G)) D
// Two launches:
//   prepare  per (chunk, head): T = (1 + A)^-1 diag(beta) and P, which no state
//            enters, so all chunks at once; keys and queries as the matrix cores'
//            operands
//   walk     per (request, head, 16 columns of the state a wave): the chunks in
//            order.  Columns of a state never meet, so a wave needs nothing of any
//            other but the operands they share in LDS.  It keeps its columns of S in
//            registers; a product's accumulator (4 consecutive rows per lane) serves
//            as the next product's operand as it is, because the order in which a
//            contraction runs over its 32 indices is free as long as both operands
//            follow it: lane group g's eight are {4g..4g+3, 16+4g..16+4g+3}.
//
// Precision: operands are f16 parts of scaled fp32 numbers.  Each matrix (for S, D
// and their like each column) is scaled by a power of two that puts its largest
// element into [2^14, 2^15), then split into a high and a low f16 part: together 22
// bits, and what lies below 2^-39 of the largest is cut.  16-bit keys and queries
// are one part, exactly.  Products of two split factors leave out low x low.  A 16-bit
// out is rounded from the same sums as an fp32 one: with single parts (half a step
// 2^-12) small outputs of large terms would be off by more than their own rounding.
// Sums of log_decay are fp64: e^(G_i - G_j) of far apart sums keeps its digits, and a
// decay of zero (-inf, taken as -10^5) stays zero.
//
// A chunk with a number that is not finite among its rows, gates or factors goes
// token by token instead (walk_tokens), as products of masked rows would spread it
// to earlier tokens.
#pragma once

#include "kvmem_internal.hpp"

#include <algorithm>
#include <type_traits>

#include "linear.hpp"

namespace kvmem_hip {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct ChunkHead {
    float from_first[kChunk];  // e^G_i
    float to_last[kChunk];     // e^(G_last - G_i)
    int32_t exp_k, exp_q, exp_t, exp_p;
    int32_t exp_last;          // of the largest to_last: 0 unless decays grow
    uint32_t by_token;         // a number that is not finite
};
static_assert(sizeof(ChunkHead) <= kHeadBytes, "");

__device__ inline uint64_t entry_of(const LinearParams &a, const Request &rq, uint32_t s, uint32_t c) {
    return (c + 1) * kChunk <= rq.count ? rq.first / kChunk + c : a.batch.n_tokens / kChunk + s;
}

// The power of two that brings numbers whose largest magnitude has the bits `m`
// into [2^14, 2^15): x * 2^-e.  At least -127, so that 2^-e is an fp32 number: the
// smallest normal ones still come to 2, 25 bits above what f16 can hold.
__device__ inline int scale_exp(uint32_t m) { return max(static_cast<int>(m >> 23) - (127 + 14), -127); }
__device__ inline float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
__device__ inline uint32_t mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr uint32_t kInf = 0x7f800000u;

#define KVMEM_MFMA16(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0)

// ------------------------------------------------------------------- prepare

// 64 rows of DK numbers, four threads a row; rows at or beyond n are zeros.
template <typename T, int DK>
__device__ inline void load_rows(const uint8_t *p, uint64_t nb, uint32_t n, RawRow<T, 8> (&raw)[DK / 32]) {
    const uint32_t row = threadIdx.x >> 2;
#pragma unroll
    for (int i = 0; i < DK / 32; ++i) {
        raw[i] = RawRow<T, 8>{};
        if (row < n) {
            load_raw<T, 8>(p + row * nb + ((threadIdx.x & 3u) * 8u + 32u * i) * sizeof(T), raw[i]);
        }
    }
}

template <typename T, int DK>
__device__ inline uint32_t max_mag(const RawRow<T, 8> (&raw)[DK / 32]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < DK / 32; ++i) {
        float x[8];
        widen<T, 8>(raw[i], x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            m = max(m, mag(x[j]));
        }
    }
    return m;
}

// Largest of two numbers over the workgroup; `lds` holds 8 words.
__device__ inline void block_max2(uint32_t &a, uint32_t &b, uint32_t *lds) {
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        a = max(a, static_cast<uint32_t>(__shfl_xor(static_cast<int>(a), x, 64)));
        b = max(b, static_cast<uint32_t>(__shfl_xor(static_cast<int>(b), x, 64)));
    }
    if ((threadIdx.x & 63u) == 0) {
        lds[threadIdx.x >> 6] = a;
        lds[4 + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = max(max(lds[0], lds[1]), max(lds[2], lds[3]));
    b = max(max(lds[4], lds[5]), max(lds[6], lds[7]));
}

// Rows as scaled f16 parts in LDS, [PARTS][64][DK + 8].
template <typename T, int DK, int PARTS>
__device__ inline void put_rows(const RawRow<T, 8> (&raw)[DK / 32], float f, _Float16 *lds) {
    const uint32_t row = threadIdx.x >> 2;
#pragma unroll
    for (int i = 0; i < DK / 32; ++i) {
        float x[8];
        widen<T, 8>(raw[i], x);
        half8_t part[2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float y = x[j] * f;
            part[0][j] = static_cast<_Float16>(y);
            part[1][j] = static_cast<_Float16>(y - static_cast<float>(part[0][j]));
        }
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
            *reinterpret_cast<half8_t *>(lds + (q * kChunk + row) * (DK + 8) + (threadIdx.x & 3u) * 8u + 32u * i) =
                part[q];
        }
    }
}

// Rows [16 m, 16 m + 16), indices [32 k, 32 k + 32) of LDS rows as an operand.
template <int DK>
__device__ inline half8_t row_frag(const _Float16 *lds, uint32_t m, uint32_t k) {
    const uint32_t lane = threadIdx.x & 63u;
    const _Float16 *p = lds + (16u * m + (lane & 15u)) * (DK + 8) + 32u * k + 4u * (lane >> 4);
    const half4_t a = *reinterpret_cast<const half4_t *>(p);
    const half4_t b = *reinterpret_cast<const half4_t *>(p + 16);
    return half8_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// Columns [16 d, 16 d + 16) as rows, tokens [32 k, 32 k + 32) as indices.
template <int DK>
__device__ inline half8_t column_frag(const _Float16 *lds, uint32_t d, uint32_t k) {
    const uint32_t lane = threadIdx.x & 63u;
    const _Float16 *p = lds + (32u * k + 4u * (lane >> 4)) * (DK + 8) + 16u * d + (lane & 15u);
    half8_t x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[j] = p[j * (DK + 8)];
        x[4 + j] = p[(16 + j) * (DK + 8)];
    }
    return x;
}

__device__ inline void put_frag(uint8_t *base, uint32_t frag, half8_t x) {
    *reinterpret_cast<half8_t *>(base + frag * kFragBytes + (threadIdx.x & 63u) * 16u) = x;
}

constexpr uint32_t kTriPitch = 68;  // floats of a row of a 64 x 64 matrix in LDS

// Row tile `m` of a lower triangle as 8 numbers per 32 columns, upper part zero.
__device__ inline void tri_row(const float *tri, uint32_t m, uint32_t k, float x[8]) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t i = 16u * m + (lane & 15u);
    const uint32_t j0 = 32u * k + 4u * (lane >> 4);
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        const float4 v = *reinterpret_cast<const float4 *>(tri + i * kTriPitch + j0 + 16u * h);
        const float y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            x[4 * h + e] = j0 + 16u * h + e <= i ? y[e] : 0.0f;
        }
    }
}

// The 16 x 32 operands of a 64 x 64 lower triangle, (row tile m, columns [32 k, 32 k + 32)):
// (1,0) (2,0) (3,0) (3,1) whole; (0,0) and (2,1), whose second 16 columns are zeros, share
// the last by their first halves.
__device__ inline constexpr bool lower_half(uint32_t m, uint32_t k) { return m == 2u * k; }
__device__ inline constexpr uint32_t lower_frag(uint32_t m, uint32_t k) { return m - 1u + k; }
constexpr uint32_t kHalvesFrag = 4;

__device__ inline void put_lower(uint8_t *base, uint32_t m, uint32_t k, half8_t x) {
    if (lower_half(m, k)) {
        *reinterpret_cast<half4_t *>(base + kHalvesFrag * kFragBytes + (threadIdx.x & 63u) * 16u + k * 8u) =
            half4_t{x[0], x[1], x[2], x[3]};
    } else {
        put_frag(base, lower_frag(m, k), x);
    }
}

// c += tile (m, k) of a lower triangle times x, or (FLIP) x times its transpose.
template <bool FLIP>
__device__ inline f32x4_t mul_lower(const half8_t *tri, uint32_t m, uint32_t k, half8_t x, f32x4_t c) {
    if (lower_half(m, k)) {
        const half8_t f = tri[kHalvesFrag];
        const half4_t a = k == 0 ? half4_t{f[0], f[1], f[2], f[3]} : half4_t{f[4], f[5], f[6], f[7]};
        const half4_t b = {x[0], x[1], x[2], x[3]};
        return FLIP ? __builtin_amdgcn_mfma_f32_16x16x16f16(b, a, c, 0, 0, 0)
                    : __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
    }
    const half8_t a = tri[lower_frag(m, k)];
    return FLIP ? KVMEM_MFMA16(x, a, c) : KVMEM_MFMA16(a, x, c);
}

// c += a b over 16 indices, fp32: a row of `a` is read from LDS rows, b's rows
// 4g..4g+3 of column lane % 16 are in registers (as an accumulator holds them).
// `take`: whether the lane's four numbers of `a` count (else zeros).
__device__ inline f32x4_t mul16(const float *a_rows, f32x4_t b, f32x4_t c, bool take = true) {
    const uint32_t lane = threadIdx.x & 63u;
    float4 a = *reinterpret_cast<const float4 *>(a_rows + (lane & 15u) * kTriPitch + 4u * (lane >> 4));
    a.x = take ? a.x : 0.0f, a.y = take ? a.y : 0.0f, a.z = take ? a.z : 0.0f, a.w = take ? a.w : 0.0f;
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b[2], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b[3], c, 0, 0, 0);
}

// K's and Q's parts, later A (then P) and T.
template <int DK, int PARTS> constexpr uint32_t prep_lds() {
    constexpr uint32_t rows = 2u * PARTS * kChunk * (DK + 8) * 2u;
    constexpr uint32_t tri = 2u * kChunk * kTriPitch * 4u;
    return rows > tri ? rows : tri;
}

// Decays and beta of a chunk's tokens in one head, one token a lane (every wave holds
// them): G is the running sum of log_decay.
struct ChunkGates {
    double G;
    float beta;
    bool odd;  // a gate that is not finite (or a decay that grows without bound)
};

__device__ inline ChunkGates load_gates(const ChunkParams &p, uint64_t row0, uint32_t n, uint32_t h) {
    const uint32_t lane = threadIdx.x & 63u;
    float decay = 0.0f;
    ChunkGates x{0.0, 0.0f, false};
    if (lane < n) {
        if (p.a.decay) {
            decay = *reinterpret_cast<const float *>(p.a.decay + (row0 + lane) * p.a.decay_nb + h * 4u);
        }
        if (p.delta) {
            x.beta = *reinterpret_cast<const float *>(p.a.beta + (row0 + lane) * p.a.beta_nb + h * 4u);
        }
    }
    x.odd = !(decay < INFINITY) || !(mag(x.beta) < kInf);
    x.G = decay < -1e5f ? -1e5 : static_cast<double>(decay);
    if (p.a.decay) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double y = __shfl_up(x.G, d, 64);
            x.G += lane >= static_cast<uint32_t>(d) ? y : 0.0;
        }
    }
    return x;
}

// e^x of a difference of sums: the rounding of x log2 e costs |x| 2^-25 of a result
// that falls as e^x, so at most 2^-25 of 1.
__device__ inline float exp_diff(double x) {
    return __builtin_amdgcn_exp2f(static_cast<float>(x * 0x1.71547652b82fep+0));
}

// A workgroup takes `heads` heads of one key head, for which K K^T and Q K^T are the
// same: all of them where workgroups are many, one where they are few.  (1 + A)^-1 goes
// by blocks of 16: a wave inverts one on the diagonal, by substitution inside blocks of
// 8, and then makes its column of blocks downwards by products.  Three workgroups share a
// compute unit (35 KB of LDS, 168 registers; four would spill: 520 us for 405 of the
// second call below). Bound by its chain of steps between barriers: waves wait half their
// time, vector instructions take 41 %, matrix units 10 % of the busy cycles. 8192 tokens
// of one bf16 request, 48 heads of 128 x 128: 91-93 us; eight of up to 4096 tokens, 32
// heads: 143-157 us, 408 MB written.
template <typename T, int DK, bool DELTA>
__global__ __launch_bounds__(kPrepThreads, DK <= 128 ? 3 : 1) void linear_prepare_kernel(const ChunkParams p,
                                                                                         const uint32_t heads) {
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    constexpr int KS = DK / 32;
    __shared__ __align__(16) uint8_t lds[prep_lds<DK, PARTS>()];
    __shared__ uint32_t words[16];
    const uint32_t per = p.a.n_head / heads;
    const uint32_t h0 = blockIdx.x % per * heads, c = blockIdx.x / per, s = blockIdx.y;
    const Request rq = request_of(p.a.batch, s);
    if (c * kChunk >= rq.count) {
        return;
    }
    const uint32_t n = min(kChunk, rq.count - c * kChunk);
    const uint64_t row0 = static_cast<uint64_t>(rq.first) + c * kChunk;
    const uint64_t entry = entry_of(p.a, rq, s, c);
    const uint32_t hk = h0 / p.a.group;
    uint8_t *keys = p.keys + (entry * (p.a.n_head / p.a.group) + hk) * p.key_bytes;
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    RawRow<T, 8> raw_k[KS], raw_q[KS] = {};  // without an out: no queries, zeros
    load_rows<T, DK>(p.a.k + row0 * p.a.k_nb2 + hk * p.a.k_nb1, p.a.k_nb2, n, raw_k);
    if (p.outs) {
        load_rows<T, DK>(p.a.q + row0 * p.a.q_nb2 + hk * p.a.q_nb1, p.a.q_nb2, n, raw_q);
    }
    ChunkGates gates = load_gates(p, row0, n, h0);
    uint32_t mk = max_mag<T, DK>(raw_k), mq = max_mag<T, DK>(raw_q);
    block_max2(mk, mq, words);
    const bool odd_rows = mk >= kInf || mq >= kInf;
    const int exp_k = scale_exp(mk), exp_q = scale_exp(mq);
    _Float16 *k16 = reinterpret_cast<_Float16 *>(lds);
    _Float16 *q16 = k16 + PARTS * kChunk * (DK + 8);
    put_rows<T, DK, PARTS>(raw_k, pow2(-exp_k), k16);
    put_rows<T, DK, PARTS>(raw_q, pow2(-exp_q), q16);
    __syncthreads();

    // the key head's operands, by its first head
    if (h0 % p.a.group == 0) {
#pragma unroll
        for (uint32_t part = 0; part < PARTS; ++part) {
            const _Float16 *kp = k16 + part * kChunk * (DK + 8);
            const _Float16 *qp = q16 + part * kChunk * (DK + 8);
            uint8_t *out = keys + part * (12u * KS * kFragBytes);
#pragma unroll
            for (uint32_t k = 0; k < KS; ++k) {
                put_frag(out, w * KS + k, row_frag<DK>(kp, w, k));
                put_frag(out, 4u * KS + w * KS + k, row_frag<DK>(qp, w, k));
            }
#pragma unroll
            for (uint32_t i = 0; i < KS; ++i) {  // 2 KS tiles of 16 columns x 2 halves, over 4 waves
                const uint32_t f = w * KS + i;
                put_frag(out, 8u * KS + f, column_frag<DK>(kp, f >> 1, f & 1u));
            }
        }
    }

    // row tile w of K K^T and Q K^T
    f32x4_t kk[4], qk[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        kk[j] = qk[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        if (j > w) {
            continue;
        }
#pragma unroll
        for (uint32_t k = 0; k < KS; ++k) {
            const half8_t b = row_frag<DK>(k16, j, k);
            const half8_t a = row_frag<DK>(k16, w, k);
            half8_t b2, a2;
            if constexpr (PARTS == 2) {
                b2 = row_frag<DK>(k16 + kChunk * (DK + 8), j, k);
            }
            if constexpr (DELTA) {
                kk[j] = KVMEM_MFMA16(a, b, kk[j]);
                if constexpr (PARTS == 2) {
                    a2 = row_frag<DK>(k16 + kChunk * (DK + 8), w, k);
                    kk[j] = KVMEM_MFMA16(a, b2, kk[j]);
                    kk[j] = KVMEM_MFMA16(a2, b, kk[j]);
                }
            }
            const half8_t aq = row_frag<DK>(q16, w, k);
            qk[j] = KVMEM_MFMA16(aq, b, qk[j]);
            if constexpr (PARTS == 2) {
                a2 = row_frag<DK>(q16 + kChunk * (DK + 8), w, k);
                qk[j] = KVMEM_MFMA16(aq, b2, qk[j]);
                qk[j] = KVMEM_MFMA16(a2, b, qk[j]);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            kk[j][r] = __builtin_amdgcn_ldexpf(kk[j][r], 2 * exp_k);
            qk[j][r] = __builtin_amdgcn_ldexpf(qk[j][r], exp_k + exp_q) * p.a.scale;
        }
        __builtin_amdgcn_sched_barrier(0);  // a tile's operands at a time, to keep to the registers of three workgroups
    }
    float *tri_a = reinterpret_cast<float *>(lds);
    float *tri_t = tri_a + kChunk * kTriPitch;
    for (uint32_t h = h0; h < h0 + heads; ++h) {
        uint8_t *head = p.heads + (entry * p.a.n_head + h) * p.head_bytes;
        if (h != h0) {
            gates = load_gates(p, row0, n, h);
        }
        const double G = gates.G, G_last = __shfl(G, 63, 64);
        const float beta = gates.beta;
        const float from_first = expf(static_cast<float>(G)), to_last = expf(static_cast<float>(G_last - G));
        bool odd = odd_rows || gates.odd || !(from_first < INFINITY) || !(to_last < INFINITY);
        __syncthreads();  // K and Q, or the head before, are read: A and T take their place
        double Gi[4];
        float bi[4];
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            const int i = static_cast<int>(16u * w + 4u * g + r);
            Gi[r] = __shfl(G, i, 64);
            bi[r] = __shfl(beta, i, 64);
        }
        f32x4_t pk[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if (j > w) {
                continue;
            }
            const uint32_t col = 16u * j + (lane & 15u);
            const double Gj = __shfl(G, static_cast<int>(col), 64);
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                const uint32_t i = 16u * w + 4u * g + r;
                const float f = p.a.decay ? exp_diff(Gi[r] - Gj) : 1.0f;
                if constexpr (DELTA) {
                    tri_a[i * kTriPitch + col] = col < i ? kk[j][r] * f * bi[r] : 0.0f;
                }
                pk[j][r] = qk[j][r] * f;
            }
        }
        if constexpr (DELTA) {
            __syncthreads();
            // 1 + A's diagonal block w: its two 8 x 8 diagonal blocks inverted by forward
            // substitution (lane (any, b, c) has column c of block b), together D; with L the
            // block below them, the inverse is D - D L D
            const uint32_t c8 = lane & 7u, b8 = lane & 8u;
            float *a = tri_a + 16u * w * kTriPitch + 16u * w;
            float *t = tri_t + 16u * w * kTriPitch + 16u * w;
            float x[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                float y = c8 == i ? 1.0f : 0.0f;
#pragma unroll
                for (uint32_t k = 0; k < i; ++k) {
                    y = __builtin_fmaf(-a[(b8 + i) * kTriPitch + b8 + k], x[k], y);
                }
                x[i] = y;
            }
            if (g < 2) {  // group 0 the blocks, group 1 the zeros beside them
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    t[(b8 + i) * kTriPitch + (g == 0 ? b8 : b8 ^ 8u) + c8] = g == 0 ? x[i] : 0.0f;
                }
            }
            __syncthreads();
            f32x4_t col[4];
            const float bw = __shfl(beta, static_cast<int>(16u * w + (lane & 15u)), 64);
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                col[0][r] = t[(4u * g + r) * kTriPitch + (lane & 15u)];
            }
            f32x4_t ld = mul16(a, col[0], f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, (lane & 15u) >= 8u && g < 2);
            ld = mul16(t, ld, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
            col[0] -= ld;
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                t[(4u * g + r) * kTriPitch + (lane & 15u)] = col[0][r];
            }
            __syncthreads();
            // column w of blocks downwards: T_iw = -T_ii sum_k A_ik T_kw
#pragma unroll
            for (uint32_t d = 1; d < 4; ++d) {
                col[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
                if (w + d < 4) {
                    f32x4_t y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (uint32_t k = 0; k < 3; ++k) {
                        if (k < d) {
                            y = mul16(tri_a + 16u * (w + d) * kTriPitch + 16u * (w + k), col[k], y);
                        }
                    }
                    y = mul16(tri_t + 16u * (w + d) * kTriPitch + 16u * (w + d), y, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
                    col[d] = -y;
                }
            }
            __syncthreads();  // A and the diagonal blocks are read
#pragma unroll
            for (uint32_t d = 0; d < 4; ++d) {
                if (w + d < 4) {
#pragma unroll
                    for (uint32_t r = 0; r < 4; ++r) {
                        tri_t[(16u * (w + d) + 4u * g + r) * kTriPitch + 16u * w + (lane & 15u)] = col[d][r] * bw;
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if (j > w) {
                continue;
            }
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                tri_a[(16u * w + 4u * g + r) * kTriPitch + 16u * j + (lane & 15u)] = pk[j][r];
            }
        }
        __syncthreads();
        float xt[2][8], xp[2][8];
        uint32_t mt = 0, mp = 0;
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
            if (k > w / 2) {
                continue;
            }
            if constexpr (DELTA) {
                tri_row(tri_t, w, k, xt[k]);
            }
            tri_row(tri_a, w, k, xp[k]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                mt = DELTA ? max(mt, mag(xt[k][i])) : 0u;
                mp = max(mp, mag(xp[k][i]));
            }
        }
        block_max2(mt, mp, words + 8);
        odd = odd || mt >= kInf || mp >= kInf;
        const int exp_t = scale_exp(mt), exp_p = scale_exp(mp);
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
            if (k > w / 2) {
                continue;
            }
            uint8_t *at = head + kHeadBytes;
            half8_t hi, lo;
            if constexpr (DELTA) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = xt[k][i] * pow2(-exp_t);
                    hi[i] = static_cast<_Float16>(y);
                    lo[i] = static_cast<_Float16>(y - static_cast<float>(hi[i]));
                }
                put_lower(at, w, k, hi);
                put_lower(at + kLowerFrags * kFragBytes, w, k, lo);
                at += 2u * kLowerFrags * kFragBytes;
            }
            if (p.outs) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = xp[k][i] * pow2(-exp_p);
                    hi[i] = static_cast<_Float16>(y);
                    lo[i] = static_cast<_Float16>(y - static_cast<float>(hi[i]));
                }
                put_lower(at, w, k, hi);
                put_lower(at + kLowerFrags * kFragBytes, w, k, lo);
            }
        }
        if (w == 0) {
            ChunkHead *out = reinterpret_cast<ChunkHead *>(head);
            out->from_first[lane] = from_first;
            out->to_last[lane] = to_last;
            const bool any = __any(odd);
            uint32_t top = mag(to_last);
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) {
                top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), x, 64)));
            }
            // to_last <= 2^exp_last; the last token's is 1
            const int exp_last = top == __float_as_uint(1.0f) ? 0 : static_cast<int>(top >> 23) - 126;
            if (lane == 0) {
                out->exp_k = exp_k;
                out->exp_q = exp_q;
                out->exp_t = exp_t;
                out->exp_p = exp_p;
                out->exp_last = exp_last;
                out->by_token = any;
            }
        }
    }
}

// ---------------------------------------------------------------------- walk

template <typename T> __device__ inline float load_one(const uint8_t *p) {
    return static_cast<float>(*reinterpret_cast<const T *>(p));
}

__device__ inline void store_one(uint8_t *p, int type, uint64_t i, float x) {
    if (type == KVMEM_TYPE_F32) {
        reinterpret_cast<float *>(p)[i] = x;
    } else if (type == KVMEM_TYPE_F16) {
        reinterpret_cast<_Float16 *>(p)[i] = static_cast<_Float16>(x);
    } else {
        reinterpret_cast<__bf16 *>(p)[i] = static_cast<__bf16>(x);
    }
}

__device__ inline half8_t get_frag(const uint8_t *base, uint32_t frag) {
    return *reinterpret_cast<const half8_t *>(base + frag * kFragBytes + (threadIdx.x & 63u) * 16u);
}

// The largest of a column's four lanes (l, l ^ 16, l ^ 32, l ^ 48): two exchanges of
// rows of 16 and of halves of the wave, each of a number with its own copy.
__device__ inline uint32_t column_max(uint32_t m) {
    auto x = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = max(static_cast<uint32_t>(x[0]), static_cast<uint32_t>(x[1]));
    x = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    return max(static_cast<uint32_t>(x[0]), static_cast<uint32_t>(x[1]));
}

// The largest magnitude of a lane's numbers, NaN left out.
template <int TILES> __device__ inline float lane_max(const f32x4_t (&x)[TILES]) {
    float m[4] = {};
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(m[2 * (t & 1)]) : "v"(x[t][0]), "v"(x[t][1]));
        asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(m[2 * (t & 1) + 1]) : "v"(x[t][2]), "v"(x[t][3]));
    }
    asm("v_max3_f32 %0, %0, %1, %2" : "+v"(m[0]) : "v"(m[1]), "v"(m[2]));
    return __builtin_fmaxf(m[0], m[3]);
}

// A column's numbers (tiles of 16 rows, 4 of each in every lane of the column) as
// two f16 parts of x * 2^-e.  The mixed-precision FMAs round
// x f and x f - high to f16 without a step in fp32: two instructions a number.  No
// number here is a matrix instruction's own result (its readers would have to wait
// inside the block); an instruction stands between a half word's write and its use.
template <int TILES> __device__ inline int column_exp(const f32x4_t (&x)[TILES]) {
    return scale_exp(column_max(__float_as_uint(lane_max<TILES>(x))));
}

typedef uint32_t words4_t __attribute__((ext_vector_type(4)));

template <int TILES>
__device__ inline void split(const f32x4_t (&x)[TILES], int e, half8_t (&hi)[TILES / 2], half8_t (&lo)[TILES / 2]) {
    const float f = pow2(-e);
#pragma unroll
    for (int t = 0; t < TILES; t += 2) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            asm("v_fma_mixlo_f16 %0, %4, %8, 0\n\t"
                "v_fma_mixlo_f16 %1, %6, %8, 0\n\t"
                "v_fma_mixhi_f16 %0, %5, %8, 0\n\t"
                "v_fma_mixhi_f16 %1, %7, %8, 0\n\t"
                "v_fma_mixlo_f16 %2, %4, %8, -%0 op_sel_hi:[0,0,1]\n\t"
                "v_fma_mixlo_f16 %3, %6, %8, -%1 op_sel_hi:[0,0,1]\n\t"
                "v_fma_mixhi_f16 %2, %5, %8, -%0 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
                "v_fma_mixhi_f16 %3, %7, %8, -%1 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
                "s_nop 0"
                : "=&v"(h[2 * u]), "=&v"(h[2 * u + 1]), "=&v"(l[2 * u]), "=&v"(l[2 * u + 1])
                : "v"(x[t + u][0]), "v"(x[t + u][1]), "v"(x[t + u][2]), "v"(x[t + u][3]), "v"(f));
        }
        hi[t / 2] = __builtin_bit_cast(half8_t, words4_t{h[0], h[1], h[2], h[3]});
        lo[t / 2] = __builtin_bit_cast(half8_t, words4_t{l[0], l[1], l[2], l[3]});
    }
}

// Lets the scheduler put `valu` vector instructions behind each of `n` matrix ones: a
// matrix instruction of 16 x 16 x 32 runs 16 cycles, in which four others can start.
template <int N, int VALU> __device__ inline void interleave() {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
    }
}

// A chunk's tokens one by one, on the wave's 16 columns of the state (rows
// 16 d + 4 g + r in s[d][r]).
template <typename T, int DK>
__device__ inline __attribute__((always_inline)) void walk_tokens(const ChunkParams &p, f32x4_t (&s)[DK / 16],
                                                                  uint64_t row0, uint32_t n, uint32_t h, uint32_t hk,
                                                                  uint32_t col, bool with_out) {
    const uint32_t g = (threadIdx.x & 63u) >> 4;
    for (uint32_t t = 0; t < n; ++t) {
        const uint64_t row = row0 + t;
        const uint8_t *k = p.a.k + row * p.a.k_nb2 + hk * p.a.k_nb1;
        const float a = p.a.decay ? expf(*reinterpret_cast<const float *>(p.a.decay + row * p.a.decay_nb + h * 4u))
                                  : 1.0f;
        float kd[DK / 16][4];
#pragma unroll
        for (int d = 0; d < DK / 16; ++d) {
            RawRow<T, 4> raw;
            load_raw<T, 4>(k + (16u * d + 4u * g) * sizeof(T), raw);
            widen<T, 4>(raw, kd[d]);
        }
        float x = load_one<T>(p.a.v + row * p.a.v_nb2 + h * p.a.v_nb1 + col * sizeof(T));
        if (p.delta) {
            float u = 0.0f;
#pragma unroll
            for (int d = 0; d < DK / 16; ++d) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    u = __builtin_fmaf(s[d][r], kd[d][r], u);
                }
            }
            u += __shfl_xor(u, 16, 64);
            u += __shfl_xor(u, 32, 64);
            const float b = *reinterpret_cast<const float *>(p.a.beta + row * p.a.beta_nb + h * 4u);
            x = b * __builtin_fmaf(-a, u, x);
        }
#pragma unroll
        for (int d = 0; d < DK / 16; ++d) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[d][r] = __builtin_fmaf(kd[d][r], x, a * s[d][r]);
            }
        }
        if (with_out) {
            const uint8_t *q = p.a.q + row * p.a.q_nb2 + hk * p.a.q_nb1;
            float o = 0.0f;
#pragma unroll
            for (int d = 0; d < DK / 16; ++d) {
                RawRow<T, 4> raw;
                float qd[4];
                load_raw<T, 4>(q + (16u * d + 4u * g) * sizeof(T), raw);
                widen<T, 4>(raw, qd);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    o = __builtin_fmaf(s[d][r], qd[r], o);
                }
            }
            o += __shfl_xor(o, 16, 64);
            o += __shfl_xor(o, 32, 64);
            if (g == 0) {
                store_one(p.a.out, p.a.out_type, (row * p.a.n_head + h) * p.a.dim_v + col, p.a.scale * o);
            }
        }
    }
}

// Four numbers of rows `row`, row + 16, row + 32 and row + 48, of which `rows` exist.
template <typename T>
__device__ inline void store_rows(uint8_t *to, uint64_t step, uint32_t row, uint32_t rows, const float (&y)[4][4]) {
    if (rows == kChunk) {
#pragma unroll
        for (uint32_t m = 0; m < 4; ++m) {
            store_row<T, 4>(to + m * step, y[m]);
        }
        return;
    }
#pragma unroll
    for (uint32_t m = 0; m < 4; ++m) {
        if (16u * m + row < rows) {
            store_row<T, 4>(to + m * step, y[m]);
        }
    }
}

typedef __attribute__((address_space(3))) void lds_void_t;

template <int N>
__device__ inline void get_frags(const uint8_t *base, uint32_t frag, half8_t (&x)[N]) {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        x[i] = get_frag(base, frag + i);
    }
}

// A chunk in LDS: its keys' operands [K Q K^T][part], then its head's (ChunkHead, T, P),
// as they lie in its entries, then its values.
template <typename T, int DK, bool DELTA, bool OUT, int WAVES> struct ChunkSpace {
    static constexpr uint32_t parts = sizeof(T) == 4 ? 2 : 1;
    static constexpr uint32_t key_frags = 12 * (DK / 32) * parts;
    static constexpr uint32_t head_frags = 1 + (DELTA ? 2 * kLowerFrags : 0) + (OUT ? 2 * kLowerFrags : 0);
    static constexpr uint32_t row_bytes = WAVES * 16 * sizeof(T);  // of the values
    static constexpr uint32_t rest = head_frags * kFragBytes + kChunk * row_bytes;
    static constexpr uint32_t most = 160 * 1024;
    // the keys' operands go through LDS where one chunk fits, chunks alternate between
    // two places where two fit
    static constexpr bool keys = key_frags * kFragBytes + rest <= most;
    static constexpr uint32_t bytes = (keys ? key_frags * kFragBytes : 0) + rest;
    static constexpr uint32_t places = 2 * bytes <= most ? 2 : 1;
};

// Every wave's LDS reads are done before another may write there.
__device__ inline void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Segments' states one behind the other, in place: what a segment adds becomes the
// state behind it, S_x = decay_x S_(x-1) + added_x.  The first one's holds the call's
// state already, and the last one's is the second pass's.  Four elements a thread;
// segments are read eight at a time, since a chain of loads would cost each of them a
// latency.
constexpr uint32_t kScanThreads = 256;
constexpr uint32_t kScanAtOnce = 8;

static __global__ __launch_bounds__(kScanThreads) void linear_scan_kernel(const ChunkParams p) {
    const uint32_t s = blockIdx.y;
    const Request rq = request_of(p.a.batch, s);
    const uint32_t last = rq.count ? (rq.count - 1u) / (p.seg_chunks * kChunk) : 0u;
    if (last < 2) {
        return;
    }
    const uint64_t of_head = static_cast<uint64_t>(p.dim_k) * p.a.dim_v, of_seg = of_head * p.a.n_head;
    const uint64_t at = (static_cast<uint64_t>(blockIdx.x) * kScanThreads + threadIdx.x) * 4u;
    if (at >= of_seg) {
        return;
    }
    float *made = p.seg_states + s * p.segs * of_seg + at;
    const float *decays = p.seg_decays + static_cast<uint64_t>(s) * p.segs * p.a.n_head + at / of_head;
    f32x4_t state = *reinterpret_cast<const f32x4_t *>(made);
    for (uint32_t x0 = 1; x0 < last; x0 += kScanAtOnce) {
        f32x4_t added[kScanAtOnce];
        float decay[kScanAtOnce];
#pragma unroll
        for (uint32_t i = 0; i < kScanAtOnce; ++i) {
            const uint32_t x = min(x0 + i, last - 1u);
            added[i] = *reinterpret_cast<const f32x4_t *>(made + x * of_seg);
            decay[i] = decays[static_cast<uint64_t>(x) * p.a.n_head];
        }
#pragma unroll
        for (uint32_t i = 0; i < kScanAtOnce; ++i) {
            if (x0 + i < last) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    state[e] = state[e] == 0.0f ? added[i][e] : __builtin_fmaf(decay[i], state[e], added[i][e]);
                }
                *reinterpret_cast<f32x4_t *>(made + (x0 + i) * of_seg) = state;
            }
        }
    }
}

// The request that the workgroups of `rank` take: the longest ones first, so that the
// last to end are short (eight bf16 prompts of up to 4096 tokens, 32 heads of 128 x 128:
// 375-390 us, 430 in their own order).  Beyond a wave's lanes of requests, in their own order.
__device__ inline uint32_t request_by_length(const LinearParams &a, uint32_t rank) {
    if (a.n_seq == 1 || a.n_seq > 64) {
        return rank;
    }
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t count = lane < a.n_seq ? request_of(a.batch, lane).count : 0u;
    uint32_t before = 0;  // longer ones, and as long ones in front of it
    for (uint32_t j = 0; j < a.n_seq; ++j) {
        const uint32_t other = __builtin_amdgcn_readlane(count, j);
        before += other > count || (other == count && j < lane) ? 1u : 0u;
    }
    return static_cast<uint32_t>(__builtin_ctzll(__ballot(lane < a.n_seq && before == rank)));
}

// WAVES waves compute, 16 columns each, and as many bring the next chunk into LDS: a
// wave issues one instruction at a time, and those for the copies would cost the
// computing ones a third of a chunk's time (8192 tokens, 48 heads of 128 x 128: 728 us
// with loads of their own, 493 with these waves, at that step).
//
// Bound by one wave's instructions: a chunk of 128 x 128 takes it 132 matrix
// instructions (2110 cycles) and 690 vector ones (2750), of which little overlaps, as
// each product waits for the one before, 7000 cycles = 3.1 us in all.  8192 tokens take
// 128 of these, one behind the other: 401-417 us on 96 compute units (a column of the
// state needs the whole chunk before it), 48 heads of 128 x 128.
template <typename T, int DK, bool DELTA, bool OUT, int WAVES>
__global__ __launch_bounds__(128 * WAVES, 1) void linear_walk_kernel(const ChunkParams p) {
    typedef ChunkSpace<T, DK, DELTA, OUT, WAVES> Space;
    constexpr int PARTS = Space::parts, KS = DK / 32, TILES = DK / 16;
    __shared__ __align__(16) uint8_t lds[Space::places * Space::bytes];
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t slices = p.a.dim_v / (16u * WAVES);
    // workgroups go round the 8 XCDs: each XCD takes neighbouring heads, whose columns
    // read the same operands through its L2
    const uint32_t unit = (blockIdx.x % kXcds) * (gridDim.x / kXcds) + blockIdx.x / kXcds;
    if (unit >= p.a.n_head * slices) {
        return;
    }
    const uint32_t h = unit / slices, s_id = request_by_length(p.a, blockIdx.y);
    const uint32_t col0 = (unit % slices) * (16u * WAVES);
    const uint32_t hk = h / p.a.group;
    Request rq = request_of(p.a.batch, s_id);
    rq.first = __builtin_amdgcn_readfirstlane(rq.first);
    rq.count = __builtin_amdgcn_readfirstlane(rq.count);
    // the chunks of this workgroup's segment: the first pass leaves behind every segment
    // but the last the state that it alone makes, the second starts from those
    uint32_t c0 = 0, limit = rq.count;
    uint32_t seg = 0, last_seg = 0;
    if constexpr (!DELTA) {
        if (p.segs > 1) {
            const uint32_t of_seg = p.seg_chunks * kChunk;
            seg = blockIdx.z;
            last_seg = rq.count ? (rq.count - 1u) / of_seg : 0u;
            if (seg > last_seg ||
                (p.second_pass ? seg == 0 || (!OUT && seg < last_seg) : seg == last_seg && seg > 0)) {
                return;
            }
            c0 = seg * p.seg_chunks;
            limit = min(rq.count, (seg + 1) * of_seg);
        }
    }
    const uint64_t key_step = p.key_bytes * (p.a.n_head / p.a.group), head_step = p.head_bytes * p.a.n_head;
    const uint8_t *keys = p.keys + hk * p.key_bytes, *heads = p.heads + h * p.head_bytes;  // of entry 0
    constexpr uint32_t head_at = Space::keys ? Space::key_frags * kFragBytes : 0;
    constexpr uint32_t values_at = head_at + Space::head_frags * kFragBytes;

    if (w >= WAVES) {
        const uint32_t lw = w - WAVES;
        const uint32_t lane16 = lane * 16u;
        constexpr uint32_t lanes = Space::row_bytes / 16;  // of a row of values
        const uint32_t row = lane / lanes;
        const uint8_t *values =
            p.a.v + rq.first * p.a.v_nb2 + h * p.a.v_nb1 + col0 * sizeof(T) + (lane % lanes) * 16u;
        auto frags = [&](const uint8_t *from, uint8_t *to, auto count) {
            constexpr uint32_t N = decltype(count)::value;
#pragma unroll
            for (uint32_t i = 0; i < (N + WAVES - 1) / WAVES; ++i) {
                if ((i + 1) * WAVES <= N || i * WAVES + lw < N) {
                    const uint32_t f = (i * WAVES + lw) * kFragBytes;
                    __builtin_amdgcn_global_load_lds(as_global(from + f) + lane16, (lds_void_t *) (to + f), 16, 0, 0);
                }
            }
        };
        auto request = [&](uint32_t c, uint8_t *to) {
            const uint64_t entry = entry_of(p.a, rq, s_id, c);
            if constexpr (Space::keys) {
                frags(keys + entry * key_step, to, std::integral_constant<uint32_t, Space::key_frags>{});
            }
            frags(heads + entry * head_step, to + head_at, std::integral_constant<uint32_t, Space::head_frags>{});
            const uint32_t n = min(kChunk, rq.count - c * kChunk);
#pragma unroll
            for (uint32_t i = 0; i < (lanes + WAVES - 1) / WAVES; ++i) {
                const uint32_t x = i * WAVES + lw;  // of `lanes` groups of 64 / lanes rows
                if (x < lanes) {
                    const uint32_t t = min(x * (64 / lanes) + row, n - 1u);
                    __builtin_amdgcn_global_load_lds(as_global(values + static_cast<uint64_t>(c * kChunk + t) * p.a.v_nb2),
                                                     (lds_void_t *) (to + values_at + x * kFragBytes), 16, 0, 0);
                }
            }
        };
        if (Space::places == 2 && c0 * kChunk < limit) {
            request(c0, lds + (c0 & 1u) * Space::bytes);
        }
        for (uint32_t c = c0; c * kChunk < limit; ++c) {
            if (Space::places == 1) {
                lds_barrier();  // the chunk before is read
                request(c, lds);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            lds_barrier();
            if (Space::places == 2 && (c + 1) * kChunk < limit) {
                request(c + 1, lds + ((c + 1) & 1u) * Space::bytes);
            }
        }
        return;
    }

    const uint32_t col = col0 + 16u * w + (lane & 15u);
    const uint64_t at = (static_cast<uint64_t>(rq.slot) * p.a.n_head + h) * DK * p.a.dim_v + col;
    // operand i of K (at 0), Q (4 KS) or K^T (8 KS), its first or second part
    auto frag_index = [](uint32_t matrix, uint32_t i, uint32_t part) { return part * 12u * KS + matrix + i; };
    f32x4_t s[TILES];
#pragma unroll
    for (int d = 0; d < TILES; ++d) {
        s[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const uint64_t seg_at = static_cast<uint64_t>(s_id) * p.segs * p.a.n_head + h;  // the request's first segment
    if (!DELTA && p.second_pass) {
        const float *made = p.seg_states + (seg_at + (seg - 1u) * p.a.n_head) * DK * p.a.dim_v + col;
#pragma unroll
        for (int d = 0; d < TILES; ++d) {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                s[d][r] = made[static_cast<uint64_t>(16u * d + 4u * g + r) * p.a.dim_v];
            }
        }
    } else if (seg == 0 && p.a.state && rq.has_slot) {
#pragma unroll
        for (int d = 0; d < TILES; ++d) {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                s[d][r] = p.a.state[at + static_cast<uint64_t>(16u * d + 4u * g + r) * p.a.dim_v];
            }
        }
    }
    const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint64_t out_row = static_cast<uint64_t>(p.a.n_head) * p.a.dim_v;
    const uint32_t esz = p.a.out_type == KVMEM_TYPE_F32 ? 4u : 2u;
    const uint32_t out_at = ((lane & 15u) * static_cast<uint32_t>(out_row) + 4u * g) * esz;
    const bool with_out = OUT && (seg == 0 || p.second_pass);
    float decayed = 1.0f;  // over the segment
    for (uint32_t c = c0; c * kChunk < limit; ++c) {
        const uint32_t n = min(kChunk, rq.count - c * kChunk);
        const uint64_t row0 = static_cast<uint64_t>(rq.first) + c * kChunk;
        const uint32_t rows = with_out ? n : 0u;
        const uint8_t *here = lds + (Space::places == 2 ? (c & 1u) * Space::bytes : 0u);
        const uint8_t *kp = here;
        if constexpr (!Space::keys) {
            kp = keys + entry_of(p.a, rq, s_id, c) * key_step;
        }
        const uint8_t *head = here + head_at;
        const ChunkHead *ch = reinterpret_cast<const ChunkHead *>(head);
        const uint8_t *frag_t = head + kHeadBytes;
        const uint8_t *frag_p = frag_t + (DELTA ? 2u * kLowerFrags * kFragBytes : 0u);
        if (Space::places == 1) {
            lds_barrier();  // the chunk before is read
        }
        lds_barrier();

        // the products' operands are read 8 at a time, a group ahead of their use
        half8_t kq[2][8];
        auto read8 = [&](half8_t(&to)[8], uint32_t matrix, uint32_t k) {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {  // K, Q: four row tiles of steps k, k + 1; K^T: operands 4k..4k+7
                to[i] = get_frag(kp, frag_index(matrix, matrix == 8 * KS ? 4 * k + i : (i & 3u) * KS + k + (i >> 2), 0));
            }
        };
        constexpr uint32_t behind_k = OUT ? 4 * KS : 8 * KS;  // what the first product's operands are followed by
        read8(kq[0], DELTA ? 0 : behind_k, 0);
        const uint8_t *vp = here + values_at + 4u * g * Space::row_bytes + (16u * w + (lane & 15u)) * sizeof(T);
        f32x4_t v[4];
#pragma unroll
        for (uint32_t m = 0; m < 4; ++m) {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                v[m][r] = load_one<T>(vp + (16u * m + r) * Space::row_bytes);
            }
        }
        half8_t hi[KS], lo[KS];
        const int exp_s = column_exp<TILES>(s);
        split<TILES>(s, exp_s, hi, lo);
        int es[4];  // of columns 4 g + r
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            es[r] = __shfl(exp_s, static_cast<int>(4u * g) + r, 64);
        }
        f32x4_t d[4] = {zero, zero, zero, zero}, o[4] = {zero, zero, zero, zero};
        half8_t tf[DELTA ? 2 * kLowerFrags : 1], pf[OUT ? 2 * kLowerFrags : 1];
        if constexpr (DELTA) {
#pragma unroll
            for (uint32_t k = 0; k < KS; k += 2) {
                if (k + 2 < KS) {
                    read8(kq[(k / 2 + 1) & 1], 0, k + 2);
                } else {
                    read8(kq[(k / 2 + 1) & 1], behind_k, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (uint32_t x = 0; x < (PARTS == 2 ? 6 : 4); ++x) {  // sums in between do not wait for each other
#pragma unroll
                    for (uint32_t m = 0; m < 4; ++m) {
                        half8_t a;
                        if (x >= 4) {
                            a = get_frag(kp, frag_index(0, m * KS + k + (x & 1u), 1));
                        } else {
                            a = kq[(k / 2) & 1][4 * (x & 1u) + m];
                        }
                        d[m] = KVMEM_MFMA16(a, x == 2 || x == 3 ? lo[k + (x & 1u)] : hi[k + (x & 1u)], d[m]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        constexpr int Q0 = DELTA ? (KS / 2) & 1 : 0;  // where Q's first group is
        f32x4_t first[4];
        float out_first[4];
        const int exp_k = ch->exp_k, exp_q = ch->exp_q, exp_t = ch->exp_t, exp_p = ch->exp_p;
        if constexpr (OUT) {
#pragma unroll
            for (uint32_t k = 0; k < KS; k += 2) {  // transposed: columns of the state are rows of the accumulator
                constexpr uint32_t KT = 8 * KS;
                if (k + 2 < KS) {
                    read8(kq[(Q0 + k / 2 + 1) & 1], 4 * KS, k + 2);
                } else {
                    read8(kq[(Q0 + k / 2 + 1) & 1], KT, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (uint32_t x = 0; x < (PARTS == 2 ? 6 : 4); ++x) {
#pragma unroll
                    for (uint32_t m = 0; m < 4; ++m) {
                        half8_t a;
                        if (x >= 4) {
                            a = get_frag(kp, frag_index(4 * KS, m * KS + k + (x & 1u), 1));
                        } else {
                            a = kq[(Q0 + k / 2) & 1][4 * (x & 1u) + m];
                        }
                        o[m] = KVMEM_MFMA16(x == 2 || x == 3 ? lo[k + (x & 1u)] : hi[k + (x & 1u)], a, o[m]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        constexpr int T0 = OUT ? (Q0 + KS / 2) & 1 : Q0;  // where K^T's first group is
        if constexpr (DELTA) {
#pragma unroll
            for (uint32_t m = 0; m < 4; ++m) {
                first[m] = *reinterpret_cast<const f32x4_t *>(ch->from_first + 16u * m + 4u * g);
            }
            get_frags(frag_t, 0, tf);
        }
        // rows behind the last token repeat it: the factors' zeros meet them
        f32x4_t odd = zero;  // NaN where a value is not finite
#pragma unroll
        for (uint32_t m = 0; m < 4; ++m) {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                odd[r] = __builtin_fmaf(v[m][r], 0.0f, odd[r]);
            }
        }
        const float any_odd = (odd[0] + odd[1]) + (odd[2] + odd[3]);
        const float whole = ch->from_first[kChunk - 1];
        if constexpr (!DELTA) {
            decayed *= whole;
        }
        if (__builtin_expect(__any(any_odd != any_odd || ch->by_token != 0), 0)) {
            walk_tokens<T, DK>(p, s, row0, n, h, hk, col, with_out);
            continue;
        }
        half8_t dh[2], dl[2];
        if constexpr (DELTA) {
            f32x4_t rest[4];
#pragma unroll
            for (uint32_t m = 0; m < 4; ++m) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    rest[m][r] =
                        __builtin_fmaf(-first[m][r], __builtin_amdgcn_ldexpf(d[m][r], exp_k + exp_s), v[m][r]);
                }
                d[m] = zero;
            }
            const int exp_r = column_exp<4>(rest), e = exp_t + exp_r;
            split<4>(rest, exp_r, dh, dl);
#pragma unroll
            for (uint32_t k = 0; k < 2; ++k) {
#pragma unroll
                for (uint32_t x = 0; x < 3; ++x) {
#pragma unroll
                    for (uint32_t m = 2 * k; m < 4; ++m) {
                        d[m] = mul_lower<false>(tf + (x == 2 ? kLowerFrags : 0u), m, k, x == 1 ? dl[k] : dh[k], d[m]);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (OUT) {
                get_frags(frag_p, 0, pf);
            }
#pragma unroll
            for (int m = 0; m < 4; ++m) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    d[m][r] = __builtin_amdgcn_ldexpf(d[m][r], e);
                }
            }
        } else {
            if constexpr (OUT) {
                get_frags(frag_p, 0, pf);
            }
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                d[m] = v[m];
            }
        }
        f32x4_t last[4];
#pragma unroll
        for (uint32_t m = 0; m < 4; ++m) {
            last[m] = *reinterpret_cast<const f32x4_t *>(ch->to_last + 16u * m + 4u * g);
            out_first[m] = p.a.scale * ch->from_first[16u * m + (lane & 15u)];
        }
        const int exp_d = column_exp<4>(d);
        if constexpr (OUT) {
            f32x4_t pd[4] = {zero, zero, zero, zero};
            split<4>(d, exp_d, dh, dl);
#pragma unroll
            for (uint32_t k = 0; k < 2; ++k) {
#pragma unroll
                for (uint32_t x = 0; x < 3; ++x) {
#pragma unroll
                    for (uint32_t m = 2 * k; m < 4; ++m) {
                        pd[m] = mul_lower<true>(pf + (x == 2 ? kLowerFrags : 0u), m, k, x == 1 ? dl[k] : dh[k], pd[m]);
                    }
                }
            }
            uint8_t *out = p.a.out + (row0 * out_row + h * p.a.dim_v + col0 + 16u * w) * esz;
            int ed[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                es[r] += exp_q;
                ed[r] = __shfl(exp_d, static_cast<int>(4u * g) + r, 64) + exp_p;
            }
            float y[4][4];
#pragma unroll
            for (uint32_t m = 0; m < 4; ++m) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    // both terms as they are: the scale of a column of zeros or next to nothing
                    // would carry P D beyond fp32
                    y[m][r] = __builtin_fmaf(out_first[m], __builtin_amdgcn_ldexpf(o[m][r], es[r]),
                                             __builtin_amdgcn_ldexpf(pd[m][r], ed[r]));
                }
            }
            // one choice of the type for all four rows
            if (p.a.out_type == KVMEM_TYPE_F32) {
                store_rows<float>(out + out_at, 16u * out_row * esz, lane & 15u, rows, y);
            } else if (p.a.out_type == KVMEM_TYPE_F16) {
                store_rows<_Float16>(out + out_at, 16u * out_row * esz, lane & 15u, rows, y);
            } else {
                store_rows<__bf16>(out + out_at, 16u * out_row * esz, lane & 15u, rows, y);
            }
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            d[m] *= last[m];
        }
        // |d| to_last is at most 2^exp_last times what |d| was scaled to, and a finite
        // number times 2^-113 at most 2^15
        const int exp_x = min(exp_d + ch->exp_last, 113);
        split<4>(d, exp_x, dh, dl);
        const int exp_y = exp_x + exp_k;
        f32x4_t y[2][4];
        auto update = [&](uint32_t t0) {
#pragma unroll
            for (uint32_t t = 0; t < 4; ++t) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[t0 + t][r] = __builtin_fmaf(whole, s[t0 + t][r],
                                                  __builtin_amdgcn_ldexpf(y[(t0 / 4) & 1][t][r], exp_y));
                }
            }
        };
#pragma unroll
        for (uint32_t t0 = 0; t0 < TILES; t0 += 4) {  // four sums at a time, the four before added meanwhile
            if (t0 + 4 < TILES) {
                read8(kq[(T0 + t0 / 4 + 1) & 1], 8 * KS, t0 / 2 + 2);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (uint32_t k = 0; k < 2; ++k) {
                half8_t second[4];
                if constexpr (PARTS == 2) {
                    // together: one by one each would wait for memory where keys are not in LDS
                    // (F32, 256 x 256, without the delta rule: 2048 tokens of 8 heads 242 us, 170 so)
#pragma unroll
                    for (uint32_t t = 0; t < 4; ++t) {
                        second[t] = get_frag(kp, frag_index(8 * KS, 2 * (t0 + t) + k, 1));
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (uint32_t x = 0; x < (PARTS == 2 ? 3 : 2); ++x) {
#pragma unroll
                    for (uint32_t t = 0; t < 4; ++t) {
                        half8_t a;
                        if (x == 2) {
                            a = second[t];
                        } else {
                            a = kq[(T0 + t0 / 4) & 1][2 * t + k];
                        }
                        f32x4_t &to = y[(t0 / 4) & 1][t];
                        to = KVMEM_MFMA16(a, x == 1 ? dl[k] : dh[k], k == 0 && x == 0 ? zero : to);
                    }
                }
            }
            if (t0 >= 4) {
                update(t0 - 4);
                interleave<16, 2>();
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        update(TILES - 4);
    }
    if (!DELTA && seg < last_seg) {
        if (!p.second_pass) {
            float *made = p.seg_states + (seg_at + seg * p.a.n_head) * DK * p.a.dim_v + col;
#pragma unroll
            for (int d = 0; d < TILES; ++d) {
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r) {
                    made[static_cast<uint64_t>(16u * d + 4u * g + r) * p.a.dim_v] = s[d][r];
                }
            }
            if (col == 0 && g == 0) {
                p.seg_decays[seg_at + seg * p.a.n_head] = decayed;
            }
        }
        return;
    }
    if (p.a.state_out && rq.has_slot) {
#pragma unroll
        for (int d = 0; d < TILES; ++d) {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                p.a.state_out[at + static_cast<uint64_t>(16u * d + 4u * g + r) * p.a.dim_v] = s[d][r];
            }
        }
    }
}

// A workgroup takes a chunk of one key head for all its heads where those fill the
// CUs twice, else for one head.  48 heads of 16 key heads, the whole call: 1024 tokens
// (256 chunks of key heads) 79.8 us together and 75.4 alone, 2048 tokens 132 and 136,
// 8192 tokens 486 and 502.
constexpr uint32_t kPrepFull = 512;

template <typename T, int DK>
static void prepare(hipStream_t stream, const ChunkParams &p) {
    const uint64_t groups = static_cast<uint64_t>(p.chunks) * (p.a.n_head / p.a.group) * p.a.n_seq;
    const uint32_t heads = groups >= kPrepFull ? p.a.group : 1u;
    const dim3 grid(p.chunks * (p.a.n_head / heads), p.a.n_seq);
    if (p.delta) {
        linear_prepare_kernel<T, DK, true><<<grid, kPrepThreads, 0, stream>>>(p, heads);
    } else {
        linear_prepare_kernel<T, DK, false><<<grid, kPrepThreads, 0, stream>>>(p, heads);
    }
}

// 64 columns a workgroup where a head has them and two chunks of that width fit into
// LDS, else 32.  A chunk takes a wave the same time either way (one request of 8192
// tokens, 48 heads of 128 x 128: 486 us, 485 by 32), and wide workgroups read the
// operands half as often (eight of up to 4096 tokens, 32 heads: 385 us, 583 by 32).
template <typename T, int DK, bool DELTA, bool OUT>
static void walk_cols(hipStream_t stream, const ChunkParams &p) {
    constexpr bool wide = ChunkSpace<T, DK, DELTA, OUT, 4>::places == 2;
    const uint32_t cols = wide && p.a.dim_v % 64 == 0 ? 64u : 32u;
    const uint32_t units = p.a.n_head * (p.a.dim_v / cols);
    const dim3 grid((units + kXcds - 1) / kXcds * kXcds, p.a.n_seq, p.segs);
    if constexpr (wide) {
        if (cols == 64) {
            linear_walk_kernel<T, DK, DELTA, OUT, 4><<<grid, 512, 0, stream>>>(p);
            return;
        }
    }
    linear_walk_kernel<T, DK, DELTA, OUT, 2><<<grid, 256, 0, stream>>>(p);
}

template <typename T, int DK>
static void launch_type(hipStream_t stream, const ChunkParams &p) {
    prepare<T, DK>(stream, p);
    if (hipPeekAtLastError() != hipSuccess) {
        return;  // factors that were not written must not be read
    }
    if (p.delta) {
        p.outs ? walk_cols<T, DK, true, true>(stream, p) : walk_cols<T, DK, true, false>(stream, p);
        return;
    }
    p.outs ? walk_cols<T, DK, false, true>(stream, p) : walk_cols<T, DK, false, false>(stream, p);
    if (p.segs > 1 && hipPeekAtLastError() == hipSuccess) {
        const uint64_t quads = static_cast<uint64_t>(p.a.n_head) * p.dim_k * p.a.dim_v / 4;
        const dim3 grid(static_cast<uint32_t>((quads + kScanThreads - 1) / kScanThreads), p.a.n_seq);
        linear_scan_kernel<<<grid, kScanThreads, 0, stream>>>(p);
        if (hipPeekAtLastError() != hipSuccess) {
            return;
        }
        ChunkParams second = p;
        second.second_pass = 1;
        p.outs ? walk_cols<T, DK, false, true>(stream, second) : walk_cols<T, DK, false, false>(stream, second);
    }
}

template <typename T>
static void launch_dims(hipStream_t stream, const ChunkParams &p) {
    if (p.dim_k == 64) {
        launch_type<T, 64>(stream, p);
    } else if (p.dim_k == 128) {
        launch_type<T, 128>(stream, p);
    } else {
        launch_type<T, 256>(stream, p);
    }
}

}  // namespace kvmem_hip
