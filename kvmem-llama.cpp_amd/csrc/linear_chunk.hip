// Linear attention by chunks of 64 tokens, for prompts (the formulas are those of
// linear.hip; a_t = exp(log_decay_t), G_i the chunk's sum of log_decay up to token i).
// With S the state before the chunk, D the chunk's rows d_i, and
//     A_ij = beta_i (k_i . k_j) e^(G_i - G_j)   j < i
//     P_ij =        (q_i . k_j) e^(G_i - G_j)   j <= i
// the recurrence is, in products of matrices,
//     D  = (1 + A)^-1 diag(beta) (V - diag(e^G) K S)      (V itself without beta)
//     O  = scale (diag(e^G) Q S + P D)
//     S' = e^(G_last) S + K^T diag(e^(G_last - G)) D
// Two launches:
//   prepare  per (chunk, head): T = (1 + A)^-1 diag(beta) and P, which no state
//            enters, so all chunks at once; keys and queries as the matrix cores'
//            operands
//   walk     per (request, head, 16 or 32 columns of the state): the chunks in
//            order.  Columns of a state never meet, so a wave needs nothing of any
//            other: no barrier, no LDS.  It keeps its columns of S in accumulator
//            registers; a product's accumulator (4 consecutive rows per lane) serves
//            as the next product's operand as it is, because the order in which a
//            contraction runs over its 32 indices is free as long as both operands
//            follow it: lane group g's eight are {4g..4g+3, 16+4g..16+4g+3}.
//
// Precision: operands are f16 parts of scaled fp32 numbers.  Each matrix (for S, D
// and their like each column) is scaled by a power of two that puts its largest
// element into [2^11, 2^12), then split into a high and a low f16 part: together 22
// bits, and what lies below 2^-36 of the largest is cut.  16-bit keys and queries
// are one part, exactly.  Products of two split factors leave out low x low.  What
// reaches only a 16-bit result takes fewer parts: for a bf16 out (half a step
// 2^-9) the scores, D and S enter the output's products by their high part (half a
// step 2^-12).  Sums of log_decay are fp64: e^(G_i - G_j) of far apart sums
// keeps its digits, and a decay of zero (-inf, taken as -10^5) stays zero.
//
// A chunk with a number that is not finite among its rows, gates or factors goes
// token by token instead (walk_tokens), as products of masked rows would spread it
// to earlier tokens.
#include "kvmem_internal.hpp"

#include <algorithm>
#include <type_traits>

#include "linear.hpp"

namespace kvmem_hip {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr uint32_t kFragBytes = 1024;  // a 16 x 32 operand of f16: 16 bytes a lane
constexpr uint32_t kLowerFrags = 6;    // of a 64 x 64 lower triangle: (0,0) (1,0) (2,0) (2,1) (3,0) (3,1)
constexpr uint32_t kHeadBytes = 1024;  // a head's entry begins with ChunkHead

struct ChunkHead {
    float from_first[kChunk];  // e^G_i
    float to_last[kChunk];     // e^(G_last - G_i)
    int32_t exp_k, exp_q, exp_t, exp_p;
    uint32_t by_token;         // a number that is not finite
};
static_assert(sizeof(ChunkHead) <= kHeadBytes, "");

struct ChunkParams {
    LinearParams a;
    uint8_t *keys;   // [entries][key heads]: fragments of K, Q, K^T
    uint8_t *heads;  // [entries][heads]: ChunkHead, fragments of T, P
    uint64_t key_bytes, head_bytes;
    uint32_t chunks;
    int type;
    uint32_t dim_k;
    uint32_t delta, outs, p_parts;
    uint32_t cols;
};

__device__ inline uint64_t entry_of(const Request &rq, uint32_t s, uint32_t c) {
    return static_cast<uint64_t>(rq.first / kChunk) + s + c;
}

// The power of two that brings numbers whose largest magnitude has the bits `m`
// into [2^11, 2^12): x * 2^-e.  Kept inside what one fp32 factor can be.
__device__ inline int scale_exp(uint32_t m) {
    const int e = static_cast<int>(m >> 23) - (127 + 11);
    return m == 0 ? 0 : e < -100 ? -100 : e > 116 ? 116 : e;
}
__device__ inline float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
__device__ inline uint32_t mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr uint32_t kInf = 0x7f800000u;

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

__device__ inline uint32_t lower_frag(uint32_t m, uint32_t k) { return m < 2 ? m : 2u * m - 2u + k; }

// c += a b over 16 indices, fp32: a row of `a` is read from LDS rows, b's rows
// 4g..4g+3 of column lane % 16 are in registers (as an accumulator holds them).
__device__ inline f32x4_t mul16(const float *a_rows, f32x4_t b, f32x4_t c) {
    const uint32_t lane = threadIdx.x & 63u;
    const float4 a = *reinterpret_cast<const float4 *>(a_rows + (lane & 15u) * kTriPitch + 4u * (lane >> 4));
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b[2], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b[3], c, 0, 0, 0);
}

// K's and Q's parts, later A, T and P.
template <int DK, int PARTS> constexpr uint32_t prep_lds() {
    constexpr uint32_t rows = 2u * PARTS * kChunk * (DK + 8) * 2u;
    constexpr uint32_t tri = 3u * kChunk * kTriPitch * 4u;
    return rows > tri ? rows : tri;
}

template <typename T, int DK>
__global__ __launch_bounds__(kPrepThreads) void linear_prepare_kernel(const ChunkParams p) {
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    constexpr int KS = DK / 32;
    __shared__ __align__(16) uint8_t lds[prep_lds<DK, PARTS>()];
    __shared__ uint32_t words[16];
    const uint32_t h = blockIdx.x % p.a.n_head, c = blockIdx.x / p.a.n_head, s = blockIdx.y;
    const Request rq = request_of(p.a.batch, s);
    if (c * kChunk >= rq.count) {
        return;
    }
    const uint32_t n = min(kChunk, rq.count - c * kChunk);
    const uint64_t row0 = static_cast<uint64_t>(rq.first) + c * kChunk;
    const uint64_t entry = entry_of(rq, s, c);
    const uint32_t hk = h / p.a.group;
    uint8_t *keys = p.keys + (entry * (p.a.n_head / p.a.group) + hk) * p.key_bytes;
    uint8_t *head = p.heads + (entry * p.a.n_head + h) * p.head_bytes;
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // decays: every wave has all 64 sums, one a lane
    float decay = 0.0f, beta = 0.0f;
    if (lane < n) {
        if (p.a.decay) {
            decay = *reinterpret_cast<const float *>(p.a.decay + (row0 + lane) * p.a.decay_nb + h * 4u);
        }
        if (p.delta) {
            beta = *reinterpret_cast<const float *>(p.a.beta + (row0 + lane) * p.a.beta_nb + h * 4u);
        }
    }
    bool odd = !(decay < INFINITY) || !(mag(beta) < kInf);
    double G = decay < -1e5f ? -1e5 : static_cast<double>(decay);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const double y = __shfl_up(G, x, 64);
        G += lane >= static_cast<uint32_t>(x) ? y : 0.0;
    }
    const double G_last = __shfl(G, 63, 64);
    const float from_first = expf(static_cast<float>(G));
    const float to_last = expf(static_cast<float>(G_last - G));
    odd = odd || !(from_first < INFINITY) || !(to_last < INFINITY);

    RawRow<T, 8> raw_k[KS], raw_q[KS];
    load_rows<T, DK>(p.a.k + row0 * p.a.k_nb2 + hk * p.a.k_nb1, p.a.k_nb2, n, raw_k);
    uint32_t mk = max_mag<T, DK>(raw_k), mq = 0;
    if (p.outs) {
        load_rows<T, DK>(p.a.q + row0 * p.a.q_nb2 + hk * p.a.q_nb1, p.a.q_nb2, n, raw_q);
        mq = max_mag<T, DK>(raw_q);
    }
    block_max2(mk, mq, words);
    odd = odd || mk >= kInf || mq >= kInf;
    const int exp_k = scale_exp(mk), exp_q = scale_exp(mq);
    _Float16 *k16 = reinterpret_cast<_Float16 *>(lds);
    _Float16 *q16 = k16 + PARTS * kChunk * (DK + 8);
    put_rows<T, DK, PARTS>(raw_k, pow2(-exp_k), k16);
    if (p.outs) {
        put_rows<T, DK, PARTS>(raw_q, pow2(-exp_q), q16);
    }
    __syncthreads();

    // the key head's operands, by its first head
    if (h % p.a.group == 0) {
#pragma unroll
        for (uint32_t part = 0; part < PARTS; ++part) {
            const _Float16 *kp = k16 + part * kChunk * (DK + 8);
            const _Float16 *qp = q16 + part * kChunk * (DK + 8);
            uint8_t *out = keys + part * (12u * KS * kFragBytes);
#pragma unroll
            for (uint32_t k = 0; k < KS; ++k) {
                put_frag(out, w * KS + k, row_frag<DK>(kp, w, k));
                if (p.outs) {
                    put_frag(out, 4u * KS + w * KS + k, row_frag<DK>(qp, w, k));
                }
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
            if (p.delta) {
                kk[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, kk[j], 0, 0, 0);
                if constexpr (PARTS == 2) {
                    a2 = row_frag<DK>(k16 + kChunk * (DK + 8), w, k);
                    kk[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b2, kk[j], 0, 0, 0);
                    kk[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a2, b, kk[j], 0, 0, 0);
                }
            }
            if (p.outs) {
                const half8_t aq = row_frag<DK>(q16, w, k);
                qk[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(aq, b, qk[j], 0, 0, 0);
                if constexpr (PARTS == 2) {
                    a2 = row_frag<DK>(q16 + kChunk * (DK + 8), w, k);
                    qk[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(aq, b2, qk[j], 0, 0, 0);
                    qk[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a2, b, qk[j], 0, 0, 0);
                }
            }
        }
    }
    __syncthreads();  // K and Q are read: A, T and P take their place
    float *tri_a = reinterpret_cast<float *>(lds);
    float *tri_t = tri_a + kChunk * kTriPitch;
    float *tri_p = tri_t + kChunk * kTriPitch;
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
            const double Gi = __shfl(G, static_cast<int>(i), 64);
            const float bi = __shfl(beta, static_cast<int>(i), 64);
            const float f = expf(static_cast<float>(Gi - Gj));
            if (p.delta) {
                tri_a[i * kTriPitch + col] =
                    col < i ? __builtin_amdgcn_ldexpf(kk[j][r] * f, 2 * exp_k) * bi : 0.0f;
            }
            if (p.outs) {
                tri_p[i * kTriPitch + col] = col <= i ? __builtin_amdgcn_ldexpf(qk[j][r] * f, exp_k + exp_q) : 0.0f;
            }
        }
    }
    if (p.delta) {
        __syncthreads();
        // 1 + A's diagonal blocks inverted by forward substitution: lane (any, c) has
        // column c of block w
        const float *a = tri_a + 16u * w * kTriPitch + 16u * w;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float y = (lane & 15u) == static_cast<uint32_t>(i) ? 1.0f : 0.0f;
#pragma unroll
            for (int k = 0; k < i; ++k) {
                y = __builtin_fmaf(-a[i * kTriPitch + k], x[k], y);
            }
            x[i] = y;
        }
        float *t = tri_t + 16u * w * kTriPitch + 16u * w;
        if (g == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                t[i * kTriPitch + lane] = x[i];
            }
        }
        __syncthreads();
        // column w of blocks downwards: T_iw = -T_ii sum_k A_ik T_kw
        f32x4_t col[4];
        const float bw = __shfl(beta, static_cast<int>(16u * w + (lane & 15u)), 64);
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            col[0][r] = t[(4u * g + r) * kTriPitch + (lane & 15u)];
        }
        f32x4_t first = col[0];
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
        __syncthreads();  // the diagonal blocks are read: they are scaled by beta now too
#pragma unroll
        for (uint32_t d = 0; d < 4; ++d) {
            if (w + d < 4) {
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r) {
                    const float y = d == 0 ? first[r] : col[d][r];
                    tri_t[(16u * (w + d) + 4u * g + r) * kTriPitch + 16u * w + (lane & 15u)] = y * bw;
                }
            }
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
        if (p.delta) {
            tri_row(tri_t, w, k, xt[k]);
        }
        if (p.outs) {
            tri_row(tri_p, w, k, xp[k]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            mt = p.delta ? max(mt, mag(xt[k][i])) : 0u;
            mp = p.outs ? max(mp, mag(xp[k][i])) : 0u;
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
        const uint32_t f = lower_frag(w, k);
        uint8_t *at = head + kHeadBytes;
        half8_t hi, lo;
        if (p.delta) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = xt[k][i] * pow2(-exp_t);
                hi[i] = static_cast<_Float16>(y);
                lo[i] = static_cast<_Float16>(y - static_cast<float>(hi[i]));
            }
            put_frag(at, f, hi);
            put_frag(at, kLowerFrags + f, lo);
            at += 2u * kLowerFrags * kFragBytes;
        }
        if (p.outs) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = xp[k][i] * pow2(-exp_p);
                hi[i] = static_cast<_Float16>(y);
                lo[i] = static_cast<_Float16>(y - static_cast<float>(hi[i]));
            }
            put_frag(at, f, hi);
            if (p.p_parts == 2) {
                put_frag(at, kLowerFrags + f, lo);
            }
        }
    }
    if (w == 0) {
        ChunkHead *out = reinterpret_cast<ChunkHead *>(head);
        out->from_first[lane] = from_first;
        out->to_last[lane] = to_last;
        const bool any = __any(odd);
        if (lane == 0) {
            out->exp_k = exp_k;
            out->exp_q = exp_q;
            out->exp_t = exp_t;
            out->exp_p = exp_p;
            out->by_token = any;
        }
    }
}

// ---------------------------------------------------------------------- walk

__device__ inline float load_one(const uint8_t *p, int type, uint64_t i) {
    if (type == KVMEM_TYPE_F32) {
        return reinterpret_cast<const float *>(p)[i];
    }
    const uint16_t x = reinterpret_cast<const uint16_t *>(p)[i];
    return type == KVMEM_TYPE_F16 ? static_cast<float>(__builtin_bit_cast(_Float16, x))
                                  : __uint_as_float(static_cast<uint32_t>(x) << 16);
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

// A column's numbers (tiles of 16 rows, 4 of each in every lane of the column) as
// two f16 parts of x * 2^-e, e the column's own.
template <int TILES>
__device__ inline int split(const f32x4_t (&x)[TILES], half8_t (&hi)[TILES / 2], half8_t (&lo)[TILES / 2]) {
    uint32_t m = 0;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            m = max(m, mag(x[t][r]));
        }
    }
    m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 16, 64)));
    m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 32, 64)));
    const int e = scale_exp(m);
    const float f = pow2(-e);
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float y = x[t][r] * f;
            const _Float16 a = static_cast<_Float16>(y);
            hi[t / 2][4 * (t & 1) + r] = a;
            lo[t / 2][4 * (t & 1) + r] = static_cast<_Float16>(y - static_cast<float>(a));
        }
    }
    return e;
}

#define KVMEM_MFMA16(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0)

// A chunk's tokens one by one, on the wave's NT x 16 columns of the state (rows
// 16 d + 4 g + r in s[.][d][r]).
template <int DK, int NT>
__device__ inline __attribute__((always_inline)) void walk_tokens(const ChunkParams &p, f32x4_t (&s)[NT][DK / 16], uint64_t row0,
                                                      uint32_t n, uint32_t h, uint32_t hk, uint32_t col) {
    const uint32_t g = (threadIdx.x & 63u) >> 4;
    for (uint32_t t = 0; t < n; ++t) {
        const uint64_t row = row0 + t;
        const uint8_t *k = p.a.k + row * p.a.k_nb2 + hk * p.a.k_nb1;
        const float a = p.a.decay ? expf(*reinterpret_cast<const float *>(p.a.decay + row * p.a.decay_nb + h * 4u))
                                  : 1.0f;
        float kd[DK / 16][4];
#pragma unroll
        for (int d = 0; d < DK / 16; ++d) {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                kd[d][r] = load_one(k, p.type, 16u * d + 4u * g + r);
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float x = load_one(p.a.v + row * p.a.v_nb2 + h * p.a.v_nb1, p.type, col + 16u * j);
            if (p.delta) {
                float u = 0.0f;
#pragma unroll
                for (int d = 0; d < DK / 16; ++d) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        u = __builtin_fmaf(s[j][d][r], kd[d][r], u);
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
                    s[j][d][r] = __builtin_fmaf(kd[d][r], x, a * s[j][d][r]);
                }
            }
            if (p.outs) {
                const uint8_t *q = p.a.q + row * p.a.q_nb2 + hk * p.a.q_nb1;
                float o = 0.0f;
#pragma unroll
                for (int d = 0; d < DK / 16; ++d) {
#pragma unroll
                    for (uint32_t r = 0; r < 4; ++r) {
                        o = __builtin_fmaf(s[j][d][r], load_one(q, p.type, 16u * d + 4u * g + r), o);
                    }
                }
                o += __shfl_xor(o, 16, 64);
                o += __shfl_xor(o, 32, 64);
                if (g == 0) {
                    store_one(p.a.out, p.a.out_type, (row * p.a.n_head + h) * p.a.dim_v + col + 16u * j,
                              p.a.scale * o);
                }
            }
        }
    }
}

template <int N>
__device__ inline void get_frags(const uint8_t *base, uint32_t frag, half8_t (&x)[N]) {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        x[i] = get_frag(base, frag + i);
    }
}

// What a chunk needs first, requested while the chunk before it is computed.
template <int NT, int PARTS, int KEYS> struct ChunkRows {
    half8_t k[KEYS];                       // operands of K (delta rule)
    uint32_t v[NT][16];                    // values as they lie in memory, rows 16 m + 4 g + r
    uint32_t by_token;
};

struct ChunkGates {
    f32x4_t first[4], last[4];  // e^G, e^(G_last - G) of rows 16 m + 4 g + r
    float out_first[4];         // e^G of rows 16 m + lane % 16
    float whole;
    int exp_k, exp_q, exp_t, exp_p;
};

template <int DK, int NT, int PARTS, bool DELTA, bool FINE>
__global__ __launch_bounds__(64, 1) void linear_walk_kernel(const ChunkParams p) {
    constexpr int KS = DK / 32, TILES = DK / 16;
    // operands of a matrix of keys: all parts requested ahead where registers hold them
    constexpr bool AHEAD = DK * PARTS <= 128;
    constexpr bool LATE = DK * PARTS >= 256;  // K^T only once K's registers are free
    constexpr int KEYS = AHEAD && DELTA ? 4 * KS * PARTS : 1;
    constexpr int ROWS = AHEAD ? 4 * KS * PARTS : 1;
    typedef ChunkRows<NT, PARTS, KEYS> Rows;
    const uint32_t lane = threadIdx.x, g = lane >> 4;
    const uint32_t slices = p.a.dim_v / (16u * NT);
    const uint32_t h = blockIdx.x / slices, s_id = blockIdx.y;
    const uint32_t col = (blockIdx.x % slices) * (16u * NT) + (lane & 15u);
    const uint32_t hk = h / p.a.group;
    Request rq = request_of(p.a.batch, s_id);
    rq.first = __builtin_amdgcn_readfirstlane(rq.first);
    rq.count = __builtin_amdgcn_readfirstlane(rq.count);
    const uint64_t at = (static_cast<uint64_t>(rq.slot) * p.a.n_head + h) * DK * p.a.dim_v + col;
    const uint64_t entry0 = entry_of(rq, s_id, 0);
    const uint64_t key_step = p.key_bytes * (p.a.n_head / p.a.group), head_step = p.head_bytes * p.a.n_head;
    const uint8_t *keys = p.keys + entry0 * key_step + hk * p.key_bytes;
    const uint8_t *head = p.heads + entry0 * head_step + h * p.head_bytes;
    const uint8_t *values = p.a.v + rq.first * p.a.v_nb2 + h * p.a.v_nb1;

    // operand i of K (at 0), Q (4 KS) or K^T (8 KS), its first or second part
    auto frag_index = [](uint32_t matrix, uint32_t i, uint32_t part) { return part * 12u * KS + matrix + i; };
    auto request_rows = [&](uint32_t c, Rows &x) {
        const uint8_t *kp = keys + c * key_step;
        const ChunkHead *ch = reinterpret_cast<const ChunkHead *>(head + c * head_step);
        const uint32_t n = min(kChunk, rq.count - c * kChunk);
        x.by_token = ch->by_token;
        if constexpr (AHEAD && DELTA) {
#pragma unroll
            for (uint32_t part = 0; part < PARTS; ++part) {
#pragma unroll
                for (uint32_t i = 0; i < 4 * KS; ++i) {
                    x.k[part * 4 * KS + i] = get_frag(kp, frag_index(0, i, part));
                }
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < NT; ++j) {
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
                const uint32_t row = 16u * (i >> 2) + 4u * g + (i & 3u);
                const uint8_t *to = values + static_cast<uint64_t>(c * kChunk + min(row, n - 1u)) * p.a.v_nb2;
                if constexpr (PARTS == 2) {
                    x.v[j][i] = reinterpret_cast<const uint32_t *>(to)[col + 16u * j];
                } else {
                    x.v[j][i] = reinterpret_cast<const uint16_t *>(to)[col + 16u * j];
                }
            }
        }
    };

    f32x4_t s[NT][TILES];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int d = 0; d < TILES; ++d) {
            s[j][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    if (p.a.state && rq.has_slot) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int d = 0; d < TILES; ++d) {
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r) {
                    s[j][d][r] =
                        p.a.state[at + static_cast<uint64_t>(16u * d + 4u * g + r) * p.a.dim_v + 16u * j];
                }
            }
        }
    }
    const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
    Rows next;
    if (rq.count) {
        request_rows(0, next);
    }
    for (uint32_t c = 0; c * kChunk < rq.count; ++c) {
        const Rows x = next;
        const uint32_t n = min(kChunk, rq.count - c * kChunk);
        const uint64_t row0 = static_cast<uint64_t>(rq.first) + c * kChunk;
        const uint8_t *kp = keys + c * key_step;
        const uint8_t *frag_t = head + c * head_step + kHeadBytes;
        const uint8_t *frag_p = frag_t + (DELTA ? 2u * kLowerFrags * kFragBytes : 0u);
        half8_t qf[ROWS], tf[DELTA ? 2 * kLowerFrags : 1], pf[(FINE ? 2 : 1) * kLowerFrags], kt[ROWS];
        if constexpr (AHEAD) {
            if (p.outs) {
#pragma unroll
                for (uint32_t i = 0; i < 4 * KS * PARTS; ++i) {
                    qf[i] = get_frag(kp, frag_index(4 * KS, i % (4 * KS), i / (4 * KS)));
                }
            }
        }
        ChunkGates z;
        const ChunkHead *ch = reinterpret_cast<const ChunkHead *>(head + c * head_step);
#pragma unroll
        for (uint32_t m = 0; m < 4; ++m) {
            z.first[m] = *reinterpret_cast<const f32x4_t *>(ch->from_first + 16u * m + 4u * g);
            z.last[m] = *reinterpret_cast<const f32x4_t *>(ch->to_last + 16u * m + 4u * g);
            z.out_first[m] = ch->from_first[16u * m + (lane & 15u)];
        }
        z.exp_k = ch->exp_k, z.exp_q = ch->exp_q, z.exp_t = ch->exp_t, z.exp_p = ch->exp_p;
        z.whole = ch->from_first[kChunk - 1];
        if constexpr (DELTA) {
            get_frags(frag_t, 0, tf);
        }
        __builtin_amdgcn_sched_barrier(0);
        f32x4_t v[NT][4];
        uint32_t odd = x.by_token;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
                const uint32_t w = x.v[j][i];
                const float f = PARTS == 2 ? __uint_as_float(w)
                                : p.type == KVMEM_TYPE_F16
                                    ? static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w)))
                                    : __uint_as_float(w << 16);
                v[j][i >> 2][i & 3u] = 16u * (i >> 2) + 4u * g + (i & 3u) < n ? f : 0.0f;
                odd |= mag(v[j][i >> 2][i & 3u]) >= kInf;
            }
        }
        if (__builtin_expect(__any(odd), 0)) {
            walk_tokens<DK, NT>(p, s, row0, n, h, hk, col);
            if ((c + 1) * kChunk < rq.count) {
                request_rows(c + 1, next);
            }
            continue;
        }
        half8_t hi[NT][KS], lo[NT][KS];
        int exp_s[NT];
        f32x4_t d[NT][4], o[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            exp_s[j] = split<TILES>(s[j], hi[j], lo[j]);
            if constexpr (DELTA) {
#pragma unroll
                for (uint32_t m = 0; m < 4; ++m) {
                    d[j][m] = zero;
                }
#pragma unroll
                for (uint32_t k = 0; k < KS; ++k) {
#pragma unroll
                    for (uint32_t m = 0; m < 4; ++m) {
                        const uint32_t i = m * KS + k;
                        const half8_t a = AHEAD ? x.k[AHEAD ? i : 0] : get_frag(kp, frag_index(0, i, 0));
                        d[j][m] = KVMEM_MFMA16(a, hi[j][k], d[j][m]);
                        d[j][m] = KVMEM_MFMA16(a, lo[j][k], d[j][m]);
                        if constexpr (PARTS == 2) {
                            const half8_t b =
                                AHEAD ? x.k[AHEAD ? 4 * KS + i : 0] : get_frag(kp, frag_index(0, i, 1));
                            d[j][m] = KVMEM_MFMA16(b, hi[j][k], d[j][m]);
                        }
                    }
                }
            }
        }
        if (p.outs) {
            get_frags(frag_p, 0, pf);
        }
        if constexpr (AHEAD && !LATE) {
#pragma unroll
            for (uint32_t i = 0; i < 4 * KS * PARTS; ++i) {
                kt[i] = get_frag(kp, frag_index(8 * KS, i % (4 * KS), i / (4 * KS)));
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (p.outs) {  // transposed: columns of the state are rows of the accumulator
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (uint32_t m = 0; m < 4; ++m) {
                    o[j][m] = zero;
                }
#pragma unroll
                for (uint32_t k = 0; k < KS; ++k) {
#pragma unroll
                    for (uint32_t m = 0; m < 4; ++m) {
                        const uint32_t i = m * KS + k;
                        const half8_t a = AHEAD ? qf[AHEAD ? i : 0] : get_frag(kp, frag_index(4 * KS, i, 0));
                        o[j][m] = KVMEM_MFMA16(hi[j][k], a, o[j][m]);
                        if constexpr (FINE) {
                            o[j][m] = KVMEM_MFMA16(lo[j][k], a, o[j][m]);
                            if constexpr (PARTS == 2) {
                                const half8_t b =
                                    AHEAD ? qf[AHEAD ? 4 * KS + i : 0] : get_frag(kp, frag_index(4 * KS, i, 1));
                                o[j][m] = KVMEM_MFMA16(hi[j][k], b, o[j][m]);
                            }
                        }
                    }
                }
            }
        }
        if constexpr (DELTA) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                f32x4_t rest[4];
#pragma unroll
                for (int m = 0; m < 4; ++m) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        rest[m][r] = __builtin_fmaf(
                            -z.first[m][r], __builtin_amdgcn_ldexpf(d[j][m][r], z.exp_k + exp_s[j]), v[j][m][r]);
                    }
                }
                half8_t rh[2], rl[2];
                const int e = z.exp_t + split<4>(rest, rh, rl);
#pragma unroll
                for (uint32_t m = 0; m < 4; ++m) {
                    d[j][m] = zero;
#pragma unroll
                    for (uint32_t k = 0; k <= m / 2; ++k) {
                        const uint32_t f = lower_frag(m, k);
                        d[j][m] = KVMEM_MFMA16(tf[f], rh[k], d[j][m]);
                        d[j][m] = KVMEM_MFMA16(tf[f], rl[k], d[j][m]);
                        d[j][m] = KVMEM_MFMA16(tf[kLowerFrags + f], rh[k], d[j][m]);
                    }
                }
#pragma unroll
                for (int m = 0; m < 4; ++m) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        d[j][m][r] = __builtin_amdgcn_ldexpf(d[j][m][r], e);
                    }
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    d[j][m] = v[j][m];
                }
            }
        }
        if constexpr (AHEAD && LATE) {
#pragma unroll
            for (uint32_t i = 0; i < 4 * KS * PARTS; ++i) {
                kt[i] = get_frag(kp, frag_index(8 * KS, i % (4 * KS), i / (4 * KS)));
            }
        }
        if constexpr (!LATE) {
            if ((c + 1) * kChunk < rq.count) {
                request_rows(c + 1, next);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (p.outs) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                half8_t dh[2], dl[2];
                const int exp_d = split<4>(d[j], dh, dl);
                f32x4_t pd[4];
#pragma unroll
                for (uint32_t m = 0; m < 4; ++m) {
                    pd[m] = zero;
#pragma unroll
                    for (uint32_t k = 0; k <= m / 2; ++k) {
                        const uint32_t f = lower_frag(m, k);
                        pd[m] = KVMEM_MFMA16(dh[k], pf[f], pd[m]);
                        if constexpr (FINE) {
                            pd[m] = KVMEM_MFMA16(dl[k], pf[f], pd[m]);
                            pd[m] = KVMEM_MFMA16(dh[k], pf[kLowerFrags + f], pd[m]);
                        }
                    }
                }
                int es[4], ed[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    es[r] = __shfl(exp_s[j], static_cast<int>(4u * g) + r, 64) + z.exp_q;
                    ed[r] = __shfl(exp_d, static_cast<int>(4u * g) + r, 64) + z.exp_p;
                }
                const uint32_t dv = col - (lane & 15u) + 16u * j + 4u * g;
#pragma unroll
                for (uint32_t m = 0; m < 4; ++m) {
                    const uint32_t i = 16u * m + (lane & 15u);
                    float y[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        y[r] = p.a.scale * __builtin_fmaf(z.out_first[m], __builtin_amdgcn_ldexpf(o[j][m][r], es[r]),
                                                          __builtin_amdgcn_ldexpf(pd[m][r], ed[r]));
                    }
                    if (i < n) {
                        const uint64_t to = ((row0 + i) * p.a.n_head + h) * p.a.dim_v + dv;
                        if (p.a.out_type == KVMEM_TYPE_F32) {
                            store_row<float, 4>(p.a.out + to * 4, y);
                        } else if (p.a.out_type == KVMEM_TYPE_F16) {
                            store_row<_Float16, 4>(p.a.out + to * 2, y);
                        } else {
                            store_row<__bf16, 4>(p.a.out + to * 2, y);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                d[j][m] *= z.last[m];
            }
            half8_t dh[2], dl[2];
            const int e = split<4>(d[j], dh, dl) + z.exp_k;
#pragma unroll
            for (uint32_t t = 0; t < TILES; ++t) {
                f32x4_t y = zero;
#pragma unroll
                for (uint32_t k = 0; k < 2; ++k) {
                    const uint32_t i = 2u * t + k;
                    const half8_t a = AHEAD ? kt[AHEAD ? i : 0] : get_frag(kp, frag_index(8 * KS, i, 0));
                    y = KVMEM_MFMA16(a, dh[k], y);
                    y = KVMEM_MFMA16(a, dl[k], y);
                    if constexpr (PARTS == 2) {
                        const half8_t b = AHEAD ? kt[AHEAD ? 4 * KS + i : 0] : get_frag(kp, frag_index(8 * KS, i, 1));
                        y = KVMEM_MFMA16(b, dh[k], y);
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[j][t][r] = __builtin_fmaf(z.whole, s[j][t][r], __builtin_amdgcn_ldexpf(y[r], e));
                }
            }
        }
        if constexpr (LATE) {
            if ((c + 1) * kChunk < rq.count) {
                request_rows(c + 1, next);
            }
        }
    }
    if (p.a.state_out && rq.has_slot) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int d = 0; d < TILES; ++d) {
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r) {
                    p.a.state_out[at + static_cast<uint64_t>(16u * d + 4u * g + r) * p.a.dim_v + 16u * j] = s[j][d][r];
                }
            }
        }
    }
}

template <typename T, int DK>
static void prepare(hipStream_t stream, const ChunkParams &p) {
    linear_prepare_kernel<T, DK><<<dim3(p.chunks * p.a.n_head, p.a.n_seq), kPrepThreads, 0, stream>>>(p);
}

template <int DK, int NT, int PARTS>
static void walk(hipStream_t stream, const ChunkParams &p) {
    const dim3 grid(p.a.n_head * (p.a.dim_v / (16u * NT)), p.a.n_seq);
    const bool fine = p.p_parts == 2;  // the output takes both parts
    if (p.delta) {
        fine ? linear_walk_kernel<DK, NT, PARTS, true, true><<<grid, 64, 0, stream>>>(p)
             : linear_walk_kernel<DK, NT, PARTS, true, false><<<grid, 64, 0, stream>>>(p);
    } else {
        fine ? linear_walk_kernel<DK, NT, PARTS, false, true><<<grid, 64, 0, stream>>>(p)
             : linear_walk_kernel<DK, NT, PARTS, false, false><<<grid, 64, 0, stream>>>(p);
    }
}

template <int DK>
static void launch(hipStream_t stream, const ChunkParams &p) {
    if (p.type == KVMEM_TYPE_F32) {
        prepare<float, DK>(stream, p);
    } else if (p.type == KVMEM_TYPE_F16) {
        prepare<_Float16, DK>(stream, p);
    } else {
        prepare<__bf16, DK>(stream, p);
    }
    if (hipPeekAtLastError() != hipSuccess) {
        return;  // factors that were not written must not be read
    }
    if (p.type == KVMEM_TYPE_F32) {
        walk<DK, 1, 2>(stream, p);
    } else {
        walk<DK, 1, 1>(stream, p);
    }
}

bool load_linear_chunk_kernels() {
    return load_kernel_object(&linear_prepare_kernel<float, 64>);
}

ChunkPlan plan_chunks(const kvmem_hip_linear_args *a, uint32_t max_q) {
    ChunkPlan pl;
    if (max_q < kChunkFrom) {
        return pl;
    }
    pl.chunked = true;
    const uint32_t parts = a->type == KVMEM_TYPE_F32 ? 2 : 1;
    pl.p_parts = !a->out ? 0 : a->out_type == KVMEM_TYPE_BF16 ? 1 : 2;
    pl.chunks = (max_q + kChunk - 1) / kChunk;
    pl.entries = a->n_tokens / kChunk + a->n_seq + 1;
    pl.key_bytes = static_cast<uint64_t>(parts) * 12 * (a->head_dim_k / 32) * kFragBytes;
    pl.head_bytes = kHeadBytes + ((a->beta ? 2 : 0) + pl.p_parts) * kLowerFrags * kFragBytes;
    pl.cols = 16;
    pl.bytes = pl.entries * (pl.key_bytes * a->n_head_k + pl.head_bytes * a->n_head);
    return pl;
}

void launch_linear_chunks(hipStream_t stream, int type, uint32_t dim_k, const ChunkPlan &pl, const LinearParams &a,
                          uint8_t *workspace) {
    ChunkParams p{};
    p.a = a;
    p.keys = workspace;
    p.heads = workspace + pl.entries * pl.key_bytes * (a.n_head / a.group);
    p.key_bytes = pl.key_bytes;
    p.head_bytes = pl.head_bytes;
    p.chunks = pl.chunks;
    p.type = type;
    p.dim_k = dim_k;
    p.delta = a.beta != nullptr;
    p.outs = a.out != nullptr;
    p.p_parts = static_cast<uint32_t>(pl.p_parts);
    p.cols = pl.cols;
    if (dim_k == 64) {
        launch<64>(stream, p);
    } else if (dim_k == 128) {
        launch<128>(stream, p);
    } else {
        launch<256>(stream, p);
    }
}

}  // namespace kvmem_hip
