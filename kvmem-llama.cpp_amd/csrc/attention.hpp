// Attention of new tokens over the pool's rows: what the kernels and the host
// side share (kvmem_hip_attention, attention.hip).
#pragma once

#include "kvmem_internal.hpp"

namespace kvmem_hip {

constexpr uint32_t kRowTile = 16;       // query rows of a decode workgroup
constexpr uint32_t kPrefillWaves = 8;
constexpr uint32_t kPrefillRows = 32 * kPrefillWaves;
constexpr uint32_t kWaves = 4;          // of a decode workgroup
// Softmax weights are 2^(x - top + shift) before they are rounded to f16.  A
// row's `top` follows its maximum only when that has grown by more than
// kTopSlack (log2), so the sums are rarely scaled down again; weights then stay
// below 2^15, and those down to 2^-20 of 2^top are normal f16 numbers.
constexpr float kWeightShift = 6.0f;
constexpr float kTopSlack = 9.0f;
constexpr float kLog2e = 1.4426950408889634f;

// Waves of the decode kernel on a SIMD.  Two, but one where a step's rows, on
// their way in registers, would make two spill: f16 or q8_0 rows of 256, f16 rows
// of 128 beside f16 or q8_0 ones.  One has as many bytes in flight.
// Two / one, in us, one request: q8_0, 256 wide, 32768 keys 57 / 31, q8_0 keys and
// q4_0 values, 65500 keys 58 / 42; f16, 128 wide, 32768 keys 38 / 31.  32 ragged
// ones up to 8192 keys, 128 wide: f16 183 / 136, q8_0 keys and f16 values 238 / 131.
// The other way round: q5_0, 256 wide, 131072 keys 75 / 82, q8_0, 128 wide, the 32
// 98 / 134.
constexpr int decode_waves(int tk, int tv, int d) {
    const bool wide_k = tk == KVMEM_TYPE_F16 || tk == KVMEM_TYPE_Q8_0;
    const bool wide_v = tv == KVMEM_TYPE_F16 || tv == KVMEM_TYPE_Q8_0;
    const bool half = tk == KVMEM_TYPE_F16 || tv == KVMEM_TYPE_F16;
    return (d == 256 && (wide_k || wide_v)) || (d == 128 && wide_k && wide_v && half) ? 1 : 2;
}

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
    uint32_t room;              // keys the table and max_kv leave room for, at least 1
    uint32_t chunk;             // keys of one part
    uint32_t n_parts;           // parts of the longest request
    uint32_t T_mul, T_shift;    // j / T as the upper word of j * T_mul, shifted (T > 1)
    uint32_t row_tile;          // rows of one workgroup
    uint32_t row_tiles;         // of the longest request
    uint32_t units;             // decode: (request, part) pairs, padded to a multiple of 8;
                                // prefill: (request, part, KV head)
    int32_t causal;
    int32_t q_bf16;
    int32_t out_type;
    uint32_t hadamard;
    uint32_t join_one;          // rows of a single part are joined (and rotated) too
    float scale;
};

// The block of key j < 2^31.
__device__ inline uint32_t block_of(const AttnParams &p, uint32_t j) {
    return p.T == 1u ? j : __umulhi(j, p.T_mul) >> p.T_shift;
}

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


// E neighbouring output elements, from element e.
template <int E>
__device__ inline void store_elems(uint8_t *out, int type, uint64_t e, const float *x) {
    typedef float f_t __attribute__((ext_vector_type(E)));
    typedef _Float16 h_t __attribute__((ext_vector_type(E)));
    typedef __bf16 b_t __attribute__((ext_vector_type(E)));
    f_t v;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        v[i] = x[i];
    }
    if (type == KVMEM_TYPE_F32) {
        *reinterpret_cast<f_t *>(out + 4 * e) = v;
    } else if (type == KVMEM_TYPE_F16) {
        *reinterpret_cast<h_t *>(out + 2 * e) = __builtin_convertvector(v, h_t);
    } else {
        *reinterpret_cast<b_t *>(out + 2 * e) = __builtin_convertvector(v, b_t);
    }
}

// Walsh-Hadamard rotation of rows of which each lane holds E neighbouring
// elements (a run of `width` stands in width / E lanes from a multiple of that):
// butterflies of span 1 .. E/2 inside the lane, the others with lane ^ span/E.
// All lanes of the wave call.
template <uint32_t M, int E>
__device__ inline void rotate_span(float *x, uint32_t lane) {
    const bool upper = lane & M;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float y = lane_xor<M>(x[i]);
        x[i] = upper ? y - x[i] : x[i] + y;
    }
}
template <int E>
__device__ inline void rotate_lanes(float *x, uint32_t width, uint32_t lane) {
    const float f = 1.0f / sqrtf(static_cast<float>(width));
#pragma unroll
    for (int i = 0; i < E; ++i) {
        x[i] *= f;
    }
#pragma unroll
    for (int h = 1; h < E; h <<= 1) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (!(i & h)) {
                const float u = x[i];
                const float v = x[i + h];
                x[i] = u + v;
                x[i + h] = u - v;
            }
        }
    }
    // width is at least 64
    rotate_span<1, E>(x, lane);
    rotate_span<2, E>(x, lane);
    rotate_span<4, E>(x, lane);
    rotate_span<8, E>(x, lane);
    if (width > 16u * E) {
        rotate_span<16, E>(x, lane);
    }
    if (width > 32u * E) {
        rotate_span<32, E>(x, lane);
    }
}

// How a call is laid out on the chip.
struct AttnPlan {
    bool prefill;              // the kernel for many queries
    uint32_t row_tile, row_tiles, chunk, n_parts, units;
    uint64_t grid;
    bool joined;               // a joining kernel follows
    size_t o_bytes, ml_bytes;  // workspace: sums, then maxima and weights
};

// Keys of a step: about the same bytes for every head size (9 KiB of q4_0 keys
// and values), enough in flight per compute unit to stream.
constexpr uint32_t step_keys(uint32_t d) { return 32u * (256u / d); }
// Launches the decode or prefill kernel of key type TK (one translation unit
// each).
template <int TK>
void launch_attention(hipStream_t stream, int type_v, uint32_t head_dim, const AttnPlan &pl, const AttnParams &p);
// Loads the unit's kernels onto the device (a first launch inside a capture must not).
template <int TK>
bool load_attention();
extern template bool load_attention<KVMEM_TYPE_Q4_0>();
extern template bool load_attention<KVMEM_TYPE_Q5_0>();
extern template bool load_attention<KVMEM_TYPE_Q8_0>();
extern template bool load_attention<KVMEM_TYPE_F16>();
extern template void launch_attention<KVMEM_TYPE_Q4_0>(hipStream_t, int, uint32_t, const AttnPlan &, const AttnParams &);
extern template void launch_attention<KVMEM_TYPE_Q5_0>(hipStream_t, int, uint32_t, const AttnPlan &, const AttnParams &);
extern template void launch_attention<KVMEM_TYPE_Q8_0>(hipStream_t, int, uint32_t, const AttnPlan &, const AttnParams &);
extern template void launch_attention<KVMEM_TYPE_F16>(hipStream_t, int, uint32_t, const AttnPlan &, const AttnParams &);

}  // namespace kvmem_hip
