// Device code shared by the kernels of recurrent layers (conv_rows.hip,
// linear.hip): a request's tokens and state slot from the batch's arrays, and
// rows of F32, F16 and BF16 in groups of consecutive elements.
#pragma once

#include "kvmem_internal.hpp"

#include <type_traits>

namespace kvmem_hip {

// The batch arrays of kvmem_hip_conv_args and kvmem_hip_linear_args.
struct BatchArgs {
    const uint32_t *q_start;
    const uint32_t *n_use;
    const uint32_t *slots;
    uint32_t n_tokens;
    uint32_t max_q;
    uint32_t n_slots;
};

struct Request {
    uint32_t first;  // row of token 0
    uint32_t count;  // tokens that take part
    uint32_t slot;   // state entry
    bool has_slot;
};

// Request s, with every length from device memory cut to the call's bounds.
__device__ inline Request request_of(const BatchArgs &b, uint32_t s) {
    Request r;
    uint32_t end = s < b.n_tokens ? s + 1u : s;
    r.first = s;
    if (b.q_start) {
        r.first = b.q_start[s];
        end = b.q_start[s + 1];
    }
    end = end < b.n_tokens ? end : b.n_tokens;
    r.count = end > r.first ? end - r.first : 0u;
    r.count = r.count < b.max_q ? r.count : b.max_q;
    if (b.n_use) {
        const uint32_t u = b.n_use[s];
        r.count = u < r.count ? u : r.count;
    }
    r.slot = b.slots ? b.slots[s] : s;
    r.has_slot = r.slot < b.n_slots;
    return r;
}

inline bool float_type_ok(int t) { return t == KVMEM_TYPE_F32 || t == KVMEM_TYPE_F16 || t == KVMEM_TYPE_BF16; }
inline uint32_t float_type_size(int t) { return t == KVMEM_TYPE_F32 ? 4u : 2u; }

// N consecutive elements as they lie in memory.
template <typename T, int N> struct RawRow {
    uint32_t w[N * sizeof(T) / 4];
};

template <typename T, int N>
__device__ inline void load_raw(const void *p, RawRow<T, N> &r) {
    constexpr int words = N * static_cast<int>(sizeof(T)) / 4;
    if constexpr (words % 4 == 0) {
#pragma unroll
        for (int i = 0; i < words / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
            r.w[4 * i] = v.x;
            r.w[4 * i + 1] = v.y;
            r.w[4 * i + 2] = v.z;
            r.w[4 * i + 3] = v.w;
        }
    } else {
        static_assert(words == 2, "rows of 8 or of multiples of 16 bytes");
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        r.w[0] = v.x;
        r.w[1] = v.y;
    }
}

template <typename T, int N>
__device__ inline void widen(const RawRow<T, N> &r, float x[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __uint_as_float(r.w[i]);
        } else if constexpr (std::is_same_v<T, __bf16>) {
            x[i] = __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
        } else {
            x[i] = static_cast<float>(
                __builtin_bit_cast(_Float16, static_cast<uint16_t>(i & 1 ? r.w[i / 2] >> 16 : r.w[i / 2])));
        }
    }
}

// Rounded once, to nearest even.
template <typename T, int N>
__device__ inline void store_row(void *p, const float x[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            reinterpret_cast<float4 *>(p)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        }
    } else {
        uint32_t w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            typedef T pair_t __attribute__((ext_vector_type(2)));
            const pair_t v = {static_cast<T>(x[2 * i]), static_cast<T>(x[2 * i + 1])};
            w[i] = __builtin_bit_cast(uint32_t, v);
        }
        if constexpr (N == 4) {
            *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 8; ++i) {
                reinterpret_cast<uint4 *>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            }
        }
    }
}

}  // namespace kvmem_hip
