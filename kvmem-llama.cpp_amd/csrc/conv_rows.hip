// The short causal convolution of a recurrent layer's projections with its
// state, SiLU and the L2 norm of query and key heads, in one pass
// (kvmem_hip_conv_rows):
//     y[t][c] = act(bias[c] + sum_j weight[c][j] x[t - (width-1) + j][c])
//     y / sqrt(sum over a run of norm_dim channels of y^2 + eps)
//
// Each row is read once and written once: bytes bound it for many tokens, one
// trip to memory for few.  A lane owns 8 consecutive channels and walks a tile of
// tokens with the last width-1 rows in registers, so that a row is read again only
// where a tile begins; a wave spans 512 channels and a norm's run lies inside it,
// its sum an exchange between the run's lanes.  The wave of a request's first
// tile alone touches the request's state: it reads the old rows before it writes
// the new ones, lane by lane, so a state is updated in place without a race.
//
// Measured: 8191 tokens x 10240 channels of bf16, width 4, SiLU and norms of 4096
// channels 70 us = 4.8 TB/s of 336 MB read and written (a copy kernel reaches 6.07);
// vector instructions are 60 % of the busy cycles.  One token 4.7 us.  Rows of F32, whose
// SiLU carries its exponent's rounding and divides in full: 148 us = 4.5 TB/s of 671 MB,
// one token 6.2 us.
#include "kvmem_internal.hpp"

#include <algorithm>
#include <type_traits>

#include "recurrent.hpp"

namespace kvmem_hip {

constexpr uint32_t kConvThreads = 256;
constexpr uint32_t kConvWaves = kConvThreads / 64;
constexpr uint32_t kConvChannels = 512;  // of a wave
// Tokens of a wave's tile.  8191 tokens x 10240 channels of bf16, tiles of 8 / 16 / 32 /
// 64: 77.6 / 70.0 / 73.6 / 76.6 us (rows read again where tiles begin, against waves
// to fill the chip); 32 requests of 6 tokens 8.5 us with each.
constexpr uint32_t kConvTile = 16;
constexpr uint32_t kConvMaxWidth = 8;

struct ConvParams {
    BatchArgs batch;
    const uint8_t *x;
    uint64_t x_nb;
    const float *weight;
    const float *bias;
    const uint8_t *state;
    uint8_t *state_out;
    uint8_t *out;
    uint32_t n_channels;
    uint32_t blocks;         // of 512 channels
    uint32_t units;          // (tile, channel block) pairs of a request
    uint32_t norm_channels;
    uint32_t norm_lanes;     // lanes of a run
    float eps;
    bool silu;
    bool vec;                // 16 bytes at a time
    bool weight_vec;
    uint32_t tile;           // tokens
};

// The lane's 8 channels of a row; `n` of them exist (all or none where VEC).
template <typename T, bool VEC>
__device__ inline void load8(const uint8_t *p, uint32_t n, RawRow<T, 8> &r) {
    if constexpr (VEC) {
        load_raw<T, 8>(p, r);
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        if constexpr (sizeof(T) == 4) {
            r.w[i] = i < n ? reinterpret_cast<const uint32_t *>(p)[i] : 0u;
        } else {
            const uint32_t h = i < n ? reinterpret_cast<const uint16_t *>(p)[i] : 0u;
            r.w[i / 2] = i & 1 ? r.w[i / 2] | h << 16 : h;
        }
    }
}

template <typename T, bool VEC>
__device__ inline void store8(uint8_t *p, uint32_t n, const float x[8]) {
    if constexpr (VEC) {
        if (n) {
            store_row<T, 8>(p, x);
        }
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        if (i < n) {
            reinterpret_cast<T *>(p)[i] = static_cast<T>(x[i]);
        }
    }
}

// Sum over the `lanes` (a power of two) neighbours that hold a run.
__device__ inline float sum_lanes(float v, uint32_t lanes) {
    if (lanes > 1) v += lane_xor<1>(v);
    if (lanes > 2) v += lane_xor<2>(v);
    if (lanes > 4) v += lane_xor<4>(v);
    if (lanes > 8) v += lane_xor<8>(v);
    if (lanes > 16) v += lane_xor<16>(v);
    if (lanes > 32) v += lane_xor<32>(v);
    return v;
}

// y / (1 + e^-y).  For rows that stay fp32 the exponent's rounding, up to |y| half
// units of the result's last place, is carried along (log2 e in two parts).
template <bool EXACT>
__device__ inline float silu(float y) {
    constexpr float log2e = 0x1.715476p+0f;
    const float t = -y * log2e;
    float e = __builtin_amdgcn_exp2f(t);
    if constexpr (EXACT) {
        const float rest = __builtin_fmaf(-y, log2e, -t) - y * 0x1.4ae0bep-26f;
        // e^-y of 0 and infinity stay
        e = e < 0x1p126f ? __builtin_fmaf(e, rest * 0x1.62e430p-1f, e) : e;
        return y / (1.0f + e);
    }
    return y * __builtin_amdgcn_rcpf(1.0f + e);
}

// The norm of a run: 1 / sqrt(sum of squares + eps) times y.
__device__ inline void norm_run(const ConvParams &p, bool norm, float (&y)[8]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s = __builtin_fmaf(y[i], y[i], s);
    }
    s = sum_lanes(s, p.norm_lanes);
    float f = __builtin_amdgcn_rsqf(s + p.eps);
    // squares beyond fp32, or nothing of them left: fp64 holds them all
    if (__builtin_expect(__any(norm && !(s < 0x1p126f && s + p.eps > 0x1p-100f)), 0)) {
        double d = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            d = __builtin_fma(static_cast<double>(y[i]), static_cast<double>(y[i]), d);
        }
        for (uint32_t m = 1; m < p.norm_lanes; m <<= 1) {
            d += __shfl_xor(d, static_cast<int>(m), 64);
        }
        d += static_cast<double>(p.eps);
        const double g = d == 0.0 ? 0.0 : 1.0 / sqrt(d);
        if (norm) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[i] = static_cast<float>(static_cast<double>(y[i]) * g);
            }
        }
        f = 1.0f;
    }
    f = norm ? f : 1.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y[i] *= f;
    }
}

template <typename T, int W, bool VEC>
__global__ __launch_bounds__(kConvThreads) void conv_rows_kernel(const ConvParams p) {
    constexpr int U = 4;  // rows requested together
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t unit = blockIdx.x * kConvWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= p.units) {
        return;
    }
    const uint32_t tile = unit / p.blocks, block = unit % p.blocks;
    uint32_t c0 = (block * 64u + lane) * 8u;
    const uint32_t n = c0 < p.n_channels ? (p.n_channels - c0 < 8u ? p.n_channels - c0 : 8u) : 0u;
    c0 = n ? c0 : 0u;  // lanes without channels read the first ones and store nothing
    const Request rq = request_of(p.batch, blockIdx.y);
    const uint32_t t0 = tile * p.tile;
    if (tile != 0 && t0 >= rq.count) {
        return;
    }
    const uint64_t row_bytes = static_cast<uint64_t>(p.n_channels) * sizeof(T);
    const uint8_t *x = p.x + rq.first * p.x_nb + c0 * sizeof(T);
    const uint64_t entry = static_cast<uint64_t>(rq.slot) * (W - 1) * row_bytes + c0 * sizeof(T);
    const bool old = p.state && rq.has_slot;
    const uint32_t t1 = rq.count < t0 + p.tile ? rq.count : t0 + p.tile;

    if (p.out && t0 < t1) {
        float h[W - 1 + U][8];
        RawRow<T, 8> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            load8<T, VEC>(x + (t0 + u < t1 ? t0 + u : t1 - 1) * p.x_nb, n, raw[u]);
        }
        RawRow<T, 8> before[W - 1];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            before[j] = RawRow<T, 8>{};
            if (tile != 0) {
                load8<T, VEC>(x + (t0 - (W - 1) + j) * p.x_nb, n, before[j]);
            } else if (old) {
                load8<T, VEC>(p.state + entry + j * row_bytes, n, before[j]);
            }
        }
        float w[8 * W];
        const float *weight = p.weight + static_cast<uint64_t>(c0) * W;
        if (VEC && p.weight_vec) {
#pragma unroll
            for (int i = 0; i < 2 * W; ++i) {
                const float4 v = reinterpret_cast<const float4 *>(weight)[i];
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8 * W; ++i) {
                w[i] = static_cast<uint32_t>(i / W) < n ? weight[i] : 0.0f;
            }
        }
        float bias[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            bias[i] = p.bias && i < n ? p.bias[c0 + i] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            widen<T, 8>(before[j], h[j]);
        }
        const bool norm = n && c0 < p.norm_channels;
        const bool any_norm = block * kConvChannels < p.norm_channels;
        uint8_t *out = p.out + static_cast<uint64_t>(rq.first) * row_bytes + c0 * sizeof(T);
        for (uint32_t t = t0; t < t1; t += U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                widen<T, 8>(raw[u], h[W - 1 + u]);
            }
            if (t + U < t1) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t at = t + U + u;
                    load8<T, VEC>(x + (at < t1 ? at : t1 - 1) * p.x_nb, n, raw[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t + u >= t1) {
                    break;
                }
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    y[i] = bias[i];
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        y[i] = __builtin_fmaf(w[i * W + j], h[u + j][i], y[i]);
                    }
                }
                if (p.silu) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        y[i] = silu<sizeof(T) == 4>(y[i]);
                    }
                }
                if (any_norm) {
                    norm_run(p, norm, y);
                }
                store8<T, VEC>(out + (t + u) * row_bytes, n, y);
            }
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    h[j][i] = h[U + j][i];
                }
            }
        }
    }
    if (tile == 0 && p.state_out && rq.has_slot) {
        // the last W-1 of (old rows, new rows); ascending, so that in place a row is
        // read before it is overwritten
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            const uint32_t at = rq.count + j;
            RawRow<T, 8> r{};
            if (at >= W - 1) {
                load8<T, VEC>(x + static_cast<uint64_t>(at - (W - 1)) * p.x_nb, n, r);
            } else if (old) {
                load8<T, VEC>(p.state + entry + at * row_bytes, n, r);
            }
            float v[8];
            widen<T, 8>(r, v);
            store8<T, VEC>(p.state_out + entry + j * row_bytes, n, v);
        }
    }
}

template <typename T, int W>
static void launch_conv(hipStream_t stream, uint32_t width, dim3 grid, const ConvParams &p) {
    if constexpr (W <= static_cast<int>(kConvMaxWidth)) {
        if (width == W) {
            if (p.vec) {
                conv_rows_kernel<T, W, true><<<grid, kConvThreads, 0, stream>>>(p);
            } else {
                conv_rows_kernel<T, W, false><<<grid, kConvThreads, 0, stream>>>(p);
            }
        } else {
            launch_conv<T, W + 1>(stream, width, grid, p);
        }
    }
}

bool load_conv_rows_kernels() {
    return load_kernel_object(&conv_rows_kernel<float, 2, true>);
}

}  // namespace kvmem_hip

using namespace kvmem_hip;

extern "C" {

int kvmem_hip_conv_rows(kvmem_hip_ctx *ctx, const kvmem_hip_conv_args *a) {
    if (!ctx) {
        return KVMEM_HIP_ERR_INVALID;
    }
    if (!a) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "conv_rows: null arguments");
    }
    if (!float_type_ok(a->type)) {
        return fail(ctx, KVMEM_HIP_ERR_UNSUPPORTED, "conv_rows: rows must be F32, F16 or BF16");
    }
    if (a->width < 2 || a->width > kConvMaxWidth) {
        return fail(ctx, KVMEM_HIP_ERR_UNSUPPORTED, "conv_rows: width must be 2 to 8");
    }
    const uint32_t esz = float_type_size(a->type);
    if (a->n_channels == 0 || a->n_channels > (1u << 24)) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "conv_rows: 1 to 2^24 channels");
    }
    if (a->norm_channels) {
        if (a->norm_dim < 32 || a->norm_dim > 512 || (a->norm_dim & (a->norm_dim - 1))) {
            return fail(ctx, KVMEM_HIP_ERR_UNSUPPORTED, "conv_rows: norm_dim must be 32, 64, 128, 256 or 512");
        }
        if (a->norm_channels > a->n_channels || a->norm_channels % a->norm_dim) {
            return fail(ctx, KVMEM_HIP_ERR_INVALID, "conv_rows: norm_channels must be whole runs of the channels");
        }
        if (!(a->eps >= 0.0f)) {
            return fail(ctx, KVMEM_HIP_ERR_INVALID, "conv_rows: eps must not be negative");
        }
    }
    if (a->n_seq > 65535) {
        return fail(ctx, KVMEM_HIP_ERR_UNSUPPORTED, "conv_rows: at most 65535 requests");
    }
    if (a->n_tokens > (1u << 26)) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "conv_rows: too many tokens");
    }
    if (!a->out && !a->state_out) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "conv_rows: no destination");
    }
    if ((a->n_tokens && !a->x) || (a->out && !a->weight)) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "conv_rows: null rows or weights");
    }
    const uintptr_t rows = reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->state) |
                           reinterpret_cast<uintptr_t>(a->state_out) | reinterpret_cast<uintptr_t>(a->out) |
                           a->x_nb;
    const uintptr_t words = reinterpret_cast<uintptr_t>(a->weight) | reinterpret_cast<uintptr_t>(a->bias) |
                            reinterpret_cast<uintptr_t>(a->q_start) | reinterpret_cast<uintptr_t>(a->n_use) |
                            reinterpret_cast<uintptr_t>(a->slots);
    if (rows % esz || words % 4) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "conv_rows: arrays and strides must be aligned to their elements");
    }
    if (a->out && (a->out == a->x || a->out == a->state || a->out == a->state_out)) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "conv_rows: out must not overlap the other rows");
    }
    if (a->n_seq == 0) {
        return KVMEM_HIP_OK;
    }
    ConvParams p{};
    p.batch = {a->q_start, a->n_use, a->slots, a->n_tokens, a->q_start ? a->max_q : std::min(a->max_q, 1u),
               a->n_slots};
    p.x = static_cast<const uint8_t *>(a->x);
    p.x_nb = a->x_nb;
    p.weight = a->weight;
    p.bias = a->bias;
    p.state = static_cast<const uint8_t *>(a->state);
    p.state_out = static_cast<uint8_t *>(a->state_out);
    p.out = static_cast<uint8_t *>(a->out);
    p.n_channels = a->n_channels;
    p.norm_channels = a->norm_channels;
    p.norm_lanes = a->norm_channels ? a->norm_dim / 8 : 1;
    p.eps = a->eps;
    p.silu = a->silu != 0;
    p.vec = rows % 16 == 0 && a->n_channels % 8 == 0;
    p.blocks = (a->n_channels + kConvChannels - 1) / kConvChannels;
    const uint32_t most = std::min(p.batch.max_q, a->n_tokens);
    p.weight_vec = reinterpret_cast<uintptr_t>(a->weight) % 16 == 0;
    p.tile = kConvTile;
    const uint64_t tiles = a->out ? std::max(1u, (most + p.tile - 1) / p.tile) : 1u;
    const uint64_t units = tiles * p.blocks;
    // a dispatch counts its work items in 32 bits
    if ((units + kConvWaves - 1) / kConvWaves * kConvThreads * a->n_seq >= uint64_t{1} << 32) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "conv_rows: too many requests of max_q tokens for one launch");
    }
    p.units = static_cast<uint32_t>(units);
    (void) hipSetDevice(ctx->device);
    if (injected_fail(ctx, KVMEM_HIP_FAIL_LAUNCH, "conv_rows launch")) {
        return KVMEM_HIP_ERR_RUNTIME;
    }
    const dim3 grid((p.units + kConvWaves - 1) / kConvWaves, a->n_seq);
    if (a->type == KVMEM_TYPE_F32) {
        launch_conv<float, 2>(ctx->stream, a->width, grid, p);
    } else if (a->type == KVMEM_TYPE_F16) {
        launch_conv<_Float16, 2>(ctx->stream, a->width, grid, p);
    } else {
        launch_conv<__bf16, 2>(ctx->stream, a->width, grid, p);
    }
    return hip_ok(ctx, hipGetLastError(), "conv_rows launch") ? KVMEM_HIP_OK : KVMEM_HIP_ERR_RUNTIME;
}

}  // extern "C"
