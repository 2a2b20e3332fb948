// Linear attention through a decaying state per request and head
// (kvmem_hip_linear_attention): with a = exp(log_decay), for each token
//     d = v                         (or d = beta (v - a S^T k), the delta rule)
//     o = scale (a S^T q + (k . q) d)
//     S = a S + k (x) d
#include "kvmem_internal.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "linear.hpp"

namespace kvmem_hip {

// ------------------------------------------------------------ token by token
// A wave owns 32 columns of a head's state for all the request's tokens: lane
// (r, c) of 8 x 8 keeps rows [r*R, r*R + R) of columns 4c..4c+3 in registers, so
// that a row of the state is a whole 128-byte line of 8 lanes.  The columns of a
// state never meet (S^T k and S^T q are sums over rows): waves need nothing of
// each other, and a token costs one exchange over the 8 row groups, S^T k and
// S^T q together (o follows from the old state: S' ^T q = a S^T q + (k . q) d).
// Bytes bound it: the state is read once and written once.  Measured, 48 heads of 128 x
// 128: 64 requests of a token 80 us = 5.0 TB/s of 405 MB (a copy kernel reaches 6.07);
// 8 requests of 6 tokens 14.6 us, 52 MB, then a wave's 1.2 us a token, dependent
// products and exchanges; one token of one request 4.1 us.
// By 16 columns a wave, whose rows are half lines: 107, 16.8 and 3.9 us.
constexpr uint32_t kStepCols = 32;

template <typename T, int R> struct StepRows {
    RawRow<T, R> k, q;
    RawRow<T, 4> v;
    float decay, beta;
};

template <typename T, int R>
__device__ inline void load_step(const LinearParams &p, uint64_t row, uint32_t h, uint32_t hk, uint32_t r, uint32_t c,
                                 StepRows<T, R> &s) {
    load_raw<T, R>(p.k + row * p.k_nb2 + hk * p.k_nb1 + r * (R * sizeof(T)), s.k);
    if (p.out) {
        load_raw<T, R>(p.q + row * p.q_nb2 + hk * p.q_nb1 + r * (R * sizeof(T)), s.q);
    }
    load_raw<T, 4>(p.v + row * p.v_nb2 + h * p.v_nb1 + c * sizeof(T), s.v);
    s.decay = p.decay ? *reinterpret_cast<const float *>(p.decay + row * p.decay_nb + h * 4u) : 0.0f;
    s.beta = p.beta ? *reinterpret_cast<const float *>(p.beta + row * p.beta_nb + h * 4u) : 0.0f;
}

// Moves between lanes by the VALU: through LDS six tokens of eight requests take 15.2
// us for 14.6.
__device__ inline float sum_row_groups(float v) {
    v += lane_xor<8>(v);
    auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

template <typename T, int DK>
__global__ __launch_bounds__(64) void linear_step_kernel(const LinearParams p) {
    constexpr int R = DK / 8;
    const uint32_t lane = threadIdx.x;
    const uint32_t r = lane >> 3;
    const uint32_t h = blockIdx.x / p.slices;
    const uint32_t c = (blockIdx.x % p.slices) * kStepCols + (lane & 7u) * 4u;
    const uint32_t hk = h / p.group;
    const Request rq = request_of(p.batch, blockIdx.y);
    const uint64_t entry = ((static_cast<uint64_t>(rq.slot) * p.n_head + h) * DK + r * R) * p.dim_v + c;
    float s[R][4];
    if (p.state && rq.has_slot) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float4 x = *reinterpret_cast<const float4 *>(p.state + entry + static_cast<uint64_t>(i) * p.dim_v);
            s[i][0] = x.x, s[i][1] = x.y, s[i][2] = x.z, s[i][3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
        }
    }
    StepRows<T, R> next;
    if (rq.count) {
        load_step<T, R>(p, rq.first, h, hk, r, c, next);
    }
    for (uint32_t t = 0; t < rq.count; ++t) {
        const StepRows<T, R> now = next;
        if (t + 1 < rq.count) {
            load_step<T, R>(p, rq.first + t + 1, h, hk, r, c, next);
        }
        float k[R], v[4];
        widen<T, R>(now.k, k);
        widen<T, 4>(now.v, v);
        const float a = p.decay ? expf(now.decay) : 1.0f;
        float d[4] = {v[0], v[1], v[2], v[3]};
        float u[4] = {}, w[4] = {}, kq = 0.0f;
        if (p.beta) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u[j] = __builtin_fmaf(s[i][j], k[i], u[j]);
                }
            }
        }
        if (p.out) {
            float q[R];
            widen<T, R>(now.q, q);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                kq = __builtin_fmaf(k[i], q[i], kq);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[j] = __builtin_fmaf(s[i][j], q[i], w[j]);
                }
            }
        }
        if (p.beta) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                d[j] = now.beta * __builtin_fmaf(-a, sum_row_groups(u[j]), v[j]);
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = __builtin_fmaf(k[i], d[j], a * s[i][j]);
            }
        }
        if (p.out) {
            kq = sum_row_groups(kq);
            float o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = p.scale * __builtin_fmaf(kq, d[j], a * sum_row_groups(w[j]));
            }
            if (r == 0) {
                const uint64_t at = ((static_cast<uint64_t>(rq.first) + t) * p.n_head + h) * p.dim_v + c;
                if (p.out_type == KVMEM_TYPE_F32) {
                    store_row<float, 4>(p.out + at * 4, o);
                } else if (p.out_type == KVMEM_TYPE_F16) {
                    store_row<_Float16, 4>(p.out + at * 2, o);
                } else {
                    store_row<__bf16, 4>(p.out + at * 2, o);
                }
            }
        }
    }
    if (p.state_out && rq.has_slot) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            *reinterpret_cast<float4 *>(p.state_out + entry + static_cast<uint64_t>(i) * p.dim_v) =
                make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
        }
    }
}

template <typename T>
static void launch_step(hipStream_t stream, uint32_t dim_k, const LinearParams &p) {
    const dim3 grid(p.n_head * p.slices, p.n_seq);
    if (dim_k == 64) {
        linear_step_kernel<T, 64><<<grid, 64, 0, stream>>>(p);
    } else if (dim_k == 128) {
        linear_step_kernel<T, 128><<<grid, 64, 0, stream>>>(p);
    } else {
        linear_step_kernel<T, 256><<<grid, 64, 0, stream>>>(p);
    }
}

bool load_linear_kernels() {
    return load_kernel_object(&linear_step_kernel<float, 64>) && load_linear_chunks_f32() &&
           load_linear_chunks_f16() && load_linear_chunks_bf16();
}

// Tokens a request from which a call goes by chunks.  A chunk costs the same for one
// token as for 64, and the chunks' kernels take longer to begin; token by token, a wave
// alone on its SIMD needs 1.2 us a token, and many share the FMAs.  Measured, us by
// chunks / by tokens, 48 heads of 128 x 128 (192 waves of states a request):
//   bf16, 1 request    16 tokens 17.6 /  20.9    12 tokens  17.6 /  16.6
//   bf16, 8 requests   24 tokens 40.3 /  35.9    32 tokens  41.0 /  44.7
//   bf16, 64 requests  56 tokens 296  /  283     64 tokens  298  /  318
//   F32, 1 request     16 tokens 20.7 /  20.6    24 tokens  21.1 /  29.5
//   F32, 8 requests    32 tokens 62.5 /  46.3    48 tokens  62.9 /  63.4
//   F32, 64 requests  128 tokens 722  /  633    192 tokens  876  /  927
// Heads of 64 x 64 cross near there (F16, 8 heads without the delta rule, 64 requests: 32
// tokens 25.2 / 26.7; F32, 64 heads, 64 requests: 192 tokens 482 / 483).  16 heads of 256 x
// 256 do for 8 requests (32 tokens 53.9 / 64.3), for 64 requests only from some 90 tokens
// on (64 tokens 435 / 390, 80 tokens 497 / 474).
static uint32_t chunk_from(const kvmem_hip_linear_args *a) {
    const uint64_t waves = static_cast<uint64_t>(a->n_seq) * a->n_head * (a->head_dim_v / kStepCols);
    const bool f32 = a->type == KVMEM_TYPE_F32;
    if (waves < 4096) {
        return f32 && waves >= 1024 ? 48 : 24;
    }
    return f32 ? 256 : 56;
}

static ChunkPlan plan_chunks(const kvmem_hip_linear_args *a, uint32_t max_q) {
    ChunkPlan pl;
    if (a->n_seq == 0 || max_q < chunk_from(a)) {
        return pl;
    }
    pl.chunked = true;
    const uint32_t parts = a->type == KVMEM_TYPE_F32 ? 2 : 1;
    pl.chunks = (max_q + kChunk - 1) / kChunk;
    pl.entries = a->n_tokens / kChunk + a->n_seq;
    pl.key_bytes = static_cast<uint64_t>(parts) * 12 * (a->head_dim_k / 32) * kFragBytes;
    pl.head_bytes = kHeadBytes + ((a->beta ? 2 : 0) + (a->out ? 2 : 0)) * kLowerFrags * kFragBytes;
    pl.bytes = pl.entries * (pl.key_bytes * a->n_head_k + pl.head_bytes * a->n_head);
    // Without the delta rule states add up: what a segment of chunks adds is made before
    // what lies behind it is known, in a first pass, and a second one walks the segments
    // again.  Worth it where the CUs are a quarter full or less and segments hold enough
    // chunks to pay for their states' traffic.  One piece / segments, us: F16, heads of
    // 64 x 64, 8 heads, 1024 tokens 41.5 / 24.2, 8192 tokens 251 / 47, eight requests of
    // up to 4096 tokens 145 / 96; bf16, 32 heads of 128 x 128, 8192 tokens 375 / 240; F32,
    // 8 heads of 256 x 256, 2048 tokens 292 / 170; what the conditions leave whole: bf16, 16
    // heads of 256 x 256, 1024 tokens 94.6 / 100 and 4096 tokens 333 / 340, 32 heads of
    // 128 x 128, two requests of up to 2048 tokens 111 / 121.
    const bool narrow = a->head_dim_v % 64 || a->head_dim_k * float_type_size(a->type) > 256;  // 32 columns a workgroup
    const uint64_t groups = static_cast<uint64_t>(a->n_seq) * a->n_head * (a->head_dim_v / (narrow ? 32 : 64));
    const uint32_t segs = static_cast<uint32_t>(std::min<uint64_t>(256 / groups, pl.chunks / (a->head_dim_k / 32)));
    if (!a->beta && segs >= 4) {
        pl.seg_chunks = (pl.chunks + segs - 1) / segs;
        pl.segs = (pl.chunks + pl.seg_chunks - 1) / pl.seg_chunks;
        const uint64_t entries = static_cast<uint64_t>(a->n_seq) * pl.segs * a->n_head;
        pl.seg_states = pl.bytes;
        pl.seg_decays = pl.seg_states + entries * a->head_dim_k * a->head_dim_v * sizeof(float);
        pl.bytes = (pl.seg_decays + entries * sizeof(float) + 15) / 16 * 16;
    }
    return pl;
}

static void launch_linear_chunks(hipStream_t stream, int type, uint32_t dim_k, const ChunkPlan &pl,
                                 const LinearParams &a, uint8_t *workspace) {
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
    p.segs = pl.segs;
    p.seg_chunks = pl.seg_chunks;
    p.seg_states = reinterpret_cast<float *>(workspace + pl.seg_states);
    p.seg_decays = reinterpret_cast<float *>(workspace + pl.seg_decays);
    if (type == KVMEM_TYPE_F32) {
        launch_linear_chunks_f32(stream, p);
    } else if (type == KVMEM_TYPE_F16) {
        launch_linear_chunks_f16(stream, p);
    } else {
        launch_linear_chunks_bf16(stream, p);
    }
}

// Tokens of a request, at most.
static uint32_t most_tokens(const kvmem_hip_linear_args *a) {
    return std::min(a->q_start ? a->max_q : std::min(a->max_q, 1u), a->n_tokens);
}

// What is wrong with a call's arguments (null: nothing), and its status.
static const char *check_linear(const kvmem_hip_linear_args *a, int &code) {
    code = KVMEM_HIP_ERR_INVALID;
    if (!a) {
        return "linear_attention: null arguments";
    }
    if (!float_type_ok(a->type) || !float_type_ok(a->out_type)) {
        code = KVMEM_HIP_ERR_UNSUPPORTED;
        return "linear_attention: rows must be F32, F16 or BF16";
    }
    if ((a->head_dim_k != 64 && a->head_dim_k != 128 && a->head_dim_k != 256) || a->head_dim_v == 0 ||
        a->head_dim_v % 32 || a->head_dim_v > 512) {
        code = KVMEM_HIP_ERR_UNSUPPORTED;
        return "linear_attention: head_dim_k must be 64, 128 or 256, head_dim_v a multiple of 32 up to 512";
    }
    if (a->n_head_k == 0 || a->n_head == 0 || a->n_head > 4096 || a->n_head % a->n_head_k) {
        return "linear_attention: 1 to 4096 heads, a multiple of the key heads";
    }
    if (a->n_seq > 65535) {
        code = KVMEM_HIP_ERR_UNSUPPORTED;
        return "linear_attention: at most 65535 requests";
    }
    if (a->n_tokens > (1u << 26)) {
        return "linear_attention: too many tokens";
    }
    if (!a->out && !a->state_out) {
        return "linear_attention: no destination";
    }
    if (a->n_tokens && (!a->k || !a->v || (a->out && !a->q))) {
        return "linear_attention: null rows";
    }
    uintptr_t rows = reinterpret_cast<uintptr_t>(a->k) | a->k_nb1 | a->k_nb2 | reinterpret_cast<uintptr_t>(a->v) |
                     a->v_nb1 | a->v_nb2 | reinterpret_cast<uintptr_t>(a->state) |
                     reinterpret_cast<uintptr_t>(a->state_out) | reinterpret_cast<uintptr_t>(a->out);
    if (a->out) {
        rows |= reinterpret_cast<uintptr_t>(a->q) | a->q_nb1 | a->q_nb2;
    }
    if (rows % 16) {
        return "linear_attention: rows, strides, states and out must be 16-byte aligned";
    }
    const uintptr_t words = reinterpret_cast<uintptr_t>(a->log_decay) | reinterpret_cast<uintptr_t>(a->beta) |
                            a->decay_nb | a->beta_nb | reinterpret_cast<uintptr_t>(a->q_start) |
                            reinterpret_cast<uintptr_t>(a->n_use) | reinterpret_cast<uintptr_t>(a->slots);
    if (words % 4) {
        return "linear_attention: arrays must be 4-byte aligned";
    }
    if (a->out && (a->out == a->q || a->out == a->k || a->out == a->v || a->out == a->state ||
                   a->out == a->state_out)) {
        return "linear_attention: out must not overlap the other arrays";
    }
    if (!(a->scale >= 0.0f) || std::isinf(a->scale)) {
        return "linear_attention: scale must not be negative";
    }
    // a dispatch counts its work items in 32 bits
    const ChunkPlan pl = plan_chunks(a, most_tokens(a));
    const uint64_t waves = static_cast<uint64_t>(a->n_head) * 
                               ((a->head_dim_v + 31) / 32) + kXcds;
    const uint64_t chunks = static_cast<uint64_t>(a->n_head) * pl.chunks;
    if (std::max(waves * 256, chunks * kPrepThreads) * a->n_seq >= uint64_t{1} << 32) {
        return "linear_attention: too many requests for one launch";
    }
    code = KVMEM_HIP_OK;
    return nullptr;
}

}  // namespace kvmem_hip

using namespace kvmem_hip;

extern "C" {

size_t kvmem_hip_linear_attention_workspace(const kvmem_hip_linear_args *a) {
    int code = 0;
    if (check_linear(a, code) || a->n_seq == 0) {
        return 0;
    }
    return plan_chunks(a, most_tokens(a)).bytes;
}

int kvmem_hip_linear_attention(kvmem_hip_ctx *ctx, const kvmem_hip_linear_args *a) {
    if (!ctx) {
        return KVMEM_HIP_ERR_INVALID;
    }
    int code = 0;
    if (const char *why = check_linear(a, code)) {
        return fail(ctx, code, why);
    }
    if (a->n_seq == 0) {
        return KVMEM_HIP_OK;
    }
    LinearParams p{};
    p.batch = {a->q_start, a->n_use, a->slots, a->n_tokens, a->q_start ? a->max_q : std::min(a->max_q, 1u),
               a->n_slots};
    p.q = static_cast<const uint8_t *>(a->q);
    p.k = static_cast<const uint8_t *>(a->k);
    p.v = static_cast<const uint8_t *>(a->v);
    p.q_nb1 = a->q_nb1, p.q_nb2 = a->q_nb2;
    p.k_nb1 = a->k_nb1, p.k_nb2 = a->k_nb2;
    p.v_nb1 = a->v_nb1, p.v_nb2 = a->v_nb2;
    p.decay = reinterpret_cast<const uint8_t *>(a->log_decay);
    p.beta = reinterpret_cast<const uint8_t *>(a->beta);
    p.decay_nb = a->decay_nb;
    p.beta_nb = a->beta_nb;
    p.state = a->state;
    p.state_out = a->state_out;
    p.out = static_cast<uint8_t *>(a->out);
    p.out_type = a->out_type;
    p.n_seq = a->n_seq;
    p.n_head = a->n_head;
    p.group = a->n_head / a->n_head_k;
    p.dim_v = a->head_dim_v;
    p.slices = a->head_dim_v / kStepCols;
    p.scale = a->scale > 0.0f ? a->scale : 1.0f / sqrtf(static_cast<float>(a->head_dim_k));
    (void) hipSetDevice(ctx->device);
    const ChunkPlan pl = plan_chunks(a, most_tokens(a));
    uint8_t *ws = nullptr;
    if (pl.chunked) {
        if (const int rc = call_workspace(ctx, ctx->linear_scratch, a->workspace, a->workspace_bytes, pl.bytes,
                                          "linear_attention", &ws)) {
            return rc;
        }
    }
    if (injected_fail(ctx, KVMEM_HIP_FAIL_LAUNCH, "linear_attention launch")) {
        return KVMEM_HIP_ERR_RUNTIME;
    }
    if (pl.chunked) {
        launch_linear_chunks(ctx->stream, a->type, a->head_dim_k, pl, p, ws);
    } else if (a->type == KVMEM_TYPE_F32) {
        launch_step<float>(ctx->stream, a->head_dim_k, p);
    } else if (a->type == KVMEM_TYPE_F16) {
        launch_step<_Float16>(ctx->stream, a->head_dim_k, p);
    } else {
        launch_step<__bf16>(ctx->stream, a->head_dim_k, p);
    }
    return hip_ok(ctx, hipGetLastError(), "linear_attention launch") ? KVMEM_HIP_OK : KVMEM_HIP_ERR_RUNTIME;
}

}  // extern "C"
