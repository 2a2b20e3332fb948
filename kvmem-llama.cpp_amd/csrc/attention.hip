// Attention of new tokens over the pool's rows (kvmem_hip_attention).
#include "attention.hpp"

#include <algorithm>
#include <cmath>

namespace kvmem_hip {

// ------------------------------------------------------------- joining parts

// Parts up to which one wave joins a row (many rows of few parts: 512 tokens of 24
// heads in 5 parts, 474 us with the attention against 542 with four waves), four
// above (few rows of many: 24 rows of 64 parts 14.8 us against 15.6 with sixteen).
constexpr uint32_t kJoinParts = 8;

// The parts of a (token, head) row, 0 where this row is not joined.
__device__ inline uint32_t row_parts(const AttnParams &p, uint32_t tok, uint32_t h) {
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
        return 0;
    }
    const Span r = request_span(p, s);
    if (tok < r.first || tok - r.first >= min(r.m, p.max_q)) {
        return 0;
    }
    const uint32_t i = tok - r.first;
    // the part count of the row tile this row was in
    const uint32_t row = i * p.group + h % p.group;
    const uint32_t row0 = row / p.row_tile * p.row_tile;
    const uint32_t rows = min(p.row_tile, min(r.m, p.max_q) * p.group - row0);
    const uint32_t n = key_limit(p, r, (row0 + rows - 1u) / p.group);
    const uint32_t n_parts = max(1u, (n + p.chunk - 1u) / p.chunk);
    return n_parts == 1 && !p.join_one ? 0u : n_parts;
}

// W waves a row, one row a workgroup (W > 1: the parts are dealt to the waves and
// their sums added in the waves' order) or four (W = 1).  A lane adds D/64 dims of
// its wave's parts in order, each weighted by its maximum.  Latency-bound for few
// rows: a wave has all its parts' loads in flight at once.
template <int D, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void attn_join_kernel(AttnParams p) {
    constexpr int E = D / 64;
    typedef float dims_t __attribute__((ext_vector_type(E)));
    __shared__ float sums[W][D];
    __shared__ float totals[W];
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t row = W == 1 ? blockIdx.x * 4u + wave : blockIdx.x;
    const uint32_t tok = row / p.n_head;
    const uint32_t h = row - tok * p.n_head;
    const uint32_t n_parts = tok < p.n_tokens ? row_parts(p, tok, h) : 0u;
    if (n_parts == 0) {
        return;
    }
    const uint64_t at = row;
    const uint64_t stride = static_cast<uint64_t>(p.n_tokens) * p.n_head;
    float top = -INFINITY;
    for (uint32_t k = lane; k < n_parts; k += 64u) {
        top = fmaxf(top, p.part_ml[k * stride + at].x);
    }
    top = fmaxf(top, lane_xor<1>(top));
    top = fmaxf(top, lane_xor<2>(top));
    top = fmaxf(top, lane_xor<4>(top));
    top = fmaxf(top, lane_xor<8>(top));
    top = fmaxf(top, lane_xor<16>(top));
    top = fmaxf(top, lane_xor<32>(top));
    const float *po = p.part_o + at * D + lane * E;
    float total = 0.0f;
    dims_t x = {};
    const uint32_t k0 = W == 1 ? 0u : wave;
#pragma unroll 8
    for (uint32_t k = k0; k < n_parts; k += W) {
        const float2 ml = p.part_ml[k * stride + at];
        const float f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - top);
        total += ml.y * f;
        x += *reinterpret_cast<const dims_t *>(po + k * stride * D) * f;
    }
    if constexpr (W > 1) {
        *reinterpret_cast<dims_t *>(&sums[wave][lane * E]) = x;
        if (lane == 0) {
            totals[wave] = total;
        }
        __syncthreads();
        if (wave != 0) {
            return;
        }
#pragma unroll
        for (int w = 1; w < W; ++w) {
            total += totals[w];
            x += *reinterpret_cast<const dims_t *>(&sums[w][lane * E]);
        }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    float y[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        y[i] = x[i] * inv;
    }
    if (p.hadamard) {
        rotate_lanes<E>(y, p.hadamard, lane);
    }
    store_elems<E>(p.out, p.out_type, at * D + lane * E, y);
    if (lane == 0 && p.lse) {
        p.lse[at] = total == 0.0f ? -INFINITY : (top - kWeightShift) / kLog2e + logf(total);
    }
}

template <int D>
static void launch_join(hipStream_t stream, const AttnParams &p) {
    const uint32_t rows = p.n_tokens * p.n_head;
    if (p.n_parts <= kJoinParts) {
        attn_join_kernel<D, 1><<<(rows + 3) / 4, 256, 0, stream>>>(p);
    } else {
        attn_join_kernel<D, 4><<<rows, 256, 0, stream>>>(p);
    }
}

constexpr uint32_t kComputeUnits = 256;

// Rows of a request (tokens x heads of a KV head) above which the prefill kernel
// takes the call.  The decode kernel reads the keys again for every 16 rows, the
// prefill kernel takes some 30 us before its second step.  Measured, decode against
// prefill kernel in us, q4_0, 4 KV heads of 256:
//   one request: 126 rows over 2048 / 8192 / 32768 keys 22 / 36 / 76 against 45 / 71 / 118,
//                192 rows over 8192 61 against 75, 384 rows 92 against 82
//   two over 8192, 120 rows: 50 against 71; four over 2048, 120 rows: 35 against 49
//   eight over 8192: 60 rows 76 against 87, 96 rows 131 against 89; 96 over 2048: 49 / 49
static uint32_t decode_rows(uint32_t n_seq) {
    return std::max(64u, std::min(192u, 480u / n_seq));
}

// Workgroups a decode launch is split up to, from the steps (128 keys of 256
// elements, a step of four waves) of all requests.  Every part costs its joining
// and the pipeline's first wait: one workgroup a compute unit while there are few
// steps for each, then two, or three with many requests, which end at different
// places.  Measured, q4_0 with 4 KV heads of 256, 256 / 512 / 768 workgroups in us:
//   one request: 16384 keys 17 / 21, 32768 22 / 24, 65536 32 / 32 / 43,
//                131072 53 / 46 / 61
//   16 of 1024 keys: 17 / 19 / 19; 8 of 2048: 18 / 18 / 18
//   8 of 8192: 32 / 29 / 27; 16 of 4096: 31 / 30 / 27; 16 of 8192: 48 / 44 / 37
//   8 ragged ones up to 8192 with 5 tokens, q5_0, 2 KV heads of 64: 35 / 29 / 24
//   32 ragged ones up to 16384, 8 KV heads of 128: 172 / 142 / 116 (1024: 134)
// Where one wave takes a SIMD, a second workgroup waits for the first:
//   one request, q8_0 keys, q4_0 values, 65500 keys 42 / 48 / 59, q8_0 131072 75 / 85 / 100,
//   64 ragged ones up to 2048: 60 / 69 / 69 (16 up to 8192: 64 / 70 / 58)
static uint64_t decode_groups(uint32_t n_seq, uint64_t steps, int waves) {
    if (waves == 1) {
        return kComputeUnits;
    }
    if (n_seq < 8) {
        return steps <= 4 * kComputeUnits ? kComputeUnits : 2 * kComputeUnits;
    }
    return steps <= 2 * kComputeUnits ? kComputeUnits : 3 * kComputeUnits;
}

static AttnPlan plan_attention(const kvmem_hip_pool *pool, const kvmem_hip_attn_args *a) {
    AttnPlan pl{};
    const uint32_t max_q = a->q_start ? std::min(a->max_q, a->n_tokens) : 1u;
    const uint32_t group = a->n_head / a->n_head_kv;
    const uint64_t rows = static_cast<uint64_t>(max_q) * group;
    pl.prefill = rows > decode_rows(a->n_seq);
    pl.row_tile = pl.prefill ? kPrefillRows : kRowTile;
    pl.row_tiles = static_cast<uint32_t>((rows + pl.row_tile - 1) / pl.row_tile);
    const uint32_t quantum = step_keys(a->head_dim) * (pl.prefill ? 1u : kWaves);
    const uint64_t room = static_cast<uint64_t>(a->table_stride) * pool->block_tokens;
    const uint64_t keys = std::max<uint64_t>(1, std::min<uint64_t>(a->max_kv, room));
    const uint64_t groups = static_cast<uint64_t>(a->n_seq) * a->n_head_kv * pl.row_tiles;
    const uint64_t most = (keys + quantum - 1) / quantum;
    uint64_t parts = 1;
    if (pl.prefill) {
        // rounds of workgroups (one a compute unit) times the keys of each, and
        // for every part the joining of its rows, in keys' time
        const uint64_t join = static_cast<uint64_t>(a->n_tokens) * a->n_head / 256 + 64;
        uint64_t best = ~uint64_t{0};
        for (uint64_t k = 1; k <= std::min<uint64_t>(most, kComputeUnits) && groups * (k - 1) < 4 * kComputeUnits; ++k) {
            const uint64_t rounds = (groups * k + kComputeUnits - 1) / kComputeUnits;
            const uint64_t cost = rounds * ((keys + k - 1) / k) + (k > 1 ? k * join : 0);
            if (cost < best) {
                best = cost;
                parts = k;
            }
        }
    } else {
        const int waves = decode_waves(pool->type_k, pool->type_v, static_cast<int>(a->head_dim));
        parts = std::min(std::max<uint64_t>(1, decode_groups(a->n_seq, groups * most, waves) / groups), most);
    }
    uint64_t chunk = (keys + parts - 1) / parts;
    chunk = (chunk + quantum - 1) / quantum * quantum;
    pl.chunk = static_cast<uint32_t>(chunk);
    pl.n_parts = static_cast<uint32_t>((keys + chunk - 1) / chunk);
    if (pl.prefill) {
        pl.units = static_cast<uint32_t>(static_cast<uint64_t>(a->n_seq) * pl.n_parts * a->n_head_kv);
        pl.grid = (static_cast<uint64_t>(pl.units) * pl.row_tiles + 7) / 8 * 8;
    } else {
        // (request, part) pairs: a multiple of 8, so that the KV heads of one pair,
        // whose slices share cache lines, go to the same XCD
        const uint64_t units = (static_cast<uint64_t>(a->n_seq) * pl.n_parts + 7) / 8 * 8;
        pl.units = static_cast<uint32_t>(units);
        pl.grid = units * pl.row_tiles * a->n_head_kv;
    }
    pl.joined = pl.n_parts > 1 || (pl.prefill && pool->xf && pool->xf->hadamard_v);
    if (pl.joined) {
        const size_t heads = static_cast<size_t>(a->n_tokens) * a->n_head * pl.n_parts;
        pl.o_bytes = heads * a->head_dim * sizeof(float);
        pl.ml_bytes = heads * sizeof(float2);
    }
    return pl;
}

bool load_attention_kernels() {
    return load_kernel_object(&attn_join_kernel<64, 1>) && load_attention<KVMEM_TYPE_Q4_0>() &&
           load_attention<KVMEM_TYPE_Q5_0>() && load_attention<KVMEM_TYPE_Q8_0>() && load_attention<KVMEM_TYPE_F16>();
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
    if (p.T > 1) {
        // ceil(2^(31 + l) / T), l = ceil(log2 T): exact for every j < 2^31
        uint32_t l = 1;
        while ((uint64_t{1} << l) < p.T) {
            ++l;
        }
        p.T_mul = static_cast<uint32_t>(((uint64_t{1} << (31 + l)) + p.T - 1) / p.T);
        p.T_shift = l - 1;
    }
    p.n_slots = pool->n_slots;
    p.table_stride = a->table_stride;
    p.causal = a->causal != 0;
    p.q_bf16 = a->q_type == KVMEM_TYPE_BF16;
    p.out_type = a->out_type;
    p.hadamard = pool->xf ? pool->xf->hadamard_v : 0;
    p.scale = a->scale > 0.0f ? a->scale : 1.0f / sqrtf(static_cast<float>(a->head_dim));
    const AttnPlan pl = plan_attention(pool, a);
    // a dispatch counts its work items in 32 bits
    if (pl.grid * (pl.prefill ? 64u * kPrefillWaves : 64u * kWaves) >= uint64_t{1} << 32) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "attention: too many requests of max_q tokens for one launch");
    }
    p.room = static_cast<uint32_t>(std::max<uint64_t>(
        1, std::min<uint64_t>(p.max_kv, static_cast<uint64_t>(p.table_stride) * p.T)));
    p.chunk = pl.chunk;
    p.n_parts = pl.n_parts;
    p.row_tile = pl.row_tile;
    p.row_tiles = pl.row_tiles;
    p.join_one = pl.prefill && p.hadamard;
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
        case KVMEM_TYPE_Q4_0: launch_attention<KVMEM_TYPE_Q4_0>(ctx->stream, pool->type_v, a->head_dim, pl, p); break;
        case KVMEM_TYPE_Q5_0: launch_attention<KVMEM_TYPE_Q5_0>(ctx->stream, pool->type_v, a->head_dim, pl, p); break;
        case KVMEM_TYPE_Q8_0: launch_attention<KVMEM_TYPE_Q8_0>(ctx->stream, pool->type_v, a->head_dim, pl, p); break;
        default: launch_attention<KVMEM_TYPE_F16>(ctx->stream, pool->type_v, a->head_dim, pl, p); break;
    }
    if (pl.joined) {
        // parts that were not written must not be joined into out
        if (!hip_ok(ctx, hipGetLastError(), "attention launch")) {
            return KVMEM_HIP_ERR_RUNTIME;
        }
        if (a->head_dim == 64) {
            launch_join<64>(ctx->stream, p);
        } else if (a->head_dim == 128) {
            launch_join<128>(ctx->stream, p);
        } else {
            launch_join<256>(ctx->stream, p);
        }
    }
    return hip_ok(ctx, hipGetLastError(), "attention launch") ? KVMEM_HIP_OK : KVMEM_HIP_ERR_RUNTIME;
}

}  // extern "C"
