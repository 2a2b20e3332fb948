// Attention of new tokens over the pool's rows (kvmem_hip_attention).
//
// One workgroup per (token, query head): tiles of 256 keys, a thread per key
// for the scores, the running maximum and sum of the softmax kept over tiles,
// then a thread per value element.
#include "kvmem_internal.hpp"

#include <algorithm>
#include <cmath>

namespace kvmem_hip {

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
    uint32_t row_k, row_v;      // bytes of a cached row
    uint32_t n_tokens, n_seq, max_q, max_kv, n_head, group, T, n_slots, table_stride;
    int32_t causal;
    int32_t q_bf16;
    int32_t out_type;
    uint32_t hadamard;
    float scale;
};

// Element e of a cached row.
__device__ inline float cache_elem(const uint8_t *row, int type, uint32_t e) {
    const uint32_t g = e >> 5;
    const uint32_t i = e & 31u;
    if (type == KVMEM_TYPE_F16) {
        return static_cast<float>(reinterpret_cast<const _Float16 *>(row)[e]);
    }
    const uint32_t gb = type == KVMEM_TYPE_Q8_0 ? 34u : type == KVMEM_TYPE_Q5_0 ? 22u : 18u;
    const uint8_t *p = row + g * gb;
    const float d = static_cast<float>(*reinterpret_cast<const _Float16 *>(p));
    if (type == KVMEM_TYPE_Q8_0) {
        return d * static_cast<float>(static_cast<int8_t>(p[2 + i]));
    }
    const uint32_t b = p[gb - 16u + (i & 15u)];
    int c = static_cast<int>(i < 16u ? b & 15u : b >> 4);
    if (type == KVMEM_TYPE_Q5_0) {
        c |= ((p[2 + (i >> 3)] >> (i & 7u)) & 1) << 4;
        return d * static_cast<float>(c - 16);
    }
    return d * static_cast<float>(c - 8);
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

__global__ __launch_bounds__(256) void attention_kernel(AttnParams p, int type_k, int type_v, uint32_t D) {
    __shared__ float qs[256], ps[256], red[256];
    __shared__ uint32_t cell[256];
    const uint32_t tid = threadIdx.x;
    const uint32_t h = blockIdx.x % p.n_head;
    const uint32_t s = blockIdx.y;
    const uint32_t i = blockIdx.x / p.n_head;
    const uint32_t a = p.q_start ? min(p.q_start[s], p.n_tokens) : s;
    const uint32_t b = p.q_start ? min(p.q_start[s + 1], p.n_tokens) : s + 1;
    const uint32_t m = b > a ? b - a : 0u;
    if (i >= m || i >= p.max_q) {
        return;
    }
    const uint32_t len = p.kv_len[s];
    const uint64_t room = static_cast<uint64_t>(p.table_stride) * p.T;
    uint32_t n = static_cast<uint32_t>(min<uint64_t>(min(len, p.max_kv), room));
    if (p.causal) {
        const int64_t last = static_cast<int64_t>(len) - m + i + 1;
        n = last <= 0 ? 0u : static_cast<uint32_t>(min<int64_t>(n, last));
    }
    const uint32_t hk = h / p.group;
    const uint64_t row = static_cast<uint64_t>(a) + i;
    if (tid < D) {
        const uint8_t *q = p.q + row * p.q_nb2 + h * p.q_nb1 + tid * 2u;
        qs[tid] = p.scale * (p.q_bf16 ? static_cast<float>(*reinterpret_cast<const __bf16 *>(q))
                                      : static_cast<float>(*reinterpret_cast<const _Float16 *>(q)));
    }
    float top = -INFINITY, sum = 0.0f, acc = 0.0f;
    for (uint32_t j0 = 0; j0 < n; j0 += 256u) {
        const uint32_t j = j0 + tid;
        __syncthreads();
        float x = -INFINITY;
        cell[tid] = 0xffffffffu;
        if (j < n) {
            const uint32_t slot = p.table[static_cast<uint64_t>(s) * p.table_stride + j / p.T];
            if (slot < p.n_slots) {
                const uint32_t c = slot * p.T + j % p.T;
                cell[tid] = c;
                const uint8_t *kr = p.k + static_cast<uint64_t>(c) * p.row_k;
                x = 0.0f;
                for (uint32_t e = 0; e < D; ++e) {
                    x += qs[e] * cache_elem(kr, type_k, hk * D + e);
                }
            }
        }
        red[tid] = x;
        __syncthreads();
        float tile_top = top;
        for (uint32_t t = 0; t < 256u; ++t) {
            tile_top = fmaxf(tile_top, red[t]);
        }
        ps[tid] = cell[tid] == 0xffffffffu ? 0.0f : expf(x - tile_top);
        __syncthreads();
        if (tile_top == -INFINITY) {
            continue;
        }
        const float fade = top == -INFINITY ? 0.0f : expf(top - tile_top);
        sum *= fade;
        acc *= fade;
        top = tile_top;
        for (uint32_t t = 0; t < 256u; ++t) {
            sum += ps[t];
            if (tid < D && cell[t] != 0xffffffffu) {
                acc += ps[t] * cache_elem(p.v + static_cast<uint64_t>(cell[t]) * p.row_v, type_v, hk * D + tid);
            }
        }
    }
    float o = sum == 0.0f ? 0.0f : acc / sum;  // a NaN sum stays one
    if (p.hadamard) {
        o *= 1.0f / sqrtf(static_cast<float>(p.hadamard));
        for (uint32_t d = 1; d < p.hadamard; d <<= 1) {
            __syncthreads();
            red[tid] = o;
            __syncthreads();
            const float other = red[tid ^ d];
            o = (tid & d) ? other - o : o + other;
        }
    }
    if (tid < D) {
        store_elem(p.out, p.out_type, (row * p.n_head + h) * D + tid, o);
    }
    if (tid == 0 && p.lse) {
        p.lse[row * p.n_head + h] = sum == 0.0f ? -INFINITY : top + logf(sum);
    }
}

bool load_attention_kernels() {
    return load_kernel_object(&attention_kernel);
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
    if (a->n_seq > 65535u || a->n_tokens > (1u << 24) || a->max_kv > 0x7fffffffu) {
        return "attention: at most 65535 requests, 2^24 tokens and 2^31 keys";
    }
    if (!(a->scale >= 0.0f) || std::isinf(a->scale)) {
        return "attention: scale must be finite and not negative";
    }
    if (pool->block_tokens == 0 || static_cast<uint64_t>(pool->n_slots) * pool->block_tokens > 0x7fffffffu) {
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
    return 0;
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
    p.group = a->n_head / a->n_head_kv;
    p.T = pool->block_tokens;
    p.n_slots = pool->n_slots;
    p.table_stride = a->table_stride;
    p.causal = a->causal != 0;
    p.q_bf16 = a->q_type == KVMEM_TYPE_BF16;
    p.out_type = a->out_type;
    p.hadamard = pool->xf ? pool->xf->hadamard_v : 0;
    p.scale = a->scale > 0.0f ? a->scale : 1.0f / sqrtf(static_cast<float>(a->head_dim));
    (void) hipSetDevice(ctx->device);
    if (injected_fail(ctx, KVMEM_HIP_FAIL_LAUNCH, "attention launch")) {
        return KVMEM_HIP_ERR_RUNTIME;
    }
    attention_kernel<<<dim3(p.max_q * p.n_head, p.n_seq), 256, 0, ctx->stream>>>(p, pool->type_k, pool->type_v,
                                                                                   a->head_dim);
    return hip_ok(ctx, hipGetLastError(), "attention launch") ? KVMEM_HIP_OK : KVMEM_HIP_ERR_RUNTIME;
}

}  // extern "C"
