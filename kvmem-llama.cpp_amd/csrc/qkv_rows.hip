// The rows of new tokens, from the projections to attention's inputs, in one
// pass (kvmem_hip_qkv_rows): per head of q and k
//     y = (x * 1/sqrt(mean(x^2) + eps)) * w
//     RoPE at the token's position, Walsh-Hadamard of runs of hadamard_k
// (v: Walsh-Hadamard of runs of hadamard_v), q to its output rows, k and v
// quantized into the token's cell of the pool.
//
// Each input element is read once and each output written once: bytes bound
// it for many tokens, the launch and one trip to memory for few.  A wave takes
// a unit of 512 consecutive elements (512 / head_dim heads of one token's q, k
// or v), 8 per lane, as the stage-in's transform holds its rows: the norm's sum
// of squares and the butterflies are exchanges inside the wave, the quantizers
// are shared with the stage-in, and a row that needs no norm gets the bytes the
// stage-in would give it.  The sum of squares is fp32, 8 elements in order per
// lane and then a tree over the head's lanes; rows whose squares leave fp32's range
// are brought into it by a power of two.
//
// cos and sin of a token's rotary pairs are computed once per workgroup into
// LDS (about 70 double-precision operations a pair).  A workgroup takes several
// tokens when there are many, so that a pair's angle serves all the token's
// heads; few tokens are spread over workgroups instead, a unit per wave.  Norm
// weights and cells are read from LDS too: loads complete in order, so one
// inside the loop would wait for the unit that is read ahead.
//
// Measured, 24 + 2 x 4 heads of 256 in bf16: 8191 tokens, with the norm, into F16
// cells 56.7 us for 268 MB (4.7 TB/s, vector instructions 86 % busy; 83 us without
// reading ahead and at four waves a SIMD instead of eight), into q8_0 cells 55 us for
// 253 MB, rotated 65 us; 96 tokens 4.8 us, one token 4.6 us (the launch).
#include "kvmem_internal.hpp"
#include "row_transform.hpp"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

#pragma clang fp contract(off)

namespace kvmem_hip {

constexpr uint32_t kRowThreads = 256;
constexpr uint32_t kRowWaves = kRowThreads / 64;
constexpr uint32_t kUnit = 512;       // elements of a wave's unit
constexpr uint32_t kMaxRot = 512;     // rotary dims, head_dim
constexpr uint32_t kMaxRowTokens = 8; // tokens of a workgroup
// Workgroups for many tokens: two rounds of the eight that a compute unit holds.
// 8191 tokens of 24 + 2 x 4 heads of 256 (bf16, norm, F16 cells), 2048 / 4096 / 8192
// workgroups: 57.7 / 54.8 / 57.3 us, rotated 62.8 / 62.5 / 66.1.
constexpr uint32_t kRowGroups = 4096;

struct Theta {
    float f[kMaxRot / 2];
};

struct RowKind {
    const uint8_t *src;   // rows of the new tokens (null: none)
    uint64_t nb1, nb2;    // bytes between heads, tokens
    const float *weight;  // norm weight (null: no norm)
    uint8_t *norm_out;    // rows after the norm (null: none)
    uint8_t *out;         // rotated rows (null: none)
    uint8_t *pool;        // the layer's cache rows (null: none)
    uint32_t row_bytes;   // bytes of a cache row
    uint32_t n_head;
    uint32_t units;       // units of one token
    uint32_t hadamard;
    float hscale;
    int type;             // of the cache rows
    uint32_t vec;         // rows can be read 16 bytes at a time
};

struct RowParams {
    RowKind kind[3];      // q, k, v
    const int32_t *positions;
    const int32_t *cells;
    uint32_t n_tokens, n_cells, head_dim, n_rot;
    uint32_t tokens;      // of one workgroup
    uint32_t splits;      // workgroups that share one group of tokens
    float eps;
};

template <typename T>
struct Row8 {
    typedef T type __attribute__((ext_vector_type(8)));
};

template <typename T>
__device__ inline typename Row8<T>::type load_row8(const uint8_t *p, uint32_t vec) {
    typename Row8<T>::type v;
    if (vec) {
        v = *reinterpret_cast<const typename Row8<T>::type *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = reinterpret_cast<const T *>(p)[i];
        }
    }
    return v;
}

template <typename T>
__device__ inline void store_row8(uint8_t *p, const float x[8]) {
    typename Row8<T>::type v;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = static_cast<T>(x[i]);  // round to nearest even
    }
    *reinterpret_cast<typename Row8<T>::type *>(p) = v;
}


// Sum over the head's head_dim / 8 lanes; every lane of the wave is active.
__device__ inline float head_sum(float s, uint32_t head_dim) {
    s = s + lane_xor<1>(s);
    s = s + lane_xor<2>(s);
    s = s + lane_xor<4>(s);
    if (head_dim > 64u) {
        s = s + lane_xor<8>(s);
    }
    if (head_dim > 128u) {
        s = s + lane_xor<16>(s);
    }
    if (head_dim > 256u) {
        s = s + lane_xor<32>(s);
    }
    return s;
}

// Quantize the wave's unit into `lds` and write its `groups` groups at dst.
template <int TYPE>
__device__ inline void put_unit(const float x[8], uint8_t *lds, uint8_t *dst, uint32_t groups, uint32_t lane) {
    constexpr uint32_t GB = Fmt<TYPE>::GB;
    quant_quarter_f<TYPE>(x, lane & 3u, lds + (lane >> 2) * GB, true);
    // the wave reads back only what it wrote itself
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const uint32_t nb = groups * GB;
    // cells whose rows are no multiple of 16 bytes go out 2 bytes at a time
    const uint32_t full = (reinterpret_cast<uintptr_t>(dst) & 15u) == 0 ? (nb & ~15u) : 0u;
    for (uint32_t off = lane * 16u; off < full; off += 1024u) {
        *reinterpret_cast<uint4 *>(dst + off) = *reinterpret_cast<const uint4 *>(lds + off);
    }
    for (uint32_t off = full + lane * 2u; off < nb; off += 128u) {
        *reinterpret_cast<uint16_t *>(dst + off) = *reinterpret_cast<const uint16_t *>(lds + off);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();  // the next unit writes the same bytes
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A wave's unit: token of the workgroup, kind, heads [h0, h0 + heads).
struct Unit {
    uint32_t tl, kd, h0, heads;
};

__device__ inline Unit find_unit(const RowParams &p, uint32_t u, uint32_t per_token, uint32_t heads_per_unit) {
    Unit r;
    r.tl = u / per_token;
    uint32_t w = u - r.tl * per_token;
    r.kd = 0;
    if (w >= p.kind[0].units) {
        w -= p.kind[0].units;
        r.kd = 1;
        if (w >= p.kind[1].units) {
            w -= p.kind[1].units;
            r.kd = 2;
        }
    }
    r.h0 = w * heads_per_unit;
    r.heads = min(heads_per_unit, p.kind[r.kd].n_head - r.h0);
    return r;
}

// TI / TO: element types of the inputs and of the output rows.
template <typename TI, typename TO>
__global__ __launch_bounds__(kRowThreads, 8) void qkv_rows_kernel(RowParams p, Theta theta) {
    __shared__ __attribute__((aligned(16))) uint8_t staged[kRowWaves][16 * 64];
    // [2][head_dim] norm weights, then [tokens][n_rot / 2] cos, sin
    extern __shared__ __attribute__((aligned(16))) float weights[];
    __shared__ uint32_t cells[kMaxRowTokens];
    float2 *tab = reinterpret_cast<float2 *>(weights + 2u * p.head_dim);
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t group = blockIdx.x / p.splits;
    const uint32_t split = blockIdx.x - group * p.splits;
    const uint32_t t0 = group * p.tokens;
    const uint32_t nt = min(p.tokens, p.n_tokens - t0);
    const uint32_t half = p.n_rot / 2u;
    const uint32_t e0 = lane * 8u;
    const uint32_t head_in_unit = e0 / p.head_dim;
    const uint32_t d0 = e0 & (p.head_dim - 1u);
    const uint32_t heads_per_unit = kUnit / p.head_dim;
    const uint32_t per_token = p.kind[0].units + p.kind[1].units + p.kind[2].units;
    const uint32_t end = nt * per_token;
    const uint32_t step = p.splits * kRowWaves;
    // lanes behind the last head read it again, and write nothing
    const auto read = [&](const Unit &n) {
        const RowKind &k = p.kind[n.kd];
        const uint32_t h = n.h0 + min(head_in_unit, n.heads - 1u);
        return load_row8<TI>(k.src + h * k.nb1 + (t0 + n.tl) * k.nb2 + d0 * sizeof(TI), k.vec);
    };
    // the row a unit ahead is on its way while one is worked on, the first while
    // the angles are
    uint32_t u = split * kRowWaves + wave;
    Unit next{};
    typename Row8<TI>::type ahead{};
    if (u < end) {
        next = find_unit(p, u, per_token, heads_per_unit);
        ahead = read(next);
    }
    constexpr uint32_t kWeightsPerThread = 2 * kMaxRot / kRowThreads;
    float weight[kWeightsPerThread];
#pragma unroll
    for (uint32_t j = 0; j < kWeightsPerThread; ++j) {
        const uint32_t i = threadIdx.x + j * kRowThreads;
        const float *w = i < p.head_dim ? p.kind[0].weight : p.kind[1].weight;
        weight[j] = w && i < 2u * p.head_dim ? w[i < p.head_dim ? i : i - p.head_dim] : 1.0f;
    }
    const uint32_t cell_ahead = threadIdx.x < nt && p.cells ? static_cast<uint32_t>(p.cells[t0 + threadIdx.x]) : ~0u;
    for (uint32_t i = threadIdx.x; i < nt * half; i += kRowThreads) {
        const uint32_t t = i / half;
        float sn, cs;
        rope_sincos(static_cast<float>(p.positions[t0 + t]) * theta.f[i - t * half], sn, cs);
        tab[i] = make_float2(cs, sn);
    }
#pragma unroll
    for (uint32_t j = 0; j < kWeightsPerThread; ++j) {
        if (threadIdx.x + j * kRowThreads < 2u * p.head_dim) {
            weights[threadIdx.x + j * kRowThreads] = weight[j];
        }
    }
    if (threadIdx.x < kMaxRowTokens) {
        cells[threadIdx.x] = cell_ahead;
    }
    __syncthreads();

    while (u < end) {
        const Unit n = next;
        const uint32_t kd = n.kd, tl = n.tl, h0 = n.h0, heads = n.heads;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = static_cast<float>(ahead[i]);
        }
        u += step;
        if (u < end) {
            next = find_unit(p, u, per_token, heads_per_unit);
            ahead = read(next);
        }
        const RowKind &k = p.kind[kd];
        const uint32_t t = t0 + tl;
        const bool valid = head_in_unit < heads;
        const uint32_t h = h0 + min(head_in_unit, heads - 1u);
        if (k.weight) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                ss = ss + x[i] * x[i];
            }
            ss = head_sum(ss, p.head_dim);
            float eps = p.eps;
            // Squares that pass fp32, or fall below it where eps does not cover them: the
            // row by a power of two first (its largest elements by 2^-80 or 2^100; the
            // norm is the same, eps goes along).  The heads of a unit decide one by one.
            const bool large = !(ss < INFINITY);
            const bool small = ss < 0x1p-80f && eps < 0x1p-94f;
            // (f16's squares do not leave it)
            if (!std::is_same<TI, _Float16>::value && __any(large || small)) {
                const float up = large ? 0x1p-80f : small ? 0x1p100f : 1.0f;
                float s2 = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = x[i] * up;
                    s2 = s2 + x[i] * x[i];
                }
                ss = head_sum(s2, p.head_dim);
                eps = eps * up * up;
            }
            const float r = 1.0f / sqrtf(ss / static_cast<float>(p.head_dim) + eps);
            const float *wd = weights + kd * p.head_dim + d0;
            const float4 w0 = *reinterpret_cast<const float4 *>(wd);
            const float4 w1 = *reinterpret_cast<const float4 *>(wd + 4);
            const float wt[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = (x[i] * r) * wt[i];
            }
        }
        const uint64_t o = (static_cast<uint64_t>(t) * k.n_head + h) * p.head_dim + d0;
        if (k.norm_out && valid) {
            store_row8<TO>(k.norm_out + o * sizeof(TO), x);
        }
        if (half != 0u && kd != 2u) {
            const bool rot = d0 < p.n_rot;
            const bool first = d0 < half;
            float q[8];
            rope_partners(x, q, p.n_rot, lane, rot, first);
            if (rot) {
                const float4 *cs = reinterpret_cast<const float4 *>(tab + tl * half + (first ? d0 : d0 - half));
                const uint32_t flip = first ? 0x80000000u : 0u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 c = cs[i];
                    const float q0 = q[2 * i] * c.y;
                    const float q1 = q[2 * i + 1] * c.w;
                    x[2 * i] = x[2 * i] * c.x + __uint_as_float(__float_as_uint(q0) ^ flip);
                    x[2 * i + 1] = x[2 * i + 1] * c.z + __uint_as_float(__float_as_uint(q1) ^ flip);
                }
            }
        }
        if (k.hadamard != 0u) {
            fwht_lanes(x, k.hadamard, k.hscale, lane);
        }
        if (k.out && valid) {
            store_row8<TO>(k.out + o * sizeof(TO), x);
        }
        if (k.pool) {
            const uint32_t cell = __builtin_amdgcn_readfirstlane(cells[tl]);
            if (cell < p.n_cells) {  // -1: the token is not kept
                const uint32_t groups = heads * (p.head_dim / 32u);
                const uint32_t g0 = h0 * (p.head_dim / 32u);
                uint8_t *row = k.pool + static_cast<uint64_t>(cell) * k.row_bytes;
                uint8_t *lds = staged[wave];
                switch (k.type) {
                    case KVMEM_TYPE_Q8_0: put_unit<KVMEM_TYPE_Q8_0>(x, lds, row + g0 * 34u, groups, lane); break;
                    case KVMEM_TYPE_Q5_0: put_unit<KVMEM_TYPE_Q5_0>(x, lds, row + g0 * 22u, groups, lane); break;
                    case KVMEM_TYPE_Q4_0: put_unit<KVMEM_TYPE_Q4_0>(x, lds, row + g0 * 18u, groups, lane); break;
                    default: put_unit<KVMEM_TYPE_F16>(x, lds, row + g0 * 64u, groups, lane); break;
                }
            }
        }
    }
}

template <typename TI, typename TO>
static void launch_rows(hipStream_t stream, uint32_t grid, size_t lds, const RowParams &p, const Theta &theta) {
    qkv_rows_kernel<TI, TO><<<grid, kRowThreads, lds, stream>>>(p, theta);
}

template <typename TI>
static void launch_rows_out(hipStream_t stream, int out_type, uint32_t grid, size_t lds, const RowParams &p,
                            const Theta &theta) {
    if (out_type == KVMEM_TYPE_F32) {
        launch_rows<TI, float>(stream, grid, lds, p, theta);
    } else if (out_type == KVMEM_TYPE_F16) {
        launch_rows<TI, _Float16>(stream, grid, lds, p, theta);
    } else {
        launch_rows<TI, __bf16>(stream, grid, lds, p, theta);
    }
}

bool load_qkv_rows_kernels() {
    return load_kernel_object(&qkv_rows_kernel<float, float>);
}

static bool float_type(int t) { return t == KVMEM_TYPE_F32 || t == KVMEM_TYPE_F16 || t == KVMEM_TYPE_BF16; }

static bool width_ok(uint32_t w, uint32_t head_dim) {
    return w == 0 || (w >= 64 && w <= 512 && (w & (w - 1)) == 0 && head_dim % w == 0);
}

}  // namespace kvmem_hip

using namespace kvmem_hip;

extern "C" {

int kvmem_hip_qkv_rows(kvmem_hip_ctx *ctx, const kvmem_hip_pool *pool, uint32_t layer,
                       const kvmem_hip_qkv_args *a) {
    if (!ctx) {
        return KVMEM_HIP_ERR_INVALID;
    }
    if (!a) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: null arguments");
    }
    if (!float_type(a->type) || !float_type(a->out_type)) {
        return fail(ctx, KVMEM_HIP_ERR_UNSUPPORTED, "qkv_rows: rows must be F32, F16 or BF16");
    }
    const uint32_t D = a->head_dim;
    if (D != 64 && D != 128 && D != 256 && D != 512) {
        return fail(ctx, KVMEM_HIP_ERR_UNSUPPORTED, "qkv_rows: head_dim must be 64, 128, 256 or 512");
    }
    if ((a->q && a->n_head == 0) || ((a->k || a->v) && a->n_head_kv == 0) || a->n_head > 4096 ||
        a->n_head_kv > 4096) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: 1 to 4096 heads");
    }
    if (a->n_tokens > (1u << 26)) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: too many tokens");
    }
    if (!a->q && !a->k && !a->v) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: no rows");
    }
    if ((a->q && !a->q_out && !a->q_norm) || (a->k && !a->k_out && !a->k_norm && !pool) || (a->v && !pool)) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: rows without a destination");
    }
    const kvmem_hip_transform *xf = a->xf ? a->xf : pool ? pool->xf : nullptr;
    const uint32_t n_rot = xf ? xf->n_rot : 0;
    if (xf) {
        if (xf->head_dim != D) {
            return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: the transform has another head_dim");
        }
        if (n_rot && (n_rot % 16 != 0 || n_rot > D || !xf->theta || !a->positions)) {
            return fail(ctx, KVMEM_HIP_ERR_INVALID,
                        "qkv_rows: n_rot must be a multiple of 16 up to head_dim, with theta and positions");
        }
        if (!width_ok(xf->hadamard_k, D) || !width_ok(xf->hadamard_v, D)) {
            return fail(ctx, KVMEM_HIP_ERR_INVALID,
                        "qkv_rows: Hadamard width must be 64..512, a power of two dividing head_dim");
        }
    }
    const size_t esz = a->type == KVMEM_TYPE_F32 ? 4 : 2;
    RowParams p{};
    const void *src[3] = {a->q, a->k, a->v};
    const size_t nb1[3] = {a->q_nb1, a->k_nb1, a->v_nb1};
    const size_t nb2[3] = {a->q_nb2, a->k_nb2, a->v_nb2};
    const float *weight[3] = {a->q_weight, a->k_weight, nullptr};
    void *norm_out[3] = {a->q_norm, a->k_norm, nullptr};
    void *out[3] = {a->q_out, a->k_out, nullptr};
    for (int i = 0; i < 3; ++i) {
        RowKind &k = p.kind[i];
        if (!src[i]) {
            continue;
        }
        const uintptr_t at = reinterpret_cast<uintptr_t>(src[i]);
        if (at % esz || nb1[i] % esz || nb2[i] % esz) {
            return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: strides must be multiples of the element size");
        }
        if ((reinterpret_cast<uintptr_t>(weight[i]) | reinterpret_cast<uintptr_t>(norm_out[i]) |
             reinterpret_cast<uintptr_t>(out[i])) & 15u) {
            return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: weights and outputs must be 16-byte aligned");
        }
        k.src = static_cast<const uint8_t *>(src[i]);
        k.nb1 = nb1[i];
        k.nb2 = nb2[i];
        k.weight = weight[i];
        k.norm_out = static_cast<uint8_t *>(norm_out[i]);
        k.out = static_cast<uint8_t *>(out[i]);
        k.n_head = i == 0 ? a->n_head : a->n_head_kv;
        k.units = (k.n_head * D + kUnit - 1) / kUnit;
        k.hadamard = xf ? (i == 2 ? xf->hadamard_v : xf->hadamard_k) : 0;
        k.hscale = k.hadamard ? 1.0f / sqrtf(static_cast<float>(k.hadamard)) : 1.0f;
        k.vec = (at | nb1[i] | nb2[i]) % 16 == 0;
    }
    if (pool && (a->k || a->v)) {
        const uint64_t E = static_cast<uint64_t>(a->n_head_kv) * D;
        if (!pool->k_layers || layer >= pool->n_layers || pool->block_tokens == 0) {
            return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: no such pool layer");
        }
        if (!a->cells) {
            return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: a pool needs the tokens' cells");
        }
        if (static_cast<uint64_t>(pool->n_slots) * pool->block_tokens > 0x7fffffffu) {
            return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: cells must fit 31 bits");
        }
        const int types[3] = {0, pool->type_k, pool->type_v};
        const uint32_t embd[3] = {0, pool->n_embd_k, pool->n_embd_v};
        void *const *layers[3] = {nullptr, pool->k_layers, pool->v_layers};
        for (int i = 1; i < 3; ++i) {
            RowKind &k = p.kind[i];
            if (!k.src) {
                continue;
            }
            if (embd[i] != E) {
                return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: the pool's rows have another width");
            }
            if (!kvmem_hip_quant_ok(types[i])) {
                return fail(ctx, KVMEM_HIP_ERR_UNSUPPORTED, "qkv_rows: unsupported cache type");
            }
            if (!layers[i] || !layers[i][layer] || (reinterpret_cast<uintptr_t>(layers[i][layer]) & 15u)) {
                return fail(ctx, KVMEM_HIP_ERR_INVALID, "qkv_rows: layer pointer null or not 16-byte aligned");
            }
            k.pool = static_cast<uint8_t *>(layers[i][layer]);
            k.type = types[i];
            k.row_bytes = static_cast<uint32_t>(kvmem_hip_row_size(types[i], static_cast<int64_t>(E)));
        }
        p.cells = a->cells;
        p.n_cells = pool->n_slots * pool->block_tokens;
    }
    if (a->n_tokens == 0) {
        return KVMEM_HIP_OK;
    }
    p.positions = a->positions;
    p.n_tokens = a->n_tokens;
    p.head_dim = D;
    p.n_rot = n_rot;
    p.eps = a->eps;
    const uint32_t units = p.kind[0].units + p.kind[1].units + p.kind[2].units;
    // tokens of a workgroup: as many as leave kRowGroups workgroups; below
    // that a token's units are spread over workgroups, one unit a wave
    p.tokens = std::max(1u, std::min(kMaxRowTokens, (a->n_tokens + kRowGroups - 1) / kRowGroups));
    const uint32_t groups = (a->n_tokens + p.tokens - 1) / p.tokens;
    const uint32_t most = (p.tokens * units + kRowWaves - 1) / kRowWaves;
    p.splits = std::max(1u, std::min(most, kRowGroups / groups));
    Theta theta;
    if (n_rot) {
        std::memcpy(theta.f, xf->theta, sizeof(float) * (n_rot / 2));
    }
    const size_t lds = sizeof(float) * 2 * D + sizeof(float2) * p.tokens * (n_rot / 2);
    (void) hipSetDevice(ctx->device);
    if (injected_fail(ctx, KVMEM_HIP_FAIL_LAUNCH, "qkv_rows launch")) {
        return KVMEM_HIP_ERR_RUNTIME;
    }
    const uint32_t grid = groups * p.splits;
    if (a->type == KVMEM_TYPE_F32) {
        launch_rows_out<float>(ctx->stream, a->out_type, grid, lds, p, theta);
    } else if (a->type == KVMEM_TYPE_F16) {
        launch_rows_out<_Float16>(ctx->stream, a->out_type, grid, lds, p, theta);
    } else {
        launch_rows_out<__bf16>(ctx->stream, a->out_type, grid, lds, p, theta);
    }
    return hip_ok(ctx, hipGetLastError(), "qkv_rows launch") ? KVMEM_HIP_OK : KVMEM_HIP_ERR_RUNTIME;
}

}  // extern "C"
