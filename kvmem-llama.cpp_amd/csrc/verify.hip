// Verification of drafted tokens (kvmem_hip_verify_draft): row by row of a
// request, draft x stays where u q(x) < p(x), p = softmax(logits / temperature);
// the next token is drawn from max(p - q, 0) at the first refusal, else from the
// last row's p.
//
// Every logit is read once: bytes bound it for many rows, three short dependent
// launches for few.
//   parts    a workgroup per part of a row: the part's maximum (with its lowest
//            id) and sum of exponentials relative to it
//   decide   a workgroup per request: joins its rows' parts, tests its drafts in
//            order, and draws the next token wherever p alone decides it, from the
//            part sums first and then inside the one part that holds the border
//   rest     where a refused draft had probabilities, the parts' sums of
//            max(p - q, 0), then the draw from those
// Exponentials and sums are fp64: a draw compares a running sum with u times the
// total, and of 10^5 ids' borders fp32 sums would misplace one in a few hundred
// draws; fp64 ones none in 10^8.
#include "kvmem_internal.hpp"

#include <algorithm>
#include <cmath>

#include "recurrent.hpp"

namespace kvmem_hip {

constexpr uint32_t kVerifyThreads = 256;
constexpr uint32_t kVerifyMaxDraft = 127;
constexpr uint32_t kVerifyMaxVocab = 1u << 24;

struct Part {
    double sum;   // of exp((logit - max) / temperature); 0: nothing above -inf
    float max;    // largest logit
    uint32_t at;  // its lowest id
};

// What a request's draw needs from the decide kernel.
struct Choice {
    double scale;   // 1 / sum of the row's exponentials
    float max;      // the row's largest logit
    uint32_t row;   // of the refused draft
    uint32_t pending;  // the draw is from max(p - q, 0)
    uint32_t pad[3];
};

struct VerifyParams {
    const uint8_t *logits;
    const uint8_t *probs;
    uint64_t logits_nb, probs_nb;
    int type, probs_type;
    uint32_t n_vocab, n_rows, n_seq, max_draft;
    const uint32_t *q_start;
    const int32_t *tokens;
    const float *temperature;
    const float *u_accept;
    const float *u_sample;
    const uint32_t *kv_len;
    int32_t *tokens_out;
    uint32_t *n_accepted;
    uint32_t *n_keep;
    uint32_t *kv_len_out;
    uint32_t part;       // ids of a part
    uint32_t n_parts;    // of a row
    bool vec, probs_vec; // 16-byte aligned rows
    Part *parts;         // [n_seq][max_draft + 1][n_parts]
    double *rest;        // [n_seq][n_parts]
    Choice *choice;      // [n_seq]
};

// Rows of request s: first, and how many are looked at.
__device__ inline uint32_t rows_of(const VerifyParams &p, uint32_t s, uint32_t &count, uint32_t &all) {
    const uint32_t most = p.max_draft + 1;
    const uint64_t first = p.q_start ? p.q_start[s] : static_cast<uint64_t>(s) * most;
    uint64_t end = p.q_start ? p.q_start[s + 1] : first + most;
    all = end > first ? static_cast<uint32_t>(end - first) : 0u;
    end = end < p.n_rows ? end : p.n_rows;
    count = end > first ? static_cast<uint32_t>(end - first) : 0u;
    count = count < most ? count : most;
    return static_cast<uint32_t>(first);
}

__device__ inline float load_float(const uint8_t *p, int type, uint64_t i) {
    if (type == KVMEM_TYPE_F32) {
        return reinterpret_cast<const float *>(p)[i];
    }
    const uint16_t h = reinterpret_cast<const uint16_t *>(p)[i];
    return type == KVMEM_TYPE_F16 ? static_cast<float>(__builtin_bit_cast(_Float16, h))
                                  : __uint_as_float(static_cast<uint32_t>(h) << 16);
}

// A logit: NaN counts as -inf.
__device__ inline float load_logit(const uint8_t *p, int type, uint64_t i) {
    const float x = load_float(p, type, i);
    return x == x ? x : -INFINITY;
}

// exp((x - max) / temperature); inv = 1 / temperature.
__device__ inline double weight_of(float x, float max, double inv) {
    return x > -INFINITY ? exp((static_cast<double>(x) - static_cast<double>(max)) * inv) : 0.0;
}

__device__ inline bool better(float m, uint32_t at, float m2, uint32_t at2) {
    return m > m2 || (m == m2 && at < at2);
}

// Sum over the workgroup, in an order that never changes; every thread has it.
__device__ inline double block_sum(double v, double *lds) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        v += __shfl_xor(v, m, 64);
    }
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) {
        lds[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

__device__ inline void block_best(float &m, uint32_t &at, float *lds_m, uint32_t *lds_at) {
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const float m2 = __shfl_xor(m, x, 64);
        const uint32_t at2 = __shfl_xor(at, x, 64);
        if (better(m2, at2, m, at)) {
            m = m2, at = at2;
        }
    }
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) {
        lds_m[threadIdx.x >> 6] = m;
        lds_at[threadIdx.x >> 6] = at;
    }
    __syncthreads();
    m = lds_m[0], at = lds_at[0];
    for (int i = 1; i < 4; ++i) {
        if (better(lds_m[i], lds_at[i], m, at)) {
            m = lds_m[i], at = lds_at[i];
        }
    }
}

__device__ inline double inv_temperature(const VerifyParams &p, uint32_t s, bool &greedy) {
    const float t = p.temperature ? p.temperature[s] : 1.0f;
    greedy = !(t > 0.0f);
    return greedy ? 1.0 : 1.0 / static_cast<double>(t);
}

__global__ __launch_bounds__(kVerifyThreads) void verify_parts_kernel(const VerifyParams p) {
    __shared__ double lds_d[4];
    __shared__ float lds_m[4];
    __shared__ uint32_t lds_at[4];
    const uint32_t s = blockIdx.z, i = blockIdx.y, part = blockIdx.x;
    uint32_t count, all;
    const uint32_t first = rows_of(p, s, count, all);
    if (i >= count) {
        return;
    }
    const uint8_t *row = p.logits + (static_cast<uint64_t>(first) + i) * p.logits_nb;
    const uint32_t v0 = part * p.part, v1 = p.n_vocab - v0 < p.part ? p.n_vocab : v0 + p.part;
    bool greedy;
    const double inv = inv_temperature(p, s, greedy);
    float m = -INFINITY;
    uint32_t at = 0xffffffffu;
    for (uint32_t v = v0 + threadIdx.x; v < v1; v += kVerifyThreads) {
        const float x = load_logit(row, p.type, v);
        if (x > m) {
            m = x, at = v;
        }
    }
    block_best(m, at, lds_m, lds_at);
    double sum = 0.0;
    if (!greedy && m > -INFINITY && m < INFINITY) {
        for (uint32_t v = v0 + threadIdx.x; v < v1; v += kVerifyThreads) {
            sum += weight_of(load_logit(row, p.type, v), m, inv);
        }
        sum = block_sum(sum, lds_d);
    }
    if (threadIdx.x == 0) {
        p.parts[(static_cast<uint64_t>(s) * (p.max_draft + 1) + i) * p.n_parts + part] = Part{sum, m, at};
    }
}

// The first of n weights whose running sum passes `target`, by the whole workgroup;
// `before` is the running sum in front of it.  Where none passes, the last positive
// one (n if there is none).  w(i) is read in order, each weight twice at most.
struct PickLds {
    double sum[kVerifyThreads];
    uint32_t last[kVerifyThreads];
    double before;
    uint32_t found, fallback;
};

template <typename W>
__device__ inline uint32_t block_pick(uint32_t n, double start, double target, W w, PickLds &lds, double &before) {
    const uint32_t per = (n + kVerifyThreads - 1) / kVerifyThreads;
    const uint32_t a = min(n, threadIdx.x * per), b = min(n, a + per);
    double sum = 0.0;
    uint32_t last = n;
    for (uint32_t i = a; i < b; ++i) {
        const double x = w(i);
        sum += x;
        last = x > 0.0 ? i : last;
    }
    __syncthreads();
    lds.sum[threadIdx.x] = sum;
    lds.last[threadIdx.x] = last;
    if (threadIdx.x == 0) {
        lds.found = n;
        lds.fallback = n;
        lds.before = start;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double run = start;
        uint32_t owner = kVerifyThreads;
        for (uint32_t t = 0; t < kVerifyThreads; ++t) {
            if (lds.last[t] < n) {
                lds.fallback = t;
                lds.before = run;
                if (run + lds.sum[t] > target) {
                    owner = t;
                    break;
                }
            }
            run += lds.sum[t];
        }
        lds.found = owner;
    }
    __syncthreads();
    const uint32_t owner = lds.found < kVerifyThreads ? lds.found : lds.fallback;
    before = lds.before;
    __syncthreads();
    if (owner >= kVerifyThreads) {
        return n;  // nothing positive
    }
    if (threadIdx.x == owner) {
        double run = before;
        uint32_t at = last;
        for (uint32_t i = a; i < b; ++i) {
            const double x = w(i);
            if (x > 0.0) {
                lds.before = run;
                if (run + x > target) {
                    at = i;
                    break;
                }
            }
            run += x;
        }
        lds.found = at;
    }
    __syncthreads();
    const uint32_t found = lds.found;
    before = lds.before;
    __syncthreads();
    return found;
}

struct Row {
    double sum;
    float max;
    uint32_t at;
};

// A row's parts together, by one wave.
__device__ inline Row join_row(const VerifyParams &p, const Part *parts, double inv) {
    const uint32_t lane = threadIdx.x & 63u;
    float m = -INFINITY;
    uint32_t at = 0xffffffffu;
    for (uint32_t i = lane; i < p.n_parts; i += 64) {
        const Part x = parts[i];
        if (better(x.max, x.at, m, at)) {
            m = x.max, at = x.at;
        }
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const float m2 = __shfl_xor(m, x, 64);
        const uint32_t at2 = __shfl_xor(at, x, 64);
        if (better(m2, at2, m, at)) {
            m = m2, at = at2;
        }
    }
    double sum = 0.0;
    for (uint32_t i = lane; i < p.n_parts; i += 64) {
        const Part x = parts[i];
        sum += x.sum > 0.0 ? x.sum * weight_of(x.max, m, inv) : 0.0;
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        sum += __shfl_xor(sum, x, 64);
    }
    return Row{sum, m, at};
}

__device__ inline void write_request(const VerifyParams &p, uint32_t s, uint32_t first, uint32_t count, uint32_t all,
                                     uint32_t accepted) {
    int32_t *out = p.tokens_out + static_cast<uint64_t>(s) * (p.max_draft + 1);
    for (uint32_t i = threadIdx.x; i <= p.max_draft; i += kVerifyThreads) {
        out[i] = i < accepted ? p.tokens[first + i + 1] : -1;
    }
    if (threadIdx.x == 0) {
        const uint32_t keep = count ? accepted + 1 : 0u;
        p.n_accepted[s] = accepted;
        if (p.n_keep) {
            p.n_keep[s] = keep;
        }
        if (p.kv_len_out) {
            p.kv_len_out[s] = p.kv_len[s] - all + keep;
        }
    }
}

__device__ inline void write_token(const VerifyParams &p, uint32_t s, uint32_t accepted, uint32_t id) {
    if (threadIdx.x == 0) {
        p.tokens_out[static_cast<uint64_t>(s) * (p.max_draft + 1) + accepted] = static_cast<int32_t>(id);
    }
}

__global__ __launch_bounds__(kVerifyThreads) void verify_decide_kernel(const VerifyParams p) {
    __shared__ Row rows[kVerifyMaxDraft + 1];
    __shared__ uint8_t stays[kVerifyMaxDraft + 1];
    __shared__ PickLds lds;
    __shared__ double lds_d[4];
    const uint32_t s = blockIdx.x;
    uint32_t count, all;
    const uint32_t first = rows_of(p, s, count, all);
    bool greedy;
    const double inv = inv_temperature(p, s, greedy);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (uint32_t i = wave; i < count; i += kVerifyThreads / 64) {
        const uint64_t r = static_cast<uint64_t>(first) + i;
        const Row row =
            join_row(p, p.parts + (static_cast<uint64_t>(s) * (p.max_draft + 1) + i) * p.n_parts, inv);
        if ((threadIdx.x & 63u) == 0) {
            rows[i] = row;
            bool ok = false;
            if (i + 1 < count) {
                const uint32_t x = static_cast<uint32_t>(p.tokens[r + 1]);
                if (x < p.n_vocab && row.max > -INFINITY) {
                    if (greedy || row.max == INFINITY) {
                        ok = x == row.at;
                    } else {
                        const double e =
                            weight_of(load_logit(p.logits + r * p.logits_nb, p.type, x), row.max, inv) / row.sum;
                        const double q =
                            p.probs ? static_cast<double>(load_float(p.probs + r * p.probs_nb, p.probs_type, x)) : 1.0;
                        ok = static_cast<double>(p.u_accept[r]) * q < e;
                    }
                }
            }
            stays[i] = ok;
        }
    }
    __syncthreads();
    uint32_t accepted = 0;
    while (accepted + 1 < count && stays[accepted]) {
        ++accepted;
    }
    write_request(p, s, first, count, all, accepted);
    __syncthreads();  // tokens_out[accepted] is written again below
    if (threadIdx.x == 0) {
        p.choice[s].pending = 0;
    }
    if (count == 0) {
        return;
    }
    const Row row = rows[accepted];
    if (row.max == -INFINITY) {
        return;  // nothing to draw from: -1
    }
    if (greedy || row.max == INFINITY) {
        write_token(p, s, accepted, row.at);
        return;
    }
    const uint64_t r = static_cast<uint64_t>(first) + accepted;
    const bool refused = accepted + 1 < count;
    if (refused && p.probs) {
        if (threadIdx.x == 0) {
            p.choice[s] = Choice{1.0 / row.sum, row.max, accepted, 1u, {}};
        }
        return;
    }
    // the draw from p, without the refused draft
    const Part *parts = p.parts + (static_cast<uint64_t>(s) * (p.max_draft + 1) + accepted) * p.n_parts;
    const uint8_t *logits = p.logits + r * p.logits_nb;
    uint32_t without = refused ? static_cast<uint32_t>(p.tokens[r + 1]) : 0xffffffffu;
    without = without < p.n_vocab ? without : 0xffffffffu;
    uint32_t cut = 0xffffffffu;  // its part, and that part's sum without it
    double cut_sum = 0.0;
    double total = row.sum;
    if (without != 0xffffffffu) {
        cut = without / p.part;
        const uint32_t v0 = cut * p.part, v1 = min(p.n_vocab, v0 + p.part);
        for (uint32_t v = v0 + threadIdx.x; v < v1; v += kVerifyThreads) {
            cut_sum += v == without ? 0.0 : weight_of(load_logit(logits, p.type, v), row.max, inv);
        }
        cut_sum = block_sum(cut_sum, lds_d);
        total = 0.0;
        for (uint32_t i = threadIdx.x; i < p.n_parts; i += kVerifyThreads) {
            const Part x = parts[i];
            total += i == cut ? cut_sum : x.sum > 0.0 ? x.sum * weight_of(x.max, row.max, inv) : 0.0;
        }
        total = block_sum(total, lds_d);
        if (!(total > 0.0)) {  // the draft was all there is
            without = cut = 0xffffffffu;
            total = row.sum;
        }
    }
    const double target = static_cast<double>(p.u_sample[s]) * total;
    double before;
    const uint32_t part = block_pick(
        p.n_parts, 0.0, target,
        [&](uint32_t i) {
            const Part x = parts[i];
            return i == cut ? cut_sum : x.sum > 0.0 ? x.sum * weight_of(x.max, row.max, inv) : 0.0;
        },
        lds, before);
    if (part >= p.n_parts) {
        return;
    }
    const uint32_t v0 = part * p.part;
    const uint32_t at = block_pick(
        min(p.part, p.n_vocab - v0), before, target,
        [&](uint32_t i) {
            return v0 + i == without ? 0.0 : weight_of(load_logit(logits, p.type, v0 + i), row.max, inv);
        },
        lds, before);
    write_token(p, s, accepted, v0 + at);
}

__device__ inline double rest_of(const VerifyParams &p, const Choice &c, const uint8_t *logits, const uint8_t *probs,
                                 double inv, uint32_t v) {
    const double e = weight_of(load_logit(logits, p.type, v), c.max, inv) * c.scale -
                     static_cast<double>(load_float(probs, p.probs_type, v));
    return e > 0.0 ? e : 0.0;
}

__global__ __launch_bounds__(kVerifyThreads) void verify_rest_kernel(const VerifyParams p) {
    __shared__ double lds_d[4];
    const uint32_t s = blockIdx.y, part = blockIdx.x;
    const Choice c = p.choice[s];
    if (!c.pending) {
        return;
    }
    uint32_t count, all;
    const uint64_t r = static_cast<uint64_t>(rows_of(p, s, count, all)) + c.row;
    bool greedy;
    const double inv = inv_temperature(p, s, greedy);
    const uint8_t *logits = p.logits + r * p.logits_nb, *probs = p.probs + r * p.probs_nb;
    const uint32_t v0 = part * p.part, v1 = min(p.n_vocab, v0 + p.part);
    double sum = 0.0;
    for (uint32_t v = v0 + threadIdx.x; v < v1; v += kVerifyThreads) {
        sum += rest_of(p, c, logits, probs, inv, v);
    }
    sum = block_sum(sum, lds_d);
    if (threadIdx.x == 0) {
        p.rest[static_cast<uint64_t>(s) * p.n_parts + part] = sum;
    }
}

__global__ __launch_bounds__(kVerifyThreads) void verify_draw_kernel(const VerifyParams p) {
    __shared__ PickLds lds;
    __shared__ double lds_d[4];
    const uint32_t s = blockIdx.x;
    const Choice c = p.choice[s];
    if (!c.pending) {
        return;
    }
    uint32_t count, all;
    const uint64_t r = static_cast<uint64_t>(rows_of(p, s, count, all)) + c.row;
    bool greedy;
    const double inv = inv_temperature(p, s, greedy);
    const uint8_t *logits = p.logits + r * p.logits_nb, *probs = p.probs + r * p.probs_nb;
    const double *rest = p.rest + static_cast<uint64_t>(s) * p.n_parts;
    const Part *parts = p.parts + (static_cast<uint64_t>(s) * (p.max_draft + 1) + c.row) * p.n_parts;
    double total = 0.0;
    for (uint32_t i = threadIdx.x; i < p.n_parts; i += kVerifyThreads) {
        total += rest[i];
    }
    total = block_sum(total, lds_d);
    const bool left = total > 0.0;  // else p itself
    if (!left) {
        total = 1.0 / c.scale;
    }
    const double target = static_cast<double>(p.u_sample[s]) * total;
    double before;
    const uint32_t part = block_pick(
        p.n_parts, 0.0, target,
        [&](uint32_t i) {
            const Part x = parts[i];
            return left ? rest[i] : x.sum > 0.0 ? x.sum * weight_of(x.max, c.max, inv) : 0.0;
        },
        lds, before);
    if (part >= p.n_parts) {
        return;
    }
    const uint32_t v0 = part * p.part;
    const uint32_t at = block_pick(
        min(p.part, p.n_vocab - v0), before, target,
        [&](uint32_t i) {
            return left ? rest_of(p, c, logits, probs, inv, v0 + i)
                        : weight_of(load_logit(logits, p.type, v0 + i), c.max, inv);
        },
        lds, before);
    write_token(p, s, c.row, v0 + at);
}

bool load_verify_kernels() {
    return load_kernel_object(&verify_parts_kernel);
}

struct VerifyPlan {
    uint32_t part, n_parts;
    size_t parts_bytes, rest_bytes, choice_bytes;
};

static VerifyPlan plan_verify(const kvmem_hip_verify_args *a) {
    VerifyPlan pl;
    pl.part = 2048;
    pl.n_parts = (a->n_vocab + pl.part - 1) / pl.part;
    const size_t rows = static_cast<size_t>(a->n_seq) * (a->max_draft + 1);
    pl.parts_bytes = rows * pl.n_parts * sizeof(Part);
    pl.rest_bytes = (static_cast<size_t>(a->n_seq) * pl.n_parts * sizeof(double) + 15) / 16 * 16;
    pl.choice_bytes = a->n_seq * sizeof(Choice);
    return pl;
}

static const char *check_verify(const kvmem_hip_verify_args *a, int &code) {
    code = KVMEM_HIP_ERR_INVALID;
    if (!a) {
        return "verify_draft: null arguments";
    }
    if (!float_type_ok(a->type) || (a->probs && !float_type_ok(a->probs_type))) {
        code = KVMEM_HIP_ERR_UNSUPPORTED;
        return "verify_draft: logits and probs must be F32, F16 or BF16";
    }
    if (a->n_seq > 65535 || a->max_draft > kVerifyMaxDraft || a->n_vocab > kVerifyMaxVocab) {
        code = KVMEM_HIP_ERR_UNSUPPORTED;
        return "verify_draft: at most 65535 requests, 127 drafts, 2^24 ids";
    }
    if (a->n_vocab == 0) {
        return "verify_draft: no ids";
    }
    if (a->n_seq == 0) {
        code = KVMEM_HIP_OK;
        return nullptr;
    }
    if (!a->logits || !a->tokens || !a->u_accept || !a->u_sample || !a->tokens_out || !a->n_accepted) {
        return "verify_draft: null array";
    }
    if ((a->kv_len == nullptr) != (a->kv_len_out == nullptr)) {
        return "verify_draft: kv_len and kv_len_out go together";
    }
    const uintptr_t words = reinterpret_cast<uintptr_t>(a->q_start) | reinterpret_cast<uintptr_t>(a->tokens) |
                            reinterpret_cast<uintptr_t>(a->temperature) | reinterpret_cast<uintptr_t>(a->u_accept) |
                            reinterpret_cast<uintptr_t>(a->u_sample) | reinterpret_cast<uintptr_t>(a->kv_len) |
                            reinterpret_cast<uintptr_t>(a->tokens_out) | reinterpret_cast<uintptr_t>(a->n_accepted) |
                            reinterpret_cast<uintptr_t>(a->n_keep) | reinterpret_cast<uintptr_t>(a->kv_len_out);
    const uintptr_t at = reinterpret_cast<uintptr_t>(a->logits) | a->logits_nb;
    const uintptr_t probs_at = a->probs ? reinterpret_cast<uintptr_t>(a->probs) | a->probs_nb : 0;
    if (words % 4 || at % float_type_size(a->type) || (a->probs && probs_at % float_type_size(a->probs_type))) {
        return "verify_draft: arrays and rows must be aligned to their elements";
    }
    if (a->tokens_out == a->tokens) {
        return "verify_draft: outputs must not overlap inputs";
    }
    code = KVMEM_HIP_OK;
    return nullptr;
}

}  // namespace kvmem_hip

using namespace kvmem_hip;

extern "C" {

size_t kvmem_hip_verify_draft_workspace(const kvmem_hip_verify_args *a) {
    int code = 0;
    if (check_verify(a, code) || a->n_seq == 0) {
        return 0;
    }
    const VerifyPlan pl = plan_verify(a);
    return pl.parts_bytes + pl.rest_bytes + pl.choice_bytes;
}

int kvmem_hip_verify_draft(kvmem_hip_ctx *ctx, const kvmem_hip_verify_args *a) {
    if (!ctx) {
        return KVMEM_HIP_ERR_INVALID;
    }
    int code = 0;
    if (const char *why = check_verify(a, code)) {
        return fail(ctx, code, why);
    }
    if (a->n_seq == 0) {
        return KVMEM_HIP_OK;
    }
    const VerifyPlan pl = plan_verify(a);
    // a dispatch counts its work items in 32 bits
    if (static_cast<uint64_t>(pl.n_parts) * (a->max_draft + 1) * a->n_seq * kVerifyThreads >= uint64_t{1} << 32) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "verify_draft: too many rows for one launch");
    }
    VerifyParams p{};
    p.logits = static_cast<const uint8_t *>(a->logits);
    p.probs = static_cast<const uint8_t *>(a->probs);
    p.logits_nb = a->logits_nb;
    p.probs_nb = a->probs_nb;
    p.type = a->type;
    p.probs_type = a->probs_type;
    p.n_vocab = a->n_vocab;
    p.n_rows = a->n_rows;
    p.n_seq = a->n_seq;
    p.max_draft = a->max_draft;
    p.q_start = a->q_start;
    p.tokens = a->tokens;
    p.temperature = a->temperature;
    p.u_accept = a->u_accept;
    p.u_sample = a->u_sample;
    p.kv_len = a->kv_len;
    p.tokens_out = a->tokens_out;
    p.n_accepted = a->n_accepted;
    p.n_keep = a->n_keep;
    p.kv_len_out = a->kv_len_out;
    p.part = pl.part;
    p.n_parts = pl.n_parts;
    p.vec = ((reinterpret_cast<uintptr_t>(a->logits) | a->logits_nb) & 15u) == 0;
    p.probs_vec = ((reinterpret_cast<uintptr_t>(a->probs) | a->probs_nb) & 15u) == 0;
    (void) hipSetDevice(ctx->device);
    uint8_t *ws = nullptr;
    if (const int rc = call_workspace(ctx, ctx->verify_scratch, a->workspace, a->workspace_bytes,
                                      pl.parts_bytes + pl.rest_bytes + pl.choice_bytes, "verify_draft", &ws)) {
        return rc;
    }
    p.parts = reinterpret_cast<Part *>(ws);
    p.rest = reinterpret_cast<double *>(ws + pl.parts_bytes);
    p.choice = reinterpret_cast<Choice *>(ws + pl.parts_bytes + pl.rest_bytes);
    if (injected_fail(ctx, KVMEM_HIP_FAIL_LAUNCH, "verify_draft launch")) {
        return KVMEM_HIP_ERR_RUNTIME;
    }
    verify_parts_kernel<<<dim3(pl.n_parts, a->max_draft + 1, a->n_seq), kVerifyThreads, 0, ctx->stream>>>(p);
    // a launch that was not made must not be read by the next
    if (!hip_ok(ctx, hipGetLastError(), "verify_draft launch")) {
        return KVMEM_HIP_ERR_RUNTIME;
    }
    verify_decide_kernel<<<a->n_seq, kVerifyThreads, 0, ctx->stream>>>(p);
    if (a->probs && a->max_draft) {
        if (!hip_ok(ctx, hipGetLastError(), "verify_draft launch")) {
            return KVMEM_HIP_ERR_RUNTIME;
        }
        verify_rest_kernel<<<dim3(pl.n_parts, a->n_seq), kVerifyThreads, 0, ctx->stream>>>(p);
        verify_draw_kernel<<<a->n_seq, kVerifyThreads, 0, ctx->stream>>>(p);
    }
    return hip_ok(ctx, hipGetLastError(), "verify_draft launch") ? KVMEM_HIP_OK : KVMEM_HIP_ERR_RUNTIME;
}

}  // extern "C"
